// Attention of drafted token trees over a paged K/V cache (tree_attn.cu), internal to the library.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

namespace g4b {

struct TreeAttnArgs {
    const void* q;          // [n_tokens][heads][dim], token stride q_stride elements
    const void* k_pool;     // [pages][page_size][kv_heads][dim], page stride page_stride elements
    const void* v_pool;
    const void* k_new;      // [n_tokens][kv_heads][dim], token stride new_stride elements
    const void* v_new;
    void* out;              // [n_tokens][heads][dim], token stride out_stride elements
    const int32_t* table;   // [seqs][width] page ids
    const int32_t* lens;    // [seqs] cached tokens
    const int32_t* cu;      // [seqs + 1] first node of each sequence
    const uint32_t* mask;   // [n_tokens][mask_words]
    const int32_t* depth;   // [n_tokens], read when window > 0
    void* work;
    long long q_stride, page_stride, new_stride, out_stride;
    int seqs, n_tokens, max_nodes, pages, page_size, width, mask_words, heads, kv_heads, dim, window;
    bool bf16;
    float scale;
};

size_t tree_attn_workspace(int max_nodes, int heads, int kv_heads, int dim);
bool tree_attn_countable(const TreeAttnArgs& a);  // whether 32 bits count the tiles of all sequences and heads
cudaError_t tree_attn_launch(const TreeAttnArgs& a, cudaStream_t st);
int tree_attn_error();  // synchronizes; nonzero when a bounded wait gave up since the last call

}  // namespace g4b
