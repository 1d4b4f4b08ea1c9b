// Launchers of the paged-cache operators (pages.cu), internal to the library.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace g4b {

// A pool of pages on the device: `planes` parallel planes (one per layer's K and V), each holding
// `pages` pages of `page_size` rows. Strides in bytes; a page's rows are contiguous.
struct PagePool {
    char* base;
    long long plane_stride, page_stride;
    int planes, pages, page_size, row_bytes;
};

// The page keeping of a set of sequences: reference counts per page, a block table row and a
// length per sequence. Inputs and outputs may be the same arrays.
struct PageTables {
    const int32_t* refs;
    const int32_t* table;
    const int32_t* lens;
    int32_t* refs_out;
    int32_t* table_out;
    int32_t* lens_out;
    int pages, seqs, width, page_size;
};

constexpr int kMaxPageSeqs = 4096;  // sequences one page-keeping call handles (shared-memory prefix sums)

cudaError_t pages_reserve(const PageTables& t, const int32_t* grow, int32_t* status, cudaStream_t st);
cudaError_t pages_free(const PageTables& t, const int32_t* seqs, int n, cudaStream_t st);
cudaError_t pages_fork(const PagePool& pool, const PageTables& t, const int32_t* src, const int32_t* dst, int n,
                       int32_t* status, cudaStream_t st);
cudaError_t pages_compact(const PagePool& pool, const PageTables& t, int32_t* moves, cudaStream_t st);
cudaError_t pages_copy(const PagePool& from, const PagePool& to, const int32_t* src, const int32_t* dst, int n,
                       cudaStream_t st);
cudaError_t pages_commit(const PagePool& pool, const int32_t* table, int width, const int32_t* lens, int seqs,
                         const char* rows, long long rows_plane_stride, int n_tokens, const int32_t* cu_nodes,
                         const int32_t* path, int path_width, const int32_t* count, const int32_t* status,
                         int32_t* lens_out, cudaStream_t st);

// tree.cu
cudaError_t tree_accept(const int32_t* tokens, const int32_t* parents, const int32_t* sampled,
                        const int32_t* cu_nodes, int seqs, int n_tokens, int32_t* path, int path_width,
                        int32_t* count, int32_t* next, cudaStream_t st);

}  // namespace g4b
