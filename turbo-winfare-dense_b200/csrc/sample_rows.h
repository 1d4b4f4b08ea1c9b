// Batched token sampling (sample_rows.cu), internal to the library.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace g4b {

struct SampleRowsArgs {
    const void* logits;        // [rows][stride] of bf16 (0), fp16 (1) or fp32 (2)
    const float* uniform;      // [rows], in [0, 1)
    const float* temperature;  // [rows] or null: 1
    const int32_t* top_k;      // [rows] or null: no bound
    const float* top_p;        // [rows] or null: 1
    const float* min_p;        // [rows] or null: 0
    int32_t* token;            // [rows]
    float* prob;               // [rows] or null
    int32_t* kept;             // [rows] or null
    long long stride;
    int rows, vocab, dtype;
};

constexpr int kSampleRowsVocab = 262144;

cudaError_t sample_rows_launch(const SampleRowsArgs& a, cudaStream_t st);

}  // namespace g4b
