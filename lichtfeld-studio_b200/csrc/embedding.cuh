// Embedding lookup, the sorted order of its indices, and its gradient (embedding.cu).
#pragma once

#include "common.cuh"

namespace lfs {

int launch_embedding_fwd(int64_t n, int64_t rows, int width, const void* table, int table_dtype, const void* indices, int index_bits, float scale,
                         void* out, int out_dtype, cudaStream_t st);

size_t embedding_sort_bytes(int64_t n, int64_t rows);
int launch_embedding_sort(int64_t n, int64_t rows, const void* indices, int index_bits, int32_t* order, int32_t* sorted_rows, void* workspace, cudaStream_t st);

size_t embedding_bwd_bytes(int64_t n, int width);
int launch_embedding_bwd(int64_t n, int64_t rows, int width, const void* v_out, int dtype, const int32_t* order, const int32_t* sorted_rows, double scale,
                         int accumulate, float* v_table, void* workspace, cudaStream_t st);

}  // namespace lfs
