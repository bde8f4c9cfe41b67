// AdamW over many tensors, moments in 32 or in 8 bits (optim.cu).
#pragma once

#include "common.cuh"

namespace lfs {

int launch_adamw_tensors(int n_tensors, const lfs_adamw_tensor* tensors, double beta1, double beta2, double eps, int64_t step_count, float grad_scale,
                         cudaStream_t st);
int launch_adamw_encode(int64_t n, const float* values, int second_moment, uint8_t* codes, float* scales, cudaStream_t st);
int launch_adamw_decode(int64_t n, const uint8_t* codes, const float* scales, int second_moment, float* values, cudaStream_t st);

}  // namespace lfs
