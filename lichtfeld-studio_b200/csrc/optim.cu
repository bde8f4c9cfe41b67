// AdamW over many tensors in one launch:
//   m1 = beta1 m + (1 - beta1) g,  v1 = beta2 v + (1 - beta2) g^2
//   p  = p (1 - lr wd) - lr / (1 - beta1^t) * m1 / (sqrt(v1) / sqrt(1 - beta2^t) + eps)
//
// Moments in 8 bits: a block of 128 elements has one 32-bit scale per moment, the largest magnitude over the largest code; the first moment is
// held as e4m3 (sign, range 2^17.8), the second as e5m2 (range 2^32, so 2^16 of its square root). All arithmetic is in 32 bits; only what is
// written back is rounded, and the update uses the moments before that rounding.
//
// How it is rounded decides whether 8 bits work at all. A second moment changes by 0.1 % a step and its codes are 12 to 25 % apart, so a value that
// is rounded to the nearest code never leaves it (on gradients of changing visibility the moment settled at 1.5 times its mean, and what was rounded to zero took steps
// thousands of times too long). Here element i of step t is rounded down, or up if its fraction of a code's distance plus a threshold reaches one:
//   threshold_m = frac(i r1 + t r0), threshold_v = frac(i r0 + t r2), r0 the golden ratio's fraction, r1 and r2 those of the plastic number's powers
// The multiples of r0 and r2 spread evenly over [0, 1) (Weyl), so over the steps every moment moves by what it should on average, and a run can be
// repeated bit for bit. The second moment is not rounded down to zero, which would leave the next denominator without its history. Same gradients, 6000 steps:
// second moment 0.985 of its mean, path of the parameters 11 % off (the noise of the moments), against nearest codes 1.55 and thousands.
//
// Explicit roundings (no contracted products), so that a code does not depend on how the compiler forms an expression.
#include "optim.cuh"

#include <cmath>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace lfs {

namespace {

constexpr int kAdamWBlock = LFS_ADAMW_BLOCK;   // one warp, four elements a lane
static_assert(kAdamWBlock == 128, "");

struct AdamWTensor {
    float* p;
    const void* g;
    void *m, *v;          // float, or e4m3 and e5m2 codes
    float *ms, *vs;       // scales of the blocks; null with 32-bit moments
    int64_t n;
    float step_size;      // lr / (1 - beta1^t)
    float decay;          // 1 - lr * weight decay
    int32_t grad_dtype;
    int32_t aligned;      // whole vectors can be read and written
};

// A kernel takes its tensors as an argument: nothing is copied to the device or kept there, and a captured launch has its own copy.
template <int CAP>
struct AdamWArgs {
    AdamWTensor t[CAP];
    int32_t first[CAP + 1];   // blocks in front of tensor k
    int32_t n;
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, bc2_sqrt_rcp, grad_scale;
    uint32_t offset_m, offset_v;   // the step's part of the rounding thresholds
};
// under 4 KB and under 32 KB of arguments, which is what a launch takes
constexpr int kAdamWFew = 32, kAdamWMany = 384;

constexpr uint32_t kGolden = 0x9E3779B9u, kPlastic = 0xC13FA9A9u, kPlastic2 = 0x91E10DA5u;
constexpr float kTopM = 448.0f, kTopV = 57344.0f;
constexpr float kTiny = 0x1p-110f;   // below it a scale would not be a normal number; such a block is held as zeros

struct Block4 { float x[4]; };

// ---- 8-bit codes -------------------------------------------------------------------------------
// `a` in [0, top]: its bits, the threshold added to those that go, shifted. Below the lowest binade the codes are evenly spaced: adding its start gives
// the number that spacing as last place, and the code is counted from there.
template <int DROPPED, int LOWEST>
__device__ __forceinline__ uint32_t round_code(float a, uint32_t threshold) {
    constexpr float kLeast = LOWEST == -6 ? 0x1p-6f : 0x1p-14f;
    static_assert(LOWEST == -6 || LOWEST == -14, "");
    const bool small = a < kLeast;
    const float t = small ? __fadd_rn(a, kLeast) : a;
    return ((__float_as_uint(t) + threshold) >> DROPPED) - ((uint32_t)(126 + LOWEST + (small ? 1 : 0)) << (23 - DROPPED));
}
__device__ __forceinline__ uint32_t encode_m(float x, float inverse, uint32_t threshold) {
    if (!isfinite(x)) return 0x7F;
    const uint32_t c = round_code<20, -6>(fminf(__fmul_rn(fabsf(x), inverse), kTopM), threshold);
    return c | ((__float_as_uint(x) >> 24) & 0x80u);
}
__device__ __forceinline__ uint32_t encode_v(float x, float inverse, uint32_t threshold) {
    if (!isfinite(x)) return isinf(x) ? 0x7C : 0x7F;
    const uint32_t c = round_code<21, -14>(fminf(__fmul_rn(fabsf(x), inverse), kTopV), threshold);
    return x > 0.0f && inverse > 0.0f ? max(c, 1u) : c;
}
__device__ __forceinline__ Block4 decode_m(uint32_t codes, float scale) {
    const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xFFFFu), __NV_E4M3)));
    const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3)));
    return {__fmul_rn(lo.x, scale), __fmul_rn(lo.y, scale), __fmul_rn(hi.x, scale), __fmul_rn(hi.y, scale)};
}
__device__ __forceinline__ Block4 decode_v(uint32_t codes, float scale) {
    const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xFFFFu), __NV_E5M2)));
    const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E5M2)));
    return {__fmul_rn(lo.x, scale), __fmul_rn(lo.y, scale), __fmul_rn(hi.x, scale), __fmul_rn(hi.y, scale)};
}
// largest finite magnitude of the warp's block; the bits of numbers that are not negative are ordered like the numbers
__device__ __forceinline__ float block_max(const Block4& b) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) most = max(most, isfinite(b.x[k]) ? __float_as_uint(fabsf(b.x[k])) : 0u);
    return __uint_as_float(__reduce_max_sync(0xffffffffu, most));
}
struct Scaling { float inverse, scale; };
__device__ __forceinline__ Scaling block_scaling(float most, float top, float top_rcp) {
    if (most < kTiny) return {0.0f, 0.0f};
    return {__fdiv_rn(top, most), __fmul_rn(most, top_rcp)};
}
// codes of the warp's block, four a lane. `offset`: the step's part of the thresholds; `nearest`: half a code's distance instead.
__device__ __forceinline__ uint32_t encode_block_m(const Block4& b, uint32_t e, uint32_t offset, bool nearest, float* scale) {
    const Scaling s = block_scaling(block_max(b), kTopM, 1.0f / kTopM);
    *scale = s.scale;
    uint32_t codes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) codes |= encode_m(b.x[k], s.inverse, nearest ? 1u << 19 : ((e + k) * kPlastic2 + offset) >> 12) << (8 * k);
    return codes;
}
__device__ __forceinline__ uint32_t encode_block_v(const Block4& b, uint32_t e, uint32_t offset, bool nearest, float* scale) {
    const Scaling s = block_scaling(block_max(b), kTopV, 1.0f / kTopV);
    *scale = s.scale;
    uint32_t codes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) codes |= encode_v(b.x[k], s.inverse, nearest ? 1u << 20 : ((e + k) * kGolden + offset) >> 11) << (8 * k);
    return codes;
}

// ---- a lane's four elements ----------------------------------------------------------------------
__device__ __forceinline__ Block4 load4(const float* src, int64_t e, int64_t n, bool whole) {
    if (whole) {
        const float4 a = *reinterpret_cast<const float4*>(src + e);
        return {a.x, a.y, a.z, a.w};
    }
    Block4 b;
#pragma unroll
    for (int k = 0; k < 4; ++k) b.x[k] = e + k < n ? src[e + k] : 0.0f;
    return b;
}
__device__ __forceinline__ void store4(float* dst, int64_t e, int64_t n, bool whole, const Block4& b) {
    if (whole) {
        *reinterpret_cast<float4*>(dst + e) = make_float4(b.x[0], b.x[1], b.x[2], b.x[3]);
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (e + k < n) dst[e + k] = b.x[k];
}
__device__ __forceinline__ uint32_t load4(const uint8_t* src, int64_t e, int64_t n, bool whole) {
    if (whole) return *reinterpret_cast<const uint32_t*>(src + e);
    uint32_t codes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (e + k < n) codes |= (uint32_t)src[e + k] << (8 * k);
    return codes;
}
__device__ __forceinline__ void store4(uint8_t* dst, int64_t e, int64_t n, bool whole, uint32_t codes) {
    if (whole) {
        *reinterpret_cast<uint32_t*>(dst + e) = codes;
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (e + k < n) dst[e + k] = (uint8_t)(codes >> (8 * k));
}
__device__ __forceinline__ float half_bits(uint32_t bits, int dtype) {
    return dtype == LFS_BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half((unsigned short)bits));
}
__device__ __forceinline__ Block4 load_grad(const void* src, int dtype, int64_t e, int64_t n, bool whole) {
    if (dtype == LFS_F32) return load4(static_cast<const float*>(src), e, n, whole);
    const uint16_t* h = static_cast<const uint16_t*>(src);
    if (whole) {
        const uint2 w = *reinterpret_cast<const uint2*>(h + e);
        return {half_bits(w.x & 0xFFFFu, dtype), half_bits(w.x >> 16, dtype), half_bits(w.y & 0xFFFFu, dtype), half_bits(w.y >> 16, dtype)};
    }
    Block4 b;
#pragma unroll
    for (int k = 0; k < 4; ++k) b.x[k] = e + k < n ? half_bits(h[e + k], dtype) : 0.0f;
    return b;
}

template <int CAP>
__global__ void __launch_bounds__(256) adamw_kernel(const __grid_constant__ AdamWArgs<CAP> A) {
    const int lane = threadIdx.x & 31;
    const int warps = (int)(gridDim.x * (blockDim.x >> 5));
    const int total = A.first[A.n];
    int k = 0;
    for (int q = (int)(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)); q < total; q += warps) {
        while (q >= A.first[k + 1]) ++k;
        const AdamWTensor& T = A.t[k];
        const int64_t start = (int64_t)(q - A.first[k]) * kAdamWBlock, e = start + lane * 4;
        const bool whole = T.aligned && start + kAdamWBlock <= T.n;
        Block4 p = load4(T.p, e, T.n, whole);
        const Block4 g = load_grad(T.g, T.grad_dtype, e, T.n, whole);
        Block4 m, v;
        if (T.ms) {
            const int64_t b = start / kAdamWBlock;
            m = decode_m(load4(static_cast<const uint8_t*>(T.m), e, T.n, whole), T.ms[b]);
            v = decode_v(load4(static_cast<const uint8_t*>(T.v), e, T.n, whole), T.vs[b]);
        } else {
            m = load4(static_cast<const float*>(T.m), e, T.n, whole);
            v = load4(static_cast<const float*>(T.v), e, T.n, whole);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float gs = __fmul_rn(g.x[i], A.grad_scale);
            m.x[i] = __fadd_rn(__fmul_rn(m.x[i], A.beta1), __fmul_rn(gs, A.one_minus_beta1));
            v.x[i] = __fadd_rn(__fmul_rn(v.x[i], A.beta2), __fmul_rn(__fmul_rn(gs, A.one_minus_beta2), gs));
            const float denom = __fadd_rn(__fmul_rn(__fsqrt_rn(v.x[i]), A.bc2_sqrt_rcp), A.eps);
            p.x[i] = __fsub_rn(__fmul_rn(p.x[i], T.decay), __fdiv_rn(__fmul_rn(m.x[i], T.step_size), denom));
        }
        store4(T.p, e, T.n, whole, p);
        if (T.ms) {
            const int64_t b = start / kAdamWBlock;
            float ms, vs;
            if (!whole)   // what lies behind the tensor's end has no part in the scale (0/0 above where eps is zero)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (e + i >= T.n) m.x[i] = v.x[i] = 0.0f;
            const uint32_t mc = encode_block_m(m, (uint32_t)e, A.offset_m, false, &ms);
            const uint32_t vc = encode_block_v(v, (uint32_t)e, A.offset_v, false, &vs);
            store4(static_cast<uint8_t*>(T.m), e, T.n, whole, mc);
            store4(static_cast<uint8_t*>(T.v), e, T.n, whole, vc);
            if (lane == 0) { T.ms[b] = ms; T.vs[b] = vs; }
        } else {
            store4(static_cast<float*>(T.m), e, T.n, whole, m);
            store4(static_cast<float*>(T.v), e, T.n, whole, v);
        }
    }
}

__global__ void __launch_bounds__(256) adamw_encode_kernel(int64_t n, int64_t blocks, const float* __restrict__ values, int second, bool aligned,
                                                           uint8_t* __restrict__ codes, float* __restrict__ scales) {
    const int lane = threadIdx.x & 31;
    for (int64_t b = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); b < blocks; b += (int64_t)gridDim.x * 8) {
        const int64_t e = b * kAdamWBlock + lane * 4;
        const bool whole = aligned && (b + 1) * kAdamWBlock <= n;
        const Block4 x = load4(values, e, n, whole);
        float scale;
        const uint32_t c = second ? encode_block_v(x, 0, 0, true, &scale) : encode_block_m(x, 0, 0, true, &scale);
        store4(codes, e, n, whole, c);
        if (lane == 0) scales[b] = scale;
    }
}

__global__ void __launch_bounds__(256) adamw_decode_kernel(int64_t n, int64_t blocks, const uint8_t* __restrict__ codes, const float* __restrict__ scales,
                                                           int second, bool aligned, float* __restrict__ values) {
    const int lane = threadIdx.x & 31;
    for (int64_t b = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); b < blocks; b += (int64_t)gridDim.x * 8) {
        const int64_t e = b * kAdamWBlock + lane * 4;
        const bool whole = aligned && (b + 1) * kAdamWBlock <= n;
        const uint32_t c = load4(codes, e, n, whole);
        store4(values, e, n, whole, second ? decode_v(c, scales[b]) : decode_m(c, scales[b]));
    }
}

template <int CAP>
int launch_adamw(int count, const lfs_adamw_tensor* tensors, double beta1, double beta2, double eps, int64_t step_count, float grad_scale, cudaStream_t st) {
    static_assert(sizeof(AdamWArgs<CAP>) <= 32764, "kernel arguments");
    // the same host arithmetic as lfs_adam_step_segments
    const double bc1 = 1.0 / (1.0 - std::pow(beta1, (double)step_count));
    const double bc2 = 1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step_count));
    AdamWArgs<CAP> A;
    int64_t blocks = 0;
    A.n = 0;
    A.first[0] = 0;
    for (int k = 0; k < count; ++k) {
        const lfs_adamw_tensor& t = tensors[k];
        if (t.n == 0) continue;
        AdamWTensor& o = A.t[A.n];
        o.p = t.param; o.g = t.grad; o.m = t.exp_avg; o.v = t.exp_avg_sq; o.ms = t.exp_avg_scale; o.vs = t.exp_avg_sq_scale;
        o.n = t.n;
        o.step_size = (float)((double)t.lr * bc1);
        o.decay = (float)(1.0 - (double)t.lr * (double)t.weight_decay);
        o.grad_dtype = t.grad_dtype;
        const uintptr_t moment = t.exp_avg_scale ? 4 : 16;
        o.aligned = aligned_by(t.param, 16) && aligned_by(t.grad, 4 * dtype_bytes(t.grad_dtype)) && aligned_by(t.exp_avg, moment) && aligned_by(t.exp_avg_sq, moment);
        blocks += (t.n + kAdamWBlock - 1) / kAdamWBlock;
        if (blocks >= (int64_t)1 << 30) {
            set_error("lfs_adamw_step_tensors: more than 2^37 elements in one launch");
            return LFS_EINVAL;
        }
        A.first[++A.n] = (int32_t)blocks;
    }
    if (blocks == 0) return LFS_OK;
    A.beta1 = (float)beta1; A.beta2 = (float)beta2;
    A.one_minus_beta1 = (float)(1.0 - beta1); A.one_minus_beta2 = (float)(1.0 - beta2);
    A.eps = (float)eps; A.bc2_sqrt_rcp = (float)bc2; A.grad_scale = grad_scale;
    A.offset_m = (uint32_t)step_count * kGolden;
    A.offset_v = (uint32_t)step_count * kPlastic;
    LFS_TIMED("adamw", st);
    adamw_kernel<CAP><<<grid_for(blocks, 8, 8), 256, 0, st>>>(A);
    return check_launch("adamw");
}

}  // namespace

int launch_adamw_tensors(int n_tensors, const lfs_adamw_tensor* tensors, double beta1, double beta2, double eps, int64_t step_count, float grad_scale,
                         cudaStream_t st) {
    for (int k = 0; k < n_tensors;) {
        const int count = n_tensors - k < kAdamWMany ? n_tensors - k : kAdamWMany;
        const int rc = (count <= kAdamWFew ? launch_adamw<kAdamWFew> : launch_adamw<kAdamWMany>)(count, tensors + k, beta1, beta2, eps, step_count, grad_scale, st);
        if (rc != LFS_OK) return rc;
        k += count;
    }
    return LFS_OK;
}

int launch_adamw_encode(int64_t n, const float* values, int second_moment, uint8_t* codes, float* scales, cudaStream_t st) {
    if (n == 0) return LFS_OK;
    const int64_t blocks = (n + kAdamWBlock - 1) / kAdamWBlock;
    LFS_TIMED("adamw_state_encode", st);
    adamw_encode_kernel<<<grid_for(blocks, 8), 256, 0, st>>>(n, blocks, values, second_moment, aligned_by(values, 16) && aligned_by(codes, 4), codes, scales);
    return check_launch("adamw_state_encode");
}
int launch_adamw_decode(int64_t n, const uint8_t* codes, const float* scales, int second_moment, float* values, cudaStream_t st) {
    if (n == 0) return LFS_OK;
    const int64_t blocks = (n + kAdamWBlock - 1) / kAdamWBlock;
    LFS_TIMED("adamw_state_decode", st);
    adamw_decode_kernel<<<grid_for(blocks, 8), 256, 0, st>>>(n, blocks, codes, scales, second_moment, aligned_by(values, 16) && aligned_by(codes, 4), values);
    return check_launch("adamw_state_decode");
}

}  // namespace lfs
