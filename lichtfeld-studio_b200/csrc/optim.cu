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
constexpr int kCtas8 = 5, kCtas32 = 6;   // CTAs per SM that the registers are shared by
// under 4 KB and under 32 KB of arguments, which is what a launch takes
constexpr int kAdamWFew = 32, kAdamWMany = 384;

constexpr uint32_t kGolden = 0x9E3779B9u, kPlastic = 0xC13FA9A9u, kPlastic2 = 0x91E10DA5u;
constexpr float kTopM = 448.0f, kTopV = 57344.0f;
constexpr float kTiny = 0x1p-110f;   // below it a scale would not be a normal number; such a block is held as zeros

// Two 32-bit operations to an instruction, each rounded as the single one is.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpair(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) { f32x2 r; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }

// A lane's four elements.
struct Block4 {
    float x[4];
    __device__ __forceinline__ f32x2 get(int k) const { return pair(x[2 * k], x[2 * k + 1]); }
    __device__ __forceinline__ void set(int k, f32x2 v) { unpair(v, x[2 * k], x[2 * k + 1]); }
};
__device__ __forceinline__ Block4 times(const Block4& b, float y) {
    Block4 r;
    r.set(0, mul2(b.get(0), pair(y, y)));
    r.set(1, mul2(b.get(1), pair(y, y)));
    return r;
}

// ---- 8-bit codes -------------------------------------------------------------------------------
// Both codes are float32 with a shorter exponent and fraction. Multiplied by 2^-120 (2^-112) their smallest normal number becomes float32's, and below it both are evenly spaced, so a code is the
// upper bits of the scaled value, and rounding adds the threshold to the bits that go.
constexpr float kShiftM = 0x1p-120f, kShiftV = 0x1p-112f;
constexpr int kDroppedM = 20, kDroppedV = 21;

__device__ __forceinline__ Block4 decode4(uint32_t codes, __nv_fp8_interpretation_t kind, float scale) {
    const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xFFFFu), kind)));
    const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), kind)));
    return times(Block4{{lo.x, lo.y, hi.x, hi.y}}, scale);
}
__device__ __forceinline__ Block4 decode_m(uint32_t codes, float scale) { return decode4(codes, __NV_E4M3, scale); }
__device__ __forceinline__ Block4 decode_v(uint32_t codes, float scale) { return decode4(codes, __NV_E5M2, scale); }

__device__ __forceinline__ float max_or_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
// the largest of the warp's numbers, none of them negative; their bits are ordered like the numbers, and NaN above all
__device__ __forceinline__ float warp_max(float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x))); }
__device__ __forceinline__ float finite_or_zero(float x) { return isfinite(x) ? fabsf(x) : 0.0f; }

// The codes of the warp's block, four a lane, and its scale. `e`: the lane's first element; `offset`: the step's part of the thresholds; `nearest`: half a code's distance instead.
template <bool SECOND>
__device__ __forceinline__ uint32_t encode4(const Block4& b, uint32_t e, uint32_t offset, bool nearest, float* scale) {
    constexpr float kTop = SECOND ? kTopV : kTopM, kTopRcp = 1.0f / kTop, kShift = SECOND ? kShiftV : kShiftM;
    constexpr int kDropped = SECOND ? kDroppedV : kDroppedM;
    constexpr uint32_t kStep = SECOND ? kGolden : kPlastic2;
    float most = warp_max(max_or_nan(max_or_nan(fabsf(b.x[0]), fabsf(b.x[1])), max_or_nan(fabsf(b.x[2]), fabsf(b.x[3]))));
    const bool finite = isfinite(most);
    if (!finite) most = warp_max(fmaxf(fmaxf(finite_or_zero(b.x[0]), finite_or_zero(b.x[1])), fmaxf(finite_or_zero(b.x[2]), finite_or_zero(b.x[3]))));
    const bool held = most >= kTiny;
    const float inverse = held ? __fdiv_rn(kTop, most) : 0.0f;
    *scale = held ? __fmul_rn(most, kTopRcp) : 0.0f;
    Block4 y = times(b, inverse);
#pragma unroll
    for (int k = 0; k < 4; ++k) y.x[k] = fminf(fabsf(y.x[k]), kTop);
    y = times(y, kShift);
    uint32_t h = e * kStep + offset, codes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t threshold = nearest ? 1u << (kDropped - 1) : h >> (32 - kDropped);
        codes |= ((__float_as_uint(y.x[k]) + threshold) >> kDropped) << (8 * k);
        h += kStep;
    }
    if (SECOND) {   // what is not zero is not held as zero
        if (held && ((codes - 0x01010101u) & ~codes & 0x80808080u)) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (b.x[k] > 0.0f && !((codes >> (8 * k)) & 0xFF)) codes |= 1u << (8 * k);
        }
    } else {
        const uint32_t lo = __byte_perm(__float_as_uint(b.x[0]), __float_as_uint(b.x[1]), 0x0073), hi = __byte_perm(__float_as_uint(b.x[2]), __float_as_uint(b.x[3]), 0x7300);
        codes |= __byte_perm(lo, hi, 0x7610) & 0x80808080u;
    }
    if (!finite) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t is = isfinite(b.x[k]) ? (codes >> (8 * k)) & 0xFF : SECOND && isinf(b.x[k]) ? 0x7Cu : 0x7Fu;
            codes = (codes & ~(0xFFu << (8 * k))) | is << (8 * k);
        }
    }
    return codes;
}

// ---- memory ------------------------------------------------------------------------------------------
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
__device__ __forceinline__ float fast_root(float x) { float r; asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float fast_reciprocal(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// A lane's part of a block as it lies in memory.
template <int BITS>
struct Raw {
    Block4 p;
    uint4 g;                         // four floats, or four 16-bit numbers in x and y
    Block4 m32, v32;                 // BITS 32
    uint32_t m8, v8;                 // BITS 8
    float ms, vs;
};
__device__ __forceinline__ Block4 gradients(const uint4& g, int dtype) {
    if (dtype == LFS_F32) return {__uint_as_float(g.x), __uint_as_float(g.y), __uint_as_float(g.z), __uint_as_float(g.w)};
    return {half_bits(g.x & 0xFFFFu, dtype), half_bits(g.x >> 16, dtype), half_bits(g.y & 0xFFFFu, dtype), half_bits(g.y >> 16, dtype)};
}
__device__ __forceinline__ uint4 load_grad(const void* src, int dtype, int64_t e, int64_t n, bool whole) {
    if (dtype == LFS_F32) {
        const Block4 g = load4(static_cast<const float*>(src), e, n, whole);
        return make_uint4(__float_as_uint(g.x[0]), __float_as_uint(g.x[1]), __float_as_uint(g.x[2]), __float_as_uint(g.x[3]));
    }
    const uint16_t* h = static_cast<const uint16_t*>(src);
    if (whole) {
        const uint2 w = *reinterpret_cast<const uint2*>(h + e);
        return make_uint4(w.x, w.y, 0, 0);
    }
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = e + k < n ? h[e + k] : 0;
    return make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, 0, 0);
}
template <int BITS>
__device__ __forceinline__ void load_raw(Raw<BITS>& r, const AdamWTensor& T, int64_t start, int64_t e, bool whole) {
    r.p = load4(T.p, e, T.n, whole);
    r.g = load_grad(T.g, T.grad_dtype, e, T.n, whole);
    if constexpr (BITS == 8) {
        r.m8 = load4(static_cast<const uint8_t*>(T.m), e, T.n, whole);
        r.v8 = load4(static_cast<const uint8_t*>(T.v), e, T.n, whole);
        r.ms = T.ms[start / kAdamWBlock];
        r.vs = T.vs[start / kAdamWBlock];
    } else {
        r.m32 = load4(static_cast<const float*>(T.m), e, T.n, whole);
        r.v32 = load4(static_cast<const float*>(T.v), e, T.n, whole);
    }
}

// One warp per block, the next one's loads under way while a block is computed.
template <int CAP, int BITS>
__global__ void __launch_bounds__(256, BITS == 8 ? kCtas8 : kCtas32) adamw_kernel(const __grid_constant__ AdamWArgs<CAP> A) {
    const int lane = threadIdx.x & 31;
    const int warps = (int)(gridDim.x * (blockDim.x >> 5));
    const int total = A.first[A.n];
    int q = (int)(blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)), next = 0;
    if (q >= total) return;
    while (q >= A.first[next + 1]) ++next;
    Raw<BITS> r;
    int64_t start = (int64_t)(q - A.first[next]) * kAdamWBlock;
    load_raw<BITS>(r, A.t[next], start, start + lane * 4, A.t[next].aligned && start + kAdamWBlock <= A.t[next].n);
    for (;;) {
        const AdamWTensor& T = A.t[next];
        const int64_t at = start, e = at + lane * 4;
        const bool whole = T.aligned && at + kAdamWBlock <= T.n;
        Block4 p = r.p, m, v;
        const Block4 g = gradients(r.g, T.grad_dtype);
        if constexpr (BITS == 8) {
            m = decode_m(r.m8, r.ms);
            v = decode_v(r.v8, r.vs);
        } else {
            m = r.m32;
            v = r.v32;
        }
        q += warps;
        const bool more = q < total;
        if (more) {
            while (q >= A.first[next + 1]) ++next;
            start = (int64_t)(q - A.first[next]) * kAdamWBlock;
            load_raw<BITS>(r, A.t[next], start, start + lane * 4, A.t[next].aligned && start + kAdamWBlock <= A.t[next].n);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const f32x2 gs = mul2(g.get(i), pair(A.grad_scale, A.grad_scale));
            const f32x2 m1 = add2(mul2(m.get(i), pair(A.beta1, A.beta1)), mul2(gs, pair(A.one_minus_beta1, A.one_minus_beta1)));
            const f32x2 v1 = add2(mul2(v.get(i), pair(A.beta2, A.beta2)), mul2(mul2(gs, pair(A.one_minus_beta2, A.one_minus_beta2)), gs));
            m.set(i, m1);
            v.set(i, v1);
            // The moments are rounded step by step, since their codes depend on it; the step itself takes the fast root and reciprocal, which are off by 2^-23 of it
            // (exact ones: two thirds more instructions). A denominator is zero or normal: the root of the smallest number is 2^-74.5.
            float a, b;
            unpair(add2(mul2(pair(fast_root(v.x[2 * i]), fast_root(v.x[2 * i + 1])), pair(A.bc2_sqrt_rcp, A.bc2_sqrt_rcp)), pair(A.eps, A.eps)), a, b);
            const f32x2 step = mul2(mul2(m1, pair(T.step_size, T.step_size)), pair(fast_reciprocal(a), fast_reciprocal(b)));
            p.set(i, sub2(mul2(p.get(i), pair(T.decay, T.decay)), step));
        }
        store4(T.p, e, T.n, whole, p);
        if constexpr (BITS == 8) {
            float ms, vs;
            if (!whole)   // what lies behind the tensor's end has no part in the scale
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (e + i >= T.n) m.x[i] = v.x[i] = 0.0f;
            const uint32_t mc = encode4<false>(m, (uint32_t)e, A.offset_m, false, &ms);
            const uint32_t vc = encode4<true>(v, (uint32_t)e, A.offset_v, false, &vs);
            store4(static_cast<uint8_t*>(T.m), e, T.n, whole, mc);
            store4(static_cast<uint8_t*>(T.v), e, T.n, whole, vc);
            if (lane == 0) { T.ms[at / kAdamWBlock] = ms; T.vs[at / kAdamWBlock] = vs; }
        } else {
            store4(static_cast<float*>(T.m), e, T.n, whole, m);
            store4(static_cast<float*>(T.v), e, T.n, whole, v);
        }
        if (!more) return;
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
        const uint32_t c = second ? encode4<true>(x, 0, 0, true, &scale) : encode4<false>(x, 0, 0, true, &scale);
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

// One launch over the tensors of one kind of moments (every tensor of a list, or those that are left when the other kind has been taken out).
template <int CAP, int BITS>
int launch_adamw(int count, const lfs_adamw_tensor* const* tensors, double beta1, double beta2, double eps, int64_t step_count, float grad_scale, cudaStream_t st) {
    static_assert(sizeof(AdamWArgs<CAP>) <= 32764, "kernel arguments");
    // the same host arithmetic as lfs_adam_step_segments
    const double bc1 = 1.0 / (1.0 - std::pow(beta1, (double)step_count));
    const double bc2 = 1.0 / std::sqrt(1.0 - std::pow(beta2, (double)step_count));
    AdamWArgs<CAP> A;
    int64_t blocks = 0;
    A.n = count;
    A.first[0] = 0;
    for (int k = 0; k < count; ++k) {
        const lfs_adamw_tensor& t = *tensors[k];
        AdamWTensor& o = A.t[k];
        o.p = t.param; o.g = t.grad; o.m = t.exp_avg; o.v = t.exp_avg_sq; o.ms = t.exp_avg_scale; o.vs = t.exp_avg_sq_scale;
        o.n = t.n;
        o.step_size = (float)((double)t.lr * bc1);
        o.decay = (float)(1.0 - (double)t.lr * (double)t.weight_decay);
        o.grad_dtype = t.grad_dtype;
        const uintptr_t moment = BITS == 8 ? 4 : 16;
        o.aligned = aligned_by(t.param, 16) && aligned_by(t.grad, 4 * dtype_bytes(t.grad_dtype)) && aligned_by(t.exp_avg, moment) && aligned_by(t.exp_avg_sq, moment);
        blocks += (t.n + kAdamWBlock - 1) / kAdamWBlock;
        if (blocks >= (int64_t)1 << 30) {
            set_error("lfs_adamw_step_tensors: more than 2^37 elements in one launch");
            return LFS_EINVAL;
        }
        A.first[k + 1] = (int32_t)blocks;
    }
    A.beta1 = (float)beta1; A.beta2 = (float)beta2;
    A.one_minus_beta1 = (float)(1.0 - beta1); A.one_minus_beta2 = (float)(1.0 - beta2);
    A.eps = (float)eps; A.bc2_sqrt_rcp = (float)bc2; A.grad_scale = grad_scale;
    A.offset_m = (uint32_t)step_count * kGolden;
    A.offset_v = (uint32_t)step_count * kPlastic;
    LFS_TIMED("adamw", st);
    adamw_kernel<CAP, BITS><<<grid_for(blocks, 8, BITS == 8 ? kCtas8 : kCtas32), 256, 0, st>>>(A);
    return check_launch("adamw");
}
template <int BITS>
int launch_adamw_kind(int n_tensors, const lfs_adamw_tensor* tensors, double beta1, double beta2, double eps, int64_t step_count, float grad_scale, cudaStream_t st) {
    const lfs_adamw_tensor* some[kAdamWMany];
    for (int k = 0; k < n_tensors;) {
        int count = 0;
        for (; k < n_tensors && count < kAdamWMany; ++k)
            if (tensors[k].n > 0 && (tensors[k].exp_avg_scale != nullptr) == (BITS == 8)) some[count++] = tensors + k;
        if (count == 0) continue;
        const int rc = (count <= kAdamWFew ? launch_adamw<kAdamWFew, BITS> : launch_adamw<kAdamWMany, BITS>)(count, some, beta1, beta2, eps, step_count, grad_scale, st);
        if (rc != LFS_OK) return rc;
    }
    return LFS_OK;
}

}  // namespace

int launch_adamw_tensors(int n_tensors, const lfs_adamw_tensor* tensors, double beta1, double beta2, double eps, int64_t step_count, float grad_scale,
                         cudaStream_t st) {
    const int rc = launch_adamw_kind<32>(n_tensors, tensors, beta1, beta2, eps, step_count, grad_scale, st);
    return rc != LFS_OK ? rc : launch_adamw_kind<8>(n_tensors, tensors, beta1, beta2, eps, step_count, grad_scale, st);
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
