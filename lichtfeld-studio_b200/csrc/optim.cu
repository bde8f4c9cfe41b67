// AdamW over many tensors in one launch:
//   m1 = beta1 m + (1 - beta1) g,  v1 = beta2 v + (1 - beta2) g^2
//   p  = p (1 - lr wd) - lr / (1 - beta1^t) * m1 / (sqrt(v1) / sqrt(1 - beta2^t) + eps)
//
// Moments in 8 bits: a block of 128 elements has one 32-bit scale per moment, the largest magnitude over the largest code; the first moment is
// held as e4m3 (sign, range 2^17.8), the second as e5m2 (range 2^32, so 2^16 of its square root). All arithmetic is in 32 bits; only what is
// written back is rounded, and the update uses the moments before that rounding.
//
// How it is rounded decides whether 8 bits work at all. A second moment changes by 0.1 % a step and its codes are 12 to 25 % apart, so a value that
// is rounded to the nearest code leaves it only as far as the block's scale moves (gradients that halve beside a steady largest one: the moment stays at 4.1 times its value), and what is rounded to zero
// takes its next steps without a denominator. Here element i of step t is rounded down, or up if its fraction of a code's distance plus a threshold reaches one:
//   threshold_m = frac(i r1 + t r0), threshold_v = frac(i r0 + t r2), t the tensor's own step number, r0 the golden ratio's fraction, r1 and r2 those of the plastic number's powers
// The multiples of r0 and r2 spread evenly over [0, 1) (Weyl), so over the steps every moment moves by what it should on average, and a run can be
// repeated bit for bit. The second moment is not rounded down to zero, which would leave the next denominator without its history. 6000 steps
// of gradients that are there in half of them and become five times smaller: second moments 0.99 of their own on average, path of the parameters 11 % off (the noise of the moments); nearest codes 1.07 to 1.6, and from
// 20 % to thousands of times, by the numbers drawn. Beside a steady largest one: 0.985, 6 %. (tests/test_gpu_adamw_step.py)
//
// Explicit roundings (no contracted products), so that a code does not depend on how the compiler forms an expression.
#include "optim.cuh"

#include <algorithm>
#include <atomic>
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
    uint32_t n;
    uint32_t flags;       // the gradient's type, kAligned, and in kBefore the elements in front of these where a tensor is longer than kPiece, modulo 2^32
    float step_size;      // lr / (1 - beta1^t)
    float decay;          // 1 - lr * weight decay
    float bc2_sqrt_rcp;   // 1 / sqrt(1 - beta2^t)
    uint32_t t;           // this tensor's step number, modulo 2^32

    __device__ __forceinline__ int grad_dtype() const { return (int)(flags & 3u); }
    __device__ __forceinline__ bool aligned() const { return (flags & 4u) != 0; }
    __device__ __forceinline__ uint32_t before() const { return flags & 0xC0000000u; }
};
constexpr uint32_t kAligned = 4;   // whole vectors can be read and written
constexpr int64_t kPiece = (int64_t)1 << 30;
static_assert(LFS_F32 < 4 && LFS_BF16 < 4 && LFS_F16 < 4, "");

// A kernel takes its tensors as an argument: nothing is copied to the device or kept there, and a captured launch has its own copy.
template <int CAP>
struct AdamWArgs {
    AdamWTensor t[CAP];
    int32_t first[CAP + 1];   // tiles in front of tensor k
    int32_t n;
    float beta1, beta2, one_minus_beta1, one_minus_beta2, eps, grad_scale, minus_zero;
};
// under 4, 10 and 32 KB of arguments, the most that a launch takes (a step of 40 small tensors 6.4 us with 10 KB and 8.1 with 32)
constexpr int kAdamWFew = 32, kAdamWSome = 128, kAdamWMany = 424;

// A CTA takes a tile of kTile elements at a time, kBlocks blocks to a warp, with the next ones being copied to shared memory.
constexpr int kWarps = 8, kThreads = kWarps * 32, kBlocks = 2, kRow = kWarps * kAdamWBlock, kTile = kBlocks * kRow;
constexpr int kStages = 2, kCtas8 = 4, kCtas32 = 3;

constexpr uint32_t kGolden = 0x9E3779B9u, kPlastic = 0xC13FA9A9u, kPlastic2 = 0x91E10DA5u;
constexpr float kTopM = 448.0f, kTopV = 57344.0f;
constexpr float kTiny = 0x1p-110f;   // below it a scale would not be a normal number; such a block is held as zeros
constexpr float kNormal = 0x1p-126f;   // the scale of such a block if it has infinities

// Two 32-bit operations to an instruction, each rounded as the single one is.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpair(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) { f32x2 r; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// A product that is added to something and has to be rounded before that. A packed product and the sum behind it become one operation in spite of their .rn and of --fmad=false, and so
// do a sum with a constant zero and what follows, so the zero (-0, which changes nothing) comes from the arguments.
__device__ __forceinline__ f32x2 mul2_alone(f32x2 a, f32x2 b, f32x2 minus_zero) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(minus_zero));
    return r;
}

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
__device__ __forceinline__ float max4(const Block4& b) {
    return max_or_nan(max_or_nan(fabsf(b.x[0]), fabsf(b.x[1])), max_or_nan(fabsf(b.x[2]), fabsf(b.x[3])));
}
// the largest of the warp's numbers, none of them negative; their bits are ordered like the numbers, and NaN above all
__device__ __forceinline__ float warp_max(float x) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x))); }

struct Scaling { float inverse, scale; };
template <bool SECOND>
__device__ __forceinline__ Scaling scaling(float most) {
    constexpr float kTop = SECOND ? kTopV : kTopM, kTopRcp = 1.0f / kTop;
    const bool held = most >= kTiny;
    return {held ? __fdiv_rn(kTop, most) : 0.0f, held ? __fmul_rn(most, kTopRcp) : 0.0f};
}
// A lane's four codes. `e`: its first element; `offset`: the step's part of the thresholds; `nearest`: half a code's distance instead. What is not finite is left to the caller.
template <bool SECOND>
__device__ __forceinline__ uint32_t encode4(const Block4& b, float inverse, uint32_t e, uint32_t offset, bool nearest) {
    constexpr float kTop = SECOND ? kTopV : kTopM, kShift = SECOND ? kShiftV : kShiftM;
    constexpr int kDropped = SECOND ? kDroppedV : kDroppedM;
    constexpr uint32_t kStep = SECOND ? kGolden : kPlastic2;
    Block4 y = times(b, inverse);
#pragma unroll
    for (int k = 0; k < 4; ++k) y.x[k] = fminf(fabsf(y.x[k]), kTop);
    y = times(y, kShift);
    uint32_t h = e * kStep + offset, c[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        c[k] = (__float_as_uint(y.x[k]) + (nearest ? 1u << (kDropped - 1) : h >> (32 - kDropped))) >> kDropped;
        h += kStep;
    }
    uint32_t codes = (c[0] | c[1] << 8) | (c[2] | c[3] << 8) << 16;
    if (SECOND) {   // what is not zero is not held as zero
        if (((codes - 0x01010101u) & ~codes & 0x80808080u) && inverse > 0.0f) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (b.x[k] > 0.0f && !((codes >> (8 * k)) & 0xFF)) codes |= 1u << (8 * k);
        }
    } else {
        const uint32_t lo = __byte_perm(__float_as_uint(b.x[0]), __float_as_uint(b.x[1]), 0x0073), hi = __byte_perm(__float_as_uint(b.x[2]), __float_as_uint(b.x[3]), 0x7300);
        codes |= __byte_perm(lo, hi, 0x7610) & 0x80808080u;
    }
    return codes;
}
template <bool SECOND>
__device__ __forceinline__ uint32_t encode_block(const Block4& b, uint32_t e, uint32_t offset, bool nearest, float* scale) {
    // the scale of a block is that of its finite numbers alone
    const bool finite = isfinite(warp_max(max4(b)));
    Block4 f = b;
    if (!finite)
#pragma unroll
        for (int k = 0; k < 4; ++k) f.x[k] = isfinite(b.x[k]) ? b.x[k] : 0.0f;
    const Scaling s = scaling<SECOND>(warp_max(max4(f)));
    *scale = !finite && s.scale == 0.0f ? kNormal : s.scale;   // infinity times zero would not be infinite
    uint32_t codes = encode4<SECOND>(f, s.inverse, e, offset, nearest);
    if (!finite)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (!isfinite(b.x[k])) codes = (codes & ~(0xFFu << (8 * k))) | (SECOND && isinf(b.x[k]) ? 0x7Cu : 0x7Fu) << (8 * k);
    return codes;
}

// Both moments of the warp's block. The scale is the first moment's in the lower half of the warp and the second's in the upper one, so that one division makes both.
struct Codes { uint32_t m, v; float scale; };
__device__ __noinline__ Codes encode_not_finite(Block4 m, Block4 v, uint32_t e, uint32_t offset_m, uint32_t offset_v) {
    Codes c;
    float ms, vs;
    c.m = encode_block<false>(m, e, offset_m, false, &ms);
    c.v = encode_block<true>(v, e, offset_v, false, &vs);
    c.scale = threadIdx.x & 16 ? vs : ms;
    return c;
}
__device__ __forceinline__ Codes encode_moments(const Block4& m, const Block4& v, uint32_t e, uint32_t offset_m, uint32_t offset_v) {
    const float most_m = warp_max(max4(m)), most_v = warp_max(max4(v));
    if (!isfinite(max_or_nan(most_m, most_v))) return encode_not_finite(m, v, e, offset_m, offset_v);
    const bool upper = threadIdx.x & 16;
    const float most = upper ? most_v : most_m;
    const bool held = most >= kTiny;
    const float inverse = held ? __fdiv_rn(upper ? kTopV : kTopM, most) : 0.0f;
    Codes c;
    c.m = encode4<false>(m, __shfl_sync(0xffffffffu, inverse, 0), e, offset_m, false);
    c.v = encode4<true>(v, __shfl_sync(0xffffffffu, inverse, 16), e, offset_v, false);
    c.scale = held ? __fmul_rn(most, upper ? 1.0f / kTopV : 1.0f / kTopM) : 0.0f;
    return c;
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
// (numbers below the normal ones included: beside an eps of 1e-15 the root of 2^-126 is 2e-4)
__device__ __forceinline__ float fast_root(float x) { float r; asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float fast_reciprocal(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// The same rounded once. Very small operands take the approximations, since root and division of CUDA leave their short path for them: first moments of rows that have not been seen for some hundreds of steps
// are below the normal numbers, and a step of 59 M elements then took 311 us instead of 270.
constexpr float kShortPath = 0x1p-100f;
__device__ __forceinline__ float root(float x) {
    const bool tiny = x < kShortPath;
    const float r = __fsqrt_rn(tiny ? 1.0f : x);
    return tiny ? fast_root(x) : r;
}
__device__ __forceinline__ float quotient(float a, float b) {
    const bool tiny = fabsf(a) < kShortPath;
    const float q = __fdiv_rn(tiny ? 1.0f : a, b);
    return tiny ? __fmul_rn(a, fast_reciprocal(b)) : q;
}

struct Step {
    float grad_scale, beta1, beta2, one_minus_beta1, one_minus_beta2, bc2_sqrt_rcp, eps, minus_zero, step_size, decay;
};
// FAST: the step takes the approximate root and reciprocal, off by 2^-23 of it each. With 32-bit moments both are rounded once, which costs nothing there to 1.5 % (59 M elements 258 us either way, 266 and 270 in a
// long run; 400 small tensors 5.5). With 8-bit moments, which are themselves 2^-5 and more off, they would add half to the time (177 M elements 725 us against 480 to 520, 4.6 M 27.7 against 20.7).
template <bool FAST>
__device__ __forceinline__ void update(Block4& p, Block4& m, Block4& v, const Block4& g, const Step& S) {
    const f32x2 zero = pair(S.minus_zero, S.minus_zero);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f32x2 gs = mul2(g.get(i), pair(S.grad_scale, S.grad_scale));
        const f32x2 m1 = add2(mul2_alone(m.get(i), pair(S.beta1, S.beta1), zero), mul2_alone(gs, pair(S.one_minus_beta1, S.one_minus_beta1), zero));
        const f32x2 v1 = add2(mul2_alone(v.get(i), pair(S.beta2, S.beta2), zero), mul2_alone(mul2(gs, pair(S.one_minus_beta2, S.one_minus_beta2)), gs, zero));
        m.set(i, m1);
        v.set(i, v1);
        // The moments are rounded step by step, since their codes depend on it.
        // A denominator is zero or normal: the root of the smallest number is 2^-74.5, and an eps below 2^-126 is refused.
        const float v0 = v.x[2 * i], v2 = v.x[2 * i + 1];
        const f32x2 roots = FAST ? pair(fast_root(v0), fast_root(v2)) : pair(root(v0), root(v2));
        const f32x2 denominator = add2(mul2(roots, pair(S.bc2_sqrt_rcp, S.bc2_sqrt_rcp)), pair(S.eps, S.eps)), numerator = mul2(m1, pair(S.step_size, S.step_size));
        float a, b;
        unpair(denominator, a, b);
        f32x2 step;
        if constexpr (FAST) {
            step = mul2(numerator, pair(fast_reciprocal(a), fast_reciprocal(b)));
        } else {
            float c, d;
            unpair(numerator, c, d);
            step = pair(quotient(c, a), quotient(d, b));
        }
        p.set(i, sub2(mul2(p.get(i), pair(S.decay, S.decay)), step));
    }
}

// A warp's block of a tile that is not whole, or of a tensor that cannot be read in vectors.
template <int BITS>
__device__ __noinline__ void single_block(const AdamWTensor& T, uint32_t start, int lane, const Step& S) {
    const int64_t e = (int64_t)start + lane * 4, n = T.n;
    const bool whole = T.aligned() && start + kAdamWBlock <= T.n;
    Block4 p = load4(T.p, e, n, whole), g, m, v;
    if (T.grad_dtype() == LFS_F32) g = load4(static_cast<const float*>(T.g), e, n, whole);
    else
#pragma unroll
        for (int k = 0; k < 4; ++k) g.x[k] = e + k < n ? half_bits(static_cast<const uint16_t*>(T.g)[e + k], T.grad_dtype()) : 0.0f;
    if constexpr (BITS == 8) {
        m = decode_m(load4(static_cast<const uint8_t*>(T.m), e, n, whole), T.ms[start / kAdamWBlock]);
        v = decode_v(load4(static_cast<const uint8_t*>(T.v), e, n, whole), T.vs[start / kAdamWBlock]);
    } else {
        m = load4(static_cast<const float*>(T.m), e, n, whole);
        v = load4(static_cast<const float*>(T.v), e, n, whole);
    }
    update<BITS == 8>(p, m, v, g, S);
    store4(T.p, e, n, whole, p);
    if constexpr (BITS == 8) {
        // what lies behind the tensor's end has no part in the scale
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (e + k >= n) m.x[k] = v.x[k] = 0.0f;
        const Codes c = encode_moments(m, v, T.before() + (uint32_t)e, T.t * kGolden, T.t * kPlastic);
        store4(static_cast<uint8_t*>(T.m), e, n, whole, c.m);
        store4(static_cast<uint8_t*>(T.v), e, n, whole, c.v);
        if ((lane & 15) == 0) (lane ? T.vs : T.ms)[start / kAdamWBlock] = c.scale;
    } else {
        store4(static_cast<float*>(T.m), e, n, whole, m);
        store4(static_cast<float*>(T.v), e, n, whole, v);
    }
}

// the tensor of tile q, which is not in front of tensor k's
template <int CAP>
__device__ __forceinline__ int tensor_of(const AdamWArgs<CAP>& A, int q, int k) {
    if (CAP == kAdamWFew) {
        while (q >= A.first[k + 1]) ++k;
        return k;
    }
    if (q < A.first[k + 1]) return k;
    int lo = k + 1, hi = A.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (q < A.first[mid + 1]) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__device__ __forceinline__ void copy16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
// A tile as it lies in memory; 16-bit gradients fill the first half of g.
struct Stage {
    float p[kTile], g[kTile];
    uint8_t m[kTile], v[kTile];
    float ms[kTile / kAdamWBlock], vs[kTile / kAdamWBlock];
};
static_assert(kThreads * 4 == kRow && kTile % (8 * kThreads) == 0, "whole copies of 16 bytes a thread");

// Moments in 8 bits. Issue slots and memory are both near their limits (65 instructions for 16 bytes; 66 % of both), so the copies are wide and asynchronous: loads straight into registers wait for one another at every
// block and cost more instructions for their addresses. us for 3 M Gaussians at SH degree 3 (177 M elements): simple 1018, codes from scaled bits 755, the next block's loads under way 592, tiles copied
// ahead 515, one division and one check for both moments 459 to 510 by the GPU and the run (86 to 96 % of the copy rate). In a long run, where the clock is lower, 503 to 534 (82 to 88 %).
template <int CAP>
__global__ void __launch_bounds__(kThreads, kCtas8) adamw8_kernel(const __grid_constant__ AdamWArgs<CAP> A) {
    extern __shared__ __align__(128) char stages_s[];
    Stage* const stages = reinterpret_cast<Stage*>(stages_s);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = threadIdx.x;
    const int total = A.first[A.n];

    int ahead = 0;   // tensor of the tile whose copies are issued
    auto issue = [&](int q, Stage& s) {
        if (q < total) {
            ahead = tensor_of(A, q, ahead);
            const AdamWTensor& T = A.t[ahead];
            const uint32_t start = (uint32_t)(q - A.first[ahead]) * kTile;
            if (T.aligned() && start + kTile <= T.n) {
                const float* p = T.p + start + t * 4;
#pragma unroll
                for (int k = 0; k < kBlocks; ++k) copy16(&s.p[k * kRow + t * 4], p + k * kRow);
                if (T.grad_dtype() == LFS_F32) {
                    const float* g = static_cast<const float*>(T.g) + start + t * 4;
#pragma unroll
                    for (int k = 0; k < kBlocks; ++k) copy16(&s.g[k * kRow + t * 4], g + k * kRow);
                } else {
#pragma unroll
                    for (int k = 0; k < kTile / 8 / kThreads; ++k) copy16(&s.g[(k * kThreads + t) * 4], static_cast<const uint16_t*>(T.g) + start + (k * kThreads + t) * 8);
                }
#pragma unroll
                for (int k = 0; k < kTile / 8 / kThreads; ++k) {
                    const int piece = k * kThreads + t, of = piece % (kTile / 16) * 16;
                    if (piece < kTile / 16) copy16(&s.m[of], static_cast<const uint8_t*>(T.m) + start + of);
                    else copy16(&s.v[of], static_cast<const uint8_t*>(T.v) + start + of);
                }
                constexpr int kScales = kTile / kAdamWBlock / 4;
                if (t < kScales) copy16(&s.ms[t * 4], T.ms + start / kAdamWBlock + t * 4);
                else if (t < 2 * kScales) copy16(&s.vs[(t - kScales) * 4], T.vs + start / kAdamWBlock + (t - kScales) * 4);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int k = 0; k < kStages - 1; ++k) issue(blockIdx.x + k * gridDim.x, stages[k]);
    int now = 0, stage = 0;
    for (int q = blockIdx.x; q < total; q += gridDim.x) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncthreads();   // everybody's copies of this tile are there, and everybody is done with the stage that is filled next
        issue(q + (kStages - 1) * gridDim.x, stages[stage == 0 ? kStages - 1 : stage - 1]);
        const Stage& s = stages[stage];
        stage = stage + 1 == kStages ? 0 : stage + 1;
        now = tensor_of(A, q, now);
        const AdamWTensor& T = A.t[now];
        const Step S{A.grad_scale, A.beta1, A.beta2, A.one_minus_beta1, A.one_minus_beta2, T.bc2_sqrt_rcp, A.eps, A.minus_zero, T.step_size, T.decay};
        const uint32_t tile = (uint32_t)(q - A.first[now]) * kTile;
        if (!(T.aligned() && tile + kTile <= T.n)) {
            for (uint32_t start = tile + warp * kAdamWBlock; start < min(tile + kTile, T.n); start += kRow) single_block<8>(T, start, lane, S);
            continue;
        }
        const uint32_t e0 = tile + t * 4;
        const int dtype = T.grad_dtype();
        float* const p_out = T.p + e0;
        uint8_t *const m_out = static_cast<uint8_t*>(T.m) + e0, *const v_out = static_cast<uint8_t*>(T.v) + e0;
        float* const scale_out = (lane & 16 ? T.vs : T.ms) + tile / kAdamWBlock + warp;
        const uint32_t e_first = T.before() + e0, offset_m = T.t * kGolden, offset_v = T.t * kPlastic;
#pragma unroll
        for (int k = 0; k < kBlocks; ++k) {
            const int i = k * kRow + t * 4;
            Block4 p = load4(s.p, i, 0, true), g, m, v;
            if (dtype == LFS_F32) g = load4(s.g, i, 0, true);
            else {
                const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(s.g) + i);
                g = {half_bits(w.x & 0xFFFFu, dtype), half_bits(w.x >> 16, dtype), half_bits(w.y & 0xFFFFu, dtype), half_bits(w.y >> 16, dtype)};
            }
            m = decode_m(load4(s.m, i, 0, true), s.ms[k * kWarps + warp]);
            v = decode_v(load4(s.v, i, 0, true), s.vs[k * kWarps + warp]);
            update<true>(p, m, v, g, S);
            store4(p_out, k * kRow, 0, true, p);
            const Codes c = encode_moments(m, v, e_first + k * kRow, offset_m, offset_v);
            *reinterpret_cast<uint32_t*>(m_out + k * kRow) = c.m;
            *reinterpret_cast<uint32_t*>(v_out + k * kRow) = c.v;
            if ((lane & 15) == 0) scale_out[k * kWarps] = c.scale;
        }
    }
}

// Moments in 32 bits: memory. A tile is a block to a warp, and the next one's loads are under way while it is computed: 59 M elements 258 us, 99 % of the copy rate (simple 321); 270 to 281 in a long run, of which
// 2 % are the root and the division.
template <int CAP>
__global__ void __launch_bounds__(kThreads, kCtas32) adamw32_kernel(const __grid_constant__ AdamWArgs<CAP> A) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = threadIdx.x;
    const int total = A.first[A.n];
    float4 p4, m4, v4;
    uint4 g4;
    int ahead = 0;
    auto load = [&](int q) {
        if (q >= total) return;
        ahead = tensor_of(A, q, ahead);
        const AdamWTensor& T = A.t[ahead];
        const uint32_t tile = (uint32_t)(q - A.first[ahead]) * kRow, e = tile + t * 4;
        if (!(T.aligned() && tile + kRow <= T.n)) return;
        p4 = *reinterpret_cast<const float4*>(T.p + e);
        m4 = *reinterpret_cast<const float4*>(static_cast<const float*>(T.m) + e);
        v4 = *reinterpret_cast<const float4*>(static_cast<const float*>(T.v) + e);
        if (T.grad_dtype() == LFS_F32) g4 = *reinterpret_cast<const uint4*>(static_cast<const float*>(T.g) + e);
        else {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(T.g) + e);
            g4 = make_uint4(w.x, w.y, 0, 0);
        }
    };
    int now = 0;
    load(blockIdx.x);
    for (int q = blockIdx.x; q < total; q += gridDim.x) {
        now = tensor_of(A, q, now);
        const AdamWTensor& T = A.t[now];
        const Step S{A.grad_scale, A.beta1, A.beta2, A.one_minus_beta1, A.one_minus_beta2, T.bc2_sqrt_rcp, A.eps, A.minus_zero, T.step_size, T.decay};
        const uint32_t tile = (uint32_t)(q - A.first[now]) * kRow, e = tile + t * 4;
        const bool whole = T.aligned() && tile + kRow <= T.n;
        Block4 p{{p4.x, p4.y, p4.z, p4.w}}, m{{m4.x, m4.y, m4.z, m4.w}}, v{{v4.x, v4.y, v4.z, v4.w}}, g;
        if (T.grad_dtype() == LFS_F32) g = {__uint_as_float(g4.x), __uint_as_float(g4.y), __uint_as_float(g4.z), __uint_as_float(g4.w)};
        else g = {half_bits(g4.x & 0xFFFFu, T.grad_dtype()), half_bits(g4.x >> 16, T.grad_dtype()), half_bits(g4.y & 0xFFFFu, T.grad_dtype()), half_bits(g4.y >> 16, T.grad_dtype())};
        load(q + gridDim.x);
        if (whole) {
            update<false>(p, m, v, g, S);
            store4(T.p, e, 0, true, p);
            store4(static_cast<float*>(T.m), e, 0, true, m);
            store4(static_cast<float*>(T.v), e, 0, true, v);
        } else if (tile + warp * kAdamWBlock < T.n) single_block<32>(T, tile + warp * kAdamWBlock, lane, S);
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
        const uint32_t c = second ? encode_block<true>(x, 0, 0, true, &scale) : encode_block<false>(x, 0, 0, true, &scale);
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

struct Host {
    double beta1, beta2, eps;
    int64_t step_count;
    float grad_scale;
    cudaStream_t st;
};
// One launch over pieces of tensors with the same kind of moments.
template <int CAP, int BITS>
int launch_adamw(int count, const AdamWTensor* pieces, const Host& h) {
    static_assert(sizeof(AdamWArgs<CAP>) <= 32764, "kernel arguments");
    constexpr int kShared = kStages * (int)sizeof(Stage);
    if (BITS == 8) {
        // once per device, and again where it failed
        static std::atomic<uint64_t> asked{0};
        int device = 0;
        if (cudaGetDevice(&device) != cudaSuccess || device > 63 || !(asked.load() >> device & 1)) {
            if (cudaFuncSetAttribute(adamw8_kernel<CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared) != cudaSuccess) return check_launch("adamw");
            if (device < 64) asked.fetch_or((uint64_t)1 << device);
        }
    }
    constexpr int kElements = BITS == 8 ? kTile : kRow;   // of a tile
    AdamWArgs<CAP> A;
    int64_t tiles = 0;
    A.n = count;
    A.first[0] = 0;
    for (int k = 0; k < count; ++k) {
        A.t[k] = pieces[k];
        tiles += (pieces[k].n + kElements - 1) / kElements;   // 2^20 at the most
        A.first[k + 1] = (int32_t)tiles;
    }
    A.beta1 = (float)h.beta1; A.beta2 = (float)h.beta2;
    A.one_minus_beta1 = (float)(1.0 - h.beta1); A.one_minus_beta2 = (float)(1.0 - h.beta2);
    A.eps = (float)h.eps; A.grad_scale = h.grad_scale; A.minus_zero = -0.0f;
    LFS_TIMED("adamw", h.st);
    // With 16 tiles to a CTA and more, three CTAs per SM: us for 0.25, 0.5, 1 and 3 M Gaussians at SH degree 3 with four 42, 82, 168 and 478, with three 43, 79, 152 and 459; 30 k and 120 k 9.7 and 26.0,
    // 10.1 and 27.0. (Moments in 32 bits: 1 M in 295, 257 and 304 with four, three and two.)
    if (BITS == 8) adamw8_kernel<CAP><<<grid_for(tiles, 1, tiles >= 16ll * kCtas8 * num_sms() ? kCtas8 - 1 : kCtas8), kThreads, kShared, h.st>>>(A);
    else adamw32_kernel<CAP><<<grid_for(tiles, 1, kCtas32), kThreads, 0, h.st>>>(A);
    return check_launch("adamw");
}
template <int BITS>
int launch_adamw_kind(int n_tensors, const lfs_adamw_tensor* tensors, const Host& h) {
    AdamWTensor pieces[kAdamWMany];
    int count = 0;
    auto flush = [&] {
        const int rc = count == 0 ? LFS_OK : count <= kAdamWFew ? launch_adamw<kAdamWFew, BITS>(count, pieces, h)
                     : count <= kAdamWSome ? launch_adamw<kAdamWSome, BITS>(count, pieces, h) : launch_adamw<kAdamWMany, BITS>(count, pieces, h);
        count = 0;
        return rc;
    };
    int64_t step = 0;      // most tensors have the one number
    double bc1 = 0.0, bc2_sqrt_rcp = 0.0;
    for (int k = 0; k < n_tensors; ++k) {
        const lfs_adamw_tensor& t = tensors[k];
        if ((t.exp_avg_scale != nullptr) != (BITS == 8)) continue;
        if (t.n > 0 && h.step_count - t.missed != step) {
            step = h.step_count - t.missed;
            bc1 = 1.0 / (1.0 - std::pow(h.beta1, (double)step));   // the same host arithmetic as lfs_adam_step_segments
            bc2_sqrt_rcp = 1.0 / std::sqrt(1.0 - std::pow(h.beta2, (double)step));
        }
        const int grad_bytes = (int)dtype_bytes(t.grad_dtype), moment_bytes = BITS / 8;
        for (int64_t at = 0; at < t.n; at += kPiece) {
            if (count == kAdamWMany) {
                const int rc = flush();
                if (rc != LFS_OK) return rc;
            }
            AdamWTensor& o = pieces[count++];
            o.p = t.param + at;
            o.g = static_cast<const char*>(t.grad) + at * grad_bytes;
            o.m = static_cast<char*>(t.exp_avg) + at * moment_bytes;
            o.v = static_cast<char*>(t.exp_avg_sq) + at * moment_bytes;
            o.ms = BITS == 8 ? t.exp_avg_scale + at / kAdamWBlock : nullptr;
            o.vs = BITS == 8 ? t.exp_avg_sq_scale + at / kAdamWBlock : nullptr;
            o.n = (uint32_t)std::min(t.n - at, kPiece);
            o.step_size = (float)((double)t.lr * bc1);
            o.decay = (float)(1.0 - (double)t.lr * (double)t.weight_decay);
            o.bc2_sqrt_rcp = (float)bc2_sqrt_rcp;
            o.t = (uint32_t)step;
            const bool aligned = aligned_by(o.p, 16) && aligned_by(o.g, 16) && aligned_by(o.m, 16) && aligned_by(o.v, 16) && aligned_by(o.ms, 16) && aligned_by(o.vs, 16);
            o.flags = (uint32_t)t.grad_dtype | (aligned ? kAligned : 0u) | (uint32_t)at;
        }
    }
    return flush();
}

}  // namespace

int launch_adamw_tensors(int n_tensors, const lfs_adamw_tensor* tensors, double beta1, double beta2, double eps, int64_t step_count, float grad_scale,
                         cudaStream_t st) {
    const Host h{beta1, beta2, eps, step_count, grad_scale, st};
    const int rc = launch_adamw_kind<32>(n_tensors, tensors, h);
    return rc != LFS_OK ? rc : launch_adamw_kind<8>(n_tensors, tensors, h);
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
