// Embedding lookup with scaling, out[i] = scale * table[indices[i]], and its gradient, v_table[r] = scale * sum over the i with indices[i] = r of v_out[i].
// An index that names no row of the table (-1, or past its end) gives zeros and takes no part in the gradient.
//
// The gradient goes by the lookups in the order of their rows: every row's sum is a run of consecutive lookups, added in that order by one
// group of lanes, so nothing is added by atomics and a call repeated gives the same bits. The order is an entry point of its own: labels of a palette
// keep it over many steps.
#include "embedding.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace lfs {

namespace {

// ---- values of a row ------------------------------------------------------------------------------
template <int DTYPE> struct Element;
template <> struct Element<LFS_F32> {
    using T = float;
    static __device__ __forceinline__ float from(float x) { return x; }
    static __device__ __forceinline__ float to(float x) { return x; }
};
template <> struct Element<LFS_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float from(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 to(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Element<LFS_F16> {
    using T = __half;
    static __device__ __forceinline__ float from(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half to(float x) { return __float2half_rn(x); }
};
// V elements, read and written at once
template <int DTYPE, int V>
struct alignas(sizeof(typename Element<DTYPE>::T) * V) Pack { typename Element<DTYPE>::T x[V]; };

template <class T, T X> struct Constant { static constexpr T value = X; };

// a / d for a < 2^31 by a multiplication: m = ceil(2^(31 + s) / d), s = ceil(log2 d)
struct Divide {
    uint32_t d, m, s;
    __device__ __forceinline__ uint32_t operator()(uint32_t a) const { return d == 1 ? a : (uint32_t)(((uint64_t)a * m) >> 32) >> (s - 1); }
};
Divide divide_by(uint32_t d) {
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    return {d, d == 1 ? 0u : (uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}

// ---- lookup ------------------------------------------------------------------------------------------
// A warp writes 32 rows of `out`, 32 neighbouring pieces of V elements at a time, so that it stores whole lines wherever the rows begin. Piece e of the 32 rows belongs to row i = e / units, whose
// place in the table less its place among the 32 is the same for all its pieces: lane i holds it, and an address is that times the row's length plus a pointer that moves by a constant.
constexpr int kFwdThreads = 128, kFwdUnroll = 8;
template <int IN, int OUT, int V>
__global__ void __launch_bounds__(kFwdThreads) embedding_fwd_kernel(int64_t n, int64_t rows, int units, Divide by_units, int segments, int segment,
                                                                    const typename Element<IN>::T* __restrict__ table, const void* __restrict__ indices, int index_bits,
                                                                    float scale, typename Element<OUT>::T* __restrict__ out) {
    using In = Pack<IN, V>;
    using Out = Pack<OUT, V>;
    const int lane = threadIdx.x & 31;
    const int64_t warps = ((n + 31) / 32) * segments;
    const int step_row = (int)by_units(32), step_col = 32 - step_row * units, row_bytes = units * (int)sizeof(In);
    for (int64_t w = (int64_t)blockIdx.x * (kFwdThreads / 32) + (threadIdx.x >> 5); w < warps; w += (int64_t)gridDim.x * (kFwdThreads / 32)) {
        const int64_t group = segments == 1 ? w : w / segments, first = group * 32;
        const int from = (int)(w - group * segments) * segment;
        const int total = (int)min((int64_t)32, n - first) * units, to = min(from + segment, total);
        int64_t r = -1;
        if (first + lane < n) r = index_bits == 32 ? (int64_t) static_cast<const int32_t*>(indices)[first + lane] : static_cast<const int64_t*>(indices)[first + lane];
        const bool valid = r >= 0 && r < rows;
        const uint32_t all = __ballot_sync(0xffffffffu, valid || first + lane >= n);
        const int moved = valid ? (int)r - lane : -lane;   // a row that is there in place of one that is not
        const char* src = reinterpret_cast<const char*>(table) + (int64_t)(from + lane) * (int)sizeof(In);
        Out* dst = reinterpret_cast<Out*>(out) + first * units + (from + lane);
        const uint32_t e0 = by_units((uint32_t)(from + lane));
        int row = (int)e0, col = from + lane - row * units;
        auto take = [&](int count, auto unroll, auto checked) {   // `count` pieces of this lane are there
            constexpr int N = decltype(unroll)::value;
            constexpr bool kChecked = decltype(checked)::value;
            In x[N];
            bool there[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int m = __shfl_sync(0xffffffffu, moved, row);
                there[k] = !kChecked || ((all >> (row & 31)) & 1);
                if (N > 1 || count > 0) x[k] = *reinterpret_cast<const In*>(src + (int64_t)m * row_bytes + k * 32 * (int)sizeof(In));
                row += step_row;
                col += step_col;
                if (col >= units) { col -= units; ++row; }
            }
#pragma unroll
            for (int k = 0; k < N; ++k) {
                Out y;
#pragma unroll
                for (int j = 0; j < V; ++j) y.x[j] = Element<OUT>::to(there[k] ? __fmul_rn(Element<IN>::from(x[k].x[j]), scale) : 0.0f);
                if (N > 1 || count > 0) dst[k * 32] = y;
            }
            src += N * 32 * (int)sizeof(In);
            dst += N * 32;
        };
        int e = from;
        if (all == 0xffffffffu) {
            for (; e + kFwdUnroll * 32 <= to; e += kFwdUnroll * 32) take(0, Constant<int, kFwdUnroll>{}, Constant<bool, false>{});
            for (; e + 2 * 32 <= to; e += 2 * 32) take(0, Constant<int, 2>{}, Constant<bool, false>{});
            for (; e < to; e += 32) take(to - e - lane, Constant<int, 1>{}, Constant<bool, false>{});
        } else {
            for (; e < to; e += 32) take(to - e - lane, Constant<int, 1>{}, Constant<bool, true>{});
        }
    }
}

template <int IN, int OUT, int V>
int fwd(int64_t n, int64_t rows, int width, const void* table, const void* indices, int index_bits, float scale, void* out, cudaStream_t st) {
    const int units = width / V;
    // a warp's pieces are 32 * units, cut up where there are few rows or long ones
    const int64_t groups = (n + 31) / 32, enough = (int64_t)num_sms() * 32;
    int64_t segments = max((int64_t)(units + 127) / 128, min((enough + groups - 1) / groups, (int64_t)units));
    const int segment = (int)((units + segments - 1) / segments) * 32;
    segments = (32ll * units + segment - 1) / segment;
    embedding_fwd_kernel<IN, OUT, V><<<grid_for(groups * segments, kFwdThreads / 32, 64), kFwdThreads, 0, st>>>(
        n, rows, units, divide_by((uint32_t)units), (int)segments, segment, static_cast<const typename Element<IN>::T*>(table), indices, index_bits, scale,
        static_cast<typename Element<OUT>::T*>(out));
    return check_launch("embedding_fwd");
}
template <int IN, int OUT>
int fwd_type(int64_t n, int64_t rows, int width, const void* table, const void* indices, int index_bits, float scale, void* out, cudaStream_t st) {
    const bool whole = width % 4 == 0 && aligned_by(table, 4 * sizeof(typename Element<IN>::T)) && aligned_by(out, 4 * sizeof(typename Element<OUT>::T));
    return (whole ? fwd<IN, OUT, 4> : fwd<IN, OUT, 1>)(n, rows, width, table, indices, index_bits, scale, out, st);
}

// ---- order --------------------------------------------------------------------------------------------
// Stable radix sort of (row, position) by the row, up to 9 bits of it a pass: a CTA counts its 4096 lookups by their digit, one CTA per digit turns the
// counts into places, and the lookups go there. Lookups that name no row sort behind all others, as row `rows`.
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32, kSortItems = 16, kSortTile = kSortThreads * kSortItems, kDigitBits = 9, kDigits = 1 << kDigitBits;

struct SortPass {
    int64_t n;
    uint32_t rows;
    int shift, digits;         // digits: their number, a power of two
    int tiles;
    const void* indices;       // first pass
    int index_bits;
    const int32_t *rows_in, *at_in;   // later passes
};
template <bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const SortPass& P, int64_t i) {
    if (!FIRST) return (uint32_t)P.rows_in[i];
    const int64_t r = P.index_bits == 32 ? (int64_t) static_cast<const int32_t*>(P.indices)[i] : static_cast<const int64_t*>(P.indices)[i];
    return r >= 0 && r < (int64_t)P.rows ? (uint32_t)r : P.rows;
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortPass P, uint32_t* __restrict__ counts) {
    __shared__ uint32_t count[kDigits];
    for (int d = threadIdx.x; d < P.digits; d += kSortThreads) count[d] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kSortTile;
#pragma unroll 4
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = first + k * kSortThreads + threadIdx.x;
        const bool in = i < P.n;
        const uint32_t d = in ? (sort_key<FIRST>(P, i) >> P.shift) & (P.digits - 1) : kDigits;
        const uint32_t same = __match_any_sync(0xffffffffu, d);   // one addition for all lanes of a digit
        if (in && (int)(threadIdx.x & 31) == __ffs(same) - 1) atomicAdd(&count[d], __popc(same));
    }
    __syncthreads();
    for (int d = threadIdx.x; d < P.digits; d += kSortThreads) counts[(size_t)d * P.tiles + blockIdx.x] = count[d];
}

// exclusive prefix of one value per thread over the block of kSortThreads; the total to all threads
__device__ __forceinline__ uint32_t block_prefix(uint32_t x, uint32_t* warp_sums, uint32_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    if (lane == 31) warp_sums[warp] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    __syncthreads();
    *total = all;
    return before + s - x;
}

// counts of one digit in all tiles -> exclusive prefix over the tiles, and the digit's total
__global__ void __launch_bounds__(kSortThreads) sort_scan_kernel(int tiles, uint32_t* __restrict__ counts, uint32_t* __restrict__ totals) {
    __shared__ uint32_t warp_sums[kSortWarps];
    uint32_t* c = counts + (size_t)blockIdx.x * tiles;
    uint32_t carry = 0;
    for (int t0 = 0; t0 < tiles; t0 += kSortThreads) {
        const int t = t0 + threadIdx.x;
        const uint32_t x = t < tiles ? c[t] : 0;
        uint32_t all;
        const uint32_t before = block_prefix(x, warp_sums, &all);
        if (t < tiles) c[t] = carry + before;
        carry += all;
    }
    if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortPass P, const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                                                                  int32_t* __restrict__ rows_out, int32_t* __restrict__ at_out) {
    __shared__ uint32_t place[kSortWarps][kDigits];
    __shared__ uint32_t warp_sums[kSortWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int d = threadIdx.x; d < kSortWarps * kDigits; d += kSortThreads) (&place[0][0])[d] = 0;
    __syncthreads();
    // a warp takes 32 neighbouring lookups at a time, in their order; a lookup's rank among its warp's of the same digit
    const int64_t first = (int64_t)blockIdx.x * kSortTile + warp * (32 * kSortItems);
    uint32_t key[kSortItems], rank[kSortItems];
    int32_t at[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const int64_t i = first + k * 32 + lane;
        key[k] = i < P.n ? sort_key<FIRST>(P, i) : 0u;
        at[k] = FIRST ? (int32_t)i : i < P.n ? P.at_in[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        const bool in = first + k * 32 + lane < P.n;
        const uint32_t d = in ? (key[k] >> P.shift) & (P.digits - 1) : kDigits;
        const uint32_t same = __match_any_sync(0xffffffffu, d);
        rank[k] = in ? place[warp][d] + __popc(same & ((1u << lane) - 1)) : 0u;
        __syncwarp();
        if (in && lane == __ffs(same) - 1) place[warp][d] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    // where the digits start, where this tile's lookups of a digit start, and where each warp's
    uint32_t carry = 0;
    for (int d0 = 0; d0 < P.digits; d0 += kSortThreads) {
        const int d = d0 + threadIdx.x;
        uint32_t all;
        const uint32_t before = block_prefix(d < P.digits ? totals[d] : 0u, warp_sums, &all);
        if (d < P.digits) {
            uint32_t next = carry + before + counts[(size_t)d * P.tiles + blockIdx.x];
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t c = place[w][d];
                place[w][d] = next;
                next += c;
            }
        }
        carry += all;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; ++k) {
        if (first + k * 32 + lane < P.n) {
            const uint32_t to = place[warp][(key[k] >> P.shift) & (P.digits - 1)] + rank[k];
            rows_out[to] = (int32_t)key[k];
            at_out[to] = at[k];
        }
    }
}

struct SortPlan { int bits, passes, digit_bits, tiles; };
SortPlan sort_plan(int64_t n, int64_t rows) {
    SortPlan p{};
    while ((rows >> p.bits) != 0) ++p.bits;   // keys are 0 .. rows
    p.passes = (p.bits + kDigitBits - 1) / kDigitBits;
    p.digit_bits = (p.bits + p.passes - 1) / p.passes;
    p.tiles = (int)((n + kSortTile - 1) / kSortTile);
    return p;
}
struct SortWs {
    uint32_t *counts, *totals;
    int32_t *rows, *at;
    size_t bytes;
};
SortWs carve_sort(int64_t n, const SortPlan& p, void* base) {
    SortWs w{};
    char* at = static_cast<char*>(base);
    size_t off = 0;
    auto take = [&](size_t bytes) {
        char* q = at ? at + off : nullptr;
        off += (bytes + 255) & ~(size_t)255;
        return q;
    };
    w.counts = reinterpret_cast<uint32_t*>(take(((size_t)p.tiles << p.digit_bits) * 4));
    w.totals = reinterpret_cast<uint32_t*>(take(kDigits * 4));
    if (p.passes > 1) {
        w.rows = reinterpret_cast<int32_t*>(take((size_t)n * 4));
        w.at = reinterpret_cast<int32_t*>(take((size_t)n * 4));
    }
    w.bytes = off;
    return w;
}

// ---- gradient -------------------------------------------------------------------------------------------
// A CTA takes a stretch of the sorted lookups, and a group of lanes a part of that, a row of v_out at a time, T of them under way. A row of the table whose lookups
// lie in one group's part is written from there. Otherwise the first group that has some adds the others' sums to its own: each leaves what belongs to a row begun before it in shared
// memory. What crosses stretches is left in the workspace, [stretch][head, tail][width], for embedding_join_kernel. Rows without lookups are cleared before.
//
// Sums are held in two floats: a million gradients of one row lose nothing, and the result is the exact sum rounded once (but for ties), whatever the stretches. Sums in 64 bits
// took 273 us for a million lookups of 45 columns where these took 84: 32-bit values become 64-bit ones at a small fraction of the rate that additions have.
constexpr int kBwdThreads = 256, kStretch = 1024, kTileUnits = 128;

// A sum in two floats: every rounding of the first is exact in the second (Knuth's two-sum). Explicit roundings, so that none of it is simplified away.
struct Sum {
    float hi, lo;
    __device__ __forceinline__ void add(float x) {
        const float s = __fadd_rn(hi, x), b = __fsub_rn(s, hi);
        lo = __fadd_rn(lo, __fadd_rn(__fsub_rn(hi, __fsub_rn(s, b)), __fsub_rn(x, b)));
        hi = s;
    }
    __device__ __forceinline__ void add(const Sum& o) {
        add(o.hi);
        lo = __fadd_rn(lo, o.lo);
    }
    // the sum times scale, plus `more`, rounded once; once it is infinite or NaN the roundings say nothing
    __device__ __forceinline__ float times(float scale, float more) const {
        const float p = __fmul_rn(hi, scale);
        Sum r{more, __fmaf_rn(lo, scale, __fmaf_rn(hi, scale, -p))};
        r.add(p);
        return isfinite(r.hi) ? __fadd_rn(r.hi, r.lo) : r.hi;
    }
};
// N of them, two to an instruction
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) { f32x2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float part(f32x2 v, int k) { float a, b; asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); return k ? b : a; }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f32x2 sub2(f32x2 a, f32x2 b) { f32x2 r; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
template <int N>
struct Sums {
    static constexpr int kPairs = N / 2;
    f32x2 hi[kPairs > 0 ? kPairs : 1], lo[kPairs > 0 ? kPairs : 1];
    Sum odd;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) hi[k] = lo[k] = 0;
        odd = {0.0f, 0.0f};
    }
    __device__ __forceinline__ void add(const float (&x)[N]) {
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            const f32x2 v = pair(x[2 * k], x[2 * k + 1]), s = add2(hi[k], v), b = sub2(s, hi[k]);
            lo[k] = add2(lo[k], add2(sub2(hi[k], sub2(s, b)), sub2(v, b)));
            hi[k] = s;
        }
        if constexpr (N % 2) odd.add(x[N - 1]);
    }
    __device__ __forceinline__ Sum get(int k) const { return k < 2 * kPairs ? Sum{part(hi[k / 2], k & 1), part(lo[k / 2], k & 1)} : odd; }
};

template <int DTYPE, int V, int C, int T>
__global__ void __launch_bounds__(kBwdThreads) embedding_bwd_kernel(int64_t n, int64_t rows, int width, int log_group, int stretch,
                                                                    const typename Element<DTYPE>::T* __restrict__ v_out, const int32_t* __restrict__ order,
                                                                    const int32_t* __restrict__ sorted_rows, float scale, int accumulate,
                                                                    float* __restrict__ v_table, Sum* __restrict__ parts) {
    using In = Pack<DTYPE, V>;
    __shared__ int2 lookup_s[kStretch + 2];   // row and position; [0] and the one behind the last belong to the neighbours
    __shared__ Sum head_s[C * V][kBwdThreads];
    __shared__ uint8_t from_before_s[kBwdThreads], ends_s[kBwdThreads];   // by group: it begins inside a row, and that row ends in it
    __shared__ int total_s;
    const int64_t first = (int64_t)blockIdx.x * stretch;
    const int there = (int)min((int64_t)stretch, n - first);
    if (threadIdx.x == 0) {
        lookup_s[0].x = first > 0 ? sorted_rows[first - 1] : -1;
        lookup_s[there + 1].x = first + there < n ? sorted_rows[first + there] : -1;
        total_s = there;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < there; i += kBwdThreads) {
        const int32_t r = sorted_rows[first + i];
        lookup_s[i + 1] = make_int2(r, order[first + i]);
        if (r >= rows) atomicMin(&total_s, i);   // lookups that name no row are the last ones
    }
    __syncthreads();
    const int total = total_s;
    const int group = 1 << log_group, lane = threadIdx.x & (group - 1), g = threadIdx.x >> log_group, groups = kBwdThreads >> log_group;
    const int units = width / V, unit0 = blockIdx.y * kTileUnits + lane;
    const int share = stretch / groups, begin = min(g * share, total), end = min(begin + share, total);
    // lanes behind the last column read it again and write nothing
    const In* column[C];
#pragma unroll
    for (int k = 0; k < C; ++k) column[k] = reinterpret_cast<const In*>(v_out) + min(unit0 + (k << log_group), units - 1);
    Sums<C * V> acc;
    auto keep_head = [&] {
#pragma unroll
        for (int i = 0; i < C * V; ++i) head_s[i][threadIdx.x] = acc.get(i);
    };
    auto write_row = [&](int32_t row) {
#pragma unroll
        for (int k = 0; k < C; ++k) {
            const int u = unit0 + (k << log_group);
            if (u < units) {
                float* dst = v_table + (size_t)row * width + u * V;
#pragma unroll
                for (int j = 0; j < V; ++j) dst[j] = acc.get(k * V + j).times(scale, accumulate ? dst[j] : 0.0f);
            }
        }
    };
    acc.clear();
    int32_t row = -1;
    bool head = false, tail = false;
    if (begin < end) {
        row = lookup_s[begin + 1].x;
        const bool from_before = lookup_s[begin].x == row;
        head = from_before;
        auto take = [&](int t, auto count) {
            constexpr int N = decltype(count)::value;
            int32_t r[N];
            In x[N][C];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int2 l = lookup_s[t + i + 1];
                r[i] = l.x;
#pragma unroll
                for (int k = 0; k < C; ++k) x[i][k] = column[k][(int64_t)l.y * units];
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if (r[i] != row) {
                    if (head) keep_head();
                    else write_row(row);
                    head = false;
                    acc.clear();
                    row = r[i];
                }
                float v[C * V];
#pragma unroll
                for (int k = 0; k < C; ++k)
#pragma unroll
                    for (int j = 0; j < V; ++j) v[k * V + j] = Element<DTYPE>::from(x[i][k].x[j]);
                acc.add(v);
            }
        };
        int t = begin;
        for (; t + T <= end; t += T) take(t, Constant<int, T>{});
        for (; t < end; ++t) take(t, Constant<int, 1>{});
        const bool goes_on = lookup_s[end + 1].x == row;
        if (lane == 0) {
            from_before_s[g] = from_before;
            ends_s[g] = !head || !goes_on;
        }
        if (head) keep_head();
        else if (goes_on) tail = true;
        else write_row(row);
    }
    __syncthreads();
    // the row that goes on behind this group's part, and the one that the stretch begins inside of
    auto join = [&](int32_t joined, bool from_head) {
        int last = g + 1;
        bool open = !from_head || !ends_s[0];
        while (open && last * share < total) open = !ends_s[last++];   // parts g + 1 .. last - 1 begin inside the row
#pragma unroll
        for (int k = 0; k < C; ++k) {
            const int u = unit0 + (k << log_group);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                Sum sum = from_head ? head_s[k * V + j][threadIdx.x] : acc.get(k * V + j);
                for (int h = g + 1; h < last; ++h) sum.add(head_s[k * V + j][(h << log_group) + lane]);
                if (u < units) {
                    const int col = u * V + j;
                    if (from_head) parts[(size_t)(2 * (int64_t)blockIdx.x) * width + col] = sum;
                    else if (open) parts[(size_t)(2 * (int64_t)blockIdx.x + 1) * width + col] = sum;
                    else {
                        float* dst = v_table + (size_t)joined * width + col;
                        *dst = sum.times(scale, accumulate ? *dst : 0.0f);
                    }
                }
            }
        }
    };
    if (tail) join(row, false);
    if (g == 0 && begin < end && from_before_s[0]) join(lookup_s[1].x, true);
}

// The rows that lie in several stretches: the one that has a row's tail adds the heads of those that follow. A CTA per stretch; its threads are columns by slices of the heads.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) embedding_join_kernel(int64_t n, int64_t rows, int width, int stretch, int stretches, const int32_t* __restrict__ sorted_rows,
                                                                      float scale, int accumulate, const Sum* __restrict__ parts, float* __restrict__ v_table) {
    __shared__ Sum sum_s[kJoinThreads];
    __shared__ int next_s;
    const int c = blockIdx.x;
    const int64_t first = (int64_t)c * stretch, end = min(first + stretch, n);
    const int32_t row = sorted_rows[end - 1];
    if (row >= rows || end >= n || sorted_rows[end] != row) return;
    if (sorted_rows[first] == row && first > 0 && sorted_rows[first - 1] == row) return;   // it begins earlier
    // stretches c + 1 .. next - 1 begin inside the row
    if (threadIdx.x == 0) next_s = stretches;
    __syncthreads();
    for (int d0 = c + 1; d0 < stretches; d0 += kJoinThreads) {
        const int d = d0 + threadIdx.x;
        const bool another = d < stretches && sorted_rows[(int64_t)d * stretch] != row;
        if (another) atomicMin(&next_s, d);
        if (__syncthreads_or(another)) break;
    }
    __syncthreads();
    const int next = next_s;
    const int columns = min(width, kJoinThreads), slices = kJoinThreads / columns, slice = threadIdx.x / columns;
    for (int col0 = 0; col0 < width; col0 += columns) {
        const int col = col0 + threadIdx.x % columns;
        Sum acc{0.0f, 0.0f};
        if (slice < slices && col < width) {
            if (slice == 0) acc = parts[(size_t)(2 * (int64_t)c + 1) * width + col];
#pragma unroll 8
            for (int d = c + 1 + slice; d < next; d += slices) acc.add(parts[(size_t)(2 * (int64_t)d) * width + col]);
        }
        sum_s[threadIdx.x] = acc;
        __syncthreads();
        if (threadIdx.x < columns && col < width) {
            for (int k = 1; k < slices; ++k) acc.add(sum_s[threadIdx.x + k * columns]);
            float* dst = v_table + (size_t)row * width + col;
            *dst = acc.times(scale, accumulate ? *dst : 0.0f);
        }
        __syncthreads();
    }
}

int64_t bwd_stretches(int64_t n) { return (n + kStretch - 1) / kStretch; }

struct Bwd {
    int64_t n, rows;
    int width, log_group, accumulate;
    const void* v_out;
    const int32_t *order, *sorted_rows;
    float scale;
    float* v_table;
    Sum* parts;
    cudaStream_t st;
};
template <int DTYPE, int V, int C>
int bwd(const Bwd& b) {
    constexpr int T = C * V <= 4 ? 8 : C * V <= 8 ? 4 : 2;
    const dim3 grid((unsigned)bwd_stretches(b.n), (unsigned)((b.width / V + kTileUnits - 1) / kTileUnits));
    embedding_bwd_kernel<DTYPE, V, C, T><<<grid, kBwdThreads, 0, b.st>>>(b.n, b.rows, b.width, b.log_group, kStretch, static_cast<const typename Element<DTYPE>::T*>(b.v_out),
                                                                         b.order, b.sorted_rows, b.scale, b.accumulate, b.v_table, b.parts);
    return check_launch("embedding_bwd");
}
template <int DTYPE, int V>
int bwd_units(Bwd b) {
    // lanes of a group times units of a lane: as few as cover the row, and then as many lanes as that leaves
    const int units = min(b.width / V, kTileUnits);
    int best = 1 << 30, per_lane = 1;
    for (int log_group = 5; log_group >= 0; --log_group) {
        const int c = (units + (1 << log_group) - 1) >> log_group;
        if (c <= 4 && (c << log_group) < best) { best = c << log_group; b.log_group = log_group; per_lane = c; }
    }
    return per_lane == 1 ? bwd<DTYPE, V, 1>(b) : per_lane == 2 ? bwd<DTYPE, V, 2>(b) : per_lane == 3 ? bwd<DTYPE, V, 3>(b) : bwd<DTYPE, V, 4>(b);
}
template <int DTYPE>
int bwd_type(const Bwd& b) {
    const bool whole = b.width % 4 == 0 && aligned_by(b.v_out, 4 * sizeof(typename Element<DTYPE>::T));
    return whole ? bwd_units<DTYPE, 4>(b) : bwd_units<DTYPE, 1>(b);
}

}  // namespace

int launch_embedding_fwd(int64_t n, int64_t rows, int width, const void* table, int table_dtype, const void* indices, int index_bits, float scale,
                         void* out, int out_dtype, cudaStream_t st) {
    if (n == 0) return LFS_OK;
    LFS_TIMED("embedding_fwd", st);
    if (table_dtype == LFS_F32) return fwd_type<LFS_F32, LFS_F32>(n, rows, width, table, indices, index_bits, scale, out, st);
    if (table_dtype == LFS_BF16)
        return out_dtype == LFS_F32 ? fwd_type<LFS_BF16, LFS_F32>(n, rows, width, table, indices, index_bits, scale, out, st)
                                    : fwd_type<LFS_BF16, LFS_BF16>(n, rows, width, table, indices, index_bits, scale, out, st);
    return out_dtype == LFS_F32 ? fwd_type<LFS_F16, LFS_F32>(n, rows, width, table, indices, index_bits, scale, out, st)
                                : fwd_type<LFS_F16, LFS_F16>(n, rows, width, table, indices, index_bits, scale, out, st);
}

size_t embedding_sort_bytes(int64_t n, int64_t rows) { return carve_sort(n, sort_plan(n, rows), nullptr).bytes; }

int launch_embedding_sort(int64_t n, int64_t rows, const void* indices, int index_bits, int32_t* order, int32_t* sorted_rows, void* workspace, cudaStream_t st) {
    if (n == 0) return LFS_OK;
    LFS_TIMED("embedding_sort", st);
    const SortPlan p = sort_plan(n, rows);
    const SortWs w = carve_sort(n, p, workspace);
    for (int k = 0; k < p.passes; ++k) {
        const bool first = k == 0, mine = (p.passes - 1 - k) % 2 == 0;   // the last pass writes the caller's arrays
        SortPass P{};
        P.n = n; P.rows = (uint32_t)rows;
        P.shift = k * p.digit_bits;
        P.digits = 1 << p.digit_bits;
        P.tiles = p.tiles;
        P.indices = indices; P.index_bits = index_bits;
        P.rows_in = mine ? w.rows : sorted_rows;
        P.at_in = mine ? w.at : order;
        int32_t *rows_out = mine ? sorted_rows : w.rows, *at_out = mine ? order : w.at;
        if (first) sort_count_kernel<true><<<p.tiles, kSortThreads, 0, st>>>(P, w.counts);
        else sort_count_kernel<false><<<p.tiles, kSortThreads, 0, st>>>(P, w.counts);
        sort_scan_kernel<<<P.digits, kSortThreads, 0, st>>>(p.tiles, w.counts, w.totals);
        if (first) sort_place_kernel<true><<<p.tiles, kSortThreads, 0, st>>>(P, w.counts, w.totals, rows_out, at_out);
        else sort_place_kernel<false><<<p.tiles, kSortThreads, 0, st>>>(P, w.counts, w.totals, rows_out, at_out);
    }
    return check_launch("embedding_sort");
}

size_t embedding_bwd_bytes(int64_t n, int width) { return (size_t)bwd_stretches(n) * 2 * width * sizeof(Sum); }

int launch_embedding_bwd(int64_t n, int64_t rows, int width, const void* v_out, int dtype, const int32_t* order, const int32_t* sorted_rows, float scale,
                         int accumulate, float* v_table, void* workspace, cudaStream_t st) {
    LFS_TIMED("embedding_bwd", st);
    if (!accumulate && cudaMemsetAsync(v_table, 0, (size_t)rows * width * sizeof(float), st) != cudaSuccess) {
        set_error("lfs_embedding_bwd: memset failed");
        return LFS_ECUDA;
    }
    if (n == 0) return LFS_OK;
    const Bwd b{n, rows, width, 0, accumulate, v_out, order, sorted_rows, scale, v_table, static_cast<Sum*>(workspace), st};
    const int rc = dtype == LFS_F32 ? bwd_type<LFS_F32>(b) : dtype == LFS_BF16 ? bwd_type<LFS_BF16>(b) : bwd_type<LFS_F16>(b);
    const int64_t stretches = bwd_stretches(n);
    if (rc != LFS_OK || stretches == 1) return rc;
    embedding_join_kernel<<<(unsigned)stretches, kJoinThreads, 0, st>>>(n, rows, width, kStretch, (int)stretches, sorted_rows, b.scale, accumulate, b.parts, v_table);
    return check_launch("embedding_join");
}

}  // namespace lfs
