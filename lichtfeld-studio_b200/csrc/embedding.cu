// Embedding lookup with scaling, out[i] = scale * table[indices[i]], and its gradient, v_table[r] = scale * sum over the i with indices[i] = r of v_out[i].
// An index that names no row of the table (-1, or past its end) gives zeros and takes no part in the gradient.
//
// The gradient goes by the lookups in the order of their rows: every row's sum is a run of consecutive lookups, added in that order by one
// group of lanes, so nothing is added by atomics and a call repeated gives the same bits. The order is an entry point of its own: labels of a palette
// keep it over many steps.
#include "embedding.cuh"

#include <cmath>

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
//
// Bound by the requests that an SM can send (76 % of their rate; a store is five, and 32 neighbouring elements lie in 2.7 lines of the table where rows are no whole number of lines): 1 M rows of 45
// floats 43 us, 70 % of the copy rate, 3 M rows of 24 from half precision 53 us, 88 %. The same rows with a division for every element 79 us, with the rows' places in shared memory 48, copied to shared memory in 16-byte
// pieces first 49 (by warps) to 69, four neighbouring elements a thread 48.
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
// Stable radix sort of (row, position) by the row, up to 9 bits of it a pass: a CTA counts its lookups by their digit, one CTA per digit turns the
// counts into places, and the lookups go there. Up to 2048 lookups one CTA does all passes. Lookups that name no row sort behind all others, as row `rows`.
constexpr int kSortThreads = 256, kSortWarps = kSortThreads / 32, kDigitBits = 9, kDigits = 1 << kDigitBits;
// Lookups of a thread: few shorten the launches while there are not many tiles, more give fewer counts (one pass over 400 k lookups 16.6 us with four and 18.6 with eight, over 3 M 59 and 54).
constexpr int kItemsFew = 4, kItemsMany = 8;
constexpr int64_t kManyLookups = 1 << 20;
constexpr int kSmallSort = 2048;   // of one CTA: 6 us, where the launches take 10 to 20

struct SortPass {
    int64_t n;
    uint32_t rows;
    int shift, bits;
    int tiles;
    const void* indices;       // first pass
    int index_bits;
    const int32_t *rows_in, *at_in;   // later passes
};
__device__ __forceinline__ uint32_t index_key(const void* indices, int index_bits, uint32_t rows, int64_t i) {
    const int64_t r = index_bits == 32 ? (int64_t) static_cast<const int32_t*>(indices)[i] : static_cast<const int64_t*>(indices)[i];
    return r >= 0 && r < (int64_t)rows ? (uint32_t)r : rows;
}
template <bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const SortPass& P, int64_t i) {
    return FIRST ? index_key(P.indices, P.index_bits, P.rows, i) : (uint32_t)P.rows_in[i];
}

template <bool FIRST, int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortPass P, uint32_t* __restrict__ counts) {
    __shared__ uint32_t count[kSortWarps / 2][kDigits];   // two warps share one: less waiting for a digit that many lookups have
    const int digits = 1 << P.bits;
    let_next_start();
    for (int d = threadIdx.x; d < kSortWarps / 2 * kDigits; d += kSortThreads) (&count[0][0])[d] = 0;
    wait_for_previous();
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * (kSortThreads * ITEMS);
    uint32_t* const mine = count[threadIdx.x >> 6];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = first + k * kSortThreads + threadIdx.x;
        if (i < P.n) atomicAdd(&mine[(sort_key<FIRST>(P, i) >> P.shift) & (digits - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < digits; d += kSortThreads) {
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < kSortWarps / 2; ++w) sum += count[w][d];
        counts[(size_t)d * P.tiles + blockIdx.x] = sum;
    }
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
    let_next_start();
    wait_for_previous();
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

// A warp's ITEMS * 32 lookups, 32 neighbouring ones at a time, in their order: each one's rank among the warp's of its digit, which `count` adds up. The lanes of a digit are found by a vote for
// each of its bits. (The instruction that compares all lanes takes as long as there are different values: 27 us instead of 21 for the three launches of a pass over 20 k lookups.)
template <int ITEMS>
__device__ __forceinline__ void warp_ranks(const uint32_t (&digit)[ITEMS], int there, uint32_t* count, uint32_t (&rank)[ITEMS]) {
    const int lane = threadIdx.x & 31;
    uint32_t same[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        same[k] = __ballot_sync(0xffffffffu, k * 32 + lane < there);
#pragma unroll
        for (int b = 0; b < kDigitBits; ++b) {
            const bool one = (digit[k] >> b) & 1;
            const uint32_t votes = __ballot_sync(0xffffffffu, one);
            same[k] &= one ? votes : ~votes;
        }
    }
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const bool in = k * 32 + lane < there;
        const uint32_t before = count[digit[k]], lower = same[k] & ((1u << lane) - 1);
        rank[k] = before + __popc(lower);
        __syncwarp();
        if (in && !lower) count[digit[k]] = before + __popc(same[k]);
        __syncwarp();
    }
}
// From the warps' counts of every digit: where each warp's first lookup of a digit goes. totals: lookups of a digit in all tiles and where this tile's start among them, or null: this CTA's alone.
__device__ __forceinline__ void digit_places(uint32_t (*place)[kDigits], int digits, const uint32_t* counts, int tiles, const uint32_t* totals, uint32_t* warp_sums) {
    uint32_t carry = 0;
    for (int d0 = 0; d0 < digits; d0 += kSortThreads) {
        const int d = d0 + threadIdx.x;
        uint32_t own = 0, all;
        if (d < digits && !totals)
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) own += place[w][d];
        const uint32_t before = block_prefix(d >= digits ? 0u : totals ? totals[d] : own, warp_sums, &all);
        if (d < digits) {
            uint32_t next = carry + before + (totals ? counts[(size_t)d * tiles + blockIdx.x] : 0u);
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t c = place[w][d];
                place[w][d] = next;
                next += c;
            }
        }
        carry += all;
    }
}

template <bool FIRST, int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_place_kernel(SortPass P, const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
                                                                  int32_t* __restrict__ rows_out, int32_t* __restrict__ at_out) {
    __shared__ uint32_t place[kSortWarps][kDigits];
    __shared__ uint32_t warp_sums[kSortWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << P.bits;
    const int64_t first = (int64_t)blockIdx.x * (kSortThreads * ITEMS) + warp * (32 * ITEMS);
    uint32_t key[ITEMS], digit[ITEMS], rank[ITEMS];
    int32_t at[ITEMS];
    let_next_start();
    for (int d = threadIdx.x; d < kSortWarps * kDigits; d += kSortThreads) (&place[0][0])[d] = 0;
    wait_for_previous();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int64_t i = first + k * 32 + lane;
        key[k] = i < P.n ? sort_key<FIRST>(P, i) : 0u;
        at[k] = FIRST ? (int32_t)i : i < P.n ? P.at_in[i] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) digit[k] = (key[k] >> P.shift) & (digits - 1);
    warp_ranks<ITEMS>(digit, (int)max((int64_t)0, min(P.n - first, (int64_t)(32 * ITEMS))), place[warp], rank);
    __syncthreads();
    digit_places(place, digits, counts, P.tiles, totals, warp_sums);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        if (first + k * 32 + lane < P.n) {
            const uint32_t to = place[warp][digit[k]] + rank[k];
            rows_out[to] = (int32_t)key[k];
            at_out[to] = at[k];
        }
    }
}

// All passes over up to 32 * kSortWarps * ITEMS lookups, by one CTA.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) sort_small_kernel(int n, uint32_t rows, const void* __restrict__ indices, int index_bits, int passes, int bits,
                                                                  int32_t* __restrict__ rows_out, int32_t* __restrict__ at_out) {
    __shared__ uint32_t place[kSortWarps][kDigits];
    __shared__ uint32_t warp_sums[kSortWarps];
    __shared__ uint32_t key_s[kSortThreads * ITEMS];
    __shared__ uint16_t at_s[kSortThreads * ITEMS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, digits = 1 << bits;
    const int first = warp * (32 * ITEMS);
    uint32_t key[ITEMS], digit[ITEMS], rank[ITEMS];
    int32_t at[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int i = first + k * 32 + lane;
        key[k] = i < n ? index_key(indices, index_bits, rows, i) : 0u;
        at[k] = i;
    }
    for (int p = 0; p < passes; ++p) {
        for (int d = threadIdx.x; d < kSortWarps * kDigits; d += kSortThreads) (&place[0][0])[d] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) digit[k] = (key[k] >> (p * bits)) & (digits - 1);
        warp_ranks<ITEMS>(digit, max(0, min(n - first, 32 * ITEMS)), place[warp], rank);
        __syncthreads();
        digit_places(place, digits, nullptr, 1, nullptr, warp_sums);
        __syncthreads();
        const bool last = p + 1 == passes;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            if (first + k * 32 + lane < n) {
                const uint32_t to = place[warp][digit[k]] + rank[k];
                if (last) {
                    rows_out[to] = (int32_t)key[k];
                    at_out[to] = at[k];
                } else {
                    key_s[to] = key[k];
                    at_s[to] = (uint16_t)at[k];
                }
            }
        }
        __syncthreads();
        if (last) return;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = first + k * 32 + lane;
            if (i < n) {
                key[k] = key_s[i];
                at[k] = at_s[i];
            }
        }
    }
}

struct SortPlan { int bits, passes, digit_bits, items, tiles; };
SortPlan sort_plan(int64_t n, int64_t rows) {
    SortPlan p{};
    while ((rows >> p.bits) != 0) ++p.bits;   // keys are 0 .. rows
    p.passes = (p.bits + kDigitBits - 1) / kDigitBits;
    p.digit_bits = (p.bits + p.passes - 1) / p.passes;
    p.items = n > kManyLookups ? kItemsMany : kItemsFew;
    p.tiles = (int)((n + kSortThreads * p.items - 1) / (kSortThreads * p.items));
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
// A CTA takes a stretch of the sorted lookups, and a group of lanes a part of that, a row of v_out at a time, T of them under way. The group's lanes fetch four lookups each,
// and the next four while it works on these. A row of the table whose lookups lie in one group's part is written from there. Otherwise the first group that has some adds the others' sums to its
// own: each leaves what belongs to a row begun before it in shared memory. What crosses stretches is left in the workspace, [stretch][head, tail][width], for embedding_join_kernel. Rows
// without lookups are cleared before.
//
// Sums are held in two floats, the second gathering in float32 what the first rounds off, so the result is that of sums with twice the bits, rounded once: off by 2^-24 of itself and, for a row of k lookups, by at
// most 6 k^2 2^-48 of its addends' magnitudes (much less: a group adds a part of them). Where that second part counts, which is where large addends cancel, it depends on the cut, and so on the GPU's SMs. Sums in 64 bits
// took 273 us for a million lookups of 45 columns where these took 84: 32-bit values become 64-bit ones at a small fraction of the rate that additions have.
//
// Bound by the loads of the rows, which lie anywhere in v_out: 1 M rows of 180 bytes take 248 MB from memory, 64 bytes at a time, 40 us at the copy rate; all of the gradient takes 61 us, 3 of them
// the clearing and 5 embedding_join_kernel. Of the rest the sums are 2 and the looks for another row 4; rows that stay in L2 take 46. Neither more rows under way (eight, twelve, sixteen), nor the
// next ones while these are added (62), nor more or fewer CTAs, nor a warp to a row of 45 columns (79), nor copies to shared memory ahead (4 bytes a lane: 80) changed that.
constexpr int kBwdThreads = 256, kTileUnits = 128;
constexpr int64_t kOwnClear = 32768;   // elements of a table that a single CTA clears itself (a launch less: 1.5 us)
// CTAs per SM by the sums that a lane holds
constexpr int bwd_ctas(int sums) { return sums <= 4 ? 3 : 2; }

// A number in two floats. The lookup's scale is a float32, as its products are; here the sums have more bits than that.
struct Scale { float hi, lo; };
Scale two_floats(double x) {
    const float hi = (float)x;
    return {hi, std::isfinite(hi) ? (float)(x - hi) : 0.0f};
}

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
    // what the product of the first floats leaves of the sum times scale
    __device__ __forceinline__ float rest(Scale scale, float p) const { return __fmaf_rn(lo, scale.hi, __fmaf_rn(hi, scale.lo, __fmaf_rn(hi, scale.hi, -p))); }
    // the sum times scale, rounded once; once it is infinite or NaN the roundings say nothing
    __device__ __forceinline__ float times(Scale scale) const {
        const float p = __fmul_rn(hi, scale.hi);
        return isfinite(p) ? __fadd_rn(p, rest(scale, p)) : p;
    }
    // and added to `more`
    __device__ __forceinline__ float times(Scale scale, float more) const {
        const float p = __fmul_rn(hi, scale.hi);
        Sum r{more, rest(scale, p)};
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
__global__ void __launch_bounds__(kBwdThreads, bwd_ctas(C * V)) embedding_bwd_kernel(int64_t n, int64_t rows, int width, int log_group, int share, int clear, const typename Element<DTYPE>::T* __restrict__ v_out,
                                                                    const int32_t* __restrict__ order, const int32_t* __restrict__ sorted_rows, Scale scale, int accumulate,
                                                                    float* __restrict__ v_table, Sum* __restrict__ parts) {
    using In = Pack<DTYPE, V>;
    __shared__ __align__(16) int32_t row_s[4 * kBwdThreads], at_s[4 * kBwdThreads];
    __shared__ Sum head_s[C * V][kBwdThreads];
    __shared__ int32_t first_row_s;
    __shared__ uint8_t ends_s[kBwdThreads];   // by group: the row that it begins inside of ends in it
    const int group = 1 << log_group, lane = threadIdx.x & (group - 1), g = threadIdx.x >> log_group, groups = kBwdThreads >> log_group;
    const int units = width / V, unit0 = blockIdx.y * kTileUnits + lane;
    const int64_t first = (int64_t)blockIdx.x * share * groups;
    const int total = (int)min((int64_t)share * groups, n - first);
    const int begin = min(g * share, total), end = min(begin + share, total);
    let_next_start();
    for (int i = threadIdx.x; i < clear; i += kBwdThreads) v_table[i] = 0.0f;   // by the only CTA, before it writes a row
    int4 next_row{}, next_at{};
    auto fetch = [&](int t) {   // four lookups of this lane, from t + 4 lane on
        const int64_t i = first + t + 4 * lane;
        if (t + 4 * lane + 4 <= end) {
            next_row = *reinterpret_cast<const int4*>(sorted_rows + i);
            next_at = *reinterpret_cast<const int4*>(order + i);
        } else if (t + 4 * lane < end) {
            const int left = end - t - 4 * lane;
            next_row.x = sorted_rows[i];
            next_at.x = order[i];
            if (left > 1) { next_row.y = sorted_rows[i + 1]; next_at.y = order[i + 1]; }
            if (left > 2) { next_row.z = sorted_rows[i + 2]; next_at.z = order[i + 2]; }
        }
    };
    fetch(begin);
    const int32_t before = begin < end && first + begin > 0 ? sorted_rows[first + begin - 1] : -1, after = begin < end && first + end < n ? sorted_rows[first + end] : -1;
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
        if (row >= rows) return;
#pragma unroll
        for (int k = 0; k < C; ++k) {
            const int u = unit0 + (k << log_group);
            if (u < units) {
                float* dst = v_table + (size_t)row * width + u * V;
#pragma unroll
                for (int j = 0; j < V; ++j) dst[j] = accumulate ? acc.get(k * V + j).times(scale, dst[j]) : acc.get(k * V + j).times(scale);
            }
        }
    };
    acc.clear();
    int32_t row = -1;
    bool head = false, tail = false, from_before = false;
    const int32_t *const my_rows = row_s + 4 * group * g, *const my_at = at_s + 4 * group * g;
    auto take = [&](int t, auto count) {
        constexpr int N = decltype(count)::value;
        In x[N][C];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t at = (int64_t)my_at[t + i] * units;
#pragma unroll
            for (int k = 0; k < C; ++k) x[i][k] = column[k][at];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int32_t r = my_rows[t + i];
            if (r != row) {
                if (head) keep_head();
                else write_row(row);
                head = false;
                acc.clear();
                row = r;
            }
            float v[C * V];
#pragma unroll
            for (int k = 0; k < C; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) v[k * V + j] = Element<DTYPE>::from(x[i][k].x[j]);
            acc.add(v);
        }
    };
    if (clear) __syncthreads();
    // every group of a warp goes round as often as the others
    for (int t = 0; t < share; t += 4 * group) {
        __syncwarp();
        reinterpret_cast<int4*>(row_s)[threadIdx.x] = next_row;
        reinterpret_cast<int4*>(at_s)[threadIdx.x] = next_at;
        __syncwarp();
        fetch(begin + t + 4 * group);
        const int count = min(4 * group, end - begin - t);
        if (count <= 0) continue;
        if (t == 0) {
            row = my_rows[0];
            head = from_before = before == row;
            if (g == 0 && lane == 0) first_row_s = row;
        }
        if (my_rows[0] >= rows && row >= rows) continue;   // lookups that name no row are the last ones
        int i = 0;
        for (; i + T <= count; i += T) take(i, Constant<int, T>{});
        for (; i < count; ++i) take(i, Constant<int, 1>{});
    }
    if (begin < end) {
        const bool goes_on = after == row;
        if (lane == 0) ends_s[g] = !head || !goes_on;
        if (head) keep_head();
        else if (goes_on) tail = row < rows;
        else write_row(row);
    }
    __syncthreads();
    // Sums of the heads that follow one another: in the round of d, a group whose row has not ended in the d parts from its own on adds those of the next d.
    bool stop = begin >= end || ends_s[g];
    for (int d = 1; d < groups; d *= 2) {
        const bool more = !stop && g + d < groups && (g + d) * share < total;
        if (!__syncthreads_or(more)) break;
        Sum sum[C * V];
        bool then = true;
        if (more) {
            then = ends_s[g + d];
#pragma unroll
            for (int i = 0; i < C * V; ++i) {
                sum[i] = head_s[i][threadIdx.x];
                sum[i].add(head_s[i][threadIdx.x + (d << log_group)]);
            }
        }
        __syncthreads();
        if (more) {
            stop = then;
            if (lane == 0) ends_s[g] = then;
#pragma unroll
            for (int i = 0; i < C * V; ++i) head_s[i][threadIdx.x] = sum[i];
        }
        __syncthreads();
    }
    // the row that goes on behind this group's part, and the one that the stretch begins inside of
    const bool opens = g == 0 && begin < end && from_before && first_row_s < rows;
    const int next = g + 1;
    const bool followed = next < groups && next * share < total;
#pragma unroll
    for (int k = 0; k < C; ++k) {
        const int u = unit0 + (k << log_group);
        if (u >= units) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int col = u * V + j;
            if (opens) parts[(size_t)(2 * (int64_t)blockIdx.x) * width + col] = head_s[k * V + j][threadIdx.x];
            if (tail) {
                Sum sum = acc.get(k * V + j);
                if (followed) sum.add(head_s[k * V + j][threadIdx.x + group]);
                if (!followed || !ends_s[next]) parts[(size_t)(2 * (int64_t)blockIdx.x + 1) * width + col] = sum;
                else {
                    float* dst = v_table + (size_t)row * width + col;
                    *dst = accumulate ? sum.times(scale, *dst) : sum.times(scale);
                }
            }
        }
    }
}

// The rows that lie in several stretches: the one that has a row's tail adds the heads of those that follow. A CTA per stretch; its threads are columns by slices of the heads.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) embedding_join_kernel(int64_t n, int64_t rows, int width, int stretch, int stretches, const int32_t* __restrict__ sorted_rows,
                                                                      Scale scale, int accumulate, const Sum* __restrict__ parts, float* __restrict__ v_table) {
    __shared__ Sum sum_s[kJoinThreads];
    __shared__ int next_s;
    wait_for_previous();
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
            *dst = accumulate ? acc.times(scale, *dst) : acc.times(scale);
        }
        __syncthreads();
    }
}

// lookups of a group and number of stretches: all CTAs at once where there are that many lookups, and 4 a lane at least
struct Cut { int share; int64_t stretches; };
Cut bwd_cut(int64_t n, int log_group, int ctas, int column_tiles) {
    const int64_t groups = kBwdThreads >> log_group, slots = max(1, num_sms() * ctas / column_tiles), step = 4 << log_group;
    const int64_t share = max(step, ((n + slots * groups - 1) / (slots * groups) + 3) / 4 * 4);
    return {(int)share, (n + share * groups - 1) / (share * groups)};
}
// the most stretches that a call may have, for any alignment
int64_t bwd_stretches(int64_t n) { return (n + 4 * kBwdThreads - 1) / (4 * kBwdThreads); }

struct Bwd {
    int64_t n, rows;
    int width, log_group, accumulate;
    const void* v_out;
    const int32_t *order, *sorted_rows;
    Scale scale;
    float* v_table;
    Sum* parts;
    cudaStream_t st;
};
template <int DTYPE, int V, int C>
int bwd(const Bwd& b) {
    constexpr int T = C * V <= 8 ? 4 : 2;
    const int column_tiles = (b.width / V + kTileUnits - 1) / kTileUnits;
    const Cut cut = bwd_cut(b.n, b.log_group, bwd_ctas(C * V), column_tiles);
    const bool alone = cut.stretches == 1 && column_tiles == 1 && b.rows * b.width <= kOwnClear;
    if (!b.accumulate && !alone && cudaMemsetAsync(b.v_table, 0, (size_t)b.rows * b.width * sizeof(float), b.st) != cudaSuccess) {
        set_error("lfs_embedding_bwd: memset failed");
        return LFS_ECUDA;
    }
    embedding_bwd_kernel<DTYPE, V, C, T><<<dim3((unsigned)cut.stretches, (unsigned)column_tiles), kBwdThreads, 0, b.st>>>(
        b.n, b.rows, b.width, b.log_group, cut.share, alone && !b.accumulate ? (int)(b.rows * b.width) : 0, static_cast<const typename Element<DTYPE>::T*>(b.v_out), b.order, b.sorted_rows, b.scale, b.accumulate, b.v_table, b.parts);
    const int rc = check_launch("embedding_bwd");
    if (rc != LFS_OK || cut.stretches == 1) return rc;
    launch_beside(embedding_join_kernel, (int)cut.stretches, kJoinThreads, 0, b.st, b.n, b.rows, b.width, cut.share * (kBwdThreads >> b.log_group), (int)cut.stretches, b.sorted_rows, b.scale,
                  b.accumulate, (const Sum*)b.parts, b.v_table);
    return check_launch("embedding_join");
}
template <int DTYPE, int V>
int bwd_units(Bwd b) {
    // lanes of a group times units of a lane: as few as cover the row, and then as many lanes as that leaves
    const int units = min(b.width / V, kTileUnits);
    int best = 1 << 30, per_lane = 1;
    for (int log_group = 5; log_group >= 1; --log_group) {
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

size_t embedding_sort_bytes(int64_t n, int64_t rows) { return n <= kSmallSort ? 0 : carve_sort(n, sort_plan(n, rows), nullptr).bytes; }

// Each launch of a pass begins while the one before it ends, and waits for it before it reads.
template <bool FIRST, int ITEMS>
static void launch_sort_pass(const SortPass& P, const SortWs& w, int32_t* rows_out, int32_t* at_out, cudaStream_t st) {
    if (FIRST) launch(sort_count_kernel<FIRST, ITEMS>, P.tiles, kSortThreads, 0, st, P, w.counts);
    else launch_beside(sort_count_kernel<FIRST, ITEMS>, P.tiles, kSortThreads, 0, st, P, w.counts);
    launch_beside(sort_scan_kernel, 1 << P.bits, kSortThreads, 0, st, P.tiles, w.counts, w.totals);
    launch_beside(sort_place_kernel<FIRST, ITEMS>, P.tiles, kSortThreads, 0, st, P, (const uint32_t*)w.counts, (const uint32_t*)w.totals, rows_out, at_out);
}

int launch_embedding_sort(int64_t n, int64_t rows, const void* indices, int index_bits, int32_t* order, int32_t* sorted_rows, void* workspace, cudaStream_t st) {
    if (n == 0) return LFS_OK;
    LFS_TIMED("embedding_sort", st);
    const SortPlan p = sort_plan(n, rows);
    if (n <= kSmallSort) {
        (n <= kSortThreads ? sort_small_kernel<1> : n <= 4 * kSortThreads ? sort_small_kernel<4> : sort_small_kernel<kSmallSort / kSortThreads>)<<<1, kSortThreads, 0, st>>>(
            (int)n, (uint32_t)rows, indices, index_bits, p.passes, p.digit_bits, sorted_rows, order);
        return check_launch("embedding_sort");
    }
    const SortWs w = carve_sort(n, p, workspace);
    for (int k = 0; k < p.passes; ++k) {
        const bool mine = (p.passes - 1 - k) % 2 == 0;   // the last pass writes the caller's arrays
        SortPass P{};
        P.n = n; P.rows = (uint32_t)rows;
        P.shift = k * p.digit_bits;
        P.bits = p.digit_bits;
        P.tiles = p.tiles;
        P.indices = indices; P.index_bits = index_bits;
        P.rows_in = mine ? w.rows : sorted_rows;
        P.at_in = mine ? w.at : order;
        int32_t *rows_out = mine ? sorted_rows : w.rows, *at_out = mine ? order : w.at;
        const bool few = p.items == kItemsFew;
        (k == 0 ? few ? launch_sort_pass<true, kItemsFew> : launch_sort_pass<true, kItemsMany>
                : few ? launch_sort_pass<false, kItemsFew> : launch_sort_pass<false, kItemsMany>)(P, w, rows_out, at_out, st);
    }
    return check_launch("embedding_sort");
}

size_t embedding_bwd_bytes(int64_t n, int width) { return bwd_stretches(n) <= 1 ? 0 : (size_t)bwd_stretches(n) * 2 * width * sizeof(Sum); }

int launch_embedding_bwd(int64_t n, int64_t rows, int width, const void* v_out, int dtype, const int32_t* order, const int32_t* sorted_rows, double scale,
                         int accumulate, float* v_table, void* workspace, cudaStream_t st) {
    LFS_TIMED("embedding_bwd", st);
    if (n == 0) {
        if (!accumulate && cudaMemsetAsync(v_table, 0, (size_t)rows * width * sizeof(float), st) != cudaSuccess) {
            set_error("lfs_embedding_bwd: memset failed");
            return LFS_ECUDA;
        }
        return LFS_OK;
    }
    const Bwd b{n, rows, width, 0, accumulate, v_out, order, sorted_rows, two_floats(scale), v_table, static_cast<Sum*>(workspace), st};
    return dtype == LFS_F32 ? bwd_type<LFS_F32>(b) : dtype == LFS_BF16 ? bwd_type<LFS_BF16>(b) : bwd_type<LFS_F16>(b);
}

}  // namespace lfs
