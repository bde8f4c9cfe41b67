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
// A CTA takes a run of rows; its elements go to the threads in their order in `out`, V of a row at a time.
constexpr int kFwdThreads = 256, kFwdUnroll = 4;
template <int IN, int OUT, int V, class Index>
__global__ void __launch_bounds__(kFwdThreads) embedding_fwd_kernel(int64_t n, int64_t rows, int units, Divide by_units, int run, const typename Element<IN>::T* __restrict__ table,
                                                                    const Index* __restrict__ indices, float scale, typename Element<OUT>::T* __restrict__ out) {
    using In = Pack<IN, V>;
    using Out = Pack<OUT, V>;
    for (int64_t first = (int64_t)blockIdx.x * run; first < n; first += (int64_t)gridDim.x * run) {
        const uint32_t total = (uint32_t)(min((int64_t)run, n - first) * units);
        Out* dst = reinterpret_cast<Out*>(out) + first * units;
        for (uint32_t u0 = threadIdx.x; u0 < total; u0 += kFwdThreads * kFwdUnroll) {
            In x[kFwdUnroll];
            bool some[kFwdUnroll];
#pragma unroll
            for (int k = 0; k < kFwdUnroll; ++k) {
                const uint32_t u = u0 + k * kFwdThreads;
                some[k] = false;
                if (u < total) {
                    const uint32_t i = by_units(u);
                    const int64_t r = (int64_t)indices[first + i];
                    some[k] = r >= 0 && r < rows;
                    if (some[k]) x[k] = reinterpret_cast<const In*>(table)[r * units + (u - i * units)];
                }
            }
#pragma unroll
            for (int k = 0; k < kFwdUnroll; ++k) {
                const uint32_t u = u0 + k * kFwdThreads;
                if (u < total) {
                    Out y;
#pragma unroll
                    for (int j = 0; j < V; ++j) y.x[j] = Element<OUT>::to(some[k] ? __fmul_rn(Element<IN>::from(x[k].x[j]), scale) : 0.0f);
                    dst[u] = y;
                }
            }
        }
    }
}

template <int IN, int OUT, int V, class Index>
int fwd(int64_t n, int64_t rows, int width, const void* table, const void* indices, float scale, void* out, cudaStream_t st) {
    const int units = width / V;
    const int run = max(1, min(4096 / units, 1 << 20));
    embedding_fwd_kernel<IN, OUT, V, Index><<<grid_for((n + run - 1) / run, 1, 32), kFwdThreads, 0, st>>>(
        n, rows, units, divide_by((uint32_t)units), run, static_cast<const typename Element<IN>::T*>(table), static_cast<const Index*>(indices), scale,
        static_cast<typename Element<OUT>::T*>(out));
    return check_launch("embedding_fwd");
}
template <int IN, int OUT>
int fwd(int64_t n, int64_t rows, int width, const void* table, const void* indices, int index_bits, float scale, void* out, cudaStream_t st) {
    const bool whole = width % 4 == 0 && reinterpret_cast<uintptr_t>(table) % (4 * sizeof(typename Element<IN>::T)) == 0 &&
                       reinterpret_cast<uintptr_t>(out) % (4 * sizeof(typename Element<OUT>::T)) == 0;
    if (index_bits == 32)
        return whole ? fwd<IN, OUT, 4, int32_t>(n, rows, width, table, indices, scale, out, st) : fwd<IN, OUT, 1, int32_t>(n, rows, width, table, indices, scale, out, st);
    return whole ? fwd<IN, OUT, 4, int64_t>(n, rows, width, table, indices, scale, out, st) : fwd<IN, OUT, 1, int64_t>(n, rows, width, table, indices, scale, out, st);
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
// The sorted lookups are cut into chunks of equal length, and a group of lanes adds up one chunk, a row of v_out at a time. A row of the table whose lookups all lie
// in one chunk is written there; of the others every chunk leaves its part in the workspace, [chunk][head, tail][width], and a second launch adds the parts up
// in their order: a tail (the row starts in this chunk and goes on) and the heads of the chunks that follow. Rows without lookups are cleared first.
constexpr int kBwdThreads = 256, kBwdTokens = 4, kChunk = 64, kTileUnits = 128;

template <int DTYPE, int V, int C>
__global__ void __launch_bounds__(kBwdThreads) embedding_bwd_kernel(int64_t n, int64_t rows, int width, int log_group, int chunks, const typename Element<DTYPE>::T* __restrict__ v_out,
                                                                    const int32_t* __restrict__ order, const int32_t* __restrict__ sorted_rows, float scale, int accumulate,
                                                                    float* __restrict__ v_table, float* __restrict__ parts) {
    using In = Pack<DTYPE, V>;
    const int group = 1 << log_group, lane = threadIdx.x & (group - 1);
    const int units = width / V;
    const int unit0 = blockIdx.y * kTileUnits + lane;
    const int groups = kBwdThreads >> log_group;
    for (int64_t c = (int64_t)blockIdx.x * groups + (threadIdx.x >> log_group); c < chunks; c += (int64_t)gridDim.x * groups) {
        const int64_t begin = c * kChunk, end = min(begin + kChunk, n);
        float acc[C][V];
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[k][j] = 0.0f;
        int32_t row = sorted_rows[begin];
        const bool from_before = begin > 0 && sorted_rows[begin - 1] == row;
        const int32_t after = end < n ? sorted_rows[end] : -1;
        bool head = from_before;
        auto write = [&](bool last) {
            if (row >= rows) return;
            const bool goes_on = last && after == row;
            float* dst = head ? parts + (size_t)(2 * c) * width : goes_on ? parts + (size_t)(2 * c + 1) * width : v_table + (size_t)row * width;
            const bool direct = !head && !goes_on;
#pragma unroll
            for (int k = 0; k < C; ++k) {
                const int u = unit0 + (k << log_group);
                if (u < units) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float x = acc[k][j];
                        if (direct) {
                            x = __fmul_rn(x, scale);
                            if (accumulate) x += dst[u * V + j];
                        }
                        dst[u * V + j] = x;
                        acc[k][j] = 0.0f;
                    }
                }
            }
        };
        for (int64_t t = begin; t < end; t += kBwdTokens) {
            int32_t r[kBwdTokens];
            In x[kBwdTokens][C];
#pragma unroll
            for (int i = 0; i < kBwdTokens; ++i) {
                const bool in = t + i < end;
                r[i] = in ? sorted_rows[t + i] : -1;
                const int64_t src = in ? (int64_t)order[t + i] * units : 0;
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    const int u = unit0 + (k << log_group);
                    if (in && r[i] < rows && u < units) x[i][k] = reinterpret_cast<const In*>(v_out)[src + u];
                }
            }
#pragma unroll
            for (int i = 0; i < kBwdTokens; ++i) {
                if (r[i] < 0) break;
                if (r[i] != row) {
                    write(false);
                    row = r[i];
                    head = false;
                }
                if (r[i] >= rows) break;
#pragma unroll
                for (int k = 0; k < C; ++k) {
                    const int u = unit0 + (k << log_group);
                    if (u < units)
#pragma unroll
                        for (int j = 0; j < V; ++j) acc[k][j] += Element<DTYPE>::from(x[i][k].x[j]);
                }
            }
        }
        write(true);
    }
}

// One CTA per chunk that holds a tail: its lanes take the columns.
__global__ void __launch_bounds__(128) embedding_join_kernel(int64_t n, int64_t rows, int width, int chunks, const int32_t* __restrict__ sorted_rows, float scale, int accumulate,
                                                             const float* __restrict__ parts, float* __restrict__ v_table) {
    for (int64_t c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int64_t begin = c * kChunk, end = min(begin + kChunk, n);
        const int32_t row = sorted_rows[end - 1];
        if (row >= rows || end >= n || sorted_rows[end] != row) continue;
        if (sorted_rows[begin] == row && begin > 0 && sorted_rows[begin - 1] == row) continue;   // it started earlier
        for (int col = threadIdx.x; col < width; col += blockDim.x) {
            float acc = parts[(size_t)(2 * c + 1) * width + col];
            for (int64_t d = c + 1; d < chunks && sorted_rows[d * kChunk] == row; ++d) acc += parts[(size_t)(2 * d) * width + col];
            float x = __fmul_rn(acc, scale);
            float* dst = v_table + (size_t)row * width + col;
            if (accumulate) x += *dst;
            *dst = x;
        }
    }
}

int64_t bwd_chunks(int64_t n) { return (n + kChunk - 1) / kChunk; }

template <int DTYPE, int V, int C>
int bwd(int64_t n, int64_t rows, int width, int log_group, const void* v_out, const int32_t* order, const int32_t* sorted_rows, float scale, int accumulate, float* v_table,
        float* parts, cudaStream_t st) {
    const int64_t chunks = bwd_chunks(n);
    const dim3 grid((unsigned)grid_for(chunks << log_group, kBwdThreads, 32), (unsigned)((width / V + kTileUnits - 1) / kTileUnits));
    embedding_bwd_kernel<DTYPE, V, C><<<grid, kBwdThreads, 0, st>>>(n, rows, width, log_group, (int)chunks, static_cast<const typename Element<DTYPE>::T*>(v_out), order, sorted_rows,
                                                                     scale, accumulate, v_table, parts);
    return check_launch("embedding_bwd");
}
template <int DTYPE, int V>
int bwd(int64_t n, int64_t rows, int width, const void* v_out, const int32_t* order, const int32_t* sorted_rows, float scale, int accumulate, float* v_table, float* parts,
        cudaStream_t st) {
    const int units = min(width / V, kTileUnits);
    int log_group = 0;
    while ((4 << log_group) < units) ++log_group;
    switch ((units + (1 << log_group) - 1) >> log_group) {
        case 1: return bwd<DTYPE, V, 1>(n, rows, width, log_group, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st);
        case 2: return bwd<DTYPE, V, 2>(n, rows, width, log_group, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st);
        case 3: return bwd<DTYPE, V, 3>(n, rows, width, log_group, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st);
        default: return bwd<DTYPE, V, 4>(n, rows, width, log_group, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st);
    }
}
template <int DTYPE>
int bwd(int64_t n, int64_t rows, int width, const void* v_out, const int32_t* order, const int32_t* sorted_rows, float scale, int accumulate, float* v_table, float* parts,
        cudaStream_t st) {
    const bool whole = width % 4 == 0 && reinterpret_cast<uintptr_t>(v_out) % (4 * sizeof(typename Element<DTYPE>::T)) == 0;
    return whole ? bwd<DTYPE, 4>(n, rows, width, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st)
                 : bwd<DTYPE, 1>(n, rows, width, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st);
}

}  // namespace

int launch_embedding_fwd(int64_t n, int64_t rows, int width, const void* table, int table_dtype, const void* indices, int index_bits, float scale,
                         void* out, int out_dtype, cudaStream_t st) {
    if (n == 0) return LFS_OK;
    LFS_TIMED("embedding_fwd", st);
    if (table_dtype == LFS_F32) return fwd<LFS_F32, LFS_F32>(n, rows, width, table, indices, index_bits, scale, out, st);
    if (table_dtype == LFS_BF16)
        return out_dtype == LFS_F32 ? fwd<LFS_BF16, LFS_F32>(n, rows, width, table, indices, index_bits, scale, out, st)
                                    : fwd<LFS_BF16, LFS_BF16>(n, rows, width, table, indices, index_bits, scale, out, st);
    return out_dtype == LFS_F32 ? fwd<LFS_F16, LFS_F32>(n, rows, width, table, indices, index_bits, scale, out, st)
                                : fwd<LFS_F16, LFS_F16>(n, rows, width, table, indices, index_bits, scale, out, st);
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

size_t embedding_bwd_bytes(int64_t n, int width) { return (size_t)bwd_chunks(n) * 2 * width * sizeof(float); }

int launch_embedding_bwd(int64_t n, int64_t rows, int width, const void* v_out, int dtype, const int32_t* order, const int32_t* sorted_rows, float scale,
                         int accumulate, float* v_table, void* workspace, cudaStream_t st) {
    LFS_TIMED("embedding_bwd", st);
    if (!accumulate && cudaMemsetAsync(v_table, 0, (size_t)rows * width * sizeof(float), st) != cudaSuccess) {
        set_error("lfs_embedding_bwd: memset failed");
        return LFS_ECUDA;
    }
    if (n == 0) return LFS_OK;
    float* parts = static_cast<float*>(workspace);
    const int rc = dtype == LFS_F32 ? bwd<LFS_F32>(n, rows, width, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st)
                 : dtype == LFS_BF16 ? bwd<LFS_BF16>(n, rows, width, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st)
                                     : bwd<LFS_F16>(n, rows, width, v_out, order, sorted_rows, scale, accumulate, v_table, parts, st);
    if (rc != LFS_OK) return rc;
    const int64_t chunks = bwd_chunks(n);
    embedding_join_kernel<<<grid_for(chunks, 1, 16), 128, 0, st>>>(n, rows, width, (int)chunks, sorted_rows, scale, accumulate, parts, v_table);
    return check_launch("embedding_join");
}

}  // namespace lfs
