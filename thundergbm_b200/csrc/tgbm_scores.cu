// Operators on the scores of many classes: penalties, biases and masks (adjust), the largest scores of a row with its
// log-sum-exp (top), the distance from a teacher's largest scores with its gradient (distill).
//
// Scores are a matrix of rows x classes in float, half or bfloat16 with any two strides; a booster keeps all rows of a class
// side by side, networks all classes of a row.  All three operators are bound by memory: they do a few operations per score.
#include <cfloat>
#include <climits>
#include <cmath>

#include <cooperative_groups.h>

#include "../../include/thundergbm.h"
#include "tgbm_kernels.cuh"
#include "tgbm_scores.cuh"
#include "tgbm_scores_check.h"

namespace tgbm {
namespace {
namespace cg = cooperative_groups;

constexpr int ROW_THREADS = 256;
constexpr int FEW = 32, FEW_THREADS = 128;   // classes that a thread's registers hold, rows of a block then

// ------------------------------------------------------------------ adjust
// A block takes a tile of rows x classes.  How often a class stands in the history of its row is counted in shared memory: every
// entry of the tile's histories that falls into its classes adds one (integers: in any order the same), so a history may be
// of any length.  A few instructions per score decide the time, so there are three ways through the scores.
constexpr int ADJUST_CELLS = 8192;

// histories of `rows` rows into counts[cell(row, class - k0)]: the rows' entries lie one behind the other, so the block's threads share
// them evenly, and each finds the row of its entries among the rows' ends
constexpr int ADJUST_MOST_ROWS = 1024;
template <int MOST_ROWS, typename C>
__device__ __forceinline__ void count_histories(const AdjustArgs &a, long long n0, int rows, int k0, int classes, int *count, int cells, C &&cell) {
    __shared__ long long ends[MOST_ROWS];
    int4 *zero = reinterpret_cast<int4 *>(count);
    const long long lo = max(0ll, a.history_ptr[n0]), hi = min(a.n_history, a.history_ptr[n0 + rows]);
    if (MOST_ROWS > 1)
        for (int r = threadIdx.x; r < rows; r += ROW_THREADS) ends[r] = a.history_ptr[n0 + r + 1];
    for (int i = threadIdx.x; i < (cells + 3) / 4; i += ROW_THREADS) zero[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    constexpr int AHEAD = 4;
    for (long long h = lo + threadIdx.x; h < hi; h += AHEAD * ROW_THREADS) {
        int c[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) c[i] = h + i * ROW_THREADS < hi ? a.history[h + i * ROW_THREADS] - k0 : -1;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (c[i] < 0 || c[i] >= classes) continue;
            int x = 0, y = MOST_ROWS == 1 ? 0 : rows - 1;   // the first row that ends behind the entry
            while (x < y) {
                const int mid = (x + y) / 2;
                if (ends[mid] > h + i * ROW_THREADS) y = mid; else x = mid + 1;
            }
            atomicAdd(&count[cell(x, c[i])], 1);
        }
    }
    __syncthreads();
}
// z / r from r's reciprocal, rounded once: the product's error times the reciprocal is put back (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990), except where that error is no float.  A score that was given
// before is in almost every warp, so all scores pay for it: divisions cost the batch of 50003 x 250 4 us more.
__device__ __forceinline__ float penalised(const AdjustArgs &a, float z, int times) {
    const float up = __fmul_rn(z, a.repetition), q = __fmul_rn(z, a.inv_repetition);
    const float error = __fmaf_rn(-q, a.repetition, z);
    const float down = fabsf(z) >= 1e-30f && fabsf(q) <= FLT_MAX ? __fmaf_rn(error, a.inv_repetition, q) : q;
    return (z > 0.f ? down : up) - ((float)times * a.frequency + a.presence);
}
// the row's mask; null: all classes are allowed
__device__ __forceinline__ const unsigned *mask_of(const AdjustArgs &a, long long n) {
    if (!a.allowed) return nullptr;
    const long long m = a.allowed_row ? (long long)a.allowed_row[n] : n;
    return m >= 0 && m < a.n_masks ? a.allowed + m * a.mask_stride : nullptr;
}

// By class: a lane per row, a warp takes neighbouring classes, eight at a time: their scores are read together, and their bits lie in
// one word of the row's mask.  Class strides are ints here: an address is one instruction.
// Blocks per SM (4 x 61 registers): 31 us for 50003 x 250 with histories, 40 with 6 blocks and fewer registers.
constexpr int ADJUST_ROWS = 32, ADJUST_AHEAD = 8, ADJUST_CLASSES = ADJUST_CELLS / ADJUST_ROWS;

template <typename T, bool HISTORY>
__global__ void __launch_bounds__(ROW_THREADS, 4) k_adjust_class(AdjustArgs a, Scores<T> in, Scores<T> out) {
    constexpr int A = ADJUST_AHEAD;
    extern __shared__ __align__(16) int count[];
    const long long n0 = (long long)blockIdx.x * ADJUST_ROWS;
    const int k0 = blockIdx.y * ADJUST_CLASSES, classes = min(ADJUST_CLASSES, a.k - k0), rows = (int)min((long long)ADJUST_ROWS, a.n - n0);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, in_cls = (int)in.cls, out_cls = (int)out.cls;
    const long long n = n0 + min(lane, rows - 1);
    const int per = (classes + A * ROW_THREADS / 32 - 1) / (A * ROW_THREADS / 32) * A, from = warp * per, to = lane < rows ? min(classes, from + per) : from;
    const T *src = in.at(n, k0 + from);
    T *dst = out.at(n, k0 + from);
    T ahead[A];
    auto fetch = [&](int left) {
        if (left >= A) {
#pragma unroll
            for (int i = 0; i < A; ++i) ahead[i] = src[(long long)i * in_cls];
        } else {
#pragma unroll
            for (int i = 0; i < A; ++i)
                if (i < left) ahead[i] = src[(long long)i * in_cls];
        }
        src += (long long)A * in_cls;
    };
    fetch(to - from);   // on their way while the histories are counted
    const unsigned *mask = mask_of(a, n);
    if (HISTORY) count_histories<ADJUST_ROWS>(a, n0, rows, k0, classes, count, classes * ADJUST_ROWS, [](int r, int c) { return c * ADJUST_ROWS + r; });
    for (int c = from; c < to; c += A) {
        float z[A];
        const int k = k0 + c;   // a multiple of 8
#pragma unroll
        for (int i = 0; i < A; ++i) z[i] = score_f32(ahead[i]);
        fetch(to - c - A);
        const unsigned word = mask ? mask[k >> 5] >> (k & 31) : 0xffffffffu;
        if (HISTORY) {
            int times[A];
#pragma unroll
            for (int i = 0; i < A; ++i) times[i] = count[min(c + i, classes - 1) * ADJUST_ROWS + lane];
#pragma unroll
            for (int i = 0; i < A; ++i)
                if (times[i]) z[i] = penalised(a, z[i], times[i]);
        }
        if (a.bias) {
#pragma unroll
            for (int i = 0; i < A; ++i) z[i] += a.bias[min(k + i, a.k - 1)];
        }
#pragma unroll
        for (int i = 0; i < A; ++i)
            if (!(word >> i & 1)) z[i] = minus_inf();
        if (c + A <= to) {
#pragma unroll
            for (int i = 0; i < A; ++i) dst[(long long)i * out_cls] = score_from<T>(z[i]);
        } else {
#pragma unroll
            for (int i = 0; i < A; ++i)
                if (c + i < to) dst[(long long)i * out_cls] = score_from<T>(z[i]);
        }
        dst += (long long)A * out_cls;
    }
}

// By row, long rows: a block takes LONG_CELLS classes of a row, a thread 16 bytes at a time.  The pieces begin at the row's first 16-byte
// boundary; up to V - 1 cells in front of it go with the first piece, one by one.  EVEN: every row begins at one (256 x 131072 in 16 bits
// 49 us so, 54 without saying so; 256 x 131071 68 us).
constexpr int LONG_CELLS = 4096;

template <typename T, bool EVEN>
__global__ void __launch_bounds__(ROW_THREADS, sizeof(T) == 2 ? 8 : 6) k_adjust_long(AdjustArgs a, Scores<T> in, Scores<T> out) {
    constexpr int V = Pack<T>::V, U = LONG_CELLS / (ROW_THREADS * V);
    extern __shared__ __align__(16) int count[];   // LONG_CELLS, then V for the cells in front
    const long long n = blockIdx.x;
    const int head = EVEN ? 0 : min(a.k, (int)((16 - reinterpret_cast<uintptr_t>(in.at(n, 0)) % 16) % 16 / sizeof(T)));
    const int k0 = head + blockIdx.y * LONG_CELLS, classes = max(0, min(LONG_CELLS, a.k - k0)), front = !EVEN && blockIdx.y == 0 ? head : 0;
    const T *src = in.at(n, k0);
    T *dst = out.at(n, k0);
    Pack<T> ahead[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {   // all of them on their way while the history is counted
        const int c = (u * ROW_THREADS + threadIdx.x) * V;
        if (c + V <= classes) ahead[u].bits = *reinterpret_cast<const uint4 *>(src + c);   // (may be the memory that is written)
    }
    const unsigned *mask = mask_of(a, n);
    if (a.history_ptr)
        count_histories<1>(a, n, 1, k0 - front, classes + front, count, EVEN ? classes : LONG_CELLS + V,
                           [&](int, int c) { return EVEN ? c : c < front ? LONG_CELLS + c : c - front; });
    // one cell at a time: in front of the first boundary (c < 0), behind the last
    auto single = [&](int c, int times) {
        const int k = k0 + c;
        float z = score_f32(src[c]);
        if (times) z = penalised(a, z, times);
        if (a.bias) z += a.bias[k];
        if (mask && !(mask[k >> 5] >> (k & 31) & 1)) z = minus_inf();
        dst[c] = score_from<T>(z);
    };
    if (!EVEN && (int)threadIdx.x < front) single((int)threadIdx.x - head, a.history_ptr ? count[LONG_CELLS + threadIdx.x] : 0);
    const bool even_bias = (reinterpret_cast<uintptr_t>(a.bias + k0) & 15) == 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = (u * ROW_THREADS + threadIdx.x) * V;
        if (c >= classes) break;
        if (c + V > classes) {   // the row's last few
            for (int i = c; i < classes; ++i) single(i, a.history_ptr ? count[i] : 0);
            break;
        }
        const int k = k0 + c;
        float z[V];
        ahead[u].unpack(z);
        if (a.history_ptr) {
            int times[V], any = 0;
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const int4 m = *reinterpret_cast<const int4 *>(count + c + i);
                times[i] = m.x; times[i + 1] = m.y; times[i + 2] = m.z; times[i + 3] = m.w;
                any |= m.x | m.y | m.z | m.w;
            }
            if (any) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (times[i]) z[i] = penalised(a, z[i], times[i]);
            }
        }
        if (a.bias) {
            if (even_bias) {
#pragma unroll
                for (int i = 0; i < V; i += 4) {
                    const float4 b = __ldg(reinterpret_cast<const float4 *>(a.bias + k + i));
                    z[i] += b.x; z[i + 1] += b.y; z[i + 2] += b.z; z[i + 3] += b.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) z[i] += __ldg(a.bias + k + i);
            }
        }
        if (mask) {   // V bits, of two words where they do not lie in one
            const unsigned word = EVEN ? mask[k >> 5] >> (k & 31) : __funnelshift_r(mask[k >> 5], mask[(k + V - 1) >> 5], k & 31);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!(word >> i & 1)) z[i] = minus_inf();
        }
        Pack<T> p;
        p.pack(z);
        *reinterpret_cast<uint4 *>(dst + c) = p.bits;
    }
}

// Anything else by row, in tiles of whole rows (or parts of one): cell i of the tile is class i mod tile_classes; `inverse` is
// 2^32 / tile_classes rounded up (exact for cells below 2^16), 0 for a tile of one row.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) k_adjust_tile(AdjustArgs a, Scores<T> in, Scores<T> out, int tile_rows, int tile_classes, unsigned inverse) {
    extern __shared__ __align__(16) int count[];
    const long long n0 = (long long)blockIdx.x * tile_rows;
    const int k0 = blockIdx.y * tile_classes;
    const int rows = (int)min((long long)tile_rows, a.n - n0), classes = min(tile_classes, a.k - k0);
    if (a.history_ptr) count_histories<ADJUST_MOST_ROWS>(a, n0, rows, k0, classes, count, tile_rows * tile_classes, [&](int r, int c) { return r * tile_classes + c; });
    const unsigned *first_mask = mask_of(a, n0);
#pragma unroll 4
    for (int i = threadIdx.x; i < rows * tile_classes; i += ROW_THREADS) {
        const int r = (int)__umulhi((unsigned)i, inverse), c = i - r * tile_classes;
        if (c >= classes) continue;
        const long long n = n0 + r;
        const int k = k0 + c;
        float z = in(n, k);
        if (a.history_ptr && count[i]) z = penalised(a, z, count[i]);
        if (a.bias) z += a.bias[k];
        const unsigned *mask = tile_rows == 1 ? first_mask : mask_of(a, n);
        if (mask && !(mask[k >> 5] >> (k & 31) & 1)) z = minus_inf();
        *out.at(n, k) = score_from<T>(z);
    }
}

// ------------------------------------------------------------------ top
// A thread per row where there are few classes.  The rows of a block are written together: they lie side by side.
template <typename T, int KP>
__global__ void __launch_bounds__(FEW_THREADS) k_top_few(TopArgs a, Scores<T> in) {
    extern __shared__ float found[];   // FEW_THREADS x top values, then as many classes
    int *found_id = reinterpret_cast<int *>(found + FEW_THREADS * a.top);
    const int tid = threadIdx.x;
    for (long long n0 = (long long)blockIdx.x * FEW_THREADS; n0 < a.n; n0 += (long long)gridDim.x * FEW_THREADS) {
        const long long n = n0 + tid;
        if (n < a.n) {
            float x[KP];
            float m = minus_inf(), s = 0;
            const T *row = in.at(n, 0);
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                x[i] = i < a.k ? score_f32(row[(long long)i * (int)in.cls]) : minus_inf();
                m = fmaxf(m, x[i]);
            }
            const float top = row_top(m);
            if (a.lse) {
#pragma unroll
                for (int i = 0; i < KP; ++i) s += exp2_fast(__fsub_rn(x[i], top) * a.c);
                a.lse[n] = (float)((double)top * a.inv_t + (s == 0.f ? (double)minus_inf() : fine_log(s)));
            }
            float *values = found + tid * a.top;
            int *ids = found_id + tid * a.top;
            if (KP == 8) {   // every score counts those before it: 28 comparisons
                int rank[KP];
#pragma unroll
                for (int i = 0; i < KP; ++i) { x[i] = fmaxf(x[i], minus_inf()); rank[i] = i; }
#pragma unroll
                for (int i = 0; i < KP; ++i)
#pragma unroll
                    for (int j = i + 1; j < KP; ++j) {
                        const int after = x[j] > x[i];
                        rank[i] += after;
                        rank[j] -= after;
                    }
#pragma unroll
                for (int i = 0; i < KP; ++i)
                    if (rank[i] < a.top) { values[rank[i]] = __fadd_rn(x[i], 0.f); ids[rank[i]] = x[i] > minus_inf() ? i : -1; }
                for (int j = KP; j < a.top; ++j) { values[j] = minus_inf(); ids[j] = -1; }
            } else {   // one after the other; a score that is taken becomes -inf
                for (int j = 0; j < a.top; ++j) {
                    float v = minus_inf();
                    int id = -1;
#pragma unroll
                    for (int b = 0; b < KP; b += 16) {
                        if (b >= a.k) break;
#pragma unroll
                        for (int i = b; i < b + 16; ++i)
                            if (x[i] > v) { v = x[i]; id = i; }
                    }
#pragma unroll
                    for (int b = 0; b < KP; b += 16) {
                        if (b >= a.k) break;
#pragma unroll
                        for (int i = b; i < b + 16; ++i)
                            if (i == id) x[i] = minus_inf();
                    }
                    values[j] = __fadd_rn(v, 0.f);
                    ids[j] = id;
                }
            }
        }
        __syncthreads();
        const int cells = (int)min((long long)FEW_THREADS, a.n - n0) * a.top;
        for (int i = tid; i < cells; i += FEW_THREADS) {
            a.values[n0 * a.top + i] = found[i];
            a.ids[n0 * a.top + i] = found_id[i];
        }
        __syncthreads();
    }
}

// A block takes a tile of rows x all classes into shared memory, a warp chooses for one row after the other.  By class: the rows of
// a class are copied side by side, a cell of row r and class c lies at c * (rows + 1) + r, so that neither the copies nor the
// reads along a row meet in a bank.  By row: a warp copies its own rows.  What a warp does for a row is a few hundred
// instructions, and they decide the time: the kernels are made for the number of scores per lane (E, see WarpRow).
constexpr int TILE_ROW_CLASSES = 1024;   // by row: above, a block takes a row
constexpr int TILE_WARPS = 8, TILE_THREADS = 32 * TILE_WARPS, TILE_MOST_ROWS = 32;

template <typename T>
__device__ __noinline__ void load_tile_of(float *tile, const T *p, long long row, long long cls, bool by_class, int rows, int rows_log, int k) {
    auto copy = [](float *to, const T *from) {
        if constexpr (sizeof(T) == 4) copy_async4(to, from);
        else *to = score_f32(*from);
    };
    if (by_class) {
        const int r = threadIdx.x & ((1 << rows_log) - 1), per = TILE_THREADS >> rows_log, c0 = threadIdx.x >> rows_log;
        if (r >= rows) return;
        const T *from = p + r * row + c0 * cls;
        float *to = tile + c0 * ((1 << rows_log) + 1) + r;
        const int step = per * ((1 << rows_log) + 1);
#pragma unroll 8
        for (int c = c0; c < k; c += per, from += per * cls, to += step) copy(to, from);
    } else {
        for (int r = threadIdx.x >> 5; r < rows; r += TILE_WARPS) {
            const int lane = threadIdx.x & 31;
            const T *from = p + r * row + lane * cls;
            float *to = tile + r * k + lane;
#pragma unroll 8
            for (int c = lane; c < k; c += 32, from += 32 * cls, to += 32) copy(to, from);
        }
    }
}
__device__ __forceinline__ void load_tile(float *tile, const ScoreView &v, long long n0, bool by_class, int rows, int rows_log, int k) {
    const long long at = n0 * v.row;
    if (v.type == SCORE_F32) load_tile_of(tile, static_cast<const float *>(v.data) + at, v.row, v.cls, by_class, rows, rows_log, k);
    else if (v.type == SCORE_F16) load_tile_of(tile, static_cast<const __half *>(v.data) + at, v.row, v.cls, by_class, rows, rows_log, k);
    else load_tile_of(tile, static_cast<const __nv_bfloat16 *>(v.data) + at, v.row, v.cls, by_class, rows, rows_log, k);
}

template <int E, int G>
__global__ void __launch_bounds__(TILE_THREADS, E == 32 ? 2 : E == 16 ? 3 : 4) k_top_tile(TopArgs a, bool by_class, int rows_log) {
    extern __shared__ __align__(16) float tile[];
    __shared__ __align__(16) unsigned room[TILE_WARPS][2 * TOP_ROOM * G];
    __shared__ float sums[TILE_MOST_ROWS][2];
    const long long n0 = (long long)blockIdx.x << rows_log;
    const int rows = (int)min(1ll << rows_log, a.n - n0), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    load_tile(tile, a.in, n0, by_class, rows, rows_log, a.k);
    copies_done();
    __syncthreads();
    for (int r = warp; r < rows; r += TILE_WARPS) {
        const WarpRow<E> row(by_class ? tile + r : tile + r * a.k, by_class ? (1 << rows_log) + 1 : 1, a.k);
        if (a.lse) {
            float m = minus_inf(), s = 0;
            row.each([&](float x, int, int) { m = fmaxf(m, x); });
            m = row_top(warp_max(m));
            s = warp_sum(row.exps(m, a.c));
            if (lane == 0) { sums[r][0] = m; sums[r][1] = s; }
        }
        const long long n = n0 + r;
        warp_top<E, G>(row, a.top, room[warp], a.values + n * a.top, a.ids + n * a.top);
    }
    __syncthreads();
    if (a.lse && threadIdx.x < rows) {
        const float m = sums[threadIdx.x][0], s = sums[threadIdx.x][1];
        a.lse[n0 + threadIdx.x] = (float)((double)m * a.inv_t + (s == 0.f ? (double)minus_inf() : fine_log(s)));
    }
}

// A long row: a block takes it, or a cluster of blocks where there are few rows, each a part.  One pass.  From its first packs a
// block learns a border that at least `top` scores reach (of the threads' maxima at least `top` do); only scores that reach it are
// kept, in shared memory, and after some steps the border is raised to what `top` of the kept ones reach: whether one of a warp's
// 256 scores reaches the border decides how long the warp takes for them.  At the end the list is narrowed down until each
// entry can count those before it.  Borders are found by bisection, counting across the block.
// Where the list fills up all the same (ties, or scores that rise along the row), borders order scores and classes at once.

// Four blocks of eight warps per SM: 98 us for 64 of 1024 x 131072 in 16 bits, 107 with three, 137 with five (and fewer registers: with
// four the compiler spills 20 bytes a thread of the 16-bit kernel, 96 of the other).  k_distill_wide, 2048 x 65536 in 16 bits: 123, 119, 140.
constexpr int WIDE_THREADS = 256, WIDE_BLOCKS = 4, WIDE_WARPS = WIDE_THREADS / 32, WIDE_PACKS = 4, WIDE_CLUSTER = 8;
constexpr int WIDE_ROOM = 2048, WIDE_GROUPS = WIDE_THREADS / 2, WIDE_LAST = 256;
static_assert(WIDE_GROUPS >= SCORES_MAX_TOP && WIDE_CLUSTER * SCORES_MAX_TOP <= WIDE_ROOM, "");
typedef unsigned long long Entry;   // score_key << 32 | ~class

struct TopList {
    Entry e[WIDE_ROOM];
    Entry group[WIDE_GROUPS];
    Entry border;              // entries below it cannot be among the `top`
    int count;
};
__device__ __forceinline__ Entry entry_of(float v, int k) { return (Entry)score_key(v) << 32 | (unsigned)~k; }
constexpr Entry LOWEST_ENTRY = (Entry)LOWEST_KEY << 32;   // what is below is no score that can be chosen

// border = the top-th largest of the groups' maxima (every thread has one, those of two neighbours make a group's); all threads
__device__ __forceinline__ void find_border(TopList &l, Entry mine, int top) {
    mine = mine < LOWEST_ENTRY ? 0 : mine;
    mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
    if (!(threadIdx.x & 1)) l.group[threadIdx.x >> 1] = mine;
    __syncthreads();
    if (threadIdx.x < WIDE_GROUPS) {
        const Entry own = l.group[threadIdx.x];
        int above = 0;
#pragma unroll 8
        for (int j = 0; j < WIDE_GROUPS; j += 2) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&l.group[j]);
            above += (o.x > own) + (o.y > own);
        }
        if (own && above == top - 1 && own > l.border) l.border = own;   // (one thread at most: entries differ)
    }
    __syncthreads();
}

// Keeps the entries that reach the border, which is raised to that of their groups first, or (exactly) to the top-th largest entry,
// found bit by bit; all threads.
__device__ __noinline__ void narrow(TopList &l, int top, bool exactly) {
    constexpr int U = WIDE_ROOM / WIDE_THREADS;
    const int m = l.count;
    Entry own[U], most = 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int at = threadIdx.x + i * WIDE_THREADS;
        own[i] = at < m ? l.e[at] : 0;
        most = max(most, own[i]);
    }
    if (exactly) {
        Entry reached = 0;
        for (int bit = 63; bit >= 0; --bit) {
            const Entry trial = reached | 1ull << bit;
            int reach = 0;
#pragma unroll
            for (int i = 0; i < U; ++i) reach += __syncthreads_count(own[i] >= trial);
            if (reach >= top) reached = trial;
        }
        if (threadIdx.x == 0 && reached > l.border) l.border = reached;
        __syncthreads();
    } else {
        find_border(l, most, top);
    }
    if (threadIdx.x == 0) l.count = 0;
    __syncthreads();
    const Entry border = l.border;
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (own[i] >= border) l.e[atomicAdd(&l.count, 1)] = own[i];
    __syncthreads();
}
// (where large entries fall into few groups, the second way leaves no more than `top`, which is within `room`)
__device__ __forceinline__ void narrow_to(TopList &l, int top, int room) {
    bool exactly = false;
    while (l.count > room) {
        const int before = l.count;
        narrow(l, top, exactly);
        exactly = l.count * 2 > before;
    }
}

// Raises `low`, a key that at least `top` of what count() counts reach, towards the largest such key until no more than `enough` do;
// count(key) is the same for all threads.  Returns how many reach it, as far as was counted (`all`: nothing was).
template <typename F>
__device__ __forceinline__ int raise_key(unsigned &low, unsigned high, int top, int enough, int all, F &&count) {
    int reached = all;
    while (reached > enough && low < high) {
        const unsigned mid = low + (high - low + 1) / 2;
        const int c = count(mid);
        if (c >= top) { low = mid; reached = c; }
        else high = mid - 1;
    }
    return reached;
}
// smallest and largest of the threads' keys, for all threads
__device__ __forceinline__ void key_range(unsigned mine, unsigned (*parts)[2], unsigned &low, unsigned &high) {
    low = __reduce_min_sync(0xffffffffu, mine);
    high = __reduce_max_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0) { parts[threadIdx.x >> 5][0] = low; parts[threadIdx.x >> 5][1] = high; }
    __syncthreads();
    low = __reduce_min_sync(0xffffffffu, parts[threadIdx.x & (WIDE_WARPS - 1)][0]);
    high = __reduce_max_sync(0xffffffffu, parts[threadIdx.x & (WIDE_WARPS - 1)][1]);
}
// The border that `enough` or a few more of the list's entries reach, by their keys; drops the others if asked to.  All threads, with a
// barrier before; the list is not full.
__device__ __noinline__ void raise_border(TopList &l, int top, int enough, bool drop, unsigned (*parts)[2]) {
    constexpr int U = WIDE_ROOM / WIDE_THREADS;
    const int m = l.count;
    unsigned key[U], most = 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int at = threadIdx.x + i * WIDE_THREADS;
        key[i] = at < m ? (unsigned)(l.e[at] >> 32) : 0u;
        most = max(most, key[i]);
    }
    unsigned low, high;
    key_range(most, parts, low, high);
    low = (unsigned)(l.border >> 32);
    const int left = raise_key(low, high, top, enough, m, [&](unsigned mid) {
        int c = 0;
        for (int i = 0; i < U && i * WIDE_THREADS < m; ++i) c += __syncthreads_count(key[i] >= mid);
        return c;
    });
    if (!drop) {
        if (threadIdx.x == 0 && (Entry)low << 32 > l.border) l.border = (Entry)low << 32;
        __syncthreads();
        return;
    }
    if (left == m) return;
    Entry own[U];
#pragma unroll
    for (int i = 0; i < U; ++i) own[i] = key[i] >= low && key[i] ? l.e[threadIdx.x + i * WIDE_THREADS] : 0;
    __syncthreads();
    if (threadIdx.x == 0) {
        l.count = 0;
        if ((Entry)low << 32 > l.border) l.border = (Entry)low << 32;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < U; ++i)
        if (own[i]) l.e[atomicAdd(&l.count, 1)] = own[i];
    __syncthreads();
}

// A step's scores have filled the list: the border is raised to that of the step's own threads' maxima and the list narrowed, then the
// scores that found no room (`dropped`, the thread's V * WIDE_PACKS cells) are put in, a warp at a time.  The scores are read again: this
// is rare, and the registers are needed elsewhere.
template <typename T>
__device__ __noinline__ void make_room(TopList &l, int top, const T *cells, int packs, int k0, unsigned dropped) {
    constexpr int V = Pack<T>::V, WARP_CELLS = 32 * WIDE_PACKS * V;
    static_assert(WIDE_LAST + WARP_CELLS <= WIDE_ROOM, "");
    auto each = [&](auto &&f) {
        for (int u = 0; u < WIDE_PACKS; ++u) {
            const int at = u * WIDE_THREADS + threadIdx.x;
            if (at >= packs) break;
            for (int i = 0; i < V; ++i) f(u * V + i, entry_of(score_f32(cells[at * V + i]), k0 + at * V + i));
        }
    };
    Entry most = 0;
    each([&](int, Entry e) { most = max(most, e); });
    if (threadIdx.x == 0) l.count = min(l.count, WIDE_ROOM);
    find_border(l, most, top);
    narrow_to(l, top, WIDE_LAST);
    for (int turn = 0; turn < WIDE_WARPS; ++turn) {
        const bool full = l.count > WIDE_ROOM - WARP_CELLS;
        __syncthreads();
        if (full) {
            narrow_to(l, top, WIDE_LAST);
            __syncthreads();   // (its last step reads the count, which the warp below raises)
        }
        const Entry border = l.border;
        if ((int)(threadIdx.x >> 5) == turn && dropped)
            each([&](int bit, Entry e) {
                if ((dropped >> bit & 1) && e >= border) l.e[atomicAdd(&l.count, 1)] = e;
            });
        __syncthreads();
    }
}

template <typename T>
__global__ void __launch_bounds__(WIDE_THREADS, WIDE_BLOCKS) k_top_wide(TopArgs a, Scores<T> in) {
    constexpr int V = Pack<T>::V, STEP = WIDE_THREADS * WIDE_PACKS;
    __shared__ __align__(16) TopList l;
    __shared__ Entry best[SCORES_MAX_TOP];
    __shared__ float parts[WIDE_WARPS][2], whole[2];
    __shared__ unsigned ranges[WIDE_WARPS][2];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long n = blockIdx.x / C;
    const int per = (a.k + C - 1) / C, lo = min(a.k, rank * per), hi = min(a.k, lo + per);
    const Part<T> part(in.at(n, 0), lo, hi);
    const uint4 *body = part.body();
    uint4 w[WIDE_PACKS], ahead[WIDE_PACKS];
    auto fetch = [&](int from) {
#pragma unroll
        for (int u = 0; u < WIDE_PACKS; ++u)
            if (from + u * WIDE_THREADS + tid < part.packs) ahead[u] = __ldg(body + from + u * WIDE_THREADS + tid);
    };
    fetch(0);
    if (tid == 0) { l.count = 0; l.border = LOWEST_ENTRY; }
    __syncthreads();
    Entry border = LOWEST_ENTRY;
    float border_score = -FLT_MAX;
    Running<false> run;
    int last = 0;   // where this thread's last entry went
    auto push = [&](Entry e) {
        last = atomicAdd(&l.count, 1);
        if (last < WIDE_ROOM) l.e[last] = e;
        return last < WIDE_ROOM;
    };
    if (tid < part.head + part.tail) {   // cells of no pack, 2 V - 2 at most
        const int k = part.single(tid);
        const float x = score_f32(part.p[k]);
        run.raise(x, a.c);
        run.add(x, row_top(run.m), a.c);
        const Entry e = entry_of(x, lo + k);
        if (e >= LOWEST_ENTRY) push(e);
    }
    __syncthreads();
    for (int from = 0; from < part.packs; from += STEP) {
#pragma unroll
        for (int u = 0; u < WIDE_PACKS; ++u) w[u] = ahead[u];
        fetch(from + STEP);
        auto has = [&](int u) { return from + u * WIDE_THREADS + tid < part.packs; };
        auto each = [&](int u, auto &&f) {   // f(bit of the cell, score, class)
            Pack<T> p;
            p.bits = w[u];
            float v[V];
            p.unpack(v);
            const int k = lo + part.head + (from + u * WIDE_THREADS + tid) * V;
#pragma unroll
            for (int i = 0; i < V; ++i) f(u * V + i, v[i], k + i);
        };
        const int turn = from / STEP;
        if (turn == 0 && part.packs * V > WIDE_ROOM / 2) {
            float largest = minus_inf();
#pragma unroll
            for (int u = 0; u < WIDE_PACKS; ++u)
                if (has(u)) each(u, [&](int, float x, int) { largest = fmaxf(largest, x); });
            const unsigned mine = score_key(largest);
            unsigned low, high;
            key_range(mine, ranges, low, high);
            low = max(low, (unsigned)(LOWEST_ENTRY >> 32));
            raise_key(low, high, a.top, a.top + a.top / 4, WIDE_THREADS, [&](unsigned mid) { return __syncthreads_count(mine >= mid); });
            border = (Entry)low << 32;
            if (tid == 0) l.border = border;   // (read behind the next barrier)
        } else if (turn == 3 || turn == 7) {   // (never: 123 us for 64 of 1024 x 131072; behind 1, 2, 4 and 8 steps: 101; like this: 98)
            __syncthreads();
            raise_border(l, a.top, a.top + a.top / 4, false, ranges);
            border = l.border;
        }
        if (border > LOWEST_ENTRY) border_score = key_score((unsigned)(border >> 32));
        unsigned dropped = 0;
        last = 0;
#pragma unroll
        for (int u = 0; u < WIDE_PACKS; ++u) {
            if (!has(u)) break;
            float v[V];
            Pack<T> p;
            p.bits = w[u];
            p.unpack(v);
            float largest = v[0];
#pragma unroll
            for (int i = 1; i < V; ++i) largest = fmaxf(largest, v[i]);
            run.add_pack(v, a.c);
            if (largest >= border_score) {   // few of a lane's V scores, but most often one of some lane's
                unsigned reach = 0;
#pragma unroll
                for (int i = 0; i < V; ++i) reach |= v[i] >= border_score ? 1u << i : 0u;
                while (reach) {
                    const int i = __ffs(reach) - 1;
                    reach &= reach - 1;
                    float x = v[0];
#pragma unroll
                    for (int j = 1; j < V; ++j) x = i == j ? v[j] : x;
                    const Entry e = entry_of(x, lo + part.head + (from + u * WIDE_THREADS + tid) * V + i);
                    if (e >= border && !push(e)) dropped |= 1u << (u * V + i);
                }
            }
        }
        if (__syncthreads_or(last >= WIDE_ROOM * 3 / 4)) {   // all threads see the same: the list is full, or soon will be
            make_room(l, a.top, part.p + part.head + (long long)from * V, part.packs - from, lo + part.head + from * V, dropped);
            border = l.border;
            border_score = border > LOWEST_ENTRY ? key_score((unsigned)(border >> 32)) : -FLT_MAX;
        }
    }
    __syncthreads();
    if (l.count > WIDE_LAST) raise_border(l, a.top, WIDE_LAST, true, ranges);
    narrow_to(l, a.top, WIDE_LAST);
    run.join_warp(a.c);
    if (lane == 0) { parts[warp][0] = run.m; parts[warp][1] = run.s; }
    const int m = l.count;
    if (tid < SCORES_MAX_TOP) best[tid] = 0;
    if (tid == 0 && (m & 1)) l.e[m] = 0;   // (m < WIDE_ROOM; read in twos)
    __syncthreads();
    if (tid < m) {
        const Entry own = l.e[tid];
        int before = 0;
        for (int j = 0; j < m; j += 2) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&l.e[j]);
            before += (o.x > own) + (o.y > own);
        }
        if (before < a.top) best[before] = own;
    }
    if (warp == 0) {
        Running<false> all;
        if (lane < WIDE_WARPS) { all.m = parts[lane][0]; all.s = parts[lane][1]; }
        all.join_warp(a.c);
        if (lane == 0) { whole[0] = all.m; whole[1] = all.s; }
    }
    auto give = [&](int j, Entry e) {
        a.values[n * a.top + j] = key_score((unsigned)(e >> 32));
        a.ids[n * a.top + j] = e ? (int)~(unsigned)e : -1;
    };
    auto give_lse = [&](const Running<false> &r) {
        if (a.lse) a.lse[n] = (float)((double)row_top(r.m) * a.inv_t + (r.s == 0.f ? (double)minus_inf() : fine_log(r.s)));
    };
    if (C == 1) {
        __syncthreads();
        if (tid < a.top) give(tid, best[tid]);
        if (tid == WIDE_THREADS - 1) {
            Running<false> r;
            r.m = whole[0]; r.s = whole[1];
            give_lse(r);
        }
        return;
    }
    cluster.sync();
    if (rank == 0) {
        // the parts' lists, each in order: an entry's place is its own plus that among the others
        for (int i = tid; i < C * a.top; i += WIDE_THREADS) l.e[i] = *cluster.map_shared_rank(&best[i % a.top], i / a.top);
        __syncthreads();
        int found = 0;
        for (int i0 = 0; i0 < C * a.top; i0 += WIDE_THREADS) {
            const int i = i0 + tid;
            const Entry own = i < C * a.top ? l.e[i] : 0;
            if (own) {
                int before = i % a.top;
                for (int c = 0; c < C; ++c) {
                    if (c == i / a.top) continue;
                    int x = 0, y = a.top;   // entries [0, x) are larger, [y, top) are not
                    while (x < y) {
                        const int mid = (x + y) / 2;
                        if (l.e[c * a.top + mid] > own) x = mid + 1; else y = mid;
                    }
                    before += x;
                }
                if (before < a.top) give(before, own);
            }
            found += __syncthreads_count(own != 0);
        }
        if (tid >= found && tid < a.top) give(tid, 0);
        if (tid == 0) {
            Running<false> r;
            for (int c = 0; c < C; ++c) {
                const float *o = cluster.map_shared_rank(whole, c);
                r.join(o[0], o[1], 0.f, a.c);
            }
            give_lse(r);
        }
    }
    cluster.sync();   // (the others' shared memory is read until here)
}

// A block per row: the largest of the keys below the last one chosen, again and again.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) k_top_any(TopArgs a, Scores<T> in) {
    __shared__ unsigned long long best[ROW_THREADS / 32];
    __shared__ float part[ROW_THREADS / 32];
    const long long n = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = minus_inf();
    bool broken = false;
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
        const float v = in(n, k);
        m = fmaxf(m, v);
        broken |= v != v;
    }
    m = warp_max(m);
    if (lane == 0) part[warp] = m;
    broken = __syncthreads_or(broken);
    m = row_top(warp_max(part[lane & (ROW_THREADS / 32 - 1)]));
    __syncthreads();
    if (a.lse) {
        float s = 0;
        for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) s += exp2_fast(__fsub_rn(in(n, k), m) * a.c);
        s = warp_sum(s);
        if (lane == 0) part[warp] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            s = 0;
            for (int w = 0; w < ROW_THREADS / 32; ++w) s += part[w];
            a.lse[n] = broken ? __int_as_float(0x7fffffff) : (float)((double)m * a.inv_t + (s == 0.f ? (double)minus_inf() : fine_log(s)));
        }
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.top; ++j) {
        unsigned long long b = 0;
        for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
            const unsigned key = score_key(in(n, k));
            const unsigned long long v = (unsigned long long)key << 32 | (unsigned)~k;
            if (key && v < last && v > b) b = v;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
        __syncthreads();
        if (lane == 0) best[warp] = b;
        __syncthreads();
        for (int w = 0; w < ROW_THREADS / 32; ++w) b = max(b, best[w]);
        last = b;
        if (threadIdx.x == 0) {
            a.values[n * a.top + j] = key_score((unsigned)(b >> 32));
            a.ids[n * a.top + j] = b ? (int)~(unsigned)b : -1;
        }
    }
}

// ------------------------------------------------------------------ distill
// A block per row.  The classes that the teacher lists are marked in a bit map.
template <typename T, bool TWO>
__global__ void __launch_bounds__(ROW_THREADS) k_distill_any(DistillArgs a, Scores<T> in) {
    extern __shared__ unsigned listed_bits[];
    __shared__ TeacherSide teacher;
    __shared__ int list_id[SCORES_MAX_TOP];
    __shared__ float list_q[SCORES_MAX_TOP];
    __shared__ StudentRow student;
    __shared__ DistillRow drow;
    __shared__ float part[3][ROW_THREADS / 32];
    const long long n = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, W = ROW_THREADS / 32;
    const double inv_t = a.inv_t;
    const float c = a.c;
    for (int i = threadIdx.x; i < (a.k + 31) / 32; i += ROW_THREADS) listed_bits[i] = 0;
    __syncthreads();
    if (warp == 0) {
        const TeacherSide t = read_teacher(a, n, list_id, list_q);
        if (lane == 0) teacher = t;
        for (int j = lane; j < a.top; j += 32)
            if (list_id[j] >= 0) atomicOr(&listed_bits[list_id[j] >> 5], 1u << (list_id[j] & 31));
    }
    __syncthreads();
    auto is_listed = [&](int k) { return listed_bits[k >> 5] >> (k & 31) & 1; };
    float m = minus_inf();
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS)
        if (!is_listed(k)) m = fmaxf(m, in(n, k));
    m = warp_max(m);
    if (lane == 0) part[0][warp] = m;
    __syncthreads();
    const float base = row_top(warp_max(part[0][lane & (W - 1)]));
    float s = 0, s1 = 0;
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS)
        if (!is_listed(k)) {
            const float x = __fsub_rn(in(n, k), base);
            s += exp2_fast(x * c);
            if (TWO) s1 += exp2_fast(x * LOG2E);
        }
    s = warp_sum(s); s1 = warp_sum(s1);
    if (lane == 0) { part[1][warp] = s; part[2][warp] = s1; }
    __syncthreads();
    if (warp == 0) {
        s = lane < W ? part[1][lane] : 0.f; s1 = lane < W ? part[2][lane] : 0.f;
        s = warp_sum(s); s1 = warp_sum(s1);
        if (!TWO) s1 = s;
        StudentRow st;
        st.base = base; st.rest = s; st.rest1 = s1;
        float top = s > 0.f || s != s ? base : minus_inf();
        for (int j = lane; j < a.top; j += 32)
            if (list_id[j] >= 0) top = fmaxf(top, in(n, list_id[j]));
        st.top = row_top(warp_max(top));
        st.base = reference_of(st.base, st.rest, st.top);
        float l = 0, l1 = 0;
        double ql = 0;
        for (int j = lane; j < a.top; j += 32)
            if (list_id[j] >= 0) {
                const float z = in(n, list_id[j]), x = __fsub_rn(z, st.top);
                l += exp2_fast(x * c);
                if (TWO) l1 += exp2_fast(x * LOG2E);
                if (list_q[j] != 0.f) ql += (double)list_q[j] * (((double)z - (double)st.top) * inv_t);
            }
        l = warp_sum(l); l1 = warp_sum(l1);
        if (!TWO) l1 = l;
        ql = warp_sum(ql);
        const float low = __fsub_rn(st.base, st.top);
        st.l = l;
        st.sum = s * exp2_fast(low * c) + l;
        st.sum1 = TWO ? s1 * exp2_fast(low * LOG2E) + l1 : st.sum;
        if (lane == 0) {
            const float w = a.weights ? a.weights[n] : 1.f;
            const int label = row_label(a, n);
            student = st;
            drow = distill_row(a, teacher, st, w, label);
            if (a.loss) a.loss[n] = distill_loss(a, teacher, st, w, label, ql, label >= 0 ? in(n, label) : 0.f);
        }
    }
    __syncthreads();
    float mg = 0, mh = 0;
    if (a.gives != GIVES_LOSS) {
        const DistillRow d = drow;
        auto put = [&](int k, float2 gh) {
            const long long at = n * a.out.row + k * a.out.cls;
            if (a.gives == GIVES_PAIRS) static_cast<float2 *>(a.out.data)[at] = gh;
            else static_cast<T *>(a.out.data)[at] = score_from<T>(gh.x);
            mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y);
        };
        for (int k = threadIdx.x; k < a.k; k += ROW_THREADS)
            if (!is_listed(k)) put(k, other_gh<TWO>(d, k, in(n, k)));
        for (int j = threadIdx.x; j < a.top; j += ROW_THREADS)
            if (list_id[j] >= 0) put(list_id[j], listed_gh<TWO>(d, list_id[j], in(n, list_id[j]), list_q[j]));
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

// A thread per row where there are few classes: the row's scores and exponentials stay in registers, what the teacher says of a class
// in a column of shared memory (a class that is listed twice holds the sum).  Rows of a class are read side by side.  Instructions
// decide the time, some 1130 per 32 rows of 7 classes: what is only needed for repeats, or for a rest, is branched around.  (Eight blocks
// per SM for up to 8 classes; with two temperatures the compiler spills 44 bytes a thread then.)
template <typename T, int KP, bool TWO>
__global__ void __launch_bounds__(FEW_THREADS, KP == 8 ? 8 : KP == 16 ? 5 : 4) k_distill_few(DistillArgs a, Scores<T> in) {
    constexpr int ENTRIES = 4;   // entries of a list that stay in registers
    constexpr bool KEEP = KP <= 16;   // ... and exponentials
    __shared__ float qs[KP][FEW_THREADS];
    const int tid = threadIdx.x, K = a.k, in_cls = (int)in.cls, out_cls = (int)a.out.cls;
    const float inv_t = (float)a.inv_t;
    float mg = 0, mh = 0;
    for (long long n = (long long)blockIdx.x * FEW_THREADS + tid; n < a.n; n += (long long)gridDim.x * FEW_THREADS) {
        float x[KP];
        const T *row = in.at(n, 0);
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            x[i] = i < K ? score_f32(row[(long long)i * in_cls]) : minus_inf();
            qs[i][tid] = 0.f;
        }
        // the teacher
        const int *ids = a.ids + n * a.ids_stride;
        int id4[ENTRIES];
        float t4[ENTRIES];
#pragma unroll
        for (int e = 0; e < ENTRIES; ++e) {
            id4[e] = e < a.top ? ids[e] : -1;
            t4[e] = e < a.top ? teacher_logit(a, n, e) : 0.f;
        }
        auto each_entry = [&](auto &&f) {   // f(class, score)
#pragma unroll
            for (int e = 0; e < ENTRIES; ++e)
                if ((unsigned)id4[e] < (unsigned)K) f(id4[e], t4[e]);
            for (int e = ENTRIES; e < a.top; ++e) {
                const int id = ids[e];
                if ((unsigned)id < (unsigned)K) f(id, teacher_logit(a, n, e));
            }
        };
        TeacherSide t;
        unsigned listed = 0, repeats = 0;
        float best = minus_inf();
        bool broken = false;
        each_entry([&](int id, float l) {
            broken |= l != l;
            best = fmaxf(best, l);
            repeats |= listed & 1u << id;
            listed |= 1u << id;
        });
        const bool none = best == minus_inf() && !broken;
        double mass = 0, entropy = 0;
        float q_scale = 1.f;   // q = qs * q_scale
        t.rest = 0.f;
        t.total = none ? 0.f : 1.f;
        if (none) {
            listed = 0;
        } else if (a.lse) {
            const double L = (double)a.lse[n];
            each_entry([&](int id, float l) {
                const double lq = (double)l * a.inv_t - L, q = exp(lq);
                mass += q;
                if (q > 0) entropy += q * lq;
                qs[id][tid] += (float)q;
            });
            const double rest = __popc(listed) < K && mass < 1 ? 1.0 - mass : 0.0;
            t.rest = (float)rest;
            t.total = (float)(mass + rest);
        } else {
            float sum = 0, far = 0;
            each_entry([&](int id, float l) {
                const float e = fine_exp(l, best, a.c, a.c_low);
                sum += e;
                if (e > 0.f) far = __fmaf_rn(e, __fsub_rn(l, best) * inv_t, far);
                qs[id][tid] += e;
            });
            q_scale = fast_inverse(sum);
            mass = 1;
            if (a.loss) entropy = (double)(far * q_scale) - fine_log(sum);
        }
        if (repeats && a.loss && !none) {   // a class's share of the entropy is that of the sum
            entropy = 0;
            for (unsigned left = listed; left; left &= left - 1) {
                const float q = qs[__ffs(left) - 1][tid] * q_scale;
                if (q != 0.f) entropy += (double)q * log((double)q);
            }
        }
        // the student: the listed classes apart where the rest is a class of its own
        const unsigned apart = t.rest > 0.f ? listed : 0u;
        StudentRow s;
        float m = minus_inf(), mt = minus_inf();
#pragma unroll
        for (int i = 0; i < KP; ++i) mt = fmaxf(mt, x[i]);
        m = mt;
        if (apart) {
            m = minus_inf();
#pragma unroll
            for (int i = 0; i < KP; ++i)
                if (!(apart >> i & 1)) m = fmaxf(m, x[i]);
        }
        s.top = row_top(mt);
        s.base = row_top(m);
        s.rest = s.rest1 = 0.f;
        float l = 0, l1 = 0, e[KEEP ? KP : 1], e1[KEEP && TWO ? KP : 1];
        if (!apart) {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                const float d = __fsub_rn(x[i], s.base), v = exp2_fast(d * a.c), v1 = TWO ? exp2_fast(d * LOG2E) : 0.f;
                s.rest += v;
                if (TWO) s.rest1 += v1;
                if (KEEP) e[i] = v;
                if (KEEP && TWO) e1[i] = v1;
            }
        } else {
#pragma unroll
            for (int i = 0; i < KP; ++i) {   // (relative to the largest of its kind, as in StudentRow)
                const bool of_rest = !(apart >> i & 1);
                const float d = __fsub_rn(x[i], of_rest ? s.base : s.top), v = exp2_fast(d * a.c), v1 = TWO ? exp2_fast(d * LOG2E) : 0.f;
                if (of_rest) { s.rest += v; s.rest1 += v1; } else { l += v; l1 += v1; }
                if (KEEP) e[i] = v;
                if (KEEP && TWO) e1[i] = v1;
            }
        }
        s.base = reference_of(s.base, s.rest, s.top);
        const float low = __fsub_rn(s.base, s.top);
        s.l = l;
        s.sum = apart ? s.rest * exp2_fast(low * a.c) + l : s.rest;
        s.sum1 = !TWO ? s.sum : apart ? s.rest1 * exp2_fast(low * LOG2E) + l1 : s.rest1;
        const float w = a.weights ? a.weights[n] : 1.f;
        const int label = row_label(a, n);
        const DistillRow d = distill_row(a, t, s, w, label);
        double of_listed = 0;
        float label_score = 0;
        if (a.loss) {
#pragma unroll
            for (int i = 0; i < KP; ++i) {
                if (i == label) label_score = x[i];
                if (listed >> i & 1) {
                    const float q = qs[i][tid] * q_scale;
                    if (q != 0.f) of_listed += (double)(q * inv_t) * ((double)x[i] - (double)s.top);
                }
            }
            t.entropy = entropy;
            t.mass = mass;
            a.loss[n] = distill_loss(a, t, s, w, label, of_listed, label_score);
        }
        if (a.gives == GIVES_LOSS) continue;
        const long long at = n * a.out.row;
        float2 *pairs = static_cast<float2 *>(a.out.data) + at;
        T *grads = static_cast<T *>(a.out.data) + at;
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            if (i >= K) break;
            const bool as_listed = apart == 0 || (apart >> i & 1);   // (a class that is not listed has q = 0)
            float v, v1 = 0.f;
            if (KEEP) {
                v = e[i];
                if (TWO) v1 = e1[i];
            } else {
                const float far = __fsub_rn(x[i], as_listed ? s.top : s.base);
                v = exp2_fast(far * a.c);
                if (TWO) v1 = exp2_fast(far * LOG2E);
            }
            const float p = v * (as_listed ? d.inv_sum : d.to_p), p1 = TWO ? v1 * (as_listed ? d.inv_sum1 : d.to_p1) : p;
            const float g = as_listed ? d.soft * __fmaf_rn(d.total, p, -(qs[i][tid] * q_scale)) : v * d.to_g;
            const float2 gh = finish_gh(d, i, g, p, p1);
            if (a.gives == GIVES_PAIRS) pairs[(long long)i * out_cls] = gh;
            else grads[(long long)i * out_cls] = score_from<T>(gh.x);
            mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y);
        }
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

// A tile as in k_top_tile: the teacher's lists are read while the scores are on their way, a warp sums up one row after the other, a
// lane each finds the rows' losses and the factors of their gradients, and the gradients of unlisted classes are written the way the
// scores were read.  The cells of listed classes and labels, a few per row, are written over them: to tell them apart in that pass
// took half of its instructions.
template <int E, bool TWO, int S>
__global__ void __launch_bounds__(TILE_THREADS, E == 32 ? 2 : 4) k_distill_tile(DistillArgs a, bool by_class, int rows_log) {
    extern __shared__ __align__(16) float tile[];
    const int R = 1 << rows_log, step = by_class ? R + 1 : 1;
    int *list_id = reinterpret_cast<int *>(tile + (size_t)a.k * (by_class ? R + 1 : R));
    float *list_q = reinterpret_cast<float *>(list_id + R * a.top), *list_x = list_q + R * a.top;
    __shared__ RowSums sums[TILE_MOST_ROWS];
    __shared__ float lse[TILE_MOST_ROWS];
    __shared__ DistillRow factors[TILE_MOST_ROWS];
    __shared__ float label_scores[TILE_MOST_ROWS];
    const long long n0 = (long long)blockIdx.x << rows_log;
    const int rows = (int)min((long long)R, a.n - n0), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    load_tile(tile, a.in, n0, by_class, rows, rows_log, a.k);
    // the lists of this warp's rows: classes to list_id, the teacher's scores to list_x for now
    for (int r = warp; r < rows; r += TILE_WARPS)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int e = lane + 32 * s;
            if (e >= a.top) continue;
            copy_async4(reinterpret_cast<float *>(list_id + r * a.top + e), reinterpret_cast<const float *>(a.ids + (n0 + r) * a.ids_stride + e));
            if (a.logits_type == SCORE_F32) copy_async4(list_x + r * a.top + e, static_cast<const float *>(a.logits) + (n0 + r) * a.logits_stride + e);
            else list_x[r * a.top + e] = teacher_logit(a, n0 + r, e);
        }
    if (threadIdx.x < rows) lse[threadIdx.x] = a.lse ? a.lse[n0 + threadIdx.x] : 0.f;
    copies_done();
    __syncthreads();
    for (int r = warp; r < rows; r += TILE_WARPS) {
        int id[S];
        float t[S], q[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int e = lane + 32 * s, i = e < a.top ? list_id[r * a.top + e] : -1;
            id[s] = i >= 0 && i < a.k ? i : -1;
            t[s] = e < a.top ? list_x[r * a.top + e] : 0.f;
        }
        const TeacherSide side = teacher_of<S>(a, a.lse ? lse + r : nullptr, id, t, q, true);
        if (lane == 0) sums[r].teacher = side;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int e = lane + 32 * s;
            if (e < a.top) { list_id[r * a.top + e] = id[s]; list_q[r * a.top + e] = q[s]; }
        }
        __syncwarp();
        warp_student<E, TWO, S>(a, n0 + r, by_class ? tile + r : tile + r * a.k, step, list_id + r * a.top, list_q + r * a.top, list_x + r * a.top, sums[r]);
    }
    __syncthreads();
    if (threadIdx.x < rows) {
        const RowSums &r = sums[threadIdx.x];
        const long long n = n0 + threadIdx.x;
        const StudentRow s = student_of(a, r);
        const float w = a.weights ? a.weights[n] : 1.f;
        const int label = row_label(a, n);
        if (a.gives != GIVES_LOSS) {
            factors[threadIdx.x] = distill_row(a, r.teacher, s, w, label);
            if (label >= 0) {   // (as the listed classes' cells are: in the pass it gets, and notes, nothing)
                float *cell = by_class ? tile + label * step + threadIdx.x : tile + threadIdx.x * a.k + label;
                label_scores[threadIdx.x] = *cell;
                *cell = minus_inf();
            }
        }
        if (a.loss) a.loss[n] = distill_loss(a, r.teacher, s, w, label, r.of_listed, r.label_score);
    }
    if (a.gives == GIVES_LOSS) return;
    __syncthreads();
    float mg = 0, mh = 0;
    const int cls = (int)a.out.cls;   // (the launch sees to it)
    const bool track = a.maxbits != nullptr;
    auto note = [&](float2 gh) {
        if (track) { mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y); }
        return gh;
    };
    // cells from `first` on, `per` apart, of row r
    auto write = [&](int r, const float *z, int first, int per) {
        DistillRow d = factors[r];
        d.label = -1;
        const long long at = (n0 + r) * a.out.row + (long long)first * cls, apart = (long long)per * cls;
        const float *from = z + first * step;
        const int cells = (a.k - first + per - 1) / per, next = per * step;
        if (a.gives == GIVES_PAIRS) {
            float2 *to = static_cast<float2 *>(a.out.data) + at;
#pragma unroll 4
            for (int c = 0; c < cells; ++c, from += next, to += apart) *to = note(other_gh<TWO>(d, 0, *from));
        } else if (a.out.type == SCORE_F32) {
            float *to = static_cast<float *>(a.out.data) + at;
#pragma unroll 4
            for (int c = 0; c < cells; ++c, from += next, to += apart) *to = note(other_gh<TWO>(d, 0, *from)).x;
        } else {
            const bool half = a.out.type == SCORE_F16;
            unsigned short *to = static_cast<unsigned short *>(a.out.data) + at;
#pragma unroll 4
            for (int c = 0; c < cells; ++c, from += next, to += apart) {
                const float g = note(other_gh<TWO>(d, 0, *from)).x;
                *to = half ? __half_as_ushort(__float2half_rn(g)) : __bfloat16_as_ushort(__float2bfloat16_rn(g));
            }
        }
    };
    auto put = [&](int r, int c, float2 gh) {
        note(gh);
        const long long at = (n0 + r) * a.out.row + (long long)c * cls;
        if (a.gives == GIVES_PAIRS) static_cast<float2 *>(a.out.data)[at] = gh;
        else if (a.out.type == SCORE_F32) static_cast<float *>(a.out.data)[at] = gh.x;
        else static_cast<unsigned short *>(a.out.data)[at] = a.out.type == SCORE_F16 ? __half_as_ushort(__float2half_rn(gh.x)) : __bfloat16_as_ushort(__float2bfloat16_rn(gh.x));
    };
    if (by_class) {
        const int r = threadIdx.x & (R - 1), c = threadIdx.x >> rows_log;
        if (r < rows && c < a.k) write(r, tile + r, c, TILE_THREADS >> rows_log);
    } else {
        for (int r = warp; r < rows; r += TILE_WARPS) write(r, tile + r * a.k, lane, 32);
    }
    __syncthreads();   // what follows is written over it
    // an entry of a list each, then the labels that are not listed
    const float inv_top = 1.f / (float)a.top;
    for (int i = threadIdx.x; i < rows * a.top; i += TILE_THREADS) {
        const int c = list_id[i], r = (int)(((float)i + 0.5f) * inv_top);   // i / top: half a cell is far more than the product is off
        if (c >= 0) put(r, c, listed_gh<TWO>(factors[r], c, list_x[i], list_q[i]));
    }
    if (threadIdx.x < rows && factors[threadIdx.x].label >= 0) {
        const int r = threadIdx.x, c = factors[r].label;
        int e = 0;
        while (e < a.top && list_id[r * a.top + e] != c) ++e;
        if (e == a.top) put(r, c, other_gh<TWO>(factors[r], c, label_scores[r]));
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

// By class, up to 1024 classes: a lane per row and E neighbouring classes per warp, whose scores stay in registers from the first read to
// the gradients.  Rows are read and written side by side, and nothing is reduced within a warp: the warps of a block exchange a maximum
// and sums per row.  What the lists say is worked out by as many threads per row as there are warps.  (A warp per row from a tile in
// shared memory took 985 instructions per row of 250 classes, and they decided its time: 65 us for 50003 of them; these are 52, with
// three blocks per SM instead of four 54, with five (and fewer registers) 68.  With four the compiler spills 24 to 44 bytes a thread where a
// warp has 32 classes.)
// The cells of listed classes and labels are written over what they get with the others.
constexpr int CLASS_ROWS = 32;

struct ListSums {   // of a row's list
    TeacherSide teacher;
    double of_listed;      // sum of q (s - top) / T
    float top, l, l1;      // largest of the listed scores, sums of exponentials relative to it
    int repeats;           // a class stands in it twice
};

template <typename T, int E, int W, bool TWO>
__global__ void __launch_bounds__(32 * W, W == 8 ? 4 : W == 16 ? 2 : 1) k_distill_class(DistillArgs a, Scores<T> in) {
    constexpr int THREADS = 32 * W;
    extern __shared__ float lists[];
    __shared__ unsigned bits[W][CLASS_ROWS];
    __shared__ float part[3][W][CLASS_ROWS];
    __shared__ ListSums of_list[CLASS_ROWS];
    __shared__ DistillRow factors[CLASS_ROWS];
    __shared__ StudentRow students[CLASS_ROWS];
    __shared__ int labels[CLASS_ROWS];
    __shared__ float lse[CLASS_ROWS], weights[CLASS_ROWS], label_scores[CLASS_ROWS];
    int *list_id = reinterpret_cast<int *>(lists);               // CLASS_ROWS x top: -1 for none
    float *list_q = lists + CLASS_ROWS * a.top, *list_x = list_q + CLASS_ROWS * a.top;   // (first the teacher's scores, then masses)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = a.k, in_cls = (int)in.cls, out_cls = (int)a.out.cls;
    const long long n0 = (long long)blockIdx.x * CLASS_ROWS;
    const int rows = (int)min((long long)CLASS_ROWS, a.n - n0), k0 = warp * E;
    const long long n = n0 + min(lane, rows - 1);
    float x[E];
    {
        const T *from = in.at(n, k0);
        T raw[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (k0 + j < K) raw[j] = from[(long long)j * in_cls];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = k0 + j < K ? score_f32(raw[j]) : minus_inf();
    }
    bits[warp][lane] = 0;
    if (tid >= THREADS - CLASS_ROWS) {   // (what the rows give besides, read while the scores are on their way)
        const int label = row_label(a, n);
        of_list[lane].repeats = 0;
        labels[lane] = label;
        lse[lane] = a.lse ? a.lse[n] : 0.f;
        weights[lane] = a.weights ? a.weights[n] : 1.f;
        label_scores[lane] = label >= 0 ? in(n, label) : 0.f;
    }
    __syncthreads();
    const float inv_top = 1.f / (float)a.top;
    auto row_of = [&](int i) { return (int)(((float)i + 0.5f) * inv_top); };   // i / top: half a cell is far more than the product is off
    for (int i = tid; i < rows * a.top; i += THREADS) {
        const int r = row_of(i), e = i - r * a.top;
        int id = a.ids[(n0 + r) * a.ids_stride + e];
        if (id < 0 || id >= K) id = -1;
        list_id[i] = id;
        list_q[i] = teacher_logit(a, n0 + r, e);
        if (id >= 0) {
            const unsigned bit = 1u << (id % E);
            if (atomicOr(&bits[id / E][r], bit) & bit) of_list[r].repeats = 1;
            list_x[i] = in(n0 + r, id);
        }
    }
    __syncthreads();
    {   // unlisted scores
        const unsigned listed = bits[warp][lane];
        float m = minus_inf();
#pragma unroll
        for (int j = 0; j < E; ++j) {
            if (listed >> j & 1) x[j] = minus_inf();
            m = fmaxf(m, x[j]);
        }
        part[0][warp][lane] = m;
    }
    // the lists: W threads per row, each every W-th entry (all lanes of a warp, whether their row is there or not)
    {
        const int r = min(tid / W, rows - 1), first = tid % W, top = tid / W < rows ? a.top : 0;
        int *id = list_id + r * a.top;
        float *q = list_q + r * a.top;
        const float *xs = list_x + r * a.top;
        auto sum = [&](auto v) {
#pragma unroll
            for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            return v;
        };
        auto largest = [&](float v) {
#pragma unroll
            for (int o = W / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
            return v;
        };
        const bool repeats = of_list[r].repeats;
        if (__any_sync(0xffffffffu, repeats)) {   // rare: of a class's entries only the first counts as a class, -2 - its number marks the others
            if (repeats && first == 0)
                for (int e = 1; e < top; ++e)
                    for (int b = 0; b < e && id[e] >= 0; ++b)
                        if (id[b] == id[e]) id[e] = -2 - b;
            __syncwarp();
        }
        float best = minus_inf(), highest = minus_inf();
        int distinct = 0, broken = 0;
        for (int e = first; e < top; e += W)
            if (id[e] != -1) {
                best = fmaxf(best, q[e]);
                broken |= q[e] != q[e];
                highest = fmaxf(highest, xs[e]);
                distinct += id[e] >= 0;
            }
        best = largest(best);
        highest = largest(highest);
        broken = sum(broken);
        distinct = sum(distinct);
        const float ref = row_top(highest);
        const bool none = best == minus_inf() && !broken;
        double L = 0;
        if (a.lse) {
            L = (double)lse[r];
        } else {
            double all = 0;
            for (int e = first; e < top; e += W)
                if (id[e] != -1) all += exp(((double)q[e] - (double)best) * a.inv_t);
            L = (double)best * a.inv_t + log(sum(all));
        }
        double mass = 0, entropy = 0, of_listed = 0;
        float l = 0, l1 = 0;
        for (int e = first; e < top; e += W)
            if (id[e] != -1) {
                const double lq = (double)q[e] * a.inv_t - L, v = none ? 0.0 : exp(lq);
                const float far = __fsub_rn(xs[e], ref);
                mass += v;
                if ((float)v != 0.f) {   // (what a float does not hold is no mass, as in the other kernels)
                    entropy += v * lq;
                    of_listed += v * (((double)xs[e] - (double)ref) * a.inv_t);
                }
                if (id[e] >= 0) {
                    l += exp2_fast(far * a.c);
                    if (TWO) l1 += exp2_fast(far * LOG2E);
                }
                q[e] = (float)v;
            }
        mass = sum(mass);
        l = sum(l);
        l1 = TWO ? sum(l1) : l;
        if (a.loss) { entropy = sum(entropy); of_listed = sum(of_listed); }
        if (__any_sync(0xffffffffu, repeats)) {
            __syncwarp();
            if (repeats && first == 0) {
                for (int e = 1; e < top; ++e)
                    if (id[e] <= -2) q[-2 - id[e]] += q[e];
                entropy = 0;
                for (int e = 0; e < top; ++e)
                    if (id[e] >= 0 && q[e] != 0.f) entropy += (double)q[e] * log((double)q[e]);
            }
        }
        const double rest = a.lse && !none && distinct < K && mass < 1 ? 1.0 - mass : 0.0;
        if (first == 0 && tid / W < rows) {
            ListSums &o = of_list[r];
            o.teacher.mass = mass; o.teacher.entropy = entropy;
            o.teacher.total = none ? 0.f : (float)(mass + rest);
            o.teacher.rest = (float)rest;
            o.of_listed = of_listed; o.top = highest; o.l = l; o.l1 = l1;
        }
    }
    __syncthreads();
    float base = part[0][0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) base = fmaxf(base, part[0][w][lane]);
    const float largest_rest = base;
    base = row_top(base);
    {
        const float2 mb = make_float2(-base, -base), c2 = make_float2(a.c, a.c), one = make_float2(LOG2E, LOG2E);
        float2 s = make_float2(0.f, 0.f), s1 = s;
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            const float2 d = add2(make_float2(x[j], x[j + 1]), mb), v = mul2(d, c2);
            s = add2(s, make_float2(exp2_fast(v.x), exp2_fast(v.y)));
            if (TWO) {
                const float2 v1 = mul2(d, one);
                s1 = add2(s1, make_float2(exp2_fast(v1.x), exp2_fast(v1.y)));
            }
        }
        part[1][warp][lane] = __fadd_rn(s.x, s.y);
        if (TWO) part[2][warp][lane] = __fadd_rn(s1.x, s1.y);
    }
    __syncthreads();
    if (warp == 0) {
        const ListSums &o = of_list[min(lane, rows - 1)];
        StudentRow st;
        st.base = base;
        st.rest = st.rest1 = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            st.rest += part[1][i][lane];
            if (TWO) st.rest1 += part[2][i][lane];
        }
        if (!TWO) st.rest1 = st.rest;
        st.top = row_top(fmaxf(largest_rest, o.top));
        st.base = reference_of(st.base, st.rest, st.top);
        const float low = __fsub_rn(st.base, st.top), high = o.top == minus_inf() ? 0.f : __fsub_rn(o.top, st.top);
        st.l = o.l * exp2_fast(high * a.c);
        st.sum = st.rest * exp2_fast(low * a.c) + st.l;
        st.sum1 = TWO ? st.rest1 * exp2_fast(low * LOG2E) + o.l1 * exp2_fast(high * LOG2E) : st.sum;
        factors[lane] = distill_row(a, o.teacher, st, weights[lane], labels[lane]);
        students[lane] = st;
    }
    __syncthreads();
    if (a.loss && warp == W - 1 && lane < rows) {   // (the others go on)
        const ListSums &o = of_list[lane];
        const float high = o.top == minus_inf() ? 0.f : __fsub_rn(o.top, students[lane].top);
        a.loss[n] = distill_loss(a, o.teacher, students[lane], weights[lane], labels[lane],
                                 o.of_listed + (o.teacher.mass != 0 ? o.teacher.mass * ((double)high * a.inv_t) : 0.0), label_scores[lane]);
    }
    if (a.gives == GIVES_LOSS) return;
    float mg = 0, mh = 0;
    const bool track = a.maxbits != nullptr;
    auto put = [&](int r, int c, float2 gh) {
        if (track) { mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y); }
        const long long at = (n0 + r) * a.out.row + (long long)c * out_cls;
        if (a.gives == GIVES_PAIRS) static_cast<float2 *>(a.out.data)[at] = gh;
        else static_cast<T *>(a.out.data)[at] = score_from<T>(gh.x);
    };
    if (lane < rows) {
        DistillRow d = factors[lane];
        const int own = d.label - k0;   // (what its cell gets here is not what it keeps: it is noted then)
        d.label = -1;
        if (a.gives == GIVES_PAIRS) {
            float2 *to = static_cast<float2 *>(a.out.data) + n * a.out.row + (long long)k0 * out_cls;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                if (k0 + j >= K) break;
                const float2 gh = other_gh<TWO>(d, 0, x[j]);
                if (track && j != own) { mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y); }
                to[(long long)j * out_cls] = gh;
            }
        } else {
            T *to = static_cast<T *>(a.out.data) + n * a.out.row + (long long)k0 * out_cls;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                if (k0 + j >= K) break;
                to[(long long)j * out_cls] = score_from<T>(other_gh<TWO>(d, 0, x[j]).x);
            }
        }
    }
    __syncthreads();   // what follows is written over it: an entry of a list each, then the labels that are not listed
    for (int i = tid; i < rows * a.top; i += THREADS) {
        const int c = list_id[i], r = row_of(i);
        if (c >= 0) put(r, c, listed_gh<TWO>(factors[r], c, list_x[i], list_q[i]));
    }
    if (tid < rows) {
        const int c = labels[tid];
        if (c >= 0 && !(bits[c / E][tid] >> (c % E) & 1)) put(tid, c, other_gh<TWO>(factors[tid], c, label_scores[tid]));
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

// A long row, taken as in k_top_wide.  The first pass sums up the classes that the teacher does not list, which a bit map marks; the second
// finds the row in the L2 cache (the launch sees to it that the rows at work fit there) and writes what unlisted classes get; the
// few cells of listed classes and of the label are written over it.  (What lies between the passes is one warp's work, and the
// others wait for it: what the list says is worked out beside the first pass.)
template <typename T, bool TWO>
__global__ void __launch_bounds__(WIDE_THREADS, WIDE_BLOCKS) k_distill_wide(DistillArgs a, Scores<T> in) {
    constexpr int V = Pack<T>::V, S = SCORES_MAX_TOP / 32;
    extern __shared__ unsigned bits[];
    __shared__ int list_id[SCORES_MAX_TOP];   // -1: no class
    __shared__ float list_t[SCORES_MAX_TOP], list_x[SCORES_MAX_TOP], list_q[SCORES_MAX_TOP];   // the teacher's scores, the student's, masses
    __shared__ DistillRow factors;
    __shared__ TeacherSide teacher;
    __shared__ StudentRow student;
    __shared__ float row_lse, label_score;
    __shared__ float parts[WIDE_WARPS][3], whole[3];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long n = blockIdx.x / C;
    const int per = (a.k + C - 1) / C, lo = min(a.k, rank * per), hi = min(a.k, lo + per);
    const Part<T> part(in.at(n, 0), lo, hi);
    const uint4 *body = part.body();
    uint4 ahead[WIDE_PACKS];
    auto fetch = [&](int from) {
#pragma unroll
        for (int u = 0; u < WIDE_PACKS; ++u)
            if (from + u * WIDE_THREADS + tid < part.packs) ahead[u] = __ldg(body + from + u * WIDE_THREADS + tid);
    };
    // First pass: a warp takes 32 * WIDE_PACKS neighbouring packs at a time.  The last one works out what the list says meanwhile and
    // comes in `late` turns behind the others.
    constexpr int TURN = 32 * WIDE_PACKS;
    const int turns = (part.packs + TURN - 1) / TURN, late = turns >= 40 ? 2 : turns >= 16 ? 1 : 0;
    auto first_of = [&](int i) { return (i < late ? i * (WIDE_WARPS - 1) + warp : i * WIDE_WARPS - late + warp) * TURN + lane; };
    auto fetch_turn = [&](int i) {
        const int from = first_of(i);
#pragma unroll
        for (int u = 0; u < WIDE_PACKS; ++u)
            if (from + 32 * u < part.packs) ahead[u] = __ldg(body + from + 32 * u);
    };
    const int first_turn = warp == WIDE_WARPS - 1 ? late : 0;
    static_assert(WIDE_THREADS >= SCORES_MAX_TOP, "");
    // what the row gives besides its scores: read here, where it is waited for together with the lists
    const int label = row_label(a, n);
    const float w = a.weights ? a.weights[n] : 1.f;
    if (tid == WIDE_THREADS - 1) {
        row_lse = a.lse ? a.lse[n] : 0.f;
        label_score = label >= 0 ? in(n, label) : 0.f;
    }
    int id = -1;
    if (tid < a.top) {
        id = a.ids[n * a.ids_stride + tid];
        if (id < 0 || id >= a.k) id = -1;
    }
    fetch_turn(first_turn);
    for (int i = tid; i < (per + 31) / 32 + 1; i += WIDE_THREADS) bits[i] = 0;   // (a word more: read in twos)
    __syncthreads();
    bool repeat = false;   // in this block's part; a class stands in one part
    if (tid < a.top) {
        const int k = id - lo;
        if (id >= lo && k < hi - lo) repeat = atomicOr(&bits[k >> 5], 1u << (k & 31)) >> (k & 31) & 1;
        list_id[tid] = id;
        list_t[tid] = teacher_logit(a, n, tid);
        list_x[tid] = id >= 0 ? in(n, id) : minus_inf();
    }
    const bool repeats = __syncthreads_or(repeat) || C > 1;
    auto listed = [&](int k) { return bits[k >> 5] >> (k & 31) & 1; };   // k: cell of the part
    Running<TWO> run;
    if (tid < part.head + part.tail) {
        const int k = part.single(tid);
        if (!listed(k)) {
            const float x = score_f32(part.p[k]);
            run.raise(x, a.c);
            run.add(x, row_top(run.m), a.c);
        }
    }
    if (warp == WIDE_WARPS - 1) {
        int ids[S];
        float t[S], q[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int e = lane + 32 * s;
            ids[s] = e < a.top ? list_id[e] : -1;
            t[s] = e < a.top ? list_t[e] : 0.f;
        }
        const TeacherSide side = teacher_of<S>(a, a.lse ? &row_lse : nullptr, ids, t, q, repeats);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int e = lane + 32 * s;
            if (e < a.top) { list_id[e] = ids[s]; list_q[e] = q[s]; }
        }
        if (lane == 0) teacher = side;
    }
    for (int i = first_turn; first_of(i) - lane < part.packs; ++i) {
        uint4 w[WIDE_PACKS];
#pragma unroll
        for (int u = 0; u < WIDE_PACKS; ++u) w[u] = ahead[u];
        const int from = first_of(i);
        fetch_turn(i + 1);
#pragma unroll
        for (int u = 0; u < WIDE_PACKS; ++u) {
            const int at = from + 32 * u;
            if (at >= part.packs) break;
            Pack<T> p;
            p.bits = w[u];
            float v[V];
            p.unpack(v);
            const int k = part.head + at * V;
            const unsigned mark = __funnelshift_r(bits[k >> 5], bits[(k >> 5) + 1], k & 31) & ((1u << V) - 1);
            if (mark) {
#pragma unroll
                for (int c = 0; c < V; ++c)
                    if (mark >> c & 1) v[c] = minus_inf();
            }
            run.add_pack(v, a.c);
        }
    }
    run.join_warp(a.c);
    if (lane == 0) { parts[warp][0] = run.m; parts[warp][1] = run.s; parts[warp][2] = run.s1; }
    __syncthreads();
    {
        Running<TWO> all;
        if (lane < WIDE_WARPS) { all.m = parts[lane][0]; all.s = parts[lane][1]; all.s1 = parts[lane][2]; }
        all.join_warp(a.c);
        run = all;
    }
    if (C > 1) {
        if (tid == 0) { whole[0] = run.m; whole[1] = run.s; whole[2] = run.s1; }
        cluster.sync();
        run = Running<TWO>();
        for (int c = 0; c < C; ++c) {
            const float *o = cluster.map_shared_rank(whole, c);
            run.join(o[0], o[1], o[2], a.c);
        }
    }
    if (warp == 0) {   // the others wait: only what the second pass needs
        float top = run.m;
        for (int e = lane; e < a.top; e += 32) top = fmaxf(top, list_x[e]);
        const TeacherSide side = teacher;
        StudentRow st;
        st.base = row_top(run.m); st.rest = run.s; st.rest1 = TWO ? run.s1 : run.s;
        st.top = row_top(warp_max(top));
        st.base = reference_of(st.base, st.rest, st.top);
        float s0 = 0, s1 = 0;
        for (int e = lane; e < a.top; e += 32) {
            if (list_id[e] < 0) continue;
            const float far = __fsub_rn(list_x[e], st.top);
            s0 += exp2_fast(far * a.c);
            if (TWO) s1 += exp2_fast(far * LOG2E);
        }
        const float low = __fsub_rn(st.base, st.top);
        st.l = warp_sum(s0);
        st.sum = st.rest * exp2_fast(low * a.c) + st.l;
        st.sum1 = TWO ? st.rest1 * exp2_fast(low * LOG2E) + warp_sum(s1) : st.sum;
        if (lane == 0) {
            factors = distill_row(a, side, st, w, label);
            student = st;
        }
    }
    __syncthreads();
    if (a.gives != GIVES_LOSS) {
        DistillRow d = factors;
        T *out = static_cast<T *>(a.out.data) + n * a.out.row + lo;             // a.out.cls is 1
        float2 *pairs = static_cast<float2 *>(a.out.data) + n * a.out.row + lo;
        auto put = [&](int k, float2 gh) {
            if (a.gives == GIVES_PAIRS) pairs[k] = gh;
            else out[k] = score_from<T>(gh.x);
        };
        d.label = -1;
        if (tid < part.head + part.tail) {
            const int k = part.single(tid);
            put(k, other_gh<TWO>(d, k, score_f32(part.p[k])));
        }
        // f(scores, cell) for every pack of the thread: a loop of its own for each kind of result, with nothing to decide inside
        auto sweep = [&](auto &&f) {
            fetch(0);
            for (int from = 0; from < part.packs; from += WIDE_THREADS * WIDE_PACKS) {
                uint4 w[WIDE_PACKS];
#pragma unroll
                for (int u = 0; u < WIDE_PACKS; ++u) w[u] = ahead[u];
                fetch(from + WIDE_THREADS * WIDE_PACKS);
#pragma unroll
                for (int u = 0; u < WIDE_PACKS; ++u) {
                    const int at = from + u * WIDE_THREADS + tid;
                    if (at >= part.packs) break;
                    Pack<T> p;
                    p.bits = w[u];
                    float v[V];
                    p.unpack(v);
                    f(v, part.head + at * V);
                }
            }
        };
        const float2 mb = make_float2(-d.base, -d.base), c2 = make_float2(d.c, d.c), to_g = make_float2(d.to_g, d.to_g);
        auto gradients = [&](float(&v)[V]) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 g = mul2(exp_pair(make_float2(v[i], v[i + 1]), mb, c2), to_g);
                v[i] = g.x; v[i + 1] = g.y;
            }
        };
        auto store = [&](const float(&v)[V], int k) {
            Pack<T> p;
            p.pack(v);
            __stcs(reinterpret_cast<uint4 *>(out + k), p.bits);
        };
        const bool aligned = reinterpret_cast<uintptr_t>(out + part.head) % 16 == 0;
        if (a.gives == GIVES_PAIRS) {
            const bool twos = reinterpret_cast<uintptr_t>(pairs + part.head) % 16 == 0;
            sweep([&](float(&v)[V], int k) {
#pragma unroll
                for (int i = 0; i < V; i += 2) {
                    const float2 x = other_gh<TWO>(d, k + i, v[i]), y = other_gh<TWO>(d, k + i + 1, v[i + 1]);
                    if (twos) {
                        __stcs(reinterpret_cast<float4 *>(pairs + k + i), make_float4(x.x, x.y, y.x, y.y));
                    } else {
                        pairs[k + i] = x;
                        pairs[k + i + 1] = y;
                    }
                }
            });
        } else if (d.hard == 0.f && aligned) {
            sweep([&](float(&v)[V], int k) {
                gradients(v);
                store(v, k);
            });
        } else if (aligned) {
            sweep([&](float(&v)[V], int k) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = other_gh<TWO>(d, k + i, v[i]).x;
                store(v, k);
            });
        } else {
            sweep([&](float(&v)[V], int k) {
#pragma unroll
                for (int i = 0; i < V; ++i) out[k + i] = score_from<T>(other_gh<TWO>(d, k + i, v[i]).x);
            });
        }
        __syncthreads();   // what follows is written over it
        d.label = label;
        if (warp >= WIDE_WARPS / 2)   // (the first warps have the loss to find)
            for (int e = tid - WIDE_THREADS / 2; e < a.top; e += WIDE_THREADS / 2) {
                const int k = list_id[e] - lo;
                if (list_id[e] >= lo && k < hi - lo) put(k, listed_gh<TWO>(d, list_id[e], list_x[e], list_q[e]));
            }
        if (tid == WIDE_THREADS - 1 && label >= lo && label < hi && !listed(label - lo)) put(label - lo, other_gh<TWO>(d, label, label_score));
    }
    if (a.loss && rank == 0 && warp == 0) {
        double of_listed = 0;
        for (int e = lane; e < a.top; e += 32)
            if (list_id[e] >= 0 && list_q[e] != 0.f) of_listed += (double)list_q[e] * (((double)list_x[e] - (double)student.top) * a.inv_t);
        of_listed = warp_sum(of_listed);
        if (lane == 0) a.loss[n] = distill_loss(a, teacher, student, w, label, of_listed, label_score);
    }
    if (C > 1) cluster.sync();   // (the others' shared memory is read until they are here)
}

}  // namespace

// ------------------------------------------------------------------ launches
constexpr int FEW_BLOCKS = 148 * 16;   // at most what the GPU holds at once; the blocks walk the rows

// Rows of a tile, as a power of two from 8 to 32, and its shared memory; 0 bytes: the row is too long for a tile.  Several
// blocks should fit on an SM, so that one copies while another computes; with few rows the tiles are smaller and there are
// more of them.  (A row's result does not depend on the tile it is in.)
constexpr size_t TILE_SHARED = 190 * 1024, TILE_WANTED = 40 * 1024;
struct Tile {
    int rows_log = 5;
    size_t shared = 0;
};
Tile tile_of(int n, int k, bool by_class, size_t per_row) {
    auto shared = [&](int log) { return sizeof(float) * (size_t)k * ((1 << log) + (by_class ? 1 : 0)) + (per_row << log); };
    Tile t;
    if (!by_class && k > TILE_ROW_CLASSES) return t;
    while (t.rows_log > 3 && (shared(t.rows_log) > TILE_WANTED || (n >> t.rows_log) < 2 * 148)) --t.rows_log;
    if (shared(t.rows_log) <= TILE_SHARED) t.shared = shared(t.rows_log);
    return t;
}

void scores_adjust(const AdjustArgs &given, cudaStream_t stream) {
    if (given.n == 0) return;
    AdjustArgs a = given;
    a.inv_repetition = 1.f / a.repetition;
    const bool by_class = a.in.row < a.in.cls && a.out.row < a.out.cls && std::max(a.in.cls, a.out.cls) <= INT_MAX;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        constexpr int V = Pack<T>::V;
        const Scores<T> in = scores_of<T>(a.in), out = scores_of<T>(a.out);
        const size_t counts = a.history_ptr ? sizeof(int) * ADJUST_CELLS : 0;
        auto parts = [](long long n, int of) { return (unsigned)((n + of - 1) / of); };
        // (the boundaries of a row of scores are those of its results)
        const bool together = in.cls == 1 && out.cls == 1 && (reinterpret_cast<uintptr_t>(in.p) - reinterpret_cast<uintptr_t>(out.p)) % 16 == 0 &&
                              (in.row - out.row) % V == 0;
        if (by_class) {
            auto kern = counts ? k_adjust_class<T, true> : k_adjust_class<T, false>;
            kern<<<dim3(parts(a.n, ADJUST_ROWS), parts(a.k, ADJUST_CLASSES)), ROW_THREADS, counts, stream>>>(a, in, out);
        } else if (a.k >= ROW_THREADS * V / 2 && together) {
            // (shorter rows leave most of a block without a pack)
            const bool even = reinterpret_cast<uintptr_t>(in.p) % 16 == 0 && in.row % V == 0;
            auto kern = even ? k_adjust_long<T, true> : k_adjust_long<T, false>;
            kern<<<dim3((unsigned)a.n, parts(a.k, LONG_CELLS)), ROW_THREADS, counts ? sizeof(int) * (LONG_CELLS + V) : 0, stream>>>(a, in, out);
        } else {
            int tile_classes = std::max(2, std::min(a.k, ADJUST_CELLS));
            while (tile_classes > 1024 && (long long)a.n * parts(a.k, tile_classes) < 4 * 148) tile_classes /= 2;   // (8 x 40210: 24 us in 40 blocks)
            const int tile_rows = std::max(1, std::min(a.n, ADJUST_CELLS / 4 / tile_classes));
            static_assert(ADJUST_CELLS / 4 / 2 <= ADJUST_MOST_ROWS, "");
            const unsigned inverse = tile_rows == 1 ? 0u : (unsigned)(((1ull << 32) + tile_classes - 1) / tile_classes);
            k_adjust_tile<T><<<dim3(parts(a.n, tile_rows), parts(a.k, tile_classes)), ROW_THREADS, counts, stream>>>(a, in, out, tile_rows, tile_classes, inverse);
        }
    });
    TGBM_CUDA(cudaGetLastError());
}

// f(E) for the number of scores a lane has of a row (WarpRow)
template <typename F> void by_lane(int k, F &&f) {
    if (k <= 128) f(std::integral_constant<int, 4>{});
    else if (k <= 256) f(std::integral_constant<int, 8>{});
    else if (k <= 512) f(std::integral_constant<int, 16>{});
    else if (k <= 1024) f(std::integral_constant<int, 32>{});
    else f(std::integral_constant<int, 0>{});
}

// Blocks of a cluster for a long row: one, and more where there are not rows enough for WIDE_BLOCKS blocks per SM, or where the rows
// that are at work at once would not fit into the L2 cache for a second pass (`twice` bytes of a row; 0: there is none).
// A part is not shorter than what a block takes in one step.
int blocks_per_row(int n, int k, int size, size_t twice) {
    constexpr long long SLOTS = WIDE_BLOCKS * 148;
    constexpr size_t L2_ROOM = 80u << 20;   // (2048 x 65536 in 16 bits: 123 us; with half of that, and clusters of two, 139)
    int c = 1;
    while (c < WIDE_CLUSTER && k / (2 * c) >= WIDE_THREADS * WIDE_PACKS * 16 / size &&
           (n * (2ll * c) <= SLOTS || (twice && (size_t)std::min<long long>(n, SLOTS / c) * twice > L2_ROOM))) c *= 2;
    return c;
}
template <typename... P, typename... A>
void launch_clusters(void (*kernel)(P...), int n, int cluster, size_t smem, cudaStream_t stream, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)n * cluster)); cfg.blockDim = dim3(WIDE_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr; cfg.numAttrs = cluster > 1 ? 1 : 0;
    TGBM_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}

void scores_top(const TopArgs &given, cudaStream_t stream) {
    if (given.n == 0) return;
    TopArgs a = given;
    a.inv_t = 1.0 / (double)a.temperature;
    a.c = (float)(1.44269504088896341 * a.inv_t);
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        // (a pick of 64 takes some 300 instructions per thread, a warp from a tile some 500 per row: 12 of 37 took 121 us there for 246388 rows)
        if ((a.k <= FEW || (a.k <= 2 * FEW && a.top <= 20)) && a.in.cls <= INT_MAX) {   // (an address is one instruction then)
            const int blocks = (int)std::min(((long long)a.n + FEW_THREADS - 1) / FEW_THREADS, (long long)FEW_BLOCKS);
            const size_t smem = (size_t)FEW_THREADS * a.top * 8;
            auto go = [&](auto kern) {
                if (smem > 48 * 1024) allow_shared(kern, (size_t)FEW_THREADS * SCORES_MAX_TOP * 8);
                kern<<<blocks, FEW_THREADS, smem, stream>>>(a, scores_of<T>(a.in));
            };
            if (a.k <= 8) go(k_top_few<T, 8>);
            else if (a.k <= 16) go(k_top_few<T, 16>);
            else if (a.k <= 32) go(k_top_few<T, 32>);
            else go(k_top_few<T, 64>);
            return;
        }
        const bool by_class = a.in.row < a.in.cls;
        const Tile tile = tile_of(a.n, a.k, by_class, 0);
        if (tile.shared) {
            by_lane(a.k, [&](auto e) {
                constexpr int E = decltype(e)::value;
                auto go = [&](auto kern) {
                    if (tile.shared > 12 * 1024) allow_shared(kern, TILE_SHARED);   // (beside up to 33 KB of its own)
                    kern<<<(int)(((long long)a.n + (1 << tile.rows_log) - 1) >> tile.rows_log), TILE_THREADS, tile.shared, stream>>>(a, by_class, tile.rows_log);
                };
                if (a.top <= 20) go(k_top_tile<E, 1>);
                else if (a.top <= 40) go(k_top_tile<E, 2>);
                else if (a.top <= 80) go(k_top_tile<E, 4>);
                else go(k_top_tile<E, 8>);
            });
            return;
        }
        if (a.in.cls == 1) {
            launch_clusters(k_top_wide<T>, a.n, blocks_per_row(a.n, a.k, (int)sizeof(T), 0), 0, stream, a, scores_of<T>(a.in));
            return;
        }
        k_top_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, scores_of<T>(a.in));
    });
    TGBM_CUDA(cudaGetLastError());
}

void scores_distill(const DistillArgs &given, cudaStream_t stream) {
    if (given.n == 0) return;
    DistillArgs a = given;
    a.inv_t = 1.0 / (double)a.temperature;
    a.c = (float)(1.44269504088896341 * a.inv_t);
    a.c_low = (float)(1.44269504088896341 * a.inv_t - (double)a.c);
    const bool two = a.alpha < 1.f && a.temperature != 1.f;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        if (a.k <= FEW && std::max(a.in.cls, a.out.cls) <= INT_MAX) {
            const int blocks = (int)std::min(((long long)a.n + FEW_THREADS - 1) / FEW_THREADS, (long long)FEW_BLOCKS);
            auto go = [&](auto kern) { kern<<<blocks, FEW_THREADS, 0, stream>>>(a, scores_of<T>(a.in)); };
            if (a.k <= 8) two ? go(k_distill_few<T, 8, true>) : go(k_distill_few<T, 8, false>);
            else if (a.k <= 16) two ? go(k_distill_few<T, 16, true>) : go(k_distill_few<T, 16, false>);
            else two ? go(k_distill_few<T, 32, true>) : go(k_distill_few<T, 32, false>);
            return;
        }
        const bool by_class = a.in.row < a.in.cls || a.in.one_by_class;
        if (by_class && a.k <= SCORES_CLASS_MOST && std::max(a.in.cls, a.out.cls) <= INT_MAX) {
            const size_t smem = 12 * (size_t)CLASS_ROWS * a.top;
            const unsigned blocks = (unsigned)(((long long)a.n + CLASS_ROWS - 1) / CLASS_ROWS);
            auto go = [&](auto kern, int warps) {
                if (smem > 16 * 1024) allow_shared(kern, 12 * (size_t)CLASS_ROWS * SCORES_MAX_TOP);
                kern<<<blocks, 32 * warps, smem, stream>>>(a, scores_of<T>(a.in));
            };
            if (a.k <= 64) two ? go(k_distill_class<T, 8, 8, true>, 8) : go(k_distill_class<T, 8, 8, false>, 8);
            else if (a.k <= 128) two ? go(k_distill_class<T, 16, 8, true>, 8) : go(k_distill_class<T, 16, 8, false>, 8);
            else if (a.k <= 256) two ? go(k_distill_class<T, 32, 8, true>, 8) : go(k_distill_class<T, 32, 8, false>, 8);
            else if (a.k <= 512) two ? go(k_distill_class<T, 32, 16, true>, 16) : go(k_distill_class<T, 32, 16, false>, 16);
            else two ? go(k_distill_class<T, 32, 32, true>, 32) : go(k_distill_class<T, 32, 32, false>, 32);
            return;
        }
        const Tile tile = tile_of(a.n, a.k, by_class, 12 * (size_t)a.top);
        if (tile.shared && (a.gives == GIVES_LOSS || a.out.cls <= INT_MAX)) {
            by_lane(a.k, [&](auto e) {
                constexpr int E = decltype(e)::value;
                auto go = [&](auto kern) {
                    if (tile.shared > 40 * 1024) allow_shared(kern, TILE_SHARED);
                    kern<<<(int)(((long long)a.n + (1 << tile.rows_log) - 1) >> tile.rows_log), TILE_THREADS, tile.shared, stream>>>(a, by_class, tile.rows_log);
                };
                if (a.top <= 32) two ? go(k_distill_tile<E, true, 1>) : go(k_distill_tile<E, false, 1>);
                else two ? go(k_distill_tile<E, true, 4>) : go(k_distill_tile<E, false, 4>);
            });
            return;
        }
        if (a.in.cls == 1 && (a.gives == GIVES_LOSS || a.out.cls == 1) && !a.maxbits) {
            const int c = blocks_per_row(a.n, a.k, (int)sizeof(T), a.gives == GIVES_LOSS ? 0 : a.k * sizeof(T));
            const size_t smem = sizeof(unsigned) * (size_t)(((a.k + c - 1) / c + 31) / 32 + 1);
            auto kern = two ? k_distill_wide<T, true> : k_distill_wide<T, false>;
            if (smem > 40 * 1024) allow_shared(kern, SCORES_MAX_CLASSES / 8 + 4);
            launch_clusters(kern, a.n, c, smem, stream, a, scores_of<T>(a.in));
            return;
        }
        auto kern = two ? k_distill_any<T, true> : k_distill_any<T, false>;
        constexpr size_t most = SCORES_MAX_CLASSES / 8;
        const size_t smem = sizeof(unsigned) * (size_t)((a.k + 31) / 32);
        if (smem > 40 * 1024) allow_shared(kern, most);
        kern<<<a.n, ROW_THREADS, smem, stream>>>(a, scores_of<T>(a.in));
    });
    TGBM_CUDA(cudaGetLastError());
}

}  // namespace tgbm

// ------------------------------------------------------------------ C entries
using namespace tgbm;

extern "C" {

int tgbm_scores_adjust(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, void *d_out,
                       long long out_row_stride, long long out_class_stride, const float *d_bias, const unsigned *d_allowed, int n_masks,
                       long long mask_stride, const int *d_allowed_row, const long long *d_history_ptr, const int *d_history,
                       long long n_history, float repetition, float frequency, float presence, void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        TGBM_CHECK(repetition > 0.f && repetition <= FLT_MAX && 1.f / repetition <= FLT_MAX,
                   "the repetition penalty has to be a positive number whose reciprocal is one");
        TGBM_CHECK(std::isfinite(frequency) && std::isfinite(presence), "penalties have to be finite");
        TGBM_CHECK(n_history >= 0, "negative length of the histories");
        if (d_allowed) {
            TGBM_CHECK(n_masks >= 1, "masks without a row");
            TGBM_CHECK(mask_stride >= 0 && (n_masks == 1 || mask_stride >= (n_classes + 31) / 32), "mask rows are shorter than the classes need");
        }
        if (n_rows == 0) return;
        AdjustArgs a;
        a.n = n_rows; a.k = n_classes;
        a.in = view_of("scores", d_scores, type, n_rows, n_classes, row_stride, class_stride, false);
        a.out = view_of("out", d_out, type, n_rows, n_classes, out_row_stride, out_class_stride, true);
        const bool in_place = a.in.data == a.out.data && a.in.row == a.out.row && a.in.cls == a.out.cls;
        TGBM_CHECK(in_place || !share_memory(a.in, size_of(type), a.out, size_of(type), n_rows, n_classes), "scores and out share memory but are not the same");
        check_pointer("bias", d_bias, 4); check_pointer("masks", d_allowed, 4); check_pointer("rows' masks", d_allowed_row, 4);
        check_pointer("history", d_history_ptr, 8); check_pointer("history", d_history, 4);
        a.bias = d_bias;
        if (d_allowed) {
            TGBM_CHECK(d_allowed_row || n_masks >= n_rows, "fewer masks than rows, and none named for each row");
            a.allowed = d_allowed; a.n_masks = n_masks; a.mask_stride = mask_stride; a.allowed_row = d_allowed_row;
        }
        if (d_history_ptr && n_history > 0) {
            TGBM_CHECK(d_history != nullptr, "history: null pointer");
            a.history_ptr = d_history_ptr; a.history = d_history; a.n_history = n_history;
        }
        a.repetition = repetition; a.frequency = frequency; a.presence = presence;
        auto read = [&](const char *what, const void *p, long long bytes) {
            TGBM_CHECK(!lies_in(a.out, size_of(type), n_rows, n_classes, p, bytes), std::string("out and ") + what + " share memory");
        };
        read("bias", a.bias, 4ll * n_classes);
        if (n_masks == 1 || mask_stride == (n_classes + 31) / 32) read("masks", a.allowed, 4 * (long long)n_masks * ((n_classes + 31) / 32));
        read("rows' masks", a.allowed_row, 4ll * n_rows);
        read("histories", a.history_ptr, 8ll * n_rows + 8);
        read("histories", a.history, 4 * a.n_history);
        scores_adjust(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

int tgbm_scores_top(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int top,
                    float temperature, float *d_values, int *d_ids, float *d_lse, void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        check_list(top);
        check_temperature(temperature);
        if (n_rows == 0) return;
        TopArgs a;
        a.n = n_rows; a.k = n_classes; a.top = top; a.temperature = temperature;
        a.in = view_of("scores", d_scores, type, n_rows, n_classes, row_stride, class_stride, false);
        TGBM_CHECK(d_values && d_ids, "values or ids: null pointer");
        check_pointer("values", d_values, 4); check_pointer("ids", d_ids, 4); check_pointer("lse", d_lse, 4);
        a.values = d_values; a.ids = d_ids; a.lse = d_lse;
        scores_top(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

int tgbm_scores_distill(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int top,
                        const int *d_ids, long long ids_stride, int logits_type, const void *d_logits, long long logits_stride,
                        const float *d_lse, const int *d_labels, const float *d_weights, float temperature, float alpha, float *d_loss,
                        int gives, void *d_grad, long long grad_row_stride, long long grad_class_stride, void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        check_list(top);
        check_temperature(temperature);
        TGBM_CHECK(alpha >= 0.f && alpha <= 1.f, "alpha outside [0, 1]");
        TGBM_CHECK(gives >= TGBM_GIVES_LOSS && gives <= TGBM_GIVES_PAIRS, "unknown kind of result");
        TGBM_CHECK(logits_type >= TGBM_F32 && logits_type <= TGBM_BF16, "logits: unknown type");
        TGBM_CHECK(ids_stride >= 0 && logits_stride >= 0, "negative stride of the teacher's lists");
        if (n_rows == 0) return;
        DistillArgs a;
        a.n = n_rows; a.k = n_classes; a.top = top;
        a.in = view_of("scores", d_scores, type, n_rows, n_classes, row_stride, class_stride, false);
        TGBM_CHECK(d_ids && d_logits, "ids or logits: null pointer");
        check_pointer("ids", d_ids, 4); check_pointer("logits", d_logits, size_of(logits_type)); check_pointer("lse", d_lse, 4);
        check_pointer("labels", d_labels, 4); check_pointer("weights", d_weights, 4); check_pointer("loss", d_loss, 4);
        a.ids = d_ids; a.ids_stride = ids_stride; a.logits = d_logits; a.logits_type = logits_type; a.logits_stride = logits_stride;
        a.lse = d_lse; a.labels = d_labels; a.weights = d_weights;
        a.temperature = temperature; a.alpha = alpha; a.gives = gives; a.loss = d_loss;
        TGBM_CHECK(d_loss || gives != TGBM_GIVES_LOSS, "loss: null pointer");
        if (gives != TGBM_GIVES_LOSS) {
            const bool pairs = gives == TGBM_GIVES_PAIRS;
            TGBM_CHECK(!pairs || reinterpret_cast<uintptr_t>(d_grad) % 8 == 0, "gradient: pairs have to be aligned to 8 bytes");
            a.out = view_of("gradient", d_grad, pairs ? (int)SCORE_F32 : type, n_rows, n_classes, grad_row_stride, grad_class_stride, true);
            TGBM_CHECK(!share_memory(a.in, size_of(type), a.out, pairs ? 8 : size_of(type), n_rows, n_classes), "scores and gradient share memory");
        }
        scores_distill(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

}  // extern "C"
