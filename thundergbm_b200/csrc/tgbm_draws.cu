// Classes drawn from the scores of many classes (sample), and the loss on drawn classes with its gradient (feedback).
//
// sample decides which class a random number falls on by sums of exponentials next to one another, and a row may have 2^20
// of them: exponentials and their sums are doubles, so that the classes are those of the definition.
#include <cfloat>
#include <climits>
#include <cmath>

#include <cooperative_groups.h>

#include "../../include/thundergbm.h"
#include "tgbm_scores.cuh"
#include "tgbm_scores_check.h"
#include "tgbm_scores_long.cuh"

namespace tgbm {
namespace {
namespace cg = cooperative_groups;

constexpr int ROW_THREADS = 256, ROW_WARPS = ROW_THREADS / 32;

// ------------------------------------------------------------------ sample
// What a row's draws obey.  Numbers that come with the rows cannot be refused: a temperature that is none means a row that has no
// distribution, the others are taken as the nearest that makes sense.
struct Limits {
    double inv_t, top_p, min_p;   // top_p >= 1, min_p = 0: none
    int top_k;                    // k: none
    bool greedy, broken;
};
__device__ __forceinline__ Limits limits_of(const SampleArgs &a, long long n) {
    const float t = a.temperatures ? a.temperatures[n] : a.temperature, p = a.top_ps ? a.top_ps[n] : a.top_p, m = a.min_ps ? a.min_ps[n] : a.min_p;
    const int k = a.top_ks ? a.top_ks[n] : a.top_k;
    Limits l;
    l.broken = !(t >= 0.f && t <= FLT_MAX);
    l.greedy = t == 0.f;
    l.inv_t = t > 0.f ? 1.0 / (double)t : 0.0;
    l.top_p = p < 1.f ? fmax((double)p, 0.0) : 1.0;   // (NaN: none)
    l.min_p = m > 0.f ? fmin((double)m, 1.0) : 0.0;
    l.top_k = k > 0 && k < a.k ? k : a.k;
    return l;
}
__device__ __forceinline__ double uniform_of(const SampleArgs &a, long long i) {
    const double u = a.uniform_f64 ? static_cast<const double *>(a.uniform)[i] : (double)static_cast<const float *>(a.uniform)[i];
    return u > 0 ? u : 0.0;   // (NaN: 0; what is not below 1 falls on the last class)
}
__device__ __forceinline__ void put_draw(const SampleArgs &a, long long i, int cls, float log, float all_log) {
    a.classes[i] = cls;
    if (a.logs) a.logs[i] = log;
    if (a.all_logs) a.all_logs[i] = all_log;
}

// sum over the block, the same in all threads and every time; `parts`: one per warp
template <typename V> __device__ __forceinline__ V block_sum(V v, V *parts) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
    V s = parts[0];
#pragma unroll
    for (int i = 1; i < ROW_WARPS; ++i) s += parts[i];
    return s;
}
__device__ __forceinline__ unsigned block_max(unsigned v, unsigned *parts) {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned s = parts[0];
#pragma unroll
    for (int i = 1; i < ROW_WARPS; ++i) s = max(s, parts[i]);
    return s;
}

// A row, any strides: a block reads it again for everything that it wants to know.  Classes that may be drawn are those whose entry
// (key of the score, then the lower class) reaches a border; a warp has a segment of neighbouring classes.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) k_sample_any(SampleArgs a, Scores<T> in) {
    __shared__ double sums[ROW_WARPS];
    __shared__ unsigned keys[ROW_WARPS];
    __shared__ int counts[ROW_WARPS];
    __shared__ int tie_class;
    const long long n = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (a.k + ROW_WARPS - 1) / ROW_WARPS, lo = min(a.k, warp * per), hi = min(a.k, lo + per);
    const Limits l = limits_of(a, n);
    auto each = [&](auto &&f) {
        for (int i = lo + lane; i < hi; i += 32) f(in(n, i), i);
    };
    bool bad = l.broken;
    unsigned top_key = 0;
    each([&](float x, int) {
        if (!(x < -minus_inf())) bad = true;   // (NaN, +inf)
        top_key = max(top_key, plain_key(x));
    });
    top_key = block_max(top_key, keys);
    bad = __syncthreads_or(bad);
    if (bad || top_key < LOWEST_KEY) {
        const float v = bad ? __int_as_float(0x7fffffff) : minus_inf();
        for (int d = threadIdx.x; d < a.draws; d += ROW_THREADS) put_draw(a, n * a.draws + d, -1, v, v);
        return;
    }
    const double best = (double)key_score(top_key);
    auto weight = [&](float x) { return l.greedy ? ((double)x == best ? 1.0 : 0.0) : exp(((double)x - best) * l.inv_t); };
    auto sum_of = [&](auto &&counts_in) {
        double s = 0;
        each([&](float x, int i) {
            if (counts_in(x, i)) s += weight(x);
        });
        return block_sum(s, sums);
    };
    auto count_of = [&](auto &&counts_in) {
        int c = 0;
        each([&](float x, int i) { c += counts_in(x, i); });
        return block_sum(c, counts);
    };
    // the r-th class in order with this key
    auto nth_tie = [&](unsigned key, int r) {
        int c = 0;
        each([&](float x, int) { c += plain_key(x) == key; });
        c = warp_sum(c);
        __syncthreads();
        if (lane == 0) counts[warp] = c;
        __syncthreads();
        int before = 0;
        for (int w = 0; w < warp; ++w) before += counts[w];
        if (before < r && r <= before + c) {
            for (int i0 = lo; i0 < hi; i0 += 32) {
                const unsigned same = __ballot_sync(0xffffffffu, i0 + lane < hi && plain_key(in(n, i0 + lane)) == key);
                const int here = __popc(same);
                if (before < r && r <= before + here) {
                    const bool mine = (same >> lane & 1) && before + __popc(same & ((2u << lane) - 1)) == r;
                    if (mine) tie_class = i0 + lane;
                }
                before += here;
            }
        }
        __syncthreads();
        return tie_class;
    };
    const double all = l.greedy ? 1.0 : sum_of([&](float x, int) { return x > minus_inf(); });
    unsigned key = LOWEST_KEY;   // entries with a larger key, and those with this one up to class `last`
    int last = a.k;
    auto reaches = [&](float x, int i) {
        const unsigned k = plain_key(x);
        return k > key || (k == key && i <= last);
    };
    if (l.min_p > 0) {   // weights rise with the scores: the lowest score that is heavy enough
        unsigned k = 0;
        each([&](float x, int) {
            if (x > minus_inf() && weight(x) >= l.min_p) k = max(k, ~plain_key(x));
        });
        key = ~block_max(k, keys);
    }
    // the largest key that enough reach
    auto bisect = [&](auto &&enough) {
        unsigned low = key, high = top_key;
        while (low < high) {
            const unsigned mid = low + (high - low + 1) / 2;
            if (enough(mid)) low = mid;
            else high = mid - 1;
        }
        return low;
    };
    const int top_k = l.greedy ? 1 : l.top_k;
    if (top_k < a.k) {
        const unsigned found = bisect([&](unsigned mid) { return count_of([&](float x, int) { return plain_key(x) >= mid; }) >= top_k; });
        const int above = count_of([&](float x, int) { return plain_key(x) > found; });
        const int ties = count_of([&](float x, int) { return plain_key(x) == found; });
        key = found;
        if (above + ties > top_k) last = nth_tie(found, top_k - above);
    }
    if (l.top_p < 1 && !l.greedy) {
        const double target = l.top_p * sum_of(reaches);
        const unsigned found = bisect([&](unsigned mid) { return sum_of([&](float x, int i) { return plain_key(x) >= mid && reaches(x, i); }) >= target; });
        const double above = sum_of([&](float x, int) { return plain_key(x) > found; }), w = weight(key_score(found));
        const int ties = count_of([&](float x, int i) { return plain_key(x) == found && reaches(x, i); });
        const double need = ceil((target - above) / w);
        const int r = need >= ties ? ties : need < 1 ? 1 : (int)need;
        last = r == ties ? (found == key ? last : a.k) : nth_tie(found, r);
        key = found;
    }
    double mine = 0;
    each([&](float x, int i) {
        if (reaches(x, i)) mine += weight(x);
    });
    mine = warp_sum(mine);
    __syncthreads();
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    double mass = 0;
    for (int w = 0; w < ROW_WARPS; ++w) mass += sums[w];
    for (int d = warp; d < a.draws; d += ROW_WARPS) {
        const long long at = n * a.draws + d;
        const double target = uniform_of(a, at) * mass;
        double before = 0;   // of the segments in front; the segment is the first that goes beyond the target, or the last that has any
        int segment = 0;
        double in_front = 0;
        for (int w = 0; w < ROW_WARPS; ++w) {
            if (sums[w] > 0) { segment = w; before = in_front; }
            in_front += sums[w];
            if (in_front > target) break;
        }
        const int from = min(a.k, segment * per), to = min(a.k, from + per);
        int cls = -1;
        double its = 0;
        for (int i0 = from; i0 < to; i0 += 32) {
            const int i = i0 + lane;
            const float x = i < to ? in(n, i) : minus_inf();
            const double w = i < to && reaches(x, i) ? weight(x) : 0.0;
            double upto = w;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned has = __ballot_sync(0xffffffffu, w > 0), hit = __ballot_sync(0xffffffffu, w > 0 && before + upto > target);
            if (has) {   // (the last that has any, should rounding leave the target behind all of them)
                const int src = hit ? __ffs(hit) - 1 : 31 - __clz(has);
                cls = i0 + src;
                its = __shfl_sync(0xffffffffu, w, src);
            }
            if (hit) break;
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) put_draw(a, at, cls, (float)log(its / mass), (float)log(its / all));
    }
}

// ---- exponentials in 64 bits ------------------------------------------------------------------
// exp(d / T) for d <= 0, relative error below 2^-38: with y = 32 d log2(e) / T and n the whole number nearest to it, 2^(n / 32) is a power of two times one
// of 32 numbers (a table in shared memory), and exp of the rest, |rest| <= ln 2 / 64, five terms of its series, the first left out
// below 2^-39.  11 instructions of the fp64 units, which do half as many as the fp32 ones; the library's exp takes twice as many.
struct Powers {
    double of[32];
    __device__ __forceinline__ void fill() {   // a warp; a barrier has to follow
        const int lane = threadIdx.x & 31;
        of[lane] = exp2((double)lane * 0.03125);
    }
};
struct Exponent {
    double by;      // 32 log2(e) / T
    float about;    // the same
    bool greedy;    // 1 for d = 0, else 0
    __device__ __forceinline__ Exponent(const Limits &l) : by(l.inv_t * 46.166241308446828384), about((float)by), greedy(l.greedy) {}
    __device__ __forceinline__ double operator()(const Powers &t, float x, float top) const {
        if (greedy) return x == top ? 1.0 : 0.0;
        if (!(__fsub_rn(x, top) * about > -32000.f)) return 0.0;   // (2^-1000; -inf)
        const double y = __dmul_rn(__dsub_rn((double)x, (double)top), by), shifted = __dadd_rn(y, 6755399441055744.0);   // 1.5 * 2^52: whole numbers
        const int n = __double2loint(shifted);
        const double r = __dsub_rn(y, __dsub_rn(shifted, 6755399441055744.0));
        constexpr double A1 = 0.6931471805599453094 / 32, A2 = A1 * A1 / 2, A3 = A1 * A1 * A1 / 6, A4 = A1 * A1 * A1 * A1 / 24;
        const double p = __fma_rn(r, __fma_rn(r, __fma_rn(r, __fma_rn(r, A4, A3), A2), A1), 1.0);
        const double v = __dmul_rn(t.of[n & 31], p);
        return __hiloint2double(__double2hiint(v) + ((n >> 5) << 20), __double2loint(v));
    }
};

// ---- up to 1024 classes: a lane has a row, the W warps of a block (W = 1: each for itself) share its classes, E neighbours each ------
// What a warp's lanes know of their rows is put together through shared memory; all warps come to the same numbers in the same order,
// and so decide alike.
//
// Limits: which scores a row's draws are left to is settled by a list of the few that can be among them, in class order, in shared memory: a lane
// walks its row's list there, without a barrier, as often as it takes.  Scores that can be are those from a border on: min_p gives one, and so does
// top_p (classes with less than (1 - top_p) / classes of the mass each have less than 1 - top_p of it together); where more than LIST reach it, it is
// raised by bisection over all scores as long as enough reach it.  Rows with more all the same (limits that leave that many, ties)
// are settled by bisection over all scores.
constexpr int LIST = 56;
template <int W> struct ClassShared {
    Powers powers;
    double sums[2][W][32];
    float lows[2][W][32], highs[2][W][32], counts[2][W][32];
    double front[W][32];
    int cls[W][32];
    float score[W][32];
};
template <int W> struct ListShared {
    static constexpr int MOST = W == 1 ? 32 : LIST;   // (W = 1: up to 32 classes)
    static constexpr int APART = 36;                  // (entries i, i + 1, ... of four rows lie in different banks)
    double w[MOST][APART], mass[32], all[32];
    float x[MOST][APART], top[32];
    unsigned short k[MOST][APART];
    int size[32];
};
template <int W> struct Over {   // `turn` alternates, so that one barrier is enough
    ClassShared<W> &sh;
    int turn = 0;
    __device__ __forceinline__ void all(double &sum, float &low, float &high, float &count) {
        if constexpr (W > 1) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            sh.sums[turn][warp][lane] = sum; sh.lows[turn][warp][lane] = low; sh.highs[turn][warp][lane] = high; sh.counts[turn][warp][lane] = count;
            __syncthreads();
            sum = 0; count = 0;
#pragma unroll 8
            for (int w = 0; w < W; ++w) {
                sum += sh.sums[turn][w][lane];
                low = fminf(low, sh.lows[turn][w][lane]);
                high = fmaxf(high, sh.highs[turn][w][lane]);
                count += sh.counts[turn][w][lane];
            }
            turn ^= 1;
        }
    }
    // of the warps in front of this one
    __device__ __forceinline__ int in_front(int count, int &total) {
        total = count;
        if constexpr (W > 1) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            sh.counts[turn][warp][lane] = (float)count;
            __syncthreads();
            int before = 0;
            total = 0;
            for (int v = 0; v < W; ++v) {
                if (v == warp) before = total;
                total += (int)sh.counts[turn][v][lane];
            }
            turn ^= 1;
            return before;
        }
        return 0;
    }
    // this warp's part [front, end) of its rows' mass; last: nothing lies behind it
    __device__ __forceinline__ double shares(double mine, double &front, double &end, bool &last) {
        front = 0; end = mine; last = mine > 0;
        double mass = mine;
        if constexpr (W > 1) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            sh.front[warp][lane] = mine;
            __syncthreads();
            mass = 0;
#pragma unroll 8
            for (int v = 0; v < W; ++v) {
                const double s = sh.front[v][lane];
                if (v == warp) front = mass;
                mass += s;
                if (v == warp) end = mass;
                if (v > warp && s > 0) last = false;
            }
        }
        return mass;
    }
};
template <int W> __device__ __forceinline__ void meet() {   // the warps that share rows
    if (W > 1) __syncthreads();
    else __syncwarp();
}

// Nothing is cut off: exponentials stay in registers.
template <typename T, int E, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 1 ? 4 : W == 8 ? 2 : 1) k_sample_class(SampleArgs a, Scores<T> in) {
    __shared__ ClassShared<W> shared[W == 1 ? 4 : 1];   // (W = 1: each warp has its own)
    ClassShared<W> &sh = shared[W == 1 ? threadIdx.x >> 5 : 0];
    const int lane = threadIdx.x & 31, warp = W == 1 ? 0 : threadIdx.x >> 5, k0 = warp * E, here = a.k - k0;
    const long long n0 = (W == 1 ? blockIdx.x * 4ll + (threadIdx.x >> 5) : (long long)blockIdx.x) * 32 + lane, n = min(n0, a.n - 1ll);
    float x[E];
    {
        const T *from = in.at(n, k0);
        T raw[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (j < here) raw[j] = from[j * in.cls];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = j < here ? score_f32(raw[j]) : minus_inf();
    }
    if (warp == 0) sh.powers.fill();
    meet<W>();
    Over<W> over{sh};
    const Limits l = limits_of(a, n);
    float top = minus_inf(), least = 0, count = 0;
    double mass = 0, mine = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        top = fmaxf(top, x[j]);
        if (x[j] != x[j]) count = 1;
    }
    over.all(mass, least, top, count);
    const bool bad = l.broken || count != 0 || top == -minus_inf(), live = !bad && top != minus_inf();
    const Exponent weight(l);
    double w[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
        w[j] = live ? weight(sh.powers, x[j], top) : 0.0;
        mine += w[j];
    }
    double front, end;
    bool last;
    mass = over.shares(mine, front, end, last);
    // W draws at a time: the warp that has a draw's class puts it down, and a warp finishes a draw for all rows
    const double log_mass = live ? log(mass) : 0.0;
    for (int d0 = 0; d0 < a.draws; d0 += W) {
        const int some = min(W, a.draws - d0);
        for (int d = 0; d < some; ++d) {
            const double target = uniform_of(a, n * a.draws + d0 + d) * mass;
            const bool hit = mine > 0 && front <= target && (end > target || last);
            if (!__any_sync(0xffffffffu, hit)) continue;
            double upto = front;
            int at = 0;
            float s = 0;
            bool found = false;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (!found && w[j] > 0) {
                    upto += w[j];
                    at = j;
                    s = x[j];
                    found = upto > target;
                }
            if (hit) { sh.cls[d][lane] = k0 + at; sh.score[d][lane] = s; }
        }
        meet<W>();
        if (warp < some && n0 == n) {
            const long long at = n * a.draws + d0 + warp;
            if (live) {
                const float log = (float)(((double)sh.score[warp][lane] - (double)top) * l.inv_t - log_mass);
                put_draw(a, at, sh.cls[warp][lane], log, log);
            } else {
                const float v = bad ? __int_as_float(0x7fffffff) : minus_inf();
                put_draw(a, at, -1, v, v);
            }
        }
        meet<W>();
    }
}

__device__ __forceinline__ float middle(float low, float high) {
    const float mid = 0.5f * low + 0.5f * high;
    return mid > low && mid <= high ? mid : high;
}
// The largest score that enough of a row reaches: `measure` of the scores from there on sums up to `target` at least.  `low` (reached by enough)
// and `high` are the least and the largest score.  Halves the interval and moves its ends to scores that there are.  each(f): f(score, measure) for
// all of them; together(sum, up, down): what the other warps have, too.
template <typename F, typename G>
__device__ __forceinline__ float reached(bool active, double target, float low, float high, F &&each, G &&together) {
    while (__any_sync(0xffffffffu, active && low < high)) {
        const float mid = middle(low, high);
        double sum = 0;
        float up = -minus_inf(), down = minus_inf();
        each([&](float x, double m) {
            if (x >= mid) { sum += m; up = fminf(up, x); }
            else down = fmaxf(down, x);
        });
        together(sum, up, down);
        if (low < high) {
            if (sum >= target) low = up;
            else high = down;
        }
    }
    return low;
}
// how many of `ties` equal scores, each of weight w, are left to reach the target beside `above`
__device__ __forceinline__ int ties_left(double target, double above, double w, int ties) {
    const double need = ceil((target - above) / w);
    return need >= (double)ties ? ties : need < 1 ? 1 : (int)need;
}

// With limits: the scores lie in shared memory (row r and class k at k * apart + r), which leaves the registers to what is found out of them.
template <typename T, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 1 ? 4 : 3) k_sample_limited(SampleArgs a, Scores<T> in, int apart) {
    extern __shared__ __align__(16) unsigned char room[];
    const int lane = threadIdx.x & 31, group = W == 1 ? threadIdx.x >> 5 : 0, warp = W == 1 ? 0 : threadIdx.x >> 5;
    ClassShared<W> &sh = reinterpret_cast<ClassShared<W> *>(room)[group];   // (W = 1: each warp has its own)
    constexpr int G = W == 1 ? 4 : 1;
    ListShared<W> &list = reinterpret_cast<ListShared<W> *>(room + G * sizeof(ClassShared<W>))[group];
    float *tile = reinterpret_cast<float *>(room + G * (sizeof(ClassShared<W>) + sizeof(ListShared<W>))) + group * (size_t)apart * a.k;
    constexpr int MOST = ListShared<W>::MOST;
    const int per = (a.k + W - 1) / W, k0 = min(a.k, warp * per), k1 = min(a.k, k0 + per);
    const long long first = (blockIdx.x * (long long)G + group) * 32, n0 = first + lane, n = min(n0, a.n - 1ll);
    float top = minus_inf(), least = 0, count = 0;
    double all = 0;
    if (apart == 33) {   // by row
        for (int r = warp; r < 32; r += W) {
            const T *from = in.at(min(first + r, a.n - 1ll), 0);
#pragma unroll 8
            for (int k = lane; k < a.k; k += 32) tile[33 * k + r] = score_f32(from[k * in.cls]);
        }
        meet<W>();
    } else {
        const T *from = in.at(n, k0);
#pragma unroll 8
        for (int k = k0; k < k1; ++k, from += in.cls) tile[32 * k + lane] = score_f32(*from);
    }
    if (warp == 0) sh.powers.fill();
    float *const mine_x = tile + lane;
    auto each_score = [&](auto &&f) {
#pragma unroll 8
        for (int k = k0; k < k1; ++k) f(mine_x[k * apart], k);
    };
    Over<W> over{sh};
    each_score([&](float x, int) {
        top = fmaxf(top, x);
        if (x != x) count = 1;
    });
    over.all(all, least, top, count);
    const Limits l = limits_of(a, n);
    const bool bad = l.broken || count != 0 || top == -minus_inf(), live = !bad && top != minus_inf();
    const Exponent weight(l);
    auto weight_of = [&](float v) { return weight(sh.powers, v, top); };
    const int top_k = l.greedy ? 1 : l.top_k;
    const bool by_count = live && top_k < a.k, by_mass = live && l.top_p < 1 && !l.greedy, by_share = live && l.min_p > 0 && !l.greedy;
    const bool limited = by_count || by_mass || by_share;
    // Borders are shares of the whole mass where nothing cuts it before: a sum of doubles.  Else it is only told of (all_logs): floats.
    if (__any_sync(0xffffffffu, live && !by_count && !by_share)) {
        each_score([&](float x, int) { all += live ? weight_of(x) : 0.0; });
    } else {
        const float c = (float)(l.inv_t * 1.4426950408889634), base = live ? top : 0.f;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
        int i = 0;
        each_score([&](float x, int) {
            part[i & 3] += exp2_fast(__fsub_rn(x, base) * c);
            ++i;
        });
        all = (double)__fadd_rn(__fadd_rn(part[0], part[1]), __fadd_rn(part[2], part[3]));
    }
    least = 0; count = 0;
    {
        float high = 0;
        over.all(all, least, high, count);
    }
    if (l.greedy) all = 1.0;
    // A border that all that is left reaches, rounded down by more than its floats can be off: 2^-19 of its distance from the largest score (logf: 2^-23,
    // products 2^-24 each), of T (the share under the logarithm is rounded) and of that score.
    float low = minus_inf(), high = top;
    {
        const float t = (float)(1.0 / l.inv_t);
        float down = -FLT_MAX;
        if (l.greedy) down = 0.f;
        else if (by_share) down = logf((float)l.min_p) * t;
        else if (by_mass && !by_count) down = logf((float)((1 - l.top_p) * all / a.k)) * t;
        low = l.greedy ? top : __fadd_rn(top, down) - (fabsf(down) + t + fabsf(top)) * 2e-6f;
        if (!(low <= top)) low = down == -FLT_MAX ? minus_inf() : top;
    }
    int own = 0;
    least = -minus_inf();
    double sum = 0;
    each_score([&](float x, int) {
        if (live && x >= low && x > minus_inf()) { ++own; least = fminf(least, x); }
    });
    count = (float)own;
    const int counted = over.turn;
    over.all(sum, least, high, count);
    low = least;
    high = top;
    bool again = false;   // what was counted above is not what the list takes
    bool narrowing = limited && count > (float)MOST && (by_count || (by_mass && !by_share));   // (of what min_p leaves the whole mass is needed)
    const double enough = by_count ? (double)top_k : l.top_p * all * (1 + 1e-9);
    while (__any_sync(0xffffffffu, narrowing)) {
        again = true;
        const float mid = middle(low, high);
        float reach = 0, up = -minus_inf(), down = minus_inf();
        sum = 0;
        each_score([&](float x, int) {
            if (x >= mid) {
                reach += 1.f;
                up = fminf(up, x);
                if (narrowing && !by_count) sum += weight_of(x);
            } else if (x >= low) {
                down = fmaxf(down, x);
            }
        });
        over.all(sum, up, down, reach);
        if (narrowing) {
            if ((by_count ? (double)reach : sum) >= enough) { low = up; count = reach; }
            else high = down;
            narrowing = count > (float)MOST && low < high;
        }
    }
    const bool listed = limited && count <= (float)MOST;   // this lane's row is settled by its list
    int list_size = 0;
    if (__any_sync(0xffffffffu, listed)) {
        int at = 0;
        if (again) {
            own = 0;
            each_score([&](float x, int) { own += listed && x >= low; });
            at = over.in_front(own, list_size);
        } else {   // (the counts of a moment ago are still there)
            if constexpr (W > 1)
                for (int v = 0; v < warp; ++v) at += (int)sh.counts[counted][v][lane];
            list_size = listed ? (int)count : 0;
        }
        each_score([&](float x, int k) {
            if (listed && x >= low) {
                list.x[at][lane] = x;
                list.k[at][lane] = (unsigned short)k;
                ++at;
            }
        });
        if (warp == 0) {
            list.all[lane] = all; list.top[lane] = top;
            list.size[lane] = list_size;   // (0: not settled here)
        }
        meet<W>();
        // L lanes for a row: all warps, each for 32 / W rows
        constexpr int L = W;
        const int row = warp * (32 / W) + lane / L, sub = lane % L, size = list.size[row];
        const Limits rl = W == 1 ? l : limits_of(a, min(first + row, a.n - 1ll));
        const Exponent row_weight(rl);
        const float row_top = list.top[row];
        const int row_k = rl.greedy ? 1 : rl.top_k, longest = __reduce_max_sync(0xffffffffu, size);
        const bool cuts = size > 0 && row_k < a.k, parts = size > 0 && rl.top_p < 1 && !rl.greedy, shares = rl.min_p > 0 && !rl.greedy;
        float lowest = -minus_inf();
        int number = 0;
        double mass = 0;
        for (int i = sub; i < longest; i += L) {
            if (i >= size) continue;
            const float v = list.x[i][row];
            double m = row_weight(sh.powers, v, row_top);
            if (m < rl.min_p) m = 0;
            list.w[i][row] = m;
            if (m > 0) { ++number; lowest = fminf(lowest, v); mass += m; }
        }
        number = lanes_sum<L>(number); lowest = lanes_min<L>(lowest); mass = lanes_sum<L>(mass);
        auto each = [&](auto &&f) {
#pragma unroll 4
            for (int i = sub; i < longest; i += L)
                if (i < size) {
                    const double v = list.w[i][row];
                    if (v > 0) f(list.x[i][row], v, i);
                }
        };
        auto together = [](double &sum, float &up, float &down) { sum = lanes_sum<L>(sum); up = lanes_min<L>(up); down = lanes_max<L>(down); };
        // leaves the first r of the scores that equal `at`, and what is larger
        auto leave = [&](bool active, float at, int r, int ties) {
            each([&](float v, double, int i) {
                if (active && v < at) list.w[i][row] = 0;
            });
            if (__any_sync(0xffffffffu, active && r < ties)) {
                __syncwarp();
                if (active && r < ties && sub == 0) {
                    int seen = 0;
                    for (int i = 0; i < size; ++i)
                        if (list.w[i][row] > 0 && list.x[i][row] == at && ++seen > r) list.w[i][row] = 0;
                }
                __syncwarp();
            }
        };
        const bool cut = cuts && row_k < number;
        if (__any_sync(0xffffffffu, cut)) {
            const float at = reached(cut, (double)row_k, lowest, row_top, [&](auto &&f) { each([&](float v, double, int) { f(v, 1.0); }); }, together);
            int above = 0, ties = 0;
            each([&](float v, double, int) { above += v > at; ties += v == at; });
            leave(cut, at, row_k - lanes_sum<L>(above), lanes_sum<L>(ties));
            if (cut) lowest = at;
            mass = 0;
            each([&](float, double m, int) { mass += m; });
            mass = lanes_sum<L>(mass);
        }
        if (__any_sync(0xffffffffu, parts)) {
            // of what the limits before leave: all of it stands in the list, unless top_p alone made the border
            const double target = rl.top_p * (cuts || shares ? mass : list.all[row]);
            const float at = reached(parts, target, lowest, row_top, [&](auto &&f) { each([&](float v, double m, int) { f(v, m); }); }, together);
            double above = 0;
            int ties = 0;
            each([&](float v, double m, int) {
                if (v > at) above += m;
                ties += v == at;
            });
            ties = lanes_sum<L>(ties);
            leave(parts, at, ties_left(target, lanes_sum<L>(above), row_weight(sh.powers, at, row_top), ties), ties);
            mass = 0;
            each([&](float, double m, int) { mass += m; });
            mass = lanes_sum<L>(mass);
        }
        if (sub == 0) list.mass[row] = mass;
        meet<W>();
    }
    // the others: over all scores, what is left out becomes -inf
    const bool rest = limited && !listed;
    if (__any_sync(0xffffffffu, rest)) {
        auto each = [&](bool masses) {
            return [&, masses](auto &&f) {
                each_score([&](float x, int) {
                    if (rest && x > minus_inf()) f(x, masses ? weight_of(x) : 1.0);
                });
            };
        };
        auto together = [&](double &s, float &up, float &down) {
            float none = 0;
            over.all(s, up, down, none);
        };
        auto leave = [&](bool active, float at, int r) {
            int own = 0, total;
            each_score([&](float x, int) { own += x == at; });
            int before = over.in_front(own, total);
            each_score([&](float x, int k) {
                const bool tie = x == at;
                if (active && (x < at || (tie && before >= r))) mine_x[k * apart] = minus_inf();
                before += tie;
            });
        };
        auto over_at = [&](float at, bool masses, double &above, int &ties, float &lowest) {
            above = 0;
            float t = 0, none = 0;
            lowest = -minus_inf();
            each(masses)([&](float v, double m) {
                if (v > at) above += m;
                t += v == at ? 1.f : 0.f;
                lowest = fminf(lowest, v);
            });
            over.all(above, lowest, none, t);
            ties = (int)t;
        };
        if (rest && by_share)
            each_score([&](float x, int k) {
                if (weight_of(x) < l.min_p) mine_x[k * apart] = minus_inf();
            });
        double above;
        int ties;
        float lowest;
        const bool cut = rest && by_count;
        if (__any_sync(0xffffffffu, cut)) {
            over_at(minus_inf(), false, above, ties, lowest);
            const bool some = cut && (double)top_k < above;
            const float at = reached(some, (double)top_k, lowest, top, each(false), together);
            over_at(at, false, above, ties, lowest);
            leave(some, at, top_k - (int)above);
        }
        const bool part = rest && by_mass;
        if (__any_sync(0xffffffffu, part)) {
            over_at(minus_inf(), true, above, ties, lowest);
            const double target = l.top_p * above;
            const float at = reached(part, target, lowest, top, each(true), together);
            over_at(at, true, above, ties, lowest);
            leave(part, at, ties_left(target, above, weight_of(at), ties));
        }
    }
    double mine = 0, front, end;
    bool last;
    const bool over_all = live && !listed, some_over_all = __any_sync(0xffffffffu, over_all);
    if (some_over_all) each_score([&](float x, int) { mine += over_all ? weight_of(x) : 0.0; });
    double mass = over.shares(mine, front, end, last);
    if (listed) mass = list.mass[lane];
    double log_mass = 0, log_all = 0;
    if (live && warp < a.draws) { log_mass = log(mass); log_all = log(all); }
    for (int d0 = 0; d0 < a.draws; d0 += W) {
        const int some = min(W, a.draws - d0);
        if (some_over_all) {
            for (int d = 0; d < some; ++d) {
                const double target = uniform_of(a, n * a.draws + d0 + d) * mass;
                const bool hit = mine > 0 && front <= target && (end > target || last);
                if (!__any_sync(0xffffffffu, hit)) continue;
                double upto = front;
                int at = 0;
                float s = 0;
                bool found = false;
                each_score([&](float x, int k) {
                    const double v = hit && !found ? weight_of(x) : 0.0;
                    if (v > 0) {
                        upto += v;
                        at = k;
                        s = x;
                        found = upto > target;
                    }
                });
                if (hit) { sh.cls[d][lane] = at; sh.score[d][lane] = s; }
            }
            meet<W>();
        }
        if (warp < some) {
            int cls = -1;
            float score = 0;
            if (listed) {
                const double target = uniform_of(a, n * a.draws + d0 + warp) * mass;
                double upto = 0;
                for (int i = 0; i < list_size && (i == 0 || !(upto > target)); ++i) {
                    const double v = list.w[i][lane];
                    if (v > 0) {
                        upto += v;
                        cls = list.k[i][lane];
                        score = list.x[i][lane];
                    }
                }
            } else if (live) {
                cls = sh.cls[warp][lane];
                score = sh.score[warp][lane];
            }
            if (n0 == n) {
                const long long at = n * a.draws + d0 + warp;
                if (live) {
                    const double lw = ((double)score - (double)top) * l.inv_t;
                    put_draw(a, at, cls, (float)(lw - log_mass), (float)(lw - log_all));
                } else {
                    const float v = bad ? __int_as_float(0x7fffffff) : minus_inf();
                    put_draw(a, at, -1, v, v);
                }
            }
        }
        if (some_over_all) meet<W>();
    }
}

// ---- long rows: a cluster of up to 8 blocks (or one) holds the row in its registers -------------------------------------------
// Classes stand in the order block, u, thread, place in the pack (Hold); a segment is what a warp has of one u, 32 packs side by side.
//
// Limits: as above the scores that can be left are those from a border on, which is raised by bisection over the registers while more than
// LONG_LIST reach it.  They go into a list in the first block, in class order, and that block alone goes on: every entry counts the larger ones,
// which is its place in descending order; prefix sums in that order tell where top_p ends, prefix sums in class order which class a random number
// falls on.  Where top_p alone leaves more, what is certainly left is told from what the end of it lies among, and only that goes into the list.
// Rows with more than a list, and rows without limits, take their draws from sums per segment.
constexpr int LONG_LIST = 1024;

template <int W, int S> struct LongRow {
    Powers powers;
    double sums[W], slot_sum[2], sum, front;          // of the warps, of this block (read by the others), of the row, of the blocks in front
    float lows[W], highs[W], slot_low[2], slot_high[2], low, high;
    int counts[W], slot_count[2], count, front_count;
    double segment[S];                                // of a segment, then of all in front of it
    int segment_count[S];
    int tie, last;
    float tie_score, at;
    __align__(16) unsigned key[LONG_LIST];
    int k[LONG_LIST];
    double w[LONG_LIST], upto[LONG_LIST];
};

// The list of a row, `size` entries in class order: what is left of it (w[i] > 0), prefix sums in class order (upto), its mass.  `base`: mass of what is
// larger than all entries (only where `border`: then the last entry that is left is told, in at and last).  All threads of a block.
template <int W, int S>
__device__ __noinline__ double settle_list(LongRow<W, S> &sh, const Exponent &weight, float top, int size, double min_p, int top_k, bool by_mass, bool of_list, double top_p,
                                           double all, double base, bool border) {
    constexpr int TH = 32 * W, Q = LONG_LIST / TH;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // exclusive prefix of the threads' sums
    auto scan = [&](double own, double &whole) {
        double upto = own;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const double v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        __syncthreads();
        if (lane == 31) sh.sums[warp] = upto;
        __syncthreads();
        double before = 0;
        whole = 0;
        for (int v = 0; v < W; ++v) {
            if (v == warp) before = whole;
            whole += sh.sums[v];
        }
        return before + (upto - own);
    };
    auto count = [&](int own) {
        own = warp_sum(own);
        __syncthreads();
        if (lane == 0) sh.counts[warp] = own;
        __syncthreads();
        int s = 0;
        for (int v = 0; v < W; ++v) s += sh.counts[v];
        return s;
    };
    if (tid < 4 && size + tid < LONG_LIST) sh.key[size + tid] = 0;   // (read four at a time)
    __syncthreads();
    int place[Q], heavy = 0;
    double mine[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = q * TH + tid;
        place[q] = size;
        mine[q] = 0;
        if (i < size) {
            const unsigned own = sh.key[i];
            mine[q] = weight(sh.powers, key_score(own), top);
            heavy += mine[q] >= min_p;
            int larger = 0;   // entries in front of this one in descending order: of equal ones those of lower classes
            for (int j = 0; j < size; j += 4) {
                const uint4 o = *reinterpret_cast<const uint4 *>(&sh.key[j]);
                const unsigned over = own + (j + 4 > i);
                larger += (o.x >= over) + (o.y >= over) + (o.z >= over) + (o.w >= over);
            }
            for (int j = i & ~3; j < i; ++j) larger += sh.key[j] == own;
            place[q] = larger;
        }
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (place[q] < size) sh.w[place[q]] = mine[q];
    int keep = min(count(heavy), top_k);   // in descending order
    if (by_mass) {
        // entries tid Q + q in descending order: prefix sums
        double s = 0, whole;
#pragma unroll
        for (int q = 0; q < Q; ++q) s += tid * Q + q < keep ? sh.w[tid * Q + q] : 0.0;
        double upto = base + scan(s, whole);
        const double target = top_p * (of_list ? whole : all);
        int before = 0;   // entries in front of which the target is not reached
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (tid * Q + q < keep) {
                before += tid * Q + q == 0 || upto < target;
                upto += sh.w[tid * Q + q];
            }
        keep = count(before);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int i = q * TH + tid;
        if (i < size) {
            sh.w[i] = place[q] < keep ? mine[q] : 0.0;   // in class order now
            if (border && place[q] == keep - 1) { sh.at = key_score(sh.key[i]); sh.last = sh.k[i]; }
        }
    }
    __syncthreads();
    double s = 0, mass;
#pragma unroll
    for (int q = 0; q < Q; ++q) s += tid * Q + q < size ? sh.w[tid * Q + q] : 0.0;
    double upto = scan(s, mass);
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (tid * Q + q < size) {
            upto += sh.w[tid * Q + q];
            sh.upto[tid * Q + q] = upto;
        }
    __syncthreads();
    return sh.upto[size - 1];
}

template <typename T, int TH, int P, bool EVEN>
__global__ void __launch_bounds__(TH, 1024 / TH) k_sample_long(SampleArgs a, Scores<T> in) {
    typedef Hold<T, TH, P, EVEN> H;
    constexpr int V = H::V, W = TH / 32, S = P * W;
    __shared__ __align__(16) LongRow<W, S> sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long n = blockIdx.x / C;
    const int lo = rank * H::CELLS, cells = min(a.k - lo, H::CELLS);
    H hold;
    hold.read(in.at(n, lo), cells);
    if (warp == 0) sh.powers.fill();
    const Limits l = limits_of(a, n);
    // f(score, class - lo) in class order within u; -inf behind the last class
    auto each_of = [&](int u, auto &&f) {
        float v[V];
        if (H::first(u) < cells) hold.get(u, v);
#pragma unroll
        for (int i = 0; i < V; ++i) f(H::first(u) < cells ? v[i] : minus_inf(), H::first(u) + i);
    };
    auto each = [&](auto &&f) {
#pragma unroll
        for (int u = 0; u < P; ++u) each_of(u, f);
    };
    // of all threads of all blocks, the same everywhere; front, front_count: of the blocks in front of this one
    int turn = 0;
    double front = 0;
    int front_count = 0;
    auto total = [&](double &sum, float &low, float &high, int &count) {
        sum = warp_sum(sum); low = lanes_min<32>(low); high = lanes_max<32>(high); count = warp_sum(count);
        if (lane == 0) { sh.sums[warp] = sum; sh.lows[warp] = low; sh.highs[warp] = high; sh.counts[warp] = count; }
        __syncthreads();
        if (warp == 0) {
            sum = lanes_sum<W>(sh.sums[lane & (W - 1)]); count = lanes_sum<W>(sh.counts[lane & (W - 1)]);
            low = lanes_min<W>(sh.lows[lane & (W - 1)]); high = lanes_max<W>(sh.highs[lane & (W - 1)]);
            if (lane == 0) { sh.slot_sum[turn] = sum; sh.slot_low[turn] = low; sh.slot_high[turn] = high; sh.slot_count[turn] = count; }
        }
        if (C > 1) cluster.sync();
        if (warp == 0) {
            double before = 0, its = sum;
            int before_count = 0, its_count = count;
            if (C > 1) {
                const LongRow<W, S> *o = cluster.map_shared_rank(&sh, lane < C ? lane : 0);
                its = o->slot_sum[turn]; its_count = o->slot_count[turn]; low = o->slot_low[turn]; high = o->slot_high[turn];
                low = lanes_min<LONG_CLUSTER>(low); high = lanes_max<LONG_CLUSTER>(high);
                sum = 0; count = 0;
                for (int b = 0; b < C; ++b) {   // one after the other: where one block's part ends the next one's begins
                    if (b == rank) { before = sum; before_count = count; }
                    sum += __shfl_sync(0xffffffffu, its, b);
                    count += __shfl_sync(0xffffffffu, its_count, b);
                }
            }
            if (lane == 0) { sh.sum = sum; sh.low = low; sh.high = high; sh.count = count; sh.front = before; sh.front_count = before_count; }
        }
        __syncthreads();
        sum = sh.sum; low = sh.low; high = sh.high; count = sh.count; front = sh.front; front_count = sh.front_count;
        turn ^= 1;
    };
    // sums of the segments become those of all segments in front; returns the block's
    auto prefix = [&](auto *of) {
        auto before = of[0] - of[0];
        __syncthreads();
        if (warp == 0) {
            for (int s = 0; s < S; s += 32) {
                const auto own = s + lane < S ? of[s + lane] : before - before;
                auto upto = own;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const auto v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                if (s + lane < S) of[s + lane] = before + (upto - own);
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        __syncthreads();
    };
    float top = minus_inf(), low = -minus_inf(), none = 0;
    double sum = 0;
    int count = 0;
    each([&](float x, int) {
        top = fmaxf(top, x);
        count |= x != x;
    });
    // Each group of lanes that holds a score has a largest one, and the least of these is reached by as many scores as there are groups: the first
    // guess of a border.  Groups are as large as they may be to be top_k.
    const int top_k = l.greedy ? 1 : l.top_k, groups = max(1, a.k / H::E);   // (threads that hold all their scores)
    {
        float its = top;
#pragma unroll
        for (int o = 1; o < 32; o *= 2)
            if (groups / (2 * o) >= max(top_k < a.k ? top_k : 0, 96)) its = fmaxf(its, __shfl_xor_sync(0xffffffffu, its, o));
        low = its > minus_inf() ? its : low;
    }
    total(sum, low, top, count);
    const bool bad = l.broken || count || top == -minus_inf();
    if (bad || top == minus_inf()) {   // (the same for all blocks; none reads another's memory any more than it did before the last barrier)
        const float v = bad ? __int_as_float(0x7fffffff) : minus_inf();
        if (rank == 0)
            for (int d = tid; d < a.draws; d += TH) put_draw(a, n * a.draws + d, -1, v, v);
        if (C > 1) cluster.sync();
        return;
    }
    const Exponent weight(l);
    auto weight_of = [&](float v) { return weight(sh.powers, v, top); };
    const bool by_count = top_k < a.k, by_mass = l.top_p < 1 && !l.greedy, by_share = l.min_p > 0 && !l.greedy;
    const float guess = low;
    double all = 0;
    // what is left: larger than `at`, or equal to it and a class up to `last`
    float at = minus_inf();
    int last = a.k;
    auto left = [&](float x, int k) { return x > at || (x == at && x > minus_inf() && lo + k <= last); };
    // masses of segments, of what is left
    auto segments = [&] {
        double s[P], mine = 0;
#pragma unroll
        for (int u = 0; u < P; ++u) {
            s[u] = 0;
            each_of(u, [&](float x, int k) { s[u] += left(x, k) ? weight_of(x) : 0.0; });
        }
        constexpr int PER = 32 / P;
        mine = sums_spread<P>(s);
        if (lane % PER == 0) {
            sh.segment[lane / PER * W + warp] = mine;
            sh.segment_count[lane / PER * W + warp] = mine > 0;
        }
        mine = lane % PER == 0 ? mine : 0.0;
        float f0 = 0, f1 = 0;
        int c0 = 0;
        total(mine, f0, f1, c0);
        prefix(sh.segment);
        return mine;
    };
    double mass = 0;
    bool listed = false;
    if (by_count || by_mass || by_share) {
        const float c = (float)(l.inv_t * 1.4426950408889634);
        auto rough = [&](float x) { return exp2_fast(__fsub_rn(x, top) * c); };
        float f0 = 0, f1 = 0;
        const bool exact = !by_count && !by_share;   // top_p alone: a share of the whole mass
        if (exact) {
            each([&](float x, int) { all += weight_of(x); });
            count = 0;
            total(all, f0, f1, count);
        }
        // the border, rounded down as in k_sample_limited; what lies 750 T below the largest score has no mass in any case
        const float t = (float)(1.0 / l.inv_t);
        float down = -750.f * t;
        if (by_share) down = logf((float)l.min_p) * t;
        else if (exact) down = logf((float)((1 - l.top_p) * all / a.k)) * t;
        low = __fadd_rn(top, down) - (fabsf(down) + t + fabsf(top)) * 2e-6f;
        if (l.greedy) low = top;
        if (!(low <= top)) low = minus_inf();
        low = fmaxf(low, -FLT_MAX);
        const float base = low;
        if (by_count && guess <= top) low = fmaxf(low, guess);
        unsigned reach = 0;   // bits of this thread's scores from the border on
        auto mark = [&](float border) {
            reach = 0;
            int bit = 0;
            each([&](float x, int) {
                reach |= x >= border ? 1u << bit : 0u;
                ++bit;
            });
        };
        mark(low);
        count = __popc(reach);
        if (!exact) {
            float part = 0;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                float s = 0;
                each_of(u, [&](float x, int) { s += rough(x); });
                part += s;
            }
            all = (double)part;
            total(all, f0, f1, count);
        } else {
            total(sum, f0, f1, count);
        }
        if (l.greedy) all = 1.0;
        if (by_count && count < top_k && low > base) {   // (groups without a score: the guess was too high)
            low = base;
            mark(low);
            count = __popc(reach);
            total(sum, f0, f1, count);
        }
        float high = top;
        const bool narrowing = by_count ? top_k <= LONG_LIST : by_mass && !by_share;
        // top_p alone: masses by floats, off by less than 2^-18, tell what certainly reaches the target and what certainly does not
        const double enough = l.top_p * all * (1 + 1e-5), short_of = l.top_p * all * (1 - 1e-5);
        int above = 0;   // scores larger than `high`, which are left in any case
        bool first = !by_count && guess > low && guess < top, moved = false;
        while (narrowing && count - above > LONG_LIST && low < high) {
            const float mid = first ? guess : middle(low, high);
            first = false;
            float up = -minus_inf(), below = minus_inf();
            int c = 0;
            sum = 0;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                if (!__any_sync(0xffffffffu, reach >> (u * V) & ((1ull << V) - 1))) continue;   // (nothing from the border on)
                float part = 0;
                each_of(u, [&](float x, int) {
                    if (x >= mid) {
                        ++c;
                        up = fminf(up, x);
                        if (!by_count) part += rough(x);
                    } else if (x >= low) {
                        below = fmaxf(below, x);
                    }
                });
                sum += (double)part;
            }
            total(sum, up, below, c);
            if (by_count ? c >= top_k : sum >= enough) { low = up; count = c; moved = true; }
            else if (below > minus_inf() && (by_count || sum < short_of)) {
                high = below;
                if (!by_count) above = c;
            } else break;
        }
        // whole: all that can be left stands in the list; part: so does the border, and what is larger is left
        const bool whole = count <= LONG_LIST, part = !whole && narrowing && !by_count && count - above <= LONG_LIST;
        listed = whole;
        if (whole) above = 0;
        if (whole || part) {
            double base = 0;
            if (part) {
                each([&](float x, int) { base += x > high ? weight_of(x) : 0.0; });
            } else {
                high = top;
            }
            auto inside = [&](float x) { return x >= low && x <= high; };
            if (moved || part) {
                reach = 0;
                int bit = 0;
                each([&](float x, int) {
                    reach |= inside(x) ? 1u << bit : 0u;
                    ++bit;
                });
            }
            // into the first block's list, in class order
            auto bits = [&](int u) { return (unsigned)(reach >> (u * V) & ((1ull << V) - 1)); };
            int mine = __popc(reach);
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const int s = __reduce_add_sync(0xffffffffu, __popc(bits(u)));
                if (lane == 0) sh.segment_count[u * W + warp] = s;
            }
            total(base, f0, f1, mine);
            prefix(sh.segment_count);
            LongRow<W, S> *to = C > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const int c = __popc(bits(u));
                if (!__any_sync(0xffffffffu, c)) continue;
                int upto = c;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                int place = front_count + sh.segment_count[u * W + warp] + upto - c;
                each_of(u, [&](float x, int k) {
                    if (inside(x)) { to->key[place] = plain_key(x); to->k[place] = lo + k; ++place; }
                });
            }
            if (C > 1) cluster.sync();
            else __syncthreads();
            if (rank == 0) {
                const int size = count - above;
                mass = settle_list(sh, weight, top, size, l.min_p, top_k, by_mass, by_count || by_share, l.top_p, all, base, part);
                if (part && tid < C) {   // the border, for all blocks
                    LongRow<W, S> *o = C > 1 ? cluster.map_shared_rank(&sh, tid) : &sh;
                    o->tie_score = sh.at; o->tie = sh.last;
                }
                count = size;
            } else if (whole) {
                return;
            }
            if (part) {
                if (C > 1) cluster.sync();
                else __syncthreads();
                at = sh.tie_score; last = sh.tie;
                mass = segments();
            }
        } else {
            // over all scores
            if (by_share) {
                float lightest = -minus_inf();
                each([&](float x, int) {
                    if (x >= low && weight_of(x) >= l.min_p) lightest = fminf(lightest, x);
                });
                count = 0;
                total(sum, lightest, f1, count);
                at = lightest;
            } else {
                each([&](float x, int) { at = fminf(x > minus_inf() ? x : -minus_inf(), at == minus_inf() ? -minus_inf() : at); });
                count = 0;
                total(sum, at, f1, count);
            }
            auto together = [&](double &s, float &up, float &below) {
                int c = 0;
                total(s, up, below, c);
            };
            // the first r of the scores that equal `at`
            auto cut_ties = [&](int r) {
                int mine = 0;
#pragma unroll
                for (int u = 0; u < P; ++u) {
                    int c = 0;
                    each_of(u, [&](float x, int k) { c += x == at && lo + k <= last; });
                    mine += c;
                    const int s = __reduce_add_sync(0xffffffffu, c);
                    if (lane == 0) sh.segment_count[u * W + warp] = s;
                }
                total(sum, f0, f1, mine);
                prefix(sh.segment_count);
#pragma unroll
                for (int u = 0; u < P; ++u) {
                    int c = 0;
                    each_of(u, [&](float x, int k) { c += x == at && lo + k <= last; });
                    int upto = c;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {
                        const int v = __shfl_up_sync(0xffffffffu, upto, o);
                        if (lane >= o) upto += v;
                    }
                    int seen = front_count + sh.segment_count[u * W + warp] + upto - c;
                    each_of(u, [&](float x, int k) {
                        if (x == at && lo + k <= last && ++seen == r)
                            for (int b = 0; b < C; ++b) (C > 1 ? cluster.map_shared_rank(&sh, b) : &sh)->tie = lo + k;
                    });
                }
                if (C > 1) cluster.sync();
                else __syncthreads();
                last = sh.tie;
            };
            auto measured = [&](bool masses) {
                return [&, masses](auto &&f) {
                    each([&](float x, int k) {
                        if (left(x, k)) f(x, masses ? weight_of(x) : 1.0);
                    });
                };
            };
            auto settle = [&](bool masses, double target) {
                const float found = reached(true, target, at, top, measured(masses), together);
                double above = 0;
                int ties = 0;
                measured(masses)([&](float x, double m) {
                    if (x > found) above += m;
                    ties += x == found;
                });
                total(above, f0, f1, ties);
                const int r = masses ? ties_left(target, above, weight_of(found), ties) : (int)(target - above);
                if (found > at) { at = found; last = a.k; }
                if (r < ties) cut_ties(r);
            };
            if (by_count) {
                count = 0;
                each([&](float x, int k) { count += left(x, k); });
                total(sum, f0, f1, count);
                if (top_k < count) settle(false, (double)top_k);
            }
            if (by_mass) {
                sum = 0;
                measured(true)([&](float, double m) { sum += m; });
                count = 0;
                total(sum, f0, f1, count);
                settle(true, l.top_p * sum);
            }
            mass = segments();
        }
    } else {
        mass = all = segments();
    }
    auto put = [&](long long i, int cls, float score, double log_mass, double log_all) {
        const double lw = ((double)score - (double)top) * l.inv_t;
        put_draw(a, i, cls, (float)(lw - log_mass), (float)(lw - log_all));
    };
    if (!listed) {
        // this block's draws: those that fall into [front, front + its mass), and where nothing is left behind it also what rounding leaves there
        const double log_mass = log(mass), log_all = log(all), own_end = front + sh.slot_sum[turn ^ 1];   // (the last total was of the masses)
        bool behind = false;
        for (int b = rank + 1; b < C; ++b) behind |= cluster.map_shared_rank(&sh, b)->slot_sum[turn ^ 1] > 0;
        const bool some = own_end > front;
        for (int d = warp; d < a.draws; d += W) {
            const long long i = n * a.draws + d;
            const double target = uniform_of(a, i) * mass;
            if (!(some && front <= target && (own_end > target || !behind))) continue;
            // the last segment that begins at or before the target; the one in front of it (or behind) where it is empty
            int from = 0, to = S;
            while (to - from > 1) {
                const int mid = (from + to) / 2;
                if (front + sh.segment[mid] <= target) from = mid;
                else to = mid;
            }
            while (from > 0 && !sh.segment_count[from]) --from;
            while (from < S - 1 && !sh.segment_count[from]) ++from;
            const int cell = ((from / W) * TH + (from % W) * 32 + lane) * V;
            float x[V];
            double w[V], own = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[j] = cell < cells ? in(n, lo + cell + j) : minus_inf();
                w[j] = left(x[j], cell + j) ? weight_of(x[j]) : 0.0;
                own += w[j];
            }
            double upto = own;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const double v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            double before = front + sh.segment[from] + (upto - own);
            const unsigned has = __ballot_sync(0xffffffffu, own > 0), hit = __ballot_sync(0xffffffffu, own > 0 && before + own > target);
            const int src = hit ? __ffs(hit) - 1 : 31 - __clz(has);
            if (lane == src) {
                int cls = 0;
                float s = 0;
                bool found = false;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (!found && w[j] > 0) {
                        before += w[j];
                        cls = lo + cell + j;
                        s = x[j];
                        found = before > target;
                    }
                put(i, cls, s, log_mass, log_all);
            }
        }
        if (C > 1) cluster.sync();   // (others look at this block's sums)
        return;
    }
    const int size = count;
    for (int d = tid; d < a.draws; d += TH) {
        const long long i = n * a.draws + d;
        const double target = uniform_of(a, i) * mass;
        int from = 0, to = size - 1;   // the first entry beyond the target, or the last that is left
        while (from < to) {
            const int mid = (from + to) / 2;
            if (sh.upto[mid] > target || sh.upto[mid] >= mass) to = mid;
            else from = mid + 1;
        }
        while (from > 0 && !(sh.w[from] > 0)) --from;   // (prefix sums by different threads are not rounded alike)
        put(i, sh.k[from], key_score(sh.key[from]), log(mass), log(all));
    }
}

// ------------------------------------------------------------------ feedback
// A row's sums, relative to its largest score: sum of e = exp((s - top) / T) and of e (s - top).  What follows from them and the draws:
//   g_i = p_i (by_d (s_i - top) + flat) + [draws of i],  h_i = max(curve p_i (1 - p_i), 1e-16),  p_i = e_i to_p
struct FeedbackRow {
    float top, c, to_p, by_d, flat, curve;
    bool counts;   // without a draw that counts, or with a weight of 0, the row has no loss
};
constexpr float MIN_HESSIAN = 1e-16f;   // the softmax objective's

struct Draw {
    double term, to_log;   // loss of one draw, its derivative by the log-probability
};
__device__ __forceinline__ Draw draw_of(const FeedbackArgs &a, double lp, float its_gain, float old, float reference) {
    const double gain = (double)its_gain, r = a.old ? exp(lp - (double)old) : 1.0;
    const double held = fmin(fmax(r, (double)a.least), (double)a.most);
    Draw d;
    d.term = gain == 0 ? 0.0 : -fmin(r * gain, held * gain);   // (what weighs 0 counts for nothing, also where the ratio is infinite)
    d.to_log = gain != 0 && r * gain <= held * gain ? -r * gain : 0.0;
    if (a.kl != 0.f) {
        const double x = (double)reference - lp, e = exp(x);
        d.term += (double)a.kl * (e - x - 1);
        d.to_log += (double)a.kl * (1 - e);
    }
    return d;
}

// The row's loss, and what its gradients need; `by`: what a draw's derivative is multiplied by
__device__ __forceinline__ FeedbackRow factors_of(const FeedbackArgs &a, long long n, float w, float top, float sum, float sum_d, double log_sum, double term,
                                                  double to_log, double size, int number, bool writes, double &by) {
    const double inv_sum = sum == 0.f ? 0.0 : 1.0 / (double)sum, spread = log_sum - (double)sum_d * a.inv_t * inv_sum;   // (the entropy)
    FeedbackRow r;
    r.counts = number > 0 && w != 0.f;
    const double share = number == 1 ? 1.0 : number ? 1.0 / number : 0.0, scale = (double)w * a.inv_t;
    if (a.loss && writes) a.loss[n] = r.counts ? (float)((double)w * (term * share - (a.entropy != 0.f ? (double)a.entropy * spread : 0.0))) : 0.f;
    r.top = top; r.c = a.c;
    r.to_p = (float)inv_sum;
    r.by_d = (float)(scale * (double)a.entropy * a.inv_t);
    r.flat = (float)(scale * ((a.entropy != 0.f ? (double)a.entropy * (spread - log_sum) : 0.0) - to_log * share));
    r.curve = (float)(2 * scale * a.inv_t * (size * share + (double)a.entropy));
    by = scale * share;
    return r;
}

// What lane l has of the draws l, l + 32, ...: read early where there is something else to wait for
struct DrawsRead {
    int cls[SCORES_MAX_TOP / 32];
    float score[SCORES_MAX_TOP / 32], gain[SCORES_MAX_TOP / 32], old[SCORES_MAX_TOP / 32], reference[SCORES_MAX_TOP / 32];
    float weight;
};
template <typename T> __device__ __forceinline__ DrawsRead read_draws(const FeedbackArgs &a, const Scores<T> &in, long long n) {
    DrawsRead r;
    r.weight = a.weights ? a.weights[n] : 1.f;
#pragma unroll
    for (int j = 0; j < SCORES_MAX_TOP / 32; ++j) {
        const int e = (threadIdx.x & 31) + 32 * j;
        if (e >= a.draws) break;
        const long long at = n * a.draws + e;
        r.cls[j] = a.classes[at];
        r.gain[j] = a.gains[at];
        r.old[j] = a.old ? a.old[at] : 0.f;
        r.reference[j] = a.kl != 0.f ? a.reference[at] : 0.f;
        r.score[j] = r.cls[j] >= 0 && r.cls[j] < a.k ? in(n, r.cls[j]) : minus_inf();
    }
    return r;
}
// One warp, for the row n: logs, the loss and what its gradients need.  cls[e], extra[e]: class of draw e and what is added there (-1: nothing;
// of draws of one class the first has the sum).
__device__ __forceinline__ FeedbackRow feedback_row(const FeedbackArgs &a, long long n, float top, float sum, float sum_d, int *cls, float *extra, bool writes,
                                                     const DrawsRead &draws) {
    const int lane = threadIdx.x & 31;
    const double log_sum = sum == 0.f ? 0.0 : fine_log(sum);
    double term = 0, to_log = 0, size = 0;
    int number = 0;
#pragma unroll
    for (int j = 0; j < SCORES_MAX_TOP / 32; ++j) {
        const int e = lane + 32 * j;
        if (e >= a.draws) break;
        const long long at = n * a.draws + e;
        const int i = draws.cls[j];
        const float x = draws.score[j];
        const bool counts = x > minus_inf() || x != x;
        const double lp = counts ? ((double)x - (double)top) * a.inv_t - log_sum : (double)minus_inf();
        if (a.logs && writes) a.logs[at] = (float)lp;
        cls[e] = counts ? i : -1;
        extra[e] = 0.f;
        if (counts) {
            const Draw d = draw_of(a, lp, draws.gain[j], draws.old[j], draws.reference[j]);
            term += d.term; to_log += d.to_log; size += fabs(d.to_log);
            extra[e] = (float)d.to_log;
            ++number;
        }
    }
    number = warp_sum(number);
    term = warp_sum(term); to_log = warp_sum(to_log); size = warp_sum(size);
    __syncwarp();
    double by;
    const FeedbackRow r = factors_of(a, n, draws.weight, top, sum, sum_d, log_sum, term, to_log, size, number, writes && lane == 0, by);
    if (a.gives != GIVES_LOSS) {   // of draws of one class the first takes the sum
        float total[SCORES_MAX_TOP / 32];
        bool first[SCORES_MAX_TOP / 32];
#pragma unroll
        for (int j = 0; j < SCORES_MAX_TOP / 32; ++j) {
            const int e = lane + 32 * j;
            double s = 0;
            first[j] = e < a.draws && cls[e] >= 0;
            if (first[j])
                for (int o = 0; o < a.draws; ++o)
                    if (cls[o] == cls[e]) {
                        if (o < e) first[j] = false;
                        s += (double)extra[o];
                    }
            total[j] = (float)(s * by);
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < SCORES_MAX_TOP / 32; ++j) {
            const int e = lane + 32 * j;
            if (e >= a.draws) break;
            if (!first[j]) cls[e] = -1;
            extra[e] = total[j];
        }
        __syncwarp();
    }
    return r;
}
__device__ __forceinline__ float2 feedback_gh(const FeedbackRow &r, float s, float extra) {
    if (!r.counts) return make_float2(0.f, MIN_HESSIAN);
    const float d = __fsub_rn(s, r.top), p = exp2_fast(d * r.c) * r.to_p;
    const float cp = r.curve * p;
    return make_float2(__fmaf_rn(p, __fmaf_rn(r.by_d, fmaxf(d, -1e30f), r.flat), extra), fmaxf(__fmaf_rn(-cp, p, cp), MIN_HESSIAN));   // (p = 0 for -inf)
}
template <typename T> __device__ __forceinline__ void put_gradient(const FeedbackArgs &a, long long n, long long k, float2 gh) {
    const long long at = n * a.out.row + k * a.out.cls;
    if (a.gives == GIVES_PAIRS) static_cast<float2 *>(a.out.data)[at] = gh;
    else static_cast<T *>(a.out.data)[at] = score_from<T>(gh.x);
}

// A row, any strides, by a block in three passes.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) k_feedback_any(FeedbackArgs a, Scores<T> in) {
    __shared__ int cls[SCORES_MAX_TOP];
    __shared__ float extra[SCORES_MAX_TOP];
    __shared__ FeedbackRow shared_row;
    __shared__ float parts[3][ROW_WARPS];
    const long long n = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = minus_inf();
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) m = fmaxf(m, in(n, k));
    m = warp_max(m);
    if (lane == 0) parts[0][warp] = m;
    __syncthreads();
    const float top = row_top(warp_max(parts[0][lane & (ROW_WARPS - 1)]));
    float s = 0, sd = 0;
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
        const float d = __fsub_rn(in(n, k), top), e = exp2_fast(d * a.c);
        s += e;
        sd = __fmaf_rn(e, fmaxf(d, -1e30f), sd);
    }
    s = warp_sum(s); sd = warp_sum(sd);
    if (lane == 0) { parts[1][warp] = s; parts[2][warp] = sd; }
    __syncthreads();
    if (warp == 0) {
        s = warp_sum(lane < ROW_WARPS ? parts[1][lane] : 0.f);
        sd = warp_sum(lane < ROW_WARPS ? parts[2][lane] : 0.f);
        const FeedbackRow r = feedback_row(a, n, top, s, sd, cls, extra, true, read_draws(a, in, n));
        if (lane == 0) shared_row = r;
    }
    __syncthreads();
    float mg = 0, mh = 0;
    if (a.gives != GIVES_LOSS) {
        const FeedbackRow r = shared_row;
        auto put = [&](int k, float more) {
            const float2 gh = feedback_gh(r, in(n, k), more);
            put_gradient<T>(a, n, k, gh);
            mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y);
        };
        for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
            float more = 0;
            for (int e = 0; e < a.draws; ++e)
                if (cls[e] == k) more = extra[e];
            put(k, more);
        }
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

// Up to 1024 classes, by class (and by row up to 32): a lane has a row, W warps share its classes, E neighbours each, which stay in registers from
// the read to the gradients.  A draw of the row is worked out by one of its warps; the cells of drawn classes are written after the others.
template <typename T, int E, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 1 ? 4 : W == 8 ? 3 : W == 16 ? 2 : 1) k_feedback_class(FeedbackArgs a, Scores<T> in) {
    extern __shared__ __align__(16) unsigned char room[];
    struct Shared {
        double sums[3][W][32];
        float2 part[2][W][32];
        int number[W][32];
        unsigned drawn[W][32];
        FeedbackRow row[32];
        double by[32];
    };
    static_assert(sizeof(Shared) <= 32 * (48 * W + sizeof(FeedbackRow) + 8) + 64, "");
    constexpr int G = W == 1 ? 4 : 1;
    const int lane = threadIdx.x & 31, group = W == 1 ? threadIdx.x >> 5 : 0, warp = W == 1 ? 0 : threadIdx.x >> 5, k0 = warp * E, here = a.k - k0;
    Shared &sh = reinterpret_cast<Shared *>(room)[group];   // (W = 1: each warp has its own)
    int *cls = reinterpret_cast<int *>(room + G * sizeof(Shared)) + group * a.draws * 64;   // draws x 32
    float *extra = reinterpret_cast<float *>(cls + a.draws * 32);
    const long long n0 = (blockIdx.x * (long long)G + group) * 32 + lane, n = min(n0, a.n - 1ll);
    float x[E];
    {
        const T *from = in.at(n, k0);
        T raw[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (j < here) raw[j] = from[j * in.cls];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = j < here ? score_f32(raw[j]) : minus_inf();
    }
    float top = minus_inf();
#pragma unroll
    for (int j = 0; j < E; ++j) top = fmaxf(top, x[j]);
    sh.drawn[warp][lane] = 0;
    if constexpr (W > 1) {
        sh.part[0][warp][lane].x = top;
        __syncthreads();
#pragma unroll
        for (int v = 0; v < W; ++v) top = fmaxf(top, sh.part[0][v][lane].x);
    }
    top = row_top(top);
    float s = 0, sd = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const float d = __fsub_rn(x[j], top), e = exp2_fast(d * a.c);
        s += e;
        sd = __fmaf_rn(e, fmaxf(d, -1e30f), sd);
    }
    if constexpr (W > 1) {
        sh.part[1][warp][lane] = make_float2(s, sd);
        __syncthreads();
        float2 all = sh.part[1][0][lane];
#pragma unroll
        for (int v = 1; v < W; ++v) all = add2(all, sh.part[1][v][lane]);
        s = all.x; sd = all.y;
    } else {
        __syncwarp();
    }
    const double log_sum = s == 0.f ? 0.0 : fine_log(s);
    const int busy = min(W, a.draws);   // warps with a draw
    if (warp < busy) {
        double term = 0, to_log = 0, size = 0;
        int number = 0;
        for (int e = warp; e < a.draws; e += W) {
            const long long at = n * a.draws + e;
            const int i = a.classes[at];
            const float v = i >= 0 && i < a.k ? in(n, i) : minus_inf();
            const bool counts = v > minus_inf() || v != v;
            const double lp = counts ? ((double)v - (double)top) * a.inv_t - log_sum : (double)minus_inf();
            if (a.logs && n0 == n) a.logs[at] = (float)lp;
            cls[e * 32 + lane] = counts ? i : -1;
            float more = 0;
            if (counts) {
                const Draw d = draw_of(a, lp, a.gains[at], a.old ? a.old[at] : 0.f, a.kl != 0.f ? a.reference[at] : 0.f);
                term += d.term; to_log += d.to_log; size += fabs(d.to_log);
                more = (float)d.to_log;
                ++number;
                atomicOr(&sh.drawn[W > 1 ? i / E : 0][lane], 1u << (i % E));
            }
            extra[e * 32 + lane] = more;
        }
        sh.sums[0][warp][lane] = term; sh.sums[1][warp][lane] = to_log; sh.sums[2][warp][lane] = size; sh.number[warp][lane] = number;
    }
    meet<W>();
    if (warp == 0) {
        double term = 0, to_log = 0, size = 0;
        int number = 0;
        for (int v = 0; v < busy; ++v) { term += sh.sums[0][v][lane]; to_log += sh.sums[1][v][lane]; size += sh.sums[2][v][lane]; number += sh.number[v][lane]; }
        double by;
        sh.row[lane] = factors_of(a, n, a.weights ? a.weights[n] : 1.f, top, s, sd, log_sum, term, to_log, size, number, n0 == n, by);
        sh.by[lane] = by;
    }
    if (a.gives == GIVES_LOSS) return;
    meet<W>();
    const FeedbackRow r = sh.row[lane];
    float mg = 0, mh = 0;
    auto seen = [&](float2 gh) { mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y); };
    if (n0 == n) {
        const unsigned drawn = sh.drawn[warp][lane];
        const long long at = n * a.out.row + k0 * a.out.cls;
        const int step = (int)a.out.cls;
        if (a.gives == GIVES_PAIRS) {
            float2 *to = static_cast<float2 *>(a.out.data) + at;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (j < here && !(drawn >> j & 1)) {
                    const float2 gh = feedback_gh(r, x[j], 0.f);
                    to[(long long)j * step] = gh;
                    if (a.maxbits) seen(gh);
                }
        } else {
            T *to = static_cast<T *>(a.out.data) + at;
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (j < here && !(drawn >> j & 1)) to[(long long)j * step] = score_from<T>(feedback_gh(r, x[j], 0.f).x);
        }
        for (int e = warp; e < a.draws; e += W) {   // of draws of one class the first writes, for all
            const int i = cls[e * 32 + lane];
            if (i < 0) continue;
            double more = 0;
            bool first = true;
            for (int o = 0; o < a.draws; ++o)
                if (cls[o * 32 + lane] == i) {
                    if (o < e) { first = false; break; }
                    more += (double)extra[o * 32 + lane];
                }
            if (!first) continue;
            const float2 gh = feedback_gh(r, in(n, i), (float)(more * sh.by[lane]));
            put_gradient<T>(a, n, i, gh);
            seen(gh);
        }
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

// By row, 33 to 1024 classes: a warp has a row, E classes in each lane, 32 apart.
template <typename T, int E>
__global__ void __launch_bounds__(ROW_THREADS) k_feedback_row(FeedbackArgs a, Scores<T> in) {
    extern __shared__ __align__(16) unsigned char room[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *cls = reinterpret_cast<int *>(room) + warp * 2 * a.draws;
    float *extra = reinterpret_cast<float *>(cls + a.draws);
    const long long n = blockIdx.x * (long long)ROW_WARPS + warp;
    float mg = 0, mh = 0;
    if (n < a.n) {
        float x[E];
        const T *from = in.at(n, lane);
        T raw[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (lane + 32 * j < a.k) raw[j] = from[32 * j * in.cls];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = lane + 32 * j < a.k ? score_f32(raw[j]) : minus_inf();
        float top = minus_inf();
#pragma unroll
        for (int j = 0; j < E; ++j) top = fmaxf(top, x[j]);
        top = row_top(warp_max(top));
        float s = 0, sd = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float d = __fsub_rn(x[j], top), e = exp2_fast(d * a.c);
            s += e;
            sd = __fmaf_rn(e, fmaxf(d, -1e30f), sd);
        }
        s = warp_sum(s); sd = warp_sum(sd);
        const FeedbackRow r = feedback_row(a, n, top, s, sd, cls, extra, true, read_draws(a, in, n));
        if (a.gives != GIVES_LOSS) {
            unsigned drawn = 0;
            for (int e = 0; e < a.draws; ++e) {
                const int i = cls[e];
                if (i >= 0 && (i & 31) == lane) drawn |= 1u << (i >> 5);
            }
            auto put = [&](int i, float v, float more) {
                const float2 gh = feedback_gh(r, v, more);
                put_gradient<T>(a, n, i, gh);
                mg = fmaxf(mg, fabsf(gh.x)); mh = fmaxf(mh, gh.y);
            };
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (lane + 32 * j < a.k && !(drawn >> j & 1)) put(lane + 32 * j, x[j], 0.f);
            for (int e = lane; e < a.draws; e += 32)
                if (cls[e] >= 0) put(cls[e], in(n, cls[e]), extra[e]);
        }
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

// Long rows: a cluster of up to 8 blocks (or one) holds the row in registers.  Two exponentials per score and gradient; a thread that has no
// score of -inf needs no care for 0 times infinity.
template <int TH> struct FeedbackShared {
    float parts[3][TH / 32], moments[3];
    int cls[SCORES_MAX_TOP];
    float extra[SCORES_MAX_TOP];
    FeedbackRow row;
    DrawsRead ahead[32];   // (kept here: the registers are the row's)
};
// sums of exp((v - base) / T) and of that times (v - base), the second if asked for
template <int V, bool MASKED>
__device__ __forceinline__ void add_exps(const float (&v)[V], float base, float c, bool spread, float2 &s, float2 &sd) {
    if constexpr (V == 1) {
        const float d = __fsub_rn(v[0], base), e = exp2_fast(d * c);
        s.x += e;
        sd.x = __fmaf_rn(e, MASKED ? fmaxf(d, -1e30f) : d, sd.x);
    } else {
        const float2 mb = make_float2(-base, -base), c2 = make_float2(c, c);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            float2 d = add2(make_float2(v[i], v[i + 1]), mb);
            const float2 y = mul2(d, c2), e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
            s = add2(s, e);
            if (spread) sd = fma2(e, MASKED ? make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)) : d, sd);
        }
    }
}
template <int V, bool MASKED> __device__ __forceinline__ void gradients(const FeedbackRow &r, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = feedback_gh(r, v[0], 0.f).x;
    } else {
        const float2 mb = make_float2(-r.top, -r.top), c2 = make_float2(r.c, r.c), p2 = make_float2(r.to_p, r.to_p);
        const float2 by = make_float2(r.by_d, r.by_d), flat = make_float2(r.flat, r.flat);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 d = add2(make_float2(v[i], v[i + 1]), mb), y = mul2(d, c2);
            const float2 p = mul2(make_float2(exp2_fast(y.x), exp2_fast(y.y)), p2);
            const float2 g = mul2(p, fma2(by, MASKED ? make_float2(fmaxf(d.x, -1e30f), fmaxf(d.y, -1e30f)) : d, flat));
            v[i] = g.x; v[i + 1] = g.y;
        }
    }
}
template <typename T, int TH, int P, bool EVEN, bool FULL>
__device__ __forceinline__ void feedback_long(const FeedbackArgs &a, const Scores<T> &in, FeedbackShared<TH> &sh) {
    typedef Hold<T, TH, P, EVEN> H;
    constexpr int V = H::V, W = TH / 32;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long n = blockIdx.x / C;
    const int lo = rank * H::CELLS, cells = FULL ? H::CELLS : min(a.k - lo, H::CELLS);
    H x;
    x.read(in.at(n, lo), cells);
    if (warp == 0) sh.ahead[lane] = read_draws(a, in, n);
    float least, m;
    x.range(cells, least, m);
    const bool masked = least == minus_inf();
    m = warp_max(m);
    if (lane == 0) sh.parts[0][warp] = m;
    __syncthreads();
    m = lanes_max<W>(sh.parts[0][lane & (W - 1)]);
    const bool spread = a.entropy != 0.f;
    float s, sd;
    {
        const float base = row_top(m);
        float2 s2 = make_float2(0.f, 0.f), sd2 = s2;
        auto pass = [&](auto care) {
#pragma unroll
            for (int u = 0; u < P; ++u)
                if (FULL || H::first(u) < cells) {
                    float v[V];
                    x.get(u, v);
                    add_exps<V, decltype(care)::value>(v, base, a.c, spread, s2, sd2);
                }
        };
        masked ? pass(std::true_type{}) : pass(std::false_type{});
        s = s2.x + s2.y; sd = sd2.x + sd2.y;
    }
    s = warp_sum(s); sd = warp_sum(sd);
    if (lane == 0) { sh.parts[1][warp] = s; sh.parts[2][warp] = sd; }
    __syncthreads();
    if (warp == 0) {
        s = lanes_sum<W>(sh.parts[1][lane & (W - 1)]); sd = lanes_sum<W>(sh.parts[2][lane & (W - 1)]);
        if (C > 1 && lane == 0) { sh.moments[0] = m; sh.moments[1] = s; sh.moments[2] = sd; }
    }
    if (C > 1) cluster.sync();
    if (warp == 0) {
        if (C > 1) {
            const float *o = cluster.map_shared_rank(sh.moments, lane < C ? lane : 0);
            const float its = o[0], base = row_top(its);
            s = o[1]; sd = o[2];
            m = lanes_max<32>(its);
            const float low = __fsub_rn(base, row_top(m)), by = its == minus_inf() ? 0.f : exp2_fast(low * a.c);
            sd = lane < C && its > minus_inf() ? __fmaf_rn(low, s, sd) * by : 0.f;
            s = lane < C ? s * by : 0.f;
            s = warp_sum(s); sd = warp_sum(sd);   // (all lanes go on)
        }
        const FeedbackRow r = feedback_row(a, n, row_top(m), s, sd, sh.cls, sh.extra, rank == 0, sh.ahead[lane]);
        if (lane == 0) sh.row = r;
    }
    __syncthreads();
    if (C > 1) cluster_done();
    if (a.gives != GIVES_LOSS) {
        const FeedbackRow r = sh.row;
        const long long at = n * a.out.row + lo;
        if (a.gives == GIVES_PAIRS) {
            float2 *to = static_cast<float2 *>(a.out.data) + at;
#pragma unroll
            for (int u = 0; u < P; ++u)
                if (FULL || H::first(u) < cells) {
                    float v[V];
                    x.get(u, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) to[H::first(u) + i] = feedback_gh(r, v[i], 0.f);
                }
        } else {
            T *to = static_cast<T *>(a.out.data) + at;
            auto pass = [&](auto care) {
#pragma unroll
                for (int u = 0; u < P; ++u)
                    if (FULL || H::first(u) < cells) {
                        float v[V];
                        x.get(u, v);
                        gradients<V, decltype(care)::value>(r, v);
                        x.template set_some<V>(u, 0, v);
                        x.write(to, u);
                    }
            };
            if (!r.counts) {
#pragma unroll
                for (int u = 0; u < P; ++u)
                    if (FULL || H::first(u) < cells) {
                        const float zero[V] = {};
                        x.template set_some<V>(u, 0, zero);
                        x.write(to, u);
                    }
            } else {
                masked ? pass(std::true_type{}) : pass(std::false_type{});
            }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < a.draws; e += TH) {
            const int i = sh.cls[e];
            if (i >= lo && i < lo + cells) put_gradient<T>(a, n, i, feedback_gh(r, in(n, i), sh.extra[e]));
        }
    }
    if (C > 1) cluster_wait();   // (no block leaves while another may still read its sums)
}
template <typename T, int TH, int P, bool EVEN>
__global__ void __launch_bounds__(TH, 1024 / TH) k_feedback_long(FeedbackArgs a, Scores<T> in) {
    __shared__ FeedbackShared<TH> sh;
    if (a.k == (int)cg::this_cluster().num_blocks() * Hold<T, TH, P, EVEN>::CELLS) feedback_long<T, TH, P, EVEN, true>(a, in, sh);
    else feedback_long<T, TH, P, EVEN, false>(a, in, sh);
}
}  // namespace

// f(E, W) for kernels with a lane per row: E classes of each of W warps
template <typename F> void by_class_sizes(int k, F &&f) {
    using std::integral_constant;
    if (k <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (k <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (k <= 32) f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (k <= 64) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (k <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (k <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
}

void scores_sample(const SampleArgs &a, cudaStream_t stream) {
    if (a.n == 0) return;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        const bool by_class = a.in.row < a.in.cls || a.in.one_by_class;
        const bool limited = a.temperatures || a.top_ks || a.top_ps || a.min_ps || a.temperature == 0.f || (a.top_k > 0 && a.top_k < a.k) || a.top_p < 1.f || a.min_p > 0.f;
        const auto blocks = [&](int rows) { return (unsigned)(((long long)a.n + rows - 1) / rows); };
        if (a.k <= 512 && !limited && (by_class || a.k <= 32)) {
            by_class_sizes(a.k, [&](auto e, auto w) {
                constexpr int E = decltype(e)::value, W = decltype(w)::value;
                k_sample_class<T, E, W><<<blocks(W == 1 ? 128 : 32), W == 1 ? 128 : 32 * W, 0, stream>>>(a, scores_of<T>(a.in));
            });
            return;
        }
        if (a.k <= SCORES_CLASS_MOST && (by_class || a.k <= 32 || a.n >= 1024)) {
            const int apart = by_class ? 32 : 33;
            auto go = [&](auto kern, int groups, size_t own, int threads) {
                const size_t smem = groups * (own + sizeof(float) * apart * a.k);
                allow_shared(kern, groups == 1 ? own + sizeof(float) * 33 * SCORES_CLASS_MOST : 4 * (own + sizeof(float) * 33 * 32));
                kern<<<blocks(32 * groups), threads, smem, stream>>>(a, scores_of<T>(a.in), apart);
            };
            if (a.k <= 32) go(k_sample_limited<T, 1>, 4, sizeof(ClassShared<1>) + sizeof(ListShared<1>), 128);
            else go(k_sample_limited<T, 8>, 1, sizeof(ClassShared<8>) + sizeof(ListShared<8>), 256);
            return;
        }
        if (a.in.cls == 1 || a.k == 1) {
            const Scores<T> in = scores_of<T>(a.in);
            const bool even = a.k % Pack<T>::V == 0 && on_16(in.p, in.row, sizeof(T));
            bool done = false;
            // the smallest blocks that hold a row in a cluster of up to 8, and bigger ones before more than one where there are rows enough for every SM
            auto go = [&](auto th, auto p, auto ev) {
                constexpr bool EVEN = decltype(ev)::value;
                constexpr int TH = decltype(th)::value, P = decltype(p)::value;
                const int c = (a.k + Hold<T, TH, P, EVEN>::CELLS - 1) / Hold<T, TH, P, EVEN>::CELLS;
                if (done || c > LONG_CLUSTER) return;
                launch_long(k_sample_long<T, TH, P, EVEN>, a.n, c, TH, stream, 0, a, in);
                done = true;
            };
            using std::integral_constant;
            auto all = [&](auto ev) {
                constexpr int S = decltype(ev)::value ? sizeof(T) == 2 ? 1 : 2 : 8;   // 8 scores
                if (a.k <= 2048) go(integral_constant<int, 256>{}, integral_constant<int, S>{}, ev);
                go(integral_constant<int, 512>{}, integral_constant<int, S>{}, ev);
                go(integral_constant<int, 512>{}, integral_constant<int, 2 * S>{}, ev);
                go(integral_constant<int, 512>{}, integral_constant<int, 4 * S>{}, ev);
            };
            even ? all(std::true_type{}) : all(std::false_type{});
            if (done) return;
        }
        k_sample_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, scores_of<T>(a.in));
    });
    TGBM_CUDA(cudaGetLastError());
}

void scores_feedback(const FeedbackArgs &given, cudaStream_t stream) {
    if (given.n == 0) return;
    FeedbackArgs a = given;
    a.inv_t = 1.0 / (double)a.temperature;
    a.c = (float)(1.44269504088896341 * a.inv_t);
    a.least = (float)(1.0 - (double)a.clip_low);
    a.most = (float)(1.0 + (double)a.clip_high);
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        const Scores<T> in = scores_of<T>(a.in);
        const bool by_class = a.in.row < a.in.cls || a.in.one_by_class;
        if ((a.k <= 32 || (by_class && a.k <= SCORES_CLASS_MOST)) && std::max(a.in.cls, a.out.cls) <= INT_MAX) {
            auto go = [&](auto e, auto w) {
                constexpr int E = decltype(e)::value, W = decltype(w)::value;
                constexpr int G = W == 1 ? 4 : 1;
                auto kern = k_feedback_class<T, E, W>;
                // (beside the lists: 24 + 16 + 4 + 4 bytes of every warp's lanes, a row's factors)
                constexpr size_t own = G * 32 * (48 * (size_t)W + sizeof(FeedbackRow) + 8) + 64 * G;
                if (own + G * 256 * a.draws > 48 * 1024) allow_shared(kern, own + G * 256 * (size_t)SCORES_MAX_TOP);
                kern<<<(unsigned)((a.n + 32ll * G - 1) / (32 * G)), W == 1 ? 128 : 32 * W, own + G * 256 * a.draws, stream>>>(a, in);
            };
            using std::integral_constant;
            if (a.k > 512) go(integral_constant<int, 32>{}, integral_constant<int, 32>{});
            else by_class_sizes(a.k, go);
            return;
        }
        if (a.k <= 1024) {
            const unsigned blocks = (unsigned)(((long long)a.n + ROW_WARPS - 1) / ROW_WARPS);
            const size_t smem = 8 * (size_t)ROW_WARPS * a.draws;
            if (a.k <= 64) k_feedback_row<T, 2><<<blocks, ROW_THREADS, smem, stream>>>(a, in);
            else if (a.k <= 128) k_feedback_row<T, 4><<<blocks, ROW_THREADS, smem, stream>>>(a, in);
            else if (a.k <= 256) k_feedback_row<T, 8><<<blocks, ROW_THREADS, smem, stream>>>(a, in);
            else if (a.k <= 512) k_feedback_row<T, 16><<<blocks, ROW_THREADS, smem, stream>>>(a, in);
            else k_feedback_row<T, 32><<<blocks, ROW_THREADS, smem, stream>>>(a, in);
            return;
        }
        if (a.in.cls == 1 && (a.gives == GIVES_LOSS || a.out.cls == 1) && !a.maxbits) {
            const bool even = a.k % Pack<T>::V == 0 && on_16(in.p, in.row, sizeof(T)) && (a.gives != GIVES_GRADIENT || on_16(a.out.data, a.out.row, sizeof(T)));
            bool done = false;
            // the smallest blocks that hold a row in a cluster of up to 8, the largest ones where there are rows for several on every SM
            auto go = [&](auto th, auto p, auto last, auto ev) {
                constexpr bool EVEN = decltype(ev)::value;
                constexpr int TH = decltype(th)::value, P = decltype(p)::value;
                const int c = (a.k + Hold<T, TH, P, EVEN>::CELLS - 1) / Hold<T, TH, P, EVEN>::CELLS;
                if (done || c > LONG_CLUSTER || (!decltype(last)::value && c > 1 && (long long)a.n * c > 8 * 148)) return;
                launch_long(k_feedback_long<T, TH, P, EVEN>, a.n, c, TH, stream, 0, a, in);
                done = true;
            };
            using std::integral_constant;
            auto all = [&](auto ev) {
                constexpr bool EVEN = decltype(ev)::value;
                constexpr int S = EVEN ? sizeof(T) == 2 ? 1 : 2 : 8;   // 8 scores
                go(integral_constant<int, 256>{}, integral_constant<int, S>{}, std::false_type{}, ev);
                go(integral_constant<int, 256>{}, integral_constant<int, 2 * S>{}, std::false_type{}, ev);
                constexpr bool more = EVEN && sizeof(T) == 2;
                go(integral_constant<int, 256>{}, integral_constant<int, 4 * S>{}, integral_constant<bool, !more>{}, ev);
                go(integral_constant<int, more ? 256 : 512>{}, integral_constant<int, more ? 8 * S : 4 * S>{}, std::true_type{}, ev);
            };
            even ? all(std::true_type{}) : all(std::false_type{});
            if (done) return;
        }
        k_feedback_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, scores_of<T>(a.in));
    });
    TGBM_CUDA(cudaGetLastError());
}

}  // namespace tgbm

// ------------------------------------------------------------------ C entries
using namespace tgbm;

extern "C" {

int tgbm_scores_sample(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int draws,
                       int uniform_type, const void *d_uniform, float temperature, const float *d_temperature, int top_k, const int *d_top_k,
                       float top_p, const float *d_top_p, float min_p, const float *d_min_p, int *d_classes, float *d_logs, float *d_all_logs,
                       void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        check_draws(draws);
        TGBM_CHECK(uniform_type == TGBM_F32 || uniform_type == TGBM_F64, "random numbers: floats or doubles");
        check_limits(d_temperature ? 1.f : temperature, d_top_k ? 0 : top_k, d_top_p ? 1.f : top_p, d_min_p ? 0.f : min_p);   // (numbers of rows stand in for those)
        if (n_rows == 0) return;
        SampleArgs a;
        a.n = n_rows; a.k = n_classes; a.draws = draws;
        a.in = view_of("scores", d_scores, type, n_rows, n_classes, row_stride, class_stride, false);
        TGBM_CHECK(d_uniform && d_classes, "random numbers or classes: null pointer");
        check_pointer("random numbers", d_uniform, uniform_type == TGBM_F64 ? 8 : 4);
        check_pointer("temperatures", d_temperature, 4); check_pointer("top_k", d_top_k, 4); check_pointer("top_p", d_top_p, 4);
        check_pointer("min_p", d_min_p, 4); check_pointer("classes", d_classes, 4); check_pointer("logs", d_logs, 4);
        check_pointer("logs among all", d_all_logs, 4);
        a.uniform = d_uniform; a.uniform_f64 = uniform_type == TGBM_F64;
        a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
        a.temperatures = d_temperature; a.top_ks = d_top_k; a.top_ps = d_top_p; a.min_ps = d_min_p;
        a.classes = d_classes; a.logs = d_logs; a.all_logs = d_all_logs;
        scores_sample(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

int tgbm_scores_feedback(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, int draws,
                         const int *d_classes, const float *d_gains, const float *d_old, const float *d_reference, const float *d_weights,
                         float temperature, float clip_low, float clip_high, float kl, float entropy, float *d_loss, float *d_logs, int gives,
                         void *d_grad, long long grad_row_stride, long long grad_class_stride, void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        check_draws(draws);
        check_temperature(temperature);
        check_feedback(clip_low, clip_high, kl, entropy);
        TGBM_CHECK(kl == 0.f || d_reference || n_rows == 0, "reference: null pointer");
        TGBM_CHECK(gives >= TGBM_GIVES_LOSS && gives <= TGBM_GIVES_PAIRS, "unknown kind of result");
        if (n_rows == 0) return;
        FeedbackArgs a;
        a.n = n_rows; a.k = n_classes; a.draws = draws;
        a.in = view_of("scores", d_scores, type, n_rows, n_classes, row_stride, class_stride, false);
        TGBM_CHECK(d_classes && d_gains, "classes or gains: null pointer");
        check_pointer("classes", d_classes, 4); check_pointer("gains", d_gains, 4); check_pointer("old", d_old, 4);
        check_pointer("reference", d_reference, 4); check_pointer("weights", d_weights, 4); check_pointer("loss", d_loss, 4);
        check_pointer("logs", d_logs, 4);
        a.classes = d_classes; a.gains = d_gains; a.old = d_old; a.reference = d_reference; a.weights = d_weights;
        a.temperature = temperature; a.clip_low = clip_low; a.clip_high = clip_high; a.kl = kl; a.entropy = entropy;
        a.gives = gives; a.loss = d_loss; a.logs = d_logs;
        TGBM_CHECK(d_loss || d_logs || gives != TGBM_GIVES_LOSS, "loss: null pointer");
        if (gives != TGBM_GIVES_LOSS) {
            const bool pairs = gives == TGBM_GIVES_PAIRS;
            TGBM_CHECK(!pairs || reinterpret_cast<uintptr_t>(d_grad) % 8 == 0, "gradient: pairs have to be aligned to 8 bytes");
            a.out = view_of("gradient", d_grad, pairs ? (int)SCORE_F32 : type, n_rows, n_classes, grad_row_stride, grad_class_stride, true);
            TGBM_CHECK(!share_memory(a.in, size_of(type), a.out, pairs ? 8 : size_of(type), n_rows, n_classes), "scores and gradient share memory");
        }
        scores_feedback(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

}  // extern "C"
