// Classes drawn from the scores of many classes (sample), one for each of a row's random numbers.
#include <cfloat>
#include <climits>
#include <cmath>

#include "../../include/thundergbm.h"
#include "tgbm_sample.cuh"
#include "tgbm_scores_check.h"

namespace tgbm {
namespace {

constexpr int ROW_THREADS = 256, ROW_WARPS = ROW_THREADS / 32;

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

// What no other kernel takes (strides, more than 1024 classes by class, more than clusters hold).  A row, any strides: a block reads it again for everything that it wants to know.  Classes that may be drawn are those whose entry
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

// ---- up to 1024 classes: a lane has a row, the W warps of a block (W = 1: each for itself) share its classes, E neighbours each ------
// What a warp's lanes know of their rows is put together through shared memory; all warps come to the same numbers in the same order,
// and so decide alike.
//
// Limits: which scores a row's draws are left to is settled by a list of the few that can be among them, in class order, in shared memory: a lane
// walks its row's list there, without a barrier, as often as it takes.  Scores that can be are those from a border on: min_p gives one, and so does
// top_p (classes with less than (1 - top_p) / classes of the mass each have less than 1 - top_p of it together); where more than LIST reach it, it is
// raised by bisection over all scores as long as enough reach it.  Rows with more all the same (limits that leave that many, ties)
// are settled by bisection over all scores, by floats as far as they tell: 20000 x 1000, top_p 0.9 of a normal distribution, 1157 us, 3146 by doubles from
// the start.
// A longer list takes more rows, and leaves room for fewer blocks on an SM: with 56 entries three tiles of up to 250 classes share it.  Lists of 40, 56
// and 80 entries (us): 50003 x 250 with some 40 likely classes, top_p 0.9: 130, 95, 126; min_p 0.02 beside it: 77, 77, 98; 50003 x 250 of a normal
// distribution, top_k 50: 171, 190, 243; 20000 x 500, 100 likely classes, top_k 20: 152, 146, 217; 20000 x 1000 of a normal distribution, top_k 50,
// where one block has an SM in any case: 546, 526, 446.
constexpr int LIST = 56;
template <int W> struct ClassShared {
    Powers powers;
    double sums[2][W][32];
    float lows[2][W][32], highs[2][W][32], counts[2][W][32];
    double front[W][32];
    int cls[W][32];
    float score[W][32];
};
template <int MOST_> struct ListShared {
    static constexpr int MOST = MOST_;
    static constexpr int APART = 36;   // (entries i, i + 1, ... of four rows lie in different banks)
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

// Nothing is cut off: exponentials stay in registers.  Bound by the call and by instructions: 581012 x 7 in 17.1 us (floor 4.3).
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

// With limits: the scores lie in shared memory (row r and class k at k * apart + r), which leaves the registers to what is found out of them.  Bound by
// instructions, 1040 a row of 250 classes, 240 of them for the mass of all classes in doubles: 50003 x 250 with min_p and top_p in 98 us (floor 7.8).
// Bisection over all scores of a tile took 179 us, lists that one warp settles for all 32 rows 252, eight lanes a row, by all warps, 135.  With floats for the
// mass where it is only told it was 83 us, but its log had no digits near 0 and could lie above that among the classes left.
template <typename T, int W, int MOST>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 1 ? 4 : 3) k_sample_limited(SampleArgs a, Scores<T> in, int apart) {
    extern __shared__ __align__(16) unsigned char room[];
    const int lane = threadIdx.x & 31, group = W == 1 ? threadIdx.x >> 5 : 0, warp = W == 1 ? 0 : threadIdx.x >> 5;
    ClassShared<W> &sh = reinterpret_cast<ClassShared<W> *>(room)[group];   // (W = 1: each warp has its own)
    constexpr int G = W == 1 ? 4 : 1;
    ListShared<MOST> &list = reinterpret_cast<ListShared<MOST> *>(room + G * sizeof(ClassShared<W>))[group];
    float *tile = reinterpret_cast<float *>(room + G * (sizeof(ClassShared<W>) + sizeof(ListShared<MOST>))) + group * (size_t)apart * a.k;
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
    if (W == 1) __syncwarp();   // (W > 1: the first exchange is a barrier)
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
    // The whole mass, a sum of doubles, and the scores from a border on that all that is left reaches.  The border is rounded down by more than its floats
    // can be off: 2^-19 of its distance from the largest score (logf: 2^-23, products 2^-24 each), of T (the share under the logarithm is
    // rounded) and of that score.  Where it is a share of the whole mass, that comes first.
    float low = minus_inf(), high = top;
    auto border = [&] {
        const float t = (float)(1.0 / l.inv_t);
        float down = -FLT_MAX;
        if (l.greedy) down = 0.f;
        else if (by_share) down = logf((float)l.min_p) * t;
        else if (by_mass && !by_count) down = logf((float)((1 - l.top_p) * all / a.k)) * t;
        low = l.greedy ? top : __fadd_rn(top, down) - ((fabsf(down) + t + fabsf(top)) * 2e-6f + 1e-44f);   // (1e-44: products below 2^-126)
        if (!(low <= top)) low = down == -FLT_MAX ? minus_inf() : top;
    };
    int own = 0;
    double sum = 0;
    least = -minus_inf();
    auto look = [&](float x) {
        if (live && x >= low && x > minus_inf()) { ++own; least = fminf(least, x); }
    };
    const bool share_of_mass = __any_sync(0xffffffffu, by_mass && !by_count && !by_share);
    if (share_of_mass) {
        each_score([&](float x, int) { all += live ? weight_of(x) : 0.0; });
        float none = 0, none_high = 0;
        count = 0;
        over.all(all, none, none_high, count);
        border();
        each_score([&](float x, int) { look(x); });
    } else {
        border();
        each_score([&](float x, int) {
            all += live ? weight_of(x) : 0.0;
            look(x);
        });
        sum = all;
    }
    count = (float)own;
    const int counted = over.turn;
    over.all(sum, least, high, count);
    if (!share_of_mass) all = sum;
    if (l.greedy) all = 1.0;
    low = least;
    high = top;
    bool again = false;   // what was counted above is not what the list takes
    bool narrowing = limited && count > (float)MOST && (by_count ? top_k <= MOST : by_mass && !by_share);   // (of what min_p leaves the whole mass is needed)
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
            narrowing = count > (float)MOST && low < high && (low == up || reach < (float)MOST);   // (too few reach it, and more than the list has room for)
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
            // by floats first, as far as they tell on which side the border lies: a warp adds up to 128 in a chain (127 roundings of 2^-24), each off by
            // 2^-22 and by 3 roundings of its exponent, which is below 10 on the mean over the mass of 1024: 9.1e-6 in all
            float up_to = top;
            const float c = (float)(l.inv_t * 1.4426950408889634);
            bool told = part && floats_tell(l);
            while (__any_sync(0xffffffffu, told && lowest < up_to)) {
                const float mid = middle(lowest, up_to);
                float mass = 0, up = -minus_inf(), below = minus_inf(), none = 0;
                each_score([&](float x, int) {
                    if (x >= mid) { mass += exp2_fast(__fsub_rn(x, top) * c); up = fminf(up, x); }
                    else if (x > minus_inf()) below = fmaxf(below, x);
                });
                double s = (double)mass;
                over.all(s, up, below, none);
                if (told && lowest < up_to) {
                    if (s >= target * (1 + 2e-5)) lowest = up;
                    else if (s < target * (1 - 2e-5)) up_to = below;
                    else told = false;
                }
            }
            const float at = reached(part, target, lowest, up_to, each(true), together);
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
}  // namespace

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
                if constexpr (W <= 16) k_sample_class<T, E, W><<<blocks(W == 1 ? 128 : 32), W == 1 ? 128 : 32 * W, 0, stream>>>(a, scores_of<T>(a.in));
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
            // (a list for all classes where a warp has them: small ones, so that more blocks share an SM)
            if (a.k <= 8) go(k_sample_limited<T, 1, 8>, 4, sizeof(ClassShared<1>) + sizeof(ListShared<8>), 128);
            else if (a.k <= 32) go(k_sample_limited<T, 1, 32>, 4, sizeof(ClassShared<1>) + sizeof(ListShared<32>), 128);
            else go(k_sample_limited<T, 8, LIST>, 1, sizeof(ClassShared<8>) + sizeof(ListShared<LIST>), 256);
            return;
        }
        if ((a.in.cls == 1 || a.k == 1) && sample_long<T>(a, stream)) return;
        k_sample_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, scores_of<T>(a.in));
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

}  // extern "C"
