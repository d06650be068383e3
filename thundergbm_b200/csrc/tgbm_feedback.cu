// Loss on classes that were drawn from the scores of many classes and on the gains that followed, with its gradient (feedback).
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

template <int W> __device__ __forceinline__ void meet() {   // the warps that share rows
    if (W > 1) __syncthreads();
    else __syncwarp();
}

// A row's sums, with y = (s - top) log2(e) / T and top its largest score: sum of e = 2^y and of e y.  What follows from them and the draws:
//   g_i = p_i (by_y y_i + flat) + [draws of i],  h_i = max(curve p_i (1 - p_i), 1e-16),  p_i = e_i to_p
struct FeedbackRow {
    float top, c, to_p, by_y, flat, curve;
    bool counts;   // without a draw that counts, or with a weight of 0, the row has no loss
};
// e is 0 from -126 on: y stops here, so that e y and p (by_y y + flat) are 0 where a score is -inf, or so low that y is (0 times infinity is none)
constexpr float FAR = -200.f;
constexpr double LN2 = 0.69314718055994530942;

struct Draw {
    double term, to_log;   // loss of one draw, its derivative by the log-probability
};
__device__ __forceinline__ Draw draw_of(const FeedbackArgs &a, double lp, float its_gain, float old, float reference) {
    const double gain = (double)its_gain, r = a.old ? exp(lp - (double)old) : 1.0;
    const double held = fmin(fmax(r, (double)a.least), (double)a.most);
    Draw d;
    d.term = gain == 0 ? 0.0 : -fmin(r * gain, held * gain);   // (what weighs 0 counts for nothing, also where the ratio is infinite)
    d.to_log = gain != 0 && r * gain <= held * gain ? -r * gain : 0.0;
    if (gain != 0 && r * gain != r * gain) d.term = d.to_log = r * gain;   // (NaN: neither bound holds it)
    if (a.kl != 0.f) {
        const double x = (double)reference - lp, e = exp(x);
        d.term += (double)a.kl * (e - x - 1);
        d.to_log += (double)a.kl * (1 - e);
    }
    return d;
}

// The row's loss, and what its gradients need; `by`: what a draw's derivative is multiplied by
__device__ __forceinline__ FeedbackRow factors_of(const FeedbackArgs &a, long long n, float w, float top, float sum, float sum_y, double log_sum, double term,
                                                  double to_log, double size, int number, bool writes, double &by) {
    const double inv_sum = sum == 0.f ? 0.0 : 1.0 / (double)sum, spread = log_sum - (double)sum_y * LN2 * inv_sum;   // (the entropy)
    FeedbackRow r;
    r.counts = number > 0 && w != 0.f;
    const double share = number == 1 ? 1.0 : number ? 1.0 / number : 0.0, scale = (double)w * a.inv_t;
    if (a.loss && writes) a.loss[n] = r.counts ? (float)((double)w * (term * share - (a.entropy != 0.f ? (double)a.entropy * spread : 0.0))) : 0.f;
    r.top = top; r.c = a.c;
    r.to_p = (float)inv_sum;
    r.by_y = (float)(scale * (double)a.entropy * LN2);
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
__device__ __forceinline__ FeedbackRow feedback_row(const FeedbackArgs &a, long long n, float top, float sum, float sum_y, int *cls, float *extra, bool writes,
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
    const FeedbackRow r = factors_of(a, n, draws.weight, top, sum, sum_y, log_sum, term, to_log, size, number, writes && lane == 0, by);
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
__device__ __forceinline__ void add_exp(float x, float top, float c, float &s, float &sy) {
    const float y = __fsub_rn(x, top) * c, e = exp2_fast(y);
    s += e;
    sy = __fmaf_rn(e, fmaxf(y, FAR), sy);
}
__device__ __forceinline__ float2 feedback_gh(const FeedbackRow &r, float s, float extra) {
    if (!r.counts) return make_float2(0.f, MIN_HESSIAN);
    const float y = __fsub_rn(s, r.top) * r.c, p = exp2_fast(y) * r.to_p;
    const float cp = r.curve * p;
    return make_float2(__fmaf_rn(p, __fmaf_rn(r.by_y, fmaxf(y, FAR), r.flat), extra), fmaxf(__fmaf_rn(-cp, p, cp), MIN_HESSIAN));
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
    float s = 0, sy = 0;
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) add_exp(in(n, k), top, a.c, s, sy);
    s = warp_sum(s); sy = warp_sum(sy);
    if (lane == 0) { parts[1][warp] = s; parts[2][warp] = sy; }
    __syncthreads();
    if (warp == 0) {
        s = warp_sum(lane < ROW_WARPS ? parts[1][lane] : 0.f);
        sy = warp_sum(lane < ROW_WARPS ? parts[2][lane] : 0.f);
        const FeedbackRow r = feedback_row(a, n, top, s, sy, cls, extra, true, read_draws(a, in, n));
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
// Four draws of 50003 x 250 with pairs: 57 us (floor 23.4), instructions, 560 a row.
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
    float s = 0, sy = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) add_exp(x[j], top, a.c, s, sy);
    if constexpr (W > 1) {
        sh.part[1][warp][lane] = make_float2(s, sy);
        __syncthreads();
        float2 all = sh.part[1][0][lane];
#pragma unroll
        for (int v = 1; v < W; ++v) all = add2(all, sh.part[1][v][lane]);
        s = all.x; sy = all.y;
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
        sh.row[lane] = factors_of(a, n, a.weights ? a.weights[n] : 1.f, top, s, sy, log_sum, term, to_log, size, number, n0 == n, by);
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
        float s = 0, sy = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) add_exp(x[j], top, a.c, s, sy);
        s = warp_sum(s); sy = warp_sum(sy);
        const FeedbackRow r = feedback_row(a, n, top, s, sy, cls, extra, true, read_draws(a, in, n));
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

// Long rows: a cluster of up to 8 blocks (or one) holds the row in registers.  Two exponentials per score and gradient; a thread whose
// scores are not infinitely far from the largest needs no care for 0 times infinity.  1024 x 131072 in 16 bits: 150 us (floor 82); the rest is waiting, for the cluster and for the
// warp that works out the draws.  Blocks of 512 threads, two per SM, took 255 us, of 256 with twice the scores a thread, four per SM, 158.
template <int TH> struct FeedbackShared {
    float parts[3][TH / 32], moments[3];
    int cls[SCORES_MAX_TOP];
    float extra[SCORES_MAX_TOP];
    FeedbackRow row;
    DrawsRead ahead[32];   // (kept here: the registers are the row's)
};
// sums of e = 2^y, y = (v - base) log2(e) / T, and of e y, the second if asked for.  MASKED: y may be infinite
template <int V, bool MASKED>
__device__ __forceinline__ void add_exps(const float (&v)[V], float base, float c, bool spread, float2 &s, float2 &sy) {
    if constexpr (V == 1) {
        const float y = __fsub_rn(v[0], base) * c, e = exp2_fast(y);
        s.x += e;
        sy.x = __fmaf_rn(e, MASKED ? fmaxf(y, FAR) : y, sy.x);
    } else {
        const float2 mb = make_float2(-base, -base), c2 = make_float2(c, c);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 y = mul2(add2(make_float2(v[i], v[i + 1]), mb), c2), e = make_float2(exp2_fast(y.x), exp2_fast(y.y));
            s = add2(s, e);
            if (spread) sy = fma2(e, MASKED ? make_float2(fmaxf(y.x, FAR), fmaxf(y.y, FAR)) : y, sy);
        }
    }
}
// MASKED: by_y y may be infinite
template <int V, bool MASKED> __device__ __forceinline__ void gradients(const FeedbackRow &r, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = feedback_gh(r, v[0], 0.f).x;
    } else {
        const float2 mb = make_float2(-r.top, -r.top), c2 = make_float2(r.c, r.c), p2 = make_float2(r.to_p, r.to_p);
        const float2 by = make_float2(r.by_y, r.by_y), flat = make_float2(r.flat, r.flat);
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 y = mul2(add2(make_float2(v[i], v[i + 1]), mb), c2);
            const float2 p = mul2(make_float2(exp2_fast(y.x), exp2_fast(y.y)), p2);
            const float2 g = mul2(p, fma2(by, MASKED ? make_float2(fmaxf(y.x, FAR), fmaxf(y.y, FAR)) : y, flat));
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
    m = warp_max(m);
    if (lane == 0) sh.parts[0][warp] = m;
    __syncthreads();
    m = lanes_max<W>(sh.parts[0][lane & (W - 1)]);
    const bool spread = a.entropy != 0.f;
    float s, sy;
    {
        const float base = row_top(m);
        const bool masked = !finite(fminf(__fsub_rn(least, base), 0.f) * a.c);
        float2 s2 = make_float2(0.f, 0.f), sy2 = s2;
        auto pass = [&](auto care) {
#pragma unroll
            for (int u = 0; u < P; ++u)
                if (FULL || H::first(u) < cells) {
                    float v[V];
                    x.get(u, v);
                    add_exps<V, decltype(care)::value>(v, base, a.c, spread, s2, sy2);
                }
        };
        masked ? pass(std::true_type{}) : pass(std::false_type{});
        s = s2.x + s2.y; sy = sy2.x + sy2.y;
    }
    s = warp_sum(s); sy = warp_sum(sy);
    if (lane == 0) { sh.parts[1][warp] = s; sh.parts[2][warp] = sy; }
    __syncthreads();
    if (warp == 0) {
        s = lanes_sum<W>(sh.parts[1][lane & (W - 1)]); sy = lanes_sum<W>(sh.parts[2][lane & (W - 1)]);
        if (C > 1 && lane == 0) { sh.moments[0] = m; sh.moments[1] = s; sh.moments[2] = sy; }
    }
    if (C > 1) cluster.sync();
    if (warp == 0) {
        if (C > 1) {
            const float *o = cluster.map_shared_rank(sh.moments, lane < C ? lane : 0);
            const float its = o[0], base = row_top(its);
            s = o[1]; sy = o[2];
            m = lanes_max<32>(its);
            const float low = __fsub_rn(base, row_top(m)) * a.c, by = its == minus_inf() ? 0.f : exp2_fast(low);
            sy = lane < C && by != 0.f ? __fmaf_rn(low, s, sy) * by : 0.f;   // (a block of classes at the type's lowest number is infinitely far)
            s = lane < C ? s * by : 0.f;
            s = warp_sum(s); sy = warp_sum(sy);   // (all lanes go on)
        }
        const FeedbackRow r = feedback_row(a, n, row_top(m), s, sy, sh.cls, sh.extra, rank == 0, sh.ahead[lane]);
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
                const bool masked = !finite(fminf(__fsub_rn(least, r.top), 0.f) * r.c * r.by_y);
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
            by_class_sizes(a.k, go);
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
            // the smallest blocks that hold a row in a cluster of up to 8, the largest ones where there are rows for several on every SM: 16 bits, the largest
            // and the smallest (us): 1200 x 20000 44 and 64, 1200 x 60000 87 and 119, 300 x 60000 27 and 32; 148 x 60000 18 and 19, fewer rows 17 either way (the call)
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
