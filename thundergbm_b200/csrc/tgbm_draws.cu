// Classes drawn from the scores of many classes (sample), and the loss on drawn classes with its gradient (feedback).
//
// sample decides which class a random number falls on by sums of exponentials next to one another, and a row may have 2^20
// of them: exponentials and their sums are doubles, so that the classes are those of the definition.
#include <cfloat>
#include <climits>
#include <cmath>

#include "../../include/thundergbm.h"
#include "tgbm_scores.cuh"
#include "tgbm_scores_check.h"

namespace tgbm {
namespace {

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
__device__ __forceinline__ Draw draw_of(const FeedbackArgs &a, long long at, double lp) {
    const double gain = (double)a.gains[at], r = a.old ? exp(lp - (double)a.old[at]) : 1.0;
    const double held = fmin(fmax(r, (double)a.least), (double)a.most);
    Draw d;
    d.term = gain == 0 ? 0.0 : -fmin(r * gain, held * gain);   // (what weighs 0 counts for nothing, also where the ratio is infinite)
    d.to_log = gain != 0 && r * gain <= held * gain ? -r * gain : 0.0;
    if (a.kl != 0.f) {
        const double x = (double)a.reference[at] - lp, e = exp(x);
        d.term += (double)a.kl * (e - x - 1);
        d.to_log += (double)a.kl * (1 - e);
    }
    return d;
}

// One warp, for the row n: logs, the loss and what its gradients need.  cls[e], extra[e]: class of draw e and what is added there (-1: nothing;
// of draws of one class the first has the sum).  score(i): the row's score of class i.
template <typename F>
__device__ __forceinline__ FeedbackRow feedback_row(const FeedbackArgs &a, long long n, float top, float sum, float sum_d, int *cls, float *extra, F &&score) {
    const int lane = threadIdx.x & 31;
    const double log_sum = sum == 0.f ? 0.0 : fine_log(sum), spread = sum == 0.f ? 0.0 : log_sum - (double)sum_d * a.inv_t / (double)sum;   // (the entropy)
    const float w = a.weights ? a.weights[n] : 1.f;
    double term = 0, to_log = 0, size = 0;
    int number = 0;
    for (int e = lane; e < a.draws; e += 32) {
        const long long at = n * a.draws + e;
        const int i = a.classes[at];
        const float x = i >= 0 && i < a.k ? score(i) : minus_inf();
        const bool counts = x > minus_inf() || x != x;
        const double lp = counts ? ((double)x - (double)top) * a.inv_t - log_sum : (double)minus_inf();
        if (a.logs) a.logs[at] = (float)lp;
        cls[e] = counts ? i : -1;
        extra[e] = 0.f;
        if (counts) {
            const Draw d = draw_of(a, at, lp);
            term += d.term; to_log += d.to_log; size += fabs(d.to_log);
            extra[e] = (float)d.to_log;
            ++number;
        }
    }
    number = warp_sum(number);
    term = warp_sum(term); to_log = warp_sum(to_log); size = warp_sum(size);
    __syncwarp();
    FeedbackRow r;
    r.counts = number > 0 && w != 0.f;
    const double share = number ? 1.0 / number : 0.0, by = (double)w * a.inv_t;
    if (a.loss && lane == 0) a.loss[n] = r.counts ? (float)((double)w * (term * share - (a.entropy != 0.f ? (double)a.entropy * spread : 0.0))) : 0.f;
    r.top = top; r.c = a.c;
    r.to_p = sum == 0.f ? 0.f : 1.f / sum;
    r.by_d = (float)(by * (double)a.entropy * a.inv_t);
    r.flat = (float)(by * ((a.entropy != 0.f ? (double)a.entropy * (spread - log_sum) : 0.0) - to_log * share));
    r.curve = (float)(2 * by * a.inv_t * (size * share + (double)a.entropy));
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
            total[j] = (float)(s * by * share);
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
        const FeedbackRow r = feedback_row(a, n, top, s, sd, cls, extra, [&](int i) { return in(n, i); });
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
}  // namespace

void scores_sample(const SampleArgs &a, cudaStream_t stream) {
    if (a.n == 0) return;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
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
        TGBM_CHECK(d_temperature || (temperature >= 0.f && temperature <= FLT_MAX), "the temperature has to be a number from 0 on");
        TGBM_CHECK(d_top_k || top_k >= 0, "top_k: negative");
        TGBM_CHECK(d_top_p || (top_p >= 0.f && top_p <= 1.f), "top_p outside [0, 1]");
        TGBM_CHECK(d_min_p || (min_p >= 0.f && min_p <= 1.f), "min_p outside [0, 1]");
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
