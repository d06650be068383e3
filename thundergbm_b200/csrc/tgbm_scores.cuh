// Device code of the operators on scores (tgbm_scores.cu): element types, reductions, the teacher's side of a row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "tgbm_device.cuh"
#include "tgbm_scores.h"

namespace tgbm {

__device__ __forceinline__ float score_f32(float v) { return v; }
__device__ __forceinline__ float score_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float score_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T score_from(float v);
template <> __device__ __forceinline__ float score_from<float>(float v) { return v; }
template <> __device__ __forceinline__ __half score_from<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 score_from<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T> struct Scores {
    T *p;
    long long row, cls;
    __device__ __forceinline__ T *at(long long n, long long k) const { return p + n * row + k * cls; }
    __device__ __forceinline__ float operator()(long long n, long long k) const { return score_f32(*at(n, k)); }
};
template <typename T> Scores<T> scores_of(const ScoreView &v) { return Scores<T>{static_cast<T *>(v.data), v.row, v.cls}; }

// f<T>() for the element type
template <typename F> inline void by_type(int type, F &&f) {
    switch (type) {
    case SCORE_F32: f(float{}); break;
    case SCORE_F16: f(__half{}); break;
    case SCORE_BF16: f(__nv_bfloat16{}); break;
    default: throw Error("unknown type of scores");
    }
}

constexpr float LOG2E = 1.44269504088896341f;
__device__ __forceinline__ float minus_inf() { return __int_as_float(0xff800000); }

// 2^x, one instruction; 0 for -inf, flushes results below 2^-126 (a class that far below the row's best adds nothing to a
// float sum that holds a 1)
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// log of a float sum to about 2^-25, absolutely (logf is off by half a step of its result, which for a sum of many terms is
// several times that): the exponent is exact, the rest lies in [sqrt(1/2), sqrt(2))
__device__ __forceinline__ double fine_log(float x) {
    if (!(x >= 1.17549435e-38f && x <= 3.40282347e38f)) return (double)logf(x);
    const int b = __float_as_int(x), e = (b - 0x3f3504f3) >> 23;
    return (double)e * 0.6931471805599453 + (double)logf(__int_as_float(b - (e << 23)));
}

// exp((x - ref) / T) to a few steps of the result wherever it lies: what x - ref and the product with 1 / T lose is put back.
// c + c_low = log2(e) / T.
__device__ __forceinline__ float fine_exp(float x, float ref, float c, float c_low) {
    const float d = __fsub_rn(x, ref);
    const float b = __fsub_rn(d, x);
    const float lost = __fsub_rn(__fsub_rn(x, __fsub_rn(d, b)), __fadd_rn(ref, b));
    const float y = __fmul_rn(d, c);
    const float low = __fmaf_rn(d, c, -y) + (d * c_low + lost * c);
    return fabsf(low) < 1.f ? __fmaf_rn(exp2f(y), low * 0.693147181f, exp2f(y)) : exp2f(y);   // (not for infinities)
}

// 1 / x to one step, for normal x
__device__ __forceinline__ float fast_inverse(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// two floats in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long r, x = *reinterpret_cast<unsigned long long *>(&a), y = *reinterpret_cast<unsigned long long *>(&b);
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return *reinterpret_cast<float2 *>(&r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    unsigned long long r, x = *reinterpret_cast<unsigned long long *>(&a), y = *reinterpret_cast<unsigned long long *>(&b);
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return *reinterpret_cast<float2 *>(&r);
}
// exp((x - base) / T) of two scores; minus_base = (-base, -base), c2 = (c, c)
__device__ __forceinline__ float2 exp_pair(float2 x, float2 minus_base, float2 c2) {
    const float2 d = mul2(add2(x, minus_base), c2);
    return make_float2(exp2_fast(d.x), exp2_fast(d.y));
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <typename V> __device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Place of a score in the order of a row: larger scores first, of equal ones the lower class.  0: not a score that can be
// chosen (-inf: masked; NaN).  Adding 0 makes one of the two zeros.
__device__ __forceinline__ unsigned score_key(float v) {
    const unsigned b = __float_as_uint(__fadd_rn(v, 0.f));
    return v > minus_inf() ? ((b & 0x80000000u) ? ~b : (b | 0x80000000u)) : 0u;
}
__device__ __forceinline__ float key_score(unsigned key) {
    return key == 0u ? minus_inf() : __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ float teacher_logit(const DistillArgs &a, long long n, int e) {
    const long long at = n * a.logits_stride + e;
    if (a.logits_type == SCORE_F32) return static_cast<const float *>(a.logits)[at];
    if (a.logits_type == SCORE_F16) return score_f32(static_cast<const __half *>(a.logits)[at]);
    return score_f32(static_cast<const __nv_bfloat16 *>(a.logits)[at]);
}

// ---- the teacher's side of one row -----------------------------------------------------------
// What a row's listed scores t_j say at temperature T: q_j = exp(t_j / T - L) with L the teacher's log-sum-exp over all classes,
// or (none given) that of the listed ones; of the mass that is left, `rest`, nothing is known but that it lies on the others.
// A class that is listed twice holds the sum of both.  Worked in doubles: `rest` and the logarithms are differences of nearly
// equal numbers, and there are only a few of them per row.
struct TeacherSide {
    double entropy, mass;      // sums over the listed classes of q log q, of q
    float total, rest;         // all mass (0: the row has no teacher), what is not listed
};

// One warp; entry e = lane + 32 s of the row's list: id[s] a class (-1: none) and t[s] its score become id[s] (-1 also where the class
// stands further in front, if `repeats` are possible) and the mass q[s].
template <int S>
__device__ __forceinline__ TeacherSide teacher_of(const DistillArgs &a, const float *lse, int (&id)[S], const float (&t)[S], float (&mass_of)[S], bool repeats) {
    const int lane = threadIdx.x & 31, top = a.top;
    const double inv_t = a.inv_t;
    double u[S], q[S], lq[S];
    float best = minus_inf();
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const float v = id[s] >= 0 ? t[s] : minus_inf();
        u[s] = (double)v * inv_t;
        best = v != v ? v : best != best ? best : fmaxf(best, v);
    }
    const bool broken = __any_sync(0xffffffffu, best != best);
    best = warp_max(best);
    const bool none = best == minus_inf() && !broken;   // nothing is listed, or nothing that the teacher thinks possible
    double L;
    if (lse) {
        L = (double)*lse;
    } else {
        double sum = 0;
#pragma unroll
        for (int s = 0; s < S; ++s)
            if (s == 0 || 32 * s < top) sum += id[s] >= 0 ? exp(u[s] - (double)best * inv_t) : 0.0;
        L = (double)best * inv_t + log(warp_sum(sum));
    }
    double mass = 0, entropy = 0;
    int distinct = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        lq[s] = q[s] = 0;
        if (s > 0 && 32 * s >= top) continue;
        lq[s] = u[s] - L;
        if (id[s] >= 0 && !none) q[s] = exp(lq[s]);
        if (!repeats) continue;
        // an earlier entry of the same class takes this one's mass
        const unsigned same = __match_any_sync(0xffffffffu, id[s]);
        const int first = __ffs(same) - 1;
        if (__any_sync(0xffffffffu, id[s] >= 0 && first != lane)) {
            double sum = 0;
            for (int l = 0; l < 32; ++l) {
                const double v = __shfl_sync(0xffffffffu, q[s], l);
                if (same >> l & 1) sum += v;
            }
            if (id[s] >= 0) {
                if (first != lane) { id[s] = -1; q[s] = 0; }
                else if (same != 1u << lane) { q[s] = sum; lq[s] = log(sum); }
            }
        }
#pragma unroll
        for (int b = 0; b < s; ++b) {
            for (int l = 0; l < 32; ++l) {   // entry l of this segment against all of segment b
                const int other = __shfl_sync(0xffffffffu, id[s], l);
                const unsigned hit = __ballot_sync(0xffffffffu, other >= 0 && other == id[b]);
                if (hit) {
                    const double v = __shfl_sync(0xffffffffu, q[s], l);
                    if (hit >> lane & 1) { q[b] += v; lq[b] = log(q[b]); }
                    if (lane == l) { id[s] = -1; q[s] = 0; }
                }
            }
        }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
        mass_of[s] = (float)q[s];
        mass += q[s];
        if (q[s] != 0) entropy += q[s] * lq[s];
        distinct += __popc(__ballot_sync(0xffffffffu, id[s] >= 0));
    }
    mass = warp_sum(mass);
    if (a.loss) entropy = warp_sum(entropy);
    const double rest = lse && !none && distinct < a.k && mass < 1 ? 1.0 - mass : 0.0;
    TeacherSide r;
    r.total = none ? 0.f : (float)(mass + rest);
    r.rest = (float)rest;
    r.entropy = entropy;
    r.mass = mass;
    return r;
}

// The same from the row's list in global memory.  list_id[e], list_q[e]: what becomes of entry e.  S: segments of 32 entries that the
// list may have.
template <int S = SCORES_MAX_TOP / 32>
__device__ __forceinline__ TeacherSide read_teacher(const DistillArgs &a, long long n, int *list_id, float *list_q) {
    const int lane = threadIdx.x & 31;
    const int *ids = a.ids + n * a.ids_stride;
    int id[S];
    float t[S], q[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int e = lane + 32 * s, i = e < a.top ? ids[e] : -1;
        id[s] = i >= 0 && i < a.k ? i : -1;
        t[s] = e < a.top ? teacher_logit(a, n, e) : 0.f;
    }
    const TeacherSide r = teacher_of<S>(a, a.lse ? a.lse + n : nullptr, id, t, q, true);
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int e = lane + 32 * s;
        if (e < a.top) { list_id[e] = id[s]; list_q[e] = q[s]; }
    }
    __syncwarp();
    return r;
}

// ---- the student's side ----------------------------------------------------------------------
// Scores are taken relative to the largest of their kind, so a sum of exponentials holds a 1 and does not overflow.  "Rest"
// are the classes summed in the pass over the row -- those that the teacher does not list, or (no bucket for them is needed) all --
// and `top`, `sum`, `sum1` are those of all classes.  The rest has a reference of its own: a student far from all of it still
// gets the gradient that says which of them to raise.  Without a score above -inf in the whole row references are 0.
struct StudentRow {
    float base, rest, rest1;   // largest of the rest; sums of exp((s - base) / T) and exp(s - base)
    float top, sum, sum1;      // the same of all classes
    float l;                   // sum of exp((s - top) / T) over the classes that are not of the rest
};
// Without a score above -inf the rest has the reference of all classes: its sums are 0 there as anywhere, and what brings them from
// one reference to the other is 1, not infinite.
__device__ __forceinline__ float reference_of(float base, float rest, float top) { return rest == 0.f ? top : base; }
__device__ __forceinline__ float row_top(float largest) { return largest == minus_inf() ? 0.f : largest; }

// Factors of a row's gradients.  For class i with shares p (at T) and p1 (at 1):
//   listed:  g = soft * (total * p - q) + hard * (p1 - [label])
//   others:  g = soft * (total * p - rest * p / p_rest) + hard * (p1 - [label])
//   h = max(curve * p (1 - p) + 2 hard * p1 (1 - p1), 1e-16)
struct DistillRow {
    float base, c;            // others: e = exp((s - base) / T) = 2^((s - base) c); p = e * to_p, p1 = exp(s - base) * to_p1
    float to_p, to_p1, to_g;  // soft * (total * p - rest * p / p_rest) = e * to_g
    float top, inv_sum, inv_sum1;
    float soft, hard;         // w alpha T, w (1 - alpha)
    float total, curve;       // the teacher's mass; 2 w alpha where the row has a teacher
    int label;                // -1: none
};

constexpr float MIN_HESSIAN = 1e-16f;   // the softmax objective's

__device__ __forceinline__ float2 finish_gh(const DistillRow &d, int i, float g, float p, float p1) {
    g = __fmaf_rn(d.hard, i == d.label ? p1 - 1.f : p1, g);
    const float cp = d.curve * p, cp1 = (2.f * d.hard) * p1;
    return make_float2(g, fmaxf(__fmaf_rn(-cp, p, cp) + __fmaf_rn(-cp1, p1, cp1), MIN_HESSIAN));
}
template <bool TWO>   // the hard labels need the shares at temperature 1 as well
__device__ __forceinline__ float2 other_gh(const DistillRow &d, int i, float s) {
    const float x = __fsub_rn(s, d.base), e = exp2_fast(x * d.c), p = e * d.to_p;
    return finish_gh(d, i, e * d.to_g, p, TWO ? exp2_fast(x * LOG2E) * d.to_p1 : p);
}
template <bool TWO>
__device__ __forceinline__ float2 listed_gh(const DistillRow &d, int i, float s, float q) {
    const float x = __fsub_rn(s, d.top), p = exp2_fast(x * d.c) * d.inv_sum;
    return finish_gh(d, i, d.soft * (d.total * p - q), p, TWO ? exp2_fast(x * LOG2E) * d.inv_sum1 : p);
}

// label of a row as a class, -1 where it has none
__device__ __forceinline__ int row_label(const DistillArgs &a, long long n) {
    if (a.labels) {
        const int y = a.labels[n];
        return y >= 0 && y < a.k ? y : -1;
    }
    if (a.labels_f) {
        const float y = a.labels_f[n];
        return y >= 0.f && y < (float)a.k ? (int)y : -1;
    }
    return -1;
}

__device__ __forceinline__ DistillRow distill_row(const DistillArgs &a, const TeacherSide &t, const StudentRow &s, float w, int label) {
    DistillRow d;
    const float c = a.c;
    const float alpha = t.total == 0.f ? 0.f : a.alpha;
    const float low = __fsub_rn(s.base, s.top);
    d.base = s.base; d.top = s.top; d.c = c;
    d.inv_sum = s.sum == 0.f ? 0.f : fast_inverse(s.sum);
    d.inv_sum1 = s.sum1 == 0.f ? 0.f : fast_inverse(s.sum1);
    d.to_p = exp2_fast(low * c) * d.inv_sum;
    d.to_p1 = exp2_fast(low * LOG2E) * d.inv_sum1;
    d.label = label;
    d.soft = w * alpha * a.temperature;
    d.hard = label >= 0 ? w * (1.f - a.alpha) : 0.f;
    d.total = t.total;
    d.to_g = d.soft * (t.total * d.to_p - (t.rest > 0.f && s.rest != 0.f ? t.rest * fast_inverse(s.rest) : 0.f));
    d.curve = 2.f * w * alpha;
    return d;
}
// listed: sum over the listed classes of q (s - top) / T
__device__ __forceinline__ float distill_loss(const DistillArgs &a, const TeacherSide &t, const StudentRow &s, float w, int label,
                                              double listed, float label_score) {
    double loss = 0;
    // (a row without a score above -inf: its listed sum or its label's score is -inf already, and the loss infinite)
    double log_sum = s.sum == 0.f ? 0.0 : fine_log(s.sum);
    if (t.total != 0.f) {
        double kl = 0;
        if (t.rest > 0.f) {
            // The rest's term and those of the listed classes take most of each other away where both sides leave nearly all mass, and
            // nearly the same, to the rest: its logarithms are those of 1 - mass and 1 / (1 + ratio), not of their roundings.
            const double low = ((double)s.base - (double)s.top) * a.inv_t;
            const float ratio = s.l * exp2f(-__fsub_rn(s.base, s.top) * a.c) / s.rest;   // listed to unlisted sum
            double share;   // log of the rest's share
            if (ratio < 1.f) {
                const double more = log1p((double)ratio);
                share = -more;
                log_sum = low + fine_log(s.rest) + more;
            } else {
                share = low + fine_log(s.rest) - log_sum;
            }
            kl = (1.0 - t.mass) * (log1p(-t.mass) - share);
        }
        kl += t.entropy - (listed - t.mass * log_sum);
        if (a.alpha > 0.f) loss = (double)a.alpha * a.temperature * a.temperature * kl;   // (it may be infinite)
    }
    if (label >= 0 && a.alpha < 1.f)
        loss -= (1.0 - (double)a.alpha) * ((double)label_score - (double)s.top - (s.sum1 == 0.f ? 0.0 : fine_log(s.sum1)));
    return w == 0.f ? 0.f : (float)((double)w * loss);
}

// ---- a row whose scores lie in shared memory, one warp ---------------------------------------
// asynchronous copy of one float into shared memory
__device__ __forceinline__ void copy_async4(float *to, const float *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// The row z[i * step], i < k: lane l has the scores l, l + 32, ...  E > 0: at most 32 E scores, in registers; 0: they are read again from
// shared memory by every pass.  each(f): f(score, class) for all lanes together, -inf behind the last class.
template <int E> struct WarpRow {
    const float *z;
    int step, k;
    float x[E ? E : 1];
    __device__ __forceinline__ WarpRow(const float *z_, int step_, int k_) : z(z_), step(step_), k(k_) {
        if constexpr (E > 0) {
            const int lane = threadIdx.x & 31;
#pragma unroll
            for (int j = 0; j < E; ++j) x[j] = lane + 32 * j < k ? z[(lane + 32 * j) * step] : minus_inf();
        }
    }
    // sum of exp((x - base) / T), c as in exp_pair
    __device__ __forceinline__ float exps(float base, float c) const {
        if constexpr (E > 0) {
            const float2 mb = make_float2(-base, -base), c2 = make_float2(c, c);
            float2 s = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < E; j += 2) s = add2(s, exp_pair(make_float2(x[j], x[j + 1]), mb, c2));
            return __fadd_rn(s.x, s.y);
        } else {
            float s = 0;
            each([&](float v, int, int) { s += exp2_fast(__fsub_rn(v, base) * c); });
            return s;
        }
    }
    template <typename F> __device__ __forceinline__ void each(F &&f) const {
        const int lane = threadIdx.x & 31;
        if constexpr (E > 0) {
#pragma unroll
            for (int j = 0; j < E; ++j) f(x[j], lane + 32 * j, j);
        } else {
            for (int i = 0; i < k; i += 32) f(i + lane < k ? z[(i + lane) * step] : minus_inf(), i + lane, i / 32);
        }
    }
};

// score_key without its special cases: what cannot be chosen (-inf; NaN is made one) lies below LOWEST_KEY
constexpr unsigned LOWEST_KEY = 0x00800000u;
__device__ __forceinline__ unsigned plain_key(float v) {
    const unsigned b = __float_as_uint(__fadd_rn(fmaxf(v, minus_inf()), 0.f));
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}

// The `top` largest scores of a row, in order.  A border that at least `top` of the maxima of 32 G groups of classes reach is
// reached by at least `top` scores, and by few more as long as `top` is well below the number of groups (20 G): it is found by sorting
// the maxima or by bisection.  The scores from there on are collected in class order, and each finds its place by counting those
// before it.  Rows with too many (more than TOP_ROOM G: ties, or large scores in few groups) choose one after the other: 32 of
// 250 classes of 50003 rows took 341 us with as many groups, for almost all rows did.  `room`: TOP_ROOM G keys and as many
// classes of the warp's own.
constexpr int TOP_ROOM = 64;

template <int E, int G>
__device__ __forceinline__ void warp_top(const WarpRow<E> &row, int top, unsigned *room, float *values, int *ids) {
    const int lane = threadIdx.x & 31;
    unsigned *keys = room;
    int *place = reinterpret_cast<int *>(room + TOP_ROOM * G);
    unsigned mx[G];
#pragma unroll
    for (int g = 0; g < G; ++g) mx[g] = 0;
    row.each([&](float x, int, int j) {
        const unsigned key = plain_key(x);
        if constexpr (E > 0) {
            mx[j % G] = max(mx[j % G], key);
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g)
                if (j % G == g) mx[g] = max(mx[g], key);
        }
    });
    unsigned low;
    if constexpr (G == 1) {   // the maxima in order, largest first: lane top - 1 has the border
        unsigned v = mx[0];
#pragma unroll
        for (int size = 2; size <= 32; size *= 2)
#pragma unroll
            for (int d = size / 2; d > 0; d /= 2) {
                const unsigned o = __shfl_xor_sync(0xffffffffu, v, d);
                v = ((lane & d) == 0) == ((lane & size) == 0) ? max(v, o) : min(v, o);
            }
        low = __shfl_sync(0xffffffffu, v, top - 1);
    } else {
        unsigned high = mx[0];
        low = mx[0];
#pragma unroll
        for (int g = 1; g < G; ++g) { low = min(low, mx[g]); high = max(high, mx[g]); }
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        for (int steps = 0; steps < 20; ++steps) {   // all maxima reach `low` at first; at least `top` always do
            const unsigned mid = low + (high - low + 1) / 2;
            if (mid == low) break;
            int reach = 0;
#pragma unroll
            for (int g = 0; g < G; ++g) reach += __popc(__ballot_sync(0xffffffffu, mx[g] >= mid));
            if (reach >= top) {
                low = mid;
                if (reach <= top + top / 16) break;
            } else {
                high = mid - 1;
            }
        }
    }
    const unsigned from = max(low, LOWEST_KEY), before = (1u << lane) - 1;
    int m = 0;
    row.each([&](float x, int i, int) {
        const unsigned key = plain_key(x);
        const unsigned take = __ballot_sync(0xffffffffu, key >= from);
        const int at = m + __popc(take & before);
        if (key >= from && at < TOP_ROOM * G) { keys[at] = key; place[at] = i; }
        m += __popc(take);
    });
    if (m <= TOP_ROOM * G) {
        if (lane < 4 && m + lane < TOP_ROOM * G) keys[m + lane] = 0;   // (read four at a time)
        __syncwarp();
        for (int c = lane; c < m; c += 32) {
            const unsigned own = keys[c];
            int rank = 0;
            for (int j = 0; j < m; j += 4) {
                const uint4 o = *reinterpret_cast<const uint4 *>(keys + j);
                const unsigned over = own + (j + 4 > c);   // of equal ones the lower class, which stands in front
                rank += (o.x >= over) + (o.y >= over) + (o.z >= over) + (o.w >= over);
            }
            for (int j = c & ~3; j < c; ++j) rank += keys[j] == own;
            if (rank < top) { values[rank] = key_score(own); ids[rank] = place[c]; }
        }
        for (int j = m + lane; j < top; j += 32) { values[j] = minus_inf(); ids[j] = -1; }
    } else {
        unsigned long long last = ~0ull;
        for (int j = 0; j < top; ++j) {
            unsigned long long b = 0;
            row.each([&](float x, int i, int) {
                const unsigned key = plain_key(x);
                const unsigned long long v = (unsigned long long)key << 32 | (unsigned)~i;
                if (key >= LOWEST_KEY && v < last && v > b) b = v;
            });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
            last = b;
            if (lane == 0) { values[j] = key_score((unsigned)(b >> 32)); ids[j] = b ? (int)~(unsigned)b : -1; }
        }
    }
    __syncwarp();
}

// What one warp finds out about a row.  What follows from it is a few dozen operations per row, which lanes do for a row each.
struct RowSums {
    TeacherSide teacher;
    double of_listed;                  // sum over the listed classes of q (s - top) / T
    float base, rest, rest1, top, l, l1;   // as in StudentRow; l, l1: of the listed classes, relative to `top`
    float label_score;
};
__device__ __forceinline__ StudentRow student_of(const DistillArgs &a, const RowSums &r) {
    StudentRow s;
    s.rest = r.rest; s.rest1 = r.rest1; s.top = r.top; s.l = r.l;
    s.base = reference_of(r.base, r.rest, r.top);
    const float low = __fsub_rn(s.base, r.top);
    s.sum = r.rest * exp2_fast(low * a.c) + r.l;
    s.sum1 = r.rest1 * exp2_fast(low * LOG2E) + r.l1;
    return s;
}

// The sums of the row z[i * step], by one warp.  The cells of listed classes become -inf, their scores go to list_x.
template <int E, bool TWO, int S>
__device__ __forceinline__ void warp_student(const DistillArgs &a, long long n, float *z, int step, const int *list_id, const float *list_q, float *list_x, RowSums &out) {
    const int lane = threadIdx.x & 31, k = a.k;
    float label_score = 0;
    if (a.loss) {
        const int label = row_label(a, n);
        if (label >= 0) label_score = z[label * step];
        __syncwarp();
    }
    float x[S];
    float top = minus_inf();
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int e = lane + 32 * s;
        x[s] = minus_inf();
        if (e < a.top && list_id[e] >= 0) {
            float *cell = z + list_id[e] * step;
            x[s] = *cell;
            *cell = minus_inf();
            list_x[e] = x[s];
            top = fmaxf(top, x[s]);
        }
    }
    __syncwarp();
    float s0 = 0, s1 = 0, base;
    {
        const WarpRow<E> row(z, step, k);
        float m = minus_inf();
        row.each([&](float v, int, int) { m = fmaxf(m, v); });
        m = warp_max(m);
        base = row_top(m);
        top = row_top(fmaxf(warp_max(top), m));
        s0 = row.exps(base, a.c);
        if (TWO) s1 = row.exps(base, LOG2E);
    }
    __syncwarp();
    s0 = warp_sum(s0);
    s1 = TWO ? warp_sum(s1) : s0;
    float l = 0, l1 = 0;
    double of_listed = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        const int e = lane + 32 * s;
        if (e < a.top && list_id[e] >= 0) {
            const float d = __fsub_rn(x[s], top), q = list_q[e];
            l += exp2_fast(d * a.c);
            if (TWO) l1 += exp2_fast(d * LOG2E);
            if (a.loss && q != 0.f) of_listed += (double)q * (((double)x[s] - (double)top) * a.inv_t);
        }
    }
    l = warp_sum(l);
    l1 = TWO ? warp_sum(l1) : l;
    if (a.loss) of_listed = warp_sum(of_listed);
    if (lane == 0) {
        out.of_listed = of_listed; out.base = base; out.rest = s0; out.rest1 = s1; out.top = top; out.l = l; out.l1 = l1;
        out.label_score = label_score;
    }
    __syncwarp();
}

// ---- a long row in global memory, a block or a cluster of blocks -----------------------------
// 16 bytes of scores
template <typename T> struct Pack {
    static constexpr int V = 16 / (int)sizeof(T);
    uint4 bits;
    __device__ __forceinline__ void unpack(float (&v)[V]) const {
        const unsigned w[4] = {bits.x, bits.y, bits.z, bits.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ void pack(const float (&v)[V]) {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
            else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const unsigned *>(&h);
            } else {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const unsigned *>(&h);
            }
        }
        bits = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// The part [lo, hi) of a row whose cells lie side by side: single cells up to the first 16-byte boundary, packs, single cells.
template <typename T> struct Part {
    const T *p;
    int head, packs, tail;   // cells [0, head), head + V * packs, the rest
    __device__ __forceinline__ Part(const T *row, int lo, int hi) : p(row + lo) {
        constexpr int V = Pack<T>::V;
        const int n = hi - lo;
        head = min(n, (int)((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T)));
        packs = (n - head) / V;
        tail = n - head - packs * V;
    }
    __device__ __forceinline__ const uint4 *body() const { return reinterpret_cast<const uint4 *>(p + head); }
    // cell of the i-th single one
    __device__ __forceinline__ int single(int i) const { return i < head ? i : i + Pack<T>::V * packs; }
};

// running sum of exponentials relative to the largest score so far
template <bool TWO> struct Running {
    float m, s, s1;
    __device__ __forceinline__ Running() : m(minus_inf()), s(0.f), s1(0.f) {}
    __device__ __forceinline__ void raise(float to, float c) {
        if (to > m) {
            const float d = __fsub_rn(m, to);
            s *= exp2_fast(d * c);
            if (TWO) s1 *= exp2_fast(d * LOG2E);
            m = to;
        }
    }
    __device__ __forceinline__ void add(float x, float base, float c) {   // base = row_top(m)
        const float d = __fsub_rn(x, base);
        s += exp2_fast(d * c);
        if (TWO) s1 += exp2_fast(d * LOG2E);
    }
    template <int V> __device__ __forceinline__ void add_pack(const float (&v)[V], float c) {
        float largest = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) largest = fmaxf(largest, v[i]);
        raise(largest, c);
        const float base = -row_top(m);
        const float2 mb = make_float2(base, base), c2 = make_float2(c, c), one = make_float2(LOG2E, LOG2E);
        float2 sum = make_float2(0.f, 0.f), sum1 = sum;
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            const float2 d = add2(make_float2(v[i], v[i + 1]), mb), x = mul2(d, c2);
            sum = add2(sum, make_float2(exp2_fast(x.x), exp2_fast(x.y)));
            if (TWO) {
                const float2 x1 = mul2(d, one);
                sum1 = add2(sum1, make_float2(exp2_fast(x1.x), exp2_fast(x1.y)));
            }
        }
        s += __fadd_rn(sum.x, sum.y);
        if (TWO) s1 += __fadd_rn(sum1.x, sum1.y);
    }
    __device__ __forceinline__ void join(float om, float os, float os1, float c) {   // another one's
        const float to = fmaxf(m, om);
        const float a = m == to ? 0.f : __fsub_rn(m, to), b = om == to ? 0.f : __fsub_rn(om, to);
        s = s * exp2_fast(a * c) + os * exp2_fast(b * c);
        if (TWO) s1 = s1 * exp2_fast(a * LOG2E) + os1 * exp2_fast(b * LOG2E);
        m = to;
    }
    __device__ __forceinline__ void join_warp(float c) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            join(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), TWO ? __shfl_xor_sync(0xffffffffu, s1, o) : 0.f, c);
    }
};

}  // namespace tgbm
