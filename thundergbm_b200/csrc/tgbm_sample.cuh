// What the kernels that draw classes share: a row's limits, exponentials in 64 bits, borders by bisection.
//
// Which class a random number falls on is decided by sums of exponentials next to one another, and a row may have 2^20 of them:
// exponentials and their sums are doubles, so that the classes are those of the definition.
#pragma once
#include <cfloat>

#include "tgbm_scores.cuh"
#include "tgbm_scores_long.cuh"

namespace tgbm {

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
    // (NaN: 0.)  Below 1: a share of a mass that is then below it, so that one of those who share the mass has the draw.
    return u > 0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
}
__device__ __forceinline__ void put_draw(const SampleArgs &a, long long i, int cls, float log, float all_log) {
    a.classes[i] = cls;
    if (a.logs) a.logs[i] = log;
    if (a.all_logs) a.all_logs[i] = all_log;
}

// ---- exponentials in 64 bits ------------------------------------------------------------------
// exp(d / T) for d <= 0, relative error below 2^-38: with y = 32 d log2(e) / T and n the whole number nearest to it, 2^(n / 32) is a power of two times one
// of 32 numbers (a table in shared memory), and exp of the rest, |rest| <= ln 2 / 64, five terms of its series, the first left out
// below 2^-39.  10 instructions of the fp64 units, which do half as many as the fp32 ones; the library's exp takes twice as many.
struct Powers {
    double of[32];
    __device__ __forceinline__ void fill() {   // a warp; a barrier has to follow
        const int lane = threadIdx.x & 31;
        of[lane] = exp2((double)lane * 0.03125);
    }
};
struct Exponent {
    double by;   // 32 log2(e) / T; temperature 0: so much that any distance counts for nothing
    __device__ __forceinline__ Exponent(const Limits &l) : by(l.greedy ? 1e300 : l.inv_t * 46.166241308446828384) {}
    __device__ __forceinline__ double operator()(const Powers &t, float x, float top) const {
        const double y = __dmul_rn(__dsub_rn((double)x, (double)top), by);
        if ((unsigned)__double2hiint(y) > 0xc0df4000u) return 0.0;   // (y < -32000: 2^-1000; -inf.  y is at most 0: its sign, exponent and first digits tell)
        const double shifted = __dadd_rn(y, 6755399441055744.0);   // 1.5 * 2^52: whole numbers
        const int n = __double2loint(shifted);
        const double r = __dsub_rn(y, __dsub_rn(shifted, 6755399441055744.0));
        constexpr double A1 = 0.6931471805599453094 / 32, A2 = A1 * A1 / 2, A3 = A1 * A1 * A1 / 6, A4 = A1 * A1 * A1 * A1 / 24;
        const double p = __fma_rn(r, __fma_rn(r, __fma_rn(r, __fma_rn(r, A4, A3), A2), A1), 1.0);
        const double v = __dmul_rn(t.of[n & 31], p);
        return __hiloint2double(__double2hiint(v) + ((n >> 5) << 20), __double2loint(v));
    }
};

// May masses be sums of 2^((x - top) c) by floats, c = log2(e) / T?  Not where c is none, nor where a difference that is none would still have a mass.
__device__ __forceinline__ bool floats_tell(const Limits &l) { return l.inv_t >= 1e-30 && l.inv_t <= 2e38; }

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

// long rows (tgbm_sample_long.cuh), a source file for each type: the kernels are large
template <typename T> bool sample_long(const SampleArgs &a, cudaStream_t stream);

}  // namespace tgbm
