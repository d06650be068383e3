// Operators on the scores of many classes: penalties, biases and masks (adjust), the largest scores of a row with its
// log-sum-exp (top), distance from a teacher's largest scores with its gradient (distill), classes drawn from given random numbers
// (sample), loss on drawn classes with its gradient (feedback), rows at mean 0 and variance 1 with the way back (norm, norm_backward).
#pragma once
#include <cuda_runtime.h>

#include <cfloat>

namespace tgbm {

enum ScoreType { SCORE_F32 = 0, SCORE_F16 = 1, SCORE_BF16 = 2 };
enum DistillGives { GIVES_LOSS = 0, GIVES_GRADIENT = 1, GIVES_PAIRS = 2 };

constexpr int SCORES_MAX_CLASSES = 1 << 20, SCORES_MAX_TOP = 128;
constexpr int SCORES_CLASS_MOST = 1024;   // by class, up to here a lane takes a row whose scores the warps of a block share

// exp(x / t) is computed as 2^(x log2(e) / t), with the factor in a float
inline bool temperature_fits(float t) { return t > 0.f && t <= FLT_MAX && 1.44269504088896341 / (double)t <= (double)FLT_MAX; }

// rows x classes, class k of row n at data[n * row + k * cls]
struct ScoreView {
    void *data = nullptr;
    int type = SCORE_F32;
    long long row = 0, cls = 0;
    bool one_by_class = false;   // a single row of a matrix that is laid out by class: distill computes it, up to 1024 classes, as its neighbours
};

struct AdjustArgs {
    int n = 0, k = 0;
    ScoreView in, out;
    const float *bias = nullptr;
    const unsigned *allowed = nullptr;   // n_masks x mask_stride words, bit k & 31 of word k >> 5
    long long mask_stride = 0;
    int n_masks = 0;
    const int *allowed_row = nullptr;    // mask of a row; null: row n has mask n
    const long long *history_ptr = nullptr;
    const int *history = nullptr;
    long long n_history = 0;
    float repetition = 1.f, frequency = 0.f, presence = 0.f;
    float inv_repetition = 1.f;          // filled in by scores_adjust
};
void scores_adjust(const AdjustArgs &a, cudaStream_t stream);

struct TopArgs {
    int n = 0, k = 0, top = 0;
    ScoreView in;
    float temperature = 1.f;
    double inv_t = 1;          // filled in by scores_top, scores_distill: 1 / T, and c with exp(x / T) = 2^(x c)
    float c = 0;
    float *values = nullptr;   // n x top
    int *ids = nullptr;        // n x top
    float *lse = nullptr;      // n, or null
};
void scores_top(const TopArgs &a, cudaStream_t stream);

struct DistillArgs {
    int n = 0, k = 0, top = 0;
    ScoreView in;
    const int *ids = nullptr;
    long long ids_stride = 0;
    const void *logits = nullptr;
    int logits_type = SCORE_F32;
    long long logits_stride = 0;
    const float *lse = nullptr;       // the teacher's log-sum-exp at this temperature: what is not listed is one bucket
    const int *labels = nullptr;      // class of a row, anything outside [0, k): none
    const float *labels_f = nullptr;  // ... the same as floats (the booster's)
    const float *weights = nullptr;
    float temperature = 1.f, alpha = 1.f;
    double inv_t = 1;
    float c = 0, c_low = 0;
    int gives = GIVES_LOSS;
    float *loss = nullptr;            // n, or null
    ScoreView out;                    // gradient in the scores' type, or (gradient, hessian) pairs of floats
    unsigned *maxbits = nullptr;      // largest |gradient| and hessian as bits (the booster's rounds)
};
void scores_distill(const DistillArgs &a, cudaStream_t stream);

// Numbers that hold for all rows, or (where there is a pointer) one per row.
struct SampleArgs {
    int n = 0, k = 0, draws = 0;
    ScoreView in;
    const void *uniform = nullptr;   // n x draws floats or doubles
    bool uniform_f64 = false;
    float temperature = 1.f, top_p = 1.f, min_p = 0.f;
    int top_k = 0;                   // 0: no limit
    const float *temperatures = nullptr, *top_ps = nullptr, *min_ps = nullptr;
    const int *top_ks = nullptr;
    int *classes = nullptr;          // n x draws
    float *logs = nullptr, *all_logs = nullptr;   // n x draws each, or null
};
void scores_sample(const SampleArgs &a, cudaStream_t stream);

struct FeedbackArgs {
    int n = 0, k = 0, draws = 0;
    ScoreView in;
    const int *classes = nullptr;    // n x draws, like the three that follow
    const float *gains = nullptr;
    const float *old = nullptr;      // null: the present ones
    const float *reference = nullptr;
    const float *weights = nullptr;  // n, or null
    float temperature = 1.f, clip_low = 1.f, clip_high = FLT_MAX, kl = 0.f, entropy = 0.f;
    double inv_t = 1;                // filled in by scores_feedback, like the bounds of the ratio
    float c = 0, least = 0, most = 0;
    int gives = GIVES_LOSS;
    float *loss = nullptr;           // n, or null
    float *logs = nullptr;           // n x draws, or null
    ScoreView out;                   // gradient in the scores' type, or (gradient, hessian) pairs of floats
    unsigned *maxbits = nullptr;     // largest |gradient| and hessian as bits (the booster's rounds)
};
void scores_feedback(const FeedbackArgs &a, cudaStream_t stream);

struct NormArgs {
    int n = 0, k = 0;
    ScoreView in, out;
    const float *gain = nullptr, *bias = nullptr;
    float eps = 1e-5f;
    float *mean = nullptr, *rstd = nullptr;
};
void scores_norm(const NormArgs &a, cudaStream_t stream);

struct NormBackwardArgs {
    int n = 0, k = 0;
    ScoreView grad, in, out;
    const float *mean = nullptr, *rstd = nullptr, *gain = nullptr;
    float *to_gain = nullptr, *to_bias = nullptr;   // null: not wanted
    float *work = nullptr;                          // norm_work(n, k) floats where they are
};
long long norm_work(int n, int k);
void scores_norm_backward(const NormBackwardArgs &a, cudaStream_t stream);

}  // namespace tgbm
