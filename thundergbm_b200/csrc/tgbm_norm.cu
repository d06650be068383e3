// Rows of scores at mean 0 and variance 1 over their classes, with a gain and a bias per class (norm), and the way back with the
// gradients of gain and bias (norm_backward).  Scores of -infinity are classes that a row may not have: they are left out of its means.
#include <cfloat>
#include <climits>
#include <cmath>

#include "../../include/thundergbm.h"
#include "tgbm_scores.cuh"
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

// A row, any strides, by a block in three passes.
template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) k_norm_any(NormArgs a, Scores<T> in, Scores<T> out) {
    __shared__ float sums[ROW_WARPS];
    __shared__ int counts[ROW_WARPS];
    const long long n = blockIdx.x;
    auto each = [&](auto &&f) {
        for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
            const float x = in(n, k);
            if (x != minus_inf()) f(x);
        }
    };
    float s = 0;
    int c = 0;
    each([&](float x) { s += x; ++c; });
    const int count = block_sum(c, counts);
    const float mean = count ? block_sum(s, sums) / (float)count : 0.f;
    float q = 0;
    each([&](float x) {
        const float d = __fsub_rn(x, mean);
        q = __fmaf_rn(d, d, q);
    });
    const float rstd = count ? 1.f / sqrtf(block_sum(q, sums) / (float)count + a.eps) : 0.f;
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[n] = mean;
        if (a.rstd) a.rstd[n] = rstd;
    }
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
        const float x = in(n, k), y = __fsub_rn(x, mean) * rstd;
        *out.at(n, k) = score_from<T>(x == minus_inf() ? x : __fmaf_rn(y, a.gain ? a.gain[k] : 1.f, a.bias ? a.bias[k] : 0.f));
    }
}

template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) k_norm_backward_any(NormBackwardArgs a, Scores<T> grad, Scores<T> in, Scores<T> out) {
    __shared__ float sums[ROW_WARPS];
    __shared__ int counts[ROW_WARPS];
    const long long n = blockIdx.x;
    const float mean = a.mean[n], rstd = a.rstd[n];
    float s = 0, sx = 0;
    int c = 0;
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
        const float x = in(n, k);
        if (x == minus_inf()) continue;
        const float g = a.gain ? grad(n, k) * a.gain[k] : grad(n, k);
        s += g;
        sx = __fmaf_rn(g, __fsub_rn(x, mean) * rstd, sx);
        ++c;
    }
    const float inv = 1.f / (float)max(1, block_sum(c, counts));
    s = block_sum(s, sums) * inv;
    sx = block_sum(sx, sums) * inv;
    for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
        const float x = in(n, k);
        float r = 0;
        if (x != minus_inf()) {
            const float g = a.gain ? grad(n, k) * a.gain[k] : grad(n, k);
            r = rstd * __fsub_rn(__fsub_rn(g, s), __fsub_rn(x, mean) * rstd * sx);
        }
        *out.at(n, k) = score_from<T>(r);
    }
}

// Gradients of gain and bias: a block sums a share of the rows for 32 classes, the shares are added in order afterwards.
constexpr int SHARES = 296;
inline int shares_of(int n, int k) { return (int)std::max(1ll, std::min<long long>({(long long)SHARES, (n + 31ll) / 32, (1ll << 23) / k + 1})); }

template <typename T>
__global__ void __launch_bounds__(ROW_THREADS) k_norm_weights_any(NormBackwardArgs a, Scores<T> grad, Scores<T> in, int shares) {
    __shared__ float sums[2][ROW_WARPS][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long k = blockIdx.x * 32ll + lane, share = blockIdx.y;
    const long long from = a.n * share / shares, to = a.n * (share + 1) / shares;
    float s = 0, sx = 0;
    if (k < a.k)
        for (long long n = from + warp; n < to; n += ROW_WARPS) {
            const float x = in(n, k);
            if (x == minus_inf()) continue;
            const float g = grad(n, k);
            s += g;
            sx = __fmaf_rn(g, __fsub_rn(x, a.mean[n]) * a.rstd[n], sx);
        }
    sums[0][warp][lane] = s; sums[1][warp][lane] = sx;
    __syncthreads();
    if (warp < 2 && k < a.k) {
        double t = 0;
        for (int w = 0; w < ROW_WARPS; ++w) t += (double)sums[warp][w][lane];
        a.work[(share * 2 + warp) * a.k + k] = (float)t;
    }
}
__global__ void __launch_bounds__(ROW_THREADS) k_norm_weights_join(NormBackwardArgs a, int shares) {
    const long long i = blockIdx.x * (long long)ROW_THREADS + threadIdx.x;
    if (i >= 2ll * a.k) return;
    double t = 0;
    for (int s = 0; s < shares; ++s) t += (double)a.work[s * 2ll * a.k + i];
    if (i < a.k) a.to_bias[i] = (float)t;
    else a.to_gain[i - a.k] = (float)t;
}
}  // namespace

void scores_norm(const NormArgs &a, cudaStream_t stream) {
    if (a.n == 0) return;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        k_norm_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, scores_of<T>(a.in), scores_of<T>(a.out));
    });
    TGBM_CUDA(cudaGetLastError());
}

long long norm_work(int n, int k) { return 2ll * shares_of(n, k) * k; }

void scores_norm_backward(const NormBackwardArgs &a, cudaStream_t stream) {
    if (a.n == 0) {
        if (a.to_gain) {
            TGBM_CUDA(cudaMemsetAsync(a.to_gain, 0, sizeof(float) * a.k, stream));
            TGBM_CUDA(cudaMemsetAsync(a.to_bias, 0, sizeof(float) * a.k, stream));
        }
        return;
    }
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        const Scores<T> grad = scores_of<T>(a.grad), in = scores_of<T>(a.in), out = scores_of<T>(a.out);
        k_norm_backward_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, grad, in, out);
        if (a.to_gain) {
            const int shares = shares_of(a.n, a.k);
            k_norm_weights_any<T><<<dim3((a.k + 31) / 32, shares), ROW_THREADS, 0, stream>>>(a, grad, in, shares);
            k_norm_weights_join<<<(2 * a.k + ROW_THREADS - 1) / ROW_THREADS, ROW_THREADS, 0, stream>>>(a, shares);
        }
    });
    TGBM_CUDA(cudaGetLastError());
}

}  // namespace tgbm

// ------------------------------------------------------------------ C entries
using namespace tgbm;

extern "C" {

int tgbm_scores_norm(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, void *d_out,
                     long long out_row_stride, long long out_class_stride, const float *d_gain, const float *d_bias, float eps, float *d_mean,
                     float *d_rstd, void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        TGBM_CHECK(eps > 0.f && eps <= FLT_MAX, "eps has to be a positive number");
        if (n_rows == 0) return;
        NormArgs a;
        a.n = n_rows; a.k = n_classes; a.eps = eps;
        a.in = view_of("scores", d_scores, type, n_rows, n_classes, row_stride, class_stride, false);
        a.out = view_of("out", d_out, type, n_rows, n_classes, out_row_stride, out_class_stride, true);
        const bool in_place = a.in.data == a.out.data && a.in.row == a.out.row && a.in.cls == a.out.cls;
        TGBM_CHECK(in_place || !share_memory(a.in, size_of(type), a.out, size_of(type), n_rows, n_classes), "scores and out share memory but are not the same");
        check_pointer("gain", d_gain, 4); check_pointer("bias", d_bias, 4); check_pointer("mean", d_mean, 4); check_pointer("rstd", d_rstd, 4);
        auto read = [&](const char *what, const void *p) {
            TGBM_CHECK(!lies_in(a.out, size_of(type), n_rows, n_classes, p, 4ll * n_classes), std::string("out and ") + what + " share memory");
        };
        read("gain", d_gain); read("bias", d_bias);
        a.gain = d_gain; a.bias = d_bias; a.mean = d_mean; a.rstd = d_rstd;
        scores_norm(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

long long tgbm_scores_norm_work(int n_rows, int n_classes) {
    return n_rows < 1 || n_classes < 1 || n_classes > TGBM_SCORES_MAX_CLASSES ? 0 : 4 * norm_work(n_rows, n_classes);
}

int tgbm_scores_norm_backward(int n_rows, int n_classes, int type, const void *d_grad, long long grad_row_stride, long long grad_class_stride,
                              const void *d_scores, long long row_stride, long long class_stride, const float *d_mean, const float *d_rstd,
                              const float *d_gain, void *d_out, long long out_row_stride, long long out_class_stride, float *d_grad_gain,
                              float *d_grad_bias, void *d_work, long long work_bytes, void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        TGBM_CHECK(!d_grad_gain == !d_grad_bias, "gradients of gain and bias: both or neither");
        NormBackwardArgs a;
        a.n = n_rows; a.k = n_classes;
        check_pointer("gradient of the gain", d_grad_gain, 4); check_pointer("gradient of the bias", d_grad_bias, 4);
        a.to_gain = d_grad_gain; a.to_bias = d_grad_bias;
        if (n_rows > 0) {
            a.grad = view_of("gradient", d_grad, type, n_rows, n_classes, grad_row_stride, grad_class_stride, false);
            a.in = view_of("scores", d_scores, type, n_rows, n_classes, row_stride, class_stride, false);
            a.out = view_of("out", d_out, type, n_rows, n_classes, out_row_stride, out_class_stride, true);
            TGBM_CHECK(!share_memory(a.in, size_of(type), a.out, size_of(type), n_rows, n_classes), "scores and out share memory");
            TGBM_CHECK(!share_memory(a.grad, size_of(type), a.out, size_of(type), n_rows, n_classes), "gradient and out share memory");
            TGBM_CHECK(d_mean && d_rstd, "mean or rstd: null pointer");
            check_pointer("mean", d_mean, 4); check_pointer("rstd", d_rstd, 4); check_pointer("gain", d_gain, 4);
            a.mean = d_mean; a.rstd = d_rstd; a.gain = d_gain;
            if (d_grad_gain) {
                TGBM_CHECK(d_work && work_bytes >= tgbm_scores_norm_work(n_rows, n_classes), "work: less memory than tgbm_scores_norm_work() asks for");
                check_pointer("work", d_work, 16);
                a.work = static_cast<float *>(d_work);
            }
        }
        scores_norm_backward(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

}  // extern "C"
