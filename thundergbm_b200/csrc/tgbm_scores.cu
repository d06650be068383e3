// Operators on the scores of many classes: penalties, biases and masks (adjust), the largest scores of a row with its
// log-sum-exp (top), the distance from a teacher's largest scores with its gradient (distill).
//
// Scores are a matrix of rows x classes in float, half or bfloat16 with any two strides; a booster keeps all rows of a class
// side by side, networks all classes of a row.  All three operators are bound by memory: they do a few operations per score.
#include <cfloat>
#include <climits>
#include <cmath>

#include "../../include/thundergbm.h"
#include "tgbm_kernels.cuh"
#include "tgbm_scores.cuh"

namespace tgbm {
namespace {

constexpr int ROW_THREADS = 256;

template <typename T> struct Scores {
    T *p;
    long long row, cls;
    __device__ __forceinline__ T *at(long long n, long long k) const { return p + n * row + k * cls; }
    __device__ __forceinline__ float operator()(long long n, long long k) const { return score_f32(*at(n, k)); }
};
template <typename T> Scores<T> scores_of(const ScoreView &v) { return Scores<T>{static_cast<T *>(v.data), v.row, v.cls}; }

// f<T>() for the element type
template <typename F> void by_type(int type, F &&f) {
    switch (type) {
    case SCORE_F32: f(float{}); break;
    case SCORE_F16: f(__half{}); break;
    case SCORE_BF16: f(__nv_bfloat16{}); break;
    default: throw Error("unknown type of scores");
    }
}

// ------------------------------------------------------------------ adjust
// A block takes a tile of rows x classes.  How often a class stands in the history of its row is counted in shared memory: every
// entry of the tile's histories that falls into its classes adds one (integers: in any order the same), so a history may be
// of any length.
constexpr int ADJUST_CELLS = 8192;

template <typename T, bool BY_CLASS>
__global__ void __launch_bounds__(ROW_THREADS) k_adjust(AdjustArgs a, Scores<T> in, Scores<T> out, int tile_rows, int tile_classes) {
    extern __shared__ int count[];
    const long long n0 = (long long)blockIdx.x * tile_rows;
    const int k0 = blockIdx.y * tile_classes;
    const int rows = (int)min((long long)tile_rows, a.n - n0), classes = min(tile_classes, a.k - k0);
    const int cells = tile_rows * tile_classes;
    auto cell = [&](int r, int c) { return BY_CLASS ? c * tile_rows + r : r * tile_classes + c; };
    if (a.history_ptr) {
        for (int i = threadIdx.x; i < cells; i += ROW_THREADS) count[i] = 0;
        __syncthreads();
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int r = warp; r < rows; r += ROW_THREADS / 32) {
            const long long lo = max(0ll, a.history_ptr[n0 + r]), hi = min(a.n_history, a.history_ptr[n0 + r + 1]);
            for (long long h = lo + lane; h < hi; h += 32) {
                const int c = a.history[h] - k0;
                if (c >= 0 && c < classes) atomicAdd(&count[cell(r, c)], 1);
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < cells; i += ROW_THREADS) {
        const int r = BY_CLASS ? i % tile_rows : i / tile_classes, c = BY_CLASS ? i / tile_rows : i % tile_classes;
        if (r >= rows || c >= classes) continue;
        const long long n = n0 + r;
        const int k = k0 + c;
        float z = in(n, k);
        if (a.history_ptr) {
            const int m = count[i];
            if (m) {
                z = z > 0.f ? z / a.repetition : z * a.repetition;
                z -= (float)m * a.frequency + a.presence;
            }
        }
        if (a.bias) z += a.bias[k];
        if (a.allowed) {
            const int m = a.allowed_row ? a.allowed_row[n] : (int)n;
            if (m >= 0 && m < a.n_masks && !(a.allowed[m * a.mask_stride + (k >> 5)] >> (k & 31) & 1)) z = minus_inf();
        }
        *out.at(n, k) = score_from<T>(z);
    }
}

// ------------------------------------------------------------------ top
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
        const float c = (float)(1.44269504088896341 / (double)a.temperature);
        float s = 0;
        for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) s += exp2_fast(__fsub_rn(in(n, k), m) * c);
        s = warp_sum(s);
        if (lane == 0) part[warp] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            s = 0;
            for (int w = 0; w < ROW_THREADS / 32; ++w) s += part[w];
            a.lse[n] = broken ? __int_as_float(0x7fffffff) : (float)((double)m / (double)a.temperature + log((double)s));
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
    __shared__ TeacherRow teacher;
    __shared__ StudentRow student;
    __shared__ DistillRow drow;
    __shared__ float part[3][ROW_THREADS / 32];
    const long long n = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, W = ROW_THREADS / 32;
    const double inv_t = 1.0 / (double)a.temperature;
    const float c = (float)(1.44269504088896341 / (double)a.temperature);
    for (int i = threadIdx.x; i < (a.k + 31) / 32; i += ROW_THREADS) listed_bits[i] = 0;
    __syncthreads();
    if (warp == 0) {
        read_teacher(teacher, a, n, inv_t);
        __syncwarp();
        for (int j = lane; j < a.top; j += 32)
            if (teacher.id[j] >= 0) atomicOr(&listed_bits[teacher.id[j] >> 5], 1u << (teacher.id[j] & 31));
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
            if (teacher.id[j] >= 0) top = fmaxf(top, in(n, teacher.id[j]));
        st.top = row_top(warp_max(top));
        float l = 0, l1 = 0;
        double ql = 0, mass = 0;
        for (int j = lane; j < a.top; j += 32)
            if (teacher.id[j] >= 0) {
                const float z = in(n, teacher.id[j]), x = __fsub_rn(z, st.top);
                l += exp2_fast(x * c);
                if (TWO) l1 += exp2_fast(x * LOG2E);
                if (teacher.q[j] != 0.f) ql += (double)teacher.q[j] * (((double)z - (double)st.top) * inv_t);
                mass += teacher.q[j];
            }
        l = warp_sum(l); l1 = warp_sum(l1);
        if (!TWO) l1 = l;
        ql = warp_sum(ql); mass = warp_sum(mass);
        const float low = __fsub_rn(base, st.top);
        st.sum = s * exp2_fast(low * c) + l;
        st.sum1 = TWO ? s1 * exp2_fast(low * LOG2E) + l1 : st.sum;
        if (lane == 0) {
            const float w = a.weights ? a.weights[n] : 1.f;
            const int label = row_label(a, n);
            student = st;
            drow = distill_row(a, teacher, st, w, label);
            if (a.loss) a.loss[n] = distill_loss(a, teacher, st, w, label, ql, mass, label >= 0 ? in(n, label) : 0.f);
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
            if (teacher.id[j] >= 0) put(teacher.id[j], listed_gh<TWO>(d, teacher.id[j], in(n, teacher.id[j]), teacher.q[j]));
    }
    if (a.maxbits) track_max(mg, mh, a.maxbits);
}

}  // namespace

// ------------------------------------------------------------------ launches
void scores_adjust(const AdjustArgs &a, cudaStream_t stream) {
    if (a.n == 0) return;
    const bool by_class = a.in.row < a.in.cls;
    const int tile_rows = by_class ? 32 : std::max(1, std::min(a.n, ADJUST_CELLS / std::min(a.k, ADJUST_CELLS)));
    const int tile_classes = by_class ? ADJUST_CELLS / 32 : std::min(a.k, ADJUST_CELLS);
    const dim3 grid((unsigned)((a.n + (long long)tile_rows - 1) / tile_rows), (unsigned)((a.k + tile_classes - 1) / tile_classes));
    const size_t smem = a.history_ptr ? sizeof(int) * (size_t)tile_rows * tile_classes : 0;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        if (by_class) k_adjust<T, true><<<grid, ROW_THREADS, smem, stream>>>(a, scores_of<T>(a.in), scores_of<T>(a.out), tile_rows, tile_classes);
        else k_adjust<T, false><<<grid, ROW_THREADS, smem, stream>>>(a, scores_of<T>(a.in), scores_of<T>(a.out), tile_rows, tile_classes);
    });
    TGBM_CUDA(cudaGetLastError());
}

void scores_top(const TopArgs &a, cudaStream_t stream) {
    if (a.n == 0) return;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        k_top_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, scores_of<T>(a.in));
    });
    TGBM_CUDA(cudaGetLastError());
}

void scores_distill(const DistillArgs &a, cudaStream_t stream) {
    if (a.n == 0) return;
    const bool two = a.alpha < 1.f && a.temperature != 1.f;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
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
namespace {
using namespace tgbm;

int size_of(int type) { return type == SCORE_F32 ? 4 : 2; }

ScoreView view_of(const char *what, const void *data, int type, int n, int k, long long row, long long cls, bool written) {
    const std::string w(what);
    TGBM_CHECK(type >= SCORE_F32 && type <= SCORE_BF16, w + ": unknown type");
    TGBM_CHECK(data != nullptr, w + ": null pointer");
    TGBM_CHECK(reinterpret_cast<uintptr_t>(data) % size_of(type) == 0, w + ": not aligned for its type");
    if (n == 1) row = k == 1 ? 1 : cls * k;   // a stride that no step takes
    if (k == 1) cls = row * n;
    TGBM_CHECK(row >= 0 && cls >= 0, w + ": negative stride");
    const long long most = LLONG_MAX / 16;
    TGBM_CHECK(row <= most / n && cls <= most / k, w + ": stride too large");
    if (written) TGBM_CHECK((row >= 1 && cls > (n - 1) * row) || (cls >= 1 && row > (k - 1) * cls), w + ": strides under which cells share memory");
    ScoreView v;
    v.data = const_cast<void *>(data); v.type = type; v.row = row; v.cls = cls;
    return v;
}

// whether two matrices of n x k share memory (true also where that is not easily told)
bool share_memory(const ScoreView &a, int a_size, const ScoreView &b, int b_size, int n, int k) {
    auto end = [&](const ScoreView &v, int size) { return reinterpret_cast<uintptr_t>(v.data) + size * (uintptr_t)((n - 1) * v.row + (k - 1) * v.cls + 1); };
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a.data), pb = reinterpret_cast<uintptr_t>(b.data);
    if (end(a, a_size) <= pb || end(b, b_size) <= pa) return false;
    if (a_size != b_size || a.row != b.row || a.cls != b.cls || (pa > pb ? pa - pb : pb - pa) % a_size) return true;
    // parts of one larger matrix, side by side: `d` cells apart are `over` lines and `in` cells
    const long long d = (long long)((pa > pb ? pa - pb : pb - pa) / a_size);
    const bool by_row = a.cls <= a.row;
    const long long line = by_row ? a.row : a.cls, step = by_row ? a.cls : a.row;
    const long long lines = by_row ? n : k, cells = by_row ? k : n;
    if (line <= 0) return true;
    const long long over = d / line, in = d % line, width = (cells - 1) * step + 1;
    return (in < width && over < lines) || (line - in < width && over + 1 < lines);
}

void check_shape(int n, int k) {
    TGBM_CHECK(n >= 0, "negative number of rows");
    TGBM_CHECK(k >= 1 && k <= TGBM_SCORES_MAX_CLASSES, "number of classes outside [1, " + std::to_string(TGBM_SCORES_MAX_CLASSES) + "]");
}
void check_temperature(float t) { TGBM_CHECK(t > 0.f && t <= FLT_MAX && 1.0 / (double)t <= FLT_MAX, "the temperature has to be a positive number"); }
void check_list(int top) { TGBM_CHECK(top >= 1 && top <= TGBM_SCORES_MAX_TOP, "length of a row's list outside [1, " + std::to_string(TGBM_SCORES_MAX_TOP) + "]"); }

template <typename F> int scores_call(F &&f) {
    try {
        set_last_error("");
        f();
        return 0;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return 1;
    }
}
}  // namespace

extern "C" {

int tgbm_scores_adjust(int n_rows, int n_classes, int type, const void *d_scores, long long row_stride, long long class_stride, void *d_out,
                       long long out_row_stride, long long out_class_stride, const float *d_bias, const unsigned *d_allowed, int n_masks,
                       long long mask_stride, const int *d_allowed_row, const long long *d_history_ptr, const int *d_history,
                       long long n_history, float repetition, float frequency, float presence, void *cuda_stream) {
    return scores_call([&] {
        check_shape(n_rows, n_classes);
        TGBM_CHECK(repetition > 0.f && repetition <= FLT_MAX, "the repetition penalty has to be a positive number");
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
