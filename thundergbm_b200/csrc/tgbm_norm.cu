// Rows of scores at mean 0 and variance 1 over their classes, with a gain and a bias per class (norm), and the way back with the
// gradients of gain and bias (norm_backward).  Scores of -infinity are classes that a row may not have: they are left out of its means.
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

// sum over the block, the same in all threads and every time; `parts`: one per warp
template <int W = ROW_WARPS, typename V> __device__ __forceinline__ V block_sum(V v, V *parts) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
    V s = parts[0];
#pragma unroll
    for (int i = 1; i < W; ++i) s += parts[i];
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

// ---- by class: a lane has a row, the W warps of a block (W = 1: each for itself) share its classes, E in a row each ---------------
// Scores stay in registers from the read to the write.
__device__ __forceinline__ bool there(float x) { return x != minus_inf(); }

// Sums of two numbers over the warps that share a lane's row, the same order in every warp; `turn` alternates, so that nothing is written over
// that is still read.  From 16 warps on a warp adds for a row or two what all of them have, for all of them.
template <int W> struct Shared {
    float2 v[2][W > 1 ? W : 1][33];
    float2 sum[2][32];
};
template <int W> __device__ __forceinline__ float2 over_warps(Shared<W> &sh, int turn, float2 v) {
    if constexpr (W > 1) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        sh.v[turn][warp][lane] = v;
        __syncthreads();
        if constexpr (W <= 8) {
            v = sh.v[turn][0][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) v = add2(v, sh.v[turn][w][lane]);
        } else {
#pragma unroll
            for (int r = warp; r < 32; r += W) {
                float2 u = sh.v[turn][lane & (W - 1)][r];
#pragma unroll
                for (int o = W / 2; o > 0; o >>= 1) u = add2(u, make_float2(__shfl_xor_sync(0xffffffffu, u.x, o), __shfl_xor_sync(0xffffffffu, u.y, o)));
                if (lane == 0) sh.sum[turn][r] = u;
            }
            __syncthreads();
            v = sh.sum[turn][lane];
        }
    }
    return v;
}
// Scores k0, k0 + 1, ... of a lane's row, -inf behind the last class; what steps along the classes is one instruction per address.
template <int E, typename T> __device__ __forceinline__ void read_classes(const T *from, int cls, int here, float none, float (&x)[E]) {
    T raw[E];
    if (here >= E) {
#pragma unroll
        for (int j = 0; j < E; ++j) raw[j] = from[(long long)j * cls];
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j) raw[j] = j < here ? from[(long long)j * cls] : score_from<T>(none);
    }
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = score_f32(raw[j]);
}
template <int E, typename T, typename F> __device__ __forceinline__ void write_classes(T *to, int cls, int here, F &&value) {
    if (here >= E) {
#pragma unroll
        for (int j = 0; j < E; ++j) to[(long long)j * cls] = score_from<T>(value(j));
    } else {
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (j < here) to[(long long)j * cls] = score_from<T>(value(j));
    }
}

// 50003 x 250: 24.9 us (floor 15.3), 23 instructions per score where a tenth is masked; addresses by 64-bit steps and a test of every class's number took 55, and
// 43 us.
template <typename T, int E, int W, bool WEIGHTS>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 8 ? 4 : W == 16 ? 2 : 1) k_norm_class(NormArgs a, Scores<T> in, Scores<T> out) {
    __shared__ Shared<W> sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k0 = W == 1 ? 0 : warp * E, here = a.k - k0;
    const long long n0 = W == 1 ? (blockIdx.x * 4ll + warp) * 32 + lane : blockIdx.x * 32ll + lane, n = min(n0, a.n - 1ll);
    float x[E];
    read_classes<E>(in.at(n, k0), (int)in.cls, here, minus_inf(), x);
    float s = 0, c = 0;
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (there(x[j])) { s += x[j]; c += 1.f; }
    const float2 first = over_warps(sh, 0, make_float2(s, c));
    const float inv = 1.f / fmaxf(first.y, 1.f), mean = first.x * inv;
    float q = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const float d = __fsub_rn(x[j], mean);
        if (there(x[j])) q = __fmaf_rn(d, d, q);
    }
    q = over_warps(sh, 1, make_float2(q, 0.f)).x;
    const float rstd = first.y != 0.f ? 1.f / sqrtf(q * inv + a.eps) : 0.f;
    if (n0 != n) return;
    if (k0 == 0) {
        if (a.mean) a.mean[n] = mean;
        if (a.rstd) a.rstd[n] = rstd;
    }
    const float by = first.y != 0.f ? rstd : 1.f;   // (-inf stays what it is)
    const float *gain = a.gain ? a.gain + k0 : nullptr, *bias = a.bias ? a.bias + k0 : nullptr;
    write_classes<E>(out.at(n, k0), (int)out.cls, here, [&](int j) {
        const float y = __fsub_rn(x[j], mean) * by;
        if (!WEIGHTS) return y;
        return there(x[j]) ? __fmaf_rn(y, gain ? __ldg(gain + j) : 1.f, bias ? __ldg(bias + j) : 0.f) : x[j];
    });
    if (!WEIGHTS && !(by > 0.f && finite(mean))) {   // (and here, where (-inf - mean) by is NaN)
        T *to = out.at(n, k0);
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (j < here && !there(x[j])) to[j * out.cls] = score_from<T>(x[j]);
    }
}

// ---- by row, up to 1024 classes: L lanes have a row, E classes each, L apart -----------------------------------------
template <typename T, int L, int E>
__global__ void __launch_bounds__(ROW_THREADS) k_norm_row(NormArgs a, Scores<T> in, Scores<T> out) {
    constexpr int R = ROW_THREADS / L;
    const int l = threadIdx.x & (L - 1), K = a.k;
    const long long n0 = blockIdx.x * (long long)R + threadIdx.x / L, n = min(n0, a.n - 1ll);
    float x[E];
    {
        const T *from = in.at(n, l);
        T raw[E];
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (l + j * L < K) raw[j] = from[(long long)j * L * in.cls];
#pragma unroll
        for (int j = 0; j < E; ++j) x[j] = l + j * L < K ? score_f32(raw[j]) : minus_inf();
    }
    float s = 0;
    int c = 0;
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (there(x[j])) { s += x[j]; ++c; }
    s = lanes_sum<L>(s); c = lanes_sum<L>(c);
    const float inv = 1.f / (float)max(c, 1), mean = s * inv;
    float q = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const float d = __fsub_rn(x[j], mean);
        if (there(x[j])) q = __fmaf_rn(d, d, q);
    }
    q = lanes_sum<L>(q);
    const float rstd = c ? 1.f / sqrtf(q * inv + a.eps) : 0.f;
    if (n0 != n) return;
    if (l == 0) {
        if (a.mean) a.mean[n] = mean;
        if (a.rstd) a.rstd[n] = rstd;
    }
    T *to = out.at(n, l);
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (l + j * L < K) {
            const float y = __fsub_rn(x[j], mean) * rstd;
            to[(long long)j * L * out.cls] = score_from<T>(!there(x[j]) ? x[j] : __fmaf_rn(y, a.gain ? a.gain[l + j * L] : 1.f, a.bias ? a.bias[l + j * L] : 0.f));
        }
}

template <int V> __device__ __forceinline__ void read_floats(const float *p, float none, float (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = p ? __ldg(p) : none;
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const float4 f = p ? __ldg(reinterpret_cast<const float4 *>(p + i)) : make_float4(none, none, none, none);
            v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        }
    }
}

// sums of M numbers over a block of TH threads, the same in all of them; all threads, with two barriers
template <int TH, int M> struct LongSums {
    float part[TH / 32][M], sum[M];
};
template <int TH, int M> __device__ __forceinline__ void long_sums(LongSums<TH, M> &sh, float (&v)[M]) {
    constexpr int W = TH / 32, PER = 32 / M;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float s = sums_spread<M>(v);
    if (lane % PER == 0) sh.part[warp][lane / PER] = s;
    __syncthreads();
    if (warp < M) {
        const float t = lanes_sum<W>(sh.part[lane & (W - 1)][warp]);
        if (lane == 0) sh.sum[warp] = t;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < M; ++m) v[m] = sh.sum[m];
}

// R rows at a time: gains and biases are read once for all of them (for one row of 16-bit scores they are four times its bytes, from the L2 cache),
// and barriers and exchanges are shared.  A row whose sum is finite holds no -inf, so only the others look at every score whether it is there.
// 2048 x 65536 in 16 bits with gain and bias: 149 us (floor 82), bound by waiting for loads and for the cluster; one row at a time 168.
template <int TH, int R> struct LongShared {
    LongSums<TH, R> sum, square;
    float part[TH / 32], moments[R][3], of_row[R][2];
};
template <typename T, int TH, int P, int R, bool EVEN, bool FULL>
__device__ __forceinline__ void norm_long(const NormArgs &a, const Scores<T> &in, const Scores<T> &out, LongShared<TH, R> &sh) {
    typedef Hold<T, TH, P, EVEN> H;
    constexpr int V = H::V;
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long n0 = (long long)(blockIdx.x / C) * R;
    const int lo = rank * H::CELLS, cells = FULL ? H::CELLS : min(a.k - lo, H::CELLS), rows = (int)min((long long)R, a.n - n0);   // (no block is without a cell)
    H x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) x[r].read(in.at(n0 + min(r, rows - 1), lo), cells);
    auto each = [&](int r, auto &&f) {
#pragma unroll
        for (int u = 0; u < P; ++u)
            if (FULL || H::first(u) < cells) {
                float v[V];
                x[r].get(u, v);
                f(v);
            }
    };
    float mean[R], square[R], count[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float2 s = make_float2(0.f, 0.f);
        each(r, [&](const float (&v)[V]) {
            if constexpr (V == 1) s.x += v[0];
            else {
#pragma unroll
                for (int i = 0; i < V; i += 2) s = add2(s, make_float2(v[i], v[i + 1]));
            }
        });
        mean[r] = s.x + s.y;
    }
    long_sums<TH>(sh.sum, mean);
    bool masked = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        count[r] = (float)cells;
        masked |= !finite(mean[r]);
    }
    if (masked) {   // (the same in all threads)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (finite(mean[r])) continue;
            float s = 0, c = 0;
            each(r, [&](const float (&v)[V]) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (there(v[i])) { s += v[i]; c += 1.f; }
            });
            mean[r] = block_sum<TH / 32>(s, sh.part);
            count[r] = block_sum<TH / 32>(c, sh.part);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        mean[r] *= 1.f / fmaxf(count[r], 1.f);
        const float2 m = make_float2(-mean[r], -mean[r]);
        float2 s = make_float2(0.f, 0.f);
        if (!masked) {
            each(r, [&](const float (&v)[V]) {
                if constexpr (V == 1) {
                    const float d = __fsub_rn(v[0], mean[r]);
                    s.x = __fmaf_rn(d, d, s.x);
                } else {
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        const float2 d = add2(make_float2(v[i], v[i + 1]), m);
                        s = fma2(d, d, s);
                    }
                }
            });
        } else {
            each(r, [&](const float (&v)[V]) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = __fsub_rn(v[i], mean[r]);
                    if (there(v[i])) s.x = __fmaf_rn(d, d, s.x);
                }
            });
        }
        square[r] = s.x + s.y;
    }
    {   // of the parts' counts, means and squares those of the row; a warp per row
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const float s = sums_spread<R>(square);
        if (lane % (32 / R) == 0) sh.square.part[warp][lane / (32 / R)] = s;
        __syncthreads();
        if (warp < R) {
            const float t = lanes_sum<TH / 32>(sh.square.part[lane & (TH / 32 - 1)][warp]);
            if (lane == 0) {
                float m = mean[0], c = count[0];
#pragma unroll
                for (int r = 1; r < R; ++r)
                    if (warp == r) { m = mean[r]; c = count[r]; }
                sh.moments[warp][0] = c; sh.moments[warp][1] = m; sh.moments[warp][2] = t;
            }
            __syncwarp();
        }
        if (C > 1) cluster.sync();
        if (warp < R) {
            float c = 0, m = 0, q = 0;
            if (lane < C) {
                const float *o = C > 1 ? cluster.map_shared_rank(sh.moments[warp], lane) : sh.moments[warp];
                c = o[0]; m = o[1]; q = o[2];
            }
            const float all = lanes_sum<LONG_CLUSTER>(c), whole = lanes_sum<LONG_CLUSTER>(c * m) / fmaxf(all, 1.f), d = __fsub_rn(m, whole);
            const float sum = lanes_sum<LONG_CLUSTER>(c == 0.f ? 0.f : __fmaf_rn(c * d, d, q));
            if (lane == 0) {
                const float by = all != 0.f ? 1.f / sqrtf(sum / all + a.eps) : 0.f;
                sh.of_row[warp][0] = whole; sh.of_row[warp][1] = by;
                if (rank == 0 && warp < rows) {
                    if (a.mean) a.mean[n0 + warp] = whole;
                    if (a.rstd) a.rstd[n0 + warp] = by;
                }
            }
        }
        __syncthreads();
        if (C > 1) cluster_done();
    }
    float rstd[R];
#pragma unroll
    for (int r = 0; r < R; ++r) { mean[r] = sh.of_row[r][0]; rstd[r] = sh.of_row[r][1]; }
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (FULL || H::first(u) < cells) {
            constexpr int Q = V < 4 ? V : 4;   // (four at a time: fewer registers)
#pragma unroll
            for (int h = 0; h < V; h += Q) {
                float g[Q], b[Q];
                read_floats<Q>(a.gain ? a.gain + lo + H::first(u) + h : nullptr, 1.f, g);
                read_floats<Q>(a.bias ? a.bias + lo + H::first(u) + h : nullptr, 0.f, b);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    float f[Q];
                    x[r].get_some(u, h, f);
                    if (V == 1 || masked) {
#pragma unroll
                        for (int i = 0; i < Q; ++i)
                            if (there(f[i])) f[i] = __fmaf_rn(__fsub_rn(f[i], mean[r]) * rstd[r], g[i], b[i]);
                    } else {
                        const float2 m = make_float2(-mean[r], -mean[r]), by = make_float2(rstd[r], rstd[r]);
#pragma unroll
                        for (int i = 0; i + 1 < Q; i += 2) {
                            const float2 y = fma2(mul2(add2(make_float2(f[i], f[i + 1]), m), by), make_float2(g[i], g[i + 1]), make_float2(b[i], b[i + 1]));
                            f[i] = y.x; f[i + 1] = y.y;
                        }
                    }
                    x[r].set_some(u, h, f);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < rows) x[r].write(out.at(n0 + r, lo), u);
        }
    if (C > 1) cluster_wait();   // (no block leaves while another may still read its moments)
}
template <typename T, int TH, int P, int R, bool EVEN>
__global__ void __launch_bounds__(TH, 1024 / TH) k_norm_long(NormArgs a, Scores<T> in, Scores<T> out) {
    __shared__ LongShared<TH, R> sh;
    const int C = (int)cg::this_cluster().num_blocks();
    if (a.k == C * Hold<T, TH, P, EVEN>::CELLS) norm_long<T, TH, P, R, EVEN, true>(a, in, out, sh);
    else norm_long<T, TH, P, R, EVEN, false>(a, in, out, sh);
}

// ---- the way back ------------------------------------------------------------------------------
// Sums over the rows, for the gradients of gain and bias, are made by blocks that stay: each adds up what its rows give to a class in a
// register of the thread that has the class and puts the sum down at the end; a second kernel adds the blocks' sums in order.
constexpr int SHARES = 296, FEW_SHARES = 148 * 8;
inline int shares_of(int n, int k) {
    return (int)std::max(1ll, std::min<long long>({k <= 32 ? (long long)FEW_SHARES : (long long)SHARES, (n + 31ll) / 32, (1ll << 23) / k + 1}));
}

template <int W> struct BackShared {
    float4 v[2][W > 1 ? W : 1][33];   // (padded: a warp reads a column)
    float4 sum[2][32];
};
__device__ __forceinline__ float4 add4(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
// as over_warps, for three numbers
template <int W> __device__ __forceinline__ float4 over_warps(BackShared<W> &sh, int turn, float4 v) {
    if constexpr (W > 1) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        sh.v[turn][warp][lane] = v;
        __syncthreads();
        if constexpr (W <= 8) {
            v = sh.v[turn][0][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) v = add4(v, sh.v[turn][w][lane]);
        } else {
#pragma unroll
            for (int r = warp; r < 32; r += W) {
                float4 u = sh.v[turn][lane & (W - 1)][r];
#pragma unroll
                for (int o = W / 2; o > 0; o >>= 1)
                    u = add4(u, make_float4(__shfl_xor_sync(0xffffffffu, u.x, o), __shfl_xor_sync(0xffffffffu, u.y, o), __shfl_xor_sync(0xffffffffu, u.z, o), 0.f));
                if (lane == 0) sh.sum[turn][r] = u;
            }
            __syncthreads();
            v = sh.sum[turn][lane];
        }
    }
    return v;
}

// By class, up to 1024 classes: a lane has a row, W warps share its classes.  50003 x 250: 49 us (floor 23), 68 instructions per score.  What 32 rows give to a class is added across the lanes, which hold 32 sums
// then (16 of x g and of g each, or one kind after the other).
template <typename T, int E, int W, bool WEIGHTS>
__global__ void __launch_bounds__(W == 1 ? 128 : 32 * W, W == 1 ? 4 : W == 8 ? (E == 32 ? 2 : 4) : W == 16 ? (E == 16 ? 2 : 1) : 1)
    k_norm_backward_class(NormBackwardArgs a, Scores<T> grad, Scores<T> in, Scores<T> out) {
    constexpr int G = W == 1 ? 4 : 1;
    __shared__ BackShared<W> sh;
    __shared__ float groups[WEIGHTS && W == 1 ? 4 : 1][2][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, k0 = W == 1 ? 0 : warp * E, here = a.k - k0;
    const long long tiles = (a.n + 32ll * G - 1) / (32 * G);
    float acc[2] = {0.f, 0.f};
    int turn = 0;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long long n0 = (W == 1 ? tile * 4 + warp : tile) * 32 + lane, n = min(n0, a.n - 1ll);
        float x[E], g[E];
        read_classes<E>(in.at(n, k0), (int)in.cls, here, minus_inf(), x);
        read_classes<E>(grad.at(n, k0), (int)grad.cls, here, 0.f, g);
        const float mean = a.mean[n], rstd = a.rstd[n];
        const float *gain = a.gain ? a.gain + k0 : nullptr;
        auto gain_of = [&](int j) { return gain ? (j < here ? __ldg(gain + j) : 0.f) : 1.f; };
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        unsigned gone = 0;   // classes that the row may not have
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const bool is = there(x[j]);
            if (!is) gone |= 1u << j;
            x[j] = is ? __fsub_rn(x[j], mean) * rstd : 0.f;
            g[j] = is ? g[j] : 0.f;
            const float b = g[j] * gain_of(j);
            v.x += b;
            v.y = __fmaf_rn(b, x[j], v.y);
        }
        v.z = (float)(E - __popc(gone));
        v = over_warps(sh, turn, v);
        turn ^= 1;
        const float inv = 1.f / fmaxf(v.z, 1.f), c1 = v.x * inv, c2 = v.y * inv;
        if (n0 == n)
            write_classes<E>(out.at(n, k0), (int)out.cls, here, [&](int j) {
                return gone >> j & 1 ? 0.f : rstd * __fsub_rn(__fsub_rn(g[j] * gain_of(j), c1), x[j] * c2);
            });
        if constexpr (WEIGHTS) {
            if (n0 != n) {
#pragma unroll
                for (int j = 0; j < E; ++j) g[j] = 0.f;   // (a row that was read for another lane)
            }
            if constexpr (E <= 16) {
                float both[2 * E];
#pragma unroll
                for (int j = 0; j < E; ++j) { both[j] = g[j]; both[E + j] = g[j] * x[j]; }
                acc[0] += sums_spread<2 * E>(both);
            } else {
#pragma unroll
                for (int j = 0; j < E; ++j) x[j] *= g[j];
                acc[0] += sums_spread<E>(g);
                acc[1] += sums_spread<E>(x);
            }
        }
    }
    if constexpr (WEIGHTS) {
        float *to = a.work + blockIdx.x * 2ll * a.k;
        constexpr int M = E <= 16 ? 2 * E : E, PER = 32 / M;
        const int m = lane / PER, j = E <= 16 ? m % E : m, kind = E <= 16 ? m / E : 0;
        if constexpr (W == 1) {
            if (lane % PER == 0) {
                groups[warp][kind][j] = acc[0];
                if (E > 16) groups[warp][1][j] = acc[1];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 2 * a.k; i += 128) {
                const int which = i / a.k, c = i % a.k;
                to[i] = (groups[0][which][c] + groups[1][which][c]) + (groups[2][which][c] + groups[3][which][c]);
            }
        } else if (lane % PER == 0 && j < here) {
            to[kind * (long long)a.k + k0 + j] = acc[0];
            if (E > 16) to[a.k + k0 + j] = acc[1];
        }
    }
}

// By row, up to 1024 classes: L lanes have a row, E classes each, L apart.
template <typename T, int L, int E, bool WEIGHTS>
__global__ void __launch_bounds__(ROW_THREADS) k_norm_backward_row(NormBackwardArgs a, Scores<T> grad, Scores<T> in, Scores<T> out) {
    constexpr int R = ROW_THREADS / L;
    __shared__ float sums[WEIGHTS ? 2 * L * E : 1];
    const int l = threadIdx.x & (L - 1);
    float to_bias[E], to_gain[E];
#pragma unroll
    for (int j = 0; j < E; ++j) to_bias[j] = to_gain[j] = 0.f;
    for (long long first = blockIdx.x * (long long)R; first < a.n; first += gridDim.x * (long long)R) {
        const long long n0 = first + threadIdx.x / L, n = min(n0, a.n - 1ll);
        float x[E], g[E];
        {
            const T *xs = in.at(n, l), *gs = grad.at(n, l);
            T rx[E], rg[E];
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (l + j * L < a.k) { rx[j] = xs[(long long)j * L * in.cls]; rg[j] = gs[(long long)j * L * grad.cls]; }
#pragma unroll
            for (int j = 0; j < E; ++j) {
                x[j] = l + j * L < a.k ? score_f32(rx[j]) : minus_inf();
                g[j] = l + j * L < a.k ? score_f32(rg[j]) : 0.f;
            }
        }
        const float mean = a.mean[n], rstd = a.rstd[n];
        auto gain_of = [&](int j) { return a.gain && l + j * L < a.k ? __ldg(a.gain + l + j * L) : 1.f; };
        unsigned gone = 0;
        float s = 0, sx = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const bool is = there(x[j]);
            if (!is) gone |= 1u << j;
            x[j] = is ? __fsub_rn(x[j], mean) * rstd : 0.f;
            g[j] = is ? g[j] : 0.f;
            const float b = g[j] * gain_of(j);
            s += b;
            sx = __fmaf_rn(b, x[j], sx);
        }
        const float inv = 1.f / (float)max(1, lanes_sum<L>(E - __popc(gone))), c1 = lanes_sum<L>(s) * inv, c2 = lanes_sum<L>(sx) * inv;
        if (n0 == n) {
            T *to = out.at(n, l);
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (l + j * L < a.k) to[(long long)j * L * out.cls] = score_from<T>(gone >> j & 1 ? 0.f : rstd * __fsub_rn(__fsub_rn(g[j] * gain_of(j), c1), x[j] * c2));
            if (WEIGHTS) {
#pragma unroll
                for (int j = 0; j < E; ++j) { to_bias[j] += g[j]; to_gain[j] = __fmaf_rn(g[j], x[j], to_gain[j]); }
            }
        }
    }
    if constexpr (WEIGHTS) {
        // lanes that have the same classes, then the warps one after the other
#pragma unroll
        for (int j = 0; j < E; ++j)
#pragma unroll
            for (int o = L; o < 32; o <<= 1) {
                to_bias[j] += __shfl_xor_sync(0xffffffffu, to_bias[j], o);
                to_gain[j] += __shfl_xor_sync(0xffffffffu, to_gain[j], o);
            }
        for (int w = 0; w < ROW_WARPS; ++w) {
            if ((int)(threadIdx.x >> 5) == w && (threadIdx.x & 31) < L) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    float *b = sums + l + j * L, *g = b + L * E;
                    *b = w ? *b + to_bias[j] : to_bias[j];
                    *g = w ? *g + to_gain[j] : to_gain[j];
                }
            }
            __syncthreads();
        }
        for (int k = threadIdx.x; k < a.k; k += ROW_THREADS) {
            a.work[blockIdx.x * 2ll * a.k + k] = sums[k];
            a.work[(blockIdx.x * 2ll + 1) * a.k + k] = sums[L * E + k];
        }
    }
}

// Long rows: a cluster of up to 8 blocks (or one) takes row after row, each block the same part of every row; the next row is on its way while this one is
// worked on.  Two scores of a thread go through each instruction.  A score of -inf makes the row's second sum infinite or NaN; only then is
// every score looked at whether it is there (and in the next row from the start).  4096 x 8191 in 16 bits: 88 us (floor 31), 29 instructions per
// score by 8 warps of 254 registers; 16 scores a thread of 512 took 100, the next row of single scores in registers 176.
// Rows that begin anywhere come through shared memory, by asynchronous copies of 16 bytes and a few single scores, two rows ahead; the others
// through registers, one row ahead.
// What a thread has of scores and gradients: as it was read, or (single scores in 16 bits) both of a class in one register.
template <typename T, int TH, int P, bool EVEN> struct Both {
    typedef Hold<T, TH, P, EVEN> H;
    static constexpr int V = H::V, E = H::E;
    static constexpr bool JOINED = !EVEN && sizeof(T) == 2;
    H x, g;
    unsigned both[JOINED ? P : 1];
    // single scores, from shared memory
    __device__ __forceinline__ void take(const T *xs, const T *gs, int cells) {
#pragma unroll
        for (int u = 0; u < P; ++u) {
            const int at = min(H::first(u), cells - 1);   // (behind the last class: another one, which counts for nothing)
            if constexpr (JOINED) both[u] = (unsigned)*reinterpret_cast<const unsigned short *>(xs + at) | (unsigned)*reinterpret_cast<const unsigned short *>(gs + at) << 16;
            else { x.one[u] = xs[at]; g.one[u] = gs[at]; }
        }
    }
    __device__ __forceinline__ static float2 split(unsigned v) {
        Pack<T> pack;
        pack.bits = make_uint4(v, 0, 0, 0);
        float f[Pack<T>::V];
        pack.unpack(f);
        return make_float2(f[0], f[1]);
    }
    // the thread's scores i and i + 1 (i even) and their gradients
    __device__ __forceinline__ void pair(int i, float2 &v, float2 &w) const {
        if constexpr (JOINED) {
            const float2 a = split(both[i]), b = split(both[i + 1]);
            v = make_float2(a.x, b.x); w = make_float2(a.y, b.y);
        } else if constexpr (EVEN) {
            float a[V], b[V];
            x.get(i / V, a);
            g.get(i / V, b);
            v = make_float2(a[i % V], a[i % V + 1]); w = make_float2(b[i % V], b[i % V + 1]);
        } else {
            v = make_float2(score_f32(x.one[i]), score_f32(x.one[i + 1])); w = make_float2(score_f32(g.one[i]), score_f32(g.one[i + 1]));
        }
    }
    static __device__ __forceinline__ int cell(int i) { return EVEN ? H::first(i / V) + i % V : H::first(i); }
};

__device__ __forceinline__ void copy_async16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// rows in shared memory at a time
template <typename T, int CELLS> constexpr int LONG_STAGES = CELLS * (int)sizeof(T) <= 32768 ? 3 : 1;
template <typename T, int CELLS> constexpr size_t LONG_RING = 2 * (size_t)LONG_STAGES<T, CELLS> * (CELLS * sizeof(T) + 16);

template <typename T, int TH, int P, bool EVEN, bool WEIGHTS>
__global__ void __launch_bounds__(TH) k_norm_backward_long(NormBackwardArgs a, Scores<T> grad, Scores<T> in, Scores<T> out) {
    typedef Both<T, TH, P, EVEN> B;
    typedef typename B::H H;
    constexpr int V = B::V, E = B::E, W = TH / 32;
    __shared__ float4 parts[2][W], block[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lo = rank * H::CELLS, cells = min(a.k - lo, H::CELLS);
    const long long step = gridDim.x / C;
    float2 to_bias[WEIGHTS ? E / 2 : 1], to_gain[WEIGHTS ? E / 2 : 1], gain[E / 2];
#pragma unroll
    for (int j = 0; j < (WEIGHTS ? E / 2 : 1); ++j) to_bias[j] = to_gain[j] = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < E; i += 2) {   // (0 behind the last class: what is read there adds nothing)
        const int k0 = B::cell(i), k1 = B::cell(i + 1);
        gain[i / 2] = make_float2(k0 < cells ? a.gain ? a.gain[lo + k0] : 1.f : 0.f, k1 < cells ? a.gain ? a.gain[lo + k1] : 1.f : 0.f);
    }
    B have;
    H next_x, next_g;
    constexpr int STAGES = LONG_STAGES<T, H::CELLS>;
    extern __shared__ __align__(16) unsigned char room[];   // (not EVEN) per stage: a row's scores and gradients, placed as they lie to 16 bytes
    T *const ring = reinterpret_cast<T *>(room);
    constexpr int LINE = H::CELLS + 16 / (int)sizeof(T);
    auto shift = [](const T *p) { return (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T)); };
    T single[2];                    // the few scores around the packs of the row asked for last, on their way
    T *single_to[2] = {nullptr, nullptr};
    auto settle_single = [&] {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (single_to[i]) { *single_to[i] = single[i]; single_to[i] = nullptr; }
    };
    auto fetch = [&](long long n, int stage) {
        const T *xs = in.at(n, lo), *gs = grad.at(n, lo);
        if constexpr (EVEN) {
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const int at = min(H::first(u), cells - V);   // (behind the last class: another one, which counts for nothing)
                next_x.w[u].bits = *reinterpret_cast<const uint4 *>(xs + at);
                next_g.w[u].bits = *reinterpret_cast<const uint4 *>(gs + at);
            }
        } else {
            settle_single();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const T *from = i ? gs : xs;
                T *to = ring + (2 * stage + i) * LINE + shift(from);
                const Part<T> part(from, 0, cells);
                const uint4 *body = part.body();
                for (int c = threadIdx.x; c < part.packs; c += TH) copy_async16(reinterpret_cast<uint4 *>(to + part.head) + c, body + c);
                if ((int)threadIdx.x < part.head + part.tail) {
                    const int at = part.single(threadIdx.x);
                    single[i] = from[at];
                    single_to[i] = to + at;
                }
            }
            copies_commit();
        }
    };
    long long n = blockIdx.x / C;
    if constexpr (EVEN) {
        if (n < a.n) fetch(n, 0);
    } else {
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) {
            if (n + i * step < a.n) fetch(n + i * step, i);
            else copies_commit();
        }
    }
    int turn = 0, stage = 0;
    bool care = false;
    for (; n < a.n; n += step) {
        if constexpr (EVEN) {
#pragma unroll
            for (int u = 0; u < P; ++u) { have.x.w[u] = next_x.w[u]; have.g.w[u] = next_g.w[u]; }
            if (n + step < a.n) fetch(n + step, 0);
        } else {
            // the row that this block worked on last has left its place: all threads have passed the barrier of its sums
            const long long ahead = n + (STAGES - 1) * step;
            const int to = stage == 0 ? STAGES - 1 : stage - 1;
            if (ahead < a.n) fetch(ahead, to);
            else { settle_single(); copies_commit(); }
            if (STAGES == 1) settle_single();
            copies_wait<STAGES - 1>();
            __syncthreads();
            const T *xs = in.at(n, lo), *gs = grad.at(n, lo);
            have.take(ring + 2 * stage * LINE + shift(xs), ring + (2 * stage + 1) * LINE + shift(gs), cells);
            stage = stage == STAGES - 1 ? 0 : stage + 1;
        }
        const float mean = a.mean[n], rstd = a.rstd[n];
        const float2 minus_mean = make_float2(-mean, -mean), by = make_float2(rstd, rstd);
        auto total = [&](float (&v)[4]) {
            const float s = sums_spread<4>(v);
            if ((lane & 7) == 0) reinterpret_cast<float *>(&parts[turn][warp])[lane >> 3] = s;
            __syncthreads();
            float4 sum;
            if (C > 1) {
                if (warp == 0) {
                    const float4 p = parts[turn][lane & (W - 1)];
                    const float4 all = make_float4(lanes_sum<W>(p.x), lanes_sum<W>(p.y), lanes_sum<W>(p.z), 0.f);
                    if (lane == 0) block[turn] = all;
                }
                cluster.sync();
                const float4 p = lane < C ? *cluster.map_shared_rank(&block[turn], lane) : make_float4(0.f, 0.f, 0.f, 0.f);
                sum = make_float4(warp_sum(p.x), warp_sum(p.y), warp_sum(p.z), 0.f);
            } else {
                const float4 p = parts[turn][lane & (W - 1)];
                sum = make_float4(lanes_sum<W>(p.x), lanes_sum<W>(p.y), lanes_sum<W>(p.z), 0.f);
            }
            turn ^= 1;
            return sum;
        };
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (!care) {
            float2 s = make_float2(0.f, 0.f), sx = s;
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                float2 v, w;
                have.pair(i, v, w);
                const float2 hat = mul2(add2(v, minus_mean), by), b = mul2(w, gain[i / 2]);
                s = add2(s, b);
                sx = fma2(b, hat, sx);
            }
            float v[4] = {s.x + s.y, sx.x + sx.y, 0.f, 0.f};
            sum = total(v);
            sum.z = (float)a.k;
        }
        if (care || !finite(sum.y)) {   // (the same in all threads)
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                float2 x, w;
                have.pair(i, x, w);
                auto one = [&](float f, float g, float its, int k) {
                    if (k < cells && there(f)) {
                        const float b = g * its;
                        v[0] += b;
                        v[1] = __fmaf_rn(b, __fsub_rn(f, mean) * rstd, v[1]);
                        v[2] += 1.f;
                    }
                };
                one(x.x, w.x, gain[i / 2].x, B::cell(i));
                one(x.y, w.y, gain[i / 2].y, B::cell(i + 1));
            }
            sum = total(v);
            care = sum.z != (float)a.k;
        }
        // rstd (b - mean(b) - hat mean(b hat))
        const float inv = rstd / fmaxf(sum.z, 1.f), c1 = -sum.x * inv, c2 = -sum.y * inv;
        const float2 m1 = make_float2(c1, c1), m2 = make_float2(c2, c2);
        T *to = out.at(n, lo) + H::first(0);
        const int behind = cells - H::first(0);   // cells from this thread's first one on
        auto write = [&](auto with_care) {
            constexpr bool CARE = decltype(with_care)::value;
#pragma unroll
            for (int u = 0; u < (EVEN ? P : P / 2); ++u) {
                constexpr int N = EVEN ? V : 2;
                float r[N];
#pragma unroll
                for (int i = u * N; i < u * N + N; i += 2) {
                    float2 v, w;
                    have.pair(i, v, w);
                    float2 hat = mul2(add2(v, minus_mean), by), g = w;
                    if (CARE) {
                        if (!there(v.x)) hat.x = g.x = 0.f;
                        if (!there(v.y)) hat.y = g.y = 0.f;
                    }
                    float2 f = fma2(hat, m2, fma2(mul2(g, gain[i / 2]), by, m1));
                    if (CARE) {
                        if (!there(v.x)) f.x = 0.f;
                        if (!there(v.y)) f.y = 0.f;
                    }
                    r[i - u * N] = f.x; r[i - u * N + 1] = f.y;
                    if constexpr (WEIGHTS) {
                        to_bias[i / 2] = add2(to_bias[i / 2], g);
                        to_gain[i / 2] = fma2(g, hat, to_gain[i / 2]);
                    }
                }
                if constexpr (EVEN) {
                    if (u * TH * V < behind) {
                        Pack<T> pack;
                        pack.pack(r);
                        *reinterpret_cast<uint4 *>(to + u * TH * V) = pack.bits;
                    }
                } else {
                    if (2 * u * TH < behind) to[2 * u * TH] = score_from<T>(r[0]);
                    if ((2 * u + 1) * TH < behind) to[(2 * u + 1) * TH] = score_from<T>(r[1]);
                }
            }
        };
        care ? write(std::true_type{}) : write(std::false_type{});
    }
    if constexpr (WEIGHTS) {
        float *bias = a.work + (blockIdx.x / C) * 2ll * a.k + lo, *gains = bias + a.k;
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const int k0 = B::cell(i), k1 = B::cell(i + 1);
            if (k0 < cells) { bias[k0] = to_bias[i / 2].x; gains[k0] = to_gain[i / 2].x; }
            if (k1 < cells) { bias[k1] = to_bias[i / 2].y; gains[k1] = to_gain[i / 2].y; }
        }
    }
    if (C > 1) {   // (no block leaves while another may still read its sums)
        cluster_done();
        cluster_wait();
    }
}

// Any strides: a block sums a share of the rows for 32 classes.
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
// The sums of all blocks: a warp takes every eighth, what the warps have is added in order.
__global__ void __launch_bounds__(ROW_THREADS) k_norm_weights_join(NormBackwardArgs a, int shares) {
    __shared__ double sums[ROW_WARPS][32];
    chain_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long i = blockIdx.x * 32ll + lane;
    double t = 0;
    if (i < 2ll * a.k) {
#pragma unroll 8
        for (int s = warp; s < shares; s += ROW_WARPS) t += (double)a.work[s * 2ll * a.k + i];
    }
    sums[warp][lane] = t;
    __syncthreads();
    if (warp == 0 && i < 2ll * a.k) {
        for (int w = 1; w < ROW_WARPS; ++w) t += sums[w][lane];
        if (i < a.k) a.to_bias[i] = (float)t;
        else a.to_gain[i - a.k] = (float)t;
    }
}
}  // namespace

// f(L, E) for kernels by row: E classes of each of L lanes
template <typename F> void by_row_sizes(int k, F &&f) {
    using std::integral_constant;
    if (k <= 4) f(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    else if (k <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (k <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (k <= 32) f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (k <= 64) f(integral_constant<int, 32>{}, integral_constant<int, 2>{});
    else if (k <= 128) f(integral_constant<int, 32>{}, integral_constant<int, 4>{});
    else if (k <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (k <= 512) f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
    else f(integral_constant<int, 32>{}, integral_constant<int, 32>{});
}
constexpr int ROW_MOST = 1024;   // classes of a row that a warp's registers hold

void scores_norm(const NormArgs &a, cudaStream_t stream) {
    if (a.n == 0) return;
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        const Scores<T> in = scores_of<T>(a.in), out = scores_of<T>(a.out);
        const bool by_class = (in.row < in.cls && out.row < out.cls) || a.in.one_by_class;
        if (by_class && a.k <= SCORES_CLASS_MOST && std::max(in.cls, out.cls) <= INT_MAX) {
            by_class_sizes(a.k, [&](auto e, auto w) {
                constexpr int E = decltype(e)::value, W = decltype(w)::value;
                const long long rows = W == 1 ? 128 : 32;
                auto kern = a.gain || a.bias ? k_norm_class<T, E, W, true> : k_norm_class<T, E, W, false>;
                kern<<<(unsigned)((a.n + rows - 1) / rows), W == 1 ? 128 : 32 * W, 0, stream>>>(a, in, out);
            });
            return;
        }
        if (a.k <= ROW_MOST) {
            by_row_sizes(a.k, [&](auto l, auto e) {
                constexpr int L = decltype(l)::value, E = decltype(e)::value;
                const long long rows = ROW_THREADS / L;
                k_norm_row<T, L, E><<<(unsigned)((a.n + rows - 1) / rows), ROW_THREADS, 0, stream>>>(a, in, out);
            });
            return;
        }
        if (in.cls == 1 && out.cls == 1) {
            const bool even = a.k % Pack<T>::V == 0 && on_16(in.p, in.row, sizeof(T)) && on_16(out.p, out.row, sizeof(T)) && on_16(a.gain, 0, 4) && on_16(a.bias, 0, 4);
            bool done = false;
            // Parts of a row that 512 threads hold, and several rows at a time where the rows are many: the smaller parts first, which need more blocks
            // for a row (at most LONG_CLUSTER) and hold more rows.
            auto go = [&](auto th, auto p, auto rows, auto ev) {
                constexpr bool EVEN = decltype(ev)::value;
                constexpr int TH = decltype(th)::value, P = decltype(p)::value, R = decltype(rows)::value;
                const int c = (a.k + Hold<T, TH, P, EVEN>::CELLS - 1) / Hold<T, TH, P, EVEN>::CELLS;
                if (done || c > LONG_CLUSTER || (R > 1 && (long long)a.n * c < 2 * 148 * R)) return;
                launch_long(k_norm_long<T, TH, P, R, EVEN>, (a.n + R - 1) / R, c, TH, stream, 0, a, in, out);
                done = true;
            };
            using std::integral_constant;
            auto all = [&](auto ev) {
                constexpr int S = decltype(ev)::value ? 2 : 8;   // packs of a quarter of what a thread holds
                go(integral_constant<int, 256>{}, integral_constant<int, S>{}, integral_constant<int, 4>{}, ev);
                go(integral_constant<int, 256>{}, integral_constant<int, S>{}, integral_constant<int, 1>{}, ev);
                go(integral_constant<int, 256>{}, integral_constant<int, 2 * S>{}, integral_constant<int, 2>{}, ev);
                go(integral_constant<int, 256>{}, integral_constant<int, 2 * S>{}, integral_constant<int, 1>{}, ev);
                go(integral_constant<int, 256>{}, integral_constant<int, 4 * S>{}, integral_constant<int, 1>{}, ev);
                go(integral_constant<int, 512>{}, integral_constant<int, 4 * S>{}, integral_constant<int, 1>{}, ev);
            };
            even ? all(std::true_type{}) : all(std::false_type{});
            if (done) return;
        }
        k_norm_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, in, out);
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
    const int most = shares_of(a.n, a.k);
    int shares = 0;   // blocks that have put sums down
    by_type(a.in.type, [&](auto t) {
        using T = decltype(t);
        const Scores<T> grad = scores_of<T>(a.grad), in = scores_of<T>(a.in), out = scores_of<T>(a.out);
        const bool weights = a.to_gain != nullptr, by_class = (in.row < in.cls && grad.row < grad.cls && out.row < out.cls) || a.in.one_by_class;
        using std::integral_constant;
        if (by_class && a.k <= SCORES_CLASS_MOST && std::max({in.cls, grad.cls, out.cls}) <= INT_MAX) {
            auto go = [&](auto e, auto w) {
                constexpr int E = decltype(e)::value, W = decltype(w)::value;
                const long long rows = W == 1 ? 128 : 32;
                const int blocks = (int)std::min<long long>((a.n + rows - 1) / rows, most);
                auto kern = weights ? k_norm_backward_class<T, E, W, true> : k_norm_backward_class<T, E, W, false>;
                kern<<<blocks, W == 1 ? 128 : 32 * W, 0, stream>>>(a, grad, in, out);
                shares = blocks;
            };
            // 129 to 256 classes: 16 warps with 16 classes each rather than 8 with 32, whose scores and gradients leave room for two blocks on an SM.  16
            // and 8 warps (us): 50003 x 130 40 and 41, 200 46 and 47, 250 50 and 53, in 16 bits 150 42 and 50, 250 44 and 51; with all of 256 classes 50 and 47.
            if (a.k > 128 && a.k <= 256) go(integral_constant<int, 16>{}, integral_constant<int, 16>{});
            else by_class_sizes(a.k, go);
            return;
        }
        if (a.k <= ROW_MOST) {
            by_row_sizes(a.k, [&](auto l, auto e) {
                constexpr int L = decltype(l)::value, E = decltype(e)::value;
                const long long rows = ROW_THREADS / L;
                const int blocks = (int)std::min<long long>((a.n + rows - 1) / rows, most);
                auto kern = weights ? k_norm_backward_row<T, L, E, true> : k_norm_backward_row<T, L, E, false>;
                kern<<<blocks, ROW_THREADS, 0, stream>>>(a, grad, in, out);
                shares = blocks;
            });
            return;
        }
        bool done = false, summed = false;
        if (in.cls == 1 && grad.cls == 1 && out.cls == 1) {
            const bool even = a.k % Pack<T>::V == 0 && on_16(in.p, in.row, sizeof(T)) && on_16(grad.p, grad.row, sizeof(T)) && on_16(out.p, out.row, sizeof(T)) &&
                              on_16(a.gain, 0, 4);
            auto go = [&](auto th, auto p, auto ev, auto sums) {
                constexpr bool EVEN = decltype(ev)::value, SUMS = decltype(sums)::value;
                constexpr int TH = decltype(th)::value, P = decltype(p)::value;
                const int c = (a.k + Hold<T, TH, P, EVEN>::CELLS - 1) / Hold<T, TH, P, EVEN>::CELLS;
                if (done || c > LONG_CLUSTER) return;
                // as many clusters as the SMs hold at once, and as there is room for sums
                const int rows = (int)std::min<long long>({(long long)a.n, std::max(1, 148 / c), (long long)most});
                constexpr size_t ring = EVEN ? 0 : LONG_RING<T, Hold<T, TH, P, EVEN>::CELLS>;
                if (!EVEN) allow_shared(k_norm_backward_long<T, TH, P, EVEN, SUMS>, ring);
                launch_long(k_norm_backward_long<T, TH, P, EVEN, SUMS>, rows, c, TH, stream, ring, a, grad, in, out);
                done = true;
                if (SUMS) { summed = true; shares = rows; }
            };
            auto all = [&](auto ev) {
                constexpr int S = decltype(ev)::value ? 16 / Pack<T>::V : 16, HALF = decltype(ev)::value || sizeof(T) == 4 ? 1 : 2;   // 16 scores
                if (weights) go(integral_constant<int, 512 / HALF>{}, integral_constant<int, S * HALF>{}, ev, std::true_type{});
                go(integral_constant<int, 512 / HALF>{}, integral_constant<int, S * HALF>{}, ev, std::false_type{});
                go(integral_constant<int, 512>{}, integral_constant<int, 2 * S>{}, ev, std::false_type{});
            };
            even ? all(std::true_type{}) : all(std::false_type{});
        }
        if (!done) k_norm_backward_any<T><<<a.n, ROW_THREADS, 0, stream>>>(a, grad, in, out);
        if (weights && !summed) {
            shares = most;
            k_norm_weights_any<T><<<dim3((a.k + 31) / 32, shares), ROW_THREADS, 0, stream>>>(a, grad, in, shares);
        }
    });
    if (a.to_gain) launch_after(k_norm_weights_join, dim3((2 * a.k + 31) / 32), dim3(ROW_THREADS), 0, stream, a, shares);
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
