// What the kernels that draw, learn from draws and standardise share: sums over lanes, long rows that a block or a cluster of blocks holds in its
// registers, sizes.
#pragma once
#include <cfloat>

#include "tgbm_scores.cuh"

namespace tgbm {

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= FLT_MAX; }
template <int L, typename V> __device__ __forceinline__ V lanes_sum(V v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int L> __device__ __forceinline__ float lanes_min(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int L> __device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    unsigned long long r, x = *reinterpret_cast<unsigned long long *>(&a), y = *reinterpret_cast<unsigned long long *>(&b), z = *reinterpret_cast<unsigned long long *>(&c);
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return *reinterpret_cast<float2 *>(&r);
}
// Sums of M numbers over a warp (M a power of two up to 32): lanes exchange half of what they hold until each holds one.  Lane l has the sum
// of number l / (32 / M).
template <int M, typename F> __device__ __forceinline__ F sums_spread(F (&v)[M]) {
    const int lane = threadIdx.x & 31;
    int o = 16;
#pragma unroll
    for (int m = M; m > 1; m >>= 1, o >>= 1) {
        const bool upper = lane & o;
#pragma unroll
        for (int i = 0; i < m / 2; ++i) {
            const F give = upper ? v[i] : v[i + m / 2], keep = upper ? v[i + m / 2] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    for (; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    return v[0];
}
// The last barrier of a kernel whose blocks have read one another's shared memory: none leaves before all have.  Nothing that was written is handed
// over by it (relaxed: a release would wait for all that the block has stored).
__device__ __forceinline__ void cluster_done() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

// ---- long rows: a block, or a cluster of blocks, each with a part of the row in its registers -------------------------------
// A thread's scores: packs of 16 bytes, TH packs apart (EVEN: rows, gains and results all begin on such boundaries), or single ones, TH apart.
constexpr int LONG_CLUSTER = 8;

template <typename T, int TH, int P, bool EVEN> struct Hold {
    static constexpr int V = EVEN ? Pack<T>::V : 1, E = P * V;
    static constexpr int CELLS = TH * E;   // of a block
    static __device__ __forceinline__ int first(int u) { return (u * TH + (int)threadIdx.x) * V; }
    Pack<T> w[EVEN ? P : 1];
    T one[EVEN ? 1 : P];
    __device__ __forceinline__ void read(const T *p, int cells) {   // cells: of the part (EVEN: whole packs)
#pragma unroll
        for (int u = 0; u < P; ++u)
            if (cells == CELLS || first(u) < cells) {
                if constexpr (EVEN) w[u].bits = *reinterpret_cast<const uint4 *>(p + first(u));   // (it may be written over later: no __ldg)
                else one[u] = p[first(u)];
            }
    }
    __device__ __forceinline__ void get(int u, float (&v)[V]) const {
        if constexpr (EVEN) w[u].unpack(v);
        else v[0] = score_f32(one[u]);
    }
    // largest of a thread's scores, NaN where one is
    __device__ __forceinline__ float largest(int cells) const {
        float high = minus_inf();
        auto larger = [](float a, float b) {
            float r;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
            return r;
        };
#pragma unroll
        for (int u = 0; u < P; ++u)
            if (cells == CELLS || first(u) < cells) {
                if constexpr (EVEN && sizeof(T) == 2) {
                    typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
                    const unsigned words[4] = {w[u].bits.x, w[u].bits.y, w[u].bits.z, w[u].bits.w};
                    const T2 v = __hmax2_nan(__hmax2_nan(*reinterpret_cast<const T2 *>(&words[0]), *reinterpret_cast<const T2 *>(&words[1])),
                                             __hmax2_nan(*reinterpret_cast<const T2 *>(&words[2]), *reinterpret_cast<const T2 *>(&words[3])));
                    high = larger(high, larger(score_f32(v.x), score_f32(v.y)));
                } else {
                    float v[V];
                    get(u, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) high = larger(high, v[i]);
                }
            }
        return high;
    }
    // least and largest of a thread's scores; NaN does not count
    __device__ __forceinline__ void range(int cells, float &low, float &high) const {
        low = -minus_inf(); high = minus_inf();
        if constexpr (EVEN && sizeof(T) == 2) {
            typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
            T2 lows, highs;
            bool some = false;
#pragma unroll
            for (int u = 0; u < P; ++u)
                if (cells == CELLS || first(u) < cells) {
                    const unsigned words[4] = {w[u].bits.x, w[u].bits.y, w[u].bits.z, w[u].bits.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const T2 v = *reinterpret_cast<const T2 *>(&words[i]);
                        lows = u + i == 0 ? v : __hmin2(lows, v);
                        highs = u + i == 0 ? v : __hmax2(highs, v);
                    }
                    some = true;
                }
            if (some) {
                low = fminf(fminf(low, score_f32(lows.x)), score_f32(lows.y));
                high = fmaxf(fmaxf(high, score_f32(highs.x)), score_f32(highs.y));
            }
        } else {
#pragma unroll
            for (int u = 0; u < P; ++u)
                if (cells == CELLS || first(u) < cells) {
                    float v[V];
                    get(u, v);
#pragma unroll
                    for (int i = 0; i < V; ++i) { low = fminf(low, v[i]); high = fmaxf(high, v[i]); }
                }
        }
    }
    // cells h to h + Q of pack u
    template <int Q> __device__ __forceinline__ void get_some(int u, int h, float (&v)[Q]) const {
        if constexpr (!EVEN) v[0] = score_f32(one[u]);
        else if constexpr (Q == V) w[u].unpack(v);
        else {
            float all[V];
            w[u].unpack(all);
#pragma unroll
            for (int i = 0; i < Q; ++i) v[i] = all[h + i];
        }
    }
    template <int Q> __device__ __forceinline__ void set_some(int u, int h, const float (&v)[Q]) {
        if constexpr (!EVEN) one[u] = score_from<T>(v[0]);
        else if constexpr (Q == V) w[u].pack(v);
        else {
            Pack<T> some;
            float all[V] = {};
#pragma unroll
            for (int i = 0; i < Q; ++i) all[i] = v[i];
            some.pack(all);
            if (h == 0) { w[u].bits.x = some.bits.x; w[u].bits.y = some.bits.y; }
            else { w[u].bits.z = some.bits.x; w[u].bits.w = some.bits.y; }
        }
    }
    __device__ __forceinline__ void write(T *p, int u) const {
        if constexpr (EVEN) *reinterpret_cast<uint4 *>(p + first(u)) = w[u].bits;
        else p[first(u)] = one[u];
    }
};
// f(E, W) for kernels with a lane per row, up to 1024 classes: E classes of each of W warps
template <typename F> inline void by_class_sizes(int k, F &&f) {
    using std::integral_constant;
    if (k <= 8) f(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    else if (k <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    else if (k <= 32) f(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    else if (k <= 64) f(integral_constant<int, 8>{}, integral_constant<int, 8>{});
    else if (k <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
    else if (k <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 8>{});
    else if (k <= 512) f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
    else f(integral_constant<int, 32>{}, integral_constant<int, 32>{});
}

inline bool on_16(const void *p, long long row, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row * size % 16 == 0; }

template <typename... P, typename... A>
void launch_long(void (*kernel)(P...), long long rows, int cluster, int threads, cudaStream_t stream, size_t smem, A &&...args) {
    TGBM_CHECK(rows * cluster < 1ll << 31, "too many rows of this length for one call");   // (rows that are all the same one take no memory)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * cluster)); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr; cfg.numAttrs = cluster > 1 ? 1 : 0;
    TGBM_CUDA(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}

}  // namespace tgbm
