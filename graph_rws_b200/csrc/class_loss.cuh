// What the losses over the class axis share (linear_ce.cu, distill.cu): element types in 16-byte pieces, running softmax
// statistics, the reduction of row losses and the factor a row's gradient gets from the loss's.
#pragma once

#include <type_traits>
#include <utility>

#include "grws_common.cuh"

namespace grws {
namespace cls {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float NEG_INF = -INFINITY;

enum Reduction : int { RED_NONE = GRWS_REDUCE_NONE, RED_MEAN = GRWS_REDUCE_MEAN, RED_SUM = GRWS_REDUCE_SUM };

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of a row as fp32 values and back
template <typename T> struct Piece;      // `largest` of several pieces ignores NaN, as fmaxf does
template <> struct Piece<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[4]) {
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
};
template <> struct Piece<__half> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) {
        const __half2 *h = reinterpret_cast<const __half2 *>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        uint4 u;
        __half2 *h = reinterpret_cast<__half2 *>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        return u;
    }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) {
        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 f = __bfloat1622float2(h[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
        uint4 u;
        __nv_bfloat162 *h = reinterpret_cast<__nv_bfloat162 *>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        return u;
    }
};

template <typename T, int N> __device__ __forceinline__ float largest(const uint4 (&u)[N]) {
    if constexpr (sizeof(T) == 4) {
        float m = NEG_INF;
#pragma unroll
        for (int i = 0; i < N; ++i)
            m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(u[i].x), __uint_as_float(u[i].y))), fmaxf(__uint_as_float(u[i].z), __uint_as_float(u[i].w)));
        return m;
    } else {
        // two 16-bit numbers at a time: a maximum is exact in any type
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        T2 m[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const T2 *h = reinterpret_cast<const T2 *>(&u[i]);
            m[i] = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
        }
#pragma unroll
        for (int i = 1; i < N; ++i) m[0] = __hmax2(m[0], m[i]);
        const float a = to_float(m[0].x), b = to_float(m[0].y);
        return fmaxf(a, b);
    }
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 numbers per instruction
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// exp2((a - m) c), exp2((b - m) c) with minus_m = (-m, -m) and cc = (c, c)
__device__ __forceinline__ uint64_t exp2_pair(float a, float b, uint64_t minus_m, uint64_t cc) {
    float x, y;
    unpair2(mul2(add2(pair2(a, b), minus_m), cc), x, y);
    return pair2(exp2_approx(x), exp2_approx(y));
}

// Running maximum m and sum s = sum exp(scale * (x - m)) of a part of a row, scale * ln 2 in `c`.  A part without entries,
// or of entries that are all -inf, is (-inf, 0); subtracting 0 instead of -inf keeps its exponentials at 0.
__device__ __forceinline__ float finite_or_zero(float m) { return m == NEG_INF ? 0.0f : m; }

__device__ __forceinline__ void join_stats(float &m, float &s, float m2, float s2, float c) {
    const float top = fmaxf(m, m2), safe = finite_or_zero(top);
    s = s * exp2_approx((m - safe) * c) + s2 * exp2_approx((m2 - safe) * c);
    m = top;
}

// (up to four chains of maxima and of sums: one chain's latency would be most of the time)
template <int N> __device__ __forceinline__ void add_values(float &m, float &s, const float (&v)[N], float c) {
    if constexpr (N < 16) {
        float top = m, t = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, v[i]);
        const float safe = finite_or_zero(top);
        if (top != m) { s *= exp2_approx((m - safe) * c); m = top; }
#pragma unroll
        for (int i = 0; i < N; ++i) t += exp2_approx((v[i] - safe) * c);
        s += t;
    } else {
        float top[4];
        uint64_t t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) { top[j] = v[j]; t[j] = 0; }
#pragma unroll
        for (int i = 4; i < N; ++i) top[i % 4] = fmaxf(top[i % 4], v[i]);
        top[0] = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), m);
        const float safe = finite_or_zero(top[0]);
        if (top[0] != m) { s *= exp2_approx((m - safe) * c); m = top[0]; }
        const uint64_t minus = pair2(-safe, -safe), cc = pair2(c, c);
#pragma unroll
        for (int i = 0; i < N; i += 2) t[i / 2 % 4] = add2(t[i / 2 % 4], exp2_pair(v[i], v[i + 1], minus, cc));
        float a, b;
        unpair2(add2(add2(t[0], t[1]), add2(t[2], t[3])), a, b);
        s += a + b;
    }
}

// the same for N pieces of a row as loaded.  (c v - c max would be one instruction instead of two, but is off by 2^-24 of
// c max: a row masked with the type's lowest value would sum up infinities.)
template <typename T, int N> __device__ __forceinline__ void add_pieces(float &m, float &s, const uint4 (&u)[N], float c) {
    constexpr int E = Piece<T>::E;
    const float top = fmaxf(m, largest<T, N>(u)), safe = finite_or_zero(top);
    if (top != m) { s *= exp2_approx((m - safe) * c); m = top; }
    const uint64_t minus = pair2(-safe, -safe), cc = pair2(c, c);
    uint64_t t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float v[E];
        Piece<T>::unpack(u[i], v);
        t[i] = exp2_pair(v[0], v[1], minus, cc);
#pragma unroll
        for (int e = 2; e < E; e += 2) t[i] = add2(t[i], exp2_pair(v[e], v[e + 1], minus, cc));
    }
#pragma unroll
    for (int i = 1; i < N; ++i) t[0] = add2(t[0], t[i]);
    float x, y;
    unpair2(t[0], x, y);
    s += x + y;
}

// Kernels of one call follow each other as programmatic dependents: the next one is launched while this one still runs, sets
// itself up and waits here before it touches memory.  Every kernel waits, so each may rely on all before it.  What lies in
// memory does change during a kernel's lifetime, then: whatever is read behind the wait is read by ordinary loads.  __ldg and
// pointers that are const and __restrict__ promise that it does not; such a load may be non-coherent, and may be moved
// ahead of the wait.  (A call's inputs are no exception: the kernel before the first one may be the last of another call,
// which lets its dependents start as early.)
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
inline int launch_next(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    GRWS_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
    return GRWS_OK;
}

// The integer at i of an array of 4- or 8-byte integers
__device__ __forceinline__ int64_t load_index(const void *p, int bytes, int64_t i) {
    return bytes == 8 ? (int64_t)static_cast<const long long *>(p)[i] : (int64_t)static_cast<const int *>(p)[i];
}

// Sum of two values over the block's threads, valid in thread 0; red holds 2 * 32 floats.
__device__ __forceinline__ void block_sum2(float &a, float &b, float *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
    if (lane == 0) { red[warp] = a; red[32 + warp] = b; }
    __syncthreads();
    if (warp == 0) {
        a = lane < warps ? red[lane] : 0.0f;
        b = lane < warps ? red[32 + lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { a += __shfl_xor_sync(0xffffffffu, a, o); b += __shfl_xor_sync(0xffffffffu, b, o); }
    }
    __syncthreads();
}

// loss = sum (or mean over the counted rows) of the blocks' partial sums [blocks][2] = (loss, counted rows), added in a fixed order
__device__ __forceinline__ void finish_loss(float sum, float count, int reduction, float *loss, float *count_out) {
    *loss = reduction == RED_MEAN ? sum / count : sum;       // no counted row: 0 / 0
    *count_out = count;
}
static __global__ void __launch_bounds__(512) loss_sum_kernel(const float2 *partial, int n, int reduction,
                                                              float *__restrict__ loss, float *__restrict__ count_out) {
    __shared__ float red[64];
    float a = 0.0f, b = 0.0f;
    wait_for_previous();
    for (int i = threadIdx.x; i < n; i += blockDim.x) { const float2 p = partial[i]; a += p.x; b += p.y; }
    block_sum2(a, b, red);
    if (threadIdx.x == 0) finish_loss(a, b, reduction, loss, count_out);
}

// Factor of all rows from the gradient of the reduced loss.  Without counted rows nothing has a gradient.
__device__ __forceinline__ float loss_factor(const float *grad_loss, const float *count, int reduction) {
    const float g = *grad_loss;
    if (reduction != RED_MEAN) return g;
    const float n = *count;
    return n > 0.0f ? g / n : 0.0f;
}

// Properties of the current device, read once
constexpr int MAX_DEVICES = 64;
inline int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < MAX_DEVICES ? dev : -1;
}
inline int sm_count() {
    static int known[MAX_DEVICES];
    const int dev = current_device();
    if (dev < 0) return 148;
    int sms = __atomic_load_n(&known[dev], __ATOMIC_RELAXED);
    if (sms == 0) {
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
        __atomic_store_n(&known[dev], sms, __ATOMIC_RELAXED);
    }
    return sms;
}

}  // namespace cls
}  // namespace grws
