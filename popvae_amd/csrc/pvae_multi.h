// Operators over all tensors of a model: the global gradient norm, clipping by it, and the Adam update with that clipping
// folded in.
//
//   n = sqrt(sum_t sum_i g_ti^2),  s = min(1, c / n),  g' = s g
//
// Two launches whatever the number of tensors (a table of PVM_MAXT tensors rides in the kernel arguments; more tensors take
// more launches): pvk_sumsq leaves one float64 partial sum per workgroup, and every workgroup of the second pass adds those
// partials up for itself, in one fixed order -- no atomics, no counter to reset, no third launch -- before it scales (or
// updates) its share.  Squares and sums are float64: no float32 square over- or underflows on the way, and at 4 bytes per
// element from memory the two float64 instructions per element cost nothing.  Bound by memory: 4 bytes per element for the
// norm, 4 + 4 more for the scaled copy, 28 for the update.
//   Measured: the norm of 1.03 GB of float32 in 164 us (6.3 TB/s), of 52 MB of bf16 in 11 us (4.6 TB/s); the scaled copy of
// those 52 MB in 19 us (5.5 TB/s); the update of 257M parameters (7.2 GB) in 1373 us (5.2 TB/s; a plain copy of 4 GB reaches 4.8
// with cached and 6.0 with nontemporal accesses).  A model of 3887 SNPs: 4 + 6 us for clipping, mostly launches, and 4 + 13 us
// for the update, whose 160 chunks leave CUs without work (its 33 MB would take 7 us at the copy's rate).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

enum { PVM_MAXT = 48, PVM_THREADS = 256, PVM_CHUNK = 8192, PVM_PARTS = 2048 };

typedef float pvm_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short pvm_u16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short pvm_u16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 pvm_f16x4 __attribute__((ext_vector_type(4)));
// the same where nothing but the elements' own alignment is known (a view, an odd row stride): memory is read and written 8 and
// 16 bytes at a time all the same, the hardware takes any address
typedef pvm_f32x4 pvm_f32x4_any __attribute__((aligned(4)));
typedef pvm_u16x4 pvm_u16x4_any __attribute__((aligned(2)));
typedef pvm_f16x4 pvm_f16x4_any __attribute__((aligned(2)));
typedef pvm_u16x8 pvm_u16x8_any __attribute__((aligned(2)));

struct PvmTab {  // elements [0, n) of tensor t are chunks first[t] .. first[t + 1) of PVM_CHUNK elements
    int count;
    int first[PVM_MAXT + 1];
    const void* a[PVM_MAXT];  // gradients
    void* b[PVM_MAXT];        // scaled copy / parameters
    float* m[PVM_MAXT];
    float* v[PVM_MAXT];
    int64_t n[PVM_MAXT];
    int tile[PVM_MAXT];            // pvae_tensor.tile of b, m and v
    unsigned char dt[PVM_MAXT];    // type of a
};

__device__ __forceinline__ float pvm_bf16(unsigned short u) { return __uint_as_float((unsigned)u << 16); }
// round to nearest even; a NaN keeps its upper half with a bit that stays set
__device__ __forceinline__ unsigned short pvm_to_bf16(float f) {
    const unsigned u = __float_as_uint(f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (unsigned short)((u >> 16) | 0x40u);
    return (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
__device__ __forceinline__ float pvm_load1(const void* p, int dt, int64_t i) {
    if (dt == 0) return static_cast<const float*>(p)[i];
    if (dt == 1) return pvm_bf16(static_cast<const unsigned short*>(p)[i]);
    return (float)static_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ pvm_f32x4 pvm_load4(const void* p, int dt, int64_t i) {
    if (dt == 0) return *reinterpret_cast<const pvm_f32x4_any*>(static_cast<const float*>(p) + i);
    if (dt == 1) {
        const pvm_u16x4 u = *reinterpret_cast<const pvm_u16x4_any*>(static_cast<const unsigned short*>(p) + i);
        return (pvm_f32x4){pvm_bf16(u.x), pvm_bf16(u.y), pvm_bf16(u.z), pvm_bf16(u.w)};
    }
    const pvm_f16x4 h = *reinterpret_cast<const pvm_f16x4_any*>(static_cast<const _Float16*>(p) + i);
    return (pvm_f32x4){(float)h.x, (float)h.y, (float)h.z, (float)h.w};
}
__device__ __forceinline__ void pvm_store1(void* p, int dt, int64_t i, float x) {
    if (dt == 0) static_cast<float*>(p)[i] = x;
    else if (dt == 1) static_cast<unsigned short*>(p)[i] = pvm_to_bf16(x);
    else static_cast<_Float16*>(p)[i] = (_Float16)x;
}
__device__ __forceinline__ void pvm_store4(void* p, int dt, int64_t i, pvm_f32x4 x) {
    if (dt == 0) *reinterpret_cast<pvm_f32x4_any*>(static_cast<float*>(p) + i) = x;
    else if (dt == 1)
        *reinterpret_cast<pvm_u16x4_any*>(static_cast<unsigned short*>(p) + i) =
            (pvm_u16x4){pvm_to_bf16(x.x), pvm_to_bf16(x.y), pvm_to_bf16(x.z), pvm_to_bf16(x.w)};
    else
        *reinterpret_cast<pvm_f16x4_any*>(static_cast<_Float16*>(p) + i) =
            (pvm_f16x4){(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
}

// sixteen bytes of a tensor and what they hold
template <int DT> struct PvmVec { enum { N = 8 }; typedef pvm_u16x8 V; typedef pvm_u16x8_any M; };
template <> struct PvmVec<0> { enum { N = 4 }; typedef pvm_f32x4 V; typedef pvm_f32x4_any M; };
template <int DT> __device__ __forceinline__ float pvm_get(typename PvmVec<DT>::V v, int e) {
    if constexpr (DT == 0) return v[e];
    else if constexpr (DT == 1) return pvm_bf16(v[e]);
    else return (float)__builtin_bit_cast(_Float16, (unsigned short)v[e]);
}
template <int DT> __device__ __forceinline__ void pvm_set(typename PvmVec<DT>::V& v, int e, float x) {
    if constexpr (DT == 0) v[e] = x;
    else if constexpr (DT == 1) v[e] = pvm_to_bf16(x);
    else v[e] = __builtin_bit_cast(unsigned short, (_Float16)x);
}
#define PVM_BY_TYPE(dt, CALL)                                   \
    switch (dt) {                                               \
        case 0: { constexpr int D_ = 0; CALL; } break;          \
        case 1: { constexpr int D_ = 1; CALL; } break;          \
        default: { constexpr int D_ = 2; CALL; } break;         \
    }

__device__ __forceinline__ int pvm_find(const PvmTab& T, int chunk) {  // the tensor of a chunk: first[t] <= chunk < first[t + 1]
    int lo = 0, hi = T.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (T.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// the workgroup's sum of one float64 per thread, in a fixed order, to every thread
__device__ __forceinline__ double pvm_block_sum(double s) {
    __shared__ double red[PVM_THREADS / 64];
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    double a = red[0];
    for (int i = 1; i < PVM_THREADS / 64; ++i) a += red[i];
    __syncthreads();
    return a;
}

// the sum of squares of a whole chunk (all its loads under way together) or of the end of a tensor
template <int DT> __device__ __forceinline__ double pvm_sumsq_chunk(const void* a, int64_t i0, int64_t i1) {
    typedef typename PvmVec<DT>::V V;
    typedef typename PvmVec<DT>::M M;
    enum { N = PvmVec<DT>::N, LOADS = PVM_CHUNK / N / PVM_THREADS };
    double s = 0.0;
    auto add = [&](V v) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const double x = pvm_get<DT>(v, e);
            s = fma(x, x, s);
        }
    };
    const M* p = reinterpret_cast<const M*>(static_cast<const char*>(a) + i0 * (16 / N)) + threadIdx.x;
    if (i1 - i0 == PVM_CHUNK) {
        V v[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) v[u] = p[u * PVM_THREADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) add(v[u]);
        return s;
    }
    const int whole = (int)(i1 - i0) / N;
    for (int u = threadIdx.x; u < whole; u += PVM_THREADS, p += PVM_THREADS) add(*p);
    for (int64_t i = i0 + (int64_t)whole * N + threadIdx.x; i < i1; i += PVM_THREADS) {
        const double x = pvm_load1(a, DT, i);
        s = fma(x, x, s);
    }
    return s;
}

__global__ __launch_bounds__(PVM_THREADS) void pvk_sumsq(const PvmTab T, double* __restrict__ part) {
    const int chunks = T.first[T.count];
    double s = 0.0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = pvm_find(T, c);
        const int64_t i0 = (int64_t)(c - T.first[t]) * PVM_CHUNK, i1 = min(T.n[t], i0 + PVM_CHUNK);
        PVM_BY_TYPE(T.dt[t], s += pvm_sumsq_chunk<D_>(T.a[t], i0, i1));
    }
    s = pvm_block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the norm from the partial sums, the same in every workgroup
__device__ __forceinline__ double pvm_norm(const double* __restrict__ part, int nparts) {
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += PVM_THREADS) s += part[i];
    return sqrt(pvm_block_sum(s));
}
// min(1, c / n); NaN where n is not finite
__device__ __forceinline__ float pvm_scale(double n, double c) {
    if (!(n < __builtin_inf())) return __builtin_nanf("");
    return n <= c ? 1.f : (float)(c / n);
}

__global__ __launch_bounds__(PVM_THREADS) void pvk_norm_final(const double* __restrict__ part, int nparts, float* __restrict__ norm) {
    const double n = pvm_norm(part, nparts);
    if (threadIdx.x == 0) *norm = (float)n;
}

template <int DT> __device__ __forceinline__ void pvm_scale_chunk(const void* a, void* b, int64_t i0, int64_t i1, float s) {
    typedef typename PvmVec<DT>::V V;
    typedef typename PvmVec<DT>::M M;
    enum { N = PvmVec<DT>::N, LOADS = PVM_CHUNK / N / PVM_THREADS };
    const M* p = reinterpret_cast<const M*>(static_cast<const char*>(a) + i0 * (16 / N)) + threadIdx.x;
    M* q = reinterpret_cast<M*>(static_cast<char*>(b) + i0 * (16 / N)) + threadIdx.x;
    auto scaled = [&](V v) {
        V o;
#pragma unroll
        for (int e = 0; e < N; ++e) pvm_set<DT>(o, e, pvm_get<DT>(v, e) * s);
        return o;
    };
    if (i1 - i0 == PVM_CHUNK) {
        V v[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) v[u] = p[u * PVM_THREADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) q[u * PVM_THREADS] = scaled(v[u]);
        return;
    }
    const int whole = (int)(i1 - i0) / N;
    for (int u = threadIdx.x; u < whole; u += PVM_THREADS, p += PVM_THREADS, q += PVM_THREADS) *q = scaled(*p);
    for (int64_t i = i0 + (int64_t)whole * N + threadIdx.x; i < i1; i += PVM_THREADS) pvm_store1(b, DT, i, pvm_load1(a, DT, i) * s);
}

__global__ __launch_bounds__(PVM_THREADS) void pvk_clip_apply(const PvmTab T, const double* __restrict__ part, int nparts, double max_norm,
                                                              float* __restrict__ norm) {
    const double n = pvm_norm(part, nparts);
    const float s = pvm_scale(n, max_norm);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const int chunks = T.first[T.count];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = pvm_find(T, c);
        if (s == 1.f && T.a[t] == T.b[t]) continue;  // in place and within the bound: every value stays as it is
        const int64_t i0 = (int64_t)(c - T.first[t]) * PVM_CHUNK, i1 = min(T.n[t], i0 + PVM_CHUNK);
        PVM_BY_TYPE(T.dt[t], pvm_scale_chunk<D_>(T.a[t], T.b[t], i0, i1, s));
    }
}

struct PvmAdam {
    double lr, b1, b2;
    float eps;
    int64_t step;
    const int* step_dev;
};

// lr sqrt(1 - b2^t) / (1 - b1^t) in float64; b^t by squaring
__device__ __forceinline__ float pvm_alpha(const PvmAdam& A) {
    int64_t t = A.step_dev ? (int64_t)*A.step_dev : A.step;
    double p1 = 1.0, p2 = 1.0, q1 = A.b1, q2 = A.b2;
    for (; t > 0; t >>= 1) {
        if (t & 1) { p1 *= q1; p2 *= q2; }
        q1 *= q1;
        q2 *= q2;
    }
    return (float)(A.lr * sqrt(1.0 - p2) / (1.0 - p1));
}

__device__ __forceinline__ void pvm_adam1(float& p, float& m, float& v, float g, float alpha, float c1, float c2, float eps) {
    m += (g - m) * c1;
    v += (g * g - v) * c2;
    p -= alpha * m / (sqrtf(v) + eps);
}

// four elements at a time, two groups under way: parameters and moments pass once, past the caches
template <int DT> __device__ __forceinline__ void pvm_adam_chunk(const void* a, float* p, float* m, float* v, int tile, int64_t i0, int64_t i1,
                                                                 float s, float alpha, float c1, float c2, float eps) {
    auto at = [&](int64_t i) { return tile ? i + i / tile * 2 * tile : i; };  // i / tile * 3 tile + i % tile
    const int whole = (int)(i1 - i0) / 4;
    auto step = [&](pvm_f32x4 g, int64_t j, pvm_f32x4 p4, pvm_f32x4 m4, pvm_f32x4 v4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float pe = p4[e], me = m4[e], ve = v4[e];
            pvm_adam1(pe, me, ve, g[e] * s, alpha, c1, c2, eps);
            p4[e] = pe; m4[e] = me; v4[e] = ve;
        }
        __builtin_nontemporal_store(p4, reinterpret_cast<pvm_f32x4_any*>(p + j));
        __builtin_nontemporal_store(m4, reinterpret_cast<pvm_f32x4_any*>(m + j));
        __builtin_nontemporal_store(v4, reinterpret_cast<pvm_f32x4_any*>(v + j));
    };
    auto ld = [](const float* q) -> pvm_f32x4 { return __builtin_nontemporal_load(reinterpret_cast<const pvm_f32x4_any*>(q)); };
    int u = threadIdx.x;
    for (; u + PVM_THREADS < whole; u += 2 * PVM_THREADS) {
        const int64_t e0 = i0 + 4 * u, e1 = e0 + 4 * PVM_THREADS, j0 = at(e0), j1 = at(e1);
        const pvm_f32x4 g0 = pvm_load4(a, DT, e0), p0 = ld(p + j0), m0 = ld(m + j0), v0 = ld(v + j0);
        const pvm_f32x4 g1 = pvm_load4(a, DT, e1), p1 = ld(p + j1), m1 = ld(m + j1), v1 = ld(v + j1);
        step(g0, j0, p0, m0, v0);
        step(g1, j1, p1, m1, v1);
    }
    for (; u < whole; u += PVM_THREADS) {
        const int64_t e0 = i0 + 4 * u, j0 = at(e0);
        step(pvm_load4(a, DT, e0), j0, ld(p + j0), ld(m + j0), ld(v + j0));
    }
    for (int64_t i = i0 + (int64_t)whole * 4 + threadIdx.x; i < i1; i += PVM_THREADS) {
        const int64_t j = at(i);
        pvm_adam1(p[j], m[j], v[j], pvm_load1(a, DT, i) * s, alpha, c1, c2, eps);
    }
}

__global__ __launch_bounds__(PVM_THREADS) void pvk_adam_apply(const PvmTab T, const double* __restrict__ part, int nparts, double clip_norm,
                                                              float* __restrict__ norm, const PvmAdam A) {
    float s = 1.f;
    if (nparts) {
        const double n = pvm_norm(part, nparts);
        if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
        if (clip_norm > 0.0) s = pvm_scale(n, clip_norm);
    }
    const float alpha = pvm_alpha(A), c1 = (float)(1.0 - A.b1), c2 = (float)(1.0 - A.b2), eps = A.eps;
    const int chunks = T.first[T.count];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = pvm_find(T, c);
        const int64_t i0 = (int64_t)(c - T.first[t]) * PVM_CHUNK, i1 = min(T.n[t], i0 + PVM_CHUNK);
        PVM_BY_TYPE(T.dt[t], pvm_adam_chunk<D_>(T.a[t], static_cast<float*>(T.b[t]), T.m[t], T.v[t], T.tile[t], i0, i1, s, alpha, c1, c2, eps));
    }
}
