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
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

enum { PVM_MAXT = 48, PVM_THREADS = 256, PVM_CHUNK = 8192, PVM_PARTS = 2048 };

typedef float pvm_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short pvm_u16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 pvm_f16x4 __attribute__((ext_vector_type(4)));

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
    unsigned char vec[PVM_MAXT];   // every pointer is aligned for four elements
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
    if (dt == 0) return *reinterpret_cast<const pvm_f32x4*>(static_cast<const float*>(p) + i);
    if (dt == 1) {
        const pvm_u16x4 u = *reinterpret_cast<const pvm_u16x4*>(static_cast<const unsigned short*>(p) + i);
        return (pvm_f32x4){pvm_bf16(u.x), pvm_bf16(u.y), pvm_bf16(u.z), pvm_bf16(u.w)};
    }
    const pvm_f16x4 h = *reinterpret_cast<const pvm_f16x4*>(static_cast<const _Float16*>(p) + i);
    return (pvm_f32x4){(float)h.x, (float)h.y, (float)h.z, (float)h.w};
}
__device__ __forceinline__ void pvm_store1(void* p, int dt, int64_t i, float x) {
    if (dt == 0) static_cast<float*>(p)[i] = x;
    else if (dt == 1) static_cast<unsigned short*>(p)[i] = pvm_to_bf16(x);
    else static_cast<_Float16*>(p)[i] = (_Float16)x;
}
__device__ __forceinline__ void pvm_store4(void* p, int dt, int64_t i, pvm_f32x4 x) {
    if (dt == 0) *reinterpret_cast<pvm_f32x4*>(static_cast<float*>(p) + i) = x;
    else if (dt == 1)
        *reinterpret_cast<pvm_u16x4*>(static_cast<unsigned short*>(p) + i) =
            (pvm_u16x4){pvm_to_bf16(x.x), pvm_to_bf16(x.y), pvm_to_bf16(x.z), pvm_to_bf16(x.w)};
    else
        *reinterpret_cast<pvm_f16x4*>(static_cast<_Float16*>(p) + i) =
            (pvm_f16x4){(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
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

__global__ __launch_bounds__(PVM_THREADS) void pvk_sumsq(const PvmTab T, double* __restrict__ part) {
    const int chunks = T.first[T.count];
    double s = 0.0;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = pvm_find(T, c), dt = T.dt[t];
        const void* a = T.a[t];
        const int64_t i0 = (int64_t)(c - T.first[t]) * PVM_CHUNK, i1 = min(T.n[t], i0 + PVM_CHUNK);
        int64_t i = i0;
        if (T.vec[t]) {
            for (i = i0 + 4 * threadIdx.x; i + 3 < i1; i += 4 * PVM_THREADS) {
                const pvm_f32x4 x = pvm_load4(a, dt, i);
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fma((double)x[e], (double)x[e], s);
            }
            i = i0 + ((i1 - i0) & ~(int64_t)3);
        }
        for (i += threadIdx.x; i < i1; i += PVM_THREADS) {
            const double x = pvm_load1(a, dt, i);
            s = fma(x, x, s);
        }
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

__global__ __launch_bounds__(PVM_THREADS) void pvk_clip_apply(const PvmTab T, const double* __restrict__ part, int nparts, double max_norm,
                                                              float* __restrict__ norm) {
    const double n = pvm_norm(part, nparts);
    const float s = pvm_scale(n, max_norm);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const int chunks = T.first[T.count];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = pvm_find(T, c), dt = T.dt[t];
        const void* a = T.a[t];
        void* b = T.b[t];
        if (s == 1.f && a == b) continue;  // in place and within the bound: every value stays as it is
        const int64_t i0 = (int64_t)(c - T.first[t]) * PVM_CHUNK, i1 = min(T.n[t], i0 + PVM_CHUNK);
        int64_t i = i0;
        if (T.vec[t]) {
            for (i = i0 + 4 * threadIdx.x; i + 3 < i1; i += 4 * PVM_THREADS) pvm_store4(b, dt, i, pvm_load4(a, dt, i) * s);
            i = i0 + ((i1 - i0) & ~(int64_t)3);
        }
        for (i += threadIdx.x; i < i1; i += PVM_THREADS) pvm_store1(b, dt, i, pvm_load1(a, dt, i) * s);
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
        const int t = pvm_find(T, c), dt = T.dt[t], tile = T.tile[t];
        const void* a = T.a[t];
        float *p = static_cast<float*>(T.b[t]), *m = T.m[t], *v = T.v[t];
        const int64_t i0 = (int64_t)(c - T.first[t]) * PVM_CHUNK, i1 = min(T.n[t], i0 + PVM_CHUNK);
        auto at = [&](int64_t i) { return tile ? i + i / tile * 2 * tile : i; };  // i / tile * 3 tile + i % tile
        int64_t i = i0;
        if (T.vec[t]) {
            for (i = i0 + 4 * threadIdx.x; i + 3 < i1; i += 4 * PVM_THREADS) {
                const pvm_f32x4 g = pvm_load4(a, dt, i) * s;
                const int64_t j = at(i);
                pvm_f32x4 p4 = *reinterpret_cast<pvm_f32x4*>(p + j), m4 = *reinterpret_cast<pvm_f32x4*>(m + j),
                          v4 = *reinterpret_cast<pvm_f32x4*>(v + j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float pe = p4[e], me = m4[e], ve = v4[e];
                    pvm_adam1(pe, me, ve, g[e], alpha, c1, c2, eps);
                    p4[e] = pe; m4[e] = me; v4[e] = ve;
                }
                *reinterpret_cast<pvm_f32x4*>(p + j) = p4;
                *reinterpret_cast<pvm_f32x4*>(m + j) = m4;
                *reinterpret_cast<pvm_f32x4*>(v + j) = v4;
            }
            i = i0 + ((i1 - i0) & ~(int64_t)3);
        }
        for (i += threadIdx.x; i < i1; i += PVM_THREADS) {
            const int64_t j = at(i);
            pvm_adam1(p[j], m[j], v[j], pvm_load1(a, dt, i) * s, alpha, c1, c2, eps);
        }
    }
}
