// A dense layer as one operator: y = f(x w + b) + r, and its gradients (pvae_ops.h).
//
// All products put the weights' columns on the rows of the matrix instruction's result and x's rows on its columns: a lane
// then holds four consecutive columns of one row of y, which bias, residual, z and y are read and written in.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pvae_multi.h"

enum { PVD_F32 = 0, PVD_BF16 = 1, PVD_F16 = 2 };
enum { PVD_LINEAR = 0, PVD_RELU = 1, PVD_ELU = 2, PVD_SIGMOID = 3, PVD_TANH = 4, PVD_SILU = 5, PVD_GELU = 6 };

typedef float pvd_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 pvd_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pvd_f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned pvd_u32x4 __attribute__((ext_vector_type(4)));

template <int DT> struct PvdType { typedef unsigned short T; enum { SIZE = 2, VEC = 8 }; };
template <> struct PvdType<PVD_F32> { typedef float T; enum { SIZE = 4, VEC = 4 }; };

template <int DT> __device__ __forceinline__ float pvd_to_f32(typename PvdType<DT>::T x) {
    if constexpr (DT == PVD_F32) return x;
    else if constexpr (DT == PVD_BF16) return pvm_bf16(x);
    else return (float)__builtin_bit_cast(_Float16, x);
}
template <int DT> __device__ __forceinline__ typename PvdType<DT>::T pvd_from_f32(float x) {
    if constexpr (DT == PVD_F32) return x;
    else if constexpr (DT == PVD_BF16) return pvm_to_bf16(x);
    else return __builtin_bit_cast(unsigned short, (_Float16)x);
}

// ---------------------------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float pvd_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ __forceinline__ float pvd_phi(float z) { return __expf(-0.5f * z * z) * 0.3989422804014327f; }
__device__ __forceinline__ float pvd_Phi(float z) { return 0.5f * (1.f + erff(z * 0.7071067811865476f)); }
__device__ __forceinline__ float pvd_act(float z, int act) {
    switch (act) {
        case PVD_RELU: return z > 0.f ? z : z != z ? z : 0.f;
        case PVD_ELU: return z > 0.f ? z : expm1f(z);
        case PVD_SIGMOID: return pvd_sigmoid(z);
        case PVD_TANH: return tanhf(z);
        case PVD_SILU: return z * pvd_sigmoid(z);
        case PVD_GELU: return z * pvd_Phi(z);
        default: return z;
    }
}
__device__ __forceinline__ float pvd_act_grad(float z, int act) {
    switch (act) {
        case PVD_RELU: return z > 0.f ? 1.f : 0.f;
        case PVD_ELU: return z > 0.f ? 1.f : __expf(z);
        case PVD_SIGMOID: { const float s = pvd_sigmoid(z); return s * (1.f - s); }
        case PVD_TANH: { const float t = tanhf(z); return 1.f - t * t; }
        case PVD_SILU: { const float s = pvd_sigmoid(z); return s * (1.f + z * (1.f - s)); }
        case PVD_GELU: return pvd_Phi(z) + z * pvd_phi(z);
        default: return 1.f;
    }
}

// ---------------------------------------------------------------------------------------------
// what follows the product
// ---------------------------------------------------------------------------------------------
struct PvdOut {
    int64_t rows, cols;
    void* y;
    int64_t ldy;
    const void* bias;
    const void* res;
    int64_t ldr;
    float* pre;
    int64_t ldp;
    int act;
    int vec;  // four columns at a multiple of four may be read and written as one access everywhere
};

// z = the products of columns n .. n + 3 of row m
template <int DT> __device__ __forceinline__ void pvd_finish4(const PvdOut& O, int64_t m, int64_t n, pvd_f32x4 z) {
    typedef typename PvdType<DT>::T T;
    if (m >= O.rows || n >= O.cols) return;
    const T *bias = static_cast<const T*>(O.bias), *res = static_cast<const T*>(O.res);
    T* y = static_cast<T*>(O.y) + m * O.ldy + n;
    if (O.vec && n + 3 < O.cols) {
        if (bias) z += pvm_load4(bias, DT, n);
        if (O.pre) *reinterpret_cast<pvd_f32x4*>(O.pre + m * O.ldp + n) = z;
        pvd_f32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pvd_act(z[e], O.act);
        if (res) o += pvm_load4(res, DT, m * O.ldr + n);
        pvm_store4(y, DT, 0, o);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (n + e >= O.cols) return;
        float a = z[e];
        if (bias) a += pvd_to_f32<DT>(bias[n + e]);
        if (O.pre) O.pre[m * O.ldp + n + e] = a;
        a = pvd_act(a, O.act);
        if (res) a += pvd_to_f32<DT>(res[m * O.ldr + n + e]);
        y[e] = pvd_from_f32<DT>(a);
    }
}

// ---------------------------------------------------------------------------------------------
// The tile kernel: any size, stride and alignment.  A workgroup of four waves makes a 64 x 64 piece of the result, a wave
// 32 x 32 of it; the contraction goes through LDS 128 bytes per row at a time, the next piece on its way to registers
// meanwhile.  float32: v_mfma_f32_16x16x4 (exact float32 products); 16-bit types: 16x16x32.
// ---------------------------------------------------------------------------------------------
struct PvdOperand {  // element (row, k) at p[row * sr + k * sk]; one of the strides is 1
    const void* p;
    int64_t rows, sr, sk;
    const float* pre;  // gradient operand: p is dy and the element dy * f'(pre); pre's strides
    int64_t pr, pk;
    int act;
    int vec;  // sixteen bytes along the unit stride may be read as one access where they start at a multiple
};

enum { PVD_T = 64, PVD_LDB = 144 };  // tile edge; bytes of an LDS row: 128 and 16 that spread the rows over the banks

template <int DT, bool GRAD> struct PvdStage {
    typedef typename PvdType<DT>::T T;
    enum { VEC = PvdType<DT>::VEC, KS = 128 / PvdType<DT>::SIZE };
    alignas(16) T r[2][VEC];

    // one run of VEC elements along the unit stride: first element (row, k), `along_k` which way it runs
    __device__ __forceinline__ void run(const PvdOperand& P, int64_t row, int64_t k, int64_t k1, bool along_k, T* o) {
        const T* p = static_cast<const T*>(P.p) + row * P.sr + k * P.sk;
        const float* z = GRAD ? P.pre + row * P.pr + k * P.pk : nullptr;
        const int64_t left = along_k ? k1 - k : P.rows - row;
        if (row >= P.rows || k >= k1 || left <= 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = T(0);
            return;
        }
        if (P.vec && left >= VEC) {
            *reinterpret_cast<pvd_u32x4*>(o) = *reinterpret_cast<const pvd_u32x4*>(p);
            if (GRAD && P.act != PVD_LINEAR) {
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const pvd_f32x4 z4 = *reinterpret_cast<const pvd_f32x4*>(z + e);
#pragma unroll
                    for (int f = 0; f < 4; ++f) o[e + f] = pvd_from_f32<DT>(pvd_to_f32<DT>(o[e + f]) * pvd_act_grad(z4[f], P.act));
                }
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            o[e] = T(0);
            if (e < left) {
                o[e] = p[e];
                if (GRAD && P.act != PVD_LINEAR) o[e] = pvd_from_f32<DT>(pvd_to_f32<DT>(p[e]) * pvd_act_grad(z[e], P.act));
            }
        }
    }
    __device__ __forceinline__ void load(const PvdOperand& P, int64_t row0, int64_t k0, int64_t k1, int tid) {
        if (P.sk == 1) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = tid + 256 * u;
                run(P, row0 + (c >> 3), k0 + (c & 7) * VEC, k1, true, r[u]);
            }
        } else {  // VEC rows at k and at k + 1
            const int rg = tid % (PVD_T / VEC), kp = tid / (PVD_T / VEC);
#pragma unroll
            for (int u = 0; u < 2; ++u) run(P, row0 + rg * VEC, k0 + 2 * kp + u, k1, false, r[u]);
        }
    }
    __device__ __forceinline__ void store(const PvdOperand& P, char* s, int tid) {
        if (P.sk == 1) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = tid + 256 * u;
                *reinterpret_cast<pvd_u32x4*>(s + (c >> 3) * PVD_LDB + (c & 7) * 16) = *reinterpret_cast<const pvd_u32x4*>(r[u]);
            }
        } else {
            const int rg = tid % (PVD_T / VEC), kp = tid / (PVD_T / VEC);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                T* d = reinterpret_cast<T*>(s + (rg * VEC + e) * PVD_LDB) + 2 * kp;
                d[0] = r[0][e];
                d[1] = r[1][e];
            }
        }
    }
};

template <int DT> __device__ __forceinline__ pvd_f32x4 pvd_mfma16(pvd_u32x4 a, pvd_u32x4 b, pvd_f32x4 c) {
    if constexpr (DT == PVD_F32) {
        // sixteen k: lane group q holds k = 4 q .. 4 q + 3, one of them per instruction, the same in both operands
        const pvd_f32x4 fa = __builtin_bit_cast(pvd_f32x4, a), fb = __builtin_bit_cast(pvd_f32x4, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[e], fb[e], c, 0, 0, 0);
        return c;
    } else if constexpr (DT == PVD_BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pvd_bf16x8, a), __builtin_bit_cast(pvd_bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pvd_f16x8, a), __builtin_bit_cast(pvd_f16x8, b), c, 0, 0, 0);
    }
}

// products of x's rows [m0, m0 + 64) and the weights' columns [n0, n0 + 64) over k0 .. k1, into acc[column group][row group]
template <int DT, bool GX, bool GW>
__device__ __forceinline__ void pvd_tile(const PvdOperand& X, const PvdOperand& W, int64_t m0, int64_t n0, int64_t k0, int64_t k1,
                                         char* smem, pvd_f32x4 (&acc)[2][2]) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
    char *xs = smem, *ws = smem + PVD_T * PVD_LDB;
    PvdStage<DT, GX> sx;
    PvdStage<DT, GW> sw;
    enum { KS = PvdStage<DT, GX>::KS };
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = (pvd_f32x4){0.f, 0.f, 0.f, 0.f};
    if (k0 >= k1) return;
    sx.load(X, m0, k0, k1, tid);
    sw.load(W, n0, k0, k1, tid);
    for (int64_t k = k0; k < k1; k += KS) {
        sx.store(X, xs, tid);
        sw.store(W, ws, tid);
        __syncthreads();
        if (k + KS < k1) {
            sx.load(X, m0, k + KS, k1, tid);
            sw.load(W, n0, k + KS, k1, tid);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            pvd_u32x4 a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = *reinterpret_cast<const pvd_u32x4*>(ws + (wn + 16 * i + r) * PVD_LDB + h * 64 + q * 16);
                b[i] = *reinterpret_cast<const pvd_u32x4*>(xs + (wm + 16 * i + r) * PVD_LDB + h * 64 + q * 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = pvd_mfma16<DT>(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
}

struct PvdTileJob {
    PvdOperand X, W;
    PvdOut O;
    int64_t K;
    int mt, nt, splits;  // tiles along rows and columns, pieces of the contraction
    int64_t kper;        // contraction of a piece: a multiple of the LDS step
    float* part;         // splits > 1: [piece][rows][cols] float32
};

template <int DT, bool GX, bool GW> __device__ __forceinline__ void pvd_tile_job(const PvdTileJob& J, int64_t block, char* smem) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tiles = (int64_t)J.mt * J.nt;
    const int piece = (int)(block / tiles);
    const int64_t t = block % tiles, m0 = t / J.nt * PVD_T, n0 = t % J.nt * PVD_T;
    const int64_t k0 = piece * J.kper, k1 = min(J.K, k0 + J.kper);
    pvd_f32x4 acc[2][2];
    pvd_tile<DT, GX, GW>(J.X, J.W, m0, n0, k0, k1, smem, acc);
    const int64_t m = m0 + (wave & 1) * 32 + (lane & 15), n = n0 + (wave >> 1) * 32 + (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t mm = m + 16 * j, nn = n + 16 * i;
            if (J.splits == 1) pvd_finish4<DT>(J.O, mm, nn, acc[i][j]);
            else if (mm < J.O.rows)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (nn + e < J.O.cols) J.part[(piece * J.O.rows + mm) * J.O.cols + nn + e] = acc[i][j][e];
        }
}

template <int DT> __global__ __launch_bounds__(256) void pvk_dense_tile(const PvdTileJob J) {
    __shared__ __attribute__((aligned(16))) char smem[2 * PVD_T * PVD_LDB];
    pvd_tile_job<DT, false, false>(J, blockIdx.x, smem);
}

// the pieces of a split contraction, added in order, and what follows the product
template <int DT> __global__ __launch_bounds__(256) void pvk_dense_join(const PvdOut O, const float* __restrict__ part, int pieces) {
    const int64_t quads = (O.cols + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= O.rows * quads) return;
    const int64_t m = i / quads, n = i % quads * 4;
    pvd_f32x4 z = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < pieces; ++p)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < O.cols) z[e] += part[(p * O.rows + m) * O.cols + n + e];
    pvd_finish4<DT>(O, m, n, z);
}

// ---------------------------------------------------------------------------------------------
// Gradients, one launch: the first workgroups make dx (x-side operand g, contraction over n), the next dw (rows of x^T,
// contraction over m), the last 64 columns of dbias (and dpre) each.  g = dy f'(pre) is formed on the way into LDS.
// ---------------------------------------------------------------------------------------------
struct PvdBwdJob {
    PvdTileJob dx, dw;
    int64_t n_dx, n_dw;  // workgroups of each
    const void* dy;
    int64_t lddy;
    const float* pre;
    int64_t ldp;
    int act;
    int64_t m, n;
    void* dbias;
    float* dpre;
};

template <int DT> __global__ __launch_bounds__(256) void pvk_dense_bwd_tile(const PvdBwdJob J) {
    __shared__ __attribute__((aligned(16))) char smem[2 * PVD_T * PVD_LDB];
    typedef typename PvdType<DT>::T T;
    int64_t b = blockIdx.x;
    if (b < J.n_dx) return pvd_tile_job<DT, true, false>(J.dx, b, smem);
    b -= J.n_dx;
    if (b < J.n_dw) return pvd_tile_job<DT, false, true>(J.dw, b, smem);
    b -= J.n_dw;
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int64_t n = b * 64 + c;
    float s = 0.f;
    if (n < J.n)
        for (int64_t m = g; m < J.m; m += 4) {
            float v = pvd_to_f32<DT>(static_cast<const T*>(J.dy)[m * J.lddy + n]);
            if (J.act != PVD_LINEAR) v *= pvd_act_grad(J.pre[m * J.ldp + n], J.act);
            if (J.dpre) J.dpre[m * J.n + n] = v;
            s += v;
        }
    float* red = reinterpret_cast<float*>(smem);
    red[threadIdx.x] = s;
    __syncthreads();
    if (g == 0 && n < J.n && J.dbias)
        static_cast<T*>(J.dbias)[n] = pvd_from_f32<DT>((red[c] + red[64 + c]) + (red[128 + c] + red[192 + c]));
}
