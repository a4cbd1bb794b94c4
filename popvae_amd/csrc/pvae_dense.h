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
typedef pvd_u32x4 pvd_u32x4_any __attribute__((aligned(2)));  // sixteen bytes at any address of an element

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
// e^x = 2^t (1 + r ln 2) with t = x / ln 2 rounded and r what that lost: without r the error grows with |x| (at 20 a dozen
// units in the last place; with it two or three at any x).  r is below 2^-17 while 2^t is a number; beyond, where it may be
// anything or NaN (max takes -1), 2^t is 0 or infinite and stays so.  Results below 2^-126 are 0.
// 2504 x 128 x 100000 with sigmoid: 665 us without r, 672 with it, 698 with expf.
__device__ __forceinline__ float pvd_exp(float x) {
    const float t = x * 1.4426950408889634f;
    const float r = fmaf(x, 1.9259629911266175e-8f, fmaf(x, 1.4426950408889634f, -t));  // 1 / ln 2 in two float32
    return __builtin_amdgcn_exp2f(t) * fmaf(fminf(fmaxf(r, -1.f), 1.f), 0.6931471805599453f, 1.f);
}
__device__ __forceinline__ float pvd_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + pvd_exp(-z)); }
__device__ __forceinline__ float pvd_phi(float z) { return pvd_exp(-0.5f * z * z) * 0.3989422804014327f; }
__device__ __forceinline__ float pvd_Phi(float z) { return 0.5f * (1.f + erff(z * 0.7071067811865476f)); }
// the kind is the same for the whole launch: one branch for four values
__device__ __forceinline__ pvd_f32x4 pvd_act4(pvd_f32x4 z, int act) {
#define PVD_EACH(EXPR)                                  \
    _Pragma("unroll") for (int e = 0; e < 4; ++e) {     \
        const float x = z[e];                           \
        z[e] = EXPR;                                    \
    }                                                   \
    return z;
    switch (act) {
        case PVD_RELU: PVD_EACH(x > 0.f ? x : x != x ? x : 0.f)
        case PVD_ELU: PVD_EACH(x > 0.f ? x : expm1f(x))
        case PVD_SIGMOID: PVD_EACH(pvd_sigmoid(x))
        case PVD_TANH: PVD_EACH(tanhf(x))
        case PVD_SILU: PVD_EACH(x * pvd_sigmoid(x))
        case PVD_GELU: PVD_EACH(x * pvd_Phi(x))
        default: return z;
    }
}
__device__ __forceinline__ float pvd_silu_grad(float z) {
    const float s = pvd_sigmoid(z);
    return s * (1.f + z * (1.f - s));
}
__device__ __forceinline__ float pvd_tanh_grad(float z) {
    const float t = tanhf(z);
    return 1.f - t * t;
}
__device__ __forceinline__ pvd_f32x4 pvd_act_grad4(pvd_f32x4 z, int act) {
    switch (act) {
        case PVD_RELU: PVD_EACH(x > 0.f ? 1.f : 0.f)
        case PVD_ELU: PVD_EACH(x > 0.f ? 1.f : pvd_exp(x))
        case PVD_SIGMOID: PVD_EACH(pvd_sigmoid(x) * pvd_sigmoid(-x))
        case PVD_TANH: PVD_EACH(pvd_tanh_grad(x))
        case PVD_SILU: PVD_EACH(pvd_silu_grad(x))
        case PVD_GELU: PVD_EACH(pvd_Phi(x) + x * pvd_phi(x))
        default: return (pvd_f32x4){1.f, 1.f, 1.f, 1.f};
    }
#undef PVD_EACH
}
__device__ __forceinline__ float pvd_act(float z, int act) { return pvd_act4((pvd_f32x4){z, z, z, z}, act)[0]; }
__device__ __forceinline__ float pvd_act_grad(float z, int act) { return pvd_act_grad4((pvd_f32x4){z, z, z, z}, act)[0]; }

// ---------------------------------------------------------------------------------------------
// g = dy f'(pre) of a 16-bit type enters the products in two terms, so that a gradient is rounded once, at its end, and fits
// wherever its value does: g = UNIT (hi + LOW lo).  bf16: hi is cut off, not rounded, so that it is finite where g is; sixteen
// bits of g in all.  float16: UNIT keeps g of the largest dy and f' below the type's largest value, LOW the second term of the
// smallest g above its least: 22 bits of g, to 2^-35 at worst; hi is 0 only where g is.  What an infinite x or w makes of a
// gradient is in the first terms' sums, and so is a g that is infinite or NaN: a second terms' sum that is not finite (0 times
// infinity, infinities of both signs) is dropped.
// One rounding of g to the type would save half of the matrix work and leave a gradient off by as much again as its own
// rounding (4096 x 2048 x 4096 bf16 with GELU: 0.0024 relative to 64 bits instead of 0.0017).
// ---------------------------------------------------------------------------------------------
template <int DT> struct PvdTerms { static constexpr float UNIT = 1.f, LOW = 1.f; };
template <> struct PvdTerms<PVD_F16> { static constexpr float UNIT = 2.f, LOW = 1.f / 2048.f; };
template <int DT> __device__ __forceinline__ void pvd_terms(float g, typename PvdType<DT>::T& hi, typename PvdType<DT>::T& lo) {
    static_assert(DT != PVD_F32, "float32 products take g as it is");
    if constexpr (DT == PVD_BF16) {
        hi = (unsigned short)(__float_as_uint(g) >> 16);  // a product's NaN is quiet: its bit stays
        lo = __builtin_bit_cast(unsigned short, (__bf16)(g - pvm_bf16(hi)));
    } else {
        const float s = g * (1.f / PvdTerms<DT>::UNIT);
        hi = pvd_from_f32<DT>(s);
        if ((hi & 0x7fffu) == 0 && s != 0.f) hi |= 1;  // the least value, s's sign: lo takes it back
        lo = pvd_from_f32<DT>((s - pvd_to_f32<DT>(hi)) * (1.f / PvdTerms<DT>::LOW));
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
};

// four elements from p[i] on, `left` of which are there (zeros, and nothing stored, behind them)
__device__ __forceinline__ pvd_f32x4 pvd_load_some(const void* p, int dt, int64_t i, int left) {
    if (left >= 4) return pvm_load4(p, dt, i);
    pvd_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < left) v[e] = pvm_load1(p, dt, i + e);
    return v;
}
__device__ __forceinline__ void pvd_store_some(void* p, int dt, int64_t i, pvd_f32x4 v, int left) {
    if (left >= 4) return pvm_store4(p, dt, i, v);
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < left) pvm_store1(p, dt, i + e, v[e]);
}
__device__ __forceinline__ int pvd_left(int64_t n, int64_t cols) { return (int)min((int64_t)4, cols - n); }

// z = the products of columns n .. n + 3 of row m
template <int DT> __device__ __forceinline__ void pvd_finish4(const PvdOut& O, int64_t m, int64_t n, pvd_f32x4 z) {
    if (m >= O.rows || n >= O.cols) return;
    const int left = pvd_left(n, O.cols);
    if (O.bias) z += pvd_load_some(O.bias, DT, n, left);
    if (O.pre) pvd_store_some(O.pre, 0, m * O.ldp + n, z, left);
    pvd_f32x4 o = pvd_act4(z, O.act);
    if (O.res) o += pvd_load_some(O.res, DT, m * O.ldr + n, left);
    pvd_store_some(O.y, DT, m * O.ldy + n, o, left);
}

// ---------------------------------------------------------------------------------------------
// The tile kernel: any size, stride and alignment.  A workgroup of four waves makes a 64 x 64 piece of the result, a wave
// 32 x 32 of it; the contraction goes through LDS 128 bytes per row at a time, the next piece on its way to registers
// meanwhile.  float32: v_mfma_f32_16x16x4 (exact float32 products); 16-bit types: 16x16x32.  It serves what neither fills the
// large kernel's pipeline nor fits the slim kernel -- short contractions, few rows of weights that would have to be laid out --
// and is bound by one round trip to memory per step: 1000 x 128 x 1000 bf16 7.6 us, 64 x 4001 x 4001 bf16 22 us (1.5 TB/s).
// ---------------------------------------------------------------------------------------------
struct PvdOperand {  // element (row, k) at p[row * sr + k * sk]; one of the strides is 1
    const void* p;
    int64_t rows, sr, sk;
    const float* pre;  // gradient operand: p is dy and the element dy * f'(pre); pre's strides
    int64_t pr, pk;
    int act;
};

enum { PVD_T = 64, PVD_LDB = 144 };  // tile edge; bytes of an LDS row: 128 and 16 that spread the rows over the banks

template <int DT> struct PvdStage {
    typedef typename PvdType<DT>::T T;
    enum { VEC = PvdType<DT>::VEC, KS = 128 / PvdType<DT>::SIZE };
    alignas(16) T r[2][VEC];

    // one run of VEC elements along the unit stride: first element (row, k), `along_k` which way it runs
    __device__ __forceinline__ void run(const PvdOperand& P, int64_t row, int64_t k, int64_t k1, bool along_k, T* o) {
        const T* p = static_cast<const T*>(P.p) + row * P.sr + k * P.sk;
        const int64_t left = along_k ? k1 - k : P.rows - row;
        if (row >= P.rows || k >= k1 || left <= 0) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = T(0);
            return;
        }
        if (left >= VEC) {
            *reinterpret_cast<pvd_u32x4*>(o) = *reinterpret_cast<const pvd_u32x4_any*>(p);
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = p[min((int64_t)e, left - 1)];  // the last element again: no load waits for a branch
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[e] = e < left ? o[e] : T(0);
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
template <int DT>
__device__ __forceinline__ void pvd_tile(const PvdOperand& X, const PvdOperand& W, int64_t m0, int64_t n0, int64_t k0, int64_t k1,
                                         char* smem, pvd_f32x4 (&acc)[2][2]) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
    char *xs = smem, *ws = smem + PVD_T * PVD_LDB;
    PvdStage<DT> sx, sw;
    enum { KS = PvdStage<DT>::KS };
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

template <int DT> __global__ __launch_bounds__(256) void pvk_dense_tile(const PvdTileJob J) {
    __shared__ __attribute__((aligned(16))) char smem[2 * PVD_T * PVD_LDB];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tiles = (int64_t)J.mt * J.nt;
    const int piece = (int)(blockIdx.x / tiles);
    const int64_t t = blockIdx.x % tiles, m0 = t / J.nt * PVD_T, n0 = t % J.nt * PVD_T;
    const int64_t k0 = piece * J.kper, k1 = min(J.K, k0 + J.kper);
    pvd_f32x4 acc[2][2];
    pvd_tile<DT>(J.X, J.W, m0, n0, k0, k1, smem, acc);
    const int64_t m = m0 + (wave & 1) * 32 + (lane & 15), n = n0 + (wave >> 1) * 32 + (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t mm = m + 16 * j, nn = n + 16 * i;
            if (J.splits == 1) pvd_finish4<DT>(J.O, mm, nn, acc[i][j]);
            else if (mm < J.O.rows && nn < J.O.cols) pvd_store_some(J.part, 0, (piece * J.O.rows + mm) * J.O.cols + nn, acc[i][j], pvd_left(nn, J.O.cols));
        }
}

// ---------------------------------------------------------------------------------------------
// The slim kernel, for few rows or results too small to give the chip 64 x 64 tiles: a workgroup of eight waves makes 32 rows
// x 16 columns.  The waves take runs of the contraction in turn and read both operands straight from memory into the matrix
// instruction's registers -- one round trip instead of one per LDS step, which is what such a call spends its time on --
// and the eight partial results meet in LDS, added in order.  32 x 128 x 128 in float32: 5.0 us, nearly all of it the launch
// and two round trips; 16 x 4096 x 4096: 27 us (w at 2.5 TB/s).
// ---------------------------------------------------------------------------------------------
enum { PVD_SM = 32, PVD_SN = 16, PVD_SW = 8 };

// VEC elements of row `row` from k on, as a lane of the matrix instruction holds them, zeros outside; and z there, if g is asked for
template <int DT, bool GRAD> struct PvdSlim {
    typedef typename PvdType<DT>::T T;
    enum { VEC = PvdType<DT>::VEC };
    alignas(16) T v[VEC];
    alignas(16) float z[VEC];

    __device__ __forceinline__ void load(const PvdOperand& P, int64_t row, int64_t k, int64_t k1) {
        const bool grad = GRAD && P.act != PVD_LINEAR, in = row < P.rows;
        const bool whole = P.sk == 1 && (!grad || P.pk == 1) && k + VEC <= k1;  // z's stride is its own (dy of one column, z of more)
        const int64_t rr = min(row, P.rows - 1);
        const T* p = static_cast<const T*>(P.p) + rr * P.sr;
        const float* pz = grad ? P.pre + rr * P.pr : nullptr;
        T t[VEC];
        float f[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = 0.f;
        if (whole) {
            const pvd_u32x4 d = *reinterpret_cast<const pvd_u32x4_any*>(p + k);
            __builtin_memcpy(t, &d, 16);
            if (grad)
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const pvd_f32x4 d4 = pvm_load4(pz, 0, k + e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[e + i] = d4[i];
                }
        } else {  // what lies outside reads the last element inside instead: no load waits for a branch
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = p[min(k + e, k1 - 1) * P.sk];
            if (grad)
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] = pz[min(k + e, k1 - 1) * P.pk];
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const bool there = in && (whole || k + e < k1);
            v[e] = there ? t[e] : T(0);
            z[e] = there ? f[e] : 0.f;
        }
    }
    // v becomes g, in a 16-bit type its first term; the second goes into `lo`
    __device__ __forceinline__ void grad(int act, pvd_u32x4& lo) {
        alignas(16) T l[VEC];
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            const pvd_f32x4 d = pvd_act_grad4(*reinterpret_cast<const pvd_f32x4*>(z + e), act);
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                const float g = pvd_to_f32<DT>(v[e + f]) * d[f];
                if constexpr (DT == PVD_F32) v[e + f] = g;
                else pvd_terms<DT>(g, v[e + f], l[e + f]);
            }
        }
        if constexpr (DT != PVD_F32) lo = *reinterpret_cast<const pvd_u32x4*>(l);
    }
    __device__ __forceinline__ pvd_u32x4 bits() const { return *reinterpret_cast<const pvd_u32x4*>(v); }
};

template <int DT, bool GX, bool GW> __device__ __forceinline__ void pvd_slim_job(const PvdTileJob& J, int64_t block, float* red) {
    enum { KS = 4 * PvdType<DT>::VEC, RUN = 2 };  // contraction of one matrix instruction group; groups under way per wave
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int64_t tiles = (int64_t)J.mt * J.nt;
    const int piece = (int)(block / tiles);
    const int64_t t = block % tiles, m0 = t / J.nt * PVD_SM, n0 = t % J.nt * PVD_SN;
    const int64_t k0 = piece * J.kper, k1 = min(J.K, k0 + J.kper);
    const bool gx = GX && J.X.act != PVD_LINEAR, gw = GW && J.W.act != PVD_LINEAR;
    const int halves = m0 + 16 < J.X.rows ? 2 : 1;
    pvd_f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    pvd_f32x4 low[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};  // the second terms' products
    for (int64_t k = k0 + wave * (RUN * KS); k < k1; k += PVD_SW * RUN * KS) {
        PvdSlim<DT, GW> a[RUN];
        PvdSlim<DT, GX> b[RUN][2];
#pragma unroll
        for (int u = 0; u < RUN; ++u) {
            const int64_t kk = k + u * KS + q * PvdType<DT>::VEC;
            a[u].load(J.W, n0 + r, kk, k1);
            b[u][0].load(J.X, m0 + r, kk, k1);
            b[u][1].load(J.X, m0 + 16 + r, kk, k1);
        }
#pragma unroll
        for (int u = 0; u < RUN; ++u) {
            if (k + u * KS < k1) {  // the same for the whole wave, as is the number of halves
                pvd_u32x4 al, bl;
                if (gw) a[u].grad(J.W.act, al);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (j < halves) {
                        if (gx) b[u][j].grad(J.X.act, bl);
                        acc[j] = pvd_mfma16<DT>(a[u].bits(), b[u][j].bits(), acc[j]);
                        if (DT != PVD_F32 && gw) low[j] = pvd_mfma16<DT>(al, b[u][j].bits(), low[j]);
                        if (DT != PVD_F32 && gx) low[j] = pvd_mfma16<DT>(a[u].bits(), bl, low[j]);
                    }
            }
        }
    }
    if constexpr (DT != PVD_F32 && (GX || GW)) {
        if (gx || gw)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (fabsf(low[j][e]) < __builtin_inff()) acc[j][e] = fmaf(low[j][e], PvdTerms<DT>::LOW, acc[j][e]);
                    acc[j][e] *= PvdTerms<DT>::UNIT;
                }
    }
    // red[wave][row][16 columns]
#pragma unroll
    for (int j = 0; j < 2; ++j) *reinterpret_cast<pvd_f32x4*>(red + ((wave * PVD_SM + 16 * j + r) * PVD_SN + 4 * q)) = acc[j];
    __syncthreads();
    if (tid >= PVD_SM * PVD_SN / 4) return;
    const int row = tid >> 2, c = (tid & 3) * 4;
    pvd_f32x4 z = *reinterpret_cast<const pvd_f32x4*>(red + row * PVD_SN + c);
#pragma unroll
    for (int w = 1; w < PVD_SW; ++w) z += *reinterpret_cast<const pvd_f32x4*>(red + (w * PVD_SM + row) * PVD_SN + c);
    const int64_t m = m0 + row, n = n0 + c;
    if (J.splits == 1) pvd_finish4<DT>(J.O, m, n, z);
    else if (m < J.O.rows) pvd_store_some(J.part, 0, (piece * J.O.rows + m) * J.O.cols + n, z, pvd_left(n, J.O.cols));
}

template <int DT> __global__ __launch_bounds__(512, 4) void pvk_dense_slim(const PvdTileJob J) {
    __shared__ __attribute__((aligned(16))) float red[PVD_SW * PVD_SM * PVD_SN];
    pvd_slim_job<DT, false, false>(J, blockIdx.x, red);
}

// ---------------------------------------------------------------------------------------------
// The rows kernel, for up to four rows, float32 up to eight (one point asked for an answer): the weights are read once, and that is its time.  A
// lane holds sixteen bytes of a row of w and all rows' sums of those columns in registers; x, as float32, comes from LDS.  The
// workgroup's eight waves, and pieces of the grid, split the contraction.  Matrix instructions would compute sixteen rows for
// one and need w transposed on the way; plain ones keep up with memory as long as rows are few.  1 x 128 x 100000 in
// float32: 11.0 us = 4.7 TB/s; 1 x 128 x 1000000: 90 us = 5.8 TB/s, in bf16 39 us = 6.6 TB/s.
// w^T (contiguous along the contraction): sixteen lanes share a column instead and add up at the end.
// ---------------------------------------------------------------------------------------------
struct PvdRowsJob {
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t ldw;    // row stride of w, or of w^T
    int64_t K;
    PvdOut O;
    int splits;
    int64_t kper;   // contraction of a piece, at most PVD_RK
    int blocks;     // workgroups of a piece
    float* part;
};
enum { PVD_RK = 1024, PVD_RW = 8 };

// x's rows of [k0, k1) to LDS as float32, [row][k]; rows and k behind the end are zeros
template <int DT, int R> __device__ __forceinline__ void pvd_rows_x(const PvdRowsJob& J, int64_t k0, int64_t k1, float* xs) {
    typedef typename PvdType<DT>::T T;
    const T* x = static_cast<const T*>(J.x);
    for (int i = threadIdx.x; i < R * PVD_RK; i += 64 * PVD_RW) {
        const int r = i / PVD_RK, k = i % PVD_RK;
        if (k < ((k1 - k0 + 31) & ~31)) xs[i] = r < J.O.rows && k0 + k < k1 ? pvd_to_f32<DT>(x[r * J.ldx + k0 + k]) : 0.f;
    }
    __syncthreads();
}

template <int DT, int R> __global__ __launch_bounds__(512) void pvk_dense_rows(const PvdRowsJob J) {
    typedef typename PvdType<DT>::T T;
    enum { VEC = PvdType<DT>::VEC, COLS = 64 * VEC };
    __shared__ __attribute__((aligned(16))) float xs[R * PVD_RK];
    __shared__ __attribute__((aligned(16))) float red[PVD_RW * COLS];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int piece = blockIdx.x / J.blocks;
    const int64_t n0 = (int64_t)(blockIdx.x % J.blocks) * COLS, k0 = piece * J.kper, k1 = min(J.K, k0 + J.kper);
    pvd_rows_x<DT, R>(J, k0, k1, xs);
    float acc[R][VEC];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[r][e] = 0.f;
    const int K = (int)(k1 - k0);
    const T* w = static_cast<const T*>(J.w) + k0 * J.ldw + n0;
    // wave after wave four rows of w, eight of a lane's loads under way
    auto add = [&](const T (&v)[4][VEC], int k) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const pvd_f32x4 x4 = *reinterpret_cast<const pvd_f32x4*>(xs + r * PVD_RK + k);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[r][e] = fmaf(x4[j], pvd_to_f32<DT>(v[j][e]), acc[r][e]);
        }
    };
    const int left = (int)min((int64_t)VEC, J.O.cols - n0 - lane * VEC);
    if (left >= VEC) {
#pragma unroll 2
        for (int k = 4 * wave; k < K; k += 4 * PVD_RW) {
            alignas(16) T v[4][VEC];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (k + j < K) *reinterpret_cast<pvd_u32x4*>(v[j]) = *reinterpret_cast<const pvd_u32x4_any*>(w + (int64_t)(k + j) * J.ldw + lane * VEC);
                else *reinterpret_cast<pvd_u32x4*>(v[j]) = (pvd_u32x4){0, 0, 0, 0};
            }
            add(v, k);
        }
    } else if (left > 0) {  // the lane with the last columns; behind them the last one again, which is not stored
        for (int k = 4 * wave; k < K; k += 4 * PVD_RW) {
            T v[4][VEC];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[j][e] = w[(int64_t)min(k + j, K - 1) * J.ldw + lane * VEC + min(e, left - 1)];
#pragma unroll
            for (int j = 1; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[j][e] = k + j < K ? v[j][e] : T(0);
            add(v, k);
        }
    }
    // the waves' sums, one row of the result at a time
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= J.O.rows) break;
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
            *reinterpret_cast<pvd_f32x4*>(red + wave * COLS + lane * VEC + e) = (pvd_f32x4){acc[r][e], acc[r][e + 1], acc[r][e + 2], acc[r][e + 3]};
        __syncthreads();
        if (tid < COLS / 4) {
            pvd_f32x4 z = *reinterpret_cast<const pvd_f32x4*>(red + 4 * tid);
#pragma unroll
            for (int v = 1; v < PVD_RW; ++v) z += *reinterpret_cast<const pvd_f32x4*>(red + v * COLS + 4 * tid);
            const int64_t n = n0 + 4 * tid;
            if (J.splits == 1) pvd_finish4<DT>(J.O, r, n, z);
            else if (n < J.O.cols) pvd_store_some(J.part, 0, (piece * J.O.rows + r) * J.O.cols + n, z, pvd_left(n, J.O.cols));
        }
        __syncthreads();
    }
}

// w^T: a wave's four groups of sixteen lanes take a column each, COLS columns to a workgroup
template <int DT, int R> __global__ __launch_bounds__(512) void pvk_dense_rows_t(const PvdRowsJob J) {
    typedef typename PvdType<DT>::T T;
    enum { VEC = PvdType<DT>::VEC, COLS = 128 };
    __shared__ __attribute__((aligned(16))) float xs[R * PVD_RK];
    __shared__ __attribute__((aligned(16))) float out[R * COLS];
    const int tid = threadIdx.x, lane = tid & 15, group = tid >> 4;
    const int piece = blockIdx.x / J.blocks;
    const int64_t n0 = (int64_t)(blockIdx.x % J.blocks) * COLS, k0 = piece * J.kper, k1 = min(J.K, k0 + J.kper);
    pvd_rows_x<DT, R>(J, k0, k1, xs);
    const int K = (int)(k1 - k0);
    float acc[4][R];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) acc[c][r] = 0.f;
    // four columns of a group side by side: their loads are under way together
    for (int k = lane * VEC; k < K; k += 16 * VEC) {
        alignas(16) T v[4][VEC];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            // a column behind the last is the last again, and is not stored
            const T* p = static_cast<const T*>(J.w) + min(n0 + group + 32 * c, J.O.cols - 1) * J.ldw + k0;
            if (k + VEC <= K) {
                *reinterpret_cast<pvd_u32x4*>(v[c]) = *reinterpret_cast<const pvd_u32x4_any*>(p + k);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[c][e] = p[min(k + e, K - 1)];
#pragma unroll
                for (int e = 1; e < VEC; ++e) v[c][e] = k + e < K ? v[c][e] : T(0);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const pvd_f32x4 x4 = *reinterpret_cast<const pvd_f32x4*>(xs + r * PVD_RK + k + e);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[c][r] = fmaf(x4[j], pvd_to_f32<DT>(v[c][e + j]), acc[c][r]);
            }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float s = acc[c][r];
            for (int o = 8; o; o /= 2) s += __shfl_xor(s, o);
            if (lane == 0) out[r * COLS + group + 32 * c] = s;
        }
    __syncthreads();
    for (int i = tid; i < R * COLS / 4; i += 512) {
        const int r = i / (COLS / 4), c = i % (COLS / 4) * 4;
        if (r >= J.O.rows) return;
        const pvd_f32x4 z = *reinterpret_cast<const pvd_f32x4*>(out + r * COLS + c);
        if (J.splits == 1) pvd_finish4<DT>(J.O, r, n0 + c, z);
        else if (n0 + c < J.O.cols) pvd_store_some(J.part, 0, (piece * J.O.rows + r) * J.O.cols + n0 + c, z, pvd_left(n0 + c, J.O.cols));
    }
}

// The pieces of a split contraction, added in a fixed order, and what follows the product.  G lanes share four columns when
// there are many pieces of a small result: lane g adds pieces g, g + G, ..., the G sums are added in turn.
// Bound by its launch and the pieces' way from the L2: 4 to 5 us (eight pieces of 512 x 512 in float32 4.6).
template <int DT, int G> __global__ __launch_bounds__(256) void pvk_dense_join(const PvdOut O, const float* __restrict__ part, int pieces) {
    const int64_t quads = (O.cols + 3) / 4, i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool in = i < O.rows * quads;
    const int64_t m = in ? i / quads : 0, n = in ? i % quads * 4 : 0;
    pvd_f32x4 z = {0.f, 0.f, 0.f, 0.f};
    const int left = pvd_left(n, O.cols);
#pragma unroll 4
    for (int p = threadIdx.x % G; p < pieces; p += G) z += pvd_load_some(part, 0, (p * O.rows + m) * O.cols + n, left);
#pragma unroll
    for (int o = G / 2; o; o /= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] += __shfl_down(z[e], o, G);
    if (in && threadIdx.x % G == 0) pvd_finish4<DT>(O, m, n, z);
}

// ---------------------------------------------------------------------------------------------
// Gradients, one launch: the first workgroups make dx (x-side operand g, contraction over n), the next dw (rows of x^T,
// contraction over m), the last 64 columns of dbias (and dpre) each.  g = dy f'(pre) is formed anew by every workgroup on the
// way to the matrix instructions: for small layers a second launch costs more than that.  32 x 128 x 128 in float32: 6.0 us;
// 1 x 32 x 10589 in bf16: 15.2 us.  Bound by the round trips to memory and the launch.
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

// 64 columns of dbias (and of dpre): the workgroup's waves take rows in turn
template <int DT> __device__ __forceinline__ void pvd_bias_job(const PvdBwdJob& J, int64_t block, float* red) {
    typedef typename PvdType<DT>::T T;
    const int c = threadIdx.x & 63, g = threadIdx.x >> 6;
    const int64_t n = block * 64 + c;
    float s = 0.f;
    if (n < J.n) {
#pragma unroll 4
        for (int64_t m = g; m < J.m; m += PVD_SW) {
            float v = pvd_to_f32<DT>(static_cast<const T*>(J.dy)[m * J.lddy + n]);
            if (J.act != PVD_LINEAR) v *= pvd_act_grad(J.pre[m * J.ldp + n], J.act);
            if (J.dpre) J.dpre[m * J.n + n] = v;
            s += v;
        }
    }
    red[threadIdx.x] = s;
    __syncthreads();
    if (g == 0 && n < J.n && J.dbias) {
#pragma unroll
        for (int w = 1; w < PVD_SW; ++w) s += red[64 * w + c];
        static_cast<T*>(J.dbias)[n] = pvd_from_f32<DT>(s);
    }
}

template <int DT> __global__ __launch_bounds__(512) void pvk_dense_bwd_slim(const PvdBwdJob J) {
    __shared__ __attribute__((aligned(16))) float red[PVD_SW * PVD_SM * PVD_SN];
    int64_t b = blockIdx.x;
    if (b < J.n_dx) return pvd_slim_job<DT, true, false>(J.dx, b, red);
    b -= J.n_dx;
    if (b < J.n_dw) return pvd_slim_job<DT, false, true>(J.dw, b, red);
    pvd_bias_job<DT>(J, b - J.n_dw, red);
}

// ---------------------------------------------------------------------------------------------
// Large products, step 1: operands that the product kernel below cannot read as they are -- rows not aligned to sixteen bytes,
// or a contraction that is no multiple of 128 bytes -- are laid out anew, and g is formed from dy and z, once instead of once
// per tile: a source of R rows of C contiguous elements becomes [pad(R)][pad(C)] or its transpose [C][pad(R)], zeros behind the
// end.  One launch for up to three sources; bound by memory: dy and z of 4096 x 4096 in bf16 to both terms of g, with
// db's partial sums, 33 us (168 MB, 5.1 TB/s); of 2504 x 512 in float32 10 us, most of it launch and round trip.
// ---------------------------------------------------------------------------------------------
struct PvdPack {
    const void* p;
    int64_t R, C, ld;
    const float* pre;  // g = p * act'(pre)
    int64_t ldp;
    int act;
    void* same;        // [h_same][ld_same], the first w_same elements of a row filled, or NULL
    void* low;         // g's second terms, laid out as `same`, which holds the first; or NULL
    int64_t ld_same, w_same, h_same;
    void* tran;        // [C][ld_tran], w_tran of a row filled, or NULL
    int64_t ld_tran, w_tran;
    float* sums;       // [row tiles][C]: column sums of 64 rows each, or NULL
    float* g32;        // [R][C] float32: g unrounded, or NULL
    int rt, ct;        // tiles of 64 x 64
};
struct PvdPacks {
    int n, first[4];
    PvdPack job[3];
};

template <int DT> __global__ __launch_bounds__(256) void pvk_dense_pack(const PvdPacks P) {
    typedef typename PvdType<DT>::T T;
    enum { VEC = PvdType<DT>::VEC, PER = 64 / VEC, LD = 64 + (DT == PVD_F32 ? 1 : 2) };
    __shared__ T tile[64 * LD];
    __shared__ float colsum[4][64];
    int j = 0;
    while (j + 1 < P.n && (int)blockIdx.x >= P.first[j + 1]) ++j;
    const PvdPack& J = P.job[j];
    const int b = blockIdx.x - P.first[j], tid = threadIdx.x;
    const int64_t r0 = (int64_t)(b / J.ct) * 64, c0 = (int64_t)(b % J.ct) * 64;
    const T* p = static_cast<const T*>(J.p);
    T* same = static_cast<T*>(J.same);
    // runs of VEC columns: PER runs a row, 256 / PER rows at a time
    const int run = tid % PER, row = tid / PER;
    float sum[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
#pragma unroll
    for (int rr = row; rr < 64; rr += 256 / PER) {
        const int64_t r = r0 + rr, c = c0 + run * VEC;
        alignas(16) T v[VEC], lo[VEC];
        float f[VEC];
        const bool whole = r < J.R && c + VEC <= J.C;
        if (whole) {
            *reinterpret_cast<pvd_u32x4*>(v) = *reinterpret_cast<const pvd_u32x4_any*>(p + r * J.ld + c);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = r < J.R && c + e < J.C ? p[r * J.ld + c + e] : T(0);
        }
        if (J.sums || J.g32 || (J.pre && J.act != PVD_LINEAR)) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = pvd_to_f32<DT>(v[e]);
            if (J.pre && J.act != PVD_LINEAR) {
                alignas(16) float z[VEC];
                if (whole) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 4) *reinterpret_cast<pvd_f32x4*>(z + e) = pvm_load4(J.pre, 0, r * J.ldp + c + e);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) z[e] = r < J.R && c + e < J.C ? J.pre[r * J.ldp + c + e] : 0.f;
                }
#pragma unroll
                for (int e = 0; e < VEC; e += 4) {
                    const pvd_f32x4 d4 = pvd_act_grad4(*reinterpret_cast<const pvd_f32x4*>(z + e), J.act);
#pragma unroll
                    for (int i = e; i < e + 4; ++i) {
                        f[i] = r < J.R && c + i < J.C ? f[i] * d4[i - e] : 0.f;
                        if constexpr (DT == PVD_F32) v[i] = f[i];
                        else pvd_terms<DT>(f[i], v[i], lo[i]);
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum[e] += f[e];
            if (J.g32)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (r < J.R && c + e < J.C) J.g32[r * J.C + c + e] = f[e];
        }
        if (same && r < J.h_same && c < J.w_same) {
            *reinterpret_cast<pvd_u32x4*>(same + r * J.ld_same + c) = *reinterpret_cast<const pvd_u32x4*>(v);
            if (DT != PVD_F32 && J.low) *reinterpret_cast<pvd_u32x4*>(static_cast<T*>(J.low) + r * J.ld_same + c) = *reinterpret_cast<const pvd_u32x4*>(lo);
        }
        if (J.tran)
#pragma unroll
            for (int e = 0; e < VEC; ++e) tile[rr * LD + run * VEC + e] = v[e];
    }
    if (J.tran) {
        T* tran = static_cast<T*>(J.tran);
        __syncthreads();
        for (int cc = row; cc < 64; cc += 256 / PER) {  // here a run is VEC rows of one column
            const int64_t c = c0 + cc, r = r0 + run * VEC;
            alignas(16) T v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = tile[(run * VEC + e) * LD + cc];
            if (c < J.C && r < J.w_tran) *reinterpret_cast<pvd_u32x4*>(tran + c * J.ld_tran + r) = *reinterpret_cast<const pvd_u32x4*>(v);
        }
    }
    if (J.sums) {
        // lanes of a wave that hold the same columns are PER apart
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            for (int o = PER; o < 64; o *= 2) sum[e] += __shfl_xor(sum[e], o);
            if ((tid & 63) < PER) colsum[tid >> 6][run * VEC + e] = sum[e];
        }
        __syncthreads();
        if (tid < 64 && c0 + tid < J.C)
            J.sums[(r0 / 64) * J.C + c0 + tid] = (colsum[0][tid] + colsum[1][tid]) + (colsum[2][tid] + colsum[3][tid]);
    }
}

// ---------------------------------------------------------------------------------------------
// Large products, step 2.  A step is 128 bytes of contraction per row of either operand.  LDS holds ST of them: while the
// matrix instructions work on one, the next arrive from memory (global_load_lds, no registers in between).
//   An operand whose rows run along the contraction lies in LDS row by row, a row of 128 bytes as eight pieces of sixteen; piece
// c of row r is at slot c ^ ((r >> 1) & 7), which spreads the sixteen rows a quarter wave reads over all banks.
//   An operand whose rows run along the other side (Keras' w in the forward, x^T and g in dw) lies there as it does in memory,
// one line of contraction after another.  16-bit types are transposed on the way to registers (ds_read_b64_tr_b16: sixteen
// lanes hold four lines of sixteen elements and get four lines of one element each), float32 is read element by element.
// Pairs of pieces (float32: runs of four) of a line are exchanged by the line's number so that the lines which are read
// together lie in different banks.
// The direct loads write lane after lane, so the lanes choose their source accordingly.
//   Measured (200 calls in a row; from idle a tenth more, in a long run less, as a library product's 123 to 103 us): 4096 x
// 4096 x 4096 bf16 with bias, SiLU, residual and z 145 us = 950 TFLOP/s, without them 133 us = 1.04 PFLOP/s (a library product
// 1.12 to 1.34); both gradient products of 4096 x 2048 x 4096 in one launch 146 us = 940, with g in two terms 261 us, 1.05 PFLOP/s of
// matrix work; 2504 x 128 x 100000 float32 with sigmoid 672 us = 95 TFLOP/s, 1.6 TB/s (a library product: 150 TFLOP/s; here a
// tile has four steps only, and 1 GB of results takes a sigmoid each).  By counters the matrix pipe is busy 46 % of the first
// kernel's time, 50 % with two terms, 62 % in the float32 one, LDS is read 36 % (none of it in bank conflicts), and what is
// staged would take 46 % of it at 64 bytes a clock and CU: no unit is at its limit.  What bounds it are the waits of a step on
// each other and the results' way out, which the CU's other workgroup hides only partly.
//   Tiles are numbered so that the workgroups of one XCD (blockIdx % 8) work on neighbouring tiles and find each other's
// operands in their L2.
// ---------------------------------------------------------------------------------------------
struct PvdNtJob {
    const char *x, *w;      // [x_rows][steps * 128 bytes], row strides ldx, ldw in bytes; across: [contraction][x_rows]
    int64_t ldx, ldw;
    int x_rows, w_rows;
    int x_across, w_across;
    int64_t x_low, w_low;   // TWO: from g's first terms to its second, in bytes, on the side that is g; 0 on the other
    int steps, per, splits; // steps of 128 bytes; of each piece; pieces
    int mt, nt, band;       // tiles; rows of tiles that go together
    PvdOut O;
    float* part;            // splits > 1: [piece][rows][cols] float32
};
struct PvdNtJobs {
    int n, first[3];        // first workgroup of each product; of the column sums behind them
    PvdNtJob job[2];
    const float* sums;      // [sum_tiles][sum_cols] -> dbias
    int sum_tiles;
    int64_t sum_cols;
    void* dbias;
};

typedef __attribute__((address_space(3))) void* pvd_lptr;
typedef short pvd_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pvd_s16x4* pvd_ltr;

// Lane l's sixteen bytes at `from` go to lds + 16 l (lds: the same for the wave).  Written out because the compiler, given its
// builtin, waits for every such load in flight before each transposing read of LDS (128 x 256 bf16 tiles: 165 us instead of
// 121 for 4096^3); the loads are waited for in PvdNt::arrived, and write no registers.
__device__ __forceinline__ void pvd_load_to_lds(const char* from, char* lds) {
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(pvd_lptr)lds);
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is the compiler's own and not kept across this: so it is meant
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(from) : "memory", "m0");
#pragma clang diagnostic pop
}

// What follows the product for ROWS x 64 products of one wave in LDS (row r's piece u of four floats at slot u ^ (r & 15)):
// rows m .., columns n ..; the residuals of several rows are asked for together.
template <int DT, int ROWS> __device__ __forceinline__ void pvd_finish_rows(const PvdOut& O, int64_t m, int64_t n, const float* ep) {
    typedef typename PvdType<DT>::T T;
    const int lane = threadIdx.x & 63, er = lane >> 4, eu = lane & 15;  // sixteen lanes, four columns each, on a row
    const int64_t c = n + 4 * eu;
    if (m + ROWS <= O.rows && n + 64 <= O.cols) {
        // all of it is there: nothing but the work itself (its addresses and tests took as long as a third of the products at
        // k = 128 in float32)
        pvd_f32x4 b4 = {0.f, 0.f, 0.f, 0.f};
        if (O.bias) b4 = pvm_load4(O.bias, DT, c);
        const T* rp = static_cast<const T*>(O.res) + (m + er) * O.ldr + c;
        float* zp = O.pre + (m + er) * O.ldp + c;
        T* yp = static_cast<T*>(O.y) + (m + er) * O.ldy + c;
        const int64_t rs = 4 * O.ldr, zs = 4 * O.ldp, ys = 4 * O.ldy;
#pragma unroll 1
        for (int i0 = 0; i0 < ROWS / 4; i0 += 4) {
            pvd_f32x4 r4[4];
            if (O.res)
#pragma unroll
                for (int i = 0; i < 4; ++i, rp += rs) r4[i] = pvm_load4(rp, DT, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 4 * (i0 + i) + er;
                pvd_f32x4 z = *reinterpret_cast<const pvd_f32x4*>(ep + r * 64 + ((eu ^ (4 * i | er)) << 2));
                z += b4;
                if (O.pre) {
                    pvm_store4(zp, 0, 0, z);
                    zp += zs;
                }
                pvd_f32x4 o = pvd_act4(z, O.act);
                if (O.res) o += r4[i];
                pvm_store4(yp, DT, 0, o);
                yp += ys;
            }
        }
        return;
    }
#pragma unroll 1
    for (int r = er; r < ROWS; r += 4)
        pvd_finish4<DT>(O, m + r, c, *reinterpret_cast<const pvd_f32x4*>(ep + r * 64 + ((eu ^ (r & 15)) << 2)));
}

// EDGE: of the tile (x's rows, the weights' columns); WM x WN: waves; ST: steps that LDS holds, two or
// four; TWO: one side is g in two terms, and a piece's steps are gone through once with each
template <int DT, int EDGE, int WM, int WN, int ST, bool TWO> struct PvdNt {
    enum { WAVES = WM * WN, THREADS = 64 * WAVES, SIDE = EDGE * 128, BUF = 2 * SIDE, LDS = ST * BUF };
    enum { ROWS = EDGE / WM, FM = ROWS / 16, FN = EDGE / WN / 16 };  // a wave's rows, its fragments of either side
    enum { LOADS = 2 * EDGE / (8 * WAVES) };                         // direct loads of a wave per step
    static_assert(EDGE % (8 * WAVES) == 0, "rows are loaded eight per wave");
    static_assert(FN % 4 == 0 && LDS >= WAVES * ROWS * 256, "a wave's result goes out through its share of LDS");
    static_assert(ST == 2 || ST == 4, "what `arrived` waits for");

    enum { SIZE = PvdType<DT>::SIZE, VEC = PvdType<DT>::VEC, KST = 128 / SIZE };  // KST: contraction of a step

    // the exchange of pieces of line k of an operand across, in pieces
    static __device__ __forceinline__ int across_swap(int k) { return DT == PVD_F32 ? 4 * ((k >> 2) & 3) : 2 * ((k & 3) | ((k >> 3 & 1) << 2)); }
    // What this lane loads of rows [row0, row0 + EDGE) and step s: a step's rows are EDGE / 8 loads of a wave, load i lies at
    // i * 1024 in LDS.  Rows behind the end repeat the last ones (their results are dropped).
    template <bool ACROSS> struct Source {
        enum { N = EDGE / (8 * WAVES) };
        const char* at[N];
        int64_t step;
        __device__ __forceinline__ Source(const char* p, int64_t ld, int rows, int row0, int s) {
            const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
            step = ACROSS ? KST * ld : 128;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int i = u * WAVES + wave;
                if constexpr (ACROSS) {
                    enum { PIECES = EDGE * SIZE / 16, LINES = 64 / PIECES };  // pieces of a line, lines of a load
                    const int k = i * LINES + lane / PIECES, piece = (lane % PIECES) ^ across_swap(k);
                    at[u] = p + k * ld + (int64_t)min(row0 + piece * VEC, rows - VEC) * SIZE;
                } else {
                    const int r = min(row0 + 8 * i + (lane >> 3), rows - 1), piece = (lane & 7) ^ (4 * (i & 1) | (lane >> 4));
                    at[u] = p + r * ld + piece * 16;
                }
                at[u] += s * step;
            }
        }
        __device__ __forceinline__ void move(int64_t bytes) {
#pragma unroll
            for (int u = 0; u < N; ++u) at[u] += bytes;
        }
        __device__ __forceinline__ void load(char* lds) {  // and on to the next step
#pragma unroll
            for (int u = 0; u < N; ++u) {
                pvd_load_to_lds(at[u], lds + (u * WAVES + (threadIdx.x >> 6)) * 1024);
                at[u] += step;
            }
        }
    };
    // the fragment of rows row0 .. row0 + 15 (a multiple of sixteen) and half h of a step
    template <bool ACROSS> static __device__ __forceinline__ pvd_u32x4 fragment(const char* lds, int row0, int h) {
        const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
        if constexpr (!ACROSS) {
            return piece(lds, row0 + r16, 4 * h + q);
        } else if constexpr (DT == PVD_F32) {
            const char* at = lds + (16 * h + 4 * q) * (EDGE * 4) + ((((row0 + r16) >> 2) ^ 4 * q) << 4) + (r16 & 3) * 4;
            pvd_u32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const unsigned*>(at + e * (EDGE * 4));
            return v;
        } else {
            const int k = 32 * h + 8 * q + (r16 >> 2);  // this lane's line of the first four; k + 4 has the same exchange
            const char* at = lds + k * (EDGE * 2) + (((row0 >> 3) ^ across_swap(k)) << 4) + (r16 & 3) * 8;
            const pvd_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pvd_ltr)at);
            const pvd_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pvd_ltr)(at + 4 * (EDGE * 2)));
            return __builtin_bit_cast(pvd_u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    // all but the last `steps` steps that this wave has asked for have arrived, its own reads of LDS too; then every wave's
    static __device__ __forceinline__ void arrived(int steps) {
        if (ST == 4 && steps >= 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * LOADS) : "memory");
        else if (ST == 4 && steps == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    static __device__ __forceinline__ void same_wave() {  // LDS written by lanes of this wave is read by others of it
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    static __device__ __forceinline__ pvd_u32x4 piece(const char* lds, int r, int c) {
        return *reinterpret_cast<const pvd_u32x4*>(lds + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
    }

    template <bool XA, bool WA> static __device__ __forceinline__ void run(const PvdNtJob& J, int block, char* smem) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
        const int tiles = J.mt * J.nt, total = tiles * J.splits;
        // an XCD's workgroups, block % 8 apart, take consecutive tiles
        const int xcd = block & 7, each = total >> 3, more = total & 7;
        int t = xcd * each + min(xcd, more) + (block >> 3);
        const int pc = t / tiles;
        t -= pc * tiles;
        const int per_band = J.band * J.nt, bi = t / per_band, in = t - bi * per_band, bh = min(J.band, J.mt - bi * J.band);
        const int m0 = (bi * J.band + in % bh) * EDGE, n0 = in / bh * EDGE;
        const int s0 = pc * J.per, len = min(J.steps, s0 + J.per) - s0, steps = TWO ? 2 * len : len;
        const int wm = (wave % WM) * ROWS, wn = (wave / WM) * (EDGE / WN);
        pvd_f32x4 acc[FN][FM];
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int k = 0; k < FM; ++k) acc[i][k] = (pvd_f32x4){0.f, 0.f, 0.f, 0.f};
        Source<XA> sx(J.x, J.ldx, J.x_rows, m0, s0);
        Source<WA> sw(J.w, J.ldw, J.w_rows, n0, s0);
        // TWO: the second terms first, so that what infinities of the other side make of them can be dropped
        if (TWO) sx.move(J.x_low), sw.move(J.w_low);
        int asked = 0;
        auto get = [&](int slot) {
            sx.load(smem + slot * BUF);
            sw.load(smem + slot * BUF + SIDE);
            if (TWO && ++asked == len) {  // the piece once more, with the first terms
                sx.move(-J.x_low - len * sx.step);
                sw.move(-J.w_low - len * sw.step);
            }
        };
        auto each_sum = [&](auto f) {
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int k = 0; k < FM; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][k][e] = f(acc[i][k][e]);
        };
        // A step is two halves.  The fragments of one are read from LDS while the other is multiplied, a quarter into it --
        // across steps too: behind the first quarter of a step's second half the waves meet, and the next step's first fragments
        // come in under the rest.
        pvd_u32x4 a[2][FN], b[2][FM];
        auto read = [&](const char* lds, int h) {
#pragma unroll
            for (int i = 0; i < FN; ++i) a[h][i] = fragment<WA>(lds + SIDE, wn + 16 * i, h);
#pragma unroll
            for (int k = 0; k < FM; ++k) b[h][k] = fragment<XA>(lds, wm + 16 * k, h);
        };
        auto multiply = [&](int h, int from, int to) {
            if constexpr (DT == PVD_F32) {  // the four products of a fragment apart from each other: each adds to what the last one left
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int u = from; u < to; ++u) {
                        const int k = u / FN, i = u % FN;
                        acc[i][k] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[h][i][e]), __uint_as_float(b[h][k][e]), acc[i][k], 0, 0, 0);
                    }
            } else {
#pragma unroll
                for (int u = from; u < to; ++u) {
                    const int k = u / FN, i = u % FN;
                    acc[i][k] = pvd_mfma16<DT>(a[h][i], b[h][k], acc[i][k]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        enum { HALVES = 2, EACH = FN * FM, FIRST = EACH / 4 };
#pragma unroll
        for (int j = 0; j < ST - 1; ++j)
            if (j < steps) get(j);
        arrived(min(ST - 2, steps - 1));
        read(smem, 0);
        int cur = 0;
        for (int s = 0; s < steps; ++s) {
            const char* lds = smem + cur * BUF;
            if (s + ST - 1 < steps) get(cur == 0 ? ST - 1 : cur - 1);
#pragma unroll
            for (int h = 0; h < HALVES - 1; ++h) {
                multiply(h, 0, FIRST);
                read(lds, h + 1);
                __builtin_amdgcn_sched_barrier(0);
                multiply(h, FIRST, EACH);
            }
            multiply(HALVES - 1, 0, FIRST);
            cur = cur + 1 == ST ? 0 : cur + 1;
            if (s + 1 < steps) {
                arrived(min(ST - 2, steps - 2 - s));
                read(smem + cur * BUF, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            multiply(HALVES - 1, FIRST, EACH);
            if (TWO && s + 1 == len)  // behind the second terms
                each_sum([](float a) { return fabsf(a) < __builtin_inff() ? a * PvdTerms<DT>::LOW : 0.f; });
        }
        if (TWO && PvdTerms<DT>::UNIT != 1.f) each_sum([](float a) { return a * PvdTerms<DT>::UNIT; });
        arrived(0);
        // through LDS, 64 columns at a time, so that sixteen lanes read and write consecutive columns of a row; the sixteen pieces of
        // a row of 64 floats are spread by the row's number
        float* ep = reinterpret_cast<float*>(smem) + wave * ROWS * 64;
#pragma unroll
        for (int i0 = 0; i0 < FN; i0 += 4) {
#pragma unroll
            for (int k = 0; k < FM; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<pvd_f32x4*>(ep + (16 * k + r16) * 64 + (((4 * i + q) ^ r16) << 2)) = acc[i0 + i][k];
            same_wave();
            const int64_t m = m0 + wm, n = n0 + wn + 16 * i0;
            if (J.splits == 1) {
                pvd_finish_rows<DT, ROWS>(J.O, m, n, ep);
            } else {
                for (int row = lane >> 4; row < ROWS && m + row < J.O.rows; row += 4) {
                    const int u = lane & 15;
                    const pvd_f32x4 z = *reinterpret_cast<const pvd_f32x4*>(ep + row * 64 + ((u ^ (row & 15)) << 2));
                    if (n + 4 * u < J.O.cols)
                        pvd_store_some(J.part, 0, (pc * J.O.rows + m + row) * J.O.cols + n + 4 * u, z, pvd_left(n + 4 * u, J.O.cols));
                }
            }
            same_wave();
        }
    }
};

template <int DT, int EDGE, int WM, int WN, int ST, bool TWO>
__global__ __launch_bounds__(64 * WM * WN) void pvk_dense_nt(const PvdNtJobs P) {
    extern __shared__ __attribute__((aligned(1024))) char pvd_smem[];
    typedef typename PvdType<DT>::T T;
    const int b = blockIdx.x;
    if (b < P.first[2]) {
        const int j = b >= P.first[1];
        typedef PvdNt<DT, EDGE, WM, WN, ST, TWO> K;
        const PvdNtJob& J = P.job[j];
        if (!J.w_across) return K::template run<false, false>(J, b - P.first[j], pvd_smem);
        if (!J.x_across) return K::template run<false, true>(J, b - P.first[j], pvd_smem);
        return K::template run<true, true>(J, b - P.first[j], pvd_smem);
    }
    const int64_t c = (int64_t)(b - P.first[2]) * blockDim.x + threadIdx.x;
    if (c >= P.sum_cols) return;
    float s = 0.f;
    for (int i = 0; i < P.sum_tiles; ++i) s += P.sums[i * P.sum_cols + c];
    static_cast<T*>(P.dbias)[c] = pvd_from_f32<DT>(s);
}
