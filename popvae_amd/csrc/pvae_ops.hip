// pvae_ops.hip -- the operators of include/pvae_ops.h: argument checks, choice of kernel, launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <new>
#include <string>
#include <utility>
#include <vector>

#include "../../include/pvae_ops.h"
#include "pvae_dense.h"
#include "pvae_multi.h"

namespace {

thread_local char g_err[512];

int refuse(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return code;
}
int launched(const char* what) {
    const hipError_t s = hipGetLastError();
    return s == hipSuccess ? 0 : refuse(-11, "launch of %s failed: %s", what, hipGetErrorString(s));
}

int esize(int dt) { return dt == PVAE_F32 ? 4 : 2; }
bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes == 0; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// [rows][cols] with a row stride: the strides the kernels' 64-bit offsets hold
int check_matrix(const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld, int size) {
    if (rows == 0 || cols == 0) return 0;
    if (!p) return refuse(-1, "%s is NULL", name);
    if (!aligned(p, size)) return refuse(-2, "%s is not aligned to its %d-byte elements", name, size);
    if (ld < cols && rows > 1) return refuse(-2, "%s: row stride %lld below the row's %lld elements", name, (long long)ld, (long long)cols);
    if (rows > 1 && ld > (int64_t(1) << 60) / rows / size) return refuse(-2, "%s: row stride %lld too large", name, (long long)ld);
    return 0;
}
int check_sizes(int32_t dtype, int32_t act, int64_t m, int64_t k, int64_t n) {
    if (dtype < PVAE_F32 || dtype > PVAE_F16) return refuse(-2, "unknown type %d", dtype);
    if (act < PVAE_LINEAR || act > PVAE_GELU) return refuse(-2, "unknown activation %d", act);
    const int64_t top = int64_t(1) << 31;
    if (m < 0 || k < 0 || n < 0 || m >= top || k >= top || n >= top)
        return refuse(-2, "sizes m = %lld, k = %lld, n = %lld: 0 .. 2^31 - 1 each", (long long)m, (long long)k, (long long)n);
    return 0;
}
int check_weights(const void* w, int64_t k, int64_t n, int64_t sk, int64_t sn, int size) {
    if (k == 0 || n == 0) return 0;
    if (sn == 1 || n == 1) return check_matrix("w", w, k, n, sk, size);
    if (sk == 1 || k == 1) return check_matrix("w^T", w, n, k, sn, size);
    return refuse(-2, "w: neither rows nor columns are contiguous (strides %lld, %lld)", (long long)sk, (long long)sn);
}

int check_workspace(const char* what, const void* p, int64_t have, int64_t need) {
    if (need == 0) return 0;
    if (!p || have < need) return refuse(-8, "%s needs a workspace of %lld bytes (got %lld)", what, (long long)need, (long long)(p ? have : 0));
    if (!aligned(p, 16)) return refuse(-2, "the workspace is not aligned to 16 bytes");
    return 0;
}
int check_grid(int64_t blocks) {
    if (blocks > 0x7fffffff) return refuse(-2, "%lld workgroups: the operands are too large for one launch", (long long)blocks);
    return 0;
}

// The bytes of a matrix: `rows` runs of `width`, `pitch` apart (pitch 0: one row for all).  An output may not meet another
// output or an input, but may lie between the rows of one: column ranges of one buffer are apart.
struct Extent {
    const char* name;
    uintptr_t lo, hi;
    int64_t rows;
    uintptr_t pitch, width;
};
Extent extent(const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld, int size) {
    if (!p || rows == 0 || cols == 0) return {name, 0, 0, 0, 0, 0};
    if (ld == 0) rows = 1;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(p), pitch = (uintptr_t)(ld * size), width = (uintptr_t)(cols * size);
    return {name, lo, lo + (uintptr_t)(rows - 1) * pitch + width, rows, pitch, width};
}
bool meet(const Extent& a, const Extent& b) {
    if (a.lo >= b.hi || b.lo >= a.hi) return false;
    if (a.lo > b.lo) return meet(b, a);
    if ((a.rows == 1 && b.rows == 1) || (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch)) return true;
    // b's runs begin `d` behind those of a (a single row's, too), all `pitch` apart
    const uintptr_t pitch = a.rows > 1 ? a.pitch : b.pitch, d = (b.lo - a.lo) % pitch;
    return d < a.width || d + b.width > pitch;
}
int check_apart(const Extent* e, int n_out, int n) {  // e[0 .. n_out) are outputs
    for (int i = 0; i < n_out; ++i)
        for (int j = i + 1; j < n; ++j)
            if (meet(e[i], e[j])) return refuse(-2, "%s overlaps %s", e[i].name, e[j].name);
    return 0;
}
Extent weights_extent(const void* w, int64_t k, int64_t n, int64_t sk, int64_t sn, int size) {
    return sn == 1 || n == 1 ? extent("w", w, k, n, sk, size) : extent("w", w, n, k, sn, size);
}

// Arguments that passed their checks, as the choice of kernel and all plans take them: w with a single row or column may come
// with any strides, and the one that is never used becomes 1, so that one of the two always is.
template <typename Args> Args plain(const Args& a) {
    Args b = a;
    if (b.w_sk != 1 && b.w_sn != 1) (b.n == 1 ? b.w_sn : b.w_sk) = 1;
    return b;
}
// an operand of the tile and slim kernels: rows x K, one of the strides 1
PvdOperand operand(const void* p, int64_t rows, int64_t sr, int64_t sk) {
    PvdOperand o{};
    o.p = p;
    o.rows = rows;
    o.sr = sr;
    o.sk = sk;
    return o;
}
void with_grad(PvdOperand& o, const float* pre, int64_t pr, int64_t pk, int act) {
    o.pre = pre;
    o.pr = pr;
    o.pk = pk;
    o.act = act;
}
PvdOut output(int64_t rows, int64_t cols, void* y, int64_t ldy, const void* bias, const void* res, int64_t ldr, float* pre, int64_t ldp,
              int act) {
    return {rows, cols, y, ldy, bias, res, ldr, pre, ldp, act};
}

// R rows of C contiguous elements as an operand that the large kernel reads as it lies: along the contraction, or across it
bool lies_well(const void* p, int64_t R, int64_t C, int64_t ld, int size, bool along) {
    return aligned(p, 16) && (R <= 1 || ld * size % 16 == 0) && (along ? C * size % 128 == 0 : R * size % 128 == 0 && C * size % 16 == 0);
}
// Which kernel makes y (microseconds, float32 / bf16, w as Keras keeps it):
//                        rows         slim         tile         large
//      1 x  512 x  512    7.7 /  8.1   5.9 /  5.5  11.1 /  9.4  15.0 /  9.0
//      1 x   16 x 20000   4.1 /  4.3   6.5 / 11.7   6.8 /  6.4   9.9 /  9.8
//      1 x 2000 x  128    7.5 /  8.3   9.1 / 10.8  13.9 / 11.2  15.6 / 13.8
//      1 x 4096 x 4096   21.2 / 10.9  27.8 / 27.1  37.4 / 18.0  29.4 / 14.4
//      2 x 100000 x 3    17.0 / 23.8  11.2 / 12.2  25.0 / 17.1  26.2 / 20.1
//      4 x 8192 x 4096   32.8 / 22.1  49.9 / 48.2  64.7 / 26.6  48.8 / 18.9
//      8 x 3159 x 6998   29.1 / 37.8  40.1 / 36.3  64.7 / 31.4  71.1 / 38.5
//      8 x  512 x 100000 41.9 / 40.6  64.3 / 72.4  84.5 / 35.7  72.7 / 27.1
//     32 x 1024 x 1024                 9.4 /  8.1  13.4 / 10.9  12.8 / 16.5
//    256 x  512 x  512                 7.4 /  6.4  13.0 / 10.6  16.4 / 12.7
//     64 x 4096 x 4096                55.7 / 45.2  39.9 / 19.6  34.6 / 17.0
//   1000 x   16 x 4000                34.1 / 75.2  13.2 / 14.5  15.1 / 14.2
//   1000 x  128 x 1000                14.9 / 18.1  11.8 /  9.0   9.5 / 11.1
//                   ... k or n odd: w is laid out anew first
//     16 x 3216 x 2854                23.0 / 21.0  33.8 / 20.3  42.4 / 26.1
//     32 x  100 x 20000                9.4 / 13.0  13.5 /  9.1  18.3 / 15.1
//     64 x 4001 x 4001                             50.1 / 28.5  62.8 / 36.0
//    256 x 2401 x 1000                             28.5 / 18.1  33.1 / 21.1
//    512 x 4001 x 4001                            289.3 / 124.8 181.3 / 51.7
enum Kernel { ROWS, SLIM, TILE, LARGE };
Kernel dense_kernel(const pvae_dense_args& a) {
    const int64_t m = a.m, k = a.k, n = a.n;
    const int size = esize(a.dtype);
    // small results: the slim kernel's workgroups all find room, and what they read over and over (48 rows of contraction each)
    // stays small
    const int64_t slim = ceil_div(m, PVD_SM) * ceil_div(n, PVD_SN), reads = slim <= (size == 4 ? 1024 : 512) ? slim * 48 * k : INT64_MAX;
    // a few rows: the weights pass once, and the contraction is split over the chip and joined in a second launch.  The slim
    // kernel makes a small result in one (less than 4096 bytes of contraction), and needs far fewer pieces of a very long
    // contraction (w^T, whose columns it reads sixteen bytes at a time, sooner: 1 x 700 x 8000 9.0 us, rows 10.6); below 128 the
    // rows kernel does not split either.  16-bit products of more than two rows over long contractions cost the rows kernel
    // more arithmetic than reading.
    if (m <= 4 && k > 0) {
        if ((k * size < 4096 || k >= 16384) && (m > 2 || k >= 128) && reads <= int64_t(a.w_sk == 1 ? 20 : 8) << 20) return SLIM;
        if (size == 4 || m <= 2 || k < 4096) return ROWS;
    }
    if (reads <= int64_t(size == 4 ? 16 : 12) << 20) return SLIM;
    // up to eight float32 rows over large weights (16-bit ones: the large kernel is as good)
    if (size == 4 && m <= 8 && (double)k * n >= (a.w_sk == 1 ? 48 : 16) * 1048576.0) return ROWS;
    // where the large kernel would lay w out first, a few rows do not repay it: up to 32 the slim kernel reads w once as well,
    // up to 64 the tile kernel
    const bool lies = a.w_sk == 1 ? lies_well(a.w, n, k, a.w_sn, size, true) : lies_well(a.w, k, n, a.w_sk, size, false);
    if (size == 4 && m <= (lies ? 16 : 32) && (k >= 256 || (!lies && k >= 64 && slim <= 2048))) return SLIM;
    if (!lies && m <= 64) return TILE;
    // a short contraction never fills the large kernel's pipeline; 16-bit products are over sooner, but it reads large weights
    // faster than the tile kernel (5 x 512 x 100000 bf16: 27 and 36 us)
    const double work = (double)m * n * k;
    if (size == 4 ? k >= 64 && (lies || work >= 536870912.0) : lies ? k >= 1024 || work >= 536870912.0 || (double)k * n >= 8388608.0 : work >= 1073741824.0) return LARGE;
    return TILE;
}
// The gradients: slim while what its workgroups read stays small (every value of g is formed anew for each), else large, which
// forms g once (float32 / bf16, GELU, in a graph: 100 x 256 x 256 slim 8.6 / 11.0 us, large 16.4 / 18.4; 100 x 600 x 600:
// 16.7 / 30.7 and 20.3 / 21.6; 256 x 512 x 512: 28.4 / 40.7 and 22.4 / 22.5; 32 x 512 x 4000: 45.6 / 87.4 and 20.6 / 21.4; 4000 x 64
// x 64, where the slim kernel sums db over long columns: 190 / 226 and 26.2 / 24.6)
Kernel bwd_kernel(const pvae_dense_bwd_args& a) {
    const int64_t dx = a.dx ? ceil_div(a.m, PVD_SM) * ceil_div(a.k, PVD_SN) : 0, dw = a.dw ? ceil_div(a.k, PVD_SM) * ceil_div(a.n, PVD_SN) : 0;
    const int64_t reads = dx * 48 * a.n + dw * 48 * a.m, most = esize(a.dtype) == 4 ? int64_t(10) << 20 : int64_t(3) << 19;
    return a.m <= (esize(a.dtype) == 4 ? 512 : 256) && dx + dw <= 1024 && reads <= most ? SLIM : LARGE;
}
PvdTileJob tile_job(const PvdOperand& X, const PvdOperand& W, const PvdOut& O, int64_t K, int size, bool slim) {
    PvdTileJob J{X, W, O, K, (int)ceil_div(O.rows, slim ? PVD_SM : PVD_T), (int)ceil_div(O.cols, slim ? PVD_SN : PVD_T), 1, 0, nullptr};
    // pieces: while CUs would be left without work, each with a few steps of the kernel's loop at least
    const int64_t step = slim ? PVD_SW * 2 * 64 / size : 128 / size, tiles = (int64_t)J.mt * J.nt;
    const int64_t most = std::max<int64_t>(1, K / ((slim ? 2 : 4) * step));
    const int64_t pieces = tiles ? std::min(most, std::max<int64_t>(1, (slim ? 256 : 512) / tiles)) : 1;
    J.kper = std::max<int64_t>(step, ceil_div(ceil_div(K, pieces), step) * step);
    J.splits = (int)std::max<int64_t>(1, ceil_div(K, J.kper));
    return J;
}
int64_t tile_job_bytes(const PvdTileJob& J) { return J.splits > 1 ? (int64_t)J.splits * J.O.rows * J.O.cols * 4 : 0; }

#define PVD_BY_TYPE(dt, ...)                                           \
    switch (dt) {                                                      \
        case PVAE_F32: { constexpr int D_ = PVD_F32; __VA_ARGS__; } break;    \
        case PVAE_BF16: { constexpr int D_ = PVD_BF16; __VA_ARGS__; } break;  \
        default: { constexpr int D_ = PVD_F16; __VA_ARGS__; } break;          \
    }

int launch_join(int dt, const PvdOut& O, const float* part, int pieces, hipStream_t s) {
    const int64_t quads = O.rows * ceil_div(O.cols, 4);
    // sixteen lanes to four columns where a lane of its own would leave the chip empty and walk a long way
    if (pieces >= 16 ? quads < 64 * 1024 : pieces >= 4 && quads < 16 * 1024) {
        PVD_BY_TYPE(dt, hipLaunchKernelGGL((pvk_dense_join<D_, 16>), dim3((unsigned)ceil_div(quads, 16)), dim3(256), 0, s, O, part, pieces));
    } else {
        PVD_BY_TYPE(dt, hipLaunchKernelGGL((pvk_dense_join<D_, 1>), dim3((unsigned)ceil_div(quads, 256)), dim3(256), 0, s, O, part, pieces));
    }
    return launched("dense_join");
}

// ---- a few rows: the weights read once ----
bool rows_transposed(const pvae_dense_args& a) { return a.n > 1 ? a.w_sn != 1 : a.w_sk == 1; }  // w's columns are contiguous
PvdRowsJob rows_job(const pvae_dense_args& a) {
    const int size = esize(a.dtype);
    const bool t = rows_transposed(a);
    PvdRowsJob J{};
    J.x = a.x; J.ldx = a.ldx;
    J.w = a.w; J.ldw = t ? a.w_sn : a.w_sk;
    J.K = a.k;
    J.O = output(a.m, a.n, a.y, a.ldy, a.bias, a.residual, a.ldr, a.pre, a.ldp, a.act);
    J.blocks = (int)ceil_div(a.n, t ? 128 : 64 * 16 / size);
    // pieces of the contraction: to fill the chip, of 64 at least and of PVD_RK, what LDS holds of x, at most
    const int64_t pieces = std::max(ceil_div(a.k, PVD_RK), std::min<int64_t>(std::max<int64_t>(1, a.k / 64), std::max<int64_t>(1, 512 / J.blocks)));
    J.kper = ceil_div(ceil_div(a.k, pieces), 32) * 32;
    J.splits = (int)ceil_div(a.k, J.kper);
    return J;
}
int64_t rows_bytes(const PvdRowsJob& J) { return J.splits > 1 ? (int64_t)J.splits * J.O.rows * J.O.cols * 4 : 0; }
template <int DT, int R> void launch_rows(const PvdRowsJob& J, bool t, hipStream_t s) {
    const dim3 grid((unsigned)(J.blocks * (int64_t)J.splits));
    if (t) hipLaunchKernelGGL((pvk_dense_rows_t<DT, R>), grid, dim3(512), 0, s, J);
    else hipLaunchKernelGGL((pvk_dense_rows<DT, R>), grid, dim3(512), 0, s, J);
}
int run_rows(const pvae_dense_args& a, PvdRowsJob J, void* workspace, hipStream_t s) {
    if (int rc = check_grid(J.blocks * (int64_t)J.splits)) return rc;
    J.part = static_cast<float*>(workspace);
    const bool t = rows_transposed(a);
    PVD_BY_TYPE(a.dtype, {
        if (a.m == 1) launch_rows<D_, 1>(J, t, s);
        else if (a.m == 2) launch_rows<D_, 2>(J, t, s);
        else if (D_ != PVD_F32 || a.m <= 4) launch_rows<D_, 4>(J, t, s);
        else launch_rows<PVD_F32, 8>(J, t, s);
    });
    if (int rc = launched("dense_rows")) return rc;
    return J.splits > 1 ? launch_join(a.dtype, J.O, J.part, J.splits, s) : 0;
}

// ---- large products: operands laid out (pvk_dense_pack) where they have to be, then pvk_dense_nt ----
int64_t pad_k(int64_t k, int size) { return ceil_div(k, 128 / size) * (128 / size); }
int64_t round256(int64_t b) { return ceil_div(b, 256) * 256; }

// [rows][K] as the product kernel reads it: where it lies, or laid out in the workspace at `at`
struct NtOperand {
    const void* p;
    int64_t ld;   // elements
    int rows;
    bool across;      // [K][rows]: contiguous along the rows
    int64_t low = 0;  // g's second terms: bytes from the first
};

struct NtPlan {
    PvdPacks packs{};
    PvdNtJobs jobs{};
    int64_t bytes = 0;     // workspace
    int tile = 0;          // its edge
    bool deep = false;
    bool two = false;      // g in two terms: every product goes through its contraction twice
};

struct NtBuilder {
    int dt, size;
    char* base;            // the workspace (NULL when only its size is asked for)
    NtPlan plan;
    NtBuilder(int dt_, void* ws) : dt(dt_), size(esize(dt_)), base(static_cast<char*>(ws)) {}

    void* take(int64_t bytes) {
        char* p = base + plan.bytes;
        plan.bytes += round256(bytes);
        return p;
    }
    PvdPack& source(const void* p, int64_t R, int64_t C, int64_t ld, const float* pre, int64_t ldp, int act) {
        PvdPack& J = plan.packs.job[plan.packs.n++];
        J = PvdPack{};
        J.p = p; J.R = R; J.C = C; J.ld = ld;
        J.pre = act == PVD_LINEAR ? nullptr : pre;
        J.ldp = ldp; J.act = act;
        return J;
    }
    // a row stride of a laid-out operand: an odd multiple of 128 bytes, so that a tile's rows lie in all of the L2's channels
    int64_t spread(int64_t k) const { return k * size / 128 % 2 ? k : k + 128 / size; }
    // the source's rows, as rows of the contraction (across: as its lines, whole steps of them)
    NtOperand same(PvdPack& J, bool across) {
        J.w_same = pad_k(J.C, size);
        J.h_same = across ? pad_k(J.R, size) : J.R;
        J.ld_same = spread(J.w_same);
        J.same = take(J.h_same * J.ld_same * size);
        return across ? NtOperand{J.same, J.ld_same, (int)J.w_same, true} : NtOperand{J.same, J.ld_same, (int)J.R, false};
    }
    NtOperand transposed(PvdPack& J) {
        J.w_tran = pad_k(J.R, size);
        J.ld_tran = spread(J.w_tran);
        J.tran = take(J.C * J.ld_tran * size);
        return {J.tran, J.ld_tran, (int)J.C, false};
    }
    // an operand given as memory rows (R rows of C contiguous elements): by_rows: its rows are the product's, else its columns;
    // may_across: the product takes it as it lies in that case
    NtOperand operand(const void* p, int64_t R, int64_t C, int64_t ld, bool by_rows, bool may_across) {
        if (by_rows && lies_well(p, R, C, ld, size, true)) return {p, ld, (int)R, false};
        if (!by_rows && may_across && lies_well(p, R, C, ld, size, false)) return {p, ld, (int)C, true};
        PvdPack& J = source(p, R, C, ld, nullptr, 0, PVD_LINEAR);
        return by_rows ? same(J, false) : transposed(J);
    }
    void product(const NtOperand& x, const NtOperand& w, int64_t K, const PvdOut& O) {
        PvdNtJob& J = plan.jobs.job[plan.jobs.n++];
        J = PvdNtJob{};
        J.x = static_cast<const char*>(x.p); J.ldx = x.ld * size; J.x_rows = x.rows; J.x_across = x.across; J.x_low = x.low;
        J.w = static_cast<const char*>(w.p); J.ldw = w.ld * size; J.w_rows = w.rows; J.w_across = w.across; J.w_low = w.low;
        J.steps = (int)ceil_div(K * size, 128);
        J.O = O;
    }
    // tile edge, pieces, numbering; call when all products are in
    void finish() {
        auto tile_steps = [&](int edge) {
            int64_t n = 0;
            for (int i = 0; i < plan.jobs.n; ++i) {
                const PvdNtJob& J = plan.jobs.job[i];
                n += ceil_div(J.O.rows, edge) * ceil_div(J.O.cols, edge) * J.steps;
            }
            return plan.two ? 2 * n : n;
        };
        // 128 x 128 with eight waves, two workgroups to a CU (4096^3 bf16 with residual and z, in long runs: 147 us; 128 x 256, one
        // workgroup to a CU, whose results nothing hides: 163; the products alone are 124 and 121).  float32 takes 64 x 64 (five to a CU)
        // where 128 x 128 would give the CUs less than 40 steps each -- matrix work is sixteen times slower there, and an
        // uneven last round counts -- or would spend a fifth of its work on rows and columns that are not there
        // (64 x 512 x 100000: 148 us, with 64 x 64 tiles 74).
        plan.tile = size == 4 && (tile_steps(128) < 256 * 40 || tile_steps(64) * 5 < tile_steps(128) * 16) ? 64 : 128;
        int64_t per = std::max<int64_t>(8, ceil_div(tile_steps(plan.tile), plan.tile == 64 ? 1024 : 512));
        if (plan.two) per = ceil_div(per, 2);  // steps of the contraction, each gone through twice
        int64_t tiles = 0;
        for (int i = 0; i < plan.jobs.n; ++i) {
            PvdNtJob& J = plan.jobs.job[i];
            J.mt = (int)ceil_div(J.O.rows, plan.tile);
            J.nt = (int)ceil_div(J.O.cols, plan.tile);
            // a contraction much longer than a CU's fair share is cut into pieces (each costs a write and a read of the result)
            J.per = J.steps > 2 * per ? (int)ceil_div(J.steps, ceil_div(J.steps, per)) : std::max(1, J.steps);
            J.splits = std::max(1, (int)ceil_div(J.steps, J.per));
            // a band's rows of tiles keep their operand in an XCD's L2 while the columns pass by
            J.band = (int)std::min<int64_t>(J.mt, std::max<int64_t>(4, (1 << 20) / ((int64_t)plan.tile * J.per * 128)));
            if (J.splits > 1) J.part = static_cast<float*>(take((int64_t)J.splits * J.O.rows * J.O.cols * 4));
            tiles += (int64_t)J.mt * J.nt * J.splits;
        }
        plan.deep = plan.tile == 128 && tiles <= 256;  // one workgroup to a CU: four steps in LDS instead of two
        int at = 0;
        for (int i = 0; i < plan.packs.n; ++i) {
            PvdPack& J = plan.packs.job[i];
            J.rt = (int)ceil_div(J.tran ? J.w_tran : J.h_same, 64);
            J.ct = (int)ceil_div(J.same ? J.w_same : J.C, 64);
            plan.packs.first[i] = at;
            at += J.rt * J.ct;
        }
        plan.packs.first[plan.packs.n] = at;
    }
};

template <int DT, int EDGE, int WM, int WN, int ST, bool TWO = false> int launch_nt(const PvdNtJobs& P, int blocks, hipStream_t s) {
    typedef PvdNt<DT, EDGE, WM, WN, ST, TWO> K;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(pvk_dense_nt<DT, EDGE, WM, WN, ST, TWO>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, K::LDS);
    if (e != hipSuccess) return refuse(-10, "%d bytes of LDS: %s", (int)K::LDS, hipGetErrorString(e));
    hipLaunchKernelGGL((pvk_dense_nt<DT, EDGE, WM, WN, ST, TWO>), dim3(blocks), dim3(K::THREADS), K::LDS, s, P);
    return launched("dense_nt");
}
int launch_large(int dt, NtPlan& plan, hipStream_t s) {
    if (plan.packs.n && plan.packs.first[plan.packs.n]) {
        PVD_BY_TYPE(dt, hipLaunchKernelGGL(pvk_dense_pack<D_>, dim3(plan.packs.first[plan.packs.n]), dim3(256), 0, s, plan.packs));
        if (int rc = launched("dense_pack")) return rc;
    }
    PvdNtJobs& P = plan.jobs;
    int64_t at = 0;
    for (int i = 0; i < 2; ++i) {
        P.first[i] = (int)at;
        if (i < P.n) at += (int64_t)P.job[i].mt * P.job[i].nt * P.job[i].splits;
    }
    P.first[2] = (int)at;
    if (P.dbias) at += ceil_div(P.sum_cols, plan.tile == 128 ? 512 : 256);
    if (int rc = check_grid(at)) return rc;
    int rc = 0;
    const int blocks = (int)at;
    if (blocks == 0) return 0;
    if (plan.tile == 64) rc = launch_nt<PVD_F32, 64, 4, 1, 2>(P, blocks, s);
    else if (plan.two && dt == PVD_BF16) rc = plan.deep ? launch_nt<PVD_BF16, 128, 4, 2, 4, true>(P, blocks, s) : launch_nt<PVD_BF16, 128, 4, 2, 2, true>(P, blocks, s);
    else if (plan.two) rc = plan.deep ? launch_nt<PVD_F16, 128, 4, 2, 4, true>(P, blocks, s) : launch_nt<PVD_F16, 128, 4, 2, 2, true>(P, blocks, s);
    else PVD_BY_TYPE(dt, (rc = plan.deep ? launch_nt<D_, 128, 4, 2, 4>(P, blocks, s) : launch_nt<D_, 128, 4, 2, 2>(P, blocks, s)));
    if (rc) return rc;
    for (int i = 0; i < P.n; ++i)
        if (P.job[i].splits > 1 && (rc = launch_join(dt, P.job[i].O, P.job[i].part, P.job[i].splits, s))) return rc;
    return 0;
}

NtPlan large_dense(const pvae_dense_args& a, void* ws) {
    NtBuilder B(a.dtype, ws);
    const NtOperand x = B.operand(a.x, a.m, a.k, a.ldx, true, false);
    const NtOperand w = a.w_sk == 1 ? B.operand(a.w, a.n, a.k, a.w_sn, true, true) : B.operand(a.w, a.k, a.n, a.w_sk, false, true);
    B.product(x, w, a.k, output(a.m, a.n, a.y, a.ldy, a.bias, a.residual, a.ldr, a.pre, a.ldp, a.act));
    B.finish();
    return B.plan;
}
NtPlan large_bwd(const pvae_dense_bwd_args& a, void* ws) {
    NtBuilder B(a.dtype, ws);
    // g: rows of the contraction for dx (over n), lines of it for dw (over m); its column sums, and unrounded if asked for
    PvdPack& g = B.source(a.dy, a.m, a.n, a.lddy, a.pre, a.ldp, a.act);
    NtOperand gw = B.same(g, true);
    if (B.size == 2 && g.pre) {
        g.low = B.take(g.h_same * g.ld_same * B.size);
        gw.low = static_cast<char*>(g.low) - static_cast<char*>(g.same);
        B.plan.two = true;
    }
    const NtOperand gx{gw.p, gw.ld, (int)a.m, false, gw.low};
    g.g32 = a.dpre;
    if (a.dbias) {
        g.sums = static_cast<float*>(B.take(ceil_div(a.m, 64) * a.n * 4));
        B.plan.jobs.sums = g.sums;
        B.plan.jobs.sum_tiles = (int)ceil_div(a.m, 64);
        B.plan.jobs.sum_cols = a.n;
        B.plan.jobs.dbias = a.dbias;
    }
    if (a.dx) {
        const NtOperand w = a.w_sn == 1 ? B.operand(a.w, a.k, a.n, a.w_sk, true, true) : B.operand(a.w, a.n, a.k, a.w_sn, false, true);
        B.product(gx, w, a.n, output(a.m, a.k, a.dx, a.lddx, nullptr, a.dx_add, a.ldadd, nullptr, 0, PVD_LINEAR));
    }
    if (a.dw) {
        const NtOperand x = B.operand(a.x, a.m, a.k, a.ldx, false, true);
        B.product(x, gw, a.m, output(a.k, a.n, a.dw, a.n, nullptr, nullptr, 0, nullptr, 0, PVD_LINEAR));
    }
    B.finish();
    return B.plan;
}
PvdTileJob dense_job(const pvae_dense_args& a, bool slim) {
    const int size = esize(a.dtype);
    return tile_job(operand(a.x, a.m, a.ldx, 1), operand(a.w, a.n, a.w_sn, a.w_sk),
                    output(a.m, a.n, a.y, a.ldy, a.bias, a.residual, a.ldr, a.pre, a.ldp, a.act), a.k, size, slim);
}
int check_dense(const pvae_dense_args* a) {
    if (!a) return refuse(-1, "no arguments");
    if (int rc = check_sizes(a->dtype, a->act, a->m, a->k, a->n)) return rc;
    const int size = esize(a->dtype);
    if (int rc = check_matrix("x", a->x, a->m, a->k, a->ldx, size)) return rc;
    if (int rc = check_weights(a->w, a->k, a->n, a->w_sk, a->w_sn, size)) return rc;
    if (int rc = check_matrix("y", a->y, a->m, a->n, a->ldy, size)) return rc;
    if (a->bias)
        if (int rc = check_matrix("bias", a->bias, 1, a->n, a->n, size)) return rc;
    if (a->residual)
        if (int rc = check_matrix("residual", a->residual, a->ldr == 0 ? 1 : a->m, a->n, a->ldr, size)) return rc;
    if (a->pre)
        if (int rc = check_matrix("pre", a->pre, a->m, a->n, a->ldp, 4)) return rc;
    const bool in_place = a->residual == a->y && (a->ldr == a->ldy || a->m <= 1);
    const Extent e[] = {extent("y", a->y, a->m, a->n, a->ldy, size), extent("pre", a->pre, a->m, a->n, a->ldp, 4),
                        extent("x", a->x, a->m, a->k, a->ldx, size), weights_extent(a->w, a->k, a->n, a->w_sk, a->w_sn, size),
                        extent("bias", a->bias, 1, a->n, a->n, size),
                        extent("residual", in_place ? nullptr : a->residual, a->m, a->n, a->ldr, size)};
    return check_apart(e, 2, 6);
}

struct BwdPlan {
    PvdBwdJob J;
    int64_t n_db;
};
BwdPlan bwd_plan(const pvae_dense_bwd_args& a) {
    const int size = esize(a.dtype);
    BwdPlan p{};
    PvdOperand gx = operand(a.dy, a.m, a.lddy, 1), gw = operand(a.dy, a.n, 1, a.lddy);
    with_grad(gx, a.pre, a.ldp, 1, a.act);
    with_grad(gw, a.pre, 1, a.ldp, a.act);
    // w as an operand of dx: rows are the k of the layer, the contraction its n
    if (a.dx)
        p.J.dx = tile_job(gx, operand(a.w, a.k, a.w_sk, a.w_sn),
                          output(a.m, a.k, a.dx, a.lddx, nullptr, a.dx_add, a.ldadd, nullptr, 0, PVD_LINEAR), a.n, size, true);
    if (a.dw)
        p.J.dw = tile_job(operand(a.x, a.k, 1, a.ldx), gw,
                          output(a.k, a.n, a.dw, a.n, nullptr, nullptr, 0, nullptr, 0, PVD_LINEAR), a.m, size, true);
    p.J.n_dx = a.dx ? (int64_t)p.J.dx.mt * p.J.dx.nt * p.J.dx.splits : 0;
    p.J.n_dw = a.dw ? (int64_t)p.J.dw.mt * p.J.dw.nt * p.J.dw.splits : 0;
    p.J.dy = a.dy;
    p.J.lddy = a.lddy;
    p.J.pre = a.pre;
    p.J.ldp = a.ldp;
    p.J.act = a.act;
    p.J.m = a.m;
    p.J.n = a.n;
    p.J.dbias = a.dbias;
    p.J.dpre = a.dpre;
    p.n_db = a.dbias || a.dpre ? ceil_div(a.n, 64) : 0;
    return p;
}
int64_t bwd_bytes(const BwdPlan& p) { return (p.J.n_dx ? tile_job_bytes(p.J.dx) : 0) + (p.J.n_dw ? tile_job_bytes(p.J.dw) : 0); }
int check_dense_bwd(const pvae_dense_bwd_args* a) {
    if (!a) return refuse(-1, "no arguments");
    if (int rc = check_sizes(a->dtype, a->act, a->m, a->k, a->n)) return rc;
    const int size = esize(a->dtype);
    if (int rc = check_matrix("dy", a->dy, a->lddy == 0 ? 1 : a->m, a->n, a->lddy, size)) return rc;
    if (a->act != PVAE_LINEAR)
        if (int rc = check_matrix("pre", a->pre, a->m, a->n, a->ldp, 4)) return rc;
    if (a->dw)
        if (int rc = check_matrix("x", a->x, a->m, a->k, a->ldx, size)) return rc;
    if (a->dx) {
        if (int rc = check_weights(a->w, a->k, a->n, a->w_sk, a->w_sn, size)) return rc;
        if (int rc = check_matrix("dx", a->dx, a->m, a->k, a->lddx, size)) return rc;
        if (a->dx_add)
            if (int rc = check_matrix("dx_add", a->dx_add, a->ldadd == 0 ? 1 : a->m, a->k, a->ldadd, size)) return rc;
    }
    if (a->dw && !aligned(a->dw, size)) return refuse(-2, "dw is not aligned to its elements");
    if (a->dbias && !aligned(a->dbias, size)) return refuse(-2, "dbias is not aligned to its elements");
    if (a->dpre && !aligned(a->dpre, 4)) return refuse(-2, "dpre is not aligned to its elements");
    const bool in_place = a->dx_add == a->dx && (a->ldadd == a->lddx || a->m <= 1);
    const Extent e[] = {extent("dx", a->dx, a->m, a->k, a->lddx, size), extent("dw", a->dw, a->k, a->n, a->n, size),
                        extent("dbias", a->dbias, 1, a->n, a->n, size), extent("dpre", a->dpre, a->m, a->n, a->n, 4),
                        extent("dy", a->dy, a->m, a->n, a->lddy, size), extent("pre", a->act == PVAE_LINEAR ? nullptr : a->pre, a->m, a->n, a->ldp, 4),
                        extent("x", a->dw ? a->x : nullptr, a->m, a->k, a->ldx, size),
                        a->dx ? weights_extent(a->w, a->k, a->n, a->w_sk, a->w_sn, size) : Extent{"w", 0, 0, 0, 0, 0},
                        extent("dx_add", in_place || !a->dx ? nullptr : a->dx_add, a->m, a->k, a->ldadd, size)};
    return check_apart(e, 4, 9);
}
// ---- many tensors ----
int check_tensors(const char* name, const pvae_tensor* t, int64_t count, bool tiles) {
    if (count < 0 || count > 65536) return refuse(-2, "%lld tensors: 0 .. 65536", (long long)count);
    if (count && !t) return refuse(-1, "%s is NULL", name);
    for (int64_t i = 0; i < count; ++i) {
        if (t[i].dtype < PVAE_F32 || t[i].dtype > PVAE_F16) return refuse(-2, "%s %lld: unknown type %d", name, (long long)i, t[i].dtype);
        if (t[i].n < 0 || t[i].n > (int64_t(1) << 40)) return refuse(-2, "%s %lld: %lld elements", name, (long long)i, (long long)t[i].n);
        if (t[i].n && !t[i].data) return refuse(-1, "%s %lld is NULL", name, (long long)i);
        if (!aligned(t[i].data, esize(t[i].dtype))) return refuse(-2, "%s %lld is not aligned to its elements", name, (long long)i);
        if (t[i].tile && (!tiles || t[i].tile < 0 || t[i].tile % 4 || t[i].n % t[i].tile))
            return refuse(-2, "%s %lld: bad interleave %d", name, (long long)i, t[i].tile);
    }
    return 0;
}
struct Span { uintptr_t lo, hi; };
void add_spans(std::vector<Span>& v, const pvae_tensor* t, int64_t count) {
    for (int64_t i = 0; i < count; ++i)
        if (t[i].n) {
            const uintptr_t lo = reinterpret_cast<uintptr_t>(t[i].data);
            v.push_back({lo, lo + (uintptr_t)t[i].n * esize(t[i].dtype)});
        }
}
bool overlap(std::vector<Span>& v) {
    std::sort(v.begin(), v.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
    for (size_t i = 1; i < v.size(); ++i)
        if (v[i].lo < v[i - 1].hi) return true;
    return false;
}
// whether t reads what one of the spans (sorted, disjoint) writes
bool reads_from(const std::vector<Span>& v, const pvae_tensor& t) {
    if (t.n == 0) return false;
    const uintptr_t lo = reinterpret_cast<uintptr_t>(t.data), hi = lo + (uintptr_t)t.n * esize(t.dtype);
    const auto it = std::lower_bound(v.begin(), v.end(), hi, [](const Span& s, uintptr_t h) { return s.lo < h; });
    return it != v.begin() && std::prev(it)->hi > lo;
}

// the tensors in tables of PVM_MAXT, empty ones left out: f(table) per launch; `fill` sets a table's other pointers
template <typename Fill, typename Launch> int for_tables(const pvae_tensor* g, int64_t count, Fill fill, Launch launch) {
    PvmTab T;
    T.count = 0;
    T.first[0] = 0;
    for (int64_t i = 0; i <= count; ++i) {
        const int64_t chunks = i < count ? ceil_div(g[i].n, PVM_CHUNK) : 0;
        if (T.count && (i == count || T.count == PVM_MAXT || T.first[T.count] + chunks > 0x7fffffff)) {
            if (int rc = launch(T)) return rc;
            T.count = 0;
        }
        if (i == count || chunks == 0) continue;
        const int c = T.count;
        T.a[c] = g[i].data;
        T.n[c] = g[i].n;
        T.dt[c] = (unsigned char)g[i].dtype;
        T.b[c] = nullptr;
        T.m[c] = T.v[c] = nullptr;
        T.tile[c] = 0;
        fill(T, c, i);
        T.first[c + 1] = T.first[c] + (int)chunks;
        T.count = c + 1;
    }
    return 0;
}
int tables_of(const pvae_tensor* g, int64_t count) {
    int n = 0;
    for_tables(g, count, [](PvmTab&, int, int64_t) {}, [&](PvmTab&) { ++n; return 0; });
    return n;
}
// the partial sums of g^2: at most PVM_PARTS over all launches
int launch_sumsq(const pvae_tensor* g, int64_t count, double* part, int* nparts, hipStream_t s) {
    const int tables = tables_of(g, count), each = tables ? std::max(1, std::min(1024, PVM_PARTS / tables)) : 0;
    *nparts = 0;
    return for_tables(g, count, [](PvmTab&, int, int64_t) {}, [&](PvmTab& T) {
        const int blocks = std::min(each, T.first[T.count]);
        hipLaunchKernelGGL(pvk_sumsq, dim3(blocks), dim3(PVM_THREADS), 0, s, T, part + *nparts);
        *nparts += blocks;
        return launched("sumsq");
    });
}
int launch_norm(const pvae_tensor* g, int64_t count, float* norm, void* ws, int* nparts, hipStream_t s) {
    double* part = static_cast<double*>(ws);
    if (int rc = launch_sumsq(g, count, part, nparts, s)) return rc;
    if (!norm) return 0;
    hipLaunchKernelGGL(pvk_norm_final, dim3(1), dim3(PVM_THREADS), 0, s, (const double*)part, *nparts, norm);
    return launched("norm_final");
}

template <typename F> int guarded(F f) {  // no C++ exception leaves a C entry
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return refuse(-9, "out of host memory");
    } catch (...) {
        return refuse(-9, "unexpected error");
    }
}

}  // namespace

extern "C" {

const char* pvae_ops_last_error(void) { return g_err; }

int64_t pvae_dense_workspace(const pvae_dense_args* args) {
    if (check_dense(args) || args->m == 0 || args->n == 0) return 0;
    const pvae_dense_args a = plain(*args);
    switch (dense_kernel(a)) {
        case ROWS: return rows_bytes(rows_job(a));
        case SLIM: return tile_job_bytes(dense_job(a, true));
        case TILE: return tile_job_bytes(dense_job(a, false));
        default: return large_dense(a, nullptr).bytes;
    }
}

int pvae_dense(const pvae_dense_args* args, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    if (int rc = check_dense(args)) return rc;
    if (args->m == 0 || args->n == 0) return 0;
    const pvae_dense_args a = plain(*args);
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    const Kernel kind = dense_kernel(a);
    if (kind == ROWS) {
        const PvdRowsJob J = rows_job(a);
        if (int rc = check_workspace("pvae_dense", workspace, workspace_bytes, rows_bytes(J))) return rc;
        return run_rows(a, J, workspace, s);
    }
    if (kind == LARGE) {
        NtPlan plan = large_dense(a, workspace);
        if (int rc = check_workspace("pvae_dense", workspace, workspace_bytes, plan.bytes)) return rc;
        return launch_large(a.dtype, plan, s);
    }
    PvdTileJob J = dense_job(a, kind == SLIM);
    if (int rc = check_workspace("pvae_dense", workspace, workspace_bytes, tile_job_bytes(J))) return rc;
    const int64_t blocks = (int64_t)J.mt * J.nt * J.splits;
    if (int rc = check_grid(blocks)) return rc;
    J.part = static_cast<float*>(workspace);
    if (kind == SLIM) {
        PVD_BY_TYPE(a.dtype, hipLaunchKernelGGL(pvk_dense_slim<D_>, dim3((unsigned)blocks), dim3(512), 0, s, J));
    } else {
        PVD_BY_TYPE(a.dtype, hipLaunchKernelGGL(pvk_dense_tile<D_>, dim3((unsigned)blocks), dim3(256), 0, s, J));
    }
    if (int rc = launched("dense")) return rc;
    return J.splits > 1 ? launch_join(a.dtype, J.O, J.part, J.splits, s) : 0;
}

int64_t pvae_dense_bwd_workspace(const pvae_dense_bwd_args* args) {
    if (check_dense_bwd(args)) return 0;
    const pvae_dense_bwd_args a = plain(*args);
    return bwd_kernel(a) == SLIM ? bwd_bytes(bwd_plan(a)) : large_bwd(a, nullptr).bytes;
}

int pvae_dense_bwd(const pvae_dense_bwd_args* args, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    if (int rc = check_dense_bwd(args)) return rc;
    const pvae_dense_bwd_args a = plain(*args);
    hipStream_t s = static_cast<hipStream_t>(hip_stream);
    if (bwd_kernel(a) == LARGE) {
        NtPlan plan = large_bwd(a, workspace);
        if (int rc = check_workspace("pvae_dense_bwd", workspace, workspace_bytes, plan.bytes)) return rc;
        return launch_large(a.dtype, plan, s);
    }
    BwdPlan p = bwd_plan(a);
    if (int rc = check_workspace("pvae_dense_bwd", workspace, workspace_bytes, bwd_bytes(p))) return rc;
    const int64_t blocks = p.J.n_dx + p.J.n_dw + p.n_db;
    if (blocks == 0) return 0;
    p.J.dx.part = static_cast<float*>(workspace);
    p.J.dw.part = static_cast<float*>(workspace) + (p.J.n_dx ? tile_job_bytes(p.J.dx) / 4 : 0);
    PVD_BY_TYPE(a.dtype, hipLaunchKernelGGL(pvk_dense_bwd_slim<D_>, dim3((unsigned)blocks), dim3(512), 0, s, p.J));
    if (int rc = launched("dense_bwd")) return rc;
    if (p.J.n_dx && p.J.dx.splits > 1)
        if (int rc = launch_join(a.dtype, p.J.dx.O, p.J.dx.part, p.J.dx.splits, s)) return rc;
    if (p.J.n_dw && p.J.dw.splits > 1)
        if (int rc = launch_join(a.dtype, p.J.dw.O, p.J.dw.part, p.J.dw.splits, s)) return rc;
    return 0;
}

int64_t pvae_norm_workspace(void) { return PVM_PARTS * (int64_t)sizeof(double); }

int pvae_global_norm(const pvae_tensor* g, int64_t count, float* norm, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    if (int rc = check_tensors("g", g, count, false)) return rc;
    if (!norm) return refuse(-1, "norm is NULL");
    if (int rc = check_workspace("pvae_global_norm", workspace, workspace_bytes, pvae_norm_workspace())) return rc;
    int nparts;
    return launch_norm(g, count, norm, workspace, &nparts, static_cast<hipStream_t>(hip_stream));
}

int pvae_clip_by_global_norm(const pvae_tensor* g, const pvae_tensor* out, int64_t count, double max_norm, float* norm, void* workspace,
                             int64_t workspace_bytes, void* hip_stream) {
    return guarded([&]() -> int {
        if (int rc = check_tensors("g", g, count, false)) return rc;
        if (int rc = check_tensors("out", out, count, false)) return rc;
        if (!(max_norm > 0.0)) return refuse(-2, "max_norm %g: a positive number", max_norm);
        bool in_place = true;
        for (int64_t i = 0; i < count; ++i) {
            if (out[i].n != g[i].n || out[i].dtype != g[i].dtype)
                return refuse(-2, "tensor %lld: out differs from g in size or type", (long long)i);
            in_place = in_place && (out[i].data == g[i].data || g[i].n == 0);
        }
        std::vector<Span> spans;
        spans.reserve(2 * (size_t)count);
        add_spans(spans, out, count);
        if (overlap(spans)) return refuse(-2, "two of out's tensors overlap");
        // a gradient may appear twice in g, but none may lie where another one's copy is written
        for (int64_t i = 0; i < count && !in_place; ++i)
            if (out[i].data != g[i].data && reads_from(spans, g[i])) return refuse(-2, "tensor %lld of g overlaps an output", (long long)i);
        if (int rc = check_workspace("pvae_clip_by_global_norm", workspace, workspace_bytes, pvae_norm_workspace())) return rc;
        hipStream_t s = static_cast<hipStream_t>(hip_stream);
        double* part = static_cast<double*>(workspace);
        int nparts;
        if (int rc = launch_sumsq(g, count, part, &nparts, s)) return rc;
        if (nparts == 0) return norm ? launch_norm(g, 0, norm, workspace, &nparts, s) : 0;
        return for_tables(
            g, count,
            [&](PvmTab& T, int c, int64_t i) { T.b[c] = out[i].data; },
            [&](PvmTab& T) {
                hipLaunchKernelGGL(pvk_clip_apply, dim3(std::min(2048, T.first[T.count])), dim3(PVM_THREADS), 0, s, T, (const double*)part,
                                   nparts, max_norm, norm);
                return launched("clip_apply");
            });
    });
}

int pvae_adam_step(const pvae_tensor* p, const pvae_tensor* g, const pvae_tensor* m, const pvae_tensor* v, int64_t count, double lr,
                   double beta1, double beta2, double eps, int64_t step, const int32_t* step_dev, double clip_norm, float* norm,
                   void* workspace, int64_t workspace_bytes, void* hip_stream) {
    return guarded([&]() -> int {
        if (int rc = check_tensors("p", p, count, true)) return rc;
        if (int rc = check_tensors("g", g, count, false)) return rc;
        if (int rc = check_tensors("m", m, count, true)) return rc;
        if (int rc = check_tensors("v", v, count, true)) return rc;
        if (!std::isfinite(lr) || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !((float)eps > 0) || !std::isfinite((float)eps))
            return refuse(-2, "lr %g, beta1 %g, beta2 %g, eps %g: finite, 0 <= beta < 1, eps > 0 in float32", lr, beta1, beta2, eps);
        if (!step_dev && step < 1) return refuse(-2, "step %lld: counted from 1", (long long)step);
        if (!(clip_norm >= 0)) return refuse(-2, "clip_norm %g: a positive number, or 0 for none", clip_norm);
        std::vector<Span> spans;
        spans.reserve(4 * (size_t)count);
        for (int64_t i = 0; i < count; ++i) {
            if (p[i].dtype != PVAE_F32 || m[i].dtype != PVAE_F32 || v[i].dtype != PVAE_F32)
                return refuse(-2, "tensor %lld: p, m and v are float32", (long long)i);
            if (p[i].n != g[i].n || m[i].n != g[i].n || v[i].n != g[i].n || m[i].tile != p[i].tile || v[i].tile != p[i].tile)
                return refuse(-2, "tensor %lld: p, g, m and v differ in size", (long long)i);
            if (p[i].tile && (static_cast<float*>(m[i].data) != static_cast<float*>(p[i].data) + p[i].tile ||
                              static_cast<float*>(v[i].data) != static_cast<float*>(p[i].data) + 2 * p[i].tile))
                return refuse(-2, "tensor %lld: p, m and v are not interleaved by %d elements", (long long)i, p[i].tile);
            if (p[i].tile && p[i].n) {
                const uintptr_t lo = reinterpret_cast<uintptr_t>(p[i].data);
                spans.push_back({lo, lo + (uintptr_t)p[i].n * 12});
            } else {
                add_spans(spans, p + i, 1);
                add_spans(spans, m + i, 1);
                add_spans(spans, v + i, 1);
            }
        }
        if (overlap(spans)) return refuse(-2, "two of the tensors p, m and v overlap");
        for (int64_t i = 0; i < count; ++i)
            if (reads_from(spans, g[i])) return refuse(-2, "tensor %lld: g overlaps one of p, m and v", (long long)i);
        hipStream_t s = static_cast<hipStream_t>(hip_stream);
        double* part = static_cast<double*>(workspace);
        int nparts = 0;
        if (clip_norm > 0 || norm) {
            if (int rc = check_workspace("pvae_adam_step", workspace, workspace_bytes, pvae_norm_workspace())) return rc;
            if (int rc = launch_sumsq(g, count, part, &nparts, s)) return rc;
            if (nparts == 0) return norm ? launch_norm(g, 0, norm, workspace, &nparts, s) : 0;
        }
        const PvmAdam A{lr, beta1, beta2, (float)eps, step, step_dev};
        return for_tables(
            g, count,
            [&](PvmTab& T, int c, int64_t i) {
                T.b[c] = p[i].data;
                T.m[c] = static_cast<float*>(m[i].data);
                T.v[c] = static_cast<float*>(v[i].data);
                T.tile[c] = p[i].tile;
            },
            [&](PvmTab& T) {
                hipLaunchKernelGGL(pvk_adam_apply, dim3(std::min(2048, T.first[T.count])), dim3(PVM_THREADS), 0, s, T, (const double*)part,
                                   nparts, clip_norm, norm, A);
                return launched("adam_apply");
            });
    });
}

}  // extern "C"
