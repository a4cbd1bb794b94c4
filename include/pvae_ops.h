/* pvae_ops.h -- C ABI of libpvae.so's operators on device tensors: a dense layer with everything that follows its product
 * in one pass, its gradients, clipping by the global gradient norm and the Adam update with that clipping folded in.
 *
 * They take device pointers of the caller's own tensors (the engine of pvae.h keeps its own) and run on the stream that is
 * passed, on the current device; nothing is allocated, nothing waits for the GPU, and every launch may be captured into a
 * graph.  Where a call needs scratch memory the caller passes it: pvae_*_workspace says how many bytes for those very
 * arguments, addresses and strides included; the memory belongs to the call until its work on the stream is done, and no call
 * finds in it what another one left.  Two calls that may run at the same time need a workspace each.
 *
 * Every function returns 0 or a negative code; pvae_ops_last_error() gives the calling thread's text.  A refused call has
 * launched nothing.
 */
#ifndef PVAE_OPS_H
#define PVAE_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { PVAE_F32 = 0, PVAE_BF16 = 1, PVAE_F16 = 2 };
/* f(z): z; max(z, 0); z > 0 ? z : exp(z) - 1; 1 / (1 + exp(-z)); tanh z; z / (1 + exp(-z)); z Phi(z) with Phi the normal
 * distribution function */
enum { PVAE_LINEAR = 0, PVAE_RELU = 1, PVAE_ELU = 2, PVAE_SIGMOID = 3, PVAE_TANH = 4, PVAE_SILU = 5, PVAE_GELU = 6 };

const char* pvae_ops_last_error(void);

/* y = f(x w + bias) + residual.  All tensors of one type; products and sums in float32, one rounding at the end.
 * x [m][k], y [m][n]: rows of contiguous elements, row strides ldx, ldy in elements (>= the row's length).
 * w [k][n]: element (i, j) at i * w_sk + j * w_sn, one of the two strides 1 (Keras kernels: w_sn == 1).
 * bias [n] or NULL.  residual [m][n] with row stride ldr (0: one row added to every row) or NULL.
 * pre [m][n] float32, row stride ldp, or NULL: receives z = x w + bias, which pvae_dense_bwd reads.
 * y may be the residual itself; otherwise outputs share no byte with each other or an input (they may be other columns of one
 * buffer; with row strides of different lengths their ranges have to be apart).
 * m, k, n >= 0; with k == 0 z is the bias. */
typedef struct pvae_dense_args {
    int32_t dtype, act;
    int64_t m, k, n;
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t w_sk, w_sn;
    const void* bias;
    const void* residual;
    int64_t ldr;
    void* y;
    int64_t ldy;
    float* pre;
    int64_t ldp;
} pvae_dense_args;
int64_t pvae_dense_workspace(const pvae_dense_args* a);
int pvae_dense(const pvae_dense_args* a, void* workspace, int64_t workspace_bytes, void* hip_stream);

/* The gradients of pvae_dense: g = dy * f'(pre); dx = g w^T (+ dx_add); dw = x^T g; dbias = column sums of g.  The
 * residual's gradient is dy itself.
 * dy [m][n] (lddy 0: one row for all); pre [m][n] float32 (NULL with PVAE_LINEAR); dx [m][k], dw [k][n] contiguous, dbias [n]: each may be NULL.
 * dx_add [m][k] with row stride ldadd, or NULL: added to dx before its one rounding (a layer whose residual is its own
 * input passes dy; dx may be dx_add itself).  dpre [m][n] float32 contiguous, or NULL: receives g.
 * g of a 16-bit type enters the products in two terms of the type (bf16: 16 bits of g; float16: 22 bits, to 2^-35 at worst, and
 * above the type's largest value), so dx and dw are rounded once, at their end; dbias sums the unrounded g. */
typedef struct pvae_dense_bwd_args {
    int32_t dtype, act;
    int64_t m, k, n;
    const void* dy;
    int64_t lddy;
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t w_sk, w_sn;
    const float* pre;
    int64_t ldp;
    void* dx;
    int64_t lddx;
    const void* dx_add;
    int64_t ldadd;
    void* dw;
    void* dbias;
    float* dpre;
} pvae_dense_bwd_args;
int64_t pvae_dense_bwd_workspace(const pvae_dense_bwd_args* a);
int pvae_dense_bwd(const pvae_dense_bwd_args* a, void* workspace, int64_t workspace_bytes, void* hip_stream);

/* One tensor of a model: n contiguous elements at data.  tile != 0 (pvae_adam_step's p, m and v, float32): the three live
 * interleaved in blocks of `tile` elements (a multiple of 4), element i at data[(i / tile) * 3 * tile + i % tile] -- how the
 * engine of pvae.h keeps its wide tensors. */
typedef struct pvae_tensor {
    void* data;
    int64_t n;
    int32_t dtype;
    int32_t tile;
} pvae_tensor;

/* norm = sqrt(sum over all tensors and elements of g^2), summed in float64; *norm (device, float32).  At most 65536 tensors. */
int64_t pvae_norm_workspace(void);
int pvae_global_norm(const pvae_tensor* g, int64_t count, float* norm, void* workspace, int64_t workspace_bytes,
                     void* hip_stream);
/* out = g * min(1, max_norm / norm) (max_norm > 0), each value rounded once; *norm as above, before clipping.  out's tensors
 * have g's sizes and types; out may be g (then a norm within the bound writes nothing).  A norm that is not finite makes
 * every output NaN, as Keras' global_clipnorm does. */
int pvae_clip_by_global_norm(const pvae_tensor* g, const pvae_tensor* out, int64_t count, double max_norm, float* norm,
                             void* workspace, int64_t workspace_bytes, void* hip_stream);
/* The engine's Adam (Keras': m += (g - m)(1 - beta1); v += (g^2 - v)(1 - beta2);
 * p -= lr sqrt(1 - beta2^t) / (1 - beta1^t) m / (sqrt(v) + eps)) on float32 p, m, v and gradients of any of the three types,
 * g scaled by min(1, clip_norm / norm) first (clip_norm == 0: not clipped, and norm may be NULL: no pass over g then).
 * t = step, or *step_dev (device, int32) where step_dev is not NULL: a captured graph's replays read it anew. */
int pvae_adam_step(const pvae_tensor* p, const pvae_tensor* g, const pvae_tensor* m, const pvae_tensor* v, int64_t count,
                   double lr, double beta1, double beta2, double eps, int64_t step, const int32_t* step_dev, double clip_norm,
                   float* norm, void* workspace, int64_t workspace_bytes, void* hip_stream);

#ifdef __cplusplus
}
#endif
#endif
