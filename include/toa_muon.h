/*
 * toa_muon.h -- C ABI of the MI355X (gfx950) operators for matrix-shaped parameters
 * (libtoa_muon.so): orthogonalisation of an update by Newton-Schulz products, its gradient, the
 * optimizer step built on it (Muon), and the 8-bit blocks its momentum can be kept in.
 *
 * The reference has no counterpart; conventions are those of toa_adam.h.
 *
 *   orthogonalize   X = G / (|G|_F + eps), then `steps` times
 *                   X <- a X + b (X X^T) X + c (X X^T)^2 X
 *   its gradient    of <X, D> with respect to G
 *   step            M <- momentum * M + g;   U = g + momentum * M  (nesterov; else U = M)
 *                   P <- (1 - lr * weight_decay) P - lr * r * orthogonalize(U)
 *                   r = 1, sqrt(max(1, rows / cols)) or 0.2 sqrt(max(rows, cols))
 *   8-bit blocks    128 consecutive elements share one float32 scale = max |x| / 127; an element
 *                   is an int8 code = x / scale rounded half to even and stands for
 *                   code * scale.  A block that holds a NaN or an infinity stands for NaN.
 *
 * Conventions
 *   lists     `num` matrices of any shapes; rows[i] x cols[i].  Empty ones are skipped.
 *   views     device memory on the CURRENT HIP device: element (i, j) of a matrix lies
 *             i * row_stride + j * col_stride elements behind `data`.  Any alignment and any
 *             strides; what is written must not overlap anything else of the call, except that
 *             `out` may be `in` itself in orthogonalize.
 *   dense     parameters' gradients and momentum of a step are dense, all in one memory order:
 *             their rows * cols elements lie from `data` on, with the parameter's strides.
 *   dtype     TOA_F32, TOA_F16 or TOA_BF16 (codes of toa_adam.h); all views of a call share it,
 *             except the momentum, whose type is given apart.
 *   precision products run on the matrix cores with float32 sums.  Their operands carry 22
 *             significant bits (two halves): float32 results are about as far off as those of plain
 *             float32 products.  In a bfloat16 call that keeps no iterates, those of
 *             the last orthogonalisation step may carry 11, where the coefficients keep what that
 *             adds within half a step of bfloat16 (the default ones do not).
 *   workspace device memory the call may overwrite, 256-byte aligned, as many bytes as the
 *             matching *_workspace function says; calls that may overlap in time (other streams,
 *             other captured graphs) need workspaces of their own.
 *   stream    a hipStream_t passed as void*; calls only enqueue kernels (no allocation, no copy,
 *             no memset, no synchronisation), so they can be captured.
 *   return    0; a positive hipError_t; or a negative TOA_E* (toa_muon_error_string names it).
 *             Nothing is enqueued when an argument is refused.
 *   threads   re-entrant; no global state.
 */
#ifndef TOA_MUON_H
#define TOA_MUON_H

#include <stddef.h>
#include <stdint.h>

#include "toa_adam.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    TOA_EVALUE = -5,    /* a number is out of its range (see each function)   */
    TOA_EWORKSPACE = -6 /* workspace too small or not 256-byte aligned        */
};

enum { TOA_I8 = 4 }; /* momentum type: 8-bit blocks */

/* How the step's length follows the matrix's shape. */
enum { TOA_MUON_UNIT = 0, TOA_MUON_ASPECT = 1, TOA_MUON_RMS = 2 };

typedef struct {
    void *data;
    int64_t row_stride, col_stride; /* in elements */
} toa_muon_view;

/* 1 <= steps <= 32; coefficients finite, and such that no iterate but the last can grow beyond 64
 * from a start of norm 1, and the last not beyond 1e30 (TOA_EVALUE otherwise); eps >= 0. */
typedef struct {
    int steps;
    double a, b, c, eps;
} toa_muon_series;

TOA_API int toa_muon_abi_version(void);
TOA_API const char *toa_muon_error_string(int code);

/* Bytes of workspace for a list; 0 for a list without elements.  What is refused comes through
 * `status` (may be NULL): TOA_ESIZE where a dimension is beyond 2^20. */
TOA_API size_t toa_muon_orthogonalize_workspace(int dtype, size_t num, const int64_t *rows,
                                                const int64_t *cols, const toa_muon_series *series,
                                                int keep, int *status);
TOA_API size_t toa_muon_backward_workspace(int dtype, size_t num, const int64_t *rows,
                                           const int64_t *cols, const toa_muon_series *series,
                                           int kept, int *status);

/* What the gradient needs of the forward pass -- every iterate and its products -- can be kept
 * between the two: bytes of that buffer (256-byte aligned) for a list, about 8 bytes for each
 * element of a matrix and of the square of its shorter side, for each step; lists of small
 * matrices, whose iterates are made again faster than they are read, need none in a short series. */
TOA_API size_t toa_muon_kept_bytes(int dtype, size_t num, const int64_t *rows, const int64_t *cols,
                                   const toa_muon_series *series, int *status);

/* kept: where the iterates go, or NULL.  keep / kept of the workspace functions says which. */
TOA_API int toa_muon_orthogonalize_multi(int dtype, size_t num, const int64_t *rows,
                                         const int64_t *cols, const toa_muon_view *in,
                                         const toa_muon_view *out, const toa_muon_series *series,
                                         void *kept, size_t kept_bytes, void *workspace,
                                         size_t workspace_bytes, void *stream);

/* grad_in = d<orthogonalize(in), grad_out> / d in.  kept: what the forward call with the same
 * `in`, list and series left, which is only read; or NULL: the iterates are computed again. */
TOA_API int toa_muon_orthogonalize_backward_multi(int dtype, size_t num, const int64_t *rows,
                                                  const int64_t *cols, const toa_muon_view *in,
                                                  const toa_muon_view *grad_out,
                                                  const toa_muon_view *grad_in,
                                                  const toa_muon_series *series, const void *kept,
                                                  size_t kept_bytes, void *workspace,
                                                  size_t workspace_bytes, void *stream);

/* The optimizer step (workspace as for orthogonalize).
 *   momentum_dtype  dtype, TOA_F32 or TOA_I8 (then scales[i] holds ceil(rows*cols / 128) floats)
 *   out             the parameters when `apply`, else where r * orthogonalize(U) is written (the
 *                   gradients themselves are allowed)
 *   momentum        in [0, 1); maximize steps along +g.  lr and weight_decay are read by `apply`. */
typedef struct {
    double momentum, lr, weight_decay;
    int nesterov, maximize, adjust, apply;
} toa_muon_hyper;

TOA_API int toa_muon_step_multi(int dtype, int momentum_dtype, size_t num, const int64_t *rows,
                                const int64_t *cols, const toa_muon_view *out,
                                const toa_muon_view *grads, const toa_muon_view *momentum,
                                float *const *scales, const toa_muon_hyper *hyper,
                                const toa_muon_series *series, void *workspace,
                                size_t workspace_bytes, void *stream);

/* 8-bit blocks of `num` dense arrays of n[i] elements, and back (dtype: F32, F16, BF16). */
TOA_API int toa_muon_quantize_multi(int dtype, size_t num, const void *const *in,
                                    const size_t *n, int8_t *const *codes, float *const *scales,
                                    void *stream);
TOA_API int toa_muon_dequantize_multi(int dtype, size_t num, const int8_t *const *codes,
                                      const float *const *scales, const size_t *n,
                                      void *const *out, void *stream);

#ifdef __cplusplus
}
#endif
#endif
