/* Layer norm with its gradients, and clipping by the global gradient norm, for the PPO trainer that drives the env path
 * (multigrid_amd/ppo.py: policies whose parameters and gradients carry a leading agent axis, clipped agent by agent,
 * v8_robust_ppo.py:340).  The entry points live in libmgnn.so next to those of mgrid_nn.h, whose error codes they extend;
 * multigrid_amd/norm_ops.py binds them.
 *
 * Every call enqueues its kernels on `stream` (a hipStream_t; NULL = the default stream) of the CURRENT device and returns
 * without synchronising; nothing is allocated, and nothing is kept between calls.  Workspaces belong to the caller: one
 * workspace per call in flight (two captured graphs that may run at once need one each), contents undefined before and
 * after.  Results do not depend on the launch order of workgroups: the same inputs give the same bits.
 * Pointers need the alignment of their element type only.
 */
#ifndef MGRID_NORM_H
#define MGRID_NORM_H

#include <stdint.h>
#include "mgrid_nn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MGNN_ERR_TYPE 3      /* an element type that is none of MGNN_F32 / MGNN_BF16 / MGNN_F16, or not allowed there */
#define MGNN_ERR_WORKSPACE 4 /* the workspace is too small, missing or not aligned to 8 bytes */
#define MGNN_ERR_VALUE 5     /* eps or max_norm negative or NaN, a required pointer missing, the norm's gradient list invalid */
#define MGNN_ERR_OVERLAP 6   /* a gradient that is written overlaps another one of the same call */
#define MGNN_ERR_MEMORY 7    /* no host memory for the list's tables */

#define MGNN_F32 0
#define MGNN_BF16 1
#define MGNN_F16 2

/* longest row of mgnn_layer_norm, most groups of either operator */
#define MGNN_LN_MAX_C 16384
#define MGNN_MAX_GROUPS 65535

/* y[g][r][c] = (x[g][r][c] - m) * s * weight[g][c] + bias[g][c] with m the mean of row (g, r) and s = 1 / sqrt(its mean
 * squared deviation + eps); sums, means and s are fp32.  x: groups * rows rows, `ld` elements from one to the next (ld >= C;
 * a row's elements are contiguous); y: rows contiguous, must not overlap x.  weight / bias: [groups][C] of type wtype (that of x, or
 * MGNN_F32), either may be NULL (1 and 0).  stats: NULL, or float [groups * rows][2] that receives (m, s) for the backward
 * pass.  1 <= C <= MGNN_LN_MAX_C, groups <= MGNN_MAX_GROUPS; no rows or no groups: nothing is done. */
int mgnn_layer_norm(const void* x, int64_t ld, const void* weight, const void* bias, void* y, float* stats, int64_t groups,
                    int64_t rows, int C, double eps, int type, int wtype, void* stream);

/* bytes of workspace that mgnn_layer_norm_backward wants for these sizes when it computes dweight or dbias (0 = none; -1 =
 * sizes or type that it refuses) */
int64_t mgnn_layer_norm_workspace(int64_t groups, int64_t rows, int C, int type);

/* With h = (x - m) * s and e = dy * weight:  dx = s * (e - mean(e) - h * mean(e * h)) per row,
 * dweight[g][c] = sum over r of dy * h, dbias[g][c] = sum over r of dy (zeros without rows).  dy and dx: rows contiguous;
 * dx may be dy itself.  Any of dx, dweight, dbias may be NULL (not wanted); weight NULL = 1.  dweight / dbias are of type
 * wtype.  The sums over rows are fp32, split over workgroups whose shares are added in a fixed order. */
int mgnn_layer_norm_backward(const void* x, int64_t ld, const void* dy, const void* weight, const float* stats, void* dx,
                             void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, int64_t groups, int64_t rows,
                             int C, int type, int wtype, void* stream);

/* bytes of workspace for mgnn_grad_norm and mgnn_clip_grads with this list (0 = none; -1 = a list that they refuse).
 * A list of gradients: `count` tensors of n[i] * groups contiguous elements of type[i], group g's being the g-th n[i] of them. */
int64_t mgnn_grad_norm_workspace(const int64_t* n, const int32_t* type, int64_t count, int64_t groups);

/* norms[g] = sqrt(sum over all tensors of the squares of group g's elements), accumulated in fp64 and rounded to fp32 */
int mgnn_grad_norm(const void* const* src, const int64_t* n, const int32_t* type, int64_t count, int64_t groups, float* norms,
                   void* workspace, int64_t workspace_bytes, void* stream);

/* norms as above, and dst[i] = src[i] * min(1, max_norm / (norms[g] + 1e-6)) in fp32, rounded to type[i]; a factor that is
 * NaN (a norm that is NaN) makes every element NaN.  dst[i] is src[i] (in place) or memory that no other tensor of the
 * call overlaps. */
int mgnn_clip_grads(const void* const* src, void* const* dst, const int64_t* n, const int32_t* type, int64_t count,
                    int64_t groups, double max_norm, float* norms, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
