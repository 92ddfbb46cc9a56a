/*
 * cista_optim.h -- C ABI of the training-step operators between the backward pass and the next
 * forward pass (part of libcista_hip.so, gfx950): the norm of all gradients, clipping by it, and
 * the Adam / AdamW update.  The reference trains with Adam (train_e2v.py:63-65, train_e2v.py:120);
 * it does not clip.
 *
 *   norm     N = sqrt(sum g^2)  |  sum |g|  |  max |g|      over every element of every tensor
 *   scale    c = min(1, max_norm / (N + 1e-6)),  1 for max_norm = +inf;   g <- c g
 *   Adam     g <- c g;  g <- -g (maximize);  g <- g + wd p, or p <- p (1 - lr wd) (decoupled)
 *            t <- t + 1;  m <- m + (1 - b1)(g - m);  v <- b2 v + (1 - b2) g^2
 *            p <- p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
 *
 * The norm is rounded to float32 once (sums run in float64, so squares neither overflow nor
 * vanish); it is NaN if any element is NaN.  A NaN norm makes c NaN, an infinite one makes c 0.
 * Results do not depend on timing: the order of a sum follows from the tensors' sizes and their
 * places within a 128-byte line.
 *
 * Conventions as in cista_lstc.h: device pointers, `stream` = hipStream_t as void*, no
 * allocation, no host sync (every call can be captured in a hipGraph), CISTA_* status codes.  The
 * tables of tensors are host arrays, read before the call returns.  A tensor is a dense run of
 * `numel` elements, aligned to its element type only; numel 0 is allowed (data may then be NULL).
 * One call takes up to 2^40 elements (norm), 68 G (scale, clip) or 17 G (Adam): CISTA_ERR_UNSUPPORTED.
 */
#ifndef CISTA_OPTIM_H
#define CISTA_OPTIM_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { CISTA_F32 = 0, CISTA_BF16 = 1, CISTA_F16 = 2 };                   /* element types          */
enum { CISTA_NORM_1 = 1, CISTA_NORM_2 = 2, CISTA_NORM_MAX = 3 };         /* norms                  */

typedef struct {
    void *data;
    long long numel;
    long long type;          /* CISTA_F32 / _BF16 / _F16                                          */
} cista_tensor;

/* workspace of every call below, for n tensors; 16-byte aligned, used by one call at a time */
size_t cista_optim_workspace_bytes(int n);

/* *norm = the norm of the n tensors (float32, device); n = 0 gives 0 */
int cista_grad_norm(const cista_tensor *grads, int n, int norm_kind, float *norm, void *workspace,
                    size_t workspace_bytes, void *stream);

/* grads <- c grads with a norm that is given (float32, device).  The tensors are disjoint, and the
 * norm is outside them (checked: CISTA_ERR_ALIAS). */
int cista_scale_grads(const cista_tensor *grads, int n, double max_norm, const float *norm, void *stream);

/* both: *norm = the norm before clipping, grads <- c grads; the same holds of the tensors and the norm */
int cista_clip_grads(const cista_tensor *grads, int n, int norm_kind, double max_norm, float *norm, void *workspace,
                     size_t workspace_bytes, void *stream);

typedef struct {
    void *param;             /* `type`                                                            */
    const void *grad;        /* `type`                                                            */
    float *exp_avg;          /* m                                                                 */
    float *exp_avg_sq;       /* v                                                                 */
    float *master;           /* float32 copy that is updated where param has 16 bits; NULL for F32 */
    float *step;             /* t, advanced by 1                                                  */
    long long numel;
    long long type;
} cista_adam_tensor;

typedef struct {
    double lr, beta1, beta2, eps, weight_decay;
    const float *lr_device;  /* not NULL: the learning rate is read from here when the kernels run */
    int n;                   /* how many tensors of the table belong to the group                 */
    int decoupled;           /* weight decay on the parameter (AdamW) instead of in the gradient  */
    int maximize;
    int reserved;
} cista_adam_group;

/* One step over all groups; the table holds the groups' tensors one group after the other.
 * norm_kind 0: no clipping (max_norm and norm are not used); else every gradient is scaled by c
 * of the norm over all groups, which goes to *norm; the gradients in memory stay as they are.
 * The parameters are disjoint, and so are the m, the v, the master copies and the steps, and the
 * norm is outside them and the gradients (checked: CISTA_ERR_ALIAS); nor do two of these kinds share
 * memory (not checked). */
int cista_adam_step(const cista_adam_tensor *table, const cista_adam_group *groups, int n_groups, int norm_kind,
                    double max_norm, float *norm, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* CISTA_OPTIM_H */
