/*
 * powersparse_rows.h — the row operators of a model that trains on graphs:
 * those whose sparse matrix follows from ids (embedding lookup and its gradient,
 * tokens sorted by expert and back with their gradients), the router that
 * chooses the ids, layer norm, and the end of a step (the norm and clipping of
 * many gradient tensors, AdamW). No reference counterpart.
 *
 * Same library, status codes and streams as powersparse_hip.h: every call
 * checks its arguments on the host, enqueues its kernels on `stream` and
 * returns; nothing but making a list of tensors synchronises or allocates, and
 * nothing is kept between calls. Workspaces are the caller's, of the stated
 * size or more, aligned to 16 bytes, not shared by calls that may overlap. The
 * stated sizes grow with every argument, so a workspace for the largest call
 * does for smaller ones. What a call writes (outputs, workspace) shares no byte
 * with anything else it is given, clipping in place and what AdamW updates aside;
 * PS_ERR_INVALID otherwise.
 *
 * Data may hold any value: ids and positions out of range are dropped where
 * the text says so and never followed. Arithmetic runs in 32 bits (norms in
 * 64), sums in an order that the call's sizes and ids fix (the same bits every
 * time), and what it gives is rounded to the output's type, to nearest even.
 */
#ifndef POWERSPARSE_ROWS_H
#define POWERSPARSE_ROWS_H

#include <stddef.h>
#include <stdint.h>

#include "powersparse_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of ps_rows and of gradient tensors. */
#define PS_F32 0
#define PS_F16 1
#define PS_BF16 2
/* Of optimizer states only: 8 bits, FP8 as OCP defines it, by blocks (below). */
#define PS_E4M3 3

/* Id types. */
#define PS_I32 0
#define PS_I64 1

/* A row-major matrix in device memory: element (r, c) is data[r * ld + c],
 * ld >= cols in elements. data is aligned to its element only; rows * ld stays
 * below 2^48. cols may be anything from 1 to 2^24. */
typedef struct ps_rows {
  void* data;
  long long rows, cols, ld;
  int dtype;
} ps_rows;

/* `count` ids, one after another, in device memory. */
typedef struct ps_ids {
  const void* data;
  long long count;
  int type;
} ps_ids;

/* out[i, :] = scale * table[ids[i], :], zeros where ids[i] is outside
 * [0, table->rows). out has ids->count rows; the types may differ. */
int ps_embedding_lookup(const ps_rows* table, const ps_ids* ids, float scale, const ps_rows* out,
                        ps_stream_t stream);

/* grad[v, :] = scale * (sum of grad_out[i, :] over the i with ids[i] = v), zeros
 * for rows without ids; with accumulate != 0 the sum is added to grad and other
 * rows are left alone. Ids outside [0, grad->rows) and those equal to padding_idx
 * (negative: none) take no part. At most 2^30 ids, 2^31 - 2 rows. A row's terms
 * are added in the order of i, in parts where there are many: where these are cut
 * follows from the count, the width and the other ids, so the same row's last
 * bits may differ in a batch of another size. */
size_t ps_embedding_grad_workspace_bytes(long long count, long long cols, long long table_rows);
int ps_embedding_grad(const ps_ids* ids, const ps_rows* grad_out, float scale,
                      long long padding_idx, int accumulate, const ps_rows* grad, void* workspace,
                      size_t workspace_bytes, ps_stream_t stream);

/* Stable sort of slots by expert. ids: the experts of slot i, i = token *
 * top_k + k. order: the slots by (expert, i), the dropped ones (id outside [0,
 * experts)) last; position[order[s]] = s, -1 for dropped slots;
 * offsets[e], e = 0 .. experts: the slots of experts below e. 1 to 1024
 * experts, at most 2^30 slots. */
size_t ps_expert_sort_workspace_bytes(long long slots, int experts);
int ps_expert_sort(const ps_ids* ids, int experts, int* order, int* position, int* offsets,
                   void* workspace, size_t workspace_bytes, ps_stream_t stream);

/* xs[position[t * top_k + k], :] = x[t, :]. position holds x->rows * top_k
 * values, all different where they are not negative; those outside [0,
 * xs->rows) are skipped, and rows of xs that no position names are left alone.
 * x and xs have one type. */
int ps_expert_dispatch(const ps_rows* x, const int* position, int top_k, const ps_rows* xs,
                       ps_stream_t stream);

/* y[t, :] = sum over k of weights[t * top_k + k] * ys[position[t * top_k + k], :],
 * positions outside [0, ys->rows) skipped whatever their weight; weights ==
 * NULL: all ones, which is the gradient of ps_expert_dispatch. ys and y have
 * one type. */
int ps_expert_combine(const ps_rows* ys, const int* position, const float* weights, int top_k,
                      const ps_rows* y, ps_stream_t stream);

/* The gradients of ps_expert_combine: dys[p, :] = weights[s] * dy[t, :] and
 * dweights[s] = <dy[t, :], ys[p, :]> with s = t * top_k + k, p = position[s];
 * dweights[s] = 0 where p is outside [0, ys->rows); rows of dys that no
 * position names are left alone. dy, ys and dys have one type. */
int ps_expert_combine_grad(const ps_rows* dy, const ps_rows* ys, const int* position,
                           const float* weights, int top_k, const ps_rows* dys, float* dweights,
                           ps_stream_t stream);

/* The router. With p the softmax of a token's row of logits (tokens x experts):
 * ids[t * top_k + k], k = 0 .. top_k - 1, are the experts of its largest logits in
 * descending order, equal ones by ascending expert (a NaN counts as the largest, and
 * makes the token's weights NaN); weights, of the same places, their p, or with
 * normalize != 0 p divided by the sum over the chosen ones. An expert whose logit
 * is -inf is barred: never chosen. Places left over have id -1 and weight 0. mask
 * (NULL: none): a byte for each token, 0 where it is padding; such tokens, and those
 * with all experts barred, take no part and have no experts.
 * counts (experts + 1 values): how often each expert was chosen, and last the tokens
 * that take part; loss (one value) = experts * sum over e of f_e * P_e, f_e the
 * choices' share that is e's and P_e the mean of p over those tokens: 1 where all
 * is balanced, 0 without tokens. Both NULL: not wanted, nor the workspace then.
 * 1 to 1024 experts, top_k up to as many, at most 2^30 slots. */
size_t ps_expert_route_workspace_bytes(long long tokens, int experts);
int ps_expert_route(const ps_rows* logits, int top_k, int normalize, const unsigned char* mask,
                    int* ids, float* weights, int* counts, float* loss, void* workspace,
                    size_t workspace_bytes, ps_stream_t stream);

/* dlogits = the gradient of sum(dweights * weights) + *dloss * loss by the logits,
 * the choices as they are: ids (a token's all different where they are not negative)
 * and counts are what ps_expert_route gave. Counts may be summed over the ranks of
 * a job: the gradient is of the loss over all their tokens then. dweights NULL:
 * zeros; dloss (device) NULL: no loss, and counts may be NULL too. A token whose
 * first id is negative gets zeros. */
int ps_expert_route_grad(const ps_rows* logits, int top_k, int normalize, const int* ids,
                         const float* dweights, const int* counts, const float* dloss,
                         const ps_rows* dlogits, ps_stream_t stream);

/* y[r, :] = (x[r, :] - mean) * rstd * weight + bias with mean the row's mean and
 * rstd = 1 / sqrt(mean of (x - mean)^2 + eps). weight and bias hold one row of
 * x->cols elements, of any type; NULL: ones and zeros. mean and rstd, a value for
 * each row, are for the gradient (NULL: not wanted). x and y may differ in type.
 * eps is a number from 0 up; with 0 a row of one value gives NaN. */
int ps_layer_norm(const ps_rows* x, const ps_rows* weight, const ps_rows* bias, float eps,
                  const ps_rows* y, float* mean, float* rstd, ps_stream_t stream);

/* Its gradients, with xh = (x - mean) * rstd and g = dy * weight:
 * dx = rstd * (g - (mean of g) - xh * (mean of g * xh)), dweight = sum over the
 * rows of dy * xh, dbias = sum over the rows of dy. weight NULL: ones; dweight and
 * dbias, one row each, NULL: not wanted; accumulate != 0: the sums are added to
 * them. dx has x's type; dy, weight, dweight and dbias may have others. Where the
 * rows' sums are cut follows from the sizes. The workspace is 32 MB at most up to
 * 262,144 columns and 128 bytes a column beyond. */
size_t ps_layer_norm_grad_workspace_bytes(long long rows, long long cols);
int ps_layer_norm_grad(const ps_rows* dy, const ps_rows* x, const ps_rows* weight,
                       const float* mean, const float* rstd, int accumulate, const ps_rows* dx,
                       const ps_rows* dweight, const ps_rows* dbias, void* workspace,
                       size_t workspace_bytes, ps_stream_t stream);

/* The gradient tensors of a model: data[i] holds counts[i] contiguous elements
 * of dtypes[i]. out (NULL: in place) and out_dtypes name where the clipped
 * gradients go; nothing that is written may overlap another tensor, no norm may
 * lie in an output, and none be written into a gradient (PS_ERR_INVALID).
 * Uploads a table and synchronises; owns it and what the calls below work in (8
 * bytes for 4096 elements): calls on one list must not overlap. */
typedef struct ps_grad_list ps_grad_list;
int ps_grad_list_create(int tensors, void* const* data, const long long* counts,
                        const int* dtypes, void* const* out, const int* out_dtypes,
                        ps_grad_list** list);
/* Waits for nothing and may come during a capture, and while calls on the list
 * are under way: its memory goes back when the next list is made. */
void ps_grad_list_destroy(ps_grad_list* list);

/* *norm (device) = sqrt(sum of (grad_scale * g)^2 over every element), summed
 * in 64 bits; 0 for no elements. Only reads the gradients. */
int ps_grad_norm(ps_grad_list* list, float grad_scale, float* norm, ps_stream_t stream);

/* out = c * grad_scale * g with c = min(1, max_norm / (*norm + 1e-6)), norm
 * (device) as given, for instance over the ranks of a job. Where nothing would
 * change (in place, c * grad_scale = 1) nothing is read or written. A NaN norm
 * makes every output NaN, an infinite one zeros and NaN. */
int ps_clip_grads(ps_grad_list* list, float max_norm, float grad_scale, const float* norm,
                  ps_stream_t stream);

/* ps_grad_norm and ps_clip_grads in two launches, bit for bit: *norm receives the
 * norm before clipping, and that FP32 value is clipped by. */
int ps_clip_grad_norm(ps_grad_list* list, float max_norm, float grad_scale, float* norm,
                      ps_stream_t stream);

/* A parameter of `count` contiguous elements, its gradient (only read) and its
 * moments, which a step updates in place. Moments of PS_F32 begin with zeros.
 * Those of PS_E4M3 are codes, a byte an element, and scales, a pair of floats for
 * every 256 elements (the last of them may be fewer): exp_avg = code * pair[0],
 * the square root of exp_avg_sq = code * pair[1]; they too begin with zeros. copy
 * (NULL: none) receives the new parameter rounded to copy_dtype. */
typedef struct ps_adamw_tensor {
  void* param;
  const void* grad;
  void *exp_avg, *exp_avg_sq;
  float* scales;
  void* copy;
  long long count;
  int param_dtype, grad_dtype, copy_dtype;
  float weight_decay;
} ps_adamw_tensor;

/* Nothing that a step writes may overlap another argument of the list's
 * (PS_ERR_INVALID). state_dtype: PS_F32 or PS_E4M3, of all moments. Uploads a table
 * and synchronises; owns it. Steps of one list must not overlap. */
typedef struct ps_adamw_list ps_adamw_list;
int ps_adamw_list_create(int tensors, const ps_adamw_tensor* list, int state_dtype,
                         ps_adamw_list** out);
/* As ps_grad_list_destroy. */
void ps_adamw_list_destroy(ps_adamw_list* list);

/* step: the number of this update, from 1. device_lr, device_step and norm (device,
 * one value each): NULL, or read when the step runs, lr and step ignored then (a
 * device step below 1 counts as 1); none may lie in what the step writes. lr and eps
 * are numbers within FP32's range, eps from 0 up (PS_ERR_INVALID otherwise). */
typedef struct ps_adamw_options {
  double lr, beta1, beta2, eps;
  long long step;
  const float* device_lr;
  const int* device_step;
  const float* norm;
  float max_norm, grad_scale;
} ps_adamw_options;

/* With g = c * grad, c = grad_scale, or with a norm (of grad_scale * grad, as
 * ps_grad_norm gives it) grad_scale * min(1, max_norm / (*norm + 1e-6)):
 * exp_avg = beta1 * exp_avg + (1 - beta1) * g,
 * exp_avg_sq = beta2 * exp_avg_sq + (1 - beta2) * g^2,
 * param -= lr * (weight_decay * param + (exp_avg / (1 - beta1^step)) /
 * (sqrt(exp_avg_sq / (1 - beta2^step)) + eps)). A norm that is not finite: nothing
 * changes, and `step` is not to count such a call (with four counted before it the
 * first update is 0.55 of its size); a step on the device can be advanced by whether
 * the norm is finite. The parameter moves by the moments before they are rounded to 8
 * bits; there they go to either neighbouring code, by a rule of step and place that
 * keeps the mean of exp_avg and of exp_avg_sq's root over the steps, and a second moment
 * that is not zero stays so. Single elements walk about their exact course: under
 * random gradients and beta2 = 0.999 roots by 15% (rms), which makes exp_avg_sq some 4%
 * too large on average.
 * A gradient that is not finite makes its element's moments so, in 8 bits its
 * block's. */
int ps_adamw_step(ps_adamw_list* list, const ps_adamw_options* options, ps_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* POWERSPARSE_ROWS_H */
