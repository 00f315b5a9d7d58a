/*
 * powersparse_rows.h — row operators whose sparse matrix follows from ids:
 * embedding lookup and its gradient, tokens sorted by expert and back with
 * their gradients, and the norm and clipping of many gradient tensors.
 * No reference counterpart.
 *
 * Same library, status codes and streams as powersparse_hip.h: every call
 * checks its arguments on the host, enqueues its kernels on `stream` and
 * returns; nothing but ps_grad_list_create synchronises or allocates, and nothing
 * is kept between calls. Workspaces are the caller's, of the stated
 * size or more, aligned to 16 bytes, not shared by calls that may overlap. The
 * stated sizes grow with every argument, so a workspace for the largest call
 * does for smaller ones. What a call writes (outputs, workspace) shares no byte
 * with anything else it is given, clipping in place aside; PS_ERR_INVALID
 * otherwise.
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

#ifdef __cplusplus
}
#endif

#endif /* POWERSPARSE_ROWS_H */
