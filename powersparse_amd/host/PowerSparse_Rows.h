// The row operators (powersparse_rows.h) for C++ callers: the same entry points
// with errors as exceptions (PS_ERR_INVALID -> std::invalid_argument, else
// std::runtime_error), and the lists of tensors as owners. No reference
// counterpart. Matrices and ids are the C ABI's ps_rows and ps_ids; every call is
// enqueued on `stream` and returns.
#ifndef POWERSPARSE_ROWS_HOST_H
#define POWERSPARSE_ROWS_HOST_H

#include <stdexcept>
#include <vector>

#include "matrix_utils.h"
#include "powersparse_rows.h"

namespace PowerSparse {

// out[i] = scale * table[ids[i]], zeros for ids outside the table.
inline void EmbeddingLookup(const ps_rows& table, const ps_ids& ids, float scale,
                            const ps_rows& out, ps_stream_t stream = nullptr) {
  ThrowOnError(ps_embedding_lookup(&table, &ids, scale, &out, stream));
}

// grad[v] = (accumulate: +=) scale * sum of grad_out[i] over the i with ids[i] = v.
// workspace: ps_embedding_grad_workspace_bytes(ids.count, grad.cols, grad.rows).
inline void EmbeddingGrad(const ps_ids& ids, const ps_rows& grad_out, float scale,
                          const ps_rows& grad, void* workspace, size_t workspace_bytes,
                          long long padding_idx = -1, bool accumulate = false,
                          ps_stream_t stream = nullptr) {
  ThrowOnError(ps_embedding_grad(&ids, &grad_out, scale, padding_idx, accumulate, &grad, workspace,
                                 workspace_bytes, stream));
}

// The slots of `ids` by expert: order, position (-1: dropped) and offsets
// (experts + 1). workspace: ps_expert_sort_workspace_bytes(ids.count, experts).
inline void ExpertSort(const ps_ids& ids, int experts, int* order, int* position, int* offsets,
                       void* workspace, size_t workspace_bytes, ps_stream_t stream = nullptr) {
  ThrowOnError(ps_expert_sort(&ids, experts, order, position, offsets, workspace, workspace_bytes,
                              stream));
}

// xs[position[t, k]] = x[t].
inline void ExpertDispatch(const ps_rows& x, const int* position, int top_k, const ps_rows& xs,
                           ps_stream_t stream = nullptr) {
  ThrowOnError(ps_expert_dispatch(&x, position, top_k, &xs, stream));
}

// y[t] = sum over k of weights[t, k] * ys[position[t, k]].
inline void ExpertCombine(const ps_rows& ys, const int* position, const float* weights, int top_k,
                          const ps_rows& y, ps_stream_t stream = nullptr) {
  if (!weights) throw std::invalid_argument("ExpertCombine: null weights");
  ThrowOnError(ps_expert_combine(&ys, position, weights, top_k, &y, stream));
}

// The gradient of ExpertDispatch: dx[t] = sum over k of dxs[position[t, k]].
inline void ExpertDispatchGrad(const ps_rows& dxs, const int* position, int top_k,
                               const ps_rows& dx, ps_stream_t stream = nullptr) {
  ThrowOnError(ps_expert_combine(&dxs, position, nullptr, top_k, &dx, stream));
}

// The gradients of ExpertCombine.
inline void ExpertCombineGrad(const ps_rows& dy, const ps_rows& ys, const int* position,
                              const float* weights, int top_k, const ps_rows& dys, float* dweights,
                              ps_stream_t stream = nullptr) {
  ThrowOnError(ps_expert_combine_grad(&dy, &ys, position, weights, top_k, &dys, dweights, stream));
}

// The router: ids and weights (logits.rows x top_k) of every token's experts, mask
// (null: none) a byte a token. counts (experts + 1) and loss (one value), or null for
// both and the workspace: ps_expert_route_workspace_bytes(logits.rows, logits.cols).
inline void ExpertRoute(const ps_rows& logits, int top_k, int* ids, float* weights,
                        int* counts = nullptr, float* loss = nullptr, void* workspace = nullptr,
                        size_t workspace_bytes = 0, const unsigned char* mask = nullptr,
                        bool normalize = true, ps_stream_t stream = nullptr) {
  ThrowOnError(ps_expert_route(&logits, top_k, normalize, mask, ids, weights, counts, loss,
                               workspace, workspace_bytes, stream));
}

// dlogits = the gradient of sum(dweights * weights) + *dloss * loss; dweights null:
// zeros, dloss null: no loss.
inline void ExpertRouteGrad(const ps_rows& logits, int top_k, const int* ids,
                            const float* dweights, const int* counts, const float* dloss,
                            const ps_rows& dlogits, bool normalize = true,
                            ps_stream_t stream = nullptr) {
  ThrowOnError(ps_expert_route_grad(&logits, top_k, normalize, ids, dweights, counts, dloss,
                                    &dlogits, stream));
}

// y = (x - mean) * rstd * weight + bias for every row; weight and bias (one row
// each) or null, mean and rstd (a value a row) or null.
inline void LayerNorm(const ps_rows& x, const ps_rows* weight, const ps_rows* bias, float eps,
                      const ps_rows& y, float* mean = nullptr, float* rstd = nullptr,
                      ps_stream_t stream = nullptr) {
  ThrowOnError(ps_layer_norm(&x, weight, bias, eps, &y, mean, rstd, stream));
}

// The gradients of LayerNorm; dweight and dbias null: not wanted, nor the workspace
// then: ps_layer_norm_grad_workspace_bytes(x.rows, x.cols).
inline void LayerNormGrad(const ps_rows& dy, const ps_rows& x, const ps_rows* weight,
                          const float* mean, const float* rstd, const ps_rows& dx,
                          const ps_rows* dweight, const ps_rows* dbias, void* workspace,
                          size_t workspace_bytes, bool accumulate = false,
                          ps_stream_t stream = nullptr) {
  ThrowOnError(ps_layer_norm_grad(&dy, &x, weight, mean, rstd, accumulate, &dx, dweight, dbias,
                                  workspace, workspace_bytes, stream));
}

// A gradient tensor: `count` contiguous elements of `dtype` (PS_F32, ...).
struct Gradient {
  void* data;
  long long count;
  int dtype;
};

// The gradient tensors of a model and where their clipped values go.
class GradientList {
 public:
  // outs: one of the same count for each, or empty for in place.
  explicit GradientList(const std::vector<Gradient>& grads,
                        const std::vector<Gradient>& outs = {}) {
    if (!outs.empty() && outs.size() != grads.size())
      throw std::invalid_argument("GradientList: one output for each gradient");
    std::vector<void*> data, to;
    std::vector<long long> counts;
    std::vector<int> types, to_types;
    for (size_t i = 0; i < grads.size(); ++i) {
      data.push_back(grads[i].data);
      counts.push_back(grads[i].count);
      types.push_back(grads[i].dtype);
      if (outs.empty()) continue;
      if (outs[i].count != grads[i].count)
        throw std::invalid_argument("GradientList: an output of another size");
      to.push_back(outs[i].data);
      to_types.push_back(outs[i].dtype);
    }
    ThrowOnError(ps_grad_list_create(int(grads.size()), data.data(), counts.data(), types.data(),
                                     outs.empty() ? nullptr : to.data(),
                                     outs.empty() ? nullptr : to_types.data(), &list_));
  }
  ~GradientList() { ps_grad_list_destroy(list_); }
  GradientList(const GradientList&) = delete;
  GradientList& operator=(const GradientList&) = delete;

  // *norm (device) = the 2-norm of grad_scale * g.
  void Norm(float* norm, float grad_scale = 1.f, ps_stream_t stream = nullptr) const {
    ThrowOnError(ps_grad_norm(list_, grad_scale, norm, stream));
  }
  // g * grad_scale * min(1, max_norm / (*norm + 1e-6)), the norm given.
  void Clip(float max_norm, const float* norm, float grad_scale = 1.f,
            ps_stream_t stream = nullptr) const {
    ThrowOnError(ps_clip_grads(list_, max_norm, grad_scale, norm, stream));
  }
  // Both; *norm receives the norm before clipping.
  void ClipNorm(float max_norm, float* norm, float grad_scale = 1.f,
                ps_stream_t stream = nullptr) const {
    ThrowOnError(ps_clip_grad_norm(list_, max_norm, grad_scale, norm, stream));
  }

 private:
  ps_grad_list* list_ = nullptr;
};

// The tensors that AdamW updates (ps_adamw_tensor says what each holds).
class AdamWList {
 public:
  // state_dtype: PS_F32, or PS_E4M3 for moments in 8 bits.
  explicit AdamWList(const std::vector<ps_adamw_tensor>& tensors, int state_dtype = PS_F32) {
    ThrowOnError(ps_adamw_list_create(int(tensors.size()), tensors.data(), state_dtype, &list_));
  }
  ~AdamWList() { ps_adamw_list_destroy(list_); }
  AdamWList(const AdamWList&) = delete;
  AdamWList& operator=(const AdamWList&) = delete;

  void Step(const ps_adamw_options& options, ps_stream_t stream = nullptr) const {
    ThrowOnError(ps_adamw_step(list_, &options, stream));
  }

 private:
  ps_adamw_list* list_ = nullptr;
};

}  // namespace PowerSparse

#endif  // POWERSPARSE_ROWS_HOST_H
