// The router of a mixture of experts: softmax of a token's logits, its top_k
// experts and their weights, how often each expert was chosen, the loss that
// asks for balance among them, and the gradient.
//
// kLanes threads share a token, each with kPer of its logits in registers:
// expert e is element e / kLanes of lane e % kLanes. The largest logits are
// found one after another, by keys that order as the logits do; equal ones go to
// the lowest expert.
#include "ps_rows.hpp"

namespace ps {
namespace {

constexpr int kMostExperts = 1024;

// Unsigned numbers that order as logits do, 0 for barred ones (-inf), the most
// for NaN; -0 and 0 are equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  if (v != v) return ~0u;
  if (v == -INFINITY) return 0;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// (~0 comes back as a NaN)
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// Over the kLanes lanes of a token, in every one of them.
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  return lanes_all<kLanes>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int kLanes>
__device__ __forceinline__ uint32_t lanes_min(uint32_t v) {
  return lanes_all<kLanes>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}

// What the workgroups leave of the loss: sums of probabilities, and choices of
// every expert with the tokens that take part behind them.
struct RouteParts {
  float* sums;  // blocks x experts
  int* counts;  // blocks x (experts + 1)
};

template <typename T, int kLanes, int kPer, int kThreads>
__global__ __launch_bounds__(kThreads) void route_kernel(
    Mat<const T> logits, int experts, int top_k, bool normalize,
    const unsigned char* __restrict__ mask, int* __restrict__ ids, float* __restrict__ weights,
    RouteParts parts) {
  constexpr int kTokens = kThreads / kLanes;
  __shared__ int chosen[kMostExperts + 1];
  __shared__ float sums[kMostExperts];
  const int lane = threadIdx.x % kLanes;
  if (parts.sums) {
    for (int e = threadIdx.x; e <= experts; e += kThreads) {
      chosen[e] = 0;
      if (e < experts) sums[e] = 0.f;
    }
    __syncthreads();
  }
  float acc[kPer];
#pragma unroll
  for (int r = 0; r < kPer; ++r) acc[r] = 0.f;
  // all lanes of a workgroup take the same turns, with a token or without
  for (long long t0 = (long long)blockIdx.x * kTokens; t0 < logits.rows;
       t0 += (long long)gridDim.x * kTokens) {
    const long long t = t0 + threadIdx.x / kLanes;
    const bool mine = t < logits.rows, on = mine && (!mask || mask[t]);
    uint32_t key[kPer];
    uint32_t most = 0;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int e = r * kLanes + lane;
      key[r] = on && e < experts ? key_of(float(*logits.at(t, e))) : 0;
      most = max(most, key[r]);
    }
    most = lanes_max<kLanes>(most);
    const float top = most ? value_of(most) : 0.f;  // nothing to choose: no probabilities either
    float p[kPer], s = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      p[r] = key[r] ? expf(value_of(key[r]) - top) : 0.f;
      s += p[r];
    }
    s = lanes_sum<kLanes>(s);
    const float scale = most ? 1.f / s : 0.f;
    if (parts.sums) {
#pragma unroll
      for (int r = 0; r < kPer; ++r) acc[r] += p[r] * scale;
      if (lane == 0 && most) atomicAdd(&chosen[experts], 1);
    }
    int* const ids_t = ids + t * top_k;
    float* const weights_t = weights + t * top_k;
    float total = 0.f, my_w = 0.f;
    int my_id = -1;  // slot k's are kept by lane k % kLanes
    for (int k = 0; k < top_k; ++k) {
      uint32_t best = 0, at = ~0u;
#pragma unroll
      for (int r = 0; r < kPer; ++r) best = max(best, key[r]);
      best = lanes_max<kLanes>(best);
      if (best) {
#pragma unroll
        for (int r = kPer - 1; r >= 0; --r)
          if (key[r] == best) at = uint32_t(r * kLanes + lane);
      }
      at = lanes_min<kLanes>(at);
#pragma unroll
      for (int r = 0; r < kPer; ++r)
        if (at == uint32_t(r * kLanes + lane)) key[r] = 0;
      const float w = best ? expf(value_of(best) - top) : 0.f;
      total += w;
      if (lane == k % kLanes) {
        my_id = int(at);
        my_w = normalize ? w : w * scale;
      }
      if (top_k > kLanes && (k % kLanes == kLanes - 1 || k + 1 == top_k)) {
        const int slot = k - k % kLanes + lane;
        if (slot <= k && mine) {
          if (parts.sums && my_id >= 0) atomicAdd(&chosen[my_id], 1);
          ids_t[slot] = my_id;
          weights_t[slot] = my_w;
        }
      }
    }
    if (top_k <= kLanes) {
      if (lane < top_k && mine) {
        if (parts.sums && my_id >= 0) atomicAdd(&chosen[my_id], 1);
        ids_t[lane] = my_id;
        weights_t[lane] = normalize && most ? my_w / total : my_w;
      }
    } else if (normalize && mine) {
      for (int k = lane; k < top_k; k += kLanes) weights_t[k] = most ? weights_t[k] / total : 0.f;
    }
  }
  if (!parts.sums) return;
  // The tokens of a wave, then the waves in order.
#pragma unroll
  for (int r = 0; r < kPer; ++r)
#pragma unroll
    for (int d = kLanes; d < kWave; d <<= 1) acc[r] += __shfl_xor(acc[r], d, kWave);
  for (int w = 0; w < kThreads / kWave; ++w) {
    __syncthreads();
    if (int(threadIdx.x / kWave) == w && lane_id() < kLanes)
#pragma unroll
      for (int r = 0; r < kPer; ++r)
        if (r * kLanes + lane < experts) sums[r * kLanes + lane] += acc[r];
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= experts; e += kThreads) {
    parts.counts[size_t(blockIdx.x) * (experts + 1) + e] = chosen[e];
    if (e < experts) parts.sums[size_t(blockIdx.x) * experts + e] = sums[e];
  }
}

// The workgroups' parts added up, and the loss: one workgroup, a thread an
// expert, the parts dealt to as many threads of the same expert as there are.
constexpr int kJoinThreads = 1024, kJoinAhead = 8;
__global__ __launch_bounds__(kJoinThreads) void route_join_kernel(RouteParts parts, int part_count,
                                                                  int experts, int groups,
                                                                  int* __restrict__ counts,
                                                                  float* __restrict__ loss) {
  __shared__ int count_of[kJoinThreads];
  __shared__ double sum_of[kJoinThreads];
  __shared__ int all_counts[kMostExperts];
  __shared__ double products[kMostExperts];
  const int per = kJoinThreads / groups;  // threads of a group, one an expert
  const int e = threadIdx.x % per, group = threadIdx.x / per;
  int c = 0, tokens = 0;
  double s = 0;
  if (e < experts) {
    for (int b0 = group; b0 < part_count; b0 += groups * kJoinAhead) {
      int counts_of[kJoinAhead];
      float sums_of[kJoinAhead];
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const int b = b0 + j * groups;
        counts_of[j] = b < part_count ? parts.counts[size_t(b) * (experts + 1) + e] : 0;
        sums_of[j] = b < part_count ? parts.sums[size_t(b) * experts + e] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        c += counts_of[j];
        s += double(sums_of[j]);
      }
    }
  }
  if (threadIdx.x < kWave)
    for (int b = threadIdx.x; b < part_count; b += kWave)
      tokens += parts.counts[size_t(b) * (experts + 1) + experts];
  count_of[threadIdx.x] = c;
  sum_of[threadIdx.x] = s;
  __syncthreads();
  if (group == 0) {
    for (int g = 1; g < groups; ++g) {
      c += count_of[g * per + e];
      s += sum_of[g * per + e];
    }
    if (e < experts) counts[e] = c;
    all_counts[e] = c;
    products[e] = double(c) * s;
  }
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  long long total = 0;
  double sum = 0;
  for (int i = threadIdx.x; i < per; i += kWave) {
    total += all_counts[i];
    sum += products[i];
  }
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) {
    tokens += __shfl_xor(tokens, d, kWave);
    total += __shfl_xor(total, d, kWave);
    sum += __shfl_xor(sum, d, kWave);
  }
  if (threadIdx.x == 0) {
    counts[experts] = tokens;
    *loss = tokens ? float(sum * experts / (double(tokens) * double(total))) : 0.f;
  }
}

constexpr int kRouteGradThreads = 256;
template <typename T, int kLanes, int kPer>
__global__ __launch_bounds__(kRouteGradThreads) void route_grad_kernel(
    Mat<const T> logits, int experts, int top_k, bool normalize, const int* __restrict__ ids,
    const float* __restrict__ dweights, const int* __restrict__ counts,
    const float* __restrict__ dloss, Mat<T> dlogits) {
  constexpr int kTokens = kRouteGradThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  // The loss's gradient by an expert's probability.
  float by_loss[kPer];
#pragma unroll
  for (int r = 0; r < kPer; ++r) by_loss[r] = 0.f;
  if (dloss) {
    float total = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int e = r * kLanes + lane;
      by_loss[r] = e < experts ? float(counts[e]) : 0.f;
      total += by_loss[r];
    }
    total = lanes_sum<kLanes>(total) * float(counts[experts]);
    const float scale = total > 0.f ? *dloss * float(experts) / total : 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) by_loss[r] *= scale;
  }
  for (long long t0 = (long long)blockIdx.x * kTokens; t0 < logits.rows;
       t0 += (long long)gridDim.x * kTokens) {
    const long long t = t0 + threadIdx.x / kLanes;
    const bool mine = t < logits.rows;
    const int* const ids_t = ids + t * top_k;
    const bool on = mine && ids_t[0] >= 0;
    float p[kPer], h[kPer], top = -INFINITY, s = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int e = r * kLanes + lane;
      p[r] = on && e < experts ? float(*logits.at(t, e)) : -INFINITY;
      top = fmaxf(top, p[r]);
      h[r] = by_loss[r];
    }
    top = lanes_all<kLanes>(top, [](float a, float b) { return fmaxf(a, b); });
    if (top == -INFINITY) top = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      p[r] = expf(p[r] - top);
      s += p[r];
    }
    s = lanes_sum<kLanes>(s);
    const float scale = on ? 1.f / s : 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) p[r] = on ? p[r] * scale : 0.f;
    // The chosen experts, kLanes at a time: what their weights' gradients add.
    float chosen = 0.f, dot = 0.f;
    const auto choice = [&](int k, float& w, float& dw) {
      const int id = on && k < top_k ? ids_t[k] : -1;
      const bool taken = id >= 0 && id < experts;
      w = taken ? expf(float(*logits.at(t, id)) - top) : 0.f;
      dw = taken && dweights ? dweights[t * top_k + k] : 0.f;
      return taken ? id : -1;
    };
    if (normalize) {
      for (int k = 0; k < top_k; k += kLanes) {
        float w, dw;
        choice(k + lane, w, dw);
        chosen += w;
        dot += w * dw;
      }
      chosen = lanes_sum<kLanes>(chosen);
      dot = lanes_sum<kLanes>(dot) / chosen;
    }
    float extra[kPer];
#pragma unroll
    for (int r = 0; r < kPer; ++r) extra[r] = 0.f;
    for (int k0 = 0; k0 < top_k; k0 += kLanes) {
      float w, dw;
      const int id = choice(k0 + lane, w, dw);
      const float add = normalize ? w / chosen * (dw - dot) : dw;
      const int n = min(kLanes, top_k - k0);
      for (int j = 0; j < n; ++j) {
        const int id_j = __shfl(id, j, kLanes);
        const float add_j = __shfl(add, j, kLanes);
#pragma unroll
        for (int r = 0; r < kPer; ++r)
          if (id_j == r * kLanes + lane) extra[r] += add_j;
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      if (!normalize) h[r] += extra[r];
      sum += p[r] * h[r];
    }
    sum = lanes_sum<kLanes>(sum);
    if (!mine) continue;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int e = r * kLanes + lane;
      const float g = p[r] * (h[r] - sum) + (normalize ? extra[r] : 0.f);
      if (e < experts) *dlogits.at(t, e) = T(on ? g : 0.f);
    }
  }
}

// ----------------------------------------------------------------- host side

// Workgroups of the forward pass where the loss is wanted: what they leave is
// added up by one workgroup.
constexpr long long kRouteBlocks = 256;
long long route_blocks(long long tokens, int per_block, long long most) {
  const long long n = (tokens + per_block - 1) / per_block;
  return n < most ? n : most;
}

// Calls f(lanes, logits per lane).
template <typename F>
int with_lanes(int experts, F&& f) {
  const auto call = [&](auto lanes, auto per) { return f(lanes, per); };
  using std::integral_constant;
  if (experts <= 8) return call(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  if (experts <= 16) return call(integral_constant<int, 8>{}, integral_constant<int, 2>{});
  if (experts <= 32) return call(integral_constant<int, 8>{}, integral_constant<int, 4>{});
  if (experts <= 64) return call(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  if (experts <= 128) return call(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  if (experts <= 256) return call(integral_constant<int, 32>{}, integral_constant<int, 8>{});
  if (experts <= 512) return call(integral_constant<int, 64>{}, integral_constant<int, 8>{});
  return call(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

// What is wrong with logits and top_k, or null.
const char* route_error(const ps_rows* logits, int top_k) {
  if (logits->cols > kMostExperts) return "1 to 1024 experts";
  if (top_k < 1 || top_k > logits->cols) return "1 to as many slots a token as there are experts";
  if (logits->rows > (1LL << 30) / top_k) return "more than 2^30 slots";
  return nullptr;
}

Region slots(const void* p, const ps_rows* m, int top_k) {
  return region(p, size_t(m->rows) * size_t(top_k) * 4);
}

}  // namespace
}  // namespace ps

extern "C" {

size_t ps_expert_route_workspace_bytes(long long tokens, int experts) {
  if (tokens < 0 || tokens > (1LL << 30) || experts < 1 || experts > ps::kMostExperts) return 0;
  const size_t blocks = tokens < ps::kRouteBlocks ? size_t(tokens) : size_t(ps::kRouteBlocks);
  return (blocks ? blocks : 1) * (2 * size_t(experts) + 1) * 4;
}

int ps_expert_route(const ps_rows* logits, int top_k, int normalize, const unsigned char* mask,
                    int* ids, float* weights, int* counts, float* loss, void* workspace,
                    size_t workspace_bytes, ps_stream_t stream) {
  PS_CHECK_ROWS(logits);
  if (const char* error = ps::route_error(logits, top_k))
    return ps::fail(PS_ERR_INVALID, std::string("ps_expert_route: ") + error);
  PS_CHECK_ARG((ids && weights) || !logits->rows, "ps_expert_route: null ids or weights");
  PS_CHECK_ARG(!counts == !loss, "ps_expert_route: counts and loss come together");
  const int experts = int(logits->cols);
  const size_t need = ps_expert_route_workspace_bytes(logits->rows, experts);
  PS_CHECK_ARG(!loss || (workspace && ps::aligned16(workspace) && workspace_bytes >= need),
               "ps_expert_route: workspace too small or misaligned");
  PS_CHECK_ARG(ps::aligned4(ids) && ps::aligned4(weights) && ps::aligned4(counts) &&
                   ps::aligned4(loss),
               "ps_expert_route: misaligned output");
  const ps::Region in[] = {ps::region(logits), ps::region(mask, size_t(logits->rows))};
  const ps::Region to[] = {ps::slots(ids, logits, top_k), ps::slots(weights, logits, top_k),
                           ps::region(counts, (size_t(experts) + 1) * 4), ps::region(loss, 4),
                           ps::region(loss ? workspace : nullptr, need)};
  for (int i = 0; i < 5; ++i) {
    PS_CHECK_ARG(!ps::overlap(to[i], {in[0], in[1]}),
                 "ps_expert_route: an output or the workspace overlaps an input");
    for (int k = 0; k < i; ++k)
      PS_CHECK_ARG(!ps::overlap(to[i], to[k]), "ps_expert_route: outputs and workspace overlap");
  }
  const hipStream_t st = ps::to_hip(stream);
  ps::RouteParts parts{nullptr, nullptr};
  long long blocks = 0;
  const int rc = ps::with_dtype(logits->dtype, [&](auto t) {
    return ps::with_lanes(experts, [&](auto lanes, auto per) {
      using T = decltype(t);
      // Large workgroups where there is work for them: the join's parts are few.
      const bool large = logits->rows > ps::kRouteBlocks * (256 / lanes);
      const int threads = large ? 1024 : 256;
      blocks = ps::route_blocks(logits->rows, threads / lanes, loss ? ps::kRouteBlocks : 1 << 20);
      if (loss) {
        parts.sums = static_cast<float*>(workspace);
        parts.counts = reinterpret_cast<int*>(parts.sums + blocks * experts);
      }
      if (!blocks) return int(PS_OK);
      const auto run = [&](auto kernel) {
        kernel<<<uint32_t(blocks), threads, 0, st>>>(ps::mat<const T>(logits), experts, top_k,
                                                     normalize != 0, mask, ids, weights, parts);
      };
      if (large)
        run(ps::route_kernel<T, lanes, per, 1024>);
      else
        run(ps::route_kernel<T, lanes, per, 256>);
      PS_LAUNCHED();
      return int(PS_OK);
    });
  });
  if (rc != PS_OK || !loss) return rc;
  int groups = ps::kJoinThreads;
  while (ps::kJoinThreads / groups < experts) groups /= 2;
  ps::route_join_kernel<<<1, ps::kJoinThreads, 0, st>>>(parts, int(blocks), experts, groups, counts,
                                                        loss);
  PS_LAUNCHED();
  return PS_OK;
}

int ps_expert_route_grad(const ps_rows* logits, int top_k, int normalize, const int* ids,
                         const float* dweights, const int* counts, const float* dloss,
                         const ps_rows* dlogits, ps_stream_t stream) {
  PS_CHECK_ROWS(logits);
  PS_CHECK_ROWS(dlogits);
  if (const char* error = ps::route_error(logits, top_k))
    return ps::fail(PS_ERR_INVALID, std::string("ps_expert_route_grad: ") + error);
  PS_CHECK_ARG(logits->dtype == dlogits->dtype && logits->cols == dlogits->cols &&
                   logits->rows == dlogits->rows,
               "ps_expert_route_grad: logits and dlogits differ in type or shape");
  PS_CHECK_ARG(ids || !logits->rows, "ps_expert_route_grad: null ids");
  PS_CHECK_ARG(!dloss || counts, "ps_expert_route_grad: the loss's gradient needs the counts");
  PS_CHECK_ARG(ps::aligned4(ids) && ps::aligned4(dweights) && ps::aligned4(counts) &&
                   ps::aligned4(dloss),
               "ps_expert_route_grad: misaligned input");
  const int experts = int(logits->cols);
  PS_CHECK_ARG(!ps::overlap(ps::region(dlogits),
                            {ps::region(logits), ps::slots(ids, logits, top_k),
                             ps::slots(dweights, logits, top_k),
                             ps::region(counts, (size_t(experts) + 1) * 4), ps::region(dloss, 4)}),
               "ps_expert_route_grad: dlogits overlaps an input");
  if (!logits->rows) return PS_OK;
  return ps::with_dtype(logits->dtype, [&](auto t) {
    return ps::with_lanes(experts, [&](auto lanes, auto per) {
      using T = decltype(t);
      const long long blocks = ps::route_blocks(logits->rows, ps::kRouteGradThreads / lanes, 4096);
      ps::route_grad_kernel<T, lanes, per>
          <<<uint32_t(blocks), ps::kRouteGradThreads, 0, ps::to_hip(stream)>>>(
              ps::mat<const T>(logits), experts, top_k, normalize != 0, ids, dweights, counts,
              dloss, ps::mat<T>(dlogits));
      PS_LAUNCHED();
      return int(PS_OK);
    });
  });
}

}  // extern "C"
