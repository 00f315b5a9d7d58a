// The router of a mixture of experts: softmax of a token's logits, its top_k
// experts and their weights, how often each expert was chosen, the loss that
// asks for balance among them, and the gradient.
//
// kLanes threads share a token, each with kPer of its logits in registers, kWide
// neighbours at a time. The largest logits are found one after another, by keys
// that order as the logits do; equal ones go to the lowest expert. Finding them is
// most of the work, so the keys are cut to leave room for the expert beside them: a
// maximum then says which, and as no two are equal the next one is the largest of
// the differences from it that are below zero, two operations an element. What was
// cut off decides where two keys agree in what is left: FP16 and BF16 lose nothing,
// FP32 the last 8 bits for 128 experts (11 for 1,024), and a wave that meets two
// such logits in a row, or a NaN, takes the longer way, which finds the expert
// behind its key.
#include <algorithm>

#include "ps_rows.hpp"

namespace ps {
namespace {

constexpr int kMostExperts = 1024;

// Unsigned numbers that order as logits do, NaN above all; -0 and 0 are equal.
// Barred experts (-inf) and taken ones (0) are at kBarred or below.
constexpr uint32_t kBarred = 0x007fffffu;
__device__ __forceinline__ uint32_t key_of_number(float v) {
  const int b = __float_as_int(v + 0.f);
  return uint32_t(b ^ ((b >> 31) | int(0x80000000u)));
}
__device__ __forceinline__ uint32_t key_of(float v) { return v != v ? ~0u : key_of_number(v); }
// (~0 comes back as a NaN)
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// e^x for x <= 0 by the hardware's power of two: off by 2^-24 (2 + 1.3 |x|) relative,
// as the exponent is rounded. For sums, where that averages out: the terms far below
// the largest count little.
__device__ __forceinline__ float rough_exp(float x) {
  return __builtin_amdgcn_exp2f(x * 1.44269504f);
}
// The same with what the rounding lost of x, x - t ln(2), put back by the first terms
// of the series: off by 2^-24 (3 + 0.05 |x|). (The bounds are for x = -inf, whose
// difference is no number, and whose power is 0.) For what a call gives back: weights,
// of which a token has top_k, and the gradient. 65,536 x 128 FP32 top 8 13.5 -> 13.6 us,
// with it in the sums too 14.4; the gradient of 16,384 x 512 BF16 15.4 -> 15.7.
__device__ __forceinline__ float exp_of(float x) {
  const float t = x * 1.44269504f, r = __builtin_amdgcn_exp2f(t);
  const float lost = __builtin_amdgcn_fmed3f(fmaf(t, -0.693147182f, x), -1.f, 1.f);
  return fmaf(r, lost, r);
}
// 1 / s for s from 1 up, or NaN: the hardware's and one step of Newton's iteration
// (0, a padding token's in the gradient, gives NaN, and that token zeros anyway).
__device__ __forceinline__ float reciprocal(float s) {
  const float r = __builtin_amdgcn_rcpf(s);
  return fmaf(fmaf(-s, r, 1.f), r, r);
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

// Which experts a lane of a token has: element r is expert of(r), ascending in r.
template <int kLanes, int kPer, int kWide>
struct Share {
  static_assert(kPer % kWide == 0, "");
  int first;
  __device__ __forceinline__ explicit Share(int lane) : first(lane * kWide) {}
  __device__ __forceinline__ int of(int r) const {
    return first + r / kWide * kLanes * kWide + r % kWide;
  }
  // f(r, logit) of row t, absent where the expert does not exist.
  template <typename T, typename F>
  __device__ __forceinline__ void load(const Mat<const T>& m, long long t, int experts, bool on,
                                       float absent, F&& f) const {
    using V = typename PieceOf<T, kWide>::type;
    V v[kPer / kWide];
#pragma unroll
    for (int c = 0; c < kPer / kWide; ++c) {
      v[c] = V(T(absent));
      if (on && of(c * kWide) < experts) v[c] = *reinterpret_cast<const V*>(m.at(t, of(c * kWide)));
    }
#pragma unroll
    for (int r = 0; r < kPer; ++r) f(r, float(v[r / kWide][r % kWide]));
  }
};

// What the workgroups leave of the loss: sums of probabilities, and choices of
// every expert with the tokens that take part behind them.
struct RouteParts {
  float* sums;  // blocks x experts; null: no loss is wanted
  int* counts;  // blocks x (experts + 1)
  // their totals: experts sums, experts + 1 counts
  double* all_sums;
  int* all_counts;
  int* joined;  // workgroups of the join that are done; the first kernel clears it
};

// The counts and the loss from the totals of every expert, by a wave.
template <typename Sum, typename Count>
__device__ __forceinline__ void finish(int experts, Sum&& sum_of, Count&& count_of,
                                       int* __restrict__ counts, float* __restrict__ loss) {
  long long total = 0;
  double sum = 0;
  for (int e = lane_id(); e < experts; e += kWave) {
    const int c = count_of(e);
    counts[e] = c;
    total += c;
    sum += double(c) * double(sum_of(e));
  }
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) {
    total += __shfl_xor(total, d, kWave);
    sum += __shfl_xor(sum, d, kWave);
  }
  if (lane_id()) return;
  const int tokens = count_of(experts);
  counts[experts] = tokens;
  *loss = tokens ? float(sum * experts / (double(tokens) * double(total))) : 0.f;
}

// Bound by its instructions, some 750 for the eight tokens of a wave with 128
// experts, 35 of them for each expert that is found: 65,536 x 128 FP32, 38 MB, top 8
// 13.6 us and top 1 7.3; with the sums for the loss 17.1 and the join 6. Where FP32
// logits hold BF16 numbers, nearly every wave meets two that agree and takes the longer
// way: 19.6, with the loss and its join 29; all equal 19.7 and 28.
template <typename T, int kLanes, int kPer, int kWide, int kThreads>
__global__ __launch_bounds__(kThreads) void route_kernel(
    Mat<const T> logits, int experts, int top_k, bool normalize,
    const unsigned char* __restrict__ mask, int* __restrict__ ids, float* __restrict__ weights,
    RouteParts parts, int* __restrict__ counts, float* __restrict__ loss) {
  constexpr int kTokens = kThreads / kLanes;
  constexpr int kMost = kLanes * kPer, kBits = __builtin_ctz(kMost);
  __shared__ int chosen[kMost + 1];
  __shared__ float sums[kThreads / kWave][kMost];
  const int lane = threadIdx.x % kLanes;
  const Share<kLanes, kPer, kWide> share(lane);
  int tokens = 0;
  if (parts.sums) {
    for (int e = threadIdx.x; e <= experts; e += kThreads) chosen[e] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *parts.joined = 0;
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
    uint32_t key[kPer], most = 0;  // cut, with the expert
    float p[kPer], s = 0.f;
    share.load(logits, t, experts, on, -INFINITY, [&](int r, float v) {
      p[r] = v;
      const uint32_t whole = key_of_number(v);  // (a NaN shows in the sum below)
      most = max(most, whole);
      key[r] = (whole >> (kBits + 1) << kBits) + uint32_t(kMost - 1 - share.of(r));
    });
    most = lanes_max<kLanes>(most);
    // nothing to choose: no probabilities either
    float top = most > kBarred ? value_of(most) : 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      p[r] = rough_exp(p[r] - top);
      s += p[r];
    }
    s = lanes_sum<kLanes>(s);
    const bool nan = s != s;
    if (nan) top = s;
    const bool takes_part = most > kBarred || nan;
    const float scale = takes_part ? reciprocal(s) : 0.f;
    if (parts.sums) {
#pragma unroll
      for (int r = 0; r < kPer; ++r) acc[r] += p[r] * scale;
      tokens += lane == 0 && takes_part;
    }
    // Slot k's expert is found by all lanes and kept by lane k % kLanes.
    int my_id = -1;
    bool found = top_k <= kLanes;
    if (found) {
      uint32_t best = key[0];
#pragma unroll
      for (int r = 1; r < kPer; ++r) best = max(best, key[r]);
      best = lanes_max<kLanes>(best);
      uint32_t my_best = 0, down = 0;
      for (int k = 0; k < top_k; ++k) {
        if (lane == k) my_best = best;
        down = key[0] - best;  // from 2^31 up for those below it
#pragma unroll
        for (int r = 1; r < kPer; ++r) down = max(down, key[r] - best);
        down = lanes_max<kLanes>(down);
        best += down;
      }
      // Whether a slot's key agrees with the next one's, the last slot's with that of
      // the expert after it (if there is one).
      const bool any = lane < top_k && my_best >> kBits > kBarred >> (kBits + 1);
      if (any) my_id = kMost - 1 - int(my_best & (kMost - 1));
      uint32_t next = uint32_t(__shfl_down(int(my_best), 1, kLanes));
      if (lane == top_k - 1) next = int(down) < 0 ? best : 0;
      const bool equal = any && next >> kBits == my_best >> kBits;
      found = !__any((sizeof(T) == 4 && equal) || nan);
    }
    // A place left over weighs 0 whatever the others are divided by, NaN too.
    const auto times = [](float w, float by) { return w == 0.f ? 0.f : w * by; };
    float total = 0.f;
    const auto put = [&](int k, float& w) {  // slot k, this lane's
      w = my_id >= 0 ? exp_of(float(*logits.at(t, my_id)) - top) : 0.f;
      total += w;
      ids[t * top_k + k] = my_id;
      if (parts.sums && my_id >= 0) atomicAdd(&chosen[my_id], 1);
    };
    if (!found) {
      my_id = -1;
      share.load(logits, t, experts, on, -INFINITY, [&](int r, float v) { key[r] = key_of(v); });
    }
    for (int k0 = 0; k0 < top_k; k0 += kLanes) {
      const int n = min(kLanes, top_k - k0);
      for (int k = 0; !found && k < n; ++k) {
        uint32_t best = key[0], mine_at = ~0u;
#pragma unroll
        for (int r = 1; r < kPer; ++r) best = max(best, key[r]);
        best = lanes_max<kLanes>(best);
        // The first of this lane's that are the best one, and of all lanes'.
        bool past = best <= kBarred, is[kPer];
        if (lane == k) my_id = -1;
#pragma unroll
        for (int r = 0; r < kPer; ++r) {
          is[r] = !past && key[r] == best;
          past = past || is[r];
          if (is[r]) mine_at = uint32_t(share.of(r));
        }
        const uint32_t at = lanes_min<kLanes>(mine_at);
        const bool taken = mine_at == at;
#pragma unroll
        for (int r = 0; r < kPer; ++r)
          if (is[r] && taken) key[r] = 0;
        if (lane == k) my_id = int(at);
      }
      float w = 0.f;
      if (lane < n && mine) put(k0 + lane, w);
      if (top_k <= kLanes) {
        const float sum = lanes_sum<kLanes>(total);
        const float by = normalize ? (sum == 0.f ? 0.f : reciprocal(sum)) : scale;
        if (lane < n && mine) weights[t * top_k + lane] = times(w, by);
      } else if (lane < n && mine) {
        weights[t * top_k + k0 + lane] = normalize ? w : times(w, scale);
      }
    }
    if (top_k > kLanes && normalize) {
      total = lanes_sum<kLanes>(total);
      const float by = total == 0.f ? 0.f : reciprocal(total);
      if (mine)
        for (int k = lane; k < top_k; k += kLanes)
          weights[t * top_k + k] = times(weights[t * top_k + k], by);
    }
  }
  if (!parts.sums) return;
  // The tokens of a wave, then the waves in order.
#pragma unroll
  for (int r = 0; r < kPer; ++r) acc[r] = groups_sum<kLanes>(acc[r]);
  if (lane_id() < kLanes)
#pragma unroll
    for (int r = 0; r < kPer; ++r) sums[threadIdx.x / kWave][share.of(r)] = acc[r];
  tokens = lanes_all<kWave>(tokens, [](int a, int b) { return a + b; });
  if (lane_id() == 0) atomicAdd(&chosen[experts], tokens);
  __syncthreads();
  const auto sum_of = [&](int e) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) s += sums[w][e];
    return s;
  };
  if (gridDim.x == 1) {  // nothing to join
    if (threadIdx.x < kWave)
      finish(experts, sum_of, [&](int e) { return chosen[e]; }, counts, loss);
    return;
  }
  for (int e = threadIdx.x; e <= experts; e += kThreads) {
    parts.counts[size_t(blockIdx.x) * (experts + 1) + e] = chosen[e];
    if (e < experts) parts.sums[size_t(blockIdx.x) * experts + e] = sum_of(e);
  }
}

// The workgroups' parts added up: 32 columns a workgroup, the experts' sums first,
// the counts and the tokens behind them, 32 threads each with up to 16 parts under
// way at once. The last workgroup to be done has all totals and finishes.
constexpr int kJoinCols = 32, kJoinLanes = 32, kJoinAhead = 16;
__global__ __launch_bounds__(kJoinCols* kJoinLanes) void route_join_kernel(
    RouteParts parts, int part_count, int experts, int* __restrict__ counts,
    float* __restrict__ loss) {
  __shared__ double sums[kJoinLanes][kJoinCols];
  __shared__ bool last;
  const int lane = threadIdx.x / kJoinCols, i = threadIdx.x % kJoinCols;
  const int c = blockIdx.x * kJoinCols + i, all = 2 * experts + 1;
  double s = 0;  // (counts stay exact in it)
  for (int k0 = lane; c < all && k0 < part_count; k0 += kJoinLanes * kJoinAhead) {
    uint32_t v[kJoinAhead];
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j) {
      const size_t k = k0 + j * kJoinLanes;
      v[j] = 0;
      if (k < size_t(part_count))
        v[j] = c < experts ? __float_as_uint(parts.sums[k * experts + c])
                           : uint32_t(parts.counts[k * (experts + 1) + c - experts]);
    }
#pragma unroll
    for (int j = 0; j < kJoinAhead; ++j)
      s += c < experts ? double(__uint_as_float(v[j])) : double(v[j]);
  }
  sums[lane][i] = s;
  __syncthreads();
  if (lane == 0 && c < all) {
#pragma unroll
    for (int k = 1; k < kJoinLanes; ++k) s += sums[k][i];
    if (c < experts)
      parts.all_sums[c] = s;
    else
      parts.all_counts[c - experts] = int(s);
  }
  __syncthreads();
  if (threadIdx.x == 0)  // releases this workgroup's totals, acquires the others'
    last = __hip_atomic_fetch_add(parts.joined, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
           int(gridDim.x) - 1;
  __syncthreads();
  if (!last || threadIdx.x >= kWave) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  finish(experts, [&](int e) { return parts.all_sums[e]; },
         [&](int e) { return parts.all_counts[e]; }, counts, loss);
}
// Both for few parts, in one launch: all parts of a column under way at once.
constexpr int kFewParts = 16, kFewThreads = 1024;
__global__ __launch_bounds__(kFewThreads) void route_join_few_kernel(RouteParts parts,
                                                                     int part_count, int experts,
                                                                     int* __restrict__ counts,
                                                                     float* __restrict__ loss) {
  __shared__ double sums[kMostExperts];
  __shared__ int chosen[kMostExperts + 1];
  for (int e = threadIdx.x; e <= experts; e += kFewThreads) {
    float s_of[kFewParts];
    int c_of[kFewParts];
#pragma unroll
    for (int k = 0; k < kFewParts; ++k) {
      c_of[k] = k < part_count ? parts.counts[k * (experts + 1) + e] : 0;
      s_of[k] = k < part_count && e < experts ? parts.sums[k * experts + e] : 0.f;
    }
    int c = 0;
    double s = 0;
#pragma unroll
    for (int k = 0; k < kFewParts; ++k) {
      c += c_of[k];
      s += double(s_of[k]);
    }
    chosen[e] = c;
    if (e < experts) sums[e] = s;
  }
  __syncthreads();
  if (threadIdx.x < kWave)
    finish(experts, [&](int e) { return sums[e]; }, [&](int e) { return chosen[e]; }, counts, loss);
}
// Without tokens.
__global__ __launch_bounds__(kWave) void route_nothing_kernel(int experts, int* __restrict__ counts,
                                                              float* __restrict__ loss) {
  finish(experts, [](int) { return 0.0; }, [](int) { return 0; }, counts, loss);
}

// Softmax again from the logits, which takes less than reading probabilities would.
// 65,536 x 128 FP32, 71 MB, in 19.5 us, 3.65 TB/s, near what its instructions take;
// 300,007 x 17 FP16, whose 28 MB are moved at 1.5 to 1.7 TB/s, 16 one behind another,
// 17 to 19 alone.
constexpr int kRouteGradThreads = 256;
template <typename T, int kLanes, int kPer, int kWide>
__global__ __launch_bounds__(kRouteGradThreads) void route_grad_kernel(
    Mat<const T> logits, int experts, int top_k, bool normalize, const int* __restrict__ ids,
    const float* __restrict__ dweights, const int* __restrict__ counts,
    const float* __restrict__ dloss, Mat<T> dlogits) {
  constexpr int kTokens = kRouteGradThreads / kLanes;
  // What the choices add to a token's logits, put in place by the lanes that know it
  // and read by those that have the logits, all in one wave.
  __shared__ float rows[kTokens][kLanes * kPer];
  float* const row = rows[threadIdx.x / kLanes];
  const int lane = threadIdx.x % kLanes;
  const Share<kLanes, kPer, kWide> share(lane);
#pragma unroll
  for (int r = 0; r < kPer; ++r) row[share.of(r)] = 0.f;
  wave_lds_sync();
  // The loss's gradient by an expert's probability.
  float by_loss[kPer];
#pragma unroll
  for (int r = 0; r < kPer; ++r) by_loss[r] = 0.f;
  if (dloss) {
    float total = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      const int e = share.of(r);
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
    struct Choice {
      int id;
      float logit, dw;
    };
    // Slot k's; loads that are in range whatever k and the id are need no branches.
    const long long tt = min(t, logits.rows - 1);
    const auto choice = [&](int k) {
      const long long at = tt * top_k + min(k, top_k - 1);
      const int id = ids[at];
      const bool taken = mine && k < top_k && id >= 0 && id < experts;
      Choice c{-1, 0.f, 0.f};
      const float logit = float(*logits.at(tt, taken ? id : 0));
      const float dw = dweights ? dweights[at] : 0.f;
      if (taken) c = {id, logit, dw};
      return c;
    };
    // All loads are under way before the first is waited for, but the chosen logits'.
    const int id_0 = ids[tt * top_k];
    float p[kPer], h[kPer], top = -INFINITY, s = 0.f;
    share.load(logits, tt, experts, true, -INFINITY, [&](int r, float v) { p[r] = v; });
    const Choice first = choice(lane);
    const bool on = mine && id_0 >= 0;
#pragma unroll
    for (int r = 0; r < kPer; ++r) top = fmaxf(top, p[r]);
    top = lanes_all<kLanes>(top, [](float a, float b) { return fmaxf(a, b); });
    if (top == -INFINITY) top = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      p[r] = exp_of(p[r] - top);
      s += p[r];
    }
    const float scale = reciprocal(lanes_sum<kLanes>(s));
    // What the chosen experts' weights' gradients add, kLanes of them at a time: the
    // first ones have been loaded.
    float chosen = 0.f, dot = 0.f;
    if (normalize) {
      Choice c = first;
      for (int k = 0; k < top_k; k += kLanes) {
        if (k) c = choice(k + lane);
        const float w = c.id >= 0 ? exp_of(c.logit - top) : 0.f;
        chosen += w;
        dot += w * c.dw;
      }
      chosen = reciprocal(lanes_sum<kLanes>(chosen));
      dot = lanes_sum<kLanes>(dot) * chosen;
    }
    Choice c = first;
    for (int k0 = 0; k0 < top_k; k0 += kLanes) {
      if (k0) c = choice(k0 + lane);
      if (c.id < 0) continue;
      atomicAdd(&row[c.id], normalize ? exp_of(c.logit - top) * chosen * (c.dw - dot) : c.dw);
    }
    wave_lds_sync();
    float extra[kPer], sum = 0.f;
#pragma unroll
    for (int r = 0; r < kPer; ++r) {
      extra[r] = row[share.of(r)];
      p[r] *= scale;
      h[r] = by_loss[r] + (normalize ? 0.f : extra[r]);
      sum += p[r] * h[r];
    }
    wave_lds_sync();
#pragma unroll
    for (int r = 0; r < kPer; ++r) row[share.of(r)] = 0.f;
    wave_lds_sync();
    sum = lanes_sum<kLanes>(sum);
    if (!mine) continue;
#pragma unroll
    for (int r = 0; r < kPer; r += kWide) {
      if (share.of(r) >= experts) continue;
      Floats<kWide> g;
#pragma unroll
      for (int j = 0; j < kWide; ++j) {
        const float d = p[r + j] * (h[r + j] - sum);
        g[j] = on ? normalize ? d + extra[r + j] : d : 0.f;
      }
      store_piece<kWide>(dlogits.at(t, share.of(r)), g);
    }
  }
}

// ----------------------------------------------------------------- host side

// Workgroups of the forward pass where the loss is wanted, what they leave is added
// up: at most kRouteThreads threads in all, half of what the device holds at once
// (65,536 x 128 top 8: 24.6 us, 25.8 with all of it), and no more workgroups than
// those of 512 threads.
constexpr long long kRouteThreads = 1 << 18, kRouteBlocks = kRouteThreads / 512;
long long route_blocks(long long tokens, int per_block, long long most) {
  const long long n = (tokens + per_block - 1) / per_block;
  return n < most ? n : most;
}

// Calls f(lanes, logits per lane, logits at a time). `many` (kFind: where experts
// are found): half as many lanes, which is less work in all, as a lane's part of
// finding the next expert hardly grows, and longer for a token alone (65,536 x 128
// top 8 18 -> 16 us, 16,384 x 512 20 -> 16, 300,007 x 17 FP16 20 -> 14; 512 x 64 4.3 ->
// 5.9; the gradient, which finds none, 19.3 -> 20.2 and 16.6 -> 22.5). Not for 64
// experts, 9.2 -> 10.1, nor for more slots than lanes, which the shorter way does
// not take.
template <bool kFind, typename F>
int with_lanes(int experts, int top_k, bool many, F&& f) {
  const auto call = [&](auto lanes, auto per) {
    constexpr int kWide = per < 4 ? per : 4;
    if (experts % kWide == 0) return f(lanes, per, std::integral_constant<int, kWide>{});
    return f(lanes, per, std::integral_constant<int, 1>{});
  };
  using std::integral_constant;
  if constexpr (kFind) {
    const int half = experts <= 32 ? 4 : experts <= 128 ? 8 : experts <= 256 ? 16 : 32;
    if (many && top_k <= half && experts > 8 && experts <= 512 && (experts <= 32 || experts > 64)) {
      if (experts <= 16) return call(integral_constant<int, 4>{}, integral_constant<int, 4>{});
      if (experts <= 32) return call(integral_constant<int, 4>{}, integral_constant<int, 8>{});
      const auto per = integral_constant<int, 16>{};
      if (experts <= 128) return call(integral_constant<int, 8>{}, per);
      if (experts <= 256) return call(integral_constant<int, 16>{}, per);
      return call(integral_constant<int, 32>{}, per);
    }
  }
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
  // the totals and the join's counter, then the workgroups' parts
  return size_t(experts) * 8 + (size_t(experts) + 2) * 4 + blocks * (2 * size_t(experts) + 1) * 4;
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
  if (!logits->rows) {
    if (!loss) return PS_OK;
    ps::route_nothing_kernel<<<1, ps::kWave, 0, st>>>(experts, counts, loss);
    PS_LAUNCHED();
    return PS_OK;
  }
  ps::RouteParts parts{};
  long long blocks = 0;
  const int rc = ps::with_dtype(logits->dtype, [&](auto t) {
    const bool many = logits->rows >= 8192;
    return ps::with_lanes<true>(experts, top_k, many, [&](auto lanes, auto per, auto wide) {
      using T = decltype(t);
      // Large workgroups where there is work for them, so that the parts are few, and
      // shared memory for a sum of each expert and wave.
      constexpr int kLarge = lanes * per <= 512 ? 1024 : 512;
      // One alone for what it takes in a turn: nothing is left to join (128 x 64 7.1 ->
      // 5.7 us; with two turns 8.0 -> 8.6).
      const bool alone = loss && logits->rows > 256 / lanes && logits->rows <= kLarge / lanes;
      const bool large = alone || logits->rows > 256 * (256 / lanes);
      const int threads = large ? kLarge : 256;
      const long long most =
          loss ? std::min(ps::kRouteThreads / threads, ps::kRouteBlocks) : 1LL << 20;
      blocks = ps::route_blocks(logits->rows, threads / lanes, most);
      if (loss) {
        parts.all_sums = static_cast<double*>(workspace);
        parts.all_counts = reinterpret_cast<int*>(parts.all_sums + experts);
        parts.joined = parts.all_counts + experts + 1;
        parts.counts = parts.joined + 1;
        parts.sums = reinterpret_cast<float*>(parts.counts + blocks * (experts + 1));
      }
      const auto run = [&](auto kernel) {
        kernel<<<uint32_t(blocks), threads, 0, st>>>(ps::mat<const T>(logits), experts, top_k,
                                                     normalize != 0, mask, ids, weights, parts,
                                                     counts, loss);
      };
      if (large)
        run(ps::route_kernel<T, lanes, per, wide, kLarge>);
      else
        run(ps::route_kernel<T, lanes, per, wide, 256>);
      PS_LAUNCHED();
      return int(PS_OK);
    });
  });
  if (rc != PS_OK || !loss || blocks == 1) return rc;
  if (blocks <= ps::kFewParts) {
    ps::route_join_few_kernel<<<1, ps::kFewThreads, 0, st>>>(parts, int(blocks), experts, counts,
                                                             loss);
    PS_LAUNCHED();
    return PS_OK;
  }
  const uint32_t columns = 2 * uint32_t(experts) + 1;
  ps::route_join_kernel<<<(columns + ps::kJoinCols - 1) / ps::kJoinCols,
                          ps::kJoinCols * ps::kJoinLanes, 0, st>>>(parts, int(blocks), experts,
                                                                   counts, loss);
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
    return ps::with_lanes<false>(experts, top_k, false, [&](auto lanes, auto per, auto wide) {
      using T = decltype(t);
      const long long blocks = ps::route_blocks(logits->rows, ps::kRouteGradThreads / lanes, 4096);
      ps::route_grad_kernel<T, lanes, per, wide>
          <<<uint32_t(blocks), ps::kRouteGradThreads, 0, ps::to_hip(stream)>>>(
              ps::mat<const T>(logits), experts, top_k, normalize != 0, ids, dweights, counts,
              dloss, ps::mat<T>(dlogits));
      PS_LAUNCHED();
      return int(PS_OK);
    });
  });
}

}  // extern "C"
