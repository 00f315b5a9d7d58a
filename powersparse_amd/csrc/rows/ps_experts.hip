// Tokens sorted by expert and back: the sort of the slots, the copies into
// expert order, the weighted sums back, and their gradients.
//
// With P the slots x tokens matrix that has a one where a slot is a token's,
// the dispatch is xs = P x, the combination y = P^T diag(w) ys, and their
// gradients dx = P^T dxs, dys = diag(w) P dy and dw = the dots of dy's and ys's
// rows at P's nonzeros: products by a sparse matrix whose k entries per token
// are the positions the sort gives. They are walked token by token, so a token's
// row is read or written once and the k rows of its slots are each touched once.
//
// All are bound by memory traffic: a slot's row is read or written in whole
// 16-byte pieces, and the positions (4 bytes a slot) hide behind it.
#include "ps_id_sort.hpp"
#include "ps_rows.hpp"

namespace ps {
namespace {

struct ExpertSink {
  static constexpr bool kStarts = true;
  int *order, *position, *offsets;
  uint32_t experts;
  __device__ __forceinline__ void put(uint32_t pos, uint32_t key, uint32_t slot) const {
    order[pos] = int(slot);
    position[slot] = key < experts ? int(pos) : -1;
  }
  __device__ __forceinline__ void bin_start(uint32_t bin, uint32_t start) const {
    offsets[bin] = int(start);
  }
};

// xs[position] = x, one piece of a token a thread, which writes it to every
// slot: x is read once. 16,384 tokens x 8 x 4,096 BF16: 1.21 GB in 228 us, 5.3
// TB/s.
template <typename T, int N, bool kStream>
__global__ __launch_bounds__(kRowThreads) void dispatch_kernel(Mat<const T> x,
                                                               const int* __restrict__ position,
                                                               int top_k, Mat<T> xs, Pieces p,
                                                               Items items_of) {
  const auto [first, items] = items_of.of_block(kRowThreads);
  if (threadIdx.x >= items) return;
  const Item it = ItemBase(first, p).at(threadIdx.x, p);
  const int c = p.begin(it.piece);
  using V = typename PieceOf<T, N>::type;
  const V v = *reinterpret_cast<const V*>(x.at(it.row, c));
  const int* pos = position + it.row * top_k;
  for (int k = 0; k < top_k; ++k) {
    const int q = pos[k];
    if (q < 0 || q >= xs.rows) continue;
    V* const to = reinterpret_cast<V*>(xs.at(q, c));
    if constexpr (kStream)
      __builtin_nontemporal_store(v, to);
    else
      *to = v;
  }
}

// Rows of a token's slots under way at once. Combination, with one and with four,
// us: 4 x 8 x 2,048 BF16 4.2 and 3.9, 256 x 8 x 4,096 4.8 and 4.5, 16,384 x 8 x
// 4,096 222.6 and 220.3; places left empty cost: 16,384 x 2 x 333 FP32 13.3 and
// 13.9, 30,011 x 3 x 333 28.3 and 28.9.
constexpr int kSlotsAhead = 4;

// y = sum of weighted slots, one piece of a token a thread, in the order of k.
// The same sizes: 1.22 GB in 222 us, 5.5 TB/s.
template <typename T, int N, bool kStream>
__global__ __launch_bounds__(kRowThreads) void combine_kernel(Mat<const T> ys,
                                                              const int* __restrict__ position,
                                                              const float* __restrict__ weights,
                                                              int top_k, Mat<T> y, Pieces p,
                                                              Items items_of) {
  const auto [first, items] = items_of.of_block(kRowThreads);
  if (threadIdx.x >= items) return;
  const Item it = ItemBase(first, p).at(threadIdx.x, p);
  const int c = p.begin(it.piece);
  const long long s = it.row * top_k;
  using V = typename PieceOf<T, N>::type;
  Floats<N> acc = 0.f;
  for (int k0 = 0; k0 < top_k; k0 += kSlotsAhead) {
    float w[kSlotsAhead];
    V v[kSlotsAhead];
#pragma unroll
    for (int j = 0; j < kSlotsAhead; ++j) {
      const int k = min(k0 + j, top_k - 1);
      const int q = position[s + k];
      const bool on = k0 + j < top_k && q >= 0 && q < ys.rows;
      w[j] = on && weights ? weights[s + k] : 1.f;
      v[j] = on ? *reinterpret_cast<const V*>(ys.at(q, c)) : V(T(0.f));
    }
#pragma unroll
    for (int j = 0; j < kSlotsAhead; ++j) acc += w[j] * __builtin_convertvector(v[j], Floats<N>);
  }
  store_piece<N, kStream>(y.at(it.row, c), acc);
}

// dys and the dots in one pass over dy and ys: kLanes threads a token, the
// pieces of its row among them, and one dot a slot summed over them. 16,384
// tokens x 4 x 2,048 BF16: 0.61 GB in 117 us, 5.2 TB/s.
template <typename T, int N, int kLanes, bool kStream>
__global__ __launch_bounds__(kRowThreads) void combine_grad_kernel(
    Mat<const T> dy, Mat<const T> ys, const int* __restrict__ position,
    const float* __restrict__ weights, int top_k, Mat<T> dys, float* __restrict__ dweights,
    Pieces p, Items tokens) {
  constexpr int kTokens = kRowThreads / kLanes;
  __shared__ float part[kLanes > kWave ? kSlotsAhead : 1][kRowThreads / kWave];
  const auto [first, count] = tokens.of_block(kTokens);
  const uint32_t mine = threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
  // threads without a token go along: the sums below take every lane
  const bool on = mine < count;
  const long long t = (long long)first + (on ? mine : 0);
  const int pieces = int(p.per_row.d);
  using V = typename PieceOf<T, N>::type;
  for (int k0 = 0; k0 < top_k; k0 += kSlotsAhead) {
    int q[kSlotsAhead];
    float w[kSlotsAhead], dot[kSlotsAhead];
#pragma unroll
    for (int j = 0; j < kSlotsAhead; ++j) {
      const long long s = t * top_k + min(k0 + j, top_k - 1);
      q[j] = position[s];
      w[j] = weights[s];
      if (!on || k0 + j >= top_k || q[j] < 0 || q[j] >= ys.rows) q[j] = -1;
      dot[j] = 0.f;
    }
    for (int i = lane; i < pieces; i += kLanes) {
      const int c = p.begin(i);
      const int seen = i * N - c;  // elements that the piece before has added
      const Floats<N> g = load_piece<N>(dy.at(t, c));
      V v[kSlotsAhead];
#pragma unroll
      for (int j = 0; j < kSlotsAhead; ++j)
        v[j] = q[j] >= 0 ? *reinterpret_cast<const V*>(ys.at(q[j], c)) : V(T(0.f));
#pragma unroll
      for (int j = 0; j < kSlotsAhead; ++j) {
        if (q[j] < 0) continue;
        const Floats<N> f = __builtin_convertvector(v[j], Floats<N>);
#pragma unroll
        for (int e = 0; e < N; ++e) dot[j] += e >= seen ? g[e] * f[e] : 0.f;
        store_piece<N, kStream>(dys.at(q[j], c), w[j] * g);
      }
    }
#pragma unroll
    for (int j = 0; j < kSlotsAhead; ++j)
#pragma unroll
      for (int d = (kLanes < kWave ? kLanes : kWave) / 2; d; d >>= 1)
        dot[j] += __shfl_xor(dot[j], d, kWave);
    if constexpr (kLanes > kWave) {
      __syncthreads();
      if (lane_id() == 0)
#pragma unroll
        for (int j = 0; j < kSlotsAhead; ++j) part[j][threadIdx.x / kWave] = dot[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kSlotsAhead; ++j) {
        dot[j] = 0.f;
#pragma unroll
        for (int u = 0; u < kRowThreads / kWave; ++u) dot[j] += part[j][u];
      }
    }
    if (on && lane == 0)
#pragma unroll
      for (int j = 0; j < kSlotsAhead; ++j)
        if (k0 + j < top_k) dweights[t * top_k + k0 + j] = dot[j];
  }
}

// The sort's workspace: the groups' counts, then the table.
size_t sort_bytes(const IdCut& cut, int experts) {
  return id_sort_group_bytes(cut, experts + 1) + id_sort_table_bytes(cut, experts + 1);
}

// What a value of four bytes for each slot of the tokens of m takes.
Region slots(const void* p, const ps_rows* m, int top_k) {
  return region(p, size_t(m->rows) * size_t(top_k) * 4);
}

// Calls f(lanes) with the threads a token's row gets: its pieces, one each up
// to 64, or a workgroup from 256 pieces on. Gradients of the combination, us:
// 16,384 x 4 x 2,048 BF16 134 with 64 lanes, 119 with 256; 256 x 8 x 4,096 18.3
// and 10.1; but 32,768 x 4 x 1,024 123 and 150, 65,536 x 4 x 333 FP16 74 and
// 187. Fewer lanes than pieces cost as well (333: 89 with 32), and so do idle
// ones (65,536 x 4 x 64 BF16: 14.3 with 8, 17.5 with 16, 54 with 64).
template <typename F>
int with_lanes(const Pieces& p, F&& f) {
  const uint32_t pieces = p.per_row.d;
  if (pieces >= 256) return f(std::integral_constant<int, 256>{});
  if (pieces > 32) return f(std::integral_constant<int, 64>{});
  if (pieces > 16) return f(std::integral_constant<int, 32>{});
  if (pieces > 8) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 8>{});
}

}  // namespace
}  // namespace ps

extern "C" {

size_t ps_expert_sort_workspace_bytes(long long slots, int experts) {
  if (slots < 0 || slots > (1LL << 30) || experts < 1 || experts > 1024) return 0;
  return ps::sort_bytes(ps::id_cut_most(slots), experts);
}

int ps_expert_sort(const ps_ids* ids, int experts, int* order, int* position, int* offsets,
                   void* workspace, size_t workspace_bytes, ps_stream_t stream) {
  PS_CHECK_IDS(ids);
  PS_CHECK_ARG(experts >= 1 && experts <= 1024, "ps_expert_sort: 1 to 1024 experts");
  PS_CHECK_ARG(offsets && (!ids->count || (order && position)), "ps_expert_sort: null output");
  PS_CHECK_ARG(workspace && ps::aligned16(workspace) &&
                   workspace_bytes >= ps_expert_sort_workspace_bytes(ids->count, experts),
               "ps_expert_sort: workspace too small or misaligned");
  const size_t slots = size_t(ids->count) * sizeof(int);
  const ps::Region in = ps::region(ids);
  const ps::Region to[] = {
      ps::region(order, slots), ps::region(position, slots),
      ps::region(offsets, (size_t(experts) + 1) * sizeof(int)),
      ps::region(workspace, ps::sort_bytes(ps::id_cut(ids->count), experts))};
  PS_CHECK_ARG(!ps::overlap(to[0], {in, to[1], to[2], to[3]}) &&
                   !ps::overlap(to[1], {in, to[2], to[3]}) && !ps::overlap(to[2], {in, to[3]}) &&
                   !ps::overlap(to[3], in),
               "ps_expert_sort: ids, outputs and workspace overlap");
  const ps::ExpertSink sink{order, position, offsets, uint32_t(experts)};
  ps::Digit dg{0, 1, experts + 1};
  while ((1 << dg.bits) < dg.bins) ++dg.bits;
  const uint32_t n = uint32_t(ids->count);
  const hipStream_t st = ps::to_hip(stream);
  const auto sort = [&](const auto& src) {
    if (n <= ps::kIdTile) return ps::id_sort_tile(src, sink, n, dg, 1, ps::ClearOnTheWay{}, st);
    // the groups' counts, then the table
    const size_t groups = ps::id_sort_group_bytes(ps::id_cut(n), dg.bins);
    if (groups) {
      const int rc = ps::id_clear({static_cast<uint4*>(workspace), groups / 16}, st);
      if (rc != PS_OK) return rc;
    }
    return ps::id_sort_pass(src, sink, n, dg, static_cast<char*>(workspace) + groups, workspace,
                            ps::ClearOnTheWay{}, st);
  };
  if (ids->type == PS_I64)
    return sort(ps::IdSource<long long>{static_cast<const long long*>(ids->data), experts, -1});
  return sort(ps::IdSource<int>{static_cast<const int*>(ids->data), experts, -1});
}

int ps_expert_dispatch(const ps_rows* x, const int* position, int top_k, const ps_rows* xs,
                       ps_stream_t stream) {
  PS_CHECK_ROWS(x);
  PS_CHECK_ROWS(xs);
  PS_CHECK_ARG(x->dtype == xs->dtype && x->cols == xs->cols,
               "ps_expert_dispatch: x and xs differ in type or width");
  PS_CHECK_ARG(top_k >= 1 && top_k <= 1024, "ps_expert_dispatch: 1 to 1024 slots per token");
  PS_CHECK_ARG(position || !x->rows, "ps_expert_dispatch: null positions");
  PS_CHECK_ARG(!ps::overlap(ps::region(xs), {ps::region(x), ps::slots(position, x, top_k)}),
               "ps_expert_dispatch: xs overlaps an input");
  if (!x->rows || !xs->rows) return PS_OK;
  return ps::with_dtype(x->dtype, [&](auto t) {
    using T = decltype(t);
    return ps::with_width<sizeof(T)>(x->cols, [&](auto n) {
      const ps::Pieces p(x->cols, n);
      const unsigned long long items = (unsigned long long)x->rows * p.per_row.d;
      return ps::with_flag(ps::streamed(xs, x->rows * top_k), [&](auto stream_out) {
        return ps::launch_items(items, ps::kRowThreads, [&](uint32_t blocks, ps::Items part) {
          ps::dispatch_kernel<T, n, stream_out>
              <<<blocks, ps::kRowThreads, 0, ps::to_hip(stream)>>>(
                  ps::mat<const T>(x), position, top_k, ps::mat<T>(xs), p, part);
        });
      });
    });
  });
}

int ps_expert_combine(const ps_rows* ys, const int* position, const float* weights, int top_k,
                      const ps_rows* y, ps_stream_t stream) {
  PS_CHECK_ROWS(ys);
  PS_CHECK_ROWS(y);
  PS_CHECK_ARG(ys->dtype == y->dtype && ys->cols == y->cols,
               "ps_expert_combine: ys and y differ in type or width");
  PS_CHECK_ARG(top_k >= 1 && top_k <= 1024, "ps_expert_combine: 1 to 1024 slots per token");
  PS_CHECK_ARG(position || !y->rows, "ps_expert_combine: null positions");
  PS_CHECK_ARG(!ps::overlap(ps::region(y), {ps::region(ys), ps::slots(position, y, top_k),
                                            ps::slots(weights, y, top_k)}),
               "ps_expert_combine: y overlaps an input");
  if (!y->rows) return PS_OK;
  return ps::with_dtype(y->dtype, [&](auto t) {
    using T = decltype(t);
    return ps::with_width<sizeof(T)>(y->cols, [&](auto n) {
      const ps::Pieces p(y->cols, n);
      const unsigned long long items = (unsigned long long)y->rows * p.per_row.d;
      return ps::with_flag(ps::streamed(y, y->rows), [&](auto stream_out) {
        return ps::launch_items(items, ps::kRowThreads, [&](uint32_t blocks, ps::Items part) {
          ps::combine_kernel<T, n, stream_out>
              <<<blocks, ps::kRowThreads, 0, ps::to_hip(stream)>>>(
                  ps::mat<const T>(ys), position, weights, top_k, ps::mat<T>(y), p, part);
        });
      });
    });
  });
}

int ps_expert_combine_grad(const ps_rows* dy, const ps_rows* ys, const int* position,
                           const float* weights, int top_k, const ps_rows* dys, float* dweights,
                           ps_stream_t stream) {
  PS_CHECK_ROWS(dy);
  PS_CHECK_ROWS(ys);
  PS_CHECK_ROWS(dys);
  PS_CHECK_ARG(dy->dtype == ys->dtype && dy->dtype == dys->dtype && dy->cols == ys->cols &&
                   dy->cols == dys->cols && ys->rows == dys->rows,
               "ps_expert_combine_grad: dy, ys and dys differ in type, width or rows");
  PS_CHECK_ARG(top_k >= 1 && top_k <= 1024, "ps_expert_combine_grad: 1 to 1024 slots per token");
  PS_CHECK_ARG((position && weights && dweights) || !dy->rows,
               "ps_expert_combine_grad: null positions or weights");
  const ps::Region in[] = {ps::region(dy), ps::region(ys), ps::slots(position, dy, top_k),
                           ps::slots(weights, dy, top_k)};
  PS_CHECK_ARG(!ps::overlap(ps::region(dys), {in[0], in[1], in[2], in[3]}),
               "ps_expert_combine_grad: dys overlaps an input");
  PS_CHECK_ARG(!ps::overlap(ps::slots(dweights, dy, top_k),
                            {in[0], in[1], in[2], in[3], ps::region(dys)}),
               "ps_expert_combine_grad: dweights overlaps another argument");
  if (!dy->rows) return PS_OK;
  return ps::with_dtype(dy->dtype, [&](auto t) {
    using T = decltype(t);
    return ps::with_width<sizeof(T)>(dy->cols, [&](auto n) {
      const ps::Pieces p(dy->cols, n);
      return ps::with_lanes(p, [&](auto lanes) {
        return ps::with_flag(ps::streamed(dys, dy->rows * top_k), [&](auto stream_out) {
          return ps::launch_items(
              dy->rows, ps::kRowThreads / lanes, [&](uint32_t blocks, ps::Items part) {
                ps::combine_grad_kernel<T, n, lanes, stream_out>
                    <<<blocks, ps::kRowThreads, 0, ps::to_hip(stream)>>>(
                        ps::mat<const T>(dy), ps::mat<const T>(ys), position, weights, top_k,
                        ps::mat<T>(dys), dweights, p, part);
              });
        });
      });
    });
  });
}

}  // extern "C"
