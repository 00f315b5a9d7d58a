// Embedding lookup with scaling, and its gradient by sorted ids.
//
// The lookup is a product by the matrix with a one per row at the id's column:
// a gather of rows, bound by the rows read and written.
//
// The gradient is the transposed product. Atomic additions would make its bits
// depend on their order and serialise on popular rows, so the ids are sorted
// (stably, ps_id_sort.hpp) and the gradient rows are sums over runs of equal
// ids. The sorted list is cut into chunks of kChunk entries, each one thread's
// per piece of the width:
//  - a run belongs to the chunk it starts in when it ends before the next
//    chunk's end: one thread adds all of it and writes the row;
//  - a longer run is cut at the chunks' borders, every part is kept as a row of
//    32-bit partial sums, and a second launch adds the parts in order.
// So partial sums cost traffic only for runs of more than kChunk entries, and
// no row waits for one thread to walk a popular id's whole run. Rows without
// ids are cleared by the same launch, from flags the sort sets.
#include <algorithm>

#include "ps_id_sort.hpp"
#include "ps_rows.hpp"

namespace ps {
namespace {

template <typename T, typename O, typename I, int N>
__global__ __launch_bounds__(kRowThreads) void lookup_kernel(Mat<const T> table,
                                                             const I* __restrict__ ids,
                                                             float scale, Mat<O> out, Pieces p,
                                                             Items items_of) {
  const auto [first, items] = items_of.of_block(kRowThreads);
  if (threadIdx.x >= items) return;
  const Item it = ItemBase(first, p).at(threadIdx.x, p);
  const int c = p.begin(it.piece);
  const long long id = ids[it.row];
  Floats<N> v = 0.f;
  if (id >= 0 && id < table.rows) v = scale * load_piece<N>(table.at(id, c));
  store_piece<N>(out.at(it.row, c), v);
}

constexpr uint32_t kChunk = 16;

struct FlagSink {
  static constexpr bool kStarts = false;
  uint32_t *keys, *values;
  uint8_t* flags;  // flags[row] = 1 for rows with ids (null: not wanted)
  uint32_t rows;
  __device__ __forceinline__ void put(uint32_t pos, uint32_t key, uint32_t value) const {
    keys[pos] = key;
    values[pos] = value;
    if (flags && key < rows) flags[key] = 1;
  }
  __device__ __forceinline__ void bin_start(uint32_t, uint32_t) const {}
};

// The sorted ids (keys; `rows` = takes no part) and where their rows of
// grad_out are, n of them, and the partial sums: chunk q's first run's part in
// row 2q, its last run's in row 2q + 1, ld floats apart.
struct Runs {
  const uint32_t *keys, *at;
  uint32_t n, rows;
  float* partial;
  long long ld;
  uint32_t *long_count, *long_list;  // the chunks in which long runs start
};

template <typename G, int N>
__device__ __forceinline__ void write_grad(const Mat<G>& grad, uint32_t row, int c, int seen,
                                           const Floats<N>& sum, float scale, bool accumulate) {
  G* to = grad.at(row, c);
  if (!accumulate) {
    store_piece<N>(to, scale * sum);
  } else if (seen <= 0) {
    store_piece<N>(to, load_piece<N>(to) + scale * sum);
  } else {
    // the elements that the piece before holds too are that piece's
    for (int e = seen; e < N; ++e) to[e] = G(float(to[e]) + scale * sum[e]);
  }
}

template <typename T, typename G, int N>
__device__ void sum_runs(const Runs& r, const Mat<const T>& dy, const Mat<G>& grad, float scale,
                         bool accumulate, uint32_t chunk, int piece, const Pieces& p) {
  const int c = p.begin(piece);
  const int seen = piece * N - c;
  const uint32_t b = chunk * kChunk, e = min(b + kChunk, r.n);
  uint32_t i = b;
  if (b > 0 && r.keys[b - 1] == r.keys[b]) {  // a run that starts in a chunk before
    const uint32_t k = r.keys[b];
    const bool is_long = k < r.rows && ((b > kChunk && r.keys[b - kChunk - 1] == k) ||
                                        (b + kChunk < r.n && r.keys[b + kChunk] == k));
    Floats<N> sum = 0.f;
    for (; i < e && r.keys[i] == k; ++i)
      if (is_long) sum += load_piece<N>(dy.at(r.at[i], c));
    if (is_long) store_piece<N>(r.partial + (2ull * chunk) * r.ld + c, sum);
  }
  while (i < e) {
    const uint32_t k = r.keys[i];
    if (k >= r.rows) break;  // only ids that take no part follow
    // the run ends with the chunk, or within the next one, or is long
    const uint32_t next = min(e + kChunk, r.n);
    Floats<N> sum = 0.f;
    for (; i < e && r.keys[i] == k; ++i) sum += load_piece<N>(dy.at(r.at[i], c));
    if (i == e && e < r.n && r.keys[e] == k) {
      if (next < r.n && r.keys[next] == k) {
        store_piece<N>(r.partial + (2ull * chunk + 1) * r.ld + c, sum);
        if (piece == 0) r.long_list[atomicAdd(r.long_count, 1u)] = chunk;
        break;
      }
      for (; i < next && r.keys[i] == k; ++i) sum += load_piece<N>(dy.at(r.at[i], c));
    }
    write_grad<G, N>(grad, k, c, seen, sum, scale, accumulate);
  }
}

// Workgroups [0, run_blocks) add runs, the rest clear the rows without ids.
template <typename T, typename G, int N>
__global__ __launch_bounds__(kRowThreads) void grad_runs_kernel(
    Runs r, Mat<const T> dy, Mat<G> grad, float scale, bool accumulate, Pieces p,
    uint32_t run_blocks, unsigned long long run_items, const uint8_t* __restrict__ flags,
    uint32_t rows_per_block) {
  if (blockIdx.x < run_blocks) {
    const unsigned long long first = (unsigned long long)blockIdx.x * kRowThreads;
    if (first + threadIdx.x >= run_items) return;
    const Item it = ItemBase(first, p).at(threadIdx.x, p);
    sum_runs<T, G, N>(r, dy, grad, scale, accumulate, uint32_t(it.row), it.piece, p);
    return;
  }
  const long long row0 = (long long)(blockIdx.x - run_blocks) * rows_per_block;
  const uint32_t count = uint32_t(min((long long)rows_per_block, grad.rows - row0));
  const uint32_t items = count * p.per_row.d;
  for (uint32_t j = threadIdx.x; j < items; j += kRowThreads) {
    const uint32_t q = p.per_row.div(j);
    if (!flags[row0 + q])
      store_piece<N>(grad.at(row0 + q, p.begin(int(j - q * p.per_row.d))), Floats<N>(0.f));
  }
}

// Adds the parts of the long runs: the last part of the chunk a run starts in,
// then the first parts of the chunks it reaches.
template <typename G, int N>
__global__ __launch_bounds__(kRowThreads) void grad_join_kernel(Runs r, Mat<G> grad, float scale,
                                                                bool accumulate, Pieces p) {
  const uint32_t count = *r.long_count;
  for (uint32_t l = blockIdx.x; l < count; l += gridDim.x) {
    const uint32_t chunk = r.long_list[l];
    const uint32_t k = r.keys[min((chunk + 1) * kChunk, r.n) - 1];
    for (int piece = threadIdx.x; piece < int(p.per_row.d); piece += kRowThreads) {
      const int c = p.begin(piece);
      Floats<N> sum = load_piece<N>(r.partial + (2ull * chunk + 1) * r.ld + c);
      for (uint32_t q = chunk + 1; q * kChunk < r.n && r.keys[q * kChunk] == k; ++q)
        sum += load_piece<N>(r.partial + (2ull * q) * r.ld + c);
      write_grad<G, N>(grad, k, c, piece * N - c, sum, scale, accumulate);
    }
  }
}

// The workspace of the gradient.
struct GradSpace {
  size_t keys[2], at[2], table, cleared, cleared_bytes, long_list, partial, total;
  long long ld;
};

int digit_passes(long long rows, int* bits) {
  int all = 1;
  while ((1LL << all) <= rows) ++all;  // keys 0 .. rows
  const int passes = (all + 9) / 10;
  *bits = (all + passes - 1) / passes;
  return passes;
}

GradSpace grad_space(long long n, long long cols, long long rows) {
  GradSpace s{};
  int bits = 0;
  digit_passes(rows, &bits);
  size_t at = 0;
  const auto take = [&at](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) & ~size_t(255);
    return from;
  };
  for (int k = 0; k < 2; ++k) {
    s.keys[k] = take(size_t(n) * 4);
    s.at[k] = take(size_t(n) * 4);
  }
  s.table = take(id_sort_table_bytes(n, 1 << bits));
  s.cleared_bytes = (size_t(rows) + 16 + 15) & ~size_t(15);  // the long runs' count, the flags
  s.cleared = take(s.cleared_bytes);
  const size_t chunks = size_t((n + kChunk - 1) / kChunk);
  s.long_list = take(chunks * 4);
  s.ld = (cols + 7) & ~7LL;
  s.partial = take(2 * chunks * size_t(s.ld) * 4);
  s.total = at;
  return s;
}

// Sorts the ids; returns which of the two buffers holds the result.
template <typename I>
int sort_ids(const I* ids, uint32_t n, long long rows, long long padding, char* ws,
             const GradSpace& s, uint8_t* flags, int* result, hipStream_t stream) {
  int bits = 0;
  const int passes = digit_passes(rows, &bits);
  const auto buffer = [&](size_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
  ClearOnTheWay clear{reinterpret_cast<uint4*>(ws + s.cleared), s.cleared_bytes / 16};
  for (int k = 0; k < passes; ++k) {
    const Digit dg{k * bits, bits, 1 << bits};
    const int to = k & 1;
    const FlagSink sink{buffer(s.keys[to]), buffer(s.at[to]), k == passes - 1 ? flags : nullptr,
                        uint32_t(rows)};
    const int rc =
        k == 0 ? id_sort_pass(IdSource<I>{ids, rows, padding}, sink, n, dg, ws + s.table, clear,
                              stream)
               : id_sort_pass(PairSource{buffer(s.keys[to ^ 1]), buffer(s.at[to ^ 1])}, sink, n,
                              dg, ws + s.table, ClearOnTheWay{}, stream);
    if (rc != PS_OK) return rc;
    *result = to;
  }
  return PS_OK;
}

}  // namespace
}  // namespace ps

extern "C" {

int ps_embedding_lookup(const ps_rows* table, const ps_ids* ids, float scale, const ps_rows* out,
                        ps_stream_t stream) {
  PS_CHECK_ROWS(table);
  PS_CHECK_IDS(ids);
  PS_CHECK_ROWS(out);
  PS_CHECK_ARG(table->cols == out->cols && out->rows == ids->count,
               "ps_embedding_lookup: out is not ids x table columns");
  PS_CHECK_ARG(!ps::overlap(table, out), "ps_embedding_lookup: table and out overlap");
  if (!ids->count) return PS_OK;
  const hipStream_t st = ps::to_hip(stream);
  return ps::with_dtype(table->dtype, [&](auto t) {
    return ps::with_dtype(out->dtype, [&](auto o) {
      using T = decltype(t);
      using O = decltype(o);
      return ps::with_width<(sizeof(T) < sizeof(O) ? sizeof(T) : sizeof(O))>(
          out->cols, [&](auto n) {
            const ps::Pieces p(out->cols, n);
            const unsigned long long items = (unsigned long long)out->rows * p.per_row.d;
            return ps::launch_items(items, ps::kRowThreads, [&](uint32_t blocks, ps::Items part) {
              if (ids->type == PS_I64)
                ps::lookup_kernel<T, O, long long, n><<<blocks, ps::kRowThreads, 0, st>>>(
                    ps::mat<const T>(table), static_cast<const long long*>(ids->data), scale,
                    ps::mat<O>(out), p, part);
              else
                ps::lookup_kernel<T, O, int, n><<<blocks, ps::kRowThreads, 0, st>>>(
                    ps::mat<const T>(table), static_cast<const int*>(ids->data), scale,
                    ps::mat<O>(out), p, part);
            });
          });
    });
  });
}

size_t ps_embedding_grad_workspace_bytes(long long count, long long cols, long long table_rows) {
  if (count < 0 || count > (1LL << 30) || cols < 1 || cols > (1 << 24) || table_rows < 0 ||
      table_rows > (1LL << 31) - 2)
    return 0;
  return ps::grad_space(count, cols, table_rows).total;
}

int ps_embedding_grad(const ps_ids* ids, const ps_rows* grad_out, float scale,
                      long long padding_idx, int accumulate, const ps_rows* grad, void* workspace,
                      size_t workspace_bytes, ps_stream_t stream) {
  PS_CHECK_IDS(ids);
  PS_CHECK_ROWS(grad_out);
  PS_CHECK_ROWS(grad);
  PS_CHECK_ARG(grad_out->cols == grad->cols && grad_out->rows == ids->count,
               "ps_embedding_grad: grad_out is not ids x grad columns");
  PS_CHECK_ARG(grad->rows <= (1LL << 31) - 2, "ps_embedding_grad: too many rows");
  PS_CHECK_ARG(!ps::overlap(grad_out, grad), "ps_embedding_grad: grad_out and grad overlap");
  const ps::GradSpace s = ps::grad_space(ids->count, grad->cols, grad->rows);
  PS_CHECK_ARG(workspace && ps::aligned16(workspace) && workspace_bytes >= s.total,
               "ps_embedding_grad: workspace too small or misaligned");
  if (!grad->rows || (!ids->count && accumulate)) return PS_OK;
  const hipStream_t st = ps::to_hip(stream);
  char* ws = static_cast<char*>(workspace);
  uint8_t* flags = accumulate ? nullptr : reinterpret_cast<uint8_t*>(ws + s.cleared + 16);
  const uint32_t n = uint32_t(ids->count);
  int result = 0;
  const int rc =
      ids->type == PS_I64
          ? ps::sort_ids(static_cast<const long long*>(ids->data), n, grad->rows, padding_idx, ws,
                         s, flags, &result, st)
          : ps::sort_ids(static_cast<const int*>(ids->data), n, grad->rows, padding_idx, ws, s,
                         flags, &result, st);
  if (rc != PS_OK) return rc;
  ps::Runs r{};
  r.keys = reinterpret_cast<const uint32_t*>(ws + s.keys[result]);
  r.at = reinterpret_cast<const uint32_t*>(ws + s.at[result]);
  r.n = n;
  r.rows = uint32_t(grad->rows);
  r.partial = reinterpret_cast<float*>(ws + s.partial);
  r.ld = s.ld;
  r.long_count = reinterpret_cast<uint32_t*>(ws + s.cleared);
  r.long_list = reinterpret_cast<uint32_t*>(ws + s.long_list);
  const uint32_t chunks = (n + ps::kChunk - 1) / ps::kChunk;
  return ps::with_dtype(grad_out->dtype, [&](auto t) {
    return ps::with_dtype(grad->dtype, [&](auto g) {
      using T = decltype(t);
      using G = decltype(g);
      return ps::with_width<(sizeof(T) < sizeof(G) ? sizeof(T) : sizeof(G))>(
          grad->cols, [&](auto w) {
            const ps::Pieces p(grad->cols, w);
            const unsigned long long items = (unsigned long long)chunks * p.per_row.d;
            const unsigned long long run_blocks =
                (items + ps::kRowThreads - 1) / ps::kRowThreads;
            // 64 KB and more a clearing workgroup, at most 2^20 of them
            unsigned long long per_block =
                std::max<unsigned long long>(1, 65536 / (size_t(grad->cols) * sizeof(G)));
            per_block = std::max<unsigned long long>(per_block, (grad->rows >> 20) + 1);
            const unsigned long long clear_blocks =
                flags ? (grad->rows + per_block - 1) / per_block : 0;
            PS_CHECK_ARG(run_blocks + clear_blocks < (1u << 24) &&
                             per_block * p.per_row.d < (1u << 31),
                         "ps_embedding_grad: too many elements for one launch");
            if (run_blocks + clear_blocks) {
              ps::grad_runs_kernel<T, G, w>
                  <<<uint32_t(run_blocks + clear_blocks), ps::kRowThreads, 0, st>>>(
                      r, ps::mat<const T>(grad_out), ps::mat<G>(grad), scale, accumulate != 0, p,
                      uint32_t(run_blocks), items, flags, uint32_t(per_block));
              PS_LAUNCHED();
            }
            // a long run takes more than kChunk ids
            if (n > ps::kChunk + 1) {
              ps::grad_join_kernel<G, w>
                  <<<std::min(chunks, 2048u), ps::kRowThreads, 0, st>>>(r, ps::mat<G>(grad), scale,
                                                                       accumulate != 0, p);
              PS_LAUNCHED();
            }
            return PS_OK;
          });
    });
  });
}

}  // extern "C"
