// Embedding lookup with scaling, and its gradient by sorted ids.
//
// The lookup is a product by the matrix with a one per row at the id's column:
// a gather of rows, bound by the rows read and written.
//
// The gradient is the transposed product. Atomic additions would make its bits
// depend on their order and serialise on popular rows, so the ids are sorted
// (stably, ps_id_sort.hpp) and the gradient rows are sums over runs of equal
// ids. The sorted list is cut into chunks, each one thread's per piece of the
// width:
//  - a run belongs to the chunk it starts in when it ends before the next
//    chunk's end: one thread adds all of it and writes the row;
//  - a longer run is cut at the chunks' borders, every part is kept as a row of
//    32-bit partial sums, and a second launch adds the parts: shares of them in
//    order, the shares by halves.
// The order is fixed by the sizes, the ids and the place of a run among the
// sorted ones.
// So partial sums cost traffic only for runs longer than a chunk, and no row
// waits for one thread to walk a popular id's whole run. Rows without ids are
// cleared by the same launch, from flags the sort sets.
#include <algorithm>

#include "ps_id_sort.hpp"
#include "ps_rows.hpp"

namespace ps {
namespace {

// out = scale * table[id], one piece a thread. Bound by memory: 65,536 ids of a
// 131,072 x 4,096 BF16 table 170 us, 0.54 GB written and 0.51 GB read, of which
// the popular rows come from the caches; 262,144 of a 1,000,000 x 128 FP32 table 47
// us, 5.8 TB/s.
template <typename T, typename O, typename I, int N, bool kStream>
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
  store_piece<N, kStream>(out.at(it.row, c), v);
}

// Entries per chunk: shorter ones mean more loads in flight, longer ones fewer
// parts of long runs. 4 to 16 while no more than 4096 chunks result, as latency
// counts there (FP32, with 4, 8 and 16: 1,021 ids of 96 columns 14.7, 16.2 and
// 18.7 us, 8,192 of 64 24.5, 26.1 and 28.5, 32,768 of 64 30.5, 30.8 and 33.2, drawn
// by 1/rank 31.9, 28.4 and 28.7; 65,536 of 64, which take 16, 38, 33.9 and 35.3).
// Then doubled, up to 256, while the chunks hold more than kRunThreads threads,
// four waves a SIMD, at a thread for 8 columns. That is what rows of 16 bits
// take; FP32 rows have twice the threads, rows narrower than a piece one an
// element, and beyond 256 entries the threads grow with the list.
constexpr unsigned long long kRunThreads = 1u << 18;
uint32_t chunk_size(long long n, long long cols) {
  if (n <= 16) return 16;  // one chunk: no run can be long, and no join is launched
  uint32_t c = 4;
  while (c < 16 && n / c > 4096) c *= 2;
  const unsigned long long pieces = (unsigned long long)(cols + 7) / 8;
  while (c < 256 && (unsigned long long)(n / c) * pieces > kRunThreads) c *= 2;
  return c;
}

struct FlagSink {
  static constexpr bool kStarts = false;
  uint2* pairs;
  uint8_t* flags;  // flags[row] = 1 for rows with ids (null: not wanted)
  uint32_t rows;
  __device__ __forceinline__ void put(uint32_t pos, uint32_t key, uint32_t value) const {
    pairs[pos] = uint2{key, value};
    if (flags && key < rows) flags[key] = 1;
  }
  __device__ __forceinline__ void bin_start(uint32_t, uint32_t) const {}
};

constexpr uint32_t kManyChunks = 64;

// The sorted ids (`rows` = takes no part) and where their rows of grad_out are,
// n of them, and the partial sums: chunk q's first run's part in row 2q, its
// last run's in row 2q + 1, ld floats apart.
struct Runs {
  const uint2* sorted;
  __device__ __forceinline__ uint32_t key(unsigned long long i) const { return sorted[i].x; }
  uint32_t n, rows, chunk;  // chunk: entries of a chunk
  float* partial;
  long long ld;
  // The chunks in which long runs start: those that reach up to kManyChunks
  // chunks (count 0, listed from the front) and longer ones (count 1, from the
  // back).
  uint32_t *long_count, *long_list;
  uint32_t chunks;
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

// One chunk's runs, for one piece of the width. Rows are loaded kAhead at a
// time and one batch ahead of the additions, ids two batches ahead: a row's
// address waits for its id, and a wait for loads also waits for the stores
// issued before them, so the next rows are under way before a finished run is
// written. Eight rows a batch are slower (calls of 262,147 skewed ids of 333 FP16
// columns 83.4 us instead of 80.0, 32,768 of 4,096 BF16 98.7 instead of 93.1, 1,021
// of 96 FP32 16.9 instead of 14.4).
template <typename T, typename G, int N>
__device__ void sum_runs(const Runs& r, const Mat<const T>& dy, const Mat<G>& grad, float scale,
                         bool accumulate, uint32_t chunk, int piece, const Pieces& p) {
  constexpr int kAhead = 4;
  using V = typename PieceOf<T, N>::type;
  constexpr uint32_t kNone = 0xFFFFFFFFu;  // no key
  const int c = p.begin(piece);
  const int seen = piece * N - c;
  const uint32_t size = r.chunk, b = chunk * size, e = min(b + size, r.n);
  const uint32_t next = min(e + size, r.n);
  uint32_t id[2][kAhead], at[2][kAhead];  // of the batches after the loaded one
  const auto load_ids = [&](uint32_t i, int s) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t q = min(i + j, r.n - 1);
      const uint2 pair = r.sorted[q];
      id[s][j] = pair.x;
      at[s][j] = pair.y;
    }
  };
  load_ids(b, 0);
  load_ids(b + kAhead, 1);
  // The ids around the chunk, loaded together: they come from far, and asked
  // for one after another they cost as much as the rows.
  const uint32_t first = id[0][0], last = r.key(e - 1);
  const uint32_t before = r.key(max(b, 1u) - 1), far_before = r.key(max(b, size + 1) - size - 1);
  const uint32_t behind = r.key(min(e, r.n - 1)), far_behind = r.key(min(next, r.n - 1));
  if (first >= r.rows) return;  // only ids that take no part
  // The first run may start in a chunk before: then it is that chunk's, or long.
  const bool continued = b > 0 && before == first;
  const bool head_long =
      continued && ((b > size && far_before == first) || (e < r.n && behind == first));
  // The last run may go on: then it is long, or this chunk's to the end.
  const bool own_tail =
      e < r.n && behind == last && last < r.rows && !(continued && first == last);
  const bool tail_long = own_tail && next < r.n && far_behind == last;
  const uint32_t end = own_tail && !tail_long ? next : e;

  uint32_t key[2][kAhead];
  V row[2][kAhead];
  const auto load_rows = [&](uint32_t i, int s) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const bool mine = i + j < e || (i + j < end && id[s][j] == last);
      key[s][j] = mine && id[s][j] < r.rows ? id[s][j] : kNone;
      const bool wanted = key[s][j] != kNone && !(continued && !head_long && key[s][j] == first);
      // (row 0 for the others: a load without a branch around it)
      row[s][j] = *reinterpret_cast<const V*>(dy.at(wanted ? at[s][j] : 0u, c));
    }
  };
  uint32_t current = kNone;
  bool in_head = false;
  Floats<N> sum = 0.f;
  const auto finish = [&] {
    if (current >= r.rows) return;  // nothing yet
    if (!in_head)
      write_grad<G, N>(grad, current, c, seen, sum, scale, accumulate);
    else if (head_long)
      store_piece<N>(r.partial + (2ull * chunk) * r.ld + c, sum);
  };
  load_rows(b, 0);
  for (uint32_t i = b; i < end; i += 2 * kAhead) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const uint32_t here = i + s * kAhead;
      load_ids(here + 2 * kAhead, s);
      load_rows(here + kAhead, s ^ 1);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (key[s][j] == kNone) continue;
        if (key[s][j] != current) {
          finish();
          in_head = continued && key[s][j] == first;
          current = key[s][j];
          sum = 0.f;
        }
        sum += __builtin_convertvector(row[s][j], Floats<N>);
      }
    }
    if (i + 2 * kAhead >= e && key[0][0] == kNone) break;  // the run has ended
  }
  if (tail_long) {
    store_piece<N>(r.partial + (2ull * chunk + 1) * r.ld + c, sum);
    if (piece == 0) {
      const unsigned long long far = e + (unsigned long long)kManyChunks * size;
      if (far < r.n && r.key(far) == last)
        r.long_list[r.chunks - 1 - atomicAdd(r.long_count + 1, 1u)] = chunk;
      else
        r.long_list[atomicAdd(r.long_count, 1u)] = chunk;
    }
  } else {
    finish();
  }
}

// Workgroups [0, run_blocks) add runs, the rest clear the rows without ids, so
// that the clearing's stores fill the memory while the runs wait for loads.
// Cleared rows are not read again soon: non-temporal stores, and 16 KB a
// workgroup (64 KB ones took 10% longer). Bound by memory: 32,768 BF16 rows into
// 131,072 x 4,096 FP32, 2.41 GB in 402 us, 6.0 TB/s.
constexpr uint32_t kClearItems = 4;  // per thread
template <typename T, typename G, int N>
__global__ __launch_bounds__(kRowThreads) void grad_runs_kernel(
    Runs r, Mat<const T> dy, Mat<G> grad, float scale, bool accumulate, Pieces p,
    uint32_t run_blocks, const uint8_t* __restrict__ flags, Items clear_items) {
  if (blockIdx.x < run_blocks) {
    const unsigned long long first = (unsigned long long)blockIdx.x * kRowThreads;
    if (first + threadIdx.x >= (unsigned long long)r.chunks * p.per_row.d) return;
    const Item it = ItemBase(first, p).at(threadIdx.x, p);
    sum_runs<T, G, N>(r, dy, grad, scale, accumulate, uint32_t(it.row), it.piece, p);
    return;
  }
  const unsigned long long first =
      clear_items.begin +
      (unsigned long long)(blockIdx.x - run_blocks) * (kRowThreads * kClearItems);
  const unsigned long long left = clear_items.end - first;
  const ItemBase base(first, p);
  Item it[kClearItems];
  uint8_t used[kClearItems];
#pragma unroll
  for (uint32_t u = 0; u < kClearItems; ++u) {
    const uint32_t j = u * kRowThreads + threadIdx.x;
    it[u] = base.at(j, p);
    used[u] = j < left ? flags[it[u].row] : 1;
  }
  using V = typename PieceOf<G, N>::type;
#pragma unroll
  for (uint32_t u = 0; u < kClearItems; ++u)
    if (!used[u])
      __builtin_nontemporal_store(
          V(G(0.f)), reinterpret_cast<V*>(grad.at(it[u].row, p.begin(it[u].piece))));
}

// How many of the chunks from `from` on begin inside the run of key k: every
// round asks at as many places as there are threads.
__device__ __forceinline__ uint32_t chunks_in_run(const Runs& r, uint32_t from, uint32_t k) {
  uint32_t lo = 0, hi = r.chunks - from;  // the answer's bounds
  while (lo < hi) {
    const uint32_t step = (hi - lo + kRowThreads - 1) / kRowThreads;
    const uint32_t at = lo + threadIdx.x * step;
    const uint32_t hits = __syncthreads_count(
        at < hi && r.key((unsigned long long)(from + at) * r.chunk) == k);
    if (!hits) return lo;
    hi = min(hi, lo + hits * step);
    lo += (hits - 1) * step + 1;
  }
  return lo;
}

// Adds the parts of the long run that starts in `chunk` for kJoinPieces pieces
// of the width: its last part, then the first parts of the chunks it reaches.
// The workgroup's thread groups take shares of the parts in order, and the
// shares are added by halves.
template <int kJoinPieces, typename G, int N>
__device__ void join_run(const Runs& r, const Mat<G>& grad, float scale, bool accumulate,
                         uint32_t chunk, uint32_t tile, const Pieces& p, float* part) {
  constexpr uint32_t kGroups = kRowThreads / kJoinPieces;
  const uint32_t group = threadIdx.x / kJoinPieces, lane = threadIdx.x % kJoinPieces;
  const uint32_t piece = tile * kJoinPieces + lane;
  const uint32_t k = r.key((chunk + 1) * r.chunk - 1);
  const uint32_t reached = chunks_in_run(r, chunk + 1, k);
  const uint32_t share = (reached + kGroups - 1) / kGroups;
  const uint32_t from = min(group * share, reached), to = min(from + share, reached);
  const bool on = piece < p.per_row.d;
  const int c = on ? p.begin(int(piece)) : 0;
  Floats<N> sum = 0.f;
  if (on) {
    if (group == 0) sum = load_piece<N>(r.partial + (2ull * chunk + 1) * r.ld + c);
    const float* at = r.partial + 2ull * (chunk + 1) * r.ld + c;
#pragma unroll 8
    for (uint32_t q = from; q < to; ++q) sum += load_piece<N>(at + 2ull * q * r.ld);
  }
  uint32_t half = kGroups / 2;
  while (half && half * share >= reached) half /= 2;  // groups without a share
  for (; half; half /= 2) {
    if (group >= half && group < 2 * half)
#pragma unroll
      for (int e = 0; e < N; ++e) part[((group - half) * kJoinPieces + lane) * N + e] = sum[e];
    __syncthreads();
    if (group < half)
#pragma unroll
      for (int e = 0; e < N; ++e) sum[e] += part[(group * kJoinPieces + lane) * N + e];
    __syncthreads();
  }
  if (group == 0 && on) write_grad<G, N>(grad, k, c, int(piece) * N - c, sum, scale, accumulate);
}

// Workgroups of 16 groups for runs of some parts, of 64 for those of many: 2,048
// parts of 336 columns take 12 us so, 22 with 16 groups.
constexpr int kFewPieces = 16, kManyPieces = 4;
template <typename G, int N>
__global__ __launch_bounds__(kRowThreads) void grad_join_kernel(Runs r, Mat<G> grad, float scale,
                                                                bool accumulate, Pieces p) {
  __shared__ float part[kRowThreads / 2 * N];
  const uint32_t few_tiles = (p.per_row.d + kFewPieces - 1) / kFewPieces;
  const uint32_t many_tiles = (p.per_row.d + kManyPieces - 1) / kManyPieces;
  const unsigned long long few = (unsigned long long)r.long_count[0] * few_tiles;
  const unsigned long long many = (unsigned long long)r.long_count[1] * many_tiles;
  for (unsigned long long l = blockIdx.x; l < many + few; l += gridDim.x) {
    if (l < many)
      join_run<kManyPieces, G, N>(r, grad, scale, accumulate,
                                  r.long_list[r.chunks - 1 - l / many_tiles],
                                  uint32_t(l % many_tiles), p, part);
    else
      join_run<kFewPieces, G, N>(r, grad, scale, accumulate, r.long_list[(l - many) / few_tiles],
                                 uint32_t((l - many) % few_tiles), p, part);
  }
}

// The workspace of the gradient.
struct GradSpace {
  size_t pairs[2], table, cleared, cleared_bytes, long_list, partial, total;
  size_t groups_bytes, flags;  // flags: from `cleared` on
  long long ld;
};

int digit_passes(long long rows, int* bits) {
  int all = 1;
  while ((1LL << all) <= rows) ++all;  // keys 0 .. rows
  const int passes = (all + 9) / 10;
  *bits = (all + passes - 1) / passes;
  return passes;
}

// What the parts of the workspace take.
struct GradSizes {
  size_t table, groups;  // groups: of one pass
  int passes;
  size_t chunks, partial;  // partial: floats
};

GradSpace grad_layout(long long n, long long rows, const GradSizes& z) {
  GradSpace s{};
  size_t at = 0;
  const auto take = [&at](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) & ~size_t(255);
    return from;
  };
  for (int k = 0; k < 2; ++k) s.pairs[k] = take(size_t(n) * sizeof(uint2));
  s.table = take(z.table);
  // the long runs' counts, every pass's groups, the flags
  s.groups_bytes = z.groups;
  s.flags = 16 + size_t(z.passes) * z.groups;
  s.cleared_bytes = (s.flags + size_t(rows) + 15) & ~size_t(15);
  s.cleared = take(s.cleared_bytes);
  s.long_list = take(z.chunks * 4);
  s.partial = take(z.partial * 4);
  s.total = at;
  return s;
}

long long partial_ld(long long cols) { return (cols + 7) & ~7LL; }

// The workspace of one call.
GradSpace grad_space(long long n, long long cols, long long rows) {
  int bits = 0;
  const int passes = digit_passes(rows, &bits);
  const int bins = 1 << bits;
  const IdCut cut = id_cut(n);
  const size_t chunk = chunk_size(n, cols), chunks = (size_t(n) + chunk - 1) / chunk;
  const size_t ld = size_t(partial_ld(cols));
  GradSpace s =
      grad_layout(n, rows, {id_sort_table_bytes(cut, bins), id_sort_group_bytes(cut, bins), passes,
                            chunks, 2 * chunks * ld});
  s.ld = (long long)ld;
  return s;
}

// The bytes that callers are asked for: no less than grad_space() of any call of
// as many ids, columns and rows or fewer, though longer chunks, wider tiles and
// shorter digits make some larger calls need less. Each part is bounded by what
// grows with all three:
//  - bins: 2^bits up to 1023 rows, which take one digit, and 1024 beyond;
//  - chunks: ceil(n / 4) while chunk_size() starts from 4, no more than 4097 where
//    it starts from 8, ceil(n / 16) beyond;
//  - chunks * ld: a chunk is the shortest one (bounded above), 256 entries, or
//    leaves chunks * ld / 8 <= kRunThreads, one partly filled chunk aside.
size_t grad_space_most(long long n, long long cols, long long rows) {
  int bits = 0;
  const int passes = digit_passes(rows, &bits);
  const int bins = passes > 1 ? 1024 : 1 << bits;
  const IdCut cut = id_cut_most(n);
  const auto chunks_of = [n](long long chunk) { return size_t((n + chunk - 1) / chunk); };
  const size_t chunks = std::max(std::min<size_t>(chunks_of(4), 4097), chunks_of(16));
  const size_t ld = size_t(partial_ld(cols));
  const size_t partial =
      std::min(chunks * ld, std::max(8 * size_t(kRunThreads) + ld, chunks_of(256) * ld));
  return grad_layout(n, rows, {id_sort_table_bytes(cut, bins), id_sort_group_bytes(cut, bins),
                               passes, chunks, 2 * partial})
      .total;
}

// The one workgroup that sorts a tile clears this many 16-byte words on the way
// (256 KB); more are cleared by a launch of their own (100 ids of 8 FP16 columns,
// on the way and by a launch: 15.0 and 14.9 us for 10,007 rows, 15.7 and 15.7 for
// 112,000, 16.4 and 16.0 for 250,000, 19.4 and 17.5 for 500,000; 4,000 ids 24.6 and
// 25.9 for 112,000, 25.8 and 26.2 for 250,000, 29.3 and 28.2 for 500,000).
constexpr size_t kTileClears = 16384;

// Sorts the ids; returns which of the two buffers holds the result.
template <typename I>
int sort_ids(const I* ids, uint32_t n, long long rows, long long padding, char* ws,
             const GradSpace& s, uint8_t* flags, int* result, hipStream_t stream) {
  int bits = 0;
  const int passes = digit_passes(rows, &bits);
  const auto pairs = [&](int k) { return reinterpret_cast<uint2*>(ws + s.pairs[k]); };
  ClearOnTheWay clear{reinterpret_cast<uint4*>(ws + s.cleared),
                      (flags ? s.cleared_bytes : s.flags) / 16};
  if (s.groups_bytes || (n <= kIdTile && clear.count > kTileClears)) {
    const int rc = id_clear(clear, stream);
    if (rc != PS_OK) return rc;
    clear = {};
  }
  if (n <= kIdTile) {
    *result = 0;
    return id_sort_tile(IdSource<I>{ids, rows, padding},
                        FlagSink{pairs(0), flags, uint32_t(rows)}, n, Digit{0, bits, 1 << bits},
                        passes, clear, stream);
  }
  for (int k = 0; k < passes; ++k) {
    const Digit dg{k * bits, bits, 1 << bits};
    const FlagSink sink{pairs(k & 1), k == passes - 1 ? flags : nullptr, uint32_t(rows)};
    void* const groups = ws + s.cleared + 16 + size_t(k) * s.groups_bytes;
    const int rc =
        k == 0 ? id_sort_pass(IdSource<I>{ids, rows, padding}, sink, n, dg, ws + s.table, groups,
                              clear, stream)
               : id_sort_pass(PairSource{pairs((k & 1) ^ 1)}, sink, n, dg, ws + s.table, groups,
                              ClearOnTheWay{}, stream);
    if (rc != PS_OK) return rc;
    *result = k & 1;
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
  PS_CHECK_ARG(!ps::overlap(ps::region(out), {ps::region(table), ps::region(ids)}),
               "ps_embedding_lookup: out overlaps an input");
  if (!ids->count) return PS_OK;
  const hipStream_t st = ps::to_hip(stream);
  return ps::with_dtype(table->dtype, [&](auto t) {
    return ps::with_dtype(out->dtype, [&](auto o) {
      using T = decltype(t);
      using O = decltype(o);
      return ps::with_width<(sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O))>(
          out->cols, [&](auto n) {
            const ps::Pieces p(out->cols, n);
            const unsigned long long items = (unsigned long long)out->rows * p.per_row.d;
            return ps::with_flag(ps::streamed(out, out->rows), [&](auto stream_out) {
              return ps::launch_items(items, ps::kRowThreads, [&](uint32_t blocks, ps::Items part) {
                if (ids->type == PS_I64)
                  ps::lookup_kernel<T, O, long long, n, stream_out>
                      <<<blocks, ps::kRowThreads, 0, st>>>(
                          ps::mat<const T>(table), static_cast<const long long*>(ids->data), scale,
                          ps::mat<O>(out), p, part);
                else
                  ps::lookup_kernel<T, O, int, n, stream_out><<<blocks, ps::kRowThreads, 0, st>>>(
                      ps::mat<const T>(table), static_cast<const int*>(ids->data), scale,
                      ps::mat<O>(out), p, part);
              });
            });
          });
    });
  });
}

size_t ps_embedding_grad_workspace_bytes(long long count, long long cols, long long table_rows) {
  if (count < 0 || count > (1LL << 30) || cols < 1 || cols > (1 << 24) || table_rows < 0 ||
      table_rows > (1LL << 31) - 2)
    return 0;
  return ps::grad_space_most(count, cols, table_rows);
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
  PS_CHECK_ARG(workspace && ps::aligned16(workspace) &&
                   workspace_bytes >= ps::grad_space_most(ids->count, grad->cols, grad->rows),
               "ps_embedding_grad: workspace too small or misaligned");
  const ps::GradSpace s = ps::grad_space(ids->count, grad->cols, grad->rows);
  const ps::Region read[] = {ps::region(ids), ps::region(grad_out)};
  PS_CHECK_ARG(!ps::overlap(ps::region(grad), {read[0], read[1]}),
               "ps_embedding_grad: grad overlaps an input");
  PS_CHECK_ARG(!ps::overlap(ps::region(workspace, s.total), {read[0], read[1], ps::region(grad)}),
               "ps_embedding_grad: the workspace overlaps another argument");
  if (!grad->rows || (!ids->count && accumulate)) return PS_OK;
  const hipStream_t st = ps::to_hip(stream);
  char* ws = static_cast<char*>(workspace);
  uint8_t* flags = accumulate ? nullptr : reinterpret_cast<uint8_t*>(ws + s.cleared + s.flags);
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
  r.sorted = reinterpret_cast<const uint2*>(ws + s.pairs[result]);
  r.n = n;
  r.rows = uint32_t(grad->rows);
  r.partial = reinterpret_cast<float*>(ws + s.partial);
  r.ld = s.ld;
  r.long_count = reinterpret_cast<uint32_t*>(ws + s.cleared);
  r.long_list = reinterpret_cast<uint32_t*>(ws + s.long_list);
  r.chunk = ps::chunk_size(ids->count, grad->cols);
  r.chunks = (n + r.chunk - 1) / r.chunk;
  return ps::with_dtype(grad_out->dtype, [&](auto t) {
    return ps::with_dtype(grad->dtype, [&](auto g) {
      using T = decltype(t);
      using G = decltype(g);
      return ps::with_width<(sizeof(T) > sizeof(G) ? sizeof(T) : sizeof(G))>(
          grad->cols, [&](auto w) {
            const ps::Pieces p(grad->cols, w);
            const unsigned long long run_blocks =
                ((unsigned long long)r.chunks * p.per_row.d + ps::kRowThreads - 1) /
                ps::kRowThreads;
            // The first launch takes the runs and as many rows to clear as
            // fit beside them, the others more rows.
            const unsigned long long clears =
                flags ? (unsigned long long)grad->rows * p.per_row.d : 0;
            PS_CHECK_ARG(run_blocks < (1u << 23), "ps_embedding_grad: too many ids for one launch");
            uint32_t runs = uint32_t(run_blocks);
            unsigned long long done = 0;
            do {
              const unsigned long long per_block = ps::kRowThreads * ps::kClearItems;
              const unsigned long long blocks = std::min<unsigned long long>(
                  (clears - done + per_block - 1) / per_block, 1u << 23);
              if (!(runs + blocks)) break;
              const unsigned long long end = std::min(clears, done + blocks * per_block);
              ps::grad_runs_kernel<T, G, w>
                  <<<uint32_t(runs + blocks), ps::kRowThreads, 0, st>>>(
                      r, ps::mat<const T>(grad_out), ps::mat<G>(grad), scale, accumulate != 0, p,
                      runs, flags, ps::Items{done, end});
              PS_LAUNCHED();
              runs = 0;
              done = end;
            } while (done < clears);
            // a long run holds more than a chunk
            if (n > r.chunk + 1) {
              const uint32_t tiles = (p.per_row.d + ps::kManyPieces - 1) / ps::kManyPieces;
              const unsigned long long most = (unsigned long long)r.chunks * tiles;
              ps::grad_join_kernel<G, w>
                  <<<uint32_t(std::min(most, 2048ull)), ps::kRowThreads, 0, st>>>(
                      r, ps::mat<G>(grad), scale, accumulate != 0, p);
              PS_LAUNCHED();
            }
            return PS_OK;
          });
    });
  });
}

}  // extern "C"
