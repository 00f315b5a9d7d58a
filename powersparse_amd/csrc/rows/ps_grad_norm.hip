// The norm over many gradient tensors, and clipping by it.
//
// The tensors are cut into chunks; a fixed number of workgroups walks them and
// each adds its chunks' squares in 64 bits: FP32 squares overflow from 1.8e19
// and vanish below 1e-23, and 64-bit sums hide every rounding order. One launch
// leaves a sum per workgroup, and the next launch's workgroups each add those
// (at most kBlocks, from the L2) before they scale their chunks: no atomics, so
// the same bits every time, and no launch between the two.
//
// Bound by memory: every gradient is read once for the norm and, where it
// changes, once more to be scaled. 800 M BF16 elements into FP32: 1.65 GB in 310
// us, 5.3 TB/s, then 4.9 GB in 957 us, 5.1 TB/s; in place 888 us in all. The
// second pass walks the chunks backwards, so what the first one read last may
// still be in the last-level cache.
#include <algorithm>
#include <mutex>
#include <utility>
#include <vector>

#include "ps_rows.hpp"

namespace ps {

struct GradTensor {
  const void* data;
  void* out;
  long long count;
  int dtype, out_dtype;
  long long first_chunk;
};
struct GradChunk {
  uint32_t tensor, index;  // elements [index * kChunk, ...) of the tensor
};

namespace {

constexpr int kClipThreads = 256;
constexpr uint32_t kBlocks = 2048;
// Elements of a chunk. The workgroups go through the chunks side by side, so
// small chunks keep what they touch at one time together: clipping 800 M BF16
// elements into FP32 took 951 us with 4096, 984 with 8192, 1089 with 32,768,
// 992 with 2048.
constexpr long long kChunk = 4096;

struct Grads {
  const GradTensor* tensors;
  const GradChunk* chunks;
  uint32_t chunk_count;
  bool in_place;
};

// The chunk table: the tensor that chunk q is of, by bisection.
__global__ __launch_bounds__(kClipThreads) void chunk_kernel(const GradTensor* __restrict__ tensors,
                                                             uint32_t tensor_count,
                                                             GradChunk* __restrict__ chunks,
                                                             uint32_t chunk_count) {
  const uint32_t q = blockIdx.x * kClipThreads + threadIdx.x;
  if (q >= chunk_count) return;
  uint32_t lo = 0, hi = tensor_count - 1;  // the last tensor that begins at or before q
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (tensors[mid].first_chunk <= q)
      lo = mid;
    else
      hi = mid - 1;
  }
  chunks[q] = {lo, uint32_t(q - tensors[lo].first_chunk)};
}

// Sum over the workgroup, in every thread.
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kClipThreads / kWave];
#pragma unroll
  for (int d = kWave / 2; d; d >>= 1) v += __shfl_xor(v, d, kWave);
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < kClipThreads / kWave; ++w) v += part[w];
  return v;
}

template <typename T>
__device__ double square_sum(const T* p, uint32_t count) {
  constexpr int N = 16 / sizeof(T);
  double s = 0;
  uint32_t i = threadIdx.x * N;
  for (; i + N <= count; i += kClipThreads * N) {
    const Floats<N> v = load_piece<N>(p + i);
#pragma unroll
    for (int e = 0; e < N; ++e) s += double(v[e]) * double(v[e]);
  }
  for (; i < count; ++i) s += double(float(p[i])) * double(float(p[i]));
  return s;
}

__global__ __launch_bounds__(kClipThreads) void norm_kernel(Grads g, double* __restrict__ sums) {
  double s = 0;
  for (uint32_t q = blockIdx.x; q < g.chunk_count; q += gridDim.x) {
    const GradChunk ch = g.chunks[q];
    const GradTensor t = g.tensors[ch.tensor];
    const long long from = (long long)ch.index * kChunk;
    const uint32_t count = uint32_t(min(kChunk, t.count - from));
    if (t.dtype == PS_F32)
      s += square_sum(static_cast<const f32*>(t.data) + from, count);
    else if (t.dtype == PS_F16)
      s += square_sum(static_cast<const f16*>(t.data) + from, count);
    else
      s += square_sum(static_cast<const bf16*>(t.data) + from, count);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// The norm from the workgroups' sums, in every thread.
__device__ __forceinline__ double norm_of(const double* sums, uint32_t count, double grad_scale) {
  double s = 0;
  for (uint32_t i = threadIdx.x; i < count; i += kClipThreads) s += sums[i];
  return sqrt(block_sum(s)) * fabs(grad_scale);
}

__global__ __launch_bounds__(kClipThreads) void norm_join_kernel(const double* __restrict__ sums,
                                                                 uint32_t count, double grad_scale,
                                                                 float* __restrict__ norm) {
  const double v = norm_of(sums, count, grad_scale);
  if (threadIdx.x == 0) *norm = float(v);
}

template <typename T, typename O>
__device__ void scale_chunk(const T* p, O* out, uint32_t count, float c) {
  constexpr int N = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
  uint32_t i = threadIdx.x * N;
#pragma unroll 4
  for (; i + N <= count; i += kClipThreads * N)
    store_piece<N>(out + i, c * load_piece<N>(p + i));
  for (; i < count; ++i) out[i] = O(c * float(p[i]));
}

template <typename T>
__device__ void scale_to(const GradTensor& t, long long from, uint32_t count, float c) {
  const T* p = static_cast<const T*>(t.data) + from;
  if (t.out_dtype == PS_F32)
    scale_chunk(p, static_cast<f32*>(t.out) + from, count, c);
  else if (t.out_dtype == PS_F16)
    scale_chunk(p, static_cast<f16*>(t.out) + from, count, c);
  else
    scale_chunk(p, static_cast<bf16*>(t.out) + from, count, c);
}

// sums: the norm kernel's, or null with *norm given.
__global__ __launch_bounds__(kClipThreads) void clip_kernel(Grads g,
                                                            const double* __restrict__ sums,
                                                            uint32_t sum_count, double max_norm,
                                                            double grad_scale,
                                                            float* __restrict__ norm) {
  float n;  // in 32 bits either way, so that one call clips as two do
  if (sums) {
    n = float(norm_of(sums, sum_count, grad_scale));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  } else {
    n = *norm;
  }
  const double v = n;
  const double ratio = max_norm / (v + 1e-6);
  const float c = float((ratio > 1.0 ? 1.0 : ratio) * grad_scale);  // a NaN ratio stays
  if (g.in_place && c == 1.f) return;
  for (uint32_t q = blockIdx.x; q < g.chunk_count; q += gridDim.x) {
    const GradChunk ch = g.chunks[g.chunk_count - 1 - q];
    const GradTensor t = g.tensors[ch.tensor];
    const long long from = (long long)ch.index * kChunk;
    const uint32_t count = uint32_t(min(kChunk, t.count - from));
    if (t.dtype == PS_F32)
      scale_to<f32>(t, from, count, c);
    else if (t.dtype == PS_F16)
      scale_to<f16>(t, from, count, c);
    else
      scale_to<bf16>(t, from, count, c);
  }
}

}  // namespace
}  // namespace ps

namespace ps {
namespace {

// Where a list's gradients, or its outputs, are: ranges that do not meet, in order.
class Ranges {
 public:
  void add(const void* p, size_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    ranges_.push_back({at, at + bytes});
  }
  void close() {
    std::sort(ranges_.begin(), ranges_.end(),
              [](const Range& a, const Range& b) { return a.begin < b.begin; });
    size_t kept = 0;
    for (const Range& r : ranges_) {
      if (kept && r.begin <= ranges_[kept - 1].end)
        ranges_[kept - 1].end = std::max(ranges_[kept - 1].end, r.end);
      else
        ranges_[kept++] = r;
    }
    ranges_.resize(kept);
  }
  bool meets(const void* p, size_t bytes) const {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const auto r = std::upper_bound(ranges_.begin(), ranges_.end(), at,
                                    [](uintptr_t x, const Range& range) { return x < range.end; });
    return r != ranges_.end() && r->begin < at + bytes;
  }

 private:
  struct Range {
    uintptr_t begin, end;
  };
  std::vector<Range> ranges_;
};

}  // namespace
}  // namespace ps

struct ps_grad_list {
  void* tables = nullptr;  // tensors, chunks, the workgroups' sums
  ps::Grads grads{};
  double* sums = nullptr;
  uint32_t blocks = 0;
  ps::Ranges read, written;
  ps_grad_list* retired = nullptr;  // the next destroyed list
};

namespace ps {
namespace {

// What is written must be read by nobody else: the index of a tensor whose
// output meets another tensor's data or output, or -1.
int shared_output(const std::vector<GradTensor>& table) {
  struct Range {
    uintptr_t begin, end;
    int tensor;
  };
  const auto range = [](const void* p, long long count, int dtype, size_t tensor) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    return Range{at, at + uintptr_t(count) * dtype_size(dtype), int(tensor)};
  };
  std::vector<Range> outs;
  for (size_t i = 0; i < table.size(); ++i)
    outs.push_back(range(table[i].out, table[i].count, table[i].out_dtype, i));
  std::sort(outs.begin(), outs.end(),
            [](const Range& a, const Range& b) { return a.begin < b.begin; });
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].begin < outs[i - 1].end) return outs[i].tensor;
  for (size_t i = 0; i < table.size(); ++i) {
    const Range d = range(table[i].data, table[i].count, table[i].dtype, i);
    // the first output that ends behind the data's begin
    const auto o = std::upper_bound(outs.begin(), outs.end(), d.begin,
                                    [](uintptr_t at, const Range& r) { return at < r.end; });
    if (o != outs.end() && o->begin < d.end && o->tensor != int(i)) return int(i);
  }
  return -1;
}

// Destroyed lists, whose memory goes back when the next list is made, which waits
// for the device anyway: freeing waits for it and is refused while any stream is
// captured (the capture is lost), and a list may go at any time, from a garbage
// collector too.
std::mutex g_retired_mu;
ps_grad_list* g_retired = nullptr;

void free_retired() {
  ps_grad_list* list;
  {
    std::lock_guard<std::mutex> lock(g_retired_mu);
    list = std::exchange(g_retired, nullptr);
  }
  while (list) {
    ps_grad_list* const next = list->retired;
    dev_free(list->tables);
    delete list;
    list = next;
  }
}

int build_chunks(const GradTensor* tensors, uint32_t tensor_count, GradChunk* chunks,
                 uint32_t chunk_count) {
  chunk_kernel<<<(chunk_count + kClipThreads - 1) / kClipThreads, kClipThreads>>>(
      tensors, tensor_count, chunks, chunk_count);
  PS_LAUNCHED();
  PS_HIP(hipStreamSynchronize(nullptr));
  return PS_OK;
}

int launch_norm(const ps_grad_list& l, hipStream_t stream) {
  if (!l.blocks) return PS_OK;
  norm_kernel<<<l.blocks, kClipThreads, 0, stream>>>(l.grads, l.sums);
  PS_LAUNCHED();
  return PS_OK;
}

int launch_clip(const ps_grad_list& l, uint32_t blocks, const double* sums, float max_norm,
                float grad_scale, float* norm, hipStream_t stream) {
  clip_kernel<<<blocks, kClipThreads, 0, stream>>>(l.grads, sums, l.blocks, double(max_norm),
                                                   double(grad_scale), norm);
  PS_LAUNCHED();
  return PS_OK;
}

}  // namespace
}  // namespace ps

extern "C" {

int ps_grad_list_create(int tensors, void* const* data, const long long* counts,
                        const int* dtypes, void* const* out, const int* out_dtypes,
                        ps_grad_list** list) {
  PS_CHECK_ARG(list, "ps_grad_list_create: null output");
  *list = nullptr;
  PS_CHECK_ARG(tensors >= 0 && tensors <= (1 << 24), "ps_grad_list_create: bad tensor count");
  PS_CHECK_ARG(!tensors || (data && counts && dtypes && !out == !out_dtypes),
               "ps_grad_list_create: null array");
  try {
    std::vector<ps::GradTensor> table;
    ps::Ranges read, written;
    long long total = 0, chunks = 0;
    bool in_place = true;
    for (int i = 0; i < tensors; ++i) {
      const std::string name = "ps_grad_list_create: tensor " + std::to_string(i);
      const int out_dtype = out ? out_dtypes[i] : dtypes[i];
      PS_CHECK_ARG(ps::dtype_valid(dtypes[i]) && ps::dtype_valid(out_dtype),
                   name + ": unknown element type");
      PS_CHECK_ARG(counts[i] >= 0 && counts[i] <= (1LL << 44) && total <= (1LL << 44),
                   name + ": bad count");
      if (!counts[i]) continue;
      void* const to = out ? out[i] : data[i];
      PS_CHECK_ARG(data[i] && to, name + ": null data");
      const size_t size = ps::dtype_size(dtypes[i]), out_size = ps::dtype_size(out_dtype);
      PS_CHECK_ARG(reinterpret_cast<uintptr_t>(data[i]) % size == 0 &&
                       reinterpret_cast<uintptr_t>(to) % out_size == 0,
                   name + ": misaligned data");
      PS_CHECK_ARG((to == data[i] && out_dtype == dtypes[i]) ||
                       !ps::overlap(ps::region(data[i], size_t(counts[i]) * size),
                                    ps::region(to, size_t(counts[i]) * out_size)),
                   name + ": overlaps its output");
      table.push_back({data[i], to, counts[i], dtypes[i], out_dtype, chunks});
      read.add(data[i], size_t(counts[i]) * size);
      written.add(to, size_t(counts[i]) * out_size);
      total += counts[i];
      chunks += (counts[i] + ps::kChunk - 1) / ps::kChunk;
      in_place = in_place && to == data[i];
    }
    PS_CHECK_ARG(chunks < (1LL << 31), "ps_grad_list_create: too many elements");
    PS_CHECK_ARG(ps::shared_output(table) < 0,
                 "ps_grad_list_create: an output overlaps another tensor, or a tensor is "
                 "listed twice");
    read.close();
    written.close();
    const size_t table_bytes = (table.size() * sizeof(ps::GradTensor) + 255) & ~size_t(255);
    const size_t chunk_bytes = (size_t(chunks) * sizeof(ps::GradChunk) + 255) & ~size_t(255);
    ps::free_retired();
    void* base = nullptr;
    PS_HIP(ps::dev_malloc(&base, table_bytes + chunk_bytes + ps::kBlocks * sizeof(double)));
    char* const at = static_cast<char*>(base);
    const auto* const tensor_table = reinterpret_cast<const ps::GradTensor*>(at);
    auto* const chunk_table = reinterpret_cast<ps::GradChunk*>(at + table_bytes);
    int rc = PS_OK;
    if (chunks) {
      rc = ps_memcpy_htod(at, table.data(), table.size() * sizeof(ps::GradTensor));
      if (rc == PS_OK) rc = ps::build_chunks(tensor_table, uint32_t(table.size()), chunk_table,
                                             uint32_t(chunks));
    }
    ps_grad_list* l = rc == PS_OK ? new (std::nothrow) ps_grad_list : nullptr;
    if (!l) {
      ps::dev_free(base);
      return rc != PS_OK ? rc : ps::fail(PS_ERR_RUNTIME, "ps_grad_list_create: out of memory");
    }
    l->tables = base;
    l->grads.tensors = tensor_table;
    l->grads.chunks = chunk_table;
    l->grads.chunk_count = uint32_t(chunks);
    l->grads.in_place = in_place;
    l->sums = reinterpret_cast<double*>(at + table_bytes + chunk_bytes);
    l->blocks = std::min(uint32_t(chunks), ps::kBlocks);
    l->read = std::move(read);
    l->written = std::move(written);
    *list = l;
    return PS_OK;
  } catch (const std::exception& e) {
    return ps::fail(PS_ERR_RUNTIME, std::string("ps_grad_list_create: ") + e.what());
  }
}

void ps_grad_list_destroy(ps_grad_list* list) {
  if (!list) return;
  std::lock_guard<std::mutex> lock(ps::g_retired_mu);
  list->retired = std::exchange(ps::g_retired, list);
}

int ps_grad_norm(ps_grad_list* list, float grad_scale, float* norm, ps_stream_t stream) {
  PS_CHECK_ARG(list && norm, "ps_grad_norm: null argument");
  PS_CHECK_ARG(!list->read.meets(norm, sizeof(float)),
               "ps_grad_norm: the norm lies in a gradient");
  const hipStream_t st = ps::to_hip(stream);
  const int rc = ps::launch_norm(*list, st);
  if (rc != PS_OK) return rc;
  ps::norm_join_kernel<<<1, ps::kClipThreads, 0, st>>>(list->sums, list->blocks,
                                                       double(grad_scale), norm);
  PS_LAUNCHED();
  return PS_OK;
}

int ps_clip_grads(ps_grad_list* list, float max_norm, float grad_scale, const float* norm,
                  ps_stream_t stream) {
  PS_CHECK_ARG(list && norm, "ps_clip_grads: null argument");
  PS_CHECK_ARG(!list->written.meets(norm, sizeof(float)),
               "ps_clip_grads: the norm lies in an output");
  PS_CHECK_ARG(max_norm >= 0.f, "ps_clip_grads: the bound is not a number from 0 up");
  if (!list->blocks) return PS_OK;
  return ps::launch_clip(*list, list->blocks, nullptr, max_norm, grad_scale,
                         const_cast<float*>(norm), ps::to_hip(stream));
}

int ps_clip_grad_norm(ps_grad_list* list, float max_norm, float grad_scale, float* norm,
                      ps_stream_t stream) {
  PS_CHECK_ARG(list && norm, "ps_clip_grad_norm: null argument");
  PS_CHECK_ARG(!list->read.meets(norm, sizeof(float)) &&
                   !list->written.meets(norm, sizeof(float)),
               "ps_clip_grad_norm: the norm lies in a gradient or an output");
  PS_CHECK_ARG(max_norm >= 0.f, "ps_clip_grad_norm: the bound is not a number from 0 up");
  const hipStream_t st = ps::to_hip(stream);
  const int rc = ps::launch_norm(*list, st);
  if (rc != PS_OK) return rc;
  return ps::launch_clip(*list, std::max(list->blocks, 1u), list->sums, max_norm, grad_scale,
                         norm, st);
}

}  // extern "C"
