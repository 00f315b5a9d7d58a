// What the lists of a model's tensors share (gradients with their norm, AdamW's
// parameters): the table of chunks that a launch walks, the ranges that the
// tensors lie in, and how a list's memory goes back.
#pragma once

#include <algorithm>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

#include "ps_rows.hpp"

namespace ps {

constexpr int kListThreads = 256;
// Elements of a chunk. The workgroups go through the chunks side by side, so
// small chunks keep what they touch at one time together: clipping 800 M BF16
// elements into FP32 took 951 us with 4096, 984 with 8192, 1089 with 32,768,
// 992 with 2048.
constexpr long long kChunk = 4096;

struct Chunk {
  uint32_t tensor, index;  // elements [index * kChunk, ...) of the tensor
};

// The chunk table: the tensor (with first_chunk) that chunk q is of, by bisection.
template <typename Tensor>
__global__ __launch_bounds__(kListThreads) void chunk_kernel(const Tensor* __restrict__ tensors,
                                                             uint32_t tensor_count,
                                                             Chunk* __restrict__ chunks,
                                                             uint32_t chunk_count) {
  const uint32_t q = blockIdx.x * kListThreads + threadIdx.x;
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

// Memory that a list reads or writes: ranges that do not meet, in order.
class Ranges {
 public:
  void add(const void* p, size_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    ranges_.push_back({at, at + bytes});
  }
  // Puts them in order and joins those that meet. False: two shared a byte.
  bool close() {
    std::sort(ranges_.begin(), ranges_.end(),
              [](const Range& a, const Range& b) { return a.begin < b.begin; });
    size_t kept = 0;
    bool apart = true;
    for (const Range& r : ranges_) {
      apart = apart && !(kept && r.begin < ranges_[kept - 1].end);
      if (kept && r.begin <= ranges_[kept - 1].end)
        ranges_[kept - 1].end = std::max(ranges_[kept - 1].end, r.end);
      else
        ranges_[kept++] = r;
    }
    ranges_.resize(kept);
    return apart;
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

// A list's device memory. Destroyed lists wait for the next list that is made,
// which waits for the device anyway: freeing waits for it and is refused while
// any stream is captured (the capture is lost), and a list may go at any time,
// from a garbage collector too.
struct TensorTables {
  void* tables = nullptr;
  TensorTables* retired = nullptr;  // the next destroyed list
  virtual ~TensorTables() { dev_free(tables); }
};

class RetiredLists {
 public:
  void retire(TensorTables* list) {
    std::lock_guard<std::mutex> lock(mu_);
    list->retired = std::exchange(first_, list);
  }
  void free() {
    TensorTables* list;
    {
      std::lock_guard<std::mutex> lock(mu_);
      list = std::exchange(first_, nullptr);
    }
    while (list) delete std::exchange(list, list->retired);
  }

 private:
  std::mutex mu_;
  TensorTables* first_ = nullptr;
};
inline RetiredLists g_retired_lists;

// Room for the tensor table, the chunk table and `more` bytes in one block, the
// first two filled; waits for the device.
template <typename Tensor>
struct ListTables {
  const Tensor* tensors = nullptr;
  const Chunk* chunks = nullptr;
  void* more = nullptr;
};
template <typename Tensor>
inline int make_list_tables(const std::vector<Tensor>& table, uint32_t chunk_count, size_t more,
                            void** block, ListTables<Tensor>* out) {
  const size_t table_bytes = (table.size() * sizeof(Tensor) + 255) & ~size_t(255);
  const size_t chunk_bytes = (size_t(chunk_count) * sizeof(Chunk) + 255) & ~size_t(255);
  g_retired_lists.free();
  PS_HIP(dev_malloc(block, table_bytes + chunk_bytes + more));
  char* const at = static_cast<char*>(*block);
  out->tensors = reinterpret_cast<const Tensor*>(at);
  auto* const chunks = reinterpret_cast<Chunk*>(at + table_bytes);
  out->chunks = chunks;
  out->more = at + table_bytes + chunk_bytes;
  if (!chunk_count) return PS_OK;
  const int rc = ps_memcpy_htod(at, table.data(), table.size() * sizeof(Tensor));
  if (rc != PS_OK) return rc;
  chunk_kernel<<<(chunk_count + kListThreads - 1) / kListThreads, kListThreads>>>(
      out->tensors, uint32_t(table.size()), chunks, chunk_count);
  PS_LAUNCHED();
  PS_HIP(hipStreamSynchronize(nullptr));
  return PS_OK;
}

}  // namespace ps
