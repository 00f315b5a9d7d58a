// Stable counting sort of ids, one pass per digit, for the row operators: ids
// become keys below a limit (ids out of range take the limit itself, so they
// sort last), and a pass puts the elements of one digit after another's.
//
// A pass over more than one tile counts every tile's digits, scans the counts
// (digit by digit, tile by tile) and places the elements; a single tile does it
// all in one launch. A tile is ranked wave by wave: the lanes of 64 consecutive
// elements that hold the same digit are found with one ballot per bit, an
// element's rank is (its digit's count in the wave's earlier steps) + (lower
// lanes with that digit). No atomics, so equal keys keep their order.
#pragma once

#include "ps_common.hpp"

namespace ps {

constexpr int kIdThreads = 1024;
constexpr int kIdItems = 4;  // per thread
constexpr uint32_t kIdTile = kIdThreads * kIdItems;
constexpr int kIdMaxBins = 1025;  // 1024 digits, or 1024 experts and the dropped slots

// Keys from ids: `limit` for ids outside [0, limit) and for `padding`.
template <typename I>
struct IdSource {
  const I* ids;
  long long limit, padding;
  __device__ __forceinline__ uint32_t key(uint32_t i) const {
    const long long id = ids[i];
    return uint32_t(id >= 0 && id < limit && id != padding ? id : limit);
  }
  __device__ __forceinline__ uint32_t value(uint32_t i) const { return i; }
};
struct PairSource {
  const uint32_t *keys, *values;
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return keys[i]; }
  __device__ __forceinline__ uint32_t value(uint32_t i) const { return values[i]; }
};

// Where the elements of a pass go. `bin_start` gets every digit's first
// position (Sink::kStarts only).
struct PairSink {
  static constexpr bool kStarts = false;
  uint32_t *keys, *values;
  __device__ __forceinline__ void put(uint32_t pos, uint32_t key, uint32_t value) const {
    keys[pos] = key;
    values[pos] = value;
  }
  __device__ __forceinline__ void bin_start(uint32_t, uint32_t) const {}
};

// Bytes cleared by the sort's first launch on the way (16-byte multiple).
struct ClearOnTheWay {
  uint4* data;
  size_t count;  // 16-byte words
};

// One digit of a sort: (key >> shift) & mask, `bins` digits occur, `bits` bits.
struct Digit {
  int shift, bits, bins;
};

template <typename Source>
__device__ __forceinline__ void rank_tile(const Source& src, uint32_t n, const Digit& dg,
                                          uint16_t* cnt, uint32_t (&key)[kIdItems],
                                          uint32_t (&loc)[kIdItems]) {
  const int w = threadIdx.x / kWave, lane = lane_id();
  const uint32_t mask = (1u << dg.bits) - 1u;
  const uint64_t lower = (uint64_t(1) << lane) - 1u;
  uint16_t* mine = cnt + w * dg.bins;
  for (int b = lane; b < dg.bins; b += kWave) mine[b] = 0;
  const uint32_t base = blockIdx.x * kIdTile + w * (kIdItems * kWave) + lane;
#pragma unroll
  for (int r = 0; r < kIdItems; ++r) {
    const uint32_t i = base + r * kWave;
    key[r] = i < n ? src.key(i) : 0u;
  }
  wave_lds_sync();
#pragma unroll
  for (int r = 0; r < kIdItems; ++r) {
    const bool valid = base + r * kWave < n;
    const uint32_t d = (key[r] >> dg.shift) & mask;
    uint64_t peers = __ballot(valid);
    for (int b = 0; b < dg.bits; ++b) {
      const bool one = (d >> b) & 1u;
      const uint64_t m = __ballot(one);
      peers &= one ? m : ~m;
    }
    const uint32_t before = mine[d];
    loc[r] = before + uint32_t(__popcll(peers & lower));
    wave_lds_sync();
    // the highest lane of each digit advances the wave's counter
    if (valid && (peers >> lane) == 1u) mine[d] = uint16_t(before + uint32_t(__popcll(peers)));
    wave_lds_sync();
  }
}

__device__ __forceinline__ void clear_share(const ClearOnTheWay& c) {
  for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < c.count;
       i += size_t(gridDim.x) * blockDim.x)
    c.data[i] = uint4{0, 0, 0, 0};
}

// Counts of every tile: table[digit * tiles + tile].
template <typename Source>
__global__ __launch_bounds__(kIdThreads) void id_count_kernel(Source src, uint32_t n, Digit dg,
                                                              uint32_t* __restrict__ table,
                                                              ClearOnTheWay clear) {
  __shared__ uint16_t cnt[kIdThreads / kWave * kIdMaxBins];
  clear_share(clear);
  uint32_t key[kIdItems], loc[kIdItems];
  rank_tile(src, n, dg, cnt, key, loc);
  __syncthreads();
  for (int b = threadIdx.x; b < dg.bins; b += kIdThreads) {
    uint32_t total = 0;
    for (int q = 0; q < kIdThreads / kWave; ++q) total += cnt[q * dg.bins + b];
    table[size_t(b) * gridDim.x + blockIdx.x] = total;
  }
}

// Places a tile's elements. starts: the scanned counts, or null for a single
// tile, whose own counts are scanned here.
template <typename Source, typename Sink>
__global__ __launch_bounds__(kIdThreads) void id_place_kernel(Source src, Sink sink, uint32_t n,
                                                              Digit dg,
                                                              const uint32_t* __restrict__ starts,
                                                              ClearOnTheWay clear) {
  __shared__ uint16_t cnt[kIdThreads / kWave * kIdMaxBins];
  __shared__ uint32_t start[kIdMaxBins + 1];
  __shared__ uint32_t wave_sum[kIdThreads / kWave];
  constexpr int kWaves = kIdThreads / kWave;
  const int w = threadIdx.x / kWave, lane = lane_id();
  clear_share(clear);
  uint32_t key[kIdItems], loc[kIdItems];
  rank_tile(src, n, dg, cnt, key, loc);
  __syncthreads();
  // counts -> the waves' offsets in their digit; thread t owns digits 2t, 2t + 1
  uint32_t total[2] = {0, 0};
  for (int k = 0; k < 2; ++k) {
    const int b = 2 * int(threadIdx.x) + k;
    if (b < dg.bins)
      for (int q = 0; q < kWaves; ++q) {
        const uint32_t c = cnt[q * dg.bins + b];
        cnt[q * dg.bins + b] = uint16_t(total[k]);
        total[k] += c;
      }
  }
  uint32_t first;
  if (starts) {
    first = 0;
  } else {
    uint32_t incl = total[0] + total[1];
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t t = uint32_t(__shfl_up(int(incl), d, kWave));
      if (lane >= d) incl += t;
    }
    if (lane == kWave - 1) wave_sum[w] = incl;
    __syncthreads();
    first = incl - (total[0] + total[1]);
    for (int q = 0; q < w; ++q) first += wave_sum[q];
  }
  for (int k = 0; k < 2; ++k) {
    const int b = 2 * int(threadIdx.x) + k;
    if (b < dg.bins) {
      const uint32_t s = starts ? starts[size_t(b) * gridDim.x + blockIdx.x] : first;
      start[b] = s;
      if (Sink::kStarts && blockIdx.x == 0) sink.bin_start(uint32_t(b), s);
      first += total[k];
    }
  }
  __syncthreads();
  const uint32_t mask = (1u << dg.bits) - 1u;
  const uint32_t base = blockIdx.x * kIdTile + w * (kIdItems * kWave) + lane;
#pragma unroll
  for (int r = 0; r < kIdItems; ++r) {
    const uint32_t i = base + r * kWave;
    if (i < n) {
      const uint32_t d = (key[r] >> dg.shift) & mask;
      sink.put(start[d] + cnt[w * dg.bins + d] + loc[r], key[r], src.value(i));
    }
  }
}

// Bytes of the count table and its scan for passes over n elements.
inline size_t id_sort_table_bytes(long long n, int bins) {
  const size_t tiles = size_t((n + kIdTile - 1) / kIdTile);
  if (tiles <= 1) return 0;
  const size_t table = tiles * size_t(bins);
  return ((table * 4 + 255) & ~size_t(255)) + ps_scan_workspace_bytes(table);
}

// One pass: n elements of src by digit dg into sink; table holds
// id_sort_table_bytes(n, dg.bins) bytes. `clear` is done by the first launch.
template <typename Source, typename Sink>
int id_sort_pass(const Source& src, const Sink& sink, uint32_t n, const Digit& dg, void* table,
                 const ClearOnTheWay& clear, hipStream_t stream) {
  const uint32_t tiles = n ? (n + kIdTile - 1) / kIdTile : 1;
  if (tiles == 1) {
    id_place_kernel<<<1, kIdThreads, 0, stream>>>(src, sink, n, dg, nullptr, clear);
    PS_LAUNCHED();
    return PS_OK;
  }
  uint32_t* counts = static_cast<uint32_t*>(table);
  const size_t entries = size_t(tiles) * size_t(dg.bins);
  id_count_kernel<<<tiles, kIdThreads, 0, stream>>>(src, n, dg, counts, clear);
  PS_LAUNCHED();
  const int rc = ps_exclusive_scan_u32(counts, counts, entries,
                                       static_cast<char*>(table) + ((entries * 4 + 255) & ~size_t(255)),
                                       reinterpret_cast<ps_stream_t>(stream));
  if (rc != PS_OK) return rc;
  id_place_kernel<<<tiles, kIdThreads, 0, stream>>>(src, sink, n, dg, counts, ClearOnTheWay{});
  PS_LAUNCHED();
  return PS_OK;
}

}  // namespace ps
