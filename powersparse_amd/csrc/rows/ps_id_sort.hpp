// Stable counting sort of ids, one pass per digit, for the row operators: ids
// become keys below a limit (ids out of range take the limit itself, so they
// sort last), and a pass puts the elements of one digit after another's.
//
// A tile is ranked wave by wave: the lanes of 64 consecutive elements that hold
// the same digit are found with one ballot per bit, an element's rank is (its
// digit's count in the wave's earlier steps) + (lower lanes with that digit). No
// atomics decide a place, so equal keys keep their order.
//
// Launches, at some 5 us each, are what a sort of this size costs. One tile
// takes one for all digits, the elements staying in LDS. More tiles take two a
// digit: one counts every tile's digits, and the next one's workgroups each add
// up the counts that precede their own: of every tile while they are few, of
// groups of tiles and of the tiles of one's own group beyond. The tables of
// very many tiles go through the device scan between the two.
#pragma once

#include "ps_common.hpp"

namespace ps {

constexpr int kIdThreads = 1024;
constexpr int kIdItems = 4;  // per thread, at most (one tile of eight for 8192 ids: 33.0
                             // us, two launches a digit: 25.4; 4096 ids 22.8 in one tile)
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
// Sorted pairs: x the key, y the value (where the element was).
struct PairSource {
  const uint2* pairs;
  __device__ __forceinline__ uint32_t key(uint32_t i) const { return pairs[i].x; }
  __device__ __forceinline__ uint32_t value(uint32_t i) const { return pairs[i].y; }
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

// Tiles up to which every workgroup adds up all tiles' counts, and up to which
// it does so by groups of kGroupTiles, whose clearing is a launch of its own
// (262,147 ids below 50,021: 33 us as 129 tiles in groups, 28 one by one).
constexpr uint32_t kFewTiles = 192, kGroupTiles = 32, kGroupedTiles = 1024;
constexpr int kIdWaves = kIdThreads / kWave;

// Index in the tile of item r of this thread, of `items` items a thread.
__device__ __forceinline__ uint32_t tile_item(int r, int items) {
  return (threadIdx.x / kWave) * (items * kWave) + r * kWave + lane_id();
}

// The waves' digit counts in cnt (bins per wave) and the items' ranks among
// their wave's; `valid` elements from the tile's start. Other waves may read cnt
// after a barrier.
__device__ __forceinline__ void rank_tile(const uint32_t (&key)[kIdItems], uint32_t valid,
                                          int items, const Digit& dg, uint16_t* cnt,
                                          uint32_t (&loc)[kIdItems]) {
  const int lane = lane_id();
  const uint32_t mask = (1u << dg.bits) - 1u;
  const uint64_t lower = (uint64_t(1) << lane) - 1u;
  uint16_t* mine = cnt + (threadIdx.x / kWave) * dg.bins;
  for (int b = lane; b < dg.bins; b += kWave) mine[b] = 0;
  wave_lds_sync();
#pragma unroll
  for (int r = 0; r < kIdItems; ++r) {
    if (r >= items) break;
    const bool in = tile_item(r, items) < valid;
    const uint32_t d = (key[r] >> dg.shift) & mask;
    uint64_t peers = __ballot(in);
    for (int b = 0; b < dg.bits; ++b) {
      const bool one = (d >> b) & 1u;
      const uint64_t m = __ballot(one);
      peers &= one ? m : ~m;
    }
    const uint32_t before = mine[d];
    loc[r] = before + uint32_t(__popcll(peers & lower));
    wave_lds_sync();
    // the highest lane of each digit advances the wave's counter
    if (in && (peers >> lane) == 1u) mine[d] = uint16_t(before + uint32_t(__popcll(peers)));
    wave_lds_sync();
  }
}

// Turns bin b's counts into the waves' offsets in it; returns its total.
__device__ __forceinline__ uint32_t wave_offsets(uint16_t* cnt, int bins, int b) {
  uint32_t c[kIdWaves], total = 0;
#pragma unroll
  for (int q = 0; q < kIdWaves; ++q) c[q] = cnt[q * bins + b];
#pragma unroll
  for (int q = 0; q < kIdWaves; ++q) {
    cnt[q * bins + b] = uint16_t(total);
    total += c[q];
  }
  return total;
}

// In place exclusive scan of v[0 .. bins), bins <= 2 * kIdThreads; begins and
// ends with a barrier.
__device__ __forceinline__ void scan_bins(uint32_t* v, int bins, uint32_t* wave_sum) {
  const int w = threadIdx.x / kWave, lane = lane_id(), b = 2 * threadIdx.x;
  __syncthreads();
  const uint32_t x = b < bins ? v[b] : 0u, y = b + 1 < bins ? v[b + 1] : 0u;
  uint32_t incl = x + y;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t t = uint32_t(__shfl_up(int(incl), d, kWave));
    if (lane >= d) incl += t;
  }
  if (lane == kWave - 1) wave_sum[w] = incl;
  __syncthreads();
  uint32_t first = incl - x - y;
  for (int q = 0; q < w; ++q) first += wave_sum[q];
  if (b < bins) v[b] = first;
  if (b + 1 < bins) v[b + 1] = first + x;
  __syncthreads();
}

__device__ __forceinline__ void clear_share(const ClearOnTheWay& c) {
  for (size_t i = size_t(blockIdx.x) * blockDim.x + threadIdx.x; i < c.count;
       i += size_t(gridDim.x) * blockDim.x)
    c.data[i] = uint4{0, 0, 0, 0};
}

// Counts of a tile in the table, padded to whole 16-byte loads.
__host__ __device__ inline uint32_t table_stride(int bins) { return uint32_t(bins + 3) & ~3u; }

// The count table: counts[tile * tile_stride + bin * bin_stride]; groups: the
// counts of kGroupTiles tiles together (table_stride() apart), cleared before the
// pass, or null.
struct IdTable {
  uint32_t *counts, *groups;
  size_t tile_stride, bin_stride;
};

// Counts of every tile.
template <typename Source>
__global__ __launch_bounds__(kIdThreads) void id_count_kernel(Source src, uint32_t n, int items,
                                                              Digit dg, IdTable table,
                                                              ClearOnTheWay clear) {
  __shared__ uint16_t cnt[kIdWaves * kIdMaxBins];
  const uint32_t tile = items * kIdThreads, base = blockIdx.x * tile, valid = min(n - base, tile);
  uint32_t key[kIdItems], loc[kIdItems];
#pragma unroll
  for (int r = 0; r < kIdItems; ++r)
    key[r] = r < items && tile_item(r, items) < valid ? src.key(base + tile_item(r, items)) : 0u;
  clear_share(clear);
  rank_tile(key, valid, items, dg, cnt, loc);
  __syncthreads();
  for (int b = threadIdx.x; b < dg.bins; b += kIdThreads) {
    const uint32_t c = wave_offsets(cnt, dg.bins, b);
    table.counts[blockIdx.x * table.tile_stride + b * table.bin_stride] = c;
    if (table.groups && c) 
      atomicAdd(&table.groups[blockIdx.x / kGroupTiles * table_stride(dg.bins) + b], c);
  }
}

// Adds rows first, first + step, ... below `count` of a table to `all`, and those
// below `mine` to `before`, for the four bins of one quad.
__device__ __forceinline__ void add_rows(const uint32_t* table, uint32_t quads, uint32_t quad,
                                         uint32_t first, uint32_t step, uint32_t count,
                                         uint32_t mine, uint4& all, uint4& before) {
  constexpr int kRows = 8;
  const uint4* rows = reinterpret_cast<const uint4*>(table) + quad;
  for (uint32_t t0 = first; t0 < count; t0 += kRows * step) {
    uint4 c[kRows];
#pragma unroll
    for (int u = 0; u < kRows; ++u) c[u] = rows[size_t(min(t0 + u * step, count - 1)) * quads];
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const uint32_t t = t0 + u * step;
      const uint32_t in = t < count ? ~0u : 0u, early = t < mine ? in : 0u;
      all.x += c[u].x & in;
      all.y += c[u].y & in;
      all.z += c[u].z & in;
      all.w += c[u].w & in;
      before.x += c[u].x & early;
      before.y += c[u].y & early;
      before.z += c[u].z & early;
      before.w += c[u].w & early;
    }
  }
}

// Places a tile's elements. kScanned: the counts have been scanned.
template <bool kScanned, typename Source, typename Sink>
__global__ __launch_bounds__(kIdThreads) void id_place_kernel(Source src, Sink sink, uint32_t n,
                                                              int items, Digit dg,
                                                              IdTable table) {
  __shared__ uint16_t cnt[kIdWaves * kIdMaxBins];
  __shared__ uint32_t start[kIdMaxBins + 3], ahead[kScanned ? 1 : kIdMaxBins + 3];
  __shared__ uint32_t wave_sum[kIdWaves];
  const uint32_t tile = items * kIdThreads, base = blockIdx.x * tile, valid = min(n - base, tile);
  uint32_t key[kIdItems], value[kIdItems], loc[kIdItems];
#pragma unroll
  for (int r = 0; r < kIdItems; ++r) {
    const bool in = r < items && tile_item(r, items) < valid;
    key[r] = in ? src.key(base + tile_item(r, items)) : 0u;
    value[r] = in ? src.value(base + tile_item(r, items)) : 0u;
  }
  if constexpr (!kScanned) {
    // start: all counts of a bin, ahead: the earlier tiles'. A thread adds up
    // four bins of a share of the rows, several rows' loads under way at once:
    // they were written under other L2s and come from far (one by one they
    // were 6 of the 12 us that 32,768 elements took).
    // Eight rows a thread at least, so that few bins do not meet in LDS.
    const uint32_t quads = table_stride(dg.bins) / 4;
    const uint32_t parts = min(kIdThreads / quads, (gridDim.x + 7) / 8);
    const uint32_t part = threadIdx.x / quads, quad = threadIdx.x - part * quads;
    uint4 all{}, before{};
    if (part < parts) {
      if (table.groups) {
        const uint32_t mine = blockIdx.x / kGroupTiles;
        add_rows(table.groups, quads, quad, part, parts, (gridDim.x - 1) / kGroupTiles + 1, mine,
                 all, before);
        uint4 none{};
        add_rows(table.counts, quads, quad, mine * kGroupTiles + part, parts, blockIdx.x,
                 blockIdx.x, none, before);
      } else {
        add_rows(table.counts, quads, quad, part, parts, gridDim.x, blockIdx.x, all, before);
      }
    }
    for (uint32_t b = threadIdx.x; b < 4 * quads; b += kIdThreads) start[b] = ahead[b] = 0;
    __syncthreads();
    if (part < parts) {
      uint32_t* const to[2] = {start + 4 * quad, ahead + 4 * quad};
      const uint4 from[2] = {all, before};
      for (int k = 0; k < 2; ++k) {
        atomicAdd(to[k], from[k].x);
        atomicAdd(to[k] + 1, from[k].y);
        atomicAdd(to[k] + 2, from[k].z);
        atomicAdd(to[k] + 3, from[k].w);
      }
    }
    scan_bins(start, dg.bins, wave_sum);
  } else {
    for (int b = threadIdx.x; b < dg.bins; b += kIdThreads)
      start[b] = table.counts[blockIdx.x * table.tile_stride + b * table.bin_stride];
  }
  rank_tile(key, valid, items, dg, cnt, loc);
  __syncthreads();
  for (int b = threadIdx.x; b < dg.bins; b += kIdThreads) {
    (void)wave_offsets(cnt, dg.bins, b);
    if (Sink::kStarts && blockIdx.x == 0) sink.bin_start(uint32_t(b), start[b]);
    if constexpr (!kScanned) start[b] += ahead[b];
  }
  __syncthreads();
  const uint32_t mask = (1u << dg.bits) - 1u;
#pragma unroll
  for (int r = 0; r < kIdItems; ++r) {
    if (r < items && tile_item(r, items) < valid) {
      const uint32_t d = (key[r] >> dg.shift) & mask;
      sink.put(start[d] + cnt[(threadIdx.x / kWave) * dg.bins + d] + loc[r], key[r], value[r]);
    }
  }
}

// All passes over one tile: `dg` is the first digit, the others follow it.
template <typename Source, typename Sink>
__global__ __launch_bounds__(kIdThreads) void id_sort_tile_kernel(Source src, Sink sink, uint32_t n,
                                                                  int items, Digit dg, int passes,
                                                                  ClearOnTheWay clear) {
  __shared__ uint16_t cnt[kIdWaves * kIdMaxBins];
  __shared__ uint32_t start[kIdMaxBins];
  __shared__ uint32_t wave_sum[kIdWaves];
  __shared__ uint32_t keys[kIdTile], values[kIdTile];
  uint32_t key[kIdItems], value[kIdItems], loc[kIdItems];
#pragma unroll
  for (int r = 0; r < kIdItems; ++r) {
    const bool in = r < items && tile_item(r, items) < n;
    key[r] = in ? src.key(tile_item(r, items)) : 0u;
    value[r] = in ? src.value(tile_item(r, items)) : 0u;
  }
  clear_share(clear);  // before the last pass, whose puts may mark the cleared bytes
  const uint32_t mask = (1u << dg.bits) - 1u;
  for (int k = 0; k < passes; ++k, dg.shift += dg.bits) {
    rank_tile(key, n, items, dg, cnt, loc);
    __syncthreads();
    for (int b = threadIdx.x; b < dg.bins; b += kIdThreads)
      start[b] = wave_offsets(cnt, dg.bins, b);
    scan_bins(start, dg.bins, wave_sum);
    if (Sink::kStarts && k == passes - 1)
      for (int b = threadIdx.x; b < dg.bins; b += kIdThreads) sink.bin_start(uint32_t(b), start[b]);
#pragma unroll
    for (int r = 0; r < kIdItems; ++r) {
      if (r < items && tile_item(r, items) < n) {
        const uint32_t d = (key[r] >> dg.shift) & mask;
        const uint32_t pos = start[d] + cnt[(threadIdx.x / kWave) * dg.bins + d] + loc[r];
        if (k == passes - 1) {
          sink.put(pos, key[r], value[r]);
        } else {
          keys[pos] = key[r];
          values[pos] = value[r];
        }
      }
    }
    if (k < passes - 1) {
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kIdItems; ++r) {
        const bool in = r < items && tile_item(r, items) < n;
        key[r] = in ? keys[tile_item(r, items)] : 0u;
        value[r] = in ? values[tile_item(r, items)] : 0u;
      }
    }
  }
}

static __global__ void id_clear_kernel(ClearOnTheWay clear) { clear_share(clear); }

// How n elements are cut. Every item of a thread is a step of the ranking,
// every tile a row of counts: as few items as leave no more than kFewTiles
// tiles.
struct IdCut {
  int items;
  uint32_t tiles, groups;  // groups: 0 where they are not used
};
inline IdCut id_cut(long long n) {
  IdCut c{1, 0, 0};
  while (c.items < kIdItems && n > (long long)kFewTiles * kIdThreads * c.items) c.items *= 2;
  const long long tile = (long long)c.items * kIdThreads;
  c.tiles = uint32_t((n + tile - 1) / tile);
  if (c.tiles > kFewTiles && c.tiles <= kGroupedTiles)
    c.groups = (c.tiles + kGroupTiles - 1) / kGroupTiles;
  return c;
}
// The most tiles and groups of any list of up to n elements: where the items a
// thread double the tiles are half of the kFewTiles before, and beyond
// kGroupedTiles there are no groups. What callers are asked for is sized by it,
// so that a workspace for n does for fewer.
inline IdCut id_cut_most(long long n) {
  IdCut c = id_cut(n);
  if (c.items > 1 && c.tiles < kFewTiles) c.tiles = kFewTiles;
  if (c.tiles > kGroupedTiles) c.groups = kGroupedTiles / kGroupTiles;
  return c;
}

// The workspace of a sort's passes: the count table and its scan, and, to be
// cleared before the first pass, the groups of every pass.
inline size_t id_sort_table_bytes(const IdCut& cut, int bins) {
  const size_t table = size_t(cut.tiles) * table_stride(bins);
  return ((table * 4 + 255) & ~size_t(255)) + ps_scan_workspace_bytes(table);
}
inline size_t id_sort_group_bytes(const IdCut& cut, int bins) {
  return size_t(cut.groups) * table_stride(bins) * 4;
}

// One pass over several tiles: n elements of src by digit dg into sink. table:
// id_sort_table_bytes() of id_cut(n) and dg.bins, groups: id_sort_group_bytes()
// cleared ones for this pass alone. `clear` is done by the first launch.
template <typename Source, typename Sink>
int id_sort_pass(const Source& src, const Sink& sink, uint32_t n, const Digit& dg, void* table,
                 void* groups, const ClearOnTheWay& clear, hipStream_t stream) {
  const IdCut cut = id_cut(n);
  uint32_t* counts = static_cast<uint32_t*>(table);
  const size_t entries = size_t(cut.tiles) * size_t(dg.bins);
  const bool scanned = cut.tiles > kGroupedTiles;
  const IdTable t{counts, cut.groups ? static_cast<uint32_t*>(groups) : nullptr,
                  scanned ? 1 : table_stride(dg.bins), scanned ? size_t(cut.tiles) : 1};
  id_count_kernel<<<cut.tiles, kIdThreads, 0, stream>>>(src, n, cut.items, dg, t, clear);
  PS_LAUNCHED();
  if (scanned) {
    const int rc = ps_exclusive_scan_u32(
        counts, counts, entries, static_cast<char*>(table) + ((entries * 4 + 255) & ~size_t(255)),
        reinterpret_cast<ps_stream_t>(stream));
    if (rc != PS_OK) return rc;
    id_place_kernel<true><<<cut.tiles, kIdThreads, 0, stream>>>(src, sink, n, cut.items, dg, t);
  } else {
    id_place_kernel<false><<<cut.tiles, kIdThreads, 0, stream>>>(src, sink, n, cut.items, dg, t);
  }
  PS_LAUNCHED();
  return PS_OK;
}

inline int id_clear(const ClearOnTheWay& clear, hipStream_t stream) {
  const size_t blocks = (clear.count + 255) / 256;
  id_clear_kernel<<<unsigned(blocks < 1024 ? blocks : 1024), 256, 0, stream>>>(clear);
  PS_LAUNCHED();
  return PS_OK;
}

// The whole sort when n fits one tile of kIdTile elements.
template <typename Source, typename Sink>
int id_sort_tile(const Source& src, const Sink& sink, uint32_t n, const Digit& first, int passes,
                 const ClearOnTheWay& clear, hipStream_t stream) {
  const int items = n ? int((n + kIdThreads - 1) / kIdThreads) : 1;
  id_sort_tile_kernel<<<1, kIdThreads, 0, stream>>>(src, sink, n, items, first, passes, clear);
  PS_LAUNCHED();
  return PS_OK;
}

}  // namespace ps
