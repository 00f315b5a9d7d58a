// Shared parts of the row operators (powersparse_rows.h): element types,
// 16-byte row accesses, the item -> (row, column) map and argument checks.
//
// A row of `cols` elements is moved in pieces of N (16 bytes of the wider
// type). An item is one piece of one row; items are numbered row by row and
// dealt to threads in order, so a wave's accesses are contiguous for every
// width. The last piece of a row ends with the row and overlaps the one before
// it when N does not divide cols: both write the same values there, and no row
// needs element-sized accesses. Only rows shorter than N take pieces of one
// element. Pieces are aligned to their element only, which global memory
// accesses of any width allow.
#pragma once

#include <initializer_list>

#include "powersparse_rows.h"
#include "ps_common.hpp"

namespace ps {

using f32 = float;
using f16 = _Float16;
using bf16 = __bf16;

template <typename T, int N>
struct PieceOf {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <int N>
using Floats = typename PieceOf<float, N>::type;

template <int N, typename T>
__device__ __forceinline__ Floats<N> load_piece(const T* p) {
  if constexpr (N == 1) {
    Floats<1> f;
    f[0] = float(*p);
    return f;
  } else {
    const auto v = *reinterpret_cast<const typename PieceOf<T, N>::type*>(p);
    return __builtin_convertvector(v, Floats<N>);
  }
}

// kStream: with the non-temporal hint (see streamed()).
template <int N, bool kStream = false, typename T>
__device__ __forceinline__ void store_piece(T* p, const Floats<N>& f) {
  if constexpr (N == 1) {
    *p = T(f[0]);
  } else {
    using V = typename PieceOf<T, N>::type;
    const V v = __builtin_convertvector(f, V);
    if constexpr (kStream)
      __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
    else
      *reinterpret_cast<V*>(p) = v;
  }
}

// A matrix as the kernels read it.
template <typename T>
struct Mat {
  T* data;
  long long rows, ld;
  __device__ __forceinline__ T* at(long long r, int c) const { return data + r * ld + c; }
};

// x / d and x % d for x < 2^31, d >= 1, by a multiplication (Granlund and
// Montgomery 1994): m = ceil(2^(32 + s) / d) - 2^32 with 2^(s-1) < d <= 2^s.
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t divisor) : d(divisor), m(0), s(0) {
    while ((uint64_t(1) << s) < d) ++s;
    m = uint32_t(((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t x) const {
    const uint32_t t = __umulhi(x, m);
    return uint32_t((uint64_t(t) + x) >> s);
  }
};

// Pieces per row and where piece q begins.
struct Pieces {
  int cols, width;  // width: elements per piece
  FastDiv per_row;
  Pieces(long long cols_, int width_)
      : cols(int(cols_)), width(width_), per_row(uint32_t((cols_ + width_ - 1) / width_)) {}
  __device__ __forceinline__ int begin(int q) const { return min(q * width, cols - width); }
};

constexpr int kRowThreads = 256;

// A launch's share of an operator's items (a launch holds fewer than 2^32
// threads).
struct Items {
  unsigned long long begin, end;
  struct Block {
    unsigned long long first;  // this workgroup's first item
    unsigned long long count;  // items from there to the share's end
  };
  __device__ __forceinline__ Block of_block(uint32_t per_block) const {
    const unsigned long long f = begin + (unsigned long long)blockIdx.x * per_block;
    return {f, end - f};
  }
};

// Item `j` of this workgroup, counted from the workgroup's first item `first`
// (64-bit: items may exceed 2^32), as (row, piece).
struct Item {
  long long row;
  int piece;
};
struct ItemBase {
  long long row;
  uint32_t rest;
  __device__ __forceinline__ ItemBase(unsigned long long first, const Pieces& p)
      : row((long long)(first / p.per_row.d)), rest(uint32_t(first % p.per_row.d)) {}
  __device__ __forceinline__ Item at(uint32_t j, const Pieces& p) const {
    const uint32_t t = rest + j;
    const uint32_t r = p.per_row.div(t);
    return {row + r, int(t - r * p.per_row.d)};
  }
};

// --------------------------------------------------------------- host side

inline size_t dtype_size(int dtype) { return dtype == PS_F32 ? 4 : 2; }
inline bool dtype_valid(int dtype) { return dtype >= PS_F32 && dtype <= PS_BF16; }

// What is wrong with a matrix, or null.
inline const char* rows_error(const ps_rows* m) {
  if (!m) return "null matrix";
  if (!dtype_valid(m->dtype)) return "unknown element type";
  if (m->rows < 0 || m->cols < 1 || m->cols > (1 << 24)) return "bad shape";
  if (m->ld < m->cols) return "row stride shorter than a row";
  if (m->rows && m->ld > (1LL << 48) / m->rows) return "too large";
  if (m->rows && !m->data) return "null data";
  if (reinterpret_cast<uintptr_t>(m->data) % dtype_size(m->dtype)) return "misaligned data";
  return nullptr;
}
inline const char* ids_error(const ps_ids* ids) {
  if (!ids) return "null ids";
  if (ids->type != PS_I32 && ids->type != PS_I64) return "unknown id type";
  if (ids->count < 0 || ids->count > (1LL << 30)) return "bad count";
  if (ids->count && !ids->data) return "null data";
  if (reinterpret_cast<uintptr_t>(ids->data) % (ids->type == PS_I64 ? 8 : 4))
    return "misaligned data";
  return nullptr;
}
#define PS_CHECK_ROWS(m)                                                                       \
  do {                                                                                         \
    if (const char* ps_error_ = ps::rows_error(m))                                             \
      return ps::fail(PS_ERR_INVALID, std::string(__func__) + ": " #m ": " + ps_error_);       \
  } while (0)
#define PS_CHECK_IDS(ids)                                                                      \
  do {                                                                                         \
    if (const char* ps_error_ = ps::ids_error(ids))                                            \
      return ps::fail(PS_ERR_INVALID, std::string(__func__) + ": " #ids ": " + ps_error_);     \
  } while (0)

// Device memory that a call reads or writes: rows of `bytes`, `pitch` apart.
struct Region {
  uintptr_t at;
  size_t rows, bytes, pitch;
  size_t span() const { return rows ? (rows - 1) * pitch + bytes : 0; }
};
inline Region region(const ps_rows* m) {
  const size_t size = dtype_size(m->dtype);
  return {reinterpret_cast<uintptr_t>(m->data), size_t(m->rows), size_t(m->cols) * size,
          size_t(m->ld) * size};
}
inline Region region(const void* p, size_t bytes) {
  return {reinterpret_cast<uintptr_t>(p), p && bytes ? size_t(1) : 0, bytes, bytes};
}
inline Region region(const ps_ids* ids) {
  return region(ids->data, size_t(ids->count) * (ids->type == PS_I64 ? 8 : 4));
}
// Column ranges of one wider matrix share its memory range and no byte.
inline bool overlap(const Region& a, const Region& b) {
  if (!a.span() || !b.span() || a.at >= b.at + b.span() || b.at >= a.at + a.span()) return false;
  // a single row's stride says nothing
  const size_t pitch = a.rows == 1 ? b.pitch : a.pitch;
  if ((a.rows > 1 && b.rows > 1 && a.pitch != b.pitch) || (a.rows == 1 && b.rows == 1)) return true;
  const size_t apart =
      a.at <= b.at ? (b.at - a.at) % pitch : (pitch - (a.at - b.at) % pitch) % pitch;
  return apart < a.bytes || apart + b.bytes > pitch;
}
// Whether something written meets anything else of the call. Places to write are
// taken from ids, counts and positions: what changed them under a kernel would
// send it anywhere.
inline bool overlap(const Region& written, std::initializer_list<Region> others) {
  for (const Region& o : others)
    if (overlap(written, o)) return true;
  return false;
}

template <typename T>
inline Mat<T> mat(const ps_rows* m) {
  return {static_cast<T*>(m->data), m->rows, m->ld};
}

// Calls f(T{}) with the element type of `dtype`.
template <typename F>
inline int with_dtype(int dtype, F&& f) {
  if (dtype == PS_F32) return f(f32{});
  if (dtype == PS_F16) return f(f16{});
  return f(bf16{});
}

// Whether an output is stored with the non-temporal hint: from 32 MB on, what
// the L2s hold together, where lines that have to be written out anyway push
// out those still read, and are written out while the next kernel runs. Plain ->
// hinted, us: lookups of 1,024 BF16 columns, 32 MB 11.8 -> 10.4 (with a kernel
// behind them that reads the output 22.5 -> 23.7), 512 MB 180 -> 147 (358 ->
// 350); 16 MB 7.2 -> 7.1 (12.7 -> 13.7). Sort, dispatch and combination of 16,384
// tokens x 4 x 512 BF16 59 -> 43, x 8 x 4,096 506 -> 459, their gradients 56 ->
// 52 and 689 -> 664. It loses for scattered rows that share lines and would stay
// in the last-level cache (65,536 x 4 x 333 FP16 131 -> 137; lookups into 33 of 96
// FP32 columns, 40 MB 23 -> 31), and gains for such rows that would not (32,768 x 8
// x 333 FP32 215 -> 208; 33 of 40 columns, 264 MB 161 -> 136).
constexpr size_t kStreamBytes = size_t(32) << 20;
// What counts is what a call writes: `written` rows of out at most, without the
// gaps between them.
inline bool streamed(const ps_rows* out, long long written) {
  const long long rows = written < out->rows ? written : out->rows;
  return size_t(rows) * size_t(out->cols) * dtype_size(out->dtype) >= kStreamBytes;
}

// Calls f(flag) with a runtime flag as a constant.
template <typename F>
inline int with_flag(bool flag, F&& f) {
  return flag ? f(std::true_type{}) : f(std::false_type{});
}

// Calls f(N) with the elements per piece of rows of `cols` elements, the wider
// of whose types has kSize bytes, as a constant.
template <int kSize, typename F>
inline int with_width(long long cols, F&& f) {
  constexpr int N = 16 / kSize;
  if (cols >= N) return f(std::integral_constant<int, N>{});
  return f(std::integral_constant<int, 1>{});
}

// Launches f(workgroups, Items) over `items` items, `per_block` for each
// workgroup of up to 1024 threads.
template <typename F>
inline int launch_items(unsigned long long items, uint32_t per_block, F&& f) {
  constexpr unsigned long long kBlocks = 1u << 21;
  for (unsigned long long at = 0; at < items; at += kBlocks * per_block) {
    const unsigned long long left = items - at;
    const unsigned long long blocks = (left + per_block - 1) / per_block;
    f(uint32_t(blocks < kBlocks ? blocks : kBlocks),
      Items{at, blocks < kBlocks ? items : at + kBlocks * per_block});
    PS_LAUNCHED();
  }
  return PS_OK;
}

}  // namespace ps
