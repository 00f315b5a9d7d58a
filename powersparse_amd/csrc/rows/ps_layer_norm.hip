// Layer norm of rows, and its gradients.
//
// A row's mean is taken first and its squared deviations from it second: sums of
// squares alone would cancel where the mean is large against the deviations. A row
// of up to 4,096 pieces (in the gradient 2,048 of 8 elements) stays in the registers
// of kLanes threads, kPieces each, and is read once; these threads go from row to row,
// so weight and bias are loaded once, and in the gradient a thread's columns stay the
// same: it adds up their dweight and dbias in registers and leaves one sum a
// workgroup, which a second launch adds up in order. No atomics: the same bits every
// time.
#include <algorithm>

#include "ps_rows.hpp"

namespace ps {
namespace {

// A weight or bias vector of any type; null: all `otherwise`.
struct Vec {
  const void* data;
  int dtype;
  float otherwise;
  template <int N>
  __device__ __forceinline__ Floats<N> at(int c) const {
    if (!data) return Floats<N>(otherwise);
    if (dtype == PS_F32) return load_piece<N>(static_cast<const f32*>(data) + c);
    if (dtype == PS_F16) return load_piece<N>(static_cast<const f16*>(data) + c);
    return load_piece<N>(static_cast<const bf16*>(data) + c);
  }
};

constexpr int kWideThreads = 1024;

// Sum over the workgroup, in every thread.
template <int kThreads>
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[kThreads / kWave];
  v = lanes_sum<kWave>(v);
  __syncthreads();
  if (lane_id() == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) v += part[w];
  return v;
}

// Whether a row's last piece repeats elements of the one before: the same for
// all rows. Where a thread has several pieces this is asked before their elements
// are compared, which is a quarter of the work (32,768 x 4,096 BF16, 64 threads a
// row: 203 and 101 us); where it has one, asking costs more (1,000,000 x 128 FP32:
// 193 and 209 us).
template <int N>
__device__ __forceinline__ bool repeats(const Pieces& p) {
  return int(p.per_row.d) * N != p.cols;
}
// The elements of piece q that the piece before has not counted.
template <int N, int kPieces, typename F>
__device__ __forceinline__ void each_new(const Pieces& p, int q, F&& f) {
  if (kPieces > 1 && !repeats<N>(p)) {
#pragma unroll
    for (int e = 0; e < N; ++e) f(e);
    return;
  }
  const int seen = q * N - p.begin(q);
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e >= seen) f(e);
}

// Sums over the kLanes threads of a row, in every one of them. part: room for
// them where these are a workgroup; two rooms are used in turn, so that one
// barrier does: a thread that writes a room again has passed the other's.
template <int kLanes>
struct RowParts {
  float of[2][2][kLanes > kWave ? kLanes / kWave : 1];
};
template <int kLanes, int kSums>
__device__ __forceinline__ void row_sums(float (&v)[kSums], RowParts<kLanes>& part, int turn) {
#pragma unroll
  for (int k = 0; k < kSums; ++k) v[k] = lanes_sum<(kLanes < kWave ? kLanes : kWave)>(v[k]);
  if constexpr (kLanes > kWave) {
    if (lane_id() == 0)
#pragma unroll
      for (int k = 0; k < kSums; ++k) part.of[turn][k][threadIdx.x / kWave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSums; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < kLanes / kWave; ++w) v[k] += part.of[turn][k][w];
    }
  }
}

constexpr int threads_of(int lanes) { return lanes > kRowThreads ? lanes : kRowThreads; }

// Bound by memory: x is read and y written once, the weights come from the caches.
// 1,000,000 x 128 FP32: 1.03 GB in 183 us, 5.6 TB/s; 32,768 x 4,096 BF16: 0.54 GB in
// 102 us, 5.3 TB/s. Non-temporal stores gave 1.5%.
template <typename T, typename O, int N, int kLanes, int kPieces>
__global__ __launch_bounds__(threads_of(kLanes)) void layer_norm_kernel(
    Mat<const T> x, Vec weight, Vec bias, float eps, Mat<O> y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, Pieces p) {
  constexpr int kRows = threads_of(kLanes) / kLanes;
  __shared__ RowParts<kLanes> part;
  const int lane = threadIdx.x % kLanes, pieces = int(p.per_row.d);
  using V = typename PieceOf<T, N>::type;
  // What does not fit the registers that are left (1,024 threads have half of 512's)
  // is loaded again for every row: 2,048 x 32,768 BF16 136 and 73 us, but 4,096 x
  // 16,384 FP32, which fit, 105 and 120.
  constexpr bool kHeld = kPieces * N <= (kLanes > 256 ? 16 : 32);
  Floats<N> w[kPieces], b[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int q = i * kLanes + lane;
    if (!kHeld || q >= pieces) continue;
    w[i] = weight.at<N>(p.begin(q));
    b[i] = bias.at<N>(p.begin(q));
  }
  // threads without a row go along: the sums take every lane
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < x.rows;
       r0 += (long long)gridDim.x * kRows) {
    const long long mine = r0 + threadIdx.x / kLanes, r = min(mine, x.rows - 1);
    V v[kPieces];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      if (q < pieces) v[i] = *reinterpret_cast<const V*>(x.at(r, p.begin(q)));
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      const Floats<N> f = __builtin_convertvector(v[i], Floats<N>);
      if (q < pieces) each_new<N, kPieces>(p, q, [&](int e) { s[0] += f[e]; });
    }
    row_sums(s, part, 0);
    const float mean = s[0] / float(p.cols);
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      const Floats<N> f = __builtin_convertvector(v[i], Floats<N>) - mean;
      if (q < pieces) each_new<N, kPieces>(p, q, [&](int e) { s[0] += f[e] * f[e]; });
    }
    row_sums(s, part, 1);
    const float rstd = 1.f / sqrtf(s[0] / float(p.cols) + eps);
    if (mine >= x.rows) continue;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      if (q >= pieces) continue;
      const Floats<N> f = (__builtin_convertvector(v[i], Floats<N>) - mean) * rstd;
      if constexpr (!kHeld) {
        w[i] = weight.at<N>(p.begin(q));
        b[i] = bias.at<N>(p.begin(q));
      }
      store_piece<N>(y.at(r, p.begin(q)), f * w[i] + b[i]);
    }
    if (lane == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
  }
}

// Both row sums are joined in one step. parts: see layer_norm_columns_kernel; null:
// not wanted. Bound by memory: 16,384 x 4,096 of FP32 with BF16 gradients 0.71 GB in
// 125 us, 5.6 TB/s, of which the parts are 34 MB; 30,011 x 333 FP32 0.125 GB in 23
// us, 5.5 TB/s.
template <typename T, typename O, int N, int kLanes, int kPieces>
__global__ __launch_bounds__(threads_of(kLanes)) void layer_norm_grad_kernel(
    Mat<const O> dy, Mat<const T> x, Vec weight, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, Mat<T> dx, float* __restrict__ parts, Pieces p) {
  constexpr int kThreads = threads_of(kLanes), kRows = kThreads / kLanes;
  __shared__ RowParts<kLanes> part;
  const int lane = threadIdx.x % kLanes, pieces = int(p.per_row.d);
  using V = typename PieceOf<T, N>::type;
  using G = typename PieceOf<O, N>::type;
  Floats<N> w[kPieces], dw[kPieces], db[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int q = i * kLanes + lane;
    dw[i] = db[i] = 0.f;
    if (q < pieces) w[i] = weight.at<N>(p.begin(q));
  }
  int turn = 0;
  for (long long r0 = (long long)blockIdx.x * kRows; r0 < x.rows;
       r0 += (long long)gridDim.x * kRows) {
    const long long mine = r0 + threadIdx.x / kLanes, r = min(mine, x.rows - 1);
    const float mean = mean_in[r], rstd = rstd_in[r];
    V v[kPieces];
    G g[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      if (q >= pieces) continue;
      v[i] = *reinterpret_cast<const V*>(x.at(r, p.begin(q)));
      g[i] = *reinterpret_cast<const G*>(dy.at(r, p.begin(q)));
    }
    float s[2] = {0.f, 0.f};  // of g and of g * xh
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      if (q >= pieces || mine >= x.rows) continue;
      const Floats<N> xh = (__builtin_convertvector(v[i], Floats<N>) - mean) * rstd;
      const Floats<N> f = __builtin_convertvector(g[i], Floats<N>), gw = f * w[i];
      dw[i] += f * xh;
      db[i] += f;
      each_new<N, kPieces>(p, q, [&](int e) {
        s[0] += gw[e];
        s[1] += gw[e] * xh[e];
      });
    }
    row_sums(s, part, turn);
    turn ^= 1;
    const float mean_g = s[0] / float(p.cols), mean_gx = s[1] / float(p.cols);
    if (mine >= x.rows) continue;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      if (q >= pieces) continue;
      const Floats<N> xh = (__builtin_convertvector(v[i], Floats<N>) - mean) * rstd;
      const Floats<N> gw = __builtin_convertvector(g[i], Floats<N>) * w[i];
      store_piece<N>(dx.at(r, p.begin(q)), rstd * (gw - mean_g - xh * mean_gx));
    }
  }
  if (!parts) return;
  float* const to = parts + size_t(blockIdx.x) * 2 * p.cols;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int q = i * kLanes + lane;
      if (q >= pieces) continue;
      const int c = p.begin(q);
      if (!repeats<N>(p)) {
        store_piece<N>(to + c, dw[i]);
        store_piece<N>(to + p.cols + c, db[i]);
        continue;
      }
      each_new<N, kPieces>(p, q, [&](int e) {
        to[c + e] = dw[i][e];
        to[p.cols + c + e] = db[i][e];
      });
    }
  } else {
    // The rows of the workgroup, in order: element by element through shared memory.
    __shared__ float rows[kThreads * N];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < N; ++e) rows[threadIdx.x * N + e] = half ? db[i][e] : dw[i][e];
        __syncthreads();
        for (int at = threadIdx.x; at < kLanes * N; at += kThreads) {
          const int q = i * kLanes + at / N;
          if (q >= pieces) continue;
          const int c = p.begin(q) + at % N;
          if (c < q * N) continue;  // the piece before has it
          float sum = 0.f;
#pragma unroll
          for (int m = 0; m < kRows; ++m) sum += rows[m * kLanes * N + at];
          to[half * p.cols + c] = sum;
        }
      }
    }
  }
}

// Rows of any width: a workgroup a row, which is read three times. 2,048 x 50,000 BF16,
// 0.41 GB to be read and written once, in 144 us, FP32 249: the caches have the row for
// its later reads.
template <typename T, typename O, int N>
__global__ __launch_bounds__(kWideThreads) void layer_norm_wide_kernel(
    Mat<const T> x, Vec weight, Vec bias, float eps, Mat<O> y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, Pieces p) {
  const int pieces = int(p.per_row.d);
  for (long long r = blockIdx.x; r < x.rows; r += gridDim.x) {
    float s = 0.f;
    for (int q = threadIdx.x; q < pieces; q += kWideThreads) {
      const Floats<N> v = load_piece<N>(x.at(r, p.begin(q)));
      each_new<N, 2>(p, q, [&](int e) { s += v[e]; });
    }
    const float mean = block_sum<kWideThreads>(s) / float(p.cols);
    s = 0.f;
    for (int q = threadIdx.x; q < pieces; q += kWideThreads) {
      const Floats<N> v = load_piece<N>(x.at(r, p.begin(q))) - mean;
      each_new<N, 2>(p, q, [&](int e) { s += v[e] * v[e]; });
    }
    const float rstd = 1.f / sqrtf(block_sum<kWideThreads>(s) / float(p.cols) + eps);
    for (int q = threadIdx.x; q < pieces; q += kWideThreads) {
      const int c = p.begin(q);
      const Floats<N> v = (load_piece<N>(x.at(r, c)) - mean) * rstd;
      store_piece<N>(y.at(r, c), v * weight.at<N>(c) + bias.at<N>(c));
    }
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
  }
}

// dx of rows of any width: a workgroup a row, which is read twice; the sums over the
// rows read all a third time. 2,048 x 50,000 BF16 with them, 0.61 GB to be read and
// written once, 287 us, FP32 513.
template <typename T, typename O, int N>
__global__ __launch_bounds__(kWideThreads) void layer_norm_grad_wide_kernel(
    Mat<const O> dy, Mat<const T> x, Vec weight, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, Mat<T> dx, Pieces p) {
  const int pieces = int(p.per_row.d);
  for (long long r = blockIdx.x; r < x.rows; r += gridDim.x) {
    const float mean = mean_in[r], rstd = rstd_in[r];
    float s = 0.f, sx = 0.f;
    for (int q = threadIdx.x; q < pieces; q += kWideThreads) {
      const int c = p.begin(q);
      const Floats<N> g = load_piece<N>(dy.at(r, c)) * weight.at<N>(c);
      const Floats<N> xh = (load_piece<N>(x.at(r, c)) - mean) * rstd;
      each_new<N, 2>(p, q, [&](int e) {
        s += g[e];
        sx += g[e] * xh[e];
      });
    }
    s = block_sum<kWideThreads>(s) / float(p.cols);
    sx = block_sum<kWideThreads>(sx) / float(p.cols);
    for (int q = threadIdx.x; q < pieces; q += kWideThreads) {
      const int c = p.begin(q);
      const Floats<N> g = load_piece<N>(dy.at(r, c)) * weight.at<N>(c);
      const Floats<N> xh = (load_piece<N>(x.at(r, c)) - mean) * rstd;
      store_piece<N>(dx.at(r, c), rstd * (g - s - xh * sx));
    }
  }
}

// Parts of the sums over the rows: one piece of every row of a range a thread.
// parts holds for each range dweight's sums and then dbias's.
template <typename T, typename O, int N>
__global__ __launch_bounds__(kRowThreads) void layer_norm_columns_kernel(
    Mat<const O> dy, Mat<const T> x, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, float* __restrict__ parts, Pieces p) {
  const int q = blockIdx.x * kRowThreads + threadIdx.x;
  if (q >= int(p.per_row.d)) return;
  const int c = p.begin(q);
  Floats<N> dw = 0.f, db = 0.f;
  for (long long r = blockIdx.y; r < x.rows; r += gridDim.y) {
    const Floats<N> g = load_piece<N>(dy.at(r, c));
    dw += g * ((load_piece<N>(x.at(r, c)) - mean_in[r]) * rstd_in[r]);
    db += g;
  }
  float* const to = parts + size_t(blockIdx.y) * 2 * p.cols + c;
  each_new<N, 2>(p, q, [&](int e) {
    to[e] = dw[e];
    to[p.cols + e] = db[e];
  });
}

// Where the sums over the rows go; null data: not wanted.
struct VecOut {
  void* data;
  int dtype;
  __device__ __forceinline__ void put(int c, float v, bool add) const {
    if (dtype == PS_F32)
      put_as(static_cast<f32*>(data) + c, v, add);
    else if (dtype == PS_F16)
      put_as(static_cast<f16*>(data) + c, v, add);
    else
      put_as(static_cast<bf16*>(data) + c, v, add);
  }
  template <typename T>
  static __device__ __forceinline__ void put_as(T* p, float v, bool add) {
    *p = T(add ? float(*p) + v : v);
  }
};

// The parts added up: 32 columns a workgroup, 32 threads each, with eight parts
// under way at once (one after another they cost 35 us for 1,024 parts of 333
// columns, whose few workgroups have nothing else to wait behind). The columns of
// dweight first, then dbias's.
constexpr int kJoinCols = 32, kJoinLanes = 32, kJoinAhead = 8;
constexpr int kJoinThreads = kJoinCols * kJoinLanes;
__global__ __launch_bounds__(kJoinThreads) void layer_norm_join_kernel(
    const float* __restrict__ parts, int part_count, int cols, VecOut dweight, VecOut dbias,
    bool add) {
  __shared__ float sums[kJoinLanes][kJoinCols];
  const int lane = threadIdx.x / kJoinCols, i = threadIdx.x % kJoinCols;
  const long long c = (long long)blockIdx.x * kJoinCols + i;
  float s = 0.f;
  if (c < 2LL * cols) {
    for (int k0 = lane; k0 < part_count; k0 += kJoinLanes * kJoinAhead) {
      float v[kJoinAhead];
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const int k = k0 + j * kJoinLanes;
        v[j] = k < part_count ? parts[size_t(k) * 2 * cols + c] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) s += v[j];
    }
  }
  sums[lane][i] = s;
  __syncthreads();
  if (lane || c >= 2LL * cols) return;
#pragma unroll
  for (int k = 1; k < kJoinLanes; ++k) s += sums[k][i];
  const VecOut& to = c < cols ? dweight : dbias;
  if (to.data) to.put(int(c < cols ? c : c - cols), s, add);
}

// ----------------------------------------------------------------- host side

// Ranges of rows that the sums over them are cut into: enough to fill the
// device, and no more than 32 MB of parts up to 262,144 columns; beyond, 128 bytes a
// column (sixteen ranges), 2 GB for the widest rows.
constexpr long long kParts = 1024, kFewParts = 16, kPartCells = 1 << 22;
long long part_count(long long rows, long long cols) {
  long long n = kPartCells / cols;
  n = n < kFewParts ? kFewParts : n > kParts ? kParts : n;
  return n < rows ? n : rows;
}

// Of them, the workgroups that take `turns` turns in all, eight each where 512 fill
// the device (512 and 1,024, us: 4,096 x 2,048 BF16 21 and 25, 4,096 x 512 8.6 and
// 10.3; with more turns 16,384 x 2,048 47 and 45, 65,536 x 512 FP32 88 and 80).
uint32_t fewer_parts(uint32_t parts, long long turns) {
  return uint32_t(std::min({(long long)parts, turns, std::max(turns / 8, 512LL)}));
}

Vec vec(const ps_rows* m, float otherwise) {
  return m ? Vec{m->data, m->dtype, otherwise} : Vec{nullptr, PS_F32, otherwise};
}
VecOut vec_out(const ps_rows* m) { return m ? VecOut{m->data, m->dtype} : VecOut{nullptr, PS_F32}; }
Region vec_region(const ps_rows* m) { return m ? region(m) : region(nullptr, 0); }
Region per_row(const float* p, const ps_rows* m) {
  return region(p, size_t(m->rows) * sizeof(float));
}

uint32_t wide_blocks(long long rows) { return uint32_t(rows < 4096 ? rows : 4096); }

// Workgroups of the forward pass: as many as the device holds at once, or with
// four turns each, which shares the work out more evenly and still loads the
// weights seldom (2,048, four turns and one turn: 1,000,000 x 128 FP32 193, 187
// and 185 us, 32,768 x 4,096 BF16 106, 99 and 130).
constexpr long long kNormBlocks = 2048, kMostNormBlocks = 1 << 20;
uint32_t norm_blocks(long long rows, int per_block) {
  const long long n = (rows + per_block - 1) / per_block;
  if (n <= kNormBlocks) return uint32_t(n);
  return uint32_t(std::min(std::max(n / 4, kNormBlocks), kMostNormBlocks));
}

// Calls f(lanes, pieces of a lane) for rows of p's pieces, or f(0, 0) for wider
// ones (beyond kMost pieces: the gradient's four of 8 elements would not fit
// 1,024 threads' registers, 472 us for 2,048 x 32,768 BF16, and 172 without).
// `apart`: whether 65 to 256 pieces get a workgroup a row. Forward that is faster
// where few rows leave most of the device idle (8 x 2,048 BF16 3.9 -> 2.9 us, but
// 16,384 x 1,024 12 -> 19), in the gradient, with twice the registers, from 129
// pieces on (16,384 x 2,048 BF16 47.5 -> 44.6; x 1,024 24.5 -> 31). 513 to 1,024
// pieces of 8 elements, 512 threads for 256: 16,384 x 8,192 gradients 168 -> 157;
// of 4 the other way: 16,384 x 4,096 137 -> 129.
template <int N, int kMost, bool kForward, typename F>
int with_lanes(const Pieces& p, bool apart, F&& f) {
  const uint32_t n = p.per_row.d;
  const auto call = [&](auto lanes, auto per) { return f(lanes, per); };
  using std::integral_constant;
  if (n <= 8) return call(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  if constexpr (N > 1) {  // (else fewer than 8)
    if (n <= 16) return call(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (n <= 32) return call(integral_constant<int, 32>{}, integral_constant<int, 1>{});
    if (n <= 64) return call(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (n <= 256 && apart) return call(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    if (n <= 128) return call(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if constexpr (kForward)  // (there the gradient's are apart)
      if (n <= 256) return call(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    if (n <= 512) return call(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    if (n <= 1024)
      return call(integral_constant<int, N == 8 ? 512 : 256>{},
                  integral_constant<int, N == 8 ? 2 : 4>{});
    if (n <= 2048) return call(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    if constexpr (kMost >= 4096)
      if (n <= 4096) return call(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
  }
  return call(integral_constant<int, 0>{}, integral_constant<int, 0>{});
}

}  // namespace
}  // namespace ps

#define PS_CHECK_VECTOR(m, cols_)                                                           \
  do {                                                                                      \
    if (m) {                                                                                \
      PS_CHECK_ROWS(m);                                                                     \
      PS_CHECK_ARG(m->rows == 1 && m->cols == (cols_),                                      \
                   std::string(__func__) + ": " #m " is not one row of x's columns");       \
    }                                                                                       \
  } while (0)

extern "C" {

int ps_layer_norm(const ps_rows* x, const ps_rows* weight, const ps_rows* bias, float eps,
                  const ps_rows* y, float* mean, float* rstd, ps_stream_t stream) {
  PS_CHECK_ROWS(x);
  PS_CHECK_ROWS(y);
  PS_CHECK_ARG(x->rows == y->rows && x->cols == y->cols,
               "ps_layer_norm: x and y differ in shape");
  PS_CHECK_VECTOR(weight, x->cols);
  PS_CHECK_VECTOR(bias, x->cols);
  PS_CHECK_ARG(eps >= 0.f, "ps_layer_norm: eps is not a number from 0 up");
  PS_CHECK_ARG(ps::aligned4(mean) && ps::aligned4(rstd),
               "ps_layer_norm: misaligned mean or rstd");
  const ps::Region in[] = {ps::region(x), ps::vec_region(weight), ps::vec_region(bias)};
  const ps::Region to[] = {ps::region(y), ps::per_row(mean, x), ps::per_row(rstd, x)};
  PS_CHECK_ARG(!ps::overlap(to[0], {in[0], in[1], in[2], to[1], to[2]}) &&
                   !ps::overlap(to[1], {in[0], in[1], in[2], to[2]}) &&
                   !ps::overlap(to[2], {in[0], in[1], in[2]}),
               "ps_layer_norm: an output overlaps another argument");
  if (!x->rows) return PS_OK;
  return ps::with_dtype(x->dtype, [&](auto t) {
    return ps::with_dtype(y->dtype, [&](auto o) {
      using T = decltype(t);
      using O = decltype(o);
      constexpr int kSize = sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O);
      return ps::with_width<kSize>(x->cols, [&](auto n) {
        const ps::Pieces p(x->cols, n);
        return ps::with_lanes<n, 4096, true>(p, x->rows <= 1024, [&](auto lanes, auto per) {
          const auto run = [&](auto kernel, uint32_t blocks, int threads) {
            kernel<<<blocks, threads, 0, ps::to_hip(stream)>>>(
                ps::mat<const T>(x), ps::vec(weight, 1.f), ps::vec(bias, 0.f), eps, ps::mat<O>(y),
                mean, rstd, p);
          };
          if constexpr (lanes == 0) {
            run(ps::layer_norm_wide_kernel<T, O, n>, ps::wide_blocks(x->rows), ps::kWideThreads);
          } else {
            constexpr int kThreads = ps::threads_of(lanes);
            run(ps::layer_norm_kernel<T, O, n, lanes, per>,
                ps::norm_blocks(x->rows, kThreads / lanes), kThreads);
          }
          PS_LAUNCHED();
          return int(PS_OK);
        });
      });
    });
  });
}

size_t ps_layer_norm_grad_workspace_bytes(long long rows, long long cols) {
  if (rows < 0 || rows > (1LL << 48) || cols < 1 || cols > (1 << 24)) return 0;
  // part_count's parts, or more where it rounds down
  const long long most = ps::kParts * cols < ps::kPartCells ? ps::kParts * cols : ps::kPartCells;
  const long long cells = most > ps::kFewParts * cols ? most : ps::kFewParts * cols;
  const long long all = rows < (1 << 24) && rows * cols < cells ? rows * cols : cells;
  return size_t(all < 2 ? 2 : all) * 2 * sizeof(float);
}

int ps_layer_norm_grad(const ps_rows* dy, const ps_rows* x, const ps_rows* weight,
                       const float* mean, const float* rstd, int accumulate, const ps_rows* dx,
                       const ps_rows* dweight, const ps_rows* dbias, void* workspace,
                       size_t workspace_bytes, ps_stream_t stream) {
  PS_CHECK_ROWS(dy);
  PS_CHECK_ROWS(x);
  PS_CHECK_ROWS(dx);
  PS_CHECK_ARG(dy->rows == x->rows && dy->cols == x->cols && dx->rows == x->rows &&
                   dx->cols == x->cols && dx->dtype == x->dtype,
               "ps_layer_norm_grad: dy, x and dx differ in shape, or dx and x in type");
  PS_CHECK_VECTOR(weight, x->cols);
  PS_CHECK_VECTOR(dweight, x->cols);
  PS_CHECK_VECTOR(dbias, x->cols);
  PS_CHECK_ARG((mean && rstd) || !x->rows, "ps_layer_norm_grad: null mean or rstd");
  PS_CHECK_ARG(ps::aligned4(mean) && ps::aligned4(rstd),
               "ps_layer_norm_grad: misaligned mean or rstd");
  const size_t need = ps_layer_norm_grad_workspace_bytes(x->rows, x->cols);
  const bool sums = dweight || dbias;
  PS_CHECK_ARG(!sums || (workspace && ps::aligned16(workspace) && workspace_bytes >= need),
               "ps_layer_norm_grad: workspace too small or misaligned");
  const ps::Region in[] = {ps::region(dy), ps::region(x), ps::vec_region(weight),
                           ps::per_row(mean, x), ps::per_row(rstd, x)};
  const ps::Region to[] = {ps::region(dx), ps::vec_region(dweight), ps::vec_region(dbias),
                           ps::region(sums ? workspace : nullptr, need)};
  for (int i = 0; i < 4; ++i) {
    PS_CHECK_ARG(!ps::overlap(to[i], {in[0], in[1], in[2], in[3], in[4]}),
                 "ps_layer_norm_grad: an output or the workspace overlaps an input");
    for (int k = 0; k < i; ++k)
      PS_CHECK_ARG(!ps::overlap(to[i], to[k]),
                   "ps_layer_norm_grad: outputs and workspace overlap");
  }
  const hipStream_t st = ps::to_hip(stream);
  float* const parts = static_cast<float*>(workspace);
  uint32_t part_count = uint32_t(ps::part_count(x->rows, x->cols));
  if (x->rows) {
    const int rc = ps::with_dtype(x->dtype, [&](auto t) {
      return ps::with_dtype(dy->dtype, [&](auto o) {
        using T = decltype(t);
        using O = decltype(o);
        constexpr int kSize = sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O);
        return ps::with_width<kSize>(x->cols, [&](auto n) {
          const ps::Pieces p(x->cols, n);
          constexpr int kMost = n == 8 ? 2048 : 4096;
          const bool apart = p.per_row.d > 128;
          return ps::with_lanes<n, kMost, false>(p, apart, [&](auto lanes, auto per) {
            if constexpr (lanes == 0) {
              ps::layer_norm_grad_wide_kernel<T, O, n>
                  <<<ps::wide_blocks(x->rows), ps::kWideThreads, 0, st>>>(
                      ps::mat<const O>(dy), ps::mat<const T>(x), ps::vec(weight, 1.f), mean, rstd,
                      ps::mat<T>(dx), p);
              PS_LAUNCHED();
              if (!sums) return int(PS_OK);
              const dim3 grid((p.per_row.d + ps::kRowThreads - 1) / ps::kRowThreads, part_count);
              ps::layer_norm_columns_kernel<T, O, n><<<grid, ps::kRowThreads, 0, st>>>(
                  ps::mat<const O>(dy), ps::mat<const T>(x), mean, rstd, parts, p);
            } else {
              constexpr int kThreads = ps::threads_of(lanes), kRows = kThreads / lanes;
              part_count = ps::fewer_parts(part_count, (x->rows + kRows - 1) / kRows);
              ps::layer_norm_grad_kernel<T, O, n, lanes, per><<<part_count, kThreads, 0, st>>>(
                  ps::mat<const O>(dy), ps::mat<const T>(x), ps::vec(weight, 1.f), mean, rstd,
                  ps::mat<T>(dx), sums ? parts : nullptr, p);
            }
            PS_LAUNCHED();
            return int(PS_OK);
          });
        });
      });
    });
    if (rc != PS_OK) return rc;
  }
  if (sums) {
    const uint32_t blocks = uint32_t((2 * x->cols + ps::kJoinCols - 1) / ps::kJoinCols);
    ps::layer_norm_join_kernel<<<blocks, ps::kJoinThreads, 0, st>>>(
        parts, int(part_count), int(x->cols), ps::vec_out(dweight), ps::vec_out(dbias),
        accumulate != 0);
    PS_LAUNCHED();
  }
  return PS_OK;
}

}  // extern "C"
