// AdamW over many tensors in one launch, with the moments in 32 bits or in 8.
//
// In 8 bits a moment is kept by blocks of 256 elements of a tensor: an E4M3 code
// for each, and one FP32 scale, the block's largest magnitude / 448, E4M3's
// largest value. Of the second moment the square root is kept, which halves the
// range of exponents that the codes have to span.
//
// A moment changes little in a step: by a part in 1000 with beta2 = 0.999, where
// two neighbouring codes are a part in 8 to 16 apart. Rounding to nearest would
// keep every code where it is for good. So the upper of two codes is taken where
// the fraction of the step between them is 1 - u or more, with u the fraction of
// a Weyl sequence, (i * a + t * b) / 2^32 mod 1 for element i in step t: b / 2^32
// is the golden ratio's fraction, so an element's u is spread evenly over the
// steps (Weyl's equidistribution), and its code goes up as often as its moment
// gains a step of the grid; a / 2^32 (the square root of two's fraction) spreads
// it over the elements. Under constant gradients that keeps an element within a step
// of the grid. Under random ones its moves and u have nothing in common, and it walks:
// after 2,000 steps of N(0, 1) gradients with beta2 = 0.999 the roots are off by 15%
// rms, 1.5 steps of the grid and at most 4.6, their mean by 0.6%. What is unbiased in
// the root adds its variance to the square, which is 3.4% too large then and up to
// 3.8% later (10,000 steps); the first moment (beta1 = 0.9) is off by 7% of its size.
// A second moment that is not zero never becomes zero: the step divides by it.
#include <cmath>
#include <limits>

#include "ps_tensor_list.hpp"

namespace ps {

struct AdamTensor {
  void* param;
  const void* grad;
  void *exp_avg, *exp_avg_sq;
  float* scales;  // a pair for each block
  void* copy;
  long long count, first_chunk;
  float decay;
  int param_dtype, grad_dtype, copy_dtype;
};

namespace {

// A workgroup a chunk, which is the next turn's where there are more: 2,048
// workgroups that take turns were 2,226 us for 400 M parameters with FP32 moments
// and 1,341 in 8 bits, 8,192 2,215 and 1,304, one a chunk 2,150 and 1,278.
constexpr uint32_t kAdamBlocks = 1u << 20;
constexpr int kStateBlock = 256;
constexpr uint32_t kByElement = 0x6A09E667u, kByStep = 0x9E3779B9u;

struct Adam {
  const AdamTensor* tensors;
  const Chunk* chunks;
  uint32_t chunk_count;
};

// What a call is given; the device's values instead where a pointer is not null.
struct AdamCall {
  float beta1, one_beta1, beta2, one_beta2, eps, lr;
  double log_beta1, log_beta2;  // 0 beta: -infinity
  float by_mean, by_root;       // by `step`, see AdamStep
  uint32_t step;
  const float* device_lr;
  const int* device_step;
  const float* norm;
  float max_norm, grad_scale;
};
// The same as an element needs it.
struct AdamStep {
  float beta1, one_beta1, beta2, one_beta2, eps, lr;
  float grad_scale, by_mean, by_root;  // 1 / (1 - beta1^t), 1 / sqrt(1 - beta2^t)
  uint32_t weyl;
};

__host__ __device__ inline float mean_factor(double step, double log_beta1) {
  return float(-1.0 / expm1(step * log_beta1));
}
__host__ __device__ inline float root_factor(double step, double log_beta2) {
  return float(1.0 / sqrt(-expm1(step * log_beta2)));
}

// False: the norm is not finite, nothing is to change.
__device__ __forceinline__ bool make_step(const AdamCall& c, AdamStep* s) {
  float scale = c.grad_scale;
  if (c.norm) {
    const float n = *c.norm;
    if (!(fabsf(n) < INFINITY)) return false;
    scale *= fminf(c.max_norm * (1.f / (n + 1e-6f)), 1.f);
  }
  *s = {c.beta1, c.one_beta1, c.beta2,   c.one_beta2, c.eps, c.device_lr ? *c.device_lr : c.lr,
        scale,   c.by_mean,   c.by_root, c.step * kByStep};
  if (c.device_step) {
    const int t = max(*c.device_step, 1);
    s->by_mean = mean_factor(t, c.log_beta1);
    s->by_root = root_factor(t, c.log_beta2);
    s->weyl = uint32_t(t) * kByStep;
  }
  return true;
}

// m and v after the gradient g. Every product and sum is rounded by itself, in the
// order of the formulas: what decides between two codes of an 8-bit moment is then
// the same wherever the formulas are computed in FP32, and so are the codes.
__device__ __forceinline__ void advance(const AdamStep& s, float g, float* m, float* v) {
#pragma clang fp contract(off)
  g = g * s.grad_scale;
  *m = s.beta1 * *m + s.one_beta1 * g;
  *v = s.beta2 * *v + s.one_beta2 * g * g;
}
// x / d, correctly rounded but for the rarest cases, with by = 1 / d: one step of
// Newton's iteration on the quotient (Markstein 1990).
__device__ __forceinline__ float quotient(float x, float d, float by) {
  const float q = x * by;
  return fmaf(fmaf(-q, d, x), by, q);
}
// sqrt(v), correctly rounded but for the rarest cases: the hardware's reciprocal
// root and one step of Newton's iteration on the root (Markstein 1990), numbers
// whose residual would be lost scaled by 2^64.
__device__ __forceinline__ float root_of(float v) {
  const bool small = v < 0x1p-96f;
  const float x = small ? v * 0x1p64f : v;
  const float y = __builtin_amdgcn_rsqf(x);
  const float q = x * y;
  const float r = fmaf(fmaf(-q, q, x), 0.5f * y, q);
  return x > 0.f && x < INFINITY ? (small ? r * 0x1p-32f : r) : v;  // (0, infinity and NaN)
}

// The parameter after a step by m and the root of v. The reciprocal is the
// hardware's, off by a unit in the last place: of the update, which is smaller
// than the parameter it is rounded into.
__device__ __forceinline__ float updated(const AdamStep& s, float decay, float p, float m,
                                         float root) {
  const float up = m * s.by_mean * __builtin_amdgcn_rcpf(fmaf(root, s.by_root, s.eps));
  return fmaf(-s.lr, fmaf(decay, p, up), p);
}

// Addresses from the table, as global memory: the compiler would otherwise take
// them for any kind and wait for shared memory too.
template <typename T>
using Global = __attribute__((address_space(1))) T*;
template <int N, typename T>
__device__ __forceinline__ typename PieceOf<T, N>::type raw(const T* p) {
  return *(Global<const typename PieceOf<T, N>::type>)p;
}
template <int N, typename V>
__device__ __forceinline__ Floats<N> floats(V v) {
  return __builtin_convertvector(v, Floats<N>);
}
template <int N, typename T>
__device__ __forceinline__ void put(T* p, const Floats<N>& f) {
  using V = typename PieceOf<T, N>::type;
  *(Global<V>)p = __builtin_convertvector(f, V);
}

template <int N>
__device__ __forceinline__ void store_copy(const AdamTensor& t, long long i, const Floats<N>& f) {
  if (!t.copy) return;
  if (t.copy_dtype == PS_F32)
    put<N>(static_cast<f32*>(t.copy) + i, f);
  else if (t.copy_dtype == PS_F16)
    put<N>(static_cast<f16*>(t.copy) + i, f);
  else
    put<N>(static_cast<bf16*>(t.copy) + i, f);
}

// N elements of a tensor with moments in 32 bits.
template <int N, typename P, typename G>
struct Elements {
  typename PieceOf<P, N>::type p;
  typename PieceOf<G, N>::type g;
  Floats<N> m, v;
  __device__ __forceinline__ void load(const AdamTensor& t, long long i) {
    p = raw<N>(static_cast<const P*>(t.param) + i);
    g = raw<N>(static_cast<const G*>(t.grad) + i);
    m = raw<N>(static_cast<const float*>(t.exp_avg) + i);
    v = raw<N>(static_cast<const float*>(t.exp_avg_sq) + i);
  }
  __device__ __forceinline__ void step(const AdamTensor& t, const AdamStep& s, long long i) {
    Floats<N> pf = floats<N>(p);
    const Floats<N> gf = floats<N>(g);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float me = m[e], ve = v[e];
      advance(s, gf[e], &me, &ve);
      pf[e] = updated(s, t.decay, pf[e], me, root_of(ve));
      m[e] = me;
      v[e] = ve;
    }
    put<N>(static_cast<P*>(t.param) + i, pf);
    put<N>(static_cast<float*>(t.exp_avg) + i, m);
    put<N>(static_cast<float*>(t.exp_avg_sq) + i, v);
    store_copy<N>(t, i, pf);
  }
};

template <typename P, typename G>
__device__ void chunk_f32(const AdamTensor& t, const AdamStep& s, long long from, uint32_t count) {
  constexpr int N = 4, kTurn = kListThreads * N, kTurns = int(kChunk / kTurn);
  uint32_t i = threadIdx.x * N;
  if (count == kChunk) {  // all loads before the first store, which might be to any of them
    Elements<N, P, G> all[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) all[k].load(t, from + i + k * kTurn);
#pragma unroll
    for (int k = 0; k < kTurns; ++k) all[k].step(t, s, from + i + k * kTurn);
    return;
  }
  for (; i + N <= count; i += kTurn) {
    Elements<N, P, G> some;
    some.load(t, from + i);
    some.step(t, s, from + i);
  }
  for (; i < count; ++i) {
    Elements<1, P, G> one;
    one.load(t, from + i);
    one.step(t, s, from + i);
  }
}

// The largest of magnitudes by their bits, which order as they do; a NaN is above
// all (as floats they would be compared in twice as many instructions).
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ float wave_most(uint32_t v) {
  return __uint_as_float(lanes_all<kWave>(v, [](uint32_t a, uint32_t b) { return max(a, b); }));
}
// Not below FP32's smallest normal number; a NaN stays one.
__device__ __forceinline__ float scale_of(float most) {
  const float s = most * (1.f / 448.f);
  return s < 0x1p-126f ? 0x1p-126f : s;
}

// The magnitude `a` (up to 448) on the grid of E4M3, rounded by u (32 bits). The
// grid has 20 bits of an FP32 significand less; below 2^-6 its steps stay 2^-9, as
// those of FP32 numbers from 2^-6 to 2^-5 with as many bits less do.
__device__ __forceinline__ float on_grid(float a, uint32_t u) {
  const float low = a < 0x1p-6f ? 0x1p-6f : 0.f;
  const uint32_t b = (__float_as_uint(a + low) + (u >> 12)) & 0xFFF00000u;
  return __uint_as_float(min(b, 0x43E00000u)) - low;  // 448
}

// Four elements, or n of them in a tensor's last block (zeros behind them).
template <bool kWhole, typename T>
__device__ __forceinline__ typename PieceOf<T, 4>::type some(const T* p, int n) {
  if (kWhole || n >= 4) return raw<4>(p);
  typename PieceOf<T, 4>::type v = T(0);
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) v[e] = *(Global<const T>)(p + e);
  return v;
}
template <bool kWhole, typename T>
__device__ __forceinline__ void put_some(T* p, typename PieceOf<T, 4>::type v, int n) {
  if (kWhole || n >= 4) {
    *(Global<typename PieceOf<T, 4>::type>)p = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < n) *(Global<T>)(p + e) = v[e];
}
template <bool kWhole, typename T>
__device__ __forceinline__ void put_as(T* p, const Floats<4>& f, int n) {
  put_some<kWhole>(p, __builtin_convertvector(f, typename PieceOf<T, 4>::type), n);
}
using Codes = PieceOf<uint8_t, 4>::type;
__device__ __forceinline__ Floats<4> from_codes(Codes c) {
  const int v = __builtin_bit_cast(int, c);
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(v, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
  return Floats<4>{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ Codes to_codes(const Floats<4>& f) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return __builtin_bit_cast(Codes, __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true));
}

// A block of a tensor with moments in 8 bits: a wave, four elements a lane.
template <typename P, typename G, bool kWhole>
struct Block {
  typename PieceOf<P, 4>::type p;
  typename PieceOf<G, 4>::type g;
  Codes m, r;
  Floats<2> scales;

  // `from`: the block's first element.
  __device__ __forceinline__ void load(const AdamTensor& t, long long from) {
    const long long i = from + lane_id() * 4;
    const int n = left(t, i);
    p = some<kWhole>(static_cast<const P*>(t.param) + i, n);
    g = some<kWhole>(static_cast<const G*>(t.grad) + i, n);
    m = some<kWhole>(static_cast<const uint8_t*>(t.exp_avg) + i, n);
    r = some<kWhole>(static_cast<const uint8_t*>(t.exp_avg_sq) + i, n);
    scales = raw<2>(t.scales + from / kStateBlock * 2);
  }
  __device__ __forceinline__ void step(const AdamTensor& t, const AdamStep& s, long long from) {
    const long long i = from + lane_id() * 4;
    const int n = left(t, i);
    Floats<4> pf = floats<4>(p), mf = from_codes(m) * scales[0], rf = from_codes(r) * scales[1];
    const Floats<4> gf = floats<4>(g);
    uint32_t m_most = 0, r_most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float me = mf[e], ve = rf[e] * rf[e];
      advance(s, gf[e], &me, &ve);
      const float root = root_of(ve);
      pf[e] = updated(s, t.decay, pf[e], me, root);
      mf[e] = me;
      rf[e] = root;
      m_most = max(m_most, magnitude(me));
      r_most = max(r_most, magnitude(root));
    }
    put_as<kWhole>(static_cast<P*>(t.param) + i, pf, n);
    if (t.copy) {
      if (t.copy_dtype == PS_F32)
        put_as<kWhole>(static_cast<f32*>(t.copy) + i, pf, n);
      else if (t.copy_dtype == PS_F16)
        put_as<kWhole>(static_cast<f16*>(t.copy) + i, pf, n);
      else
        put_as<kWhole>(static_cast<bf16*>(t.copy) + i, pf, n);
    }
    const float m_scale = scale_of(wave_most(m_most)), r_scale = scale_of(wave_most(r_most));
    const float by_m = 1.f / m_scale, by_r = 1.f / r_scale;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t u = uint32_t(i + e) * kByElement + s.weyl;
      mf[e] = copysignf(on_grid(quotient(fabsf(mf[e]), m_scale, by_m), u), mf[e]);
      const float least = rf[e] > 0.f ? 0x1p-9f : 0.f;
      const float code = on_grid(quotient(rf[e], r_scale, by_r), u);
      rf[e] = code < least ? least : code;
    }
    put_some<kWhole>(static_cast<uint8_t*>(t.exp_avg) + i, to_codes(mf), n);
    put_some<kWhole>(static_cast<uint8_t*>(t.exp_avg_sq) + i, to_codes(rf), n);
    if (lane_id() == 0) put<2>(t.scales + from / kStateBlock * 2, Floats<2>{m_scale, r_scale});
  }

 private:
  static __device__ __forceinline__ int left(const AdamTensor& t, long long i) {
    return kWhole ? 4 : int(max(0LL, min(4LL, t.count - i)));
  }
};

template <typename P, typename G>
__device__ void chunk_f8(const AdamTensor& t, const AdamStep& s, long long from, uint32_t count) {
  constexpr int kTurn = kListThreads / kWave * kStateBlock, kTurns = int(kChunk / kTurn);
  uint32_t i = threadIdx.x / kWave * kStateBlock;
  if (count == kChunk) {
    Block<P, G, true> all[kTurns];
#pragma unroll
    for (int k = 0; k < kTurns; ++k) all[k].load(t, from + i + k * kTurn);
#pragma unroll
    for (int k = 0; k < kTurns; ++k) all[k].step(t, s, from + i + k * kTurn);
    return;
  }
  for (; i < count; i += kTurn) {
    Block<P, G, false> one;
    one.load(t, from + i);
    one.step(t, s, from + i);
  }
}

template <bool k8, typename P, typename G>
__device__ __forceinline__ void chunk_of(const AdamTensor& t, const AdamStep& s, long long from,
                                         uint32_t count) {
  if constexpr (k8)
    chunk_f8<P, G>(t, s, from, count);
  else
    chunk_f32<P, G>(t, s, from, count);
}
template <bool k8, typename P>
__device__ __forceinline__ void chunk_of(const AdamTensor& t, const AdamStep& s, long long from,
                                         uint32_t count) {
  if (t.grad_dtype == PS_F32)
    chunk_of<k8, P, f32>(t, s, from, count);
  else if (t.grad_dtype == PS_F16)
    chunk_of<k8, P, f16>(t, s, from, count);
  else
    chunk_of<k8, P, bf16>(t, s, from, count);
}

// Bound by memory: 400 M FP32 parameters, BF16 gradients and copies, FP32 moments:
// 11.2 GB in 2,138 us, 5.2 TB/s; moments in 8 bits 6.4 GB in 1,192 us, 5.4 TB/s, with
// as much time's worth of instructions, some 100 an element, under it. With rate and
// step on the device, whose factors every thread computes in 64 bits, 0.4% and 1.5%
// more (captured: 2,087 -> 2,095 and 1,152 -> 1,170).
template <bool k8>
__global__ __launch_bounds__(kListThreads) void adamw_kernel(Adam a, AdamCall call) {
  AdamStep s;
  if (!make_step(call, &s)) return;
  for (uint32_t q = blockIdx.x; q < a.chunk_count; q += gridDim.x) {
    const Chunk ch = a.chunks[q];
    const AdamTensor t = a.tensors[ch.tensor];
    const long long from = (long long)ch.index * kChunk;
    const uint32_t count = uint32_t(min(kChunk, t.count - from));
    if (t.param_dtype == PS_F32)
      chunk_of<k8, f32>(t, s, from, count);
    else if (t.param_dtype == PS_F16)
      chunk_of<k8, f16>(t, s, from, count);
    else
      chunk_of<k8, bf16>(t, s, from, count);
  }
}

static_assert(kChunk % kStateBlock == 0, "a block lies in one chunk");

}  // namespace
}  // namespace ps

// Its tables: tensors, chunks.
struct ps_adamw_list : ps::TensorTables {
  ps::Adam adam{};
  bool in_8_bits = false;
  ps::Ranges written;
};

extern "C" {

int ps_adamw_list_create(int tensors, const ps_adamw_tensor* list, int state_dtype,
                         ps_adamw_list** out) {
  PS_CHECK_ARG(out, "ps_adamw_list_create: null output");
  *out = nullptr;
  PS_CHECK_ARG(tensors >= 0 && tensors <= (1 << 24), "ps_adamw_list_create: bad tensor count");
  PS_CHECK_ARG(!tensors || list, "ps_adamw_list_create: null array");
  PS_CHECK_ARG(state_dtype == PS_F32 || state_dtype == PS_E4M3,
               "ps_adamw_list_create: states are of PS_F32 or PS_E4M3");
  const bool in_8_bits = state_dtype == PS_E4M3;
  try {
    std::vector<ps::AdamTensor> table;
    ps::Ranges written;
    long long total = 0, chunks = 0;
    for (int i = 0; i < tensors; ++i) {
      const ps_adamw_tensor& t = list[i];
      const auto bad = [i](const char* what) {
        return "ps_adamw_list_create: tensor " + std::to_string(i) + ": " + what;
      };
      PS_CHECK_ARG(ps::dtype_valid(t.param_dtype) && ps::dtype_valid(t.grad_dtype) &&
                       (!t.copy || ps::dtype_valid(t.copy_dtype)),
                   bad("unknown element type"));
      PS_CHECK_ARG(t.count >= 0 && t.count <= (1LL << 44) && total <= (1LL << 44),
                   bad("bad count"));
      PS_CHECK_ARG(std::isfinite(t.weight_decay), bad("weight decay is not a number"));
      if (!t.count) continue;
      PS_CHECK_ARG(t.param && t.grad && t.exp_avg && t.exp_avg_sq && (!in_8_bits || t.scales),
                   bad("null data"));
      const size_t state = in_8_bits ? 1 : 4, n = size_t(t.count);
      const size_t blocks = (n + ps::kStateBlock - 1) / ps::kStateBlock;
      const auto misaligned = [](const void* p, size_t size) {
        return reinterpret_cast<uintptr_t>(p) % size != 0;
      };
      PS_CHECK_ARG(!misaligned(t.param, ps::dtype_size(t.param_dtype)) &&
                       !misaligned(t.grad, ps::dtype_size(t.grad_dtype)) &&
                       !misaligned(t.exp_avg, state) && !misaligned(t.exp_avg_sq, state) &&
                       !(in_8_bits && misaligned(t.scales, 4)) &&
                       !(t.copy && misaligned(t.copy, ps::dtype_size(t.copy_dtype))),
                   bad("misaligned data"));
      written.add(t.param, n * ps::dtype_size(t.param_dtype));
      written.add(t.exp_avg, n * state);
      written.add(t.exp_avg_sq, n * state);
      if (in_8_bits) written.add(t.scales, blocks * 2 * sizeof(float));
      if (t.copy) written.add(t.copy, n * ps::dtype_size(t.copy_dtype));
      table.push_back({t.param, t.grad, t.exp_avg, t.exp_avg_sq, in_8_bits ? t.scales : nullptr,
                       t.copy, t.count, chunks, t.weight_decay, t.param_dtype, t.grad_dtype,
                       t.copy_dtype});
      total += t.count;
      chunks += (t.count + ps::kChunk - 1) / ps::kChunk;
    }
    PS_CHECK_ARG(chunks < (1LL << 31), "ps_adamw_list_create: too many elements");
    PS_CHECK_ARG(written.close(),
                 "ps_adamw_list_create: parameters, states, scales or copies overlap, or a tensor "
                 "is listed twice");
    for (const ps::AdamTensor& t : table)
      PS_CHECK_ARG(!written.meets(t.grad, size_t(t.count) * ps::dtype_size(t.grad_dtype)),
                   "ps_adamw_list_create: a gradient overlaps what the step writes");
    std::unique_ptr<ps_adamw_list> l(new ps_adamw_list);
    ps::ListTables<ps::AdamTensor> tables;
    const int rc = ps::make_list_tables(table, uint32_t(chunks), 0, &l->tables, &tables);
    if (rc != PS_OK) return rc;
    l->adam = {tables.tensors, tables.chunks, uint32_t(chunks)};
    l->in_8_bits = in_8_bits;
    l->written = std::move(written);
    *out = l.release();
    return PS_OK;
  } catch (const std::exception& e) {
    return ps::fail(PS_ERR_RUNTIME, std::string("ps_adamw_list_create: ") + e.what());
  }
}

void ps_adamw_list_destroy(ps_adamw_list* list) {
  if (list) ps::g_retired_lists.retire(list);
}

int ps_adamw_step(ps_adamw_list* list, const ps_adamw_options* o, ps_stream_t stream) {
  PS_CHECK_ARG(list && o, "ps_adamw_step: null argument");
  PS_CHECK_ARG(o->beta1 >= 0 && o->beta1 < 1 && o->beta2 >= 0 && o->beta2 < 1,
               "ps_adamw_step: betas are from 0 up to below 1");
  constexpr double kLargest = std::numeric_limits<float>::max();  // the kernel computes in FP32
  PS_CHECK_ARG(o->eps >= 0 && o->eps <= kLargest, "ps_adamw_step: eps is not a number from 0 up");
  PS_CHECK_ARG(o->device_lr || std::fabs(o->lr) <= kLargest,
               "ps_adamw_step: the rate is not a number");
  PS_CHECK_ARG(o->device_step || o->step >= 1, "ps_adamw_step: steps are counted from 1");
  PS_CHECK_ARG(!o->norm || o->max_norm >= 0.f,
               "ps_adamw_step: the bound is not a number from 0 up");
  PS_CHECK_ARG(ps::aligned4(o->device_lr) && ps::aligned4(o->device_step) && ps::aligned4(o->norm),
               "ps_adamw_step: misaligned rate, step or norm");
  for (const void* p : {static_cast<const void*>(o->device_lr),
                        static_cast<const void*>(o->device_step),
                        static_cast<const void*>(o->norm)})
    PS_CHECK_ARG(!p || !list->written.meets(p, 4),
                 "ps_adamw_step: the rate, step or norm lies in what the step writes");
  if (!list->adam.chunk_count) return PS_OK;
  const double log_beta1 = std::log(o->beta1), log_beta2 = std::log(o->beta2);
  const double step = o->device_step ? 1.0 : double(o->step);
  const ps::AdamCall call{float(o->beta1),
                          float(1.0 - o->beta1),
                          float(o->beta2),
                          float(1.0 - o->beta2),
                          float(o->eps),
                          float(o->lr),
                          log_beta1,
                          log_beta2,
                          ps::mean_factor(step, log_beta1),
                          ps::root_factor(step, log_beta2),
                          uint32_t(o->step),
                          o->device_lr,
                          o->device_step,
                          o->norm,
                          o->max_norm,
                          o->grad_scale};
  const uint32_t blocks = std::min(list->adam.chunk_count, ps::kAdamBlocks);
  const hipStream_t st = ps::to_hip(stream);
  if (list->in_8_bits)
    ps::adamw_kernel<true><<<blocks, ps::kListThreads, 0, st>>>(list->adam, call);
  else
    ps::adamw_kernel<false><<<blocks, ps::kListThreads, 0, st>>>(list->adam, call);
  PS_LAUNCHED();
  return PS_OK;
}

}  // extern "C"
