// The distribution that a row's token is drawn from, over the whole vocabulary.
//
// x = logits / temperature (rounded to fp32, finite where the logit is), tokens in the sampler's order: x descending,
// index ascending.  min_p keeps those with exp(x - max) >= min_p, top_k the first of these,
// top_p those of these before which less than top_p of their sum stands; every cut is a
// prefix of the order, so a token stays if its order key is at or above the cut's.  Weights
// are exp(x - max) from fp64, summed in fixed point (2^-44 of the largest): sums do not
// depend on the order they are made in, and a cut falls where exact arithmetic has it unless
// two numbers agree to 11 digits.
#include "common.hpp"
#include "lif_math.hpp"

namespace spk {
namespace probs {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kIndexBits = 18;
constexpr int kMaxVocab = 1 << kIndexBits;
constexpr float kGreedyTemp = 1e-5f;
constexpr double kMassScale = 17592186044416.0;  // 2^44: 2^18 weights of at most 1 fit 64 bits

struct Shared {
  u64 hist[256];
  u64 wave[kWaves];
  u64 digit, above;
};

// Larger: earlier in the order.
__device__ __forceinline__ u64 order_key(float x, int i) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<u64>(k) << kIndexBits) | static_cast<u64>(kMaxVocab - 1 - i);
}

__device__ __forceinline__ u64 shfl_xor_u64(u64 v, int d) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), d), hi = __shfl_xor(static_cast<uint32_t>(v >> 32), d);
  return (static_cast<u64>(hi) << 32) | lo;
}

// Over the workgroup, to every thread.
template <class Op>
__device__ __forceinline__ u64 block_reduce(u64 v, Shared &sh, Op op) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = op(v, shfl_xor_u64(v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.wave[0];
  for (int w = 1; w < kWaves; ++w) v = op(v, sh.wave[w]);
  return v;
}

// A logit over the temperature; what is finite stays finite (a mask of the type's lowest value
// is no -infinity below a temperature of 1).
__device__ __forceinline__ float quotient(float v, float temp) {
  const float x = v / temp;
  return fabsf(x) == INFINITY && fabsf(v) != INFINITY ? copysignf(3.402823466e38f, x) : x;
}

template <int DT>
struct Row {
  typedef typename Elem<DT>::T E;
  const E *p;
  int V;
  float temp;
  double m, low;  // the largest x; ln min_p

  __device__ __forceinline__ float x(int i) const {
    const float v = elem_to_f32<DT>(p[i]);
    return temp < kGreedyTemp ? v : quotient(v, temp);
  }
  __device__ __forceinline__ double down(float x) const {
    const double d = static_cast<double>(x) - m;
    return static_cast<double>(x) == m ? 0.0 : d;  // (also where both are infinite)
  }
  __device__ __forceinline__ bool alive(float x) const { return down(x) >= low; }  // (a NaN is not)
  __device__ __forceinline__ u64 mass(float x) const {
    return static_cast<u64>(exp(down(x)) * kMassScale + 0.5);
  }
};

// The smallest order key of the shortest prefix whose weights reach `target`, among the
// tokens that `weight` gives one; 0 if all of them do not.
template <int DT, class Weight>
__device__ __forceinline__ u64 prefix_cut(const Row<DT> &row, Shared &sh, double target, Weight weight) {
  u64 prefix = 0, above = 0;
  for (int shift = 48; shift >= 0; shift -= 8) {
    for (int b = threadIdx.x; b < 256; b += kThreads) sh.hist[b] = 0;
    if (threadIdx.x == 0) sh.digit = 256;
    __syncthreads();
    for (int i = threadIdx.x; i < row.V; i += kThreads) {
      const float x = row.x(i);
      const u64 key = order_key(x, i);
      if ((key >> shift >> 8) != (prefix >> shift >> 8)) continue;
      const u64 w = weight(x, key);
      if (w) atomicAdd(&sh.hist[(key >> shift) & 255], w);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      u64 before = above;
      for (int b = 255; b >= 0; --b) {
        const u64 h = sh.hist[b];
        if (h && static_cast<double>(before) < target && target <= static_cast<double>(before + h)) {
          sh.digit = b;
          sh.above = before;
          break;
        }
        before += h;
      }
    }
    __syncthreads();
    const u64 digit = sh.digit;
    above = sh.above;
    __syncthreads();
    if (digit == 256) return 0;
    prefix |= digit << shift;
  }
  return prefix;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void probs_kernel(const void *logits, int64_t row_stride, int V,
                                                         const float *temperature, const int32_t *top_k,
                                                         const float *top_p, const float *min_p, float *out,
                                                         int64_t out_stride) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  Row<DT> row;
  row.p = static_cast<const typename Elem<DT>::T *>(logits) + r * row_stride;
  row.V = V;
  row.temp = temperature[r];
  const float mp = min_p ? min_p[r] : 0.f, tp = top_p ? top_p[r] : 1.f;
  const int tk = top_k ? top_k[r] : -1;
  const auto larger = [](u64 a, u64 b) { return a > b ? a : b; };
  const auto plus = [](u64 a, u64 b) { return a + b; };
  float *o = out + r * out_stride;

  u64 best = 0;
  for (int i = tid; i < V; i += kThreads) {
    const float x = row.x(i);
    if (x == x) best = larger(best, order_key(x, i));
  }
  best = block_reduce(best, sh, larger);
  const int first = kMaxVocab - 1 - static_cast<int>(best & (kMaxVocab - 1));
  const float m = best ? row.x(first) : -INFINITY;
  if (m == -INFINITY || row.temp < kGreedyTemp) {  // nothing to draw from; the first of the order
    for (int i = tid; i < V; i += kThreads) o[i] = m != -INFINITY && i == first ? 1.f : 0.f;
    return;
  }
  row.m = m;
  row.low = mp > 0.f ? log(static_cast<double>(mp)) : -INFINITY;
  u64 cut = 0;
  if (tk > 0 && tk < V)
    cut = prefix_cut(row, sh, static_cast<double>(tk), [&](float x, u64) -> u64 { return row.alive(x) ? 1 : 0; });
  auto total = [&](u64 from) {
    u64 z = 0;
    for (int i = tid; i < V; i += kThreads) {
      const float x = row.x(i);
      if (row.alive(x) && order_key(x, i) >= from) z += row.mass(x);
    }
    return block_reduce(z, sh, plus);
  };
  u64 Z = total(cut);
  if (tp < 1.f) {
    const u64 c = cut;
    cut = larger(cut, prefix_cut(row, sh, static_cast<double>(tp) * static_cast<double>(Z), [&](float x, u64 key) -> u64 {
                   return key >= c && row.alive(x) ? row.mass(x) : 0;
                 }));
    Z = total(cut);
  }
  const double scale = kMassScale / static_cast<double>(Z);
  for (int i = tid; i < V; i += kThreads) {
    const float x = row.x(i);
    o[i] = row.alive(x) && order_key(x, i) >= cut ? static_cast<float>(exp(row.down(x)) * scale) : 0.f;
  }
}

template <int DT>
void launch(const void *logits, int64_t row_stride, int rows, int V, const float *temperature, const int32_t *top_k,
            const float *top_p, const float *min_p, float *out, int64_t out_stride, hipStream_t s) {
  probs_kernel<DT><<<rows, kThreads, 0, s>>>(logits, row_stride, V, temperature, top_k, top_p, min_p, out, out_stride);
}

}  // namespace probs
}  // namespace spk

using namespace spk;

extern "C" size_t spk_sample_probs_workspace_bytes(int rows, int vocab) { return 0; }

extern "C" int spk_sample_probs(const void *logits, int logits_dtype, int64_t row_stride, int rows, int vocab,
                                const float *temperature, const int32_t *top_k, const float *top_p,
                                const float *min_p, float *probs_out, int64_t out_stride, void *workspace,
                                size_t workspace_bytes, void *stream) {
  if (!valid_float_dtype(logits_dtype))
    return fail(SPK_EINVAL, "sample_probs: logits dtype %d is not a float type", logits_dtype);
  if (rows < 0 || vocab < 1 || vocab > probs::kMaxVocab)
    return fail(SPK_EINVAL, "sample_probs: rows=%d, vocab=%d must be in [1, %d]", rows, vocab, probs::kMaxVocab);
  if (rows > 1 && out_stride < vocab) return fail(SPK_EINVAL, "sample_probs: rows of the output lie on one another");
  if (rows == 0) return SPK_OK;
  if (!logits || !temperature || !probs_out) return fail(SPK_EINVAL, "sample_probs: null pointer");
  const size_t need = spk_sample_probs_workspace_bytes(rows, vocab);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(SPK_EINVAL, "sample_probs: workspace of %zu bytes, %zu needed, aligned to 16",
                workspace ? workspace_bytes : 0, need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (logits_dtype == SPK_F32)
    probs::launch<SPK_F32>(logits, row_stride, rows, vocab, temperature, top_k, top_p, min_p, probs_out, out_stride, s);
  else if (logits_dtype == SPK_F16)
    probs::launch<SPK_F16>(logits, row_stride, rows, vocab, temperature, top_k, top_p, min_p, probs_out, out_stride, s);
  else
    probs::launch<SPK_BF16>(logits, row_stride, rows, vocab, temperature, top_k, top_p, min_p, probs_out, out_stride, s);
  return check_launch("sample_probs");
}
