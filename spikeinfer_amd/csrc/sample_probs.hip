// The distribution that a row's token is drawn from, over the whole vocabulary.
//
// x = logits / temperature (rounded to fp32, finite where the logit is), tokens in the
// sampler's order: x descending, index ascending.  min_p keeps those with exp(x - max) >=
// min_p, top_k the first of these, top_p those of these before which less than top_p of their
// sum stands; every cut is a prefix of the order, so a token stays if its order key is at or
// above the cut's.  Weights are exp(x - max) from fp64, summed in fixed point (2^-44 of the
// largest): sums do not depend on the order they are made in, and a cut falls where exact
// arithmetic has it unless two numbers agree to 11 digits.
//
// A workgroup a row.  Cuts keep few tokens as a rule, so the row is read twice, once for its
// largest and once for the candidates, those at or above a bound that the threads' maxima
// give; the cuts are then found among the candidates in LDS, the row is filled with zeros and
// the kept tokens are put in their places.  A cut by top_p needs the sum over the whole row:
// candidates count with their exact weight, the rest with fp32 exponentials, whose error is
// bounded; where the cut could fall elsewhere within that bound, or outside the candidates,
// the row goes the long way: a histogram of the exact weights over the row, then the tokens of
// the bin that holds the cut as candidates.  Without cuts the row is read for its largest,
// for the sum, and for the result.
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
constexpr int kCand = 4096;                      // candidates
constexpr int kBins = 2048;                      // 11-bit digits
constexpr int kBinsPerThread = kBins / kThreads;
constexpr int kMostK = 640;                      // largest top_k whose bound the threads' maxima give
constexpr int kOpenReach = 960;                  // maxima above the bound without one: about 2,800 candidates

struct Shared {
  u64 cand[kCand];  // order keys
  u64 hist[kBins];
  u64 wave[kWaves];
  double dwave[kWaves];
  u64 digit, above, in_digit;
  uint32_t tmax[kThreads];
  uint32_t bound;
  int count;
};

// Larger: earlier in the order.
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);  // (-0 is 0)
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ u64 order_key(float x, int i) {
  return (static_cast<u64>(value_key(x)) << kIndexBits) | static_cast<u64>(kMaxVocab - 1 - i);
}
__device__ __forceinline__ float order_value(u64 k) { return key_value(static_cast<uint32_t>(k >> kIndexBits)); }
__device__ __forceinline__ int order_index(u64 k) { return kMaxVocab - 1 - static_cast<int>(k & (kMaxVocab - 1)); }

__device__ __forceinline__ u64 shfl_u64(u64 v, int lane) {
  const uint32_t lo = __shfl(static_cast<uint32_t>(v), lane), hi = __shfl(static_cast<uint32_t>(v >> 32), lane);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ __forceinline__ u64 shfl_xor_u64(u64 v, int d) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), d), hi = __shfl_xor(static_cast<uint32_t>(v >> 32), d);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ __forceinline__ u64 shfl_up_u64(u64 v, int d) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d), hi = __shfl_up(static_cast<uint32_t>(v >> 32), d);
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
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v = op(v, sh.wave[w]);
  return v;
}
__device__ __forceinline__ double block_sum(double v, Shared &sh) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.dwave[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.dwave[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v += sh.dwave[w];
  return v;
}

// A logit over the temperature; what is finite stays finite (a mask of the type's lowest value
// is no -infinity below a temperature of 1).  inv = 1 / temp in fp64: the quotient of two
// fp32 numbers lies at least 2^-49 of itself from the middle between two fp32 numbers, and the
// product is off by at most 2^-52, so its rounding is the quotient's.
__device__ __forceinline__ float quotient(float v, double inv) {
  const float x = static_cast<float>(static_cast<double>(v) * inv);
  return fabsf(x) == INFINITY && fabsf(v) != INFINITY ? copysignf(3.402823466e38f, v) : x;
}

// A bound at or below every logit whose quotient is `x`, that of `bound`.
__device__ __forceinline__ float same_quotient(float bound, float x, float temp) {
  if (fabsf(bound) == INFINITY) return bound;
  if (x == 3.402823466e38f) bound = fminf(bound, x * temp);
  if (x == -3.402823466e38f) return -INFINITY;
  return bound - fabsf(bound) * 0x1p-22f - temp * 0x1p-148f;
}

template <int DT>
struct Row {
  typedef typename Elem<DT>::T E;
  static constexpr int W = Elem<DT>::kVec;
  typedef E Vec __attribute__((ext_vector_type(W)));
  const E *p;
  int V;
  double inv;     // 1 / temperature
  double m, low;  // the largest x; ln min_p

  // f(index, logit) for every token, in no particular order; 16-byte loads, four in flight,
  // between a head and a tail that are not aligned.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int tid = threadIdx.x;
    const int head = min(V, static_cast<int>((-(reinterpret_cast<uintptr_t>(p) / sizeof(E))) & (W - 1)));
    if (tid < head) f(tid, elem_to_f32<DT>(p[tid]));
    const int nv = (V - head) / W;
    const Vec *pv = reinterpret_cast<const Vec *>(p + head);
    auto one = [&](int v, const Vec &a) {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const E e = a[j];
        f(head + v * W + j, elem_to_f32<DT>(e));
      }
    };
    int v = tid;
    for (; v + 3 * kThreads < nv; v += 4 * kThreads) {
      Vec a[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) a[u] = pv[v + u * kThreads];
#pragma unroll
      for (int u = 0; u < 4; ++u) one(v + u * kThreads, a[u]);
    }
    for (; v < nv; v += kThreads) one(v, pv[v]);
    const int t = head + nv * W + tid;
    if (t < V) f(t, elem_to_f32<DT>(p[t]));
  }
  // The same with one copy of f, for passes that compute much (a workgroup waits for the
  // instructions that it runs through once).
  template <class F>
  __device__ __forceinline__ void each_short(F f) const {
#pragma unroll 1
    for (int i0 = threadIdx.x; i0 < V; i0 += 4 * kThreads) {
      E a[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) a[u] = p[min(i0 + u * kThreads, V - 1)];
#pragma unroll 1
      for (int i = i0; i < V && i < i0 + 4 * kThreads; i += kThreads) {
        f(i, elem_to_f32<DT>(a[0]));
        a[0] = a[1];
        a[1] = a[2];
        a[2] = a[3];
      }
    }
  }
  __device__ __forceinline__ float x(float logit) const { return quotient(logit, inv); }
  __device__ __forceinline__ double down(float x) const {
    const double d = static_cast<double>(x) - m;
    return static_cast<double>(x) == m ? 0.0 : d;  // (also where both are infinite)
  }
  __device__ __forceinline__ bool alive(float x) const { return down(x) >= low; }  // (a NaN is not)
  __device__ __forceinline__ u64 mass(float x) const {
    return static_cast<u64>(exp(down(x)) * kMassScale + 0.5);
  }
};

// The bin of sh.hist, from the top, with above < target <= above + its content, `above` being
// `base` and the bins over it, into sh.digit (kBins: none), sh.above and sh.in_digit.
__device__ __forceinline__ void select_bin(Shared &sh, u64 base, double target) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int top = kBins - 1 - kBinsPerThread * tid;
  u64 h[kBinsPerThread], sum = 0;
#pragma unroll
  for (int r = 0; r < kBinsPerThread; ++r) sum += h[r] = sh.hist[top - r];
  u64 inc = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_up_u64(inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 63) sh.wave[wave] = inc;
  if (tid == 0) sh.digit = kBins;
  __syncthreads();
  u64 before = base + inc - sum;
  for (int w = 0; w < wave; ++w) before += sh.wave[w];
#pragma unroll
  for (int r = 0; r < kBinsPerThread; ++r) {
    if (h[r] && static_cast<double>(before) < target && target <= static_cast<double>(before + h[r])) {
      sh.digit = top - r;
      sh.above = before;
      sh.in_digit = h[r];
    }
    before += h[r];
  }
  __syncthreads();
}

// The smallest order key of the shortest prefix whose weights reach `target`, among the tokens
// (order keys) that each(f) visits with a weight; 0 if they do not reach it.  Radix selection: 11-bit digits of the key, from the
// first bit in which `lo` and `hi` (bounds of the keys) differ.
template <class Each>
__device__ __forceinline__ u64 prefix_cut(Shared &sh, u64 lo, u64 hi, double target, Each each) {
  const u64 differ = lo ^ hi;
  int bits = differ ? 64 - __clzll(static_cast<long long>(differ)) : 1;
  u64 prefix = hi >> bits << bits, above = 0;
  while (bits > 0) {
    const int shift = max(bits - 11, 0);
    const uint32_t mask = (1u << (bits - shift)) - 1u;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
    each([&](u64 key, u64 w) {
      if (w && key >> bits == prefix >> bits) atomicAdd(&sh.hist[static_cast<uint32_t>(key >> shift) & mask], w);
    });
    __syncthreads();
    select_bin(sh, above, target);
    if (sh.digit == kBins) return 0;
    prefix |= sh.digit << shift;
    above = sh.above;
    bits = shift;
  }
  return prefix;
}

// A key that at least `need` of the threads' maxima reach, and about as few as can be.
__device__ __forceinline__ void find_bound(Shared &sh, uint32_t need) {
  if (threadIdx.x < 64) {
    constexpr int kPer = kThreads / 64;
    uint32_t t[kPer], top = 0;
#pragma unroll
    for (int q = 0; q < kPer; ++q) {
      t[q] = sh.tmax[q * 64 + threadIdx.x];
      top = max(top, t[q]);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d)));
    auto reach = [&](uint32_t k) {
      uint32_t c = 0;
#pragma unroll
      for (int q = 0; q < kPer; ++q) c += static_cast<uint32_t>(__popcll(__ballot(t[q] >= k)));
      return c;
    };
    uint32_t lo = 0, hi = top;  // reach(lo) >= need; 0: every token
    if (reach(1u) >= need) {
      lo = 1;
      if (reach(hi) >= need) lo = hi;
      else if (hi > (4u << 23) && reach(hi - (4u << 23)) >= need) lo = hi - (4u << 23);
      while (hi - lo > 1u) {
        const uint32_t mid = lo + ((hi - lo) >> 1), c = reach(mid);
        if (c >= need) {
          lo = mid;
          if (c <= need + (need >> 5)) break;
        } else {
          hi = mid;
        }
      }
    }
    if (threadIdx.x == 0) sh.bound = lo;
  }
  __syncthreads();
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
  const float temp = temperature[r];
  row.inv = 1.0 / static_cast<double>(temp);
  const float mp = min_p ? min_p[r] : 0.f, tp_given = top_p ? top_p[r] : 1.f;
  const float tp = tp_given <= 0.f ? 0x1p-60f : tp_given;  // (the first token stays)
  const int tk_given = top_k ? top_k[r] : -1, tk = tk_given > 0 && tk_given < V ? tk_given : 0;
  const auto larger = [](u64 a, u64 b) { return a > b ? a : b; };
  const auto plus = [](u64 a, u64 b) { return a + b; };
  float *o = out + r * out_stride;
  // 0 to every place; the kept tokens' places are written behind a barrier
  auto zeros = [&] {
    typedef float F4 __attribute__((ext_vector_type(4)));
    const int head = min(V, static_cast<int>((-(reinterpret_cast<uintptr_t>(o) / 4)) & 3));
    if (tid < head) o[tid] = 0.f;
    const int nv = (V - head) / 4;
    F4 *ov = reinterpret_cast<F4 *>(o + head);
    for (int v = tid; v < nv; v += kThreads) ov[v] = F4{0.f, 0.f, 0.f, 0.f};
    const int t = head + 4 * nv + tid;
    if (t < V) o[t] = 0.f;
  };

  // ---- the largest logit; each thread's largest as a key (0: none, a NaN is none) ----
  uint32_t mk = 0;
  row.each([&](int, float v) { mk = max(mk, v == v ? value_key(v) : 0u); });
  sh.tmax[tid] = mk;
  const uint32_t best = static_cast<uint32_t>(block_reduce(mk, sh, larger));
  if (best <= value_key(-INFINITY)) {  // nothing to draw from
    zeros();
    return;
  }
  const float most = key_value(best);
  if (!(temp >= kGreedyTemp)) {  // greedy: the first of the largest
    zeros();
    int first = V;
    row.each([&](int i, float v) { first = v == most ? min(first, i) : first; });
    first = static_cast<int>(block_reduce(static_cast<u64>(first), sh, [](u64 a, u64 b) { return a < b ? a : b; }));
    if (tid == 0) o[first] = 1.f;
    return;
  }
  row.m = row.x(most);
  row.low = mp > 0.f ? fmin(log(static_cast<double>(mp)), 0.0) : -INFINITY;  // (the largest stays)
  const bool open = tp < 1.f;

  // ---- no cut: the sum, then the result ----
  if (!tk && !open && !(mp > 0.f)) {
    double z = 0.0;
    row.each([&](int, float v) {
      const double d = row.down(row.x(v));
      if (d >= -INFINITY) z += static_cast<double>(expf(static_cast<float>(d)));
    });
    z = block_sum(z, sh);
    const float scale = static_cast<float>(1.0 / z);
    row.each([&](int i, float v) {
      const double d = row.down(row.x(v));
      o[i] = d >= -INFINITY ? expf(static_cast<float>(d)) * scale : 0.f;
    });
    return;
  }

  // ---- candidates: logits at or above a bound ----
  // Every token that a cut may keep is among them: of top_k's prefix as many are there as
  // the threads' maxima say, of min_p's all.  Without either, a prefix of about 2,800.
  u64 cut = 0, Z = 0;
  if (tk <= kMostK) {
    const bool rest_counts = open && !tk && !(mp > 0.f);
    float bound = -INFINITY;
    if (tk || rest_counts) {
      find_bound(sh, tk ? tk : kOpenReach);
      if (sh.bound > value_key(-INFINITY)) bound = key_value(sh.bound);
    }
    const float whole = row.x(bound);  // from here on up no token is missing
    bound = same_quotient(bound, whole, temp);
    if (mp > 0.f) {
      const double x = row.m + row.low;
      const float least = x <= -3.402823466e38 ? -INFINITY : static_cast<float>(x * static_cast<double>(temp));
      bound = fmaxf(bound, fabsf(least) == INFINITY ? least : least - fabsf(least) * 0x1p-20f - temp * 0x1p-148f);
    }
    if (tid == 0) sh.count = 0;
    __syncthreads();
    const float c1 = static_cast<float>(row.inv * 1.4426950408889634);
    const float c2 = static_cast<float>(row.m * 1.4426950408889634);
    float rest = 0.f;
    row.each([&](int i, float v) {
      if (v >= bound) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kCand) sh.cand[at] = order_key(row.x(v), i);
      } else if (rest_counts && v == v) {
        rest += __builtin_amdgcn_exp2f(v * c1 - c2);
      }
    });
    __syncthreads();
    const int n = sh.count;
    if (n <= kCand) {
      auto weight = [&](u64 k) -> u64 { return k >= cut && row.alive(order_value(k)) ? row.mass(order_value(k)) : 0; };
      auto cands = [&](auto f) {
        for (int j = tid; j < n; j += kThreads) f(sh.cand[j]);
      };
      auto total = [&](u64 from) {
        u64 z = 0;
        cands([&](u64 k) { z += k >= from ? weight(k) : 0; });
        return block_reduce(z, sh, plus);
      };
      u64 lo = ~0ull, hi = 0;
      cands([&](u64 k) {
        lo = min(lo, k);
        hi = max(hi, k);
      });
      lo = block_reduce(lo, sh, [](u64 a, u64 b) { return a < b ? a : b; });
      hi = block_reduce(hi, sh, larger);
      if (tk)
        cut = prefix_cut(sh, lo, hi, static_cast<double>(tk), [&](auto f) {
          cands([&](u64 k) { f(k, row.alive(order_value(k)) ? 1ull : 0ull); });
        });
      Z = total(cut);
      bool found = true;
      if (open) {
        double lowest = static_cast<double>(Z), highest = lowest;
        if (rest_counts) {
          // The exponent (at most 160 below c2, or the power is 0) is off by 2^-22 of its terms, a
          // power by a step, a sum of 2^8 terms by 2^8 half steps.
          const double s = block_sum(static_cast<double>(rest), sh) * kMassScale;
          const double off = 0x1p-15 + 0x1p-22 * (fabs(static_cast<double>(c2)) + 160.0);
          lowest += s * fmax(1.0 - off, 0.0);
          highest += s * (1.0 + off) + 1.0;
        }
        const u64 c = prefix_cut(sh, lo, hi, static_cast<double>(tp) * lowest, [&](auto f) {
          cands([&](u64 k) { f(k, weight(k)); });
        });
        if (rest_counts)  // the same cut for the largest sum there can be, and no token missing above it
          found = c && order_value(c) >= whole && static_cast<double>(tp) * highest <= static_cast<double>(total(c));
        if (found) {
          cut = larger(cut, c);
          Z = total(cut);
        }
      }
      if (found) {
        zeros();
        const double scale = kMassScale / static_cast<double>(Z);
        __syncthreads();
        cands([&](u64 k) {
          const float x = order_value(k);
          if (k >= cut && row.alive(x)) o[order_index(k)] = static_cast<float>(exp(row.down(x)) * scale);
        });
        return;
      }
    }
  }

  // ---- the long way ----
  const u64 highest_key = order_key(static_cast<float>(row.m), 0);
  cut = 0;
  if (tk)
    cut = prefix_cut(sh, 0, highest_key, static_cast<double>(tk), [&](auto f) {
      row.each_short([&](int i, float v) {
        const float x = row.x(v);
        f(order_key(x, i), row.alive(x) ? 1ull : 0ull);
      });
    });
  auto total = [&](u64 from) {
    u64 z = 0;
    row.each_short([&](int i, float v) {
      const float x = row.x(v);
      if (row.alive(x) && order_key(x, i) >= from) z += row.mass(x);
    });
    return block_reduce(z, sh, plus);
  };
  Z = total(cut);
  if (open) {
    const u64 c = cut;
    cut = larger(cut, prefix_cut(sh, 0, highest_key, static_cast<double>(tp) * static_cast<double>(Z), [&](auto f) {
                   row.each_short([&](int i, float v) {
                     const float x = row.x(v);
                     const u64 key = order_key(x, i);
                     f(key, key >= c && row.alive(x) ? row.mass(x) : 0ull);
                   });
                 }));
    Z = total(cut);
  }
  const double scale = kMassScale / static_cast<double>(Z);
  row.each_short([&](int i, float v) {
    const float x = row.x(v);
    o[i] = row.alive(x) && order_key(x, i) >= cut ? static_cast<float>(exp(row.down(x)) * scale) : 0.f;
  });
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
