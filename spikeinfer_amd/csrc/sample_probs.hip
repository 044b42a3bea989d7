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
// Two launches, the first a workgroup a slice of a row, the second one a row (more where there are
// no cuts).  Cuts keep few tokens as a rule, so:
//   * the first (slice_kernel) holds its slice in registers, fills its part of the result with
//     zeros and lists its candidates, the logits at or above a bound that so many of the
//     threads' maxima reach, with the sum of the others' weights;
//   * the second (row_kernel) finds the cuts among the candidates of a row's slices and puts
//     the kept tokens in their places.  A cut by top_p needs the sum over the whole row:
//     candidates count in fixed point, the others with the slices' sums, whose error is bounded;
//     where the cut could fall elsewhere within that bound, or below a slice's bound, the row
//     goes the long way, through histograms of the weights over the row.
// A row without cuts gets its sum from the first launch and its values from the second.
// Many rows are bound by memory (320 of 151,936 in bf16: slices 64 us, 4.5 TB/s, rows 16), few by
// the phases behind barriers (one row: 12 and 16 us, of which the weights in fp64 take 4 and 3).
// The long way takes a workgroup 130 to 230 us for 151,936 tokens, and 750 and more where a cut has
// to be found by digits.  Rows that go it, of bf16 logits:
//   * nearly flat ones under top_p (a cut below the candidates), and top_k above kMostK;
//   * masked ones, where fewer threads of a slice hold an allowed token than its bound asks for: the
//     bound is the mask's value then, and every token of the slice is listed.  Five rows with 200 and
//     2,000 tokens allowed: top_p 160 and 174 us, top_k of 50 242 and 17; with 20 allowed 158 and 763
//     (fewer than top_k: the cut lies among the masked); with 20,000 25 and 19.  min_p escapes
//     (13 to 18 us; with the type's lowest value as the mask and 20 allowed 65), rows without cuts too;
//   * rows whose likely tokens lie in one slice: in descending order top_p 219 us, top_k of 50 253.
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "lif_math.hpp"

namespace spk {
namespace probs {

typedef unsigned long long u64;

constexpr int kSliceThreads = 512;
// 16-byte vectors of a slice that a thread holds, by the elements of one: 10,240 or 12,288 tokens.
// (16-bit rows with five: one row of 151,936 29 us against 27; fp32 with three: slices of 6,144
// miss top_k's tokens too often, 77 rows of 50,257 100 us against 29.)
constexpr int slice_vecs(int vec) { return vec == 4 ? 5 : 3; }
constexpr int kRowThreads = 512;
constexpr int kIndexBits = 18;
constexpr int kMaxVocab = 1 << kIndexBits;
constexpr float kGreedyTemp = 1e-5f;
constexpr float kMost = 3.402823466e38f;         // the largest fp32 number
constexpr double kMassScale = 17592186044416.0;  // 2^44: 2^18 weights of at most 1 fit 64 bits
constexpr int kCand = 4096;                      // candidates of a row
constexpr int kBins = 1024;              // of a row's histogram: 10-bit digits
constexpr int kBinsPerThread = kBins / kRowThreads;
constexpr int kRank = 256;                       // candidates that are ranked one against the other
constexpr int kMaxSlices = kMaxVocab / (4 * slice_vecs(4) * kSliceThreads) + 2;  // of a row
constexpr int kMostK = 2048;                     // top_k beyond: the long way
constexpr int kChunk = 256;                     // candidates that a wave takes at a time

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

__device__ __forceinline__ u64 shfl_xor_u64(u64 v, int d) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), d), hi = __shfl_xor(static_cast<uint32_t>(v >> 32), d);
  return (static_cast<u64>(hi) << 32) | lo;
}
__device__ __forceinline__ u64 shfl_up_u64(u64 v, int d) {
  const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d), hi = __shfl_up(static_cast<uint32_t>(v >> 32), d);
  return (static_cast<u64>(hi) << 32) | lo;
}

// A logit over the temperature; what is finite stays finite (a mask of the type's lowest value
// is no -infinity below a temperature of 1).  inv = inverse(temp): the quotient of two
// fp32 numbers lies at least 2^-49 of itself from the middle between two fp32 numbers, and the
// product is off by at most 2^-52, so its rounding is the quotient's (below 2^-126, where the
// numbers have fewer bits, it may be the one beside it).
__device__ __forceinline__ float quotient(float v, double inv) {
  const float x = static_cast<float>(static_cast<double>(v) * inv);
  return fabsf(x) == INFINITY && fabsf(v) != INFINITY ? copysignf(kMost, v) : x;
}
// 1 / temp in fp64; of an infinite temperature a number that makes every finite logit 0 in fp32
// and leaves the infinite ones (0 would make them NaN).
__device__ __forceinline__ double inverse(float temp) {
  return temp < INFINITY ? 1.0 / static_cast<double>(temp) : 0x1p-400;
}

// A bound at or below every logit whose quotient is `x`, that of `bound`.
__device__ __forceinline__ float same_quotient(float bound, float x, float temp) {
  if (fabsf(bound) == INFINITY) return bound;
  if (x == kMost) bound = fminf(bound, x * temp);
  if (x == -kMost) return -INFINITY;
  return bound - fabsf(bound) * 0x1p-22f - temp * 0x1p-148f;
}

// exp(logit / temp - x_most) in fp32; the quotient with one correction (inv: fp32 of 1 / temp,
// inv64 = inverse(temp)).
__device__ __forceinline__ float power(float v, float temp, float inv, double inv64, float x_most) {
  const float q = v * inv;
  float x = __builtin_fmaf(__builtin_fmaf(-q, temp, v), inv, q);
  x = fabsf(q) < 1e30f && temp < INFINITY ? x : quotient(v, inv64);  // (and infinities, NaN)
  return x == x ? expf(x == x_most ? 0.f : x - x_most) : 0.f;
}

// exp(d) for -800 <= d <= 0, off by less than kPowerOff of itself: the Taylor polynomial of degree
// 11 around multiples of ln 2 (the next term is 0.3466^12 / 12! = 6.3e-15, the roundings a few of
// 1.1e-16).  Half of the library's instructions.
constexpr double kPowerOff = 0x1p-46;
__device__ __forceinline__ double power64(double d) {
  const double n = __builtin_rint(d * 1.4426950408889634);
  const double g = __builtin_fma(n, -2.3190468138462996e-17, __builtin_fma(n, -0.6931471805599453, d));
  double p = 1.0 / 39916800.0;
  p = __builtin_fma(p, g, 1.0 / 3628800.0);
  p = __builtin_fma(p, g, 1.0 / 362880.0);
  p = __builtin_fma(p, g, 1.0 / 40320.0);
  p = __builtin_fma(p, g, 1.0 / 5040.0);
  p = __builtin_fma(p, g, 1.0 / 720.0);
  p = __builtin_fma(p, g, 1.0 / 120.0);
  p = __builtin_fma(p, g, 1.0 / 24.0);
  p = __builtin_fma(p, g, 1.0 / 6.0);
  p = __builtin_fma(p, g, 0.5);
  p = __builtin_fma(p, g, 1.0);
  p = __builtin_fma(p, g, 1.0);
  return __builtin_amdgcn_ldexp(p, static_cast<int>(n));
}

enum Kind { kGreedy, kWhole, kCuts };

// A row's parameters.
struct Ask {
  float temp, min_p, top_p;
  int top_k;   // 0: none
  double inv;  // 1 / temperature
  double low;  // ln min_p
  Kind kind;
  bool open;  // a cut by top_p
};

struct Args {
  const void *logits;
  int64_t row_stride;
  int V;
  const float *temperature, *top_p, *min_p;
  const int32_t *top_k;
  float *out;
  int64_t out_stride;
  int S, cap;       // slices of a row, candidates of a slice
  int groups;       // workgroups of a row in the second launch
  int reach, most;  // threads whose maxima reach a slice's bound: without top_k; with the largest
  struct Head *heads;  // [row][slice]
  u64 *lists;          // [row][slice][cap]
};

// What a slice leaves for its row.
struct Head {
  int count;    // candidates; -1: more than fit
  float most;   // the largest logit, -infinity: none
  float whole;  // quotients from here on up are all listed
  double rest;  // sum of exp(x - its most's x) over the others (rows without cuts: over all)
};

__device__ __forceinline__ Ask ask(const Args &a, int64_t r) {
  Ask k;
  k.temp = a.temperature[r];
  k.min_p = a.min_p ? a.min_p[r] : 0.f;
  const float tp = a.top_p ? a.top_p[r] : 1.f;
  k.top_p = tp <= 0.f ? 0x1p-60f : tp;  // (the first token stays)
  const int tk = a.top_k ? a.top_k[r] : -1;
  k.top_k = tk > 0 && tk < a.V ? tk : 0;
  k.inv = inverse(k.temp);
  k.low = k.min_p > 0.f ? fmin(log(static_cast<double>(k.min_p)), 0.0) : -INFINITY;  // (the largest stays)
  k.open = k.top_p < 1.f;
  k.kind = !(k.temp >= kGreedyTemp) ? kGreedy : k.top_k || k.open || k.min_p > 0.f ? kCuts : kWhole;
  return k;
}

// ---- slices --------------------------------------------------------------------------
// A row's elements as 16-byte vectors of aligned memory: the first may begin before the row,
// the last end behind it.
template <int DT>
struct RowMem {
  typedef typename Elem<DT>::T E;
  static constexpr int W = Elem<DT>::kVec, kVecs = slice_vecs(W);
  typedef E Vec __attribute__((ext_vector_type(W)));
  const E *p;
  int V, before;  // elements of the first vector that are not the row's

  __device__ __forceinline__ RowMem(const Args &a, int64_t r) {
    p = static_cast<const E *>(a.logits) + r * a.row_stride;
    V = a.V;
    before = static_cast<int>(reinterpret_cast<uintptr_t>(p) / sizeof(E)) & (W - 1);
  }
  static __device__ __forceinline__ E none() {  // a NaN
    if constexpr (DT == SPK_F32) return __uint_as_float(0x7fc00000u);
    else return static_cast<E>(0x7fff);
  }
  __device__ __forceinline__ int first(int v) const { return v * W - before; }  // index of a vector's first element
  __device__ __forceinline__ Vec load(int v) const {
    const int i = first(v);
    if (i >= 0 && i + W <= V) return *reinterpret_cast<const Vec *>(p + i);
    Vec a;
#pragma unroll
    for (int j = 0; j < W; ++j) a[j] = i + j >= 0 && i + j < V ? p[i + j] : none();
    return a;
  }
};

// Places [i0, i1) of a row's result.
__device__ __forceinline__ void fill_zeros(float *o, int i0, int i1, int threads) {
  typedef float F4 __attribute__((ext_vector_type(4)));
  o += i0;
  const int n = i1 - i0, tid = threadIdx.x;
  const int head = min(n, static_cast<int>((-(reinterpret_cast<uintptr_t>(o) / 4)) & 3));
  if (tid < head) o[tid] = 0.f;
  const int nv = (n - head) / 4;
  F4 *ov = reinterpret_cast<F4 *>(o + head);
  for (int v = tid; v < nv; v += threads) ov[v] = F4{0.f, 0.f, 0.f, 0.f};
  const int t = head + 4 * nv + tid;
  if (t < n) o[t] = 0.f;
}

struct SliceShared {
  int32_t i[kCand];  // the candidates
  uint32_t tmax[kSliceThreads];
  float wave[kSliceThreads / 64];
  double part[kSliceThreads / 64];
  uint32_t bound;
  int count, first;
};

// A key that at least `need` of the threads' maxima reach, and about as few as can be (0: fewer
// threads have one).
__device__ __forceinline__ void find_bound(SliceShared &sh, uint32_t need) {
  if (threadIdx.x < 64) {
    constexpr int kPer = kSliceThreads / 64;
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
    uint32_t lo = 0, hi = top;
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
__global__ __launch_bounds__(kSliceThreads) void slice_kernel(Args a) {
  typedef RowMem<DT> Mem;
  typedef typename Mem::E E;
  constexpr int W = Mem::W, kVecs = Mem::kVecs;
  __shared__ SliceShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = blockIdx.x / a.S;
  const int s = static_cast<int>(blockIdx.x % a.S);
  const Mem row(a, r);
  const int v0 = s * kVecs * kSliceThreads;
  typename Mem::Vec reg[kVecs];
#pragma unroll
  for (int q = 0; q < kVecs; ++q) reg[q] = row.load(v0 + q * kSliceThreads + tid);
  const Ask k = ask(a, r);
  Head *head = a.heads + r * a.S + s;
  if (k.kind != kWhole)
    fill_zeros(a.out + r * a.out_stride, min(max(row.first(v0), 0), a.V),
               min(max(row.first(v0 + kVecs * kSliceThreads), 0), a.V), kSliceThreads);

  // f(index, logit)
  auto each = [&](auto f) {
#pragma unroll
    for (int q = 0; q < kVecs; ++q)
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const E e = reg[q][j];
        f(row.first(v0 + q * kSliceThreads + tid) + j, elem_to_f32<DT>(e));
      }
  };
  float most = -INFINITY;
  each([&](int, float v) { most = fmaxf(most, v); });
  sh.tmax[tid] = most > -INFINITY ? value_key(most) : 0u;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  if (lane == 0) sh.wave[wave] = most;
  if (tid == 0) sh.count = 0, sh.first = kMaxVocab;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSliceThreads / 64; ++w) most = fmaxf(most, sh.wave[w]);
  auto sum = [&](double v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if (lane == 0) sh.part[wave] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kSliceThreads / 64; ++w) v += sh.part[w];
    return v;
  };
  if (most == -INFINITY) {
    if (tid == 0) *head = Head{0, most, -INFINITY, 0.0};
    return;
  }
  if (k.kind == kGreedy) {
    int first = kMaxVocab;
    each([&](int i, float v) { first = v == most ? min(first, i) : first; });
    atomicMin(&sh.first, first);
    __syncthreads();
    if (tid == 0) *head = Head{sh.first, most, -INFINITY, 0.0};
    return;
  }
  const float x_most = quotient(most, k.inv);
  if (k.kind == kWhole) {
    const float inv = 1.f / k.temp;
    float z = 0.f;
    each([&](int, float v) { z += power(v, k.temp, inv, k.inv, x_most); });
    const double all = sum(z);
    if (tid == 0) *head = Head{0, most, -INFINITY, all};
    return;
  }
  // ---- candidates ----
  if (k.top_k > kMostK) {
    if (tid == 0) *head = Head{-1, most, INFINITY, 0.0};
    return;
  }
  float bound = -INFINITY;
  if (k.top_k || !(k.min_p > 0.f)) {
    find_bound(sh, k.top_k ? min(k.top_k, a.most) : a.reach);
    if (sh.bound > value_key(-INFINITY)) bound = key_value(sh.bound);
  }
  float whole = quotient(bound, k.inv);
  bound = same_quotient(bound, whole, k.temp);
  if (k.min_p > 0.f) {  // those below ln min_p under this slice's largest are none of the row's
    const double x = static_cast<double>(x_most) + k.low;
    const float least = x <= -static_cast<double>(kMost) || !(k.temp < INFINITY) ? -INFINITY : static_cast<float>(x * static_cast<double>(k.temp));
    const float lower = fabsf(least) == INFINITY ? least : least - fabsf(least) * 0x1p-20f - k.temp * 0x1p-148f;
    if (lower > bound || !k.top_k) {
      bound = lower;
      whole = -INFINITY;  // of the survivors none is missing
    }
  }
  // A thread's candidates as bits of its elements, then their indices into LDS; the values
  // are read again (one round trip for all; a branch an element took 4.4 us against 1).
  constexpr int kSlots = kVecs * W;
  static_assert(kSlots <= 64, "a bit each");
  u64 hits = 0;
  double rest = 0.0;
  if (k.open && !k.top_k && !(k.min_p > 0.f)) {
    const double m = x_most;
    int slot = 0;
    each([&](int, float v) {
      hits |= v >= bound ? 1ull << slot : 0;
      ++slot;
      // (what overflows weighs nothing beside the largest; fmax takes the difference for a NaN)
      const double d = static_cast<double>(static_cast<float>(static_cast<double>(v) * k.inv)) - m;
      rest += power64(v < bound ? fmax(d, -800.0) : -800.0);
    });
    rest = sum(rest);
  } else {
    int slot = 0;
    each([&](int, float v) {
      hits |= v >= bound ? 1ull << slot : 0;
      ++slot;
    });
  }
  const int own = __popcll(hits);
  int upto = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  int at = 0;
  if (lane == 63 && upto) at = atomicAdd(&sh.count, upto);
  at = __shfl(at, 63) + upto - own;
  __syncthreads();
  const int n = sh.count;
  if (n <= a.cap) {
    for (; hits; hits &= hits - 1) {
      const int slot = __builtin_ctzll(hits);
      sh.i[at++] = row.first(v0 + slot / W * kSliceThreads + tid) + slot % W;
    }
    __syncthreads();
    u64 *list = a.lists + (r * a.S + s) * a.cap;
#pragma unroll 4
    for (int j = tid; j < n; j += kSliceThreads) list[j] = order_key(quotient(elem_to_f32<DT>(row.p[sh.i[j]]), k.inv), sh.i[j]);
  }
  if (tid == 0) *head = Head{n <= a.cap ? n : -1, most, whole, rest};
}

// ---- rows ----------------------------------------------------------------------------
struct RowShared {
  u64 key[kCand], mass[kCand];
  u64 hist[kBins];
  u64 wave[kRowThreads / 64];
  Head head[kMaxSlices];
  u64 digit, above, pick;
  int count;
};

// Over the workgroup, to every thread.
template <class Op>
__device__ __forceinline__ u64 block_reduce(u64 v, RowShared &sh, Op op) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = op(v, shfl_xor_u64(v, d));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh.wave[0];
#pragma unroll
  for (int w = 1; w < kRowThreads / 64; ++w) v = op(v, sh.wave[w]);
  return v;
}
__device__ __forceinline__ u64 larger(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 smaller(u64 a, u64 b) { return a < b ? a : b; }
__device__ __forceinline__ u64 plus(u64 a, u64 b) { return a + b; }

// The bin of sh.hist, from the top, with above < target <= above + its content, `above` being
// `base` and the bins over it, into sh.digit (kBins: none) and sh.above.
__device__ __forceinline__ void select_bin(RowShared &sh, u64 base, double target) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int top = kBins - 1 - kBinsPerThread * tid;
  u64 h[kBinsPerThread], sum = 0;
#pragma unroll
  for (int q = 0; q < kBinsPerThread; ++q) sum += h[q] = sh.hist[top - q];
  u64 inc = sum;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const u64 o = shfl_up_u64(inc, d);
    if (lane >= d) inc += o;
  }
  __syncthreads();  // (what sh.wave held is read)
  if (lane == 63) sh.wave[wave] = inc;
  if (tid == 0) sh.digit = kBins;
  __syncthreads();
  u64 before = base + inc - sum;
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) before += w < wave ? sh.wave[w] : 0;
#pragma unroll
  for (int q = 0; q < kBinsPerThread; ++q) {
    if (h[q] && static_cast<double>(before) < target && target <= static_cast<double>(before + h[q])) {
      sh.digit = top - q;
      sh.above = before;
    }
    before += h[q];
  }
  __syncthreads();
}

// The smallest order key of the shortest prefix whose weights reach `target`, among the tokens
// (order keys) that each(f) visits with a weight, `base` of it before all of them; 0 if they do
// not reach it.  Radix selection: 10-bit digits of the key, from the first bit in which `lo` and
// `hi` (bounds of the keys) differ.
template <class Each>
__device__ __forceinline__ u64 radix_cut(RowShared &sh, u64 lo, u64 hi, u64 base, double target, Each each) {
  const u64 differ = lo ^ hi;
  int bits = differ ? 64 - __clzll(static_cast<long long>(differ)) : 1;
  u64 prefix = hi >> bits << bits, above = base;
  while (bits > 0) {
    const int shift = max(bits - 10, 0);
    const uint32_t mask = (1u << (bits - shift)) - 1u;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kRowThreads) sh.hist[b] = 0;
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

// A candidate's place: how many stand before it, and their weight.  Two threads a candidate
// (e = thread / 2, n <= kRank) take half of the others each.
struct Place {
  int rank;
  u64 before;
};
__device__ __forceinline__ Place place(const u64 *key, const u64 *mass, int n) {
  Place r{0, 0};
  const int e = threadIdx.x >> 1;
  if (e < n) {
    const u64 k = key[e];
#pragma unroll 4
    for (int j = threadIdx.x & 1; j < n; j += 2) {
      const bool first = key[j] > k;
      r.rank += first ? 1 : 0;
      r.before += first ? mass[j] : 0;
    }
    r.rank += __shfl_xor(r.rank, 1);
    r.before += shfl_xor_u64(r.before, 1);
  }
  return r;
}

// The cut as radix_cut finds it among at most kRank candidates, ranked one against the other; those
// below `from` have no weight, by_count: 1 each.
__device__ __forceinline__ u64 rank_cut(RowShared &sh, const u64 *key, const u64 *mass, int n, bool by_count, u64 from,
                                        u64 base, double target) {
  if (threadIdx.x == 0) sh.pick = 0;
  __syncthreads();
  const Place at = place(key, mass, n);
  const int e = threadIdx.x >> 1;
  if (e < n && !(threadIdx.x & 1) && key[e] >= from) {
    const u64 before = base + (by_count ? static_cast<u64>(at.rank) : at.before), w = by_count ? 1ull : mass[e];
    if (w && static_cast<double>(before) < target && target <= static_cast<double>(before + w)) sh.pick = key[e];
  }
  __syncthreads();
  return sh.pick;
}
// The cut as radix_cut finds it, among the n candidates in sh.key (sh.mass: their weights; by_count:
// 1 each), of which those below `from` have none, x between `bottom` and `top` (where they are no
// finite distance apart, the candidates are looked at).  Few are ranked.  Many go into bins of equal
// width in x first, and those of the bin that holds the cut are ranked; where that is too many as
// well (equal logits), by digits.
__device__ __forceinline__ u64 cand_cut(RowShared &sh, int n, bool by_count, u64 from, u64 base, double target, float top,
                                        float bottom) {
  if (n <= kRank) return rank_cut(sh, sh.key, sh.mass, n, by_count, from, base, target);
  u64 lo = order_key(bottom, kMaxVocab - 1), hi = order_key(top, 0);
  if (!(top - bottom < 1e30f)) {
    lo = ~0ull, hi = 0;
    for (int j = threadIdx.x; j < n; j += kRowThreads) {
      lo = smaller(lo, sh.key[j]);
      hi = larger(hi, sh.key[j]);
    }
    lo = block_reduce(lo, sh, smaller);
    hi = block_reduce(hi, sh, larger);
    top = order_value(hi), bottom = order_value(lo);
  }
  auto weight = [&](int j) -> u64 { return sh.key[j] < from ? 0 : by_count ? 1ull : sh.mass[j]; };
  const float width = top - bottom;
  if (width > 0.f && width < INFINITY) {
    const float scale = static_cast<float>(kBins) / width;
    auto bin = [&](u64 k) { return kBins - 1 - min(kBins - 1, static_cast<int>((top - order_value(k)) * scale)); };
    for (int b = threadIdx.x; b < kBins; b += kRowThreads) sh.hist[b] = 0;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < n; j += kRowThreads)
      if (const u64 w = weight(j)) atomicAdd(&sh.hist[bin(sh.key[j])], w);
    __syncthreads();
    select_bin(sh, base, target);
    if (sh.digit == kBins) return 0;
    const int digit = static_cast<int>(sh.digit);
    const u64 above = sh.above;
    __syncthreads();
    u64 *key = sh.hist, *mass = sh.hist + kRank;  // (the histogram is done with)
    for (int j = threadIdx.x; j < n; j += kRowThreads) {
      if (bin(sh.key[j]) != digit) continue;
      const int at = atomicAdd(&sh.count, 1);
      if (at < kRank) {
        key[at] = sh.key[j];
        mass[at] = sh.mass[j];
      }
    }
    __syncthreads();
    if (sh.count <= kRank) return rank_cut(sh, key, mass, sh.count, by_count, from, above, target);
  }
  return radix_cut(sh, lo, hi, base, target, [&](auto f) {
    for (int j = threadIdx.x; j < n; j += kRowThreads) f(sh.key[j], weight(j));
  });
}

template <int DT>
struct Row {
  typedef RowMem<DT> Mem;
  typedef typename Mem::E E;
  Mem mem;
  double inv, m, low;

  __device__ __forceinline__ Row(const Args &a, int64_t r, const Ask &k, float most)
      : mem(a, r), inv(k.inv), m(quotient(most, k.inv)), low(k.low) {}
  // f(index, logit) for every token, in no particular order; 16-byte loads, two in flight.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int all = (mem.before + mem.V + Mem::W - 1) / Mem::W;
    typename Mem::Vec next = mem.load(min(static_cast<int>(threadIdx.x), all - 1));
#pragma unroll 1
    for (int v = threadIdx.x; v < all; v += kRowThreads) {
      const typename Mem::Vec e = next;
      next = mem.load(min(v + kRowThreads, all - 1));
#pragma unroll
      for (int j = 0; j < Mem::W; ++j) {
        const E ej = e[j];
        f(mem.first(v) + j, elem_to_f32<DT>(ej));  // (a NaN where the row has no token)
      }
    }
  }
  __device__ __forceinline__ float x(float logit) const { return quotient(logit, inv); }
  __device__ __forceinline__ double down(float x) const {
    const double d = static_cast<double>(x) - m;
    return static_cast<double>(x) == m ? 0.0 : d;  // (also where both are infinite)
  }
  // What a slice's sum is of weights below the row's largest.
  __device__ __forceinline__ double rest(const Head &h) const {
    return h.most > -INFINITY ? h.rest * exp(down(x(h.most))) : 0.0;
  }
  __device__ __forceinline__ bool alive(float x) const { return down(x) >= low; }  // (a NaN is not)
  __device__ __forceinline__ u64 mass(float x) const {
    const double d = down(x);
    if (!(d >= low)) return 0;
    // (to the nearest: the sum's last bits are those of the integer)
    return static_cast<u64>(__double_as_longlong(power64(fmax(d, -800.0)) * kMassScale + 0x1p52)) - 0x4330000000000000ull;
  }
};

// A cut over the whole row: the tokens' weights (by_count: 1 each; below `from`: none) in bins of
// 1 / 64 of x below the largest, then the tokens of the bin that holds the cut as candidates; by
// digits of the key where they are too many, or lie too far below.  share: target is one of the
// weights' sum; then `kept` is the kept tokens' weight (0 by digits, who do not have it).
template <int DT>
__device__ __forceinline__ u64 row_cut(RowShared &sh, const Row<DT> &row, bool by_count, u64 from, double target,
                                       bool share, u64 &kept) {
  constexpr float kPerX = 64.f;
  const float top = static_cast<float>(row.m);
  auto bin = [&](float x) {  // (the largest, infinite or not, in the first)
    return x == top ? kBins - 1 : kBins - 1 - static_cast<int>(fminf((top - x) * kPerX, static_cast<float>(kBins - 1)));
  };
  auto weight = [&](float x, int i) -> u64 {  // (0 for a NaN)
    return order_key(x, i) < from ? 0 : by_count ? (row.alive(x) ? 1ull : 0ull) : row.mass(x);
  };
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kRowThreads) sh.hist[b] = 0;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  row.each([&](int i, float v) {
    const float x = row.x(v);
    if (const u64 w = weight(x, i)) atomicAdd(&sh.hist[bin(x)], w);
  });
  __syncthreads();
  if (share) {
    u64 z = 0;
    for (int b = threadIdx.x; b < kBins; b += kRowThreads) z += sh.hist[b];
    kept = block_reduce(z, sh, plus);
    target *= static_cast<double>(kept);
  }
  select_bin(sh, 0, target);
  const int digit = static_cast<int>(sh.digit);
  const u64 above = sh.above;
  if (digit == kBins) return 0;
  __syncthreads();
  if (digit > 0) {
    row.each([&](int i, float v) {
      const float x = row.x(v);
      if (!(x == x) || bin(x) != digit || order_key(x, i) < from) return;
      const int at = atomicAdd(&sh.count, 1);
      if (at < kCand) sh.key[at] = order_key(x, i);
    });
    __syncthreads();
    const int n = sh.count;
    if (n <= kCand) {
      for (int j = threadIdx.x; j < n; j += kRowThreads) sh.mass[j] = weight(order_value(sh.key[j]), order_index(sh.key[j]));
      __syncthreads();
      const u64 cut = cand_cut(sh, n, by_count, from, above, target, INFINITY, 0.f);
      if (share) {
        u64 z = 0;
        for (int j = threadIdx.x; j < n; j += kRowThreads) z += sh.key[j] >= cut ? sh.mass[j] : 0;
        kept = above + block_reduce(z, sh, plus);
      }
      return cut;
    }
    __syncthreads();
  }
  kept = 0;
  return radix_cut(sh, 0, order_key(top, 0), 0, target, [&](auto f) {
    row.each([&](int i, float v) {
      const float x = row.x(v);
      if (x == x) f(order_key(x, i), weight(x, i));
    });
  });
}

// A row whose candidates do not decide it.
template <int DT>
__device__ __forceinline__ void long_way(RowShared &sh, const Row<DT> &row, const Ask &k, float *o) {
  u64 cut = 0, weight = 0;
  if (k.top_k) cut = row_cut(sh, row, true, 0, static_cast<double>(k.top_k), false, weight);
  weight = 0;
  if (k.open) cut = larger(cut, row_cut(sh, row, false, cut, static_cast<double>(k.top_p), true, weight));
  // the kept tokens as numbers: x at least `lowest`, at or before the cut's
  const float top = static_cast<float>(row.m), at = cut ? order_value(cut) : -INFINITY;
  const int last = cut ? order_index(cut) : kMaxVocab;
  float lowest = -INFINITY;
  if (k.min_p > 0.f) {
    lowest = static_cast<float>(row.m + row.low);
    if (!row.alive(lowest)) lowest = nextafterf(lowest, INFINITY);
    else if (row.alive(nextafterf(lowest, -INFINITY))) lowest = nextafterf(lowest, -INFINITY);
  }
  auto power_of = [&](int i, float v) {  // 0 if it is not kept
    const float x = row.x(v);
    return x >= lowest && (x > at || (x == at && i <= last)) ? expf(x == top ? 0.f : x - top) : 0.f;
  };
  float scale = static_cast<float>(kMassScale / static_cast<double>(weight));
  if (!weight) {
    double z = 0.0;
    row.each([&](int i, float v) { z += static_cast<double>(power_of(i, v)); });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) z += __shfl_xor(z, d);
    double *part = reinterpret_cast<double *>(sh.wave);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = z;
    __syncthreads();
    z = 0.0;
#pragma unroll
    for (int w = 0; w < kRowThreads / 64; ++w) z += part[w];
    scale = static_cast<float>(1.0 / z);
  }
  row.each([&](int i, float v) {  // (the zeros are there)
    const float e = power_of(i, v);
    if (e > 0.f) o[i] = e * scale;
  });
}

// A row without cuts: its values, groups [v0, v1) of four.
template <int DT>
__device__ __forceinline__ void whole_row(const RowMem<DT> &mem, const Ask &k, float x_most, float scale, float *o,
                                          int part, int parts) {
  typedef typename RowMem<DT>::E E;
  typedef float F4 __attribute__((ext_vector_type(4)));
  typedef E E4 __attribute__((ext_vector_type(4), aligned(sizeof(E))));
  const int V = mem.V, head = min(V, static_cast<int>((-(reinterpret_cast<uintptr_t>(o) / 4)) & 3)), groups = (V - head) / 4;
  const int g0 = static_cast<int>(static_cast<int64_t>(groups) * part / parts);
  const int g1 = static_cast<int>(static_cast<int64_t>(groups) * (part + 1) / parts);
  const float inv = 1.f / k.temp;
  auto value = [&](E e) { return power(elem_to_f32<DT>(e), k.temp, inv, k.inv, x_most) * scale; };
#pragma unroll 4
  for (int g = g0 + static_cast<int>(threadIdx.x); g < g1; g += kRowThreads) {
    const E4 a = *reinterpret_cast<const E4 *>(mem.p + head + 4 * g);
    *reinterpret_cast<F4 *>(o + head + 4 * g) = F4{value(a[0]), value(a[1]), value(a[2]), value(a[3])};
  }
  if (part == 0) {  // (at most 3 at each end)
    const int i = static_cast<int>(threadIdx.x) < head ? static_cast<int>(threadIdx.x) : -1, t = head + 4 * groups + static_cast<int>(threadIdx.x);
    if (i >= 0) o[i] = value(mem.p[i]);
    if (t < V) o[t] = value(mem.p[t]);
  }
}

// (two workgroups a CU: the registers of the long way alone would leave room for one)
template <int DT>
__global__ __launch_bounds__(kRowThreads) __attribute__((amdgpu_waves_per_eu(4))) void row_kernel(Args a) {
  __shared__ RowShared sh;
  const int tid = threadIdx.x;
  const int rows = static_cast<int>(gridDim.x / a.groups);  // (the first workgroups of all rows first)
  const int64_t r = blockIdx.x % rows;
  const int g = static_cast<int>(blockIdx.x / rows);
  const Ask k = ask(a, r);
  if (k.kind != kWhole && g) return;
  const Head *heads = a.heads + r * a.S;
  if (tid < a.S) sh.head[tid] = heads[tid];
  __syncthreads();
  // (a lane a slice here and below, in every wave)
  const int lane = tid & 63, wave = tid >> 6;
  float most = -INFINITY;
  for (int q = lane; q < a.S; q += 64) most = fmaxf(most, sh.head[q].most);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
  float *o = a.out + r * a.out_stride;
  const Row<DT> row(a, r, k, most);

  if (k.kind == kWhole) {
    if (most == -INFINITY) {
      fill_zeros(o, static_cast<int>(static_cast<int64_t>(a.V) * g / a.groups),
                 static_cast<int>(static_cast<int64_t>(a.V) * (g + 1) / a.groups), kRowThreads);
      return;
    }
    double z = 0.0;
    for (int q = lane; q < a.S; q += 64) z += row.rest(sh.head[q]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) z += __shfl_xor(z, d);
    whole_row(row.mem, k, static_cast<float>(row.m), static_cast<float>(1.0 / z), o, g, a.groups);
    return;
  }
  if (most == -INFINITY) return;
  if (k.kind == kGreedy) {
    int first = kMaxVocab;
    for (int q = lane; q < a.S; q += 64) first = sh.head[q].most == most ? min(first, sh.head[q].count) : first;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) first = min(first, __shfl_xor(first, d));
    if (tid == 0) o[first] = 1.f;
    return;
  }

  // ---- the slices' candidates, those from `whole` on up: no token there is missing ----
  const bool rest_counts = k.open && !k.top_k && !(k.min_p > 0.f);
  bool known = true;
  float whole = -INFINITY;
  double rest = 0.0;
  for (int q = lane; q < a.S; q += 64) {
    const Head h = sh.head[q];
    known = known && h.count >= 0;
    whole = fmaxf(whole, h.whole);
    if (rest_counts) rest += row.rest(h);
  }
  known = __all(known);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    whole = fmaxf(whole, __shfl_xor(whole, d));
    rest += __shfl_xor(rest, d);
  }
  u64 below = 0;  // weight of the candidates that are not kept here
  int n = 0;
  if (known) {
    if (tid == 0) sh.count = 0;
    __syncthreads();
    // a wave kChunk of a slice's candidates at a time
    constexpr int kEach = kChunk / 64;
    const int chunks = (a.cap + kChunk - 1) / kChunk;
    for (int t = wave; t < a.S * chunks; t += kRowThreads / 64) {
      const int q = t / chunks, j0 = t % chunks * kChunk, count = sh.head[q].count;
      if (j0 >= count) continue;
      const u64 *list = a.lists + (r * a.S + q) * a.cap;
      u64 key[kEach];
      uint64_t kept[kEach];
      int all = 0;
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        const int j = j0 + 64 * u + lane;
        key[u] = j < count ? list[j] : 0;
      }
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        kept[u] = __ballot(j0 + 64 * u + lane < count && order_value(key[u]) >= whole);
        all += __popcll(kept[u]);
      }
      int base = 0;
      if (lane == 0 && all) base = atomicAdd(&sh.count, all);
      base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
      for (int u = 0; u < kEach; ++u) {
        if (j0 + 64 * u >= count) break;
        const bool keep = kept[u] >> lane & 1;
        const u64 w = keep || (j0 + 64 * u + lane < count && rest_counts) ? row.mass(order_value(key[u])) : 0;
        if (keep) {
          const int at = base + __popcll(kept[u] & ((1ull << lane) - 1));
          if (at < kCand) {
            sh.key[at] = key[u];
            sh.mass[at] = w;
          }
        } else {
          below += w;
        }
        base += __popcll(kept[u]);
      }
    }
    if (rest_counts) below = block_reduce(below, sh, plus);
    __syncthreads();
    n = sh.count;
    __syncthreads();  // (a cut counts in it anew)
    // of top_k's prefix every token is there, or every survivor of min_p
    known = n <= kCand && (rest_counts || (k.top_k && n >= k.top_k) || whole == -INFINITY ||
                           row.m + row.low >= static_cast<double>(whole));
  }
  if (known && n <= kRank) {
    // ---- few: ranked, each by two threads ----
    const Place at = place(sh.key, sh.mass, n);
    const int e = tid >> 1;
    bool kept = e < n && (!k.top_k || at.rank < k.top_k);
    const u64 w = e < n ? sh.mass[e] : 0;
    u64 Z = block_reduce(kept && !(tid & 1) ? w : 0, sh, plus);
    if (k.open) {
      double lowest = static_cast<double>(Z), highest = lowest;
      if (rest_counts) {
        lowest += static_cast<double>(below) + rest * (1.0 - kPowerOff) * kMassScale;
        highest += static_cast<double>(below) + rest * (1.0 + kPowerOff) * kMassScale;
        known = static_cast<double>(k.top_p) * highest <= static_cast<double>(Z);
      }
      const double before = static_cast<double>(at.before);
      const bool other = kept && before < static_cast<double>(k.top_p) * highest;
      kept = kept && before < static_cast<double>(k.top_p) * lowest;
      known = !__syncthreads_or(kept != other || !known);
      if (known) Z = block_reduce(kept && !(tid & 1) ? w : 0, sh, plus);
    }
    if (known) {
      if (kept && !(tid & 1)) {
        const float x = order_value(sh.key[e]);
        // below 2^-20 of the largest the fixed point has fewer digits than the result
        if (row.alive(x))
          o[order_index(sh.key[e])] = static_cast<float>((w >> 24 ? static_cast<double>(w) : exp(row.down(x)) * kMassScale) /
                                                         static_cast<double>(Z));
      }
      return;
    }
  } else if (known) {
    const float top = static_cast<float>(row.m);
    auto total = [&](u64 from) {
      u64 z = 0;
      for (int j = tid; j < n; j += kRowThreads) z += sh.key[j] >= from ? sh.mass[j] : 0;
      return block_reduce(z, sh, plus);
    };
    u64 cut = k.top_k && n >= k.top_k ? cand_cut(sh, n, true, 0, 0, static_cast<double>(k.top_k), top, whole) : 0;
    u64 Z = total(cut);
    if (k.open) {
      double lowest = static_cast<double>(Z), highest = lowest;
      if (rest_counts) {
        lowest += static_cast<double>(below) + rest * (1.0 - kPowerOff) * kMassScale;
        highest += static_cast<double>(below) + rest * (1.0 + kPowerOff) * kMassScale;
      }
      const u64 c = cand_cut(sh, n, false, cut, 0, static_cast<double>(k.top_p) * lowest, top, whole);
      cut = larger(cut, c);
      Z = total(cut);
      if (rest_counts)  // the same cut for the largest sum there can be
        known = c && static_cast<double>(k.top_p) * highest <= static_cast<double>(Z);
    }
    if (known) {
      const double scale = 1.0 / static_cast<double>(Z);
      for (int j = tid; j < n; j += kRowThreads) {
        const u64 key = sh.key[j];
        const float x = order_value(key);
        if (key >= cut && row.alive(x))
          o[order_index(key)] = static_cast<float>(
              (sh.mass[j] >> 24 ? static_cast<double>(sh.mass[j]) : exp(row.down(x)) * kMassScale) * scale);
      }
      return;
    }
  }
  __syncthreads();
  long_way(sh, row, k, o);
}

struct Plan {
  int S, cap, reach, most;
  size_t heads, lists;  // bytes
};
inline Plan plan(int rows, int V, int vec) {
  Plan p;
  const int per = vec * slice_vecs(vec) * kSliceThreads;
  p.S = (V + vec - 1 + per - 1) / per;
  p.cap = std::min(kCand, ((2 * kCand / p.S) + 63) & ~63);
  // The number of threads r whose maxima reach a bound that c tokens of a slice of random order reach:
  // r = T (1 - exp(-c / T)).  Without top_k about 2,800 candidates a row, with at most 3,000.
  const auto threads = [&](double c) {
    return std::max(1, static_cast<int>(kSliceThreads * (1.0 - std::exp(-c / p.S / kSliceThreads))));
  };
  p.reach = threads(2800.0);
  p.most = threads(3000.0);
  p.heads = (static_cast<size_t>(rows) * p.S * sizeof(Head) + 15) & ~static_cast<size_t>(15);
  p.lists = static_cast<size_t>(rows) * p.S * p.cap * sizeof(u64);
  return p;
}

template <int DT>
void launch(Args a, int rows, void *workspace, hipStream_t s) {
  const Plan p = plan(rows, a.V, Elem<DT>::kVec);
  a.S = p.S;
  a.cap = p.cap;
  a.reach = p.reach;
  a.most = p.most;
  a.heads = static_cast<Head *>(workspace);
  a.lists = reinterpret_cast<u64 *>(static_cast<char *>(workspace) + p.heads);
  const unsigned grid = static_cast<unsigned>(rows) * p.S;
  slice_kernel<DT><<<grid, kSliceThreads, 0, s>>>(a);
  // Two workgroups a CU (256 CUs), which rows without cuts use, and two a row at least: 247 rows of
  // 151,936 in bf16 88 us (103 with one, 93 with four a row), 320 rows 122 us (135 with one).  (Both before
  // slices of 12,288 16-bit logits; with them 79 and 104.)
  a.groups = std::min(p.S, std::max(2, 512 / rows));
  row_kernel<DT><<<static_cast<unsigned>(rows) * a.groups, kRowThreads, 0, s>>>(a);
}

}  // namespace probs
}  // namespace spk

using namespace spk;

extern "C" size_t spk_sample_probs_workspace_bytes(int rows, int vocab) {
  if (rows <= 0 || vocab <= 0 || vocab > probs::kMaxVocab) return 0;
  size_t most = 0;
  for (int vec : {4, 8}) {  // (the logits' type is not an argument)
    const probs::Plan p = probs::plan(rows, vocab, vec);
    most = std::max(most, p.heads + p.lists);
  }
  return most;
}

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
  if (static_cast<double>(rows) * probs::plan(1, vocab, 4).S * probs::kSliceThreads > 4294967295.0)
    return fail(SPK_EUNSUPPORTED, "sample_probs: more threads than a launch has, rows=%d vocab=%d", rows, vocab);
  if (!logits || !temperature || !probs_out) return fail(SPK_EINVAL, "sample_probs: null pointer");
  const int64_t dtype_bytes = logits_dtype == SPK_F32 ? 4 : 2;
  const size_t need = spk_sample_probs_workspace_bytes(rows, vocab);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(SPK_EINVAL, "sample_probs: workspace of %zu bytes, %zu needed, aligned to 16",
                workspace ? workspace_bytes : 0, need);
  if (on_one_another(logits, row_stride * dtype_bytes, vocab * dtype_bytes, probs_out,
                     out_stride * 4, vocab * int64_t{4}, rows))
    return fail(SPK_EINVAL, "sample_probs: the output lies on the logits");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const probs::Args a{logits, row_stride, vocab, temperature, top_p, min_p, top_k, probs_out, out_stride, 0, 0, 0, 0,
                      0, nullptr, nullptr};
  if (logits_dtype == SPK_F32) probs::launch<SPK_F32>(a, rows, workspace, s);
  else if (logits_dtype == SPK_F16) probs::launch<SPK_F16>(a, rows, workspace, s);
  else probs::launch<SPK_BF16>(a, rows, workspace, s);
  return check_launch("sample_probs");
}
