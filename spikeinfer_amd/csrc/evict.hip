// Eviction from the paged packed cache by accumulated attention weight.
//
// Per (layer, sequence, kv head): a sequence longer than the budget keeps its first
// `sinks` tokens, its last `recent` ones and, of the others, those of largest mass
// (equal masses: the lowest positions) so that `budget` stay, in their order.
//   evict_select_kernel: a workgroup a (layer, sequence, kv head) finds the smallest
//     mass that stays with a radix selection (11, 11 and 10 bits) on order-preserving
//     32-bit keys, then numbers the kept tokens with ballots and one prefix sum, in position
//     order.  The masses are read once and stay in registers, EACH to a thread, up to
//     32,768 tokens.
//   evict_move_kernel: a workgroup a kv head and two timesteps moves the kept words of K
//     and V to positions 0, 1, ...: slots are worked out once for the four planes.  A kept
//     token never moves up, so chunks in order, each read whole before it is written, move
//     in place.
// Six layers of 32 sequences of 1,500..12,000 tokens cut to 2,048 (4 timesteps, 2 kv heads of
// 64 channels) take 32 + 54 us.  The selection is bound by vector instructions (its units are busy
// 64 % of the time) and barriers.
// The move touches nearly every 64-byte line of the sequences (three of ten tokens stay, eight
// lie in a line), 166 MB, and writes 50: 4.0 TB/s of lines, and other shapes of its
// workgroups (256..1024 threads, 1..4 timesteps) measure the same within 2 % or slower.
#include "common.hpp"

namespace spk {
namespace evict {

constexpr int kMaxLayers = 64;  // layers a launch (kernel arguments)
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMoveEach = 4;  // tokens a thread and chunk
constexpr int kMoveSteps = 2; // timesteps a workgroup

struct Params {
  const float *mass;
  float *mass_out;
  int64_t ms0, ms1, ms2;  // layer, sequence, kv head
  int64_t os0, os1, os2;
  int cap;
  const int32_t *lens;
  int32_t *new_lens, *keep;
  int budget, sinks, recent;
  int N, Hkv, T, W, bs_log2;
  int max_tokens;  // what a block table addresses
  const int32_t *bt, *dt;
  int64_t bts0, bts1, dts0, dts1;
  int max_dst;  // tokens that a destination table addresses
  int in_place;
  int64_t ks0, ks1, ks2;
  int64_t num_slots;
  int layer0;
  uint32_t *kv[kMaxLayers][2];
};

__device__ __forceinline__ int length(const Params &p, int n) {
  return min(max(p.lens[n], 0), min(p.cap, p.max_tokens));
}

// Order-preserving key of a mass; -0 as +0, NaN below everything.
__device__ __forceinline__ uint32_t key_of(float m) {
  const uint32_t u = __float_as_uint(m + 0.f);
  if (m != m) return 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive sum of x over the workgroup's threads, in thread order; `total` by all.
__device__ __forceinline__ uint32_t block_sum(uint32_t x, int lane, int wave, uint32_t *waves, uint32_t &total) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const uint32_t y = __shfl_up(x, s);
    if (lane >= s) x += y;
  }
  if (lane == 63) waves[wave] = x;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    const uint32_t y = waves[w];
    before += w < wave ? y : 0;
    total += y;
  }
  return before + x;
}

// EACH: masses a thread keeps in registers (EACH * kSelThreads tokens at most); 0: none, they
// are read again where they are needed.
template <int EACH>
__global__ __launch_bounds__(kSelThreads) __attribute__((amdgpu_waves_per_eu(EACH <= 16 ? 8 : 4))) void
evict_select_kernel(Params p) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t counts[EACH ? EACH * kSelWaves : 2 * kSelWaves], waves[2][kSelWaves], found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int h = blockIdx.x, n = blockIdx.y, layer = p.layer0 + blockIdx.z;
  const int len = length(p, n), kept = min(len, p.budget);
  const float *mass = p.mass + layer * p.ms0 + n * p.ms1 + h * p.ms2;
  float *to = p.mass_out + layer * p.os0 + n * p.os1 + h * p.os2;
  int32_t *keep = p.keep + ((static_cast<int64_t>(layer) * p.N + n) * p.Hkv + h) * p.budget;
  if (h == 0 && layer == 0 && tid == 0) p.new_lens[n] = kept;

  if (len <= p.budget) {
    for (int j = tid; j < p.budget; j += kSelThreads) keep[j] = j < len ? j : -1;
    for (int j = tid; j < p.cap; j += kSelThreads)
      if (j >= len) to[j] = 0.f;
      else if (to != mass) to[j] = mass[j];
    return;
  }

  float m[EACH ? EACH : 1];
  uint32_t key[EACH ? EACH : 1];
  if constexpr (EACH > 0) {
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (i * kSelThreads < len) m[i] = mass[min(i * kSelThreads + tid, len - 1)];
#pragma unroll
    for (int i = 0; i < EACH; ++i)
      if (i * kSelThreads < len) key[i] = key_of(m[i]);
  }
  // The candidates' free-th largest key, and how many equal to it stay.
  const int lo = p.sinks, hi = len - p.recent;
  int free = p.budget - p.sinks - p.recent;
  const bool any = free > 0;
  uint32_t prefix = 0, mask = 0;
  if (any) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      auto count = [&](int j, uint32_t k, bool inside) {
        if ((inside || (j >= lo && j < hi)) && (k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
      };
      if constexpr (EACH > 0) {
#pragma unroll
        for (int i = 0; i < EACH; ++i)
          if (i * kSelThreads >= lo && (i + 1) * kSelThreads <= hi) count(0, key[i], true);
          else if (i * kSelThreads < hi) count(i * kSelThreads + tid, key[i], false);
      } else {
        for (int j0 = 0; j0 < len; j0 += 8 * kSelThreads) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = mass[min(j0 + i * kSelThreads + tid, len - 1)];
#pragma unroll
          for (int i = 0; i < 8; ++i) count(j0 + i * kSelThreads + tid, key_of(x[i]), false);
        }
      }
      __syncthreads();
      // thread t holds bins top and top - 1, the highest first
      const int top = kBins - 1 - 2 * tid;
      const uint32_t c0 = hist[top], c1 = hist[top - 1];
      uint32_t total;
      const uint32_t upto = block_sum(c0 + c1, lane, wave, waves[pass & 1], total), need = free;
      const uint32_t before = upto - c0 - c1;
      if (before < need && upto >= need) {  // one thread
        const bool first = before + c0 >= need;
        found[0] = first ? top : top - 1;
        found[1] = need - before - (first ? 0 : c0);
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= static_cast<uint32_t>(bins - 1) << shift;
      free = static_cast<int>(found[1]);
    }
  }

  // Kept tokens in position order: `sure` ones, and the first `free` equal ones.
  auto look = [&](int j, uint32_t k, bool &sure, bool &equal) {
    const bool edge = j < len && (j < lo || j >= hi), in = j >= lo && j < hi && any;
    sure = edge || (in && k > prefix);
    equal = in && k == prefix;
  };
  const uint64_t below = (1ull << lane) - 1;
  if constexpr (EACH > 0) {
    // a wave's counts of each of its EACH chunks, sure ones in the low half, then one sum
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (i * kSelThreads >= len) {
        if (lane == 0) counts[i * kSelWaves + wave] = 0;
        continue;
      }
      bool sure, equal;
      look(i * kSelThreads + tid, key[i], sure, equal);
      const uint64_t sb = __ballot(sure), eb = __ballot(equal);
      if (lane == 0) counts[i * kSelWaves + wave] = __popcll(sb) | __popcll(eb) << 16;
    }
    __syncthreads();
    const uint32_t mine = tid < EACH * kSelWaves ? counts[tid] : 0;
    uint32_t total;
    const uint32_t upto = block_sum(mine, lane, wave, waves[1], total);  // (halves stay below 2^16)
    if (tid < EACH * kSelWaves) counts[tid] = upto - mine;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int j = i * kSelThreads + tid;
      if (i * kSelThreads >= len) break;
      bool sure, equal;
      look(j, key[i], sure, equal);
      const uint64_t sb = __ballot(sure), eb = __ballot(equal);
      const uint32_t base = counts[i * kSelWaves + wave];
      const int s = (base & 0xffff) + __popcll(sb & below), e = (base >> 16) + __popcll(eb & below);
      if (sure || (equal && e < free)) {
        const int at = s + min(e, free);
        keep[at] = j;
        to[at] = m[i];
      }
    }
  } else {
    int sure0 = 0, equal0 = 0;
    for (int j0 = 0, turn = 0; j0 < len; j0 += kSelThreads, turn ^= 1) {
      const int j = j0 + tid;
      const float x = mass[min(j, len - 1)];
      bool sure, equal;
      look(j, key_of(x), sure, equal);
      const uint64_t sb = __ballot(sure), eb = __ballot(equal);
      if (lane == 0) counts[turn * kSelWaves + wave] = __popcll(sb) | __popcll(eb) << 16;
      __syncthreads();  // (all of the chunk is read: what is written below lies in it or before)
      int s = sure0, e = equal0;
      for (int w = 0; w < kSelWaves; ++w) {
        const int cs = counts[turn * kSelWaves + w] & 0xffff, ce = counts[turn * kSelWaves + w] >> 16;
        if (w < wave) {
          s += cs;
          e += ce;
        }
        sure0 += cs;
        equal0 += ce;
      }
      s += __popcll(sb & below);
      e += __popcll(eb & below);
      if (sure || (equal && e < free)) {
        const int at = s + min(e, free);
        keep[at] = j;
        to[at] = x;
      }
    }
    __syncthreads();
  }
  for (int j = kept + tid; j < p.cap; j += kSelThreads) to[j] = 0.f;
}

// A token's W words, one access (they need no more than a word's alignment).
template <int W> struct Words;
template <> struct Words<1> { typedef uint32_t type; };
template <> struct Words<2> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(4))); };
template <> struct Words<3> { typedef uint32_t type __attribute__((ext_vector_type(3), aligned(4))); };
template <> struct Words<4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4))); };

template <int W>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(Params p) {
  typedef typename Words<W>::type Token;
  const int h = blockIdx.x % p.Hkv, t0 = blockIdx.x / p.Hkv * kMoveSteps, n = blockIdx.y;
  const int len = length(p, n), kept = min(len, p.budget);
  if (p.in_place && len <= p.budget) return;
  const int32_t *keep = p.keep + ((static_cast<int64_t>(p.layer0 + blockIdx.z) * p.N + n) * p.Hkv + h) * p.budget;
  uint32_t *plane[2 * kMoveSteps];
#pragma unroll
  for (int i = 0; i < 2 * kMoveSteps; ++i)
    plane[i] = p.kv[blockIdx.z][i & 1] + min(t0 + i / 2, p.T - 1) * p.ks0 + h * p.ks1;
  const int64_t blocks = p.num_slots >> p.bs_log2;
  const int bs_mask = (1 << p.bs_log2) - 1;
  const int last = min(kept, p.max_dst) - 1;
  for (int i0 = 0; i0 <= last; i0 += kMoveThreads * kMoveEach) {
    int64_t src[kMoveEach], dst[kMoveEach];
#pragma unroll
    for (int e = 0; e < kMoveEach; ++e) {
      const int i = min(i0 + e * kMoveThreads + static_cast<int>(threadIdx.x), last);
      const int from = keep[i];
      const int64_t a = p.bt[n * p.bts0 + (from >> p.bs_log2) * p.bts1], b = p.dt[n * p.dts0 + (i >> p.bs_log2) * p.dts1];
      src[e] = a < 0 || a >= blocks ? -1 : ((a << p.bs_log2) | (from & bs_mask)) * p.ks2;
      dst[e] = b < 0 || b >= blocks || i0 + e * kMoveThreads + static_cast<int>(threadIdx.x) > last
                   ? -1 : ((b << p.bs_log2) | (i & bs_mask)) * p.ks2;
      if (src[e] == dst[e]) dst[e] = -1;
    }
    Token x[2 * kMoveSteps][kMoveEach];
#pragma unroll
    for (int k = 0; k < 2 * kMoveSteps; ++k)
#pragma unroll
      for (int e = 0; e < kMoveEach; ++e) {
        x[k][e] = Token(0);
        if (src[e] >= 0 && dst[e] >= 0) __builtin_memcpy(&x[k][e], plane[k] + src[e], 4 * W);
      }
    __builtin_amdgcn_s_waitcnt(0);  // the chunk's words are here before any is overwritten
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2 * kMoveSteps; ++k) {
      if (t0 + k / 2 >= p.T) continue;
#pragma unroll
      for (int e = 0; e < kMoveEach; ++e)
        if (dst[e] >= 0) __builtin_memcpy(plane[k] + dst[e], &x[k][e], 4 * W);
    }
  }
}

// Masses in registers as the longest sequence needs them, against reading them five times
// (evictions captured and replayed): 2 a thread 13.4 us, reading 18.2, 32 a thread 28.9 (one layer,
// 2,000 tokens to 512); 8 a thread 30.4, 16 a thread 34.2, reading 40.3 (one layer of 8,000 to
// 2,048); 16 a thread 79, reading 101, 32 a thread (one workgroup a CU) 104 (the six layers above);
// 32 a thread 55, reading 72 (one layer of 20,000 to 4,096), and 205, reading 245 (six layers of
// 32 sequences of 17,000..32,768 to 2,048).
static void launch_select(const Params &p, dim3 grid, hipStream_t s) {
  const int tokens = p.cap < p.max_tokens ? p.cap : p.max_tokens;  // the longest sequence
  if (tokens <= 2 * kSelThreads) evict_select_kernel<2><<<grid, kSelThreads, 0, s>>>(p);
  else if (tokens <= 8 * kSelThreads) evict_select_kernel<8><<<grid, kSelThreads, 0, s>>>(p);
  else if (tokens <= 16 * kSelThreads) evict_select_kernel<16><<<grid, kSelThreads, 0, s>>>(p);
  else if (tokens <= 32 * kSelThreads) evict_select_kernel<32><<<grid, kSelThreads, 0, s>>>(p);
  else evict_select_kernel<0><<<grid, kSelThreads, 0, s>>>(p);
}

}  // namespace evict
}  // namespace spk

using namespace spk;

extern "C" int spk_evict(const SpkCacheLayer *layers, int nlayers, const int64_t cache_strides[3], int64_t num_slots,
                         const float *mass, const int64_t mass_strides[3], float *mass_out,
                         const int64_t mass_out_strides[3], int64_t cap, const int32_t *block_tables,
                         int64_t bt_stride0, int64_t bt_stride1, int max_blocks, const int32_t *dst_tables,
                         int64_t dt_stride0, int64_t dt_stride1, int max_dst_blocks, const int32_t *seq_lens,
                         int32_t *new_lens, int32_t *keep, int budget, int sinks, int recent, int T, int N, int Hkv,
                         int head_dim, int block_size, void *stream) {
  if (nlayers < 0 || T <= 0 || N < 0 || Hkv <= 0 || head_dim <= 0 || cap < 0 || max_blocks < 0 || num_slots < 0 ||
      max_dst_blocks < 0)
    return fail(SPK_EINVAL, "evict: bad sizes layers=%d T=%d N=%d Hkv=%d D=%d", nlayers, T, N, Hkv, head_dim);
  if (budget <= 0 || sinks < 0 || recent < 0 || static_cast<int64_t>(sinks) + recent > budget)
    return fail(SPK_EINVAL, "evict: budget=%d does not hold %d first and %d last tokens", budget, sinks, recent);
  if (head_dim > 128) return fail(SPK_EUNSUPPORTED, "evict: head_dim=%d (at most 128)", head_dim);
  if (!is_pow2(block_size)) return fail(SPK_EINVAL, "evict: block_size=%d is not a power of two", block_size);
  const int64_t tokens = static_cast<int64_t>(max_blocks) * block_size;
  const int64_t room = dst_tables ? static_cast<int64_t>(max_dst_blocks) * block_size : tokens;
  if (tokens > (1 << 30) || cap > (1 << 30) || room > (1 << 30) || budget > (1 << 30))
    return fail(SPK_EUNSUPPORTED, "evict: sequences of %lld tokens (at most 2^30)", (long long)tokens);
  if (room < budget && room < tokens)
    return fail(SPK_EINVAL, "evict: destination tables of %lld tokens for a budget of %d", (long long)room, budget);
  if (nlayers == 0 || N == 0) return SPK_OK;
  if (N > 65535 || static_cast<int64_t>(T) * Hkv > (1 << 16))
    return fail(SPK_EUNSUPPORTED, "evict: N=%d T=%d Hkv=%d", N, T, Hkv);
  if (!layers || !seq_lens || !new_lens || !keep || (cap > 0 && (!mass || !mass_out)) || (tokens > 0 && !block_tables))
    return fail(SPK_EINVAL, "evict: null pointer");
  for (int i = 0; i < nlayers; ++i)
    if (num_slots > 0 && (!layers[i].k || !layers[i].v)) return fail(SPK_EINVAL, "evict: null pointer in layer %d", i);
  if ((T > 1 && !cache_strides[0]) || (Hkv > 1 && !cache_strides[1]) || (num_slots > 1 && !cache_strides[2]))
    return fail(SPK_EINVAL, "evict: words of a cache lie on one another");
  if (cap > 0 && ((nlayers > 1 && !mass_out_strides[0]) || (N > 1 && !mass_out_strides[1]) || (Hkv > 1 && !mass_out_strides[2])))
    return fail(SPK_EINVAL, "evict: rows of mass_out lie on one another");
  const int twice = shared_cache(num_slots > 0 ? nlayers : 0, [&](int i) { return std::make_pair(layers[i].k, layers[i].v); });
  if (twice >= 0) return fail(SPK_EINVAL, "evict: layer %d has one cache twice, or another layer's", twice);
  evict::Params p{};
  p.mass = mass; p.ms0 = mass_strides[0]; p.ms1 = mass_strides[1]; p.ms2 = mass_strides[2];
  p.mass_out = mass_out; p.os0 = mass_out_strides[0]; p.os1 = mass_out_strides[1]; p.os2 = mass_out_strides[2];
  p.cap = static_cast<int>(cap); p.lens = seq_lens; p.new_lens = new_lens; p.keep = keep;
  p.budget = budget; p.sinks = sinks; p.recent = recent;
  p.N = N; p.Hkv = Hkv; p.T = T; p.W = (head_dim + 31) / 32; p.bs_log2 = ilog2(block_size);
  p.max_tokens = static_cast<int>(tokens);
  p.bt = block_tables; p.bts0 = bt_stride0; p.bts1 = bt_stride1;
  p.in_place = !dst_tables;
  p.dt = dst_tables ? dst_tables : block_tables;
  p.dts0 = dst_tables ? dt_stride0 : bt_stride0;
  p.dts1 = dst_tables ? dt_stride1 : bt_stride1;
  p.max_dst = static_cast<int>(room);
  p.ks0 = cache_strides[0]; p.ks1 = cache_strides[1]; p.ks2 = cache_strides[2];
  p.num_slots = num_slots;
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (int i = 0; i < nlayers; i += evict::kMaxLayers) {
    const int m = nlayers - i < evict::kMaxLayers ? nlayers - i : evict::kMaxLayers;
    p.layer0 = i;
    for (int k = 0; k < m; ++k) {
      p.kv[k][0] = reinterpret_cast<uint32_t *>(layers[i + k].k);
      p.kv[k][1] = reinterpret_cast<uint32_t *>(layers[i + k].v);
    }
    evict::launch_select(p, dim3(Hkv, N, m), s);
    int rc = check_launch("evict");
    if (rc) return rc;
    const dim3 grid((T + evict::kMoveSteps - 1) / evict::kMoveSteps * Hkv, N, m);
    switch (p.W) {
      case 1: evict::evict_move_kernel<1><<<grid, evict::kMoveThreads, 0, s>>>(p); break;
      case 2: evict::evict_move_kernel<2><<<grid, evict::kMoveThreads, 0, s>>>(p); break;
      case 3: evict::evict_move_kernel<3><<<grid, evict::kMoveThreads, 0, s>>>(p); break;
      default: evict::evict_move_kernel<4><<<grid, evict::kMoveThreads, 0, s>>>(p); break;
    }
    rc = check_launch("evict");
    if (rc) return rc;
  }
  return SPK_OK;
}
