// Eviction from the paged packed cache by accumulated attention weight.
//
// Per (layer, sequence, kv head): a sequence longer than the budget keeps its first
// `sinks` tokens, its last `recent` ones and, of the others, those of largest mass
// (equal masses: the lowest positions) so that `budget` stay, in their order.
//   evict_select_kernel: a workgroup a (layer, sequence, kv head) finds the smallest
//     mass that stays with a radix selection on order-preserving 32-bit keys, then
//     numbers the kept tokens with ballots and prefix sums, in position order.
//   evict_move_kernel: a workgroup a (t, kv head, K or V) plane moves the kept words
//     to positions 0, 1, ...  A kept token never moves up, so chunks in order, each
//     read whole before it is written, move in place.
#include "common.hpp"

namespace spk {
namespace evict {

constexpr int kMaxLayers = 64;  // layers a launch (kernel arguments)
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256;
constexpr int kMoveEach = 4;  // tokens a thread and chunk

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

__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(Params p) {
  __shared__ uint32_t hist[kBins];
  __shared__ int counts[2][2][kSelWaves];
  __shared__ uint32_t found[2];
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

  // The candidates' free-th largest key, and how many equal to it stay.
  const int lo = p.sinks, hi = len - p.recent;
  int free = p.budget - p.sinks - p.recent;
  uint32_t prefix = 0, mask = 0;
  if (free > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
      for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int j = lo + tid; j < hi; j += kSelThreads) {
        const uint32_t k = key_of(mass[j]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
      }
      __syncthreads();
      if (wave == 0) {  // a lane holds kBins / 64 bins, the highest first
        constexpr int kEach = kBins / 64;
        const int top = kBins - 1 - lane * kEach;
        uint32_t sum = 0;
        for (int b = 0; b < kEach; ++b) sum += hist[top - b];
        uint32_t upto = sum;
        for (int s = 1; s < 64; s <<= 1) {
          const uint32_t y = __shfl_up(upto, s);
          if (lane >= s) upto += y;
        }
        uint32_t before = upto - sum;
        if (before < static_cast<uint32_t>(free) && upto >= static_cast<uint32_t>(free)) {
          int b = 0;
          while (before + hist[top - b] < static_cast<uint32_t>(free)) before += hist[top - b++];
          found[0] = top - b;
          found[1] = free - before;
        }
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= static_cast<uint32_t>(bins - 1) << shift;
      free = found[1];
    }
  }
  const bool any = p.budget > p.sinks + p.recent;

  // Kept tokens in position order: `sure` ones, and the first `free` equal ones.
  int sure0 = 0, equal0 = 0;
  for (int j0 = 0, turn = 0; j0 < len; j0 += kSelThreads, turn ^= 1) {
    const int j = j0 + tid;
    float m = 0.f;
    bool sure = false, equal = false;
    if (j < len) {
      m = mass[j];
      const uint32_t k = key_of(m);
      const bool edge = j < lo || j >= hi;
      sure = edge || (any && k > prefix);
      equal = !edge && any && k == prefix;
    }
    const uint64_t sb = __ballot(sure), eb = __ballot(equal);
    if (lane == 0) {
      counts[turn][0][wave] = __popcll(sb);
      counts[turn][1][wave] = __popcll(eb);
    }
    __syncthreads();
    int s = sure0, e = equal0;
    for (int w = 0; w < kSelWaves; ++w) {
      const int cs = counts[turn][0][w], ce = counts[turn][1][w];
      if (w < wave) {
        s += cs;
        e += ce;
      }
      sure0 += cs;
      equal0 += ce;
    }
    const uint64_t below = (1ull << lane) - 1;
    s += __popcll(sb & below);
    e += __popcll(eb & below);
    if (sure || (equal && e < free)) {
      const int at = s + min(e, free);
      keep[at] = j;
      to[at] = m;
    }
  }
  __syncthreads();
  for (int j = kept + tid; j < p.cap; j += kSelThreads) to[j] = 0.f;
}

template <int W>
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(Params p) {
  const int which = blockIdx.x & 1, h = (blockIdx.x >> 1) % p.Hkv, t = (blockIdx.x >> 1) / p.Hkv;
  const int n = blockIdx.y;
  const int len = length(p, n), kept = min(len, p.budget);
  if (p.in_place && len <= p.budget) return;
  const int32_t *keep = p.keep + ((static_cast<int64_t>(p.layer0 + blockIdx.z) * p.N + n) * p.Hkv + h) * p.budget;
  uint32_t *base = p.kv[blockIdx.z][which] + t * p.ks0 + h * p.ks1;
  const int64_t blocks = p.num_slots >> p.bs_log2;
  const int bs_mask = (1 << p.bs_log2) - 1;
  auto slot = [&](const int32_t *table, int64_t stride, int pos) -> int64_t {
    const int64_t phys = table[(pos >> p.bs_log2) * stride];
    return phys < 0 || phys >= blocks ? -1 : (phys << p.bs_log2) | (pos & bs_mask);
  };
  for (int i0 = 0; i0 < kept; i0 += kMoveThreads * kMoveEach) {
    uint32_t x[kMoveEach][W];
    int64_t dst[kMoveEach];
#pragma unroll
    for (int e = 0; e < kMoveEach; ++e) {
      const int i = i0 + e * kMoveThreads + threadIdx.x;
      dst[e] = -1;
      if (i >= kept || i >= p.max_dst) continue;
      const int64_t src = slot(p.bt + n * p.bts0, p.bts1, keep[i]);
      dst[e] = slot(p.dt + n * p.dts0, p.dts1, i);
      if (src == dst[e]) dst[e] = -1;
#pragma unroll
      for (int w = 0; w < W; ++w) x[e][w] = src < 0 ? 0u : base[src * p.ks2 + w];
    }
    __builtin_amdgcn_s_waitcnt(0);  // the chunk's words are here before any is overwritten
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kMoveEach; ++e)
      if (dst[e] >= 0)
#pragma unroll
        for (int w = 0; w < W; ++w) base[dst[e] * p.ks2 + w] = x[e][w];
  }
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
    evict::evict_select_kernel<<<dim3(Hkv, N, m), evict::kSelThreads, 0, s>>>(p);
    int rc = check_launch("evict");
    if (rc) return rc;
    const dim3 grid(2 * T * Hkv, N, m);
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
