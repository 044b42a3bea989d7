// Attention weight that the cached tokens of a sequence get from its last rows.
//
// Row i of a sequence's m rows is the token at position len - m + i and sees the
// positions up to its own:
//   mass[n, g, j] (+)= sum over t, query heads h of kv head g, rows i of
//                      exp(popc(q & k_j) * scale) / sum_j' exp(popc(q & k_j') * scale).
// Of more than max_rows rows the last max_rows count; rows that the buffer lacks never do.
//
// MI355X design: scores of 16 rows and 16 keys are one fp4 product over 128 channels
// (v_mfma_scale_f32_16x16x128_f8f6f4, a spike of both as 1, block scales that leave the
// score's table offset in the accumulator's bits, as spike_tiles.hpp has it), a weight is a
// look-up in LDS.  128 channels are 4 / WP timesteps of a head (WP: words of a head, a power
// of two): a product's 16 rows are 4 * WP of each of these timesteps, whose words stand in
// their own quarter or half of the channels beside zeros, so that decoding (7 rows of 4
// timesteps at 64 channels) fills 14 of 16 rows and every lane loads one word of a key.
//   Few rows (a decode step): a workgroup takes kPart keys, their words requested at once and
//     kept, and all row tiles, one a timestep group.  One launch sums the rows' weights (keys
//     as the product's rows: a lane adds its own row's weights), another adds the parts' sums
//     in their order, then the weights over them (keys as its columns: a lane adds its own
//     key's); with one part a single launch does both.
//   Many rows: den_rows_kernel has kPart keys in its waves' registers and goes through kRows row
//     tiles; mass_rows_kernel has 128 keys, and its waves share the row tiles.
// The order of all sums is the sequence's own, whatever the batch.
//
// Bound by instruction issue and latency: 4 timesteps, 14 query and 2 kv heads of 64 channels,
// one row of each of 64 sequences of 4,096..16,384 tokens takes 17.7 + 21.6 us a dispatch (42 MB of
// keys, read twice, the second time mostly from the caches: 2.1 TB/s), where vector units are busy
// 52 % of the time: a product has 24 vector instructions beside it, four look-ups and their sums
// and the key's five.  The rest is the chain lengths, table, words, LDS table, barrier, with
// nothing under it.  Windows of up to 32 rows of 8 sequences of 2,000..8,000 tokens take 18.1 +
// 20.9 us, vector units busy 62 and 55 %.
#include <type_traits>

#include "spike_tiles.hpp"

namespace spk {
namespace mass {

using namespace tiles;

constexpr int kStep = 64;      // keys a wave takes at once: four products' columns
constexpr int kPart = 1024;    // keys of a partial sum
// Waves that share kPart keys, each with kSteps steps.  Of 4, 8 and 16 (captured and replayed):
// 10.9, 10 and 9..11 us for a row of 700 tokens, 40.6, 41.0 and 55.4 for one of each of 64 sequences
// of 4,096..16,384.
constexpr int kWaves = 8;
constexpr int kSteps = kPart / (kWaves * kStep);
constexpr int kRows = 4;       // many rows: row tiles of a workgroup
constexpr int kShare = 4;      // waves that share the row tiles of their keys
constexpr int kMassKeys = 128;
constexpr int kChunk = 64;     // row tiles whose denominators are in LDS

struct Params {
  const uint32_t *q;           // words of (t, row, query head)
  int64_t qs0, qs1, qs2;
  const uint32_t *k;           // cache (t, kv head, slot)
  int64_t ks0, ks1, ks2;
  int64_t num_slots;
  const int32_t *bt;
  int64_t bts0, bts1;
  const int32_t *lens, *starts;
  float *mass;
  int64_t ms0, ms1, cap;
  int accumulate;
  int64_t rows;
  uint32_t rep_mul;            // inverse_of(nrep)
  int N, max_rows, T, Hkv, nrep, W, D, bs_log2, max_blocks;
  int tgroups;                 // timestep groups
  int rtiles;                  // most row tiles of a timestep group
  int parts;                   // most parts of a sequence
  float *den;                  // [N, Hkv, parts, tgroups, rtiles, 16]
  float tab[kTab];             // exp((s - D) * scale)
};

struct Seq {
  int64_t first;
  int m, len, parts;
  int open;    // the position of the first row: keys up to it are seen by all rows
  int rtiles;  // row tiles of a timestep group
};

template <int WP>
__device__ __forceinline__ Seq sequence(const Params &p, int n) {
  Seq s;
  const int64_t a = p.starts ? p.starts[n] : n, e = p.starts ? max<int64_t>(p.starts[n + 1], a) : n + 1;
  s.first = max(max<int64_t>(a, e - p.max_rows), 0);
  s.m = static_cast<int>(max<int64_t>(min(e, p.rows) - s.first, 0));
  s.len = min(max(p.lens[n], 0), p.max_blocks << p.bs_log2);
  s.open = s.len - static_cast<int>(max<int64_t>(e - s.first, 0));
  s.parts = (s.len + kPart - 1) / kPart;
  s.rtiles = (s.m * p.nrep + 4 * WP - 1) / (4 * WP);
  return s;
}

__device__ __forceinline__ int row_of(const Params &p, int r) {  // r / nrep
  return p.nrep == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), p.rep_mul));
}

// Row tile `rt` of a timestep group: its rows 4 * WP * rt .. of each timestep.  A product's row
// y: timestep y / (4 * WP) of the group, row y % (4 * WP) of the tile.
template <int WP>
__device__ __forceinline__ int tile_row(const Params &p, int rt, int y) {  // of the sequence's rows
  return row_of(p, rt * 4 * WP + y % (4 * WP));
}
template <int WP>
__device__ __forceinline__ bool has_row(const Params &p, const Seq &s, int tg, int rt, int y) {
  return tile_row<WP>(p, rt, y) < s.m && tg * (4 / WP) + y / (4 * WP) < p.T;
}

// 32 bits as 32 fp4 values, 8 of each 4th bit: a key's bits stay where they are (0.5, 1 and 2,
// and the sign's at 2), the query's hold what makes their products 1.
__device__ __forceinline__ v8i key_bits(uint32_t w) {
  v8i r = {};
  r[0] = static_cast<int>(w & 0x11111111u);
  r[1] = static_cast<int>(w & 0x22222222u);
  r[2] = static_cast<int>(w & 0x44444444u);
  r[3] = static_cast<int>(w >> 1 & 0x44444444u);
  return r;
}
__device__ __forceinline__ v8i query_bits(uint32_t w) {
  v8i r = {};
  r[0] = static_cast<int>(w << 2 & 0x44444444u);
  r[1] = static_cast<int>(w & 0x22222222u);
  r[2] = static_cast<int>(w >> 2 & 0x11111111u);
  r[3] = static_cast<int>(w >> 3 & 0x11111111u);
  return r;
}

// A lane's query word of a row tile (row l % 16, block l / 16 of the product's channels).
template <int WP>
__device__ __forceinline__ uint32_t query_word(const Params &p, const Seq &s, int kvh, int tg, int rt, int lane) {
  const int y = lane & 15, dt = y / (4 * WP), t = tg * (4 / WP) + dt, w = (lane >> 4) - dt * WP;
  const int r = rt * 4 * WP + y % (4 * WP), row = row_of(p, r);
  const bool in = row < s.m && t < p.T && w >= 0 && w < WP && w < p.W;
  const uint32_t x =
      p.q[in ? t * p.qs0 + (s.first + row) * p.qs1 + (kvh * p.nrep + r - row * p.nrep) * p.qs2 + w : int64_t(0)];
  return in ? x : 0u;
}

// A lane's words of a step's four key tiles (lane l: key l % 16 of a tile, block l / 16 of
// the product's channels).  Keys behind the sequence read its last block, what they give is
// dropped; so is, by the queries' zeros, what a block of no timestep or word gives.
// PAGE: blocks are of 16 slots or more, a key tile lies in one and its place is scalar (41.0 us
// where lanes' own places take 43.5, 64 sequences of 4,096..16,384 tokens, captured and replayed;
// with many rows there is no difference).
template <int WP, bool PAGE>
struct Keys {
  const Params &p;
  const int32_t *table;
  const uint32_t *base;
  uint32_t nblocks;
  int last_block, y;
  struct Places {
    int64_t at[4];
    bool ok[4];
  };
  __device__ __forceinline__ Keys(const Params &p, const Seq &s, int n, int kvh, int lane) : p(p) {
    table = p.bt + n * p.bts0;
    base = p.k + kvh * p.ks1;
    nblocks = static_cast<uint32_t>(min<int64_t>(p.num_slots >> p.bs_log2, 0xffffffffll));
    last_block = (s.len - 1) >> p.bs_log2;
    y = lane & 15;
  }
  __device__ __forceinline__ const uint32_t *words(int tg, int lane) const {
    const int t = tg * (4 / WP) + (lane >> 4) / WP, w = (lane >> 4) % WP;
    const uint32_t *at = base + (t < p.T ? t : 0) * p.ks0 + (w < p.W ? w : 0);
    return PAGE ? at + y * p.ks2 : at;
  }
  __device__ __forceinline__ Places places(int j0) const {
    Places r;
    uint32_t phys[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + 16 * u + (PAGE ? 0 : y);
      phys[u] = static_cast<uint32_t>(table[min(j >> p.bs_log2, last_block) * p.bts1]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + 16 * u + (PAGE ? 0 : y);
      if constexpr (PAGE) phys[u] = __builtin_amdgcn_readfirstlane(phys[u]);
      r.ok[u] = phys[u] < nblocks;
      r.at[u] = r.ok[u] ? ((static_cast<int64_t>(phys[u]) << p.bs_log2) | (j & ((1 << p.bs_log2) - 1))) * p.ks2 : 0;
    }
    return r;
  }
};

__device__ __forceinline__ v4f score(const v8i &a, const v8i &b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{}, 4, 4, 0, 54, 0, 53);
}

__device__ __forceinline__ float weight(uint32_t tab0, float score) {
  return *reinterpret_cast<const SPK_LDS float *>(static_cast<uintptr_t>(tab0 + __float_as_uint(score)));
}

// What 16 keys at j give a row's denominator (lane: row l % 16, keys j + 4 * (l / 16) + 0..3;
// `lim`: the last key that the row sees).
template <bool MASK>
__device__ __forceinline__ float row_weights(uint32_t tab0, const v8i &q, const v8i &k, int j, int lane, int lim) {
  const v4f a = score(k, q);
  float w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = weight(tab0, a[e]);
    if (MASK) w[e] = j + 4 * (lane >> 4) + e <= lim ? w[e] : 0.f;
  }
  return (w[0] + w[1]) + (w[2] + w[3]);
}

// What a tile's rows 4 * (l / 16) + 0..3 give a lane's key j.
template <bool MASK>
__device__ __forceinline__ float key_weights(uint32_t tab0, const v8i &q, const v8i &k, int j, const v4f &inv,
                                             const int (&lim)[4], float sum) {
  const v4f a = score(q, k);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float w = weight(tab0, a[e]);
    if (MASK) w = j <= lim[e] ? w : 0.f;
    sum = __builtin_fmaf(w, inv[e], sum);
  }
  return sum;
}

// Sum of the parts' denominators, in their order.
__device__ __forceinline__ float parts_sum(const Params &p, const Seq &s, const float *at) {
  float d = 0.f;
  for (int pt = 0; pt < s.parts; pt += 8) {  // eight on their way at once
    float y[8];
#pragma unroll
    for (int v = 0; v < 8; ++v)
      y[v] = at[static_cast<int64_t>(min(pt + v, s.parts - 1)) * p.tgroups * p.rtiles * 16];
#pragma unroll
    for (int v = 0; v < 8; ++v) d += pt + v < s.parts ? y[v] : 0.f;
  }
  return d;
}

enum Pass { kDen, kMass, kBoth };

// Few rows: one row tile for each of RT or fewer timestep groups.
template <int WP, int RT, bool PAGE, Pass PASS>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(4))) void few_rows_kernel(Params p) {
  struct Smem {
    float tab[kTab + 3];  // first: a score's accumulator is its entry's LDS address
    float sum[kWaves][RT][16];
    float inv[RT][16];
  };
  __shared__ Smem sm;
  const uint32_t tab0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPK_LDS char *)(void *)sm.tab));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.y % p.Hkv, n = blockIdx.y / p.Hkv;
  const Seq s = sequence<WP>(p, n);
  const int64_t from = static_cast<int64_t>(blockIdx.x) * kPart;
  float *mass = p.mass + n * p.ms0 + kvh * p.ms1;
  if constexpr (PASS != kDen) {
    if (!p.accumulate)
      for (int64_t j = max<int64_t>(from, s.rtiles ? s.len : 0) + tid; j < min(p.cap, from + kPart); j += kWaves * 64)
        mass[j] = 0.f;
  }
  if (from >= s.len || s.rtiles == 0) return;
  if (tid <= p.D) sm.tab[tid] = p.tab[tid];

  const Keys<WP, PAGE> keys(p, s, n, kvh, lane);
  const int j1 = static_cast<int>(from) + wave * kStep;
  uint32_t x[kSteps][RT][4];
  bool ok[kSteps][4];
  float old[kSteps];
  {
    const uint32_t *at[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) at[i] = keys.words(min(i, p.tgroups - 1), lane);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const typename Keys<WP, PAGE>::Places to = keys.places(j1 + st * kWaves * kStep);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        ok[st][u] = to.ok[u];
#pragma unroll
        for (int i = 0; i < RT; ++i) x[st][i][u] = at[i][to.at[u]];
      }
    }
  }
  const int end = static_cast<int>(min<int64_t>(min<int64_t>(s.len, p.cap), from + kPart));
  if constexpr (PASS != kDen) {
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int j = j1 + st * kWaves * kStep + lane;
      old[st] = p.accumulate && j < end ? mass[j] : 0.f;
    }
  }
  v8i q[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) q[i] = query_bits(i < p.tgroups ? query_word<WP>(p, s, kvh, i, 0, lane) : 0u);
  const int open = s.open;
  float *den = p.den + (static_cast<int64_t>(blockIdx.y) * p.parts + (PASS == kDen ? blockIdx.x : 0)) * p.tgroups * 16;
  if constexpr (PASS == kMass) {
    if (tid < p.tgroups * 16) {
      const float d = parts_sum(p, s, den + tid);
      sm.inv[tid / 16][tid % 16] = d > 0.f && has_row<WP>(p, s, tid / 16, 0, tid % 16) ? 1.f / d : 0.f;
    }
  }
  __syncthreads();

  if constexpr (PASS != kMass) {
    float l[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) l[i] = 0.f;
    const int lim = open + tile_row<WP>(p, 0, lane & 15);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int j0 = j1 + st * kWaves * kStep;
      auto add = [&](auto mask) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          if (i >= p.tgroups) continue;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            l[i] += row_weights<decltype(mask)::value>(tab0, q[i], key_bits(ok[st][u] ? x[st][i][u] : 0u), j0 + 16 * u,
                                                       lane, lim);
        }
      };
      if (j0 + kStep - 1 <= open) add(std::false_type{});
      else if (j0 < s.len) add(std::true_type{});
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      l[i] += __shfl_xor(l[i], 16);
      l[i] += __shfl_xor(l[i], 32);
      if (lane < 16) sm.sum[wave][i][lane] = l[i];
    }
    __syncthreads();
    if (tid < p.tgroups * 16) {
      const int i = tid / 16, y = tid % 16;
      float d = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) d += sm.sum[w][i][y];
      if constexpr (PASS == kDen) den[tid] = d;
      else sm.inv[i][y] = d > 0.f && has_row<WP>(p, s, i, 0, y) ? 1.f / d : 0.f;
    }
    if constexpr (PASS == kBoth) __syncthreads();
  }
  if constexpr (PASS != kDen) {
    v4f inv[RT];
    int lim[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) lim[e] = open + tile_row<WP>(p, 0, 4 * (lane >> 4) + e);
#pragma unroll
    for (int i = 0; i < RT; ++i) inv[i] = *reinterpret_cast<const v4f *>(&sm.inv[i][4 * (lane >> 4)]);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int j0 = j1 + st * kWaves * kStep;
      if (j0 >= end) break;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      auto add = [&](auto mask) {
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          if (i >= p.tgroups) continue;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            sum[u] = key_weights<decltype(mask)::value>(tab0, q[i], key_bits(ok[st][u] ? x[st][i][u] : 0u),
                                                        j0 + 16 * u + (lane & 15), inv[i], lim, sum[u]);
        }
      };
      if (j0 + kStep - 1 <= open) add(std::false_type{});
      else add(std::true_type{});
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        sum[u] += __shfl_xor(sum[u], 16);
        sum[u] += __shfl_xor(sum[u], 32);
      }
      // lane l: key l of the step
      const float y = lane < 32 ? (lane < 16 ? sum[0] : sum[1]) : (lane < 48 ? sum[2] : sum[3]);
      if (j0 + lane < end) mass[j0 + lane] = old[st] + y;
    }
  }
}

// Many rows: denominators of kRows row tiles of a timestep group over kPart keys.  A wave keeps
// its keys and goes through the row tiles in a loop.  With four of them both kernels take 41 us
// captured and replayed for windows of up to 32 rows of 8 sequences of 2,000..8,000 tokens (two 46,
// eight 43).
template <int WP>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(4))) void den_rows_kernel(Params p) {
  struct Smem {
    float tab[kTab + 3];
    float sum[kWaves][kRows][16];
  };
  __shared__ Smem sm;
  const uint32_t tab0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPK_LDS char *)(void *)sm.tab));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int chunks = (p.rtiles + kRows - 1) / kRows;
  const int part = blockIdx.x % p.parts, group = blockIdx.x / p.parts;
  const int tg = group / chunks, rt0 = (group - tg * chunks) * kRows;
  const int kvh = blockIdx.y % p.Hkv, n = blockIdx.y / p.Hkv;
  const Seq s = sequence<WP>(p, n);
  if (part >= s.parts || rt0 >= s.rtiles) return;
  if (tid <= p.D) sm.tab[tid] = p.tab[tid];
  const Keys<WP, false> keys(p, s, n, kvh, lane);
  const int j1 = part * kPart + wave * kStep, tiles = min(kRows, s.rtiles - rt0);
  v8i k[kSteps][4];
  uint32_t qw = query_word<WP>(p, s, kvh, tg, rt0, lane);
  {
    uint32_t x[kSteps][4];
    bool ok[kSteps][4];
    const uint32_t *at = keys.words(tg, lane);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const typename Keys<WP, false>::Places to = keys.places(j1 + st * kWaves * kStep);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        ok[st][u] = to.ok[u];
        x[st][u] = at[to.at[u]];
      }
    }
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int u = 0; u < 4; ++u) k[st][u] = key_bits(ok[st][u] ? x[st][u] : 0u);
  }
  __syncthreads();
  const int open = s.open;
#pragma unroll 1
  for (int i = 0; i < tiles; ++i) {
    const v8i q = query_bits(qw);
    qw = query_word<WP>(p, s, kvh, tg, rt0 + min(i + 1, tiles - 1), lane);  // the next tile's
    float l = 0.f;
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int j0 = j1 + st * kWaves * kStep;
      if (j0 + kStep - 1 <= open) {
#pragma unroll
        for (int u = 0; u < 4; ++u) l += row_weights<false>(tab0, q, k[st][u], j0 + 16 * u, lane, 0);
      } else if (j0 < s.len) {
        const int lim = open + tile_row<WP>(p, rt0 + i, lane & 15);
#pragma unroll
        for (int u = 0; u < 4; ++u) l += row_weights<true>(tab0, q, k[st][u], j0 + 16 * u, lane, lim);
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (lane < 16) sm.sum[wave][i][lane] = l;
  }
  __syncthreads();
  if (tid < tiles * 16) {
    float d = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) d += sm.sum[w][tid / 16][tid % 16];
    p.den[(((static_cast<int64_t>(blockIdx.y) * p.parts + part) * p.tgroups + tg) * p.rtiles + rt0) * 16 + tid] = d;
  }
}

// Many rows: the weights of kMassKeys keys; kShare waves go through the row tiles of 64, four
// by four (so a sequence of few rows has the sums of few_rows_kernel, a wave's).
template <int WP>
__global__ __launch_bounds__(kMassKeys * kShare) __attribute__((amdgpu_waves_per_eu(4))) void mass_rows_kernel(Params p) {
  constexpr int kThreads = kMassKeys * kShare;
  struct Smem {
    float tab[kTab + 3];
    union {
      float inv[kChunk][16];
      float sum[kShare][kMassKeys];
    };
  };
  __shared__ Smem sm;
  const uint32_t tab0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPK_LDS char *)(void *)sm.tab));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), share = wave % kShare;
  const int kvh = blockIdx.y % p.Hkv, n = blockIdx.y / p.Hkv;
  const Seq s = sequence<WP>(p, n);
  float *mass = p.mass + n * p.ms0 + kvh * p.ms1;
  const int64_t from = static_cast<int64_t>(blockIdx.x) * kMassKeys, stop = min(p.cap, from + kMassKeys);
  if (!p.accumulate)
    for (int64_t j = max<int64_t>(from, s.rtiles ? s.len : 0) + tid; j < stop; j += kThreads) mass[j] = 0.f;
  if (from >= s.len || s.rtiles == 0) return;
  if (tid <= p.D) sm.tab[tid] = p.tab[tid];
  const Keys<WP, false> keys(p, s, n, kvh, lane);
  const int j0 = static_cast<int>(from) + wave / kShare * kStep, open = s.open;
  const int end = min(s.len, static_cast<int>(stop)), tiles = s.rtiles * p.tgroups;
  const typename Keys<WP, false>::Places places = keys.places(j0);
  const float *den = p.den + static_cast<int64_t>(blockIdx.y) * p.parts * p.tgroups * p.rtiles * 16;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  v8i k[4];
  // the wave's tiles: tile x is row tile x % rtiles of timestep group x / rtiles
  int tg = 0, rt = 4 * share, have = -1;
  auto settle = [&] {
    while (rt >= s.rtiles) {
      rt -= s.rtiles;
      ++tg;
    }
  };
  settle();
  uint32_t qw = tg < p.tgroups ? query_word<WP>(p, s, kvh, tg, rt, lane) : 0u;
  for (int c0 = 0; c0 < tiles; c0 += kChunk) {
    if (c0) __syncthreads();
    for (int v = tid; v < min(kChunk, tiles - c0) * 16; v += kThreads) {
      const int x = c0 + v / 16, xg = x / s.rtiles, xr = x - xg * s.rtiles, y = v % 16;
      const float d = parts_sum(p, s, den + static_cast<int64_t>(xg * p.rtiles + xr) * 16 + y);
      sm.inv[v / 16][y] = d > 0.f && has_row<WP>(p, s, xg, xr, y) ? 1.f / d : 0.f;
    }
    __syncthreads();
    for (int x = c0 + 4 * share, step; x < min(c0 + kChunk, tiles); x += step) {
      if (tg != have) {
        const uint32_t *at = keys.words(tg, lane);
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = at[places.at[u]];
#pragma unroll
        for (int u = 0; u < 4; ++u) k[u] = key_bits(places.ok[u] ? w[u] : 0u);
        have = tg;
      }
      const v8i q = query_bits(qw);
      const int row0 = rt;
      step = x % 4 == 3 ? 4 * kShare - 3 : 1;
      rt += step;
      settle();
      qw = tg < p.tgroups ? query_word<WP>(p, s, kvh, tg, rt, lane) : 0u;  // the next tile's
      const v4f inv = *reinterpret_cast<const v4f *>(&sm.inv[x - c0][4 * (lane >> 4)]);
      int lim[4];
      if (j0 + kStep - 1 <= open) {
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[u] = key_weights<false>(tab0, q, k[u], 0, inv, lim, sum[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) lim[e] = open + tile_row<WP>(p, row0, 4 * (lane >> 4) + e);
#pragma unroll
        for (int u = 0; u < 4; ++u)
          sum[u] = key_weights<true>(tab0, q, k[u], j0 + 16 * u + (lane & 15), inv, lim, sum[u]);
      }
    }
  }
  __syncthreads();  // (the denominators' place takes the sums)
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    sum[u] += __shfl_xor(sum[u], 16);
    sum[u] += __shfl_xor(sum[u], 32);
    if (lane < 16) sm.sum[share][j0 - static_cast<int>(from) + 16 * u + lane] = sum[u];
  }
  __syncthreads();
  if (tid < kMassKeys && from + tid < end) {
    const float x = (sm.sum[0][tid] + sm.sum[1][tid]) + (sm.sum[2][tid] + sm.sum[3][tid]);
    mass[from + tid] = p.accumulate ? mass[from + tid] + x : x;
  }
}

// exp((s - D) * scale), s = 0..D.
inline void build_weights(float scale, int D, float *tab) {
  static thread_local float last_scale = -1.f, last[kTab];
  static thread_local int last_d = 0;
  if (scale != last_scale || D != last_d) {
    for (int i = 0; i <= D; ++i) last[i] = static_cast<float>(std::exp((i - D) * static_cast<double>(scale)));
    last_scale = scale;
    last_d = D;
  }
  std::memcpy(tab, last, sizeof(float) * (D + 1));
}

// Words of a head as the products have them, timestep groups, row tiles of one, parts.
struct Plan {
  int wp, tgroups, rtiles, parts;
  size_t bytes;
};
inline Plan plan(int T, int N, int Hq, int Hkv, int D, int max_rows, int block_size, int max_blocks) {
  Plan r;
  const int W = (D + 31) / 32;
  r.wp = W == 3 ? 4 : W;
  const int64_t rows = static_cast<int64_t>(max_rows) * (Hq / Hkv);
  r.tgroups = (T + 4 / r.wp - 1) / (4 / r.wp);
  r.rtiles = static_cast<int>((rows + 4 * r.wp - 1) / (4 * r.wp));
  r.parts = static_cast<int>((static_cast<int64_t>(max_blocks) * block_size + kPart - 1) / kPart);
  r.bytes = static_cast<size_t>(N) * Hkv * r.parts * r.tgroups * r.rtiles * 16 * sizeof(float);
  return r;
}

// With one part a launch does both passes: 11.0 us where two take 13.0 (a sequence of 700 tokens,
// captured and replayed).
template <int WP, int RT, bool PAGE>
static int launch_few(const Params &p, int64_t wide, hipStream_t s) {
  const dim3 grid((wide + kPart - 1) / kPart, p.N * p.Hkv);
  if (p.parts <= 1) {
    few_rows_kernel<WP, RT, PAGE, kBoth><<<grid, kWaves * 64, 0, s>>>(p);
  } else {
    few_rows_kernel<WP, RT, PAGE, kDen><<<dim3(p.parts, p.N * p.Hkv), kWaves * 64, 0, s>>>(p);
    few_rows_kernel<WP, RT, PAGE, kMass><<<grid, kWaves * 64, 0, s>>>(p);
  }
  return check_launch("key_mass");
}

// Few rows: one row tile in each of four timestep groups at most (a decode step's).  The
// kernels for many rows would take 133 us where these take 41 (64 sequences of 4,096..16,384
// tokens, 14 query and 2 kv heads of 64 channels, 4 timesteps, captured and replayed).  Two rows
// of such a step, or more than 8 heads a kv head of 64 channels, have two row tiles and go there.
template <int WP>
static int launch(const Params &p, hipStream_t s) {
  // (without accumulation entries behind the table become 0)
  const int64_t tokens = static_cast<int64_t>(p.max_blocks) << p.bs_log2;
  const int64_t wide = p.accumulate && tokens < p.cap ? tokens : p.cap;
  if (p.rtiles == 1 && p.tgroups <= 4) {
    const bool page = p.bs_log2 >= 4;
    if (p.tgroups <= 2) return page ? launch_few<WP, 2, true>(p, wide, s) : launch_few<WP, 2, false>(p, wide, s);
    return page ? launch_few<WP, 4, true>(p, wide, s) : launch_few<WP, 4, false>(p, wide, s);
  }
  const int chunks = (p.rtiles + kRows - 1) / kRows;
  if (p.parts > 0 && p.rows > 0)
    den_rows_kernel<WP><<<dim3(p.parts * p.tgroups * chunks, p.N * p.Hkv), kWaves * 64, 0, s>>>(p);
  mass_rows_kernel<WP><<<dim3((wide + kMassKeys - 1) / kMassKeys, p.N * p.Hkv), kMassKeys * kShare, 0, s>>>(p);
  return check_launch("key_mass");
}

}  // namespace mass
}  // namespace spk

using namespace spk;

extern "C" size_t spk_key_mass_workspace_bytes(int T, int N, int Hq, int Hkv, int head_dim, int max_rows,
                                               int block_size, int max_blocks) {
  if (T <= 0 || N <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0 || head_dim > 128 || max_rows <= 0 ||
      block_size <= 0 || max_blocks < 0)
    return 0;
  return mass::plan(T, N, Hq, Hkv, head_dim, max_rows, block_size, max_blocks).bytes;
}

extern "C" int spk_key_mass(const int32_t *q, const int64_t q_strides[3], const int32_t *k_cache,
                            const int64_t cache_strides[3], int64_t num_slots, const int32_t *block_tables,
                            int64_t bt_stride0, int64_t bt_stride1, const int32_t *seq_lens,
                            const int32_t *row_starts, float *mass, const int64_t mass_strides[2], int64_t cap,
                            int accumulate, int64_t rows, int N, int max_rows, int T, int Hq, int Hkv,
                            int head_dim, int block_size, int max_blocks, float scale, void *workspace,
                            size_t workspace_bytes, void *stream) {
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0 || N < 0 || rows < 0 || max_rows <= 0 ||
      max_blocks < 0 || num_slots < 0 || cap < 0)
    return fail(SPK_EINVAL, "key_mass: bad sizes T=%d Hq=%d Hkv=%d D=%d N=%d rows=%lld max_rows=%d", T, Hq, Hkv,
                head_dim, N, (long long)rows, max_rows);
  if (head_dim > 128) return fail(SPK_EUNSUPPORTED, "key_mass: head_dim=%d (at most 128)", head_dim);
  if (!is_pow2(block_size)) return fail(SPK_EINVAL, "key_mass: block_size=%d is not a power of two", block_size);
  if (static_cast<int64_t>(max_blocks) * block_size > (1 << 30))
    return fail(SPK_EUNSUPPORTED, "key_mass: block tables of %d x %d tokens (at most 2^30)", max_blocks, block_size);
  if (!(scale > 0.f) || scale * head_dim > 12.f)
    return fail(SPK_EINVAL, "key_mass: scale=%g outside (0, 12/head_dim]", (double)scale);
  if (N == 0 || cap == 0 || (accumulate && max_blocks == 0)) return SPK_OK;
  if (static_cast<int64_t>(N) * Hkv > 65535) return fail(SPK_EUNSUPPORTED, "key_mass: %d sequences of %d heads", N, Hkv);
  if ((rows > 0 && !q) || !seq_lens || !mass || (max_blocks > 0 && !block_tables) || (num_slots > 0 && !k_cache))
    return fail(SPK_EINVAL, "key_mass: null pointer");
  if ((N > 1 && !mass_strides[0]) || (Hkv > 1 && !mass_strides[1]))
    return fail(SPK_EINVAL, "key_mass: rows of mass lie on one another");
  const mass::Plan plan = mass::plan(T, N, Hq, Hkv, head_dim, max_rows, block_size, max_blocks);
  if (static_cast<int64_t>(max_rows) * (Hq / Hkv) > (1 << 24) ||
      static_cast<int64_t>(plan.rtiles) * plan.tgroups * plan.parts > (1 << 30) ||
      // (a launch has fewer than 2^32 threads along its first axis)
      static_cast<int64_t>((plan.rtiles + mass::kRows - 1) / mass::kRows) * plan.tgroups * plan.parts > (1 << 22) ||
      cap > (1 << 29))
    return fail(SPK_EUNSUPPORTED, "key_mass: %d rows of %d heads over %d x %d tokens", max_rows, Hq / Hkv, max_blocks,
                block_size);
  if (!tiles::divides_to(static_cast<int64_t>(plan.rtiles) * 4 * plan.wp, Hq / Hkv))
    return fail(SPK_EUNSUPPORTED, "key_mass: %d heads a kv head with %d rows", Hq / Hkv, max_rows);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
    return fail(SPK_EINVAL, "key_mass: workspace of %zu bytes, %zu needed", workspace_bytes, plan.bytes);
  mass::Params p{};
  p.q = reinterpret_cast<const uint32_t *>(q);
  p.qs0 = q_strides[0]; p.qs1 = q_strides[1]; p.qs2 = q_strides[2];
  p.k = reinterpret_cast<const uint32_t *>(k_cache);
  p.ks0 = cache_strides[0]; p.ks1 = cache_strides[1]; p.ks2 = cache_strides[2];
  p.num_slots = num_slots;
  if (num_slots < block_size && q) {  // no block of a cache: every key is dropped, the loads read q's words
    p.k = p.q;
    p.ks0 = p.ks1 = p.ks2 = 0;
  }
  p.bt = block_tables; p.bts0 = bt_stride0; p.bts1 = bt_stride1;
  p.lens = seq_lens; p.starts = row_starts;
  p.mass = mass; p.ms0 = mass_strides[0]; p.ms1 = mass_strides[1]; p.cap = cap;
  p.accumulate = accumulate; p.rows = rows; p.N = N; p.max_rows = max_rows;
  p.T = T; p.Hkv = Hkv; p.nrep = Hq / Hkv; p.D = head_dim; p.W = (head_dim + 31) / 32;
  p.rep_mul = tiles::inverse_of(p.nrep);
  p.bs_log2 = ilog2(block_size); p.max_blocks = max_blocks;
  p.tgroups = plan.tgroups; p.rtiles = plan.rtiles; p.parts = plan.parts;
  p.den = static_cast<float *>(workspace);
  mass::build_weights(scale, head_dim, p.tab);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (plan.wp) {
    case 1: return mass::launch<1>(p, s);
    case 2: return mass::launch<2>(p, s);
    default: return mass::launch<4>(p, s);
  }
}
