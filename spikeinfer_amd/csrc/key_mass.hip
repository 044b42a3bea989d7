// Attention weight that the cached tokens of a sequence get from its last rows.
//
// Row i of a sequence's m rows is the token at position len - m + i and sees the
// positions up to its own:
//   mass[n, g, j] (+)= sum over t, query heads h of kv head g, rows i of
//                      exp(popc(q & k_j) * scale) / sum_j' exp(popc(q & k_j') * scale).
//
// MI355X design: scores of 16 rows and 16 keys are one fp4 product over 128 channels
// (v_mfma_scale_f32_16x16x128_f8f6f4, bits as 0.5 in place, block scales that leave the
// score's table offset in the accumulator's bits, as spike_tiles.hpp has it), a weight is a
// look-up in LDS.  128 channels are 4 / WP timesteps of a head (WP: words of a head, a power
// of two): a product's 16 rows are 4 * WP of each of these timesteps, whose words stand in
// their own quarter or half of the channels beside zeros, so that decoding (7 rows of 4
// timesteps at 64 channels) fills 14 of 16 rows and every lane loads one word of a key.
//   den_kernel   sums the weights of a part of kPart keys for RT or fewer such row tiles
//                (keys as the product's rows: a lane adds its own row's weights);
//   mass_kernel  adds the parts' sums in their order, then the weights over the
//                denominators (keys as its columns: a lane adds its own key's).  With RT row
//                tiles or fewer (a decode step) a wave holds them and goes through its keys;
//                with more the four waves of a workgroup have the same keys and share the row
//                tiles, RT at a time, and their sums are added in wave order.
// The order of all sums is the sequence's own, whatever the batch.
#include "spike_tiles.hpp"

namespace spk {
namespace mass {

using namespace tiles;

constexpr int kWaves = 4;
constexpr int kStep = 64;      // keys a wave takes at once: four products' columns
constexpr int kPart = 1024;    // keys a workgroup

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
  uint32_t rep_mul;            // floor(r / nrep) = r * rep_mul >> 32 for every row
  int N, max_rows, T, Hkv, nrep, W, D, bs_log2, max_blocks;
  int tgroups;                 // timestep groups
  int tiles;                   // most row tiles of a sequence
  int parts;                   // most parts of a sequence
  float *den;                  // [N, Hkv, parts, tiles, 16]
  float tab[kTab];             // exp((s - D) * scale)
};

struct Seq {
  int64_t first;
  int m, len, parts;
  int rtiles, tiles;  // row tiles of a timestep group, of all
};

template <int WP>
__device__ __forceinline__ Seq sequence(const Params &p, int n) {
  Seq s;
  const int64_t a = p.starts ? p.starts[n] : n, e = p.starts ? p.starts[n + 1] : n + 1;
  s.first = min(max<int64_t>(a, 0), p.rows);
  s.m = static_cast<int>(min(min(max(e, s.first), s.first + p.max_rows), p.rows) - s.first);
  s.len = min(max(p.lens[n], 0), p.max_blocks << p.bs_log2);
  s.parts = (s.len + kPart - 1) / kPart;
  s.rtiles = (s.m * p.nrep + 4 * WP - 1) / (4 * WP);
  s.tiles = s.rtiles * p.tgroups;
  return s;
}

__device__ __forceinline__ int row_of(const Params &p, int r) {  // r / nrep
  return p.nrep == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), p.rep_mul));
}

// Row tiles of a workgroup: tile x is rows 4 * WP * (x % rtiles) .. of timestep group x / rtiles.
// A product's row y: timestep y / (4 * WP) of the group, row y % (4 * WP) of the tile.
template <int WP, int RT>
struct Rows {
  v8i q[RT];
  int tg[RT];   // timestep group (uniform; -1: no tile)
  int lim[RT];  // last key that row l % 16 of the tile sees (-1: none)

  __device__ __forceinline__ void load(const Params &p, const Seq &s, int kvh, int tile0, int lane) {
    const int y = lane & 15, b = lane >> 4;  // row, 32-channel block of the product
    const int dt = y / (4 * WP);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int x = tile0 + i;
      tg[i] = x < s.tiles ? x / s.rtiles : -1;
      const int r = (x - tg[i] * s.rtiles) * 4 * WP + y % (4 * WP);
      const int row = row_of(p, r), t = tg[i] * (4 / WP) + dt;
      const bool in = tg[i] >= 0 && row < s.m && t < p.T;
      lim[i] = in ? s.len - s.m + row : -1;
      const int w = b - dt * WP;  // this lane's word of the row's head
      q[i] = fp4_bits(in && w >= 0 && w < WP && w < p.W
                          ? p.q[t * p.qs0 + (s.first + row) * p.qs1 + (kvh * p.nrep + r - row * p.nrep) * p.qs2 + w]
                          : 0u);
    }
  }
};

// A lane's words of a step's four key tiles for one timestep group (lane l: key l % 16 of a
// tile, block l / 16 of the product's channels), as operands.
template <int WP>
struct Keys {
  const Params &p;
  const int32_t *table;
  const uint32_t *base;
  uint32_t nblocks;
  int last_block, len, y, dt, w;
  __device__ __forceinline__ Keys(const Params &p, const Seq &s, int n, int kvh, int lane) : p(p), len(s.len) {
    table = p.bt + n * p.bts0;
    base = p.k + kvh * p.ks1;
    nblocks = static_cast<uint32_t>(min<int64_t>(p.num_slots >> p.bs_log2, 0xffffffffll));
    last_block = max(s.len - 1, 0) >> p.bs_log2;
    y = lane & 15;
    dt = (lane >> 4) / WP;
    w = (lane >> 4) % WP;
  }
  // Slots of the lane's four keys, -1 where there is none.
  __device__ __forceinline__ void slots(int j0, int64_t (&at)[4]) const {
    uint32_t phys[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      phys[u] = static_cast<uint32_t>(table[min((j0 + 16 * u + y) >> p.bs_log2, last_block) * p.bts1]);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + 16 * u + y;
      at[u] = j < len && phys[u] < nblocks
                  ? ((static_cast<int64_t>(phys[u]) << p.bs_log2) | (j & ((1 << p.bs_log2) - 1))) * p.ks2
                  : -1;
    }
  }
  // (unconditional loads, dropped where there is no key or word: they are all on their way
  // before the first is waited for)
  __device__ __forceinline__ void load(int tg, const int64_t (&at)[4], uint32_t (&x)[4]) const {
    const int t = tg * (4 / WP) + dt;
    const bool in = t < p.T && w < p.W;
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = base[in && at[u] >= 0 ? t * p.ks0 + at[u] + w : 0];
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = in && at[u] >= 0 ? x[u] : 0u;
  }
};

__device__ __forceinline__ v4f score(const v8i &a, const v8i &b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{}, 4, 4, 0, 55, 0, 54);
}

__device__ __forceinline__ float weight(uint32_t tab0, float score) {
  return *reinterpret_cast<const SPK_LDS float *>(static_cast<uintptr_t>(tab0 + __float_as_uint(score)));
}

// Key words of all of a wave's steps for each row tile.
template <int WP, int RT, int STEPS>
__device__ __forceinline__ void request(const Keys<WP> &keys, const int (&tg)[RT], int j1, uint32_t (&x)[STEPS][RT][4]) {
  int64_t at[STEPS][4];
#pragma unroll
  for (int st = 0; st < STEPS; ++st) keys.slots(j1 + st * kWaves * kStep, at[st]);
#pragma unroll
  for (int st = 0; st < STEPS; ++st)
#pragma unroll
    for (int i = 0; i < RT; ++i) keys.load(max(tg[i], 0), at[st], x[st][i]);
}

template <int WP, int RT>
__global__ __launch_bounds__(kWaves * 64) void den_kernel(Params p) {
  struct Smem {
    float tab[kTab + 3];  // first: a score's accumulator is its entry's LDS address
    float sum[kWaves][RT][16];
  };
  __shared__ Smem sm;
  const uint32_t tab0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPK_LDS char *)(void *)sm.tab));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = blockIdx.x % p.parts, chunk = blockIdx.x / p.parts;
  const int kvh = blockIdx.y % p.Hkv, n = blockIdx.y / p.Hkv;
  const Seq s = sequence<WP>(p, n);
  if (part >= s.parts || chunk * RT >= s.tiles) return;
  if (tid <= p.D) sm.tab[tid] = p.tab[tid];
  Rows<WP, RT> rows;
  rows.load(p, s, kvh, chunk * RT, lane);
  const Keys<WP> keys(p, s, n, kvh, lane);
  float l[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) l[i] = 0.f;
  __syncthreads();
  const int end = min(s.len, (part + 1) * kPart), open = s.len - s.m;  // keys up to `open` are seen by all rows
  auto add = [&](int i, int u, int j0, const v8i &k) {
    const v4f a = score(k, rows.q[i]);  // lane: row l % 16, keys 4 * (l / 16) + 0..3
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = weight(tab0, a[e]);
    if (j0 + 16 * u + 15 > open) {
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = j0 + 16 * u + 4 * (lane >> 4) + e <= rows.lim[i] ? w[e] : 0.f;
    }
    l[i] += (w[0] + w[1]) + (w[2] + w[3]);
  };
  const int j1 = part * kPart + wave * kStep;
  if constexpr (RT == 2) {  // few products a key: the words of all steps are requested first
    constexpr int kSteps = kPart / (kWaves * kStep);
    uint32_t x[kSteps][RT][4];
    request<WP, RT, kSteps>(keys, rows.tg, j1, x);
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      const int j0 = j1 + st * kWaves * kStep;
      if (j0 >= end) break;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (rows.tg[i] < 0) continue;
#pragma unroll
        for (int u = 0; u < 4; ++u) add(i, u, j0, fp4_bits(x[st][i][u]));
      }
    }
  } else {
    for (int j0 = j1; j0 < end; j0 += kWaves * kStep) {
      int64_t at[4];
      keys.slots(j0, at);
      v8i k[4];
      int have = -1;
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (rows.tg[i] < 0) continue;
        if (rows.tg[i] != have) {
          uint32_t x[4];
          keys.load(rows.tg[i], at, x);
#pragma unroll
          for (int u = 0; u < 4; ++u) k[u] = fp4_bits(x[u]);
          have = rows.tg[i];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) add(i, u, j0, k[u]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    l[i] += __shfl_xor(l[i], 16);
    l[i] += __shfl_xor(l[i], 32);
    if (lane < 16) sm.sum[wave][i][lane] = l[i];
  }
  __syncthreads();
  float *to = p.den + ((static_cast<int64_t>(blockIdx.y) * p.parts + part) * p.tiles + chunk * RT) * 16;
  for (int x = tid; x < RT * 16; x += kWaves * 64)
    if (chunk * RT + x / 16 < s.tiles)
      to[x] = (sm.sum[0][x / 16][x % 16] + sm.sum[1][x / 16][x % 16]) + (sm.sum[2][x / 16][x % 16] + sm.sum[3][x / 16][x % 16]);
}

// SHARED: the waves have the same kStep * STEPS keys and share the row tiles; else each has
// STEPS steps of its own.
template <int WP, int RT, int STEPS, bool SHARED>
__global__ __launch_bounds__(kWaves * 64) void mass_kernel(Params p) {
  constexpr int kKeys = STEPS * kStep * (SHARED ? 1 : kWaves);  // of a workgroup
  struct Smem {
    float tab[kTab + 3];
    float inv[kWaves][RT][16];
    int lim[kWaves][RT][16];
    float sum[SHARED ? kWaves : 1][kKeys];
  };
  __shared__ Smem sm;
  const uint32_t tab0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPK_LDS char *)(void *)sm.tab));
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.y % p.Hkv, n = blockIdx.y / p.Hkv;
  const Seq s = sequence<WP>(p, n);
  float *mass = p.mass + n * p.ms0 + kvh * p.ms1;
  const int64_t from = static_cast<int64_t>(blockIdx.x) * kKeys, stop = min(p.cap, from + kKeys);
  if (!p.accumulate)
    for (int64_t j = max<int64_t>(from, s.len) + tid; j < stop; j += kWaves * 64) mass[j] = 0.f;
  if (from >= s.len || from >= p.cap) return;
  if (tid <= p.D) sm.tab[tid] = p.tab[tid];
  __syncthreads();
  const Keys<WP> keys(p, s, n, kvh, lane);
  const int end = min(s.len, static_cast<int>(stop)), open = s.len - s.m;  // keys up to `open` are seen by all rows
  const float *den = p.den + static_cast<int64_t>(blockIdx.y) * p.parts * p.tiles * 16;

  Rows<WP, RT> rows;
  float inv[RT][4];  // of the products' rows 4 * (l / 16) + 0..3; no row: 0
  auto take = [&](int tile0) {  // row tiles tile0 .. and their denominators, a wave by itself
    rows.load(p, s, kvh, tile0, lane);
#pragma unroll
    for (int i = 0; i < RT; i += 4) {  // lane: row l % 16 of tile i + l / 16
      const int x = i + (lane >> 4);
      float d = 0.f;
      if (x < RT && tile0 + x < s.tiles) {
        const float *at = den + (tile0 + x) * 16 + (lane & 15);
        for (int pt = 0; pt < s.parts; pt += 8) {  // eight parts' sums on their way at once
          float y[8];
#pragma unroll
          for (int v = 0; v < 8; ++v) y[v] = at[static_cast<int64_t>(min(pt + v, s.parts - 1)) * p.tiles * 16];
#pragma unroll
          for (int v = 0; v < 8; ++v) d += pt + v < s.parts ? y[v] : 0.f;
        }
      }
      if (x < RT) sm.inv[wave][x][lane & 15] = d > 0.f ? 1.f / d : 0.f;
    }
    if (lane < 16) {
#pragma unroll
      for (int i = 0; i < RT; ++i) sm.lim[wave][i][lane] = rows.lim[i];
    }
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int y = 4 * (lane >> 4) + e;
        inv[i][e] = sm.lim[wave][i][y] >= 0 ? sm.inv[wave][i][y] : 0.f;
      }
  };
  auto give = [&](int i, int u, int j0, const v8i &k, float &sum) {
    const v4f a = score(rows.q[i], k);  // lane: key l % 16, rows 4 * (l / 16) + 0..3
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = weight(tab0, a[e]);
    if (j0 + 16 * u + 15 > open) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = j0 + 16 * u + (lane & 15) <= sm.lim[wave][i][4 * (lane >> 4) + e] ? w[e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = __builtin_fmaf(w[e], inv[i][e], sum);
  };
  auto add = [&](int j0, float (&sum)[4]) {  // what the rows give the 64 keys at j0
    int64_t at[4];
    keys.slots(j0, at);
    v8i k[4];
    int have = -1;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (rows.tg[i] < 0) continue;
      if (rows.tg[i] != have) {
        uint32_t x[4];
        keys.load(rows.tg[i], at, x);
#pragma unroll
        for (int u = 0; u < 4; ++u) k[u] = fp4_bits(x[u]);
        have = rows.tg[i];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) give(i, u, j0, k[u], sum[u]);
    }
  };
  auto finish = [&](int j, float x) {
    if (j < end) mass[j] = p.accumulate ? mass[j] + x : x;
  };
  if constexpr (SHARED) {
    float sum[STEPS][4] = {};
    for (int tile0 = wave * RT; tile0 < s.tiles; tile0 += kWaves * RT) {
      take(tile0);
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
        if (from + st * kStep < end) add(static_cast<int>(from) + st * kStep, sum[st]);
      wave_lds_sync();  // (the limits are read before the next tiles' come)
    }
#pragma unroll
    for (int st = 0; st < STEPS; ++st)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float x = sum[st][u];
        x += __shfl_xor(x, 16);
        x += __shfl_xor(x, 32);
        if (lane < 16) sm.sum[wave][st * kStep + 16 * u + lane] = x;
      }
    __syncthreads();
    for (int x = tid; x < kKeys; x += kWaves * 64)
      finish(static_cast<int>(from) + x, (sm.sum[0][x] + sm.sum[1][x]) + (sm.sum[2][x] + sm.sum[3][x]));
  } else {
    // few products a key: the words of all steps are requested first
    const int j1 = static_cast<int>(from) + wave * kStep;
    int tg[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) tg[i] = i < s.tiles ? i / s.rtiles : 0;
    uint32_t words[STEPS][RT][4];
    request<WP, RT, STEPS>(keys, tg, j1, words);
    take(0);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int j0 = j1 + st * kWaves * kStep;
      if (j0 >= end) break;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (rows.tg[i] < 0) continue;
#pragma unroll
        for (int u = 0; u < 4; ++u) give(i, u, j0, fp4_bits(words[st][i][u]), sum[u]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        sum[u] += __shfl_xor(sum[u], 16);
        sum[u] += __shfl_xor(sum[u], 32);
      }
      // lane l: key l of the step
      const float x = lane < 32 ? (lane < 16 ? sum[0] : sum[1]) : (lane < 48 ? sum[2] : sum[3]);
      finish(j0 + lane, x);
    }
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

// Rows of a product's timestep, timestep groups, row tiles.
struct Plan {
  int wp, tgroups, tiles, parts;
  size_t bytes;
};
inline Plan plan(int T, int N, int Hq, int Hkv, int D, int max_rows, int block_size, int max_blocks) {
  Plan r;
  const int W = (D + 31) / 32;
  r.wp = W == 3 ? 4 : W;
  const int64_t rows = static_cast<int64_t>(max_rows) * (Hq / Hkv);
  r.tgroups = (T + 4 / r.wp - 1) / (4 / r.wp);
  r.tiles = static_cast<int>((rows + 4 * r.wp - 1) / (4 * r.wp)) * r.tgroups;
  r.parts = static_cast<int>((static_cast<int64_t>(max_blocks) * block_size + kPart - 1) / kPart);
  r.bytes = static_cast<size_t>(N) * Hkv * r.parts * r.tiles * 16 * sizeof(float);
  return r;
}

template <int WP, int RT, int STEPS, bool SHARED>
static int launch(const Params &p, hipStream_t s) {
  const int chunks = (p.tiles + RT - 1) / RT, keys = STEPS * kStep * (SHARED ? 1 : kWaves);
  // (without accumulation entries behind the table become 0)
  const int64_t tokens = static_cast<int64_t>(p.max_blocks) << p.bs_log2;
  const int64_t wide = p.accumulate && tokens < p.cap ? tokens : p.cap;
  if (p.parts > 0 && p.rows > 0) den_kernel<WP, RT><<<dim3(p.parts * chunks, p.N * p.Hkv), kWaves * 64, 0, s>>>(p);
  mass_kernel<WP, RT, STEPS, SHARED><<<dim3((wide + keys - 1) / keys, p.N * p.Hkv), kWaves * 64, 0, s>>>(p);
  return check_launch("key_mass");
}

// Row tiles a wave holds in registers: those of a decode step, or eight.
template <int WP>
static int launch_rows(const Params &p, hipStream_t s) {
  if (p.tiles <= 2) return launch<WP, 2, 4, false>(p, s);
  if (p.tiles <= 4) return launch<WP, 4, 2, false>(p, s);
  return launch<WP, 8, 2, true>(p, s);
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
  const mass::Plan plan = mass::plan(T, N, Hq, Hkv, head_dim, max_rows, block_size, max_blocks);
  if (static_cast<int64_t>(max_rows) * (Hq / Hkv) > (1 << 24) ||
      static_cast<int64_t>(plan.tiles) * plan.parts > (1 << 30) || cap > (1 << 30))
    return fail(SPK_EUNSUPPORTED, "key_mass: %d rows of %d heads over %d x %d tokens", max_rows, Hq / Hkv, max_blocks,
                block_size);
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
  // ceil(2^32 / nrep): its product with r is off by less than r * nrep, below 2^32
  p.rep_mul = static_cast<uint32_t>(((int64_t(1) << 32) + p.nrep - 1) / p.nrep);
  p.bs_log2 = ilog2(block_size); p.max_blocks = max_blocks;
  p.tgroups = plan.tgroups; p.tiles = plan.tiles; p.parts = plan.parts;
  p.den = static_cast<float *>(workspace);
  mass::build_weights(scale, head_dim, p.tab);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (plan.wp) {
    case 1: return mass::launch_rows<1>(p, s);
    case 2: return mass::launch_rows<2>(p, s);
    default: return mass::launch_rows<4>(p, s);
  }
}
