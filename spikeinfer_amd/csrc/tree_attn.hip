// Attention of drafted token trees over the paged packed cache (head_dim <= 128).
//
// Row r of a sequence (a drafted token) attends, per timestep and query head, to
// the sequence's cached context and to the drafted tokens that its mask names:
//   out = sum_j w_j bits(v_j) / sum_j w_j,  w_j = exp(popc(q & k_j) * scale).
//
// MI355X design, on the tiles of the prefill attention (spike_tiles.hpp):
//   * Rows: node r / n_rep, query head r % n_rep of one (t, kv head), in tiles of 32.
//     Keys: tiles of 32, the context's first; the tree's own start on a tile of their
//     own, so that a row's mask word is the tile's.
//   * Scores as there: one fp4 product per 64 channels leaves the score's table offset in
//     the accumulator's bits, and the weight is a look-up.
//   * Values: f16 products over two keys a register, one for the weights' high halves and one
//     for their low ones, whatever the output's type: the smallest weight, 2^15 / e^12, keeps
//     2^-21 of itself, larger ones up to 2^-23.  A v bit becomes an operand by one `and`, as
//     one of f16's exponent bits, 2^-14 or 2^-13 by the key's number % 2, and two tables of
//     weights hold what makes the products equal again.
//   * Eight waves a workgroup (four with more than 64 channels) share the key tiles' operands
//     through LDS: each prepares one of a step's tiles, two buffers of them so that one barrier
//     a step does.  Of a sequence of more than 16 rows a wave of the workgroup (128, 64) each
//     wave takes a row tile of 32 and all keys; of more than 8 two waves share a row tile, of
//     more than 4 (and with four waves of fewer) four, else all eight, each with its part of a
//     step's tiles; they are added in their order.
//   * The context is cut into parts of kPartTiles tiles (more beyond kMaxParts parts), the
//     tree's tiles belonging to the last: a workgroup each, whose sums a second launch adds in
//     their order.  So the sums depend on the sequence alone, its length and its rows, not on
//     the batch around it.
//   * Sums go to the workspace every kPartTiles tiles, also within a longer part: fp32
//     accumulators take 256 products at most (and the tree's), whatever the length.  Off from
//     float64, fp32 outputs: random words 4e-7 in the 2-norm from 2,000 to 1 << 20 tokens; keys of
//     equal weights with values of ones, the worst found, 2.4e-6 at 1 << 20 and 4e-6 at 1 << 22
//     (with one accumulator a part up to 5e-5 and 2e-4).
//
// Bound by issue: a tile of 32 rows and 32 keys of 64 channels is 9 matrix instructions with 64
// vector, 19 LDS and about 11 scalar ones, which hide behind one another only in part.  With 14
// query and 2 kv heads of 64 channels and 4 timesteps, 32 nodes on each of 16 contexts of
// 4,096..16,384 tokens, fp32, take 115..126 us, 600..655 TFLOP/s of 4 * T * Hq * nodes * keys * D
// operations (those on values done twice); matrix units are busy 44 % and vector units 57 % of
// the time.  61 nodes on 30,011 tokens, bf16, take 46 us: 569 TFLOP/s, in 240 workgroups of 64
// tiles, one a CU.  (The weights' high halves alone would take 33, and change bf16 outputs: up
// to 2^-10 of them where 2^-8 is half a step.)  At four waves a SIMD the kernel for 64 channels
// spills 68 registers, of which its unmasked loops reload 12 to 14 a step of eight tiles.
#include <type_traits>

#include "spike_tiles.hpp"

namespace spk {
namespace tree {

using namespace tiles;

// Waves a workgroup, and tiles between its barriers: eight, so that two workgroups are four
// waves a SIMD, or with the sums of more than 64 channels, four, so that two are two (71 us
// where eight take 78, captured and replayed: 8 sequences of 100..9,000 tokens, 25 nodes, 16
// query heads of 128).
constexpr int waves_of(int NC) { return NC > 2 ? 4 : 8; }
constexpr int kKeys = 32;          // keys per tile
// Tiles per part, up to kMaxParts of them.  Of 32, 64 and 128 (captured and replayed): 55, 54
// and 80 us for 61 nodes on 30,011 tokens, 53, 52 and 76 for 32 sequences of 500..5,000, 129, 136
// and 133 for 32 nodes on 16 of 4,096..16,384, 70, 71 and 95 for the case of 128 channels above.
constexpr int kPartTiles = 64;
constexpr int kMaxParts = 32;
constexpr int kMaxNodes = 1024;
constexpr int kTabStride = kTab + 3;

struct Params {
  const uint32_t *q;        // words of (t, row, query head)
  int64_t qs0, qs1, qs2;
  const uint32_t *kt, *vt;  // drafted tokens' words (t, row, kv head), the same strides
  int64_t ts0, ts1, ts2;
  const uint32_t *k, *v;    // caches (t, kv head, slot), the same strides
  int64_t ks0, ks1, ks2;
  int64_t num_slots;
  const int32_t *bt;
  int64_t bts0, bts1;
  const int32_t *lens, *starts;
  const uint32_t *masks;    // int64 words as pairs
  int mask_words;           // 32-bit words a row
  void *out;                // (t, row, query head, channel)
  int64_t os0, os1, os2;
  int out_dtype, out_vec;   // out_vec: rows take aligned 4-channel stores
  int64_t rows;
  uint32_t rep_mul;         // inverse_of(nrep)
  int units, Hkv, nrep, D, W, bs_log2, max_blocks, max_nodes;
  int rtiles;               // most row tiles of a sequence
  int groups;               // workgroups along them
  int parts;                // along its context
  int wide;                 // a plane of the caches passes 2^32 bytes
  float *ws;                // with parts > 1: sums of (sequence, unit, part, row tile)
  uint32_t tab[kTab];
};

// A sequence as the kernels take it: its rows and cached tokens, clamped to the buffers.
struct Seq {
  int64_t first;
  int nodes, ctx, ctiles, end;  // end: tiles of the context and of the tree
  int ptiles, parts;            // tiles of a part, parts
};

__device__ __forceinline__ Seq sequence(const Params &p, int n) {
  Seq s;
  s.first = min<int64_t>(max(p.starts[n], 0), p.rows);
  const int64_t end = min(max<int64_t>(p.starts[n + 1], s.first), p.rows);
  s.nodes = static_cast<int>(min<int64_t>(end - s.first, p.max_nodes));
  s.ctx = min(max(p.lens[n], 0), p.max_blocks << p.bs_log2);
  s.ctiles = (s.ctx + kKeys - 1) / kKeys;
  s.end = s.ctiles + (s.nodes + kKeys - 1) / kKeys;
  s.ptiles = kPartTiles;
  while (s.ptiles * kMaxParts < s.ctiles) s.ptiles <<= 1;
  s.parts = max(1, (s.ctiles + s.ptiles - 1) / s.ptiles);
  return s;
}

// The same for a table of `tokens` (host): most parts of a sequence.
inline int most_parts(int64_t tokens) {
  const int64_t tiles = (tokens + kKeys - 1) / kKeys;
  return tiles <= kPartTiles ? 1 : static_cast<int>(tiles < kPartTiles * kMaxParts ? (tiles + kPartTiles - 1) / kPartTiles : kMaxParts);
}

__device__ __forceinline__ int node_of(const Params &p, int r) {
  return p.nrep == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), p.rep_mul));
}

// Two tables of (hi, lo) pairs in LDS at offset 0: the weights, and half of them.
constexpr int kTables = 2;
__device__ __forceinline__ void fill_tables(const Params &p, uint32_t *tab, int tid) {
  if (tid > p.D) return;
  const uint32_t w = p.tab[tid];
  const v2h half = __builtin_bit_cast(v2h, w) * v2h{static_cast<_Float16>(0.5f), static_cast<_Float16>(0.5f)};
  tab[tid] = w;
  tab[kTabStride + tid] = __builtin_bit_cast(uint32_t, half);
}

// Query words of row `r` (score operands of its tile).
template <int NK>
__device__ __forceinline__ void load_query(const Params &p, const Seq &s, int t, int kvh, int r, int half,
                                           v8i (&qop)[NK]) {
  const int node = node_of(p, r), h = r - node * p.nrep;
  const uint32_t *qp = p.q + t * p.qs0 + (s.first + node) * p.qs1 + (kvh * p.nrep + h) * p.qs2;
#pragma unroll
  for (int k = 0; k < NK; ++k) {
    const int w = 2 * k + half;
    qop[k] = fp4_bits(w < p.W ? qp[w] : 0u);
  }
}

// A lane's key words of tile kt (lane l: key l % 32, words 2k + l / 32).  Loads are
// unconditional (indices clamped into range, the value dropped where a key is none:
// zero spikes), so that the wave waits for none of them before its use.
template <int NK>
struct Keys {
  const Params &p;
  const Seq &s;
  const int32_t *table;
  const uint32_t *kbase, *vbase, *ktree, *vtree;
  uint32_t nblocks, slot_bytes;
  int last, half, col;

  __device__ __forceinline__ Keys(const Params &p, const Seq &s, int n, int t, int kvh, int half, int col)
      : p(p), s(s), half(half), col(col) {
    table = p.bt + n * p.bts0;
    kbase = p.k + t * p.ks0 + kvh * p.ks1;
    vbase = p.v + t * p.ks0 + kvh * p.ks1;
    ktree = p.kt + t * p.ts0 + s.first * p.ts1 + kvh * p.ts2;
    vtree = p.vt + t * p.ts0 + s.first * p.ts1 + kvh * p.ts2;
    nblocks = static_cast<uint32_t>(min<int64_t>(p.num_slots >> p.bs_log2, 0xffffffffll));
    slot_bytes = static_cast<uint32_t>(p.ks2 * 4);
    last = max(s.ctx - 1, 0);
  }
  __device__ __forceinline__ uint32_t block_of(int kt) const {
    return static_cast<uint32_t>(table[(min(kt * kKeys + col, last) >> p.bs_log2) * p.bts1]);
  }
  __device__ __forceinline__ void words(const uint32_t *kp, const uint32_t *vp, uint32_t at, uint32_t (&kw)[NK],
                                        uint32_t (&vw)[NK]) const {
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const uint32_t b = at + 4 * min(2 * k + half, p.W - 1);  // (a uniform base and 32-bit bytes)
      kw[k] = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(kp) + b);
      vw[k] = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(vp) + b);
    }
  }
  __device__ __forceinline__ void load(int kt, uint32_t phys, uint32_t (&kw)[NK], uint32_t (&vw)[NK], bool &ok) const {
    if (kt < s.ctiles) {
      const int j = kt * kKeys + col;
      ok = j < s.ctx && phys < nblocks;
      const uint32_t low = static_cast<uint32_t>(j & ((1 << p.bs_log2) - 1));
      if (!p.wide) {
        words(kbase, vbase, ok ? ((phys << p.bs_log2) | low) * slot_bytes : 0u, kw, vw);
      } else {
        const int64_t at = ok ? ((static_cast<int64_t>(phys) << p.bs_log2) | low) * p.ks2 : 0;
        words(kbase + at, vbase + at, 0, kw, vw);
      }
    } else {
      const int j = (kt - s.ctiles) * kKeys + col;
      ok = j < s.nodes;
      const int64_t at = ok ? j * p.ts1 : 0;
      words(ktree + at, vtree + at, 0, kw, vw);
    }
  }
  // Loaded words as a tile's shared operands: keys as fp4, and per channel tile a lane's
  // channel l % 32 as bits of its keys: bit 8 * (e >> 2) + (e & 3) for its e-th key,
  // e < 16, which is key 8 * (e >> 2) + 4 * (l / 32) + (e & 3) of the tile.
  __device__ __forceinline__ void operands(const uint32_t (&kw)[NK], const uint32_t (&vw)[NK], bool ok, int lane,
                                           v8i (&kop)[NK], uint32_t (&vt)[2 * NK]) const {
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const bool in = ok && 2 * k + half < p.W;
      kop[k] = fp4_bits(in ? kw[k] : 0u);
      const uint32_t x = transpose32(in ? vw[k] : 0u, lane);
      const auto sw = __builtin_amdgcn_permlane32_swap(x, x, false, false);
      vt[2 * k] = sw[0] >> (4 * half);
      vt[2 * k + 1] = sw[1] >> (4 * half);
    }
  }
};

// Keys of tile kt that a row sees, as bits of the tile (`word`: the row's mask words).
__device__ __forceinline__ uint32_t seen(const Seq &s, int kt, const uint32_t *word, int half) {
  const int nt = kt - s.ctiles, left = nt < 0 ? s.ctx - kt * kKeys : s.nodes - nt * kKeys;
  uint32_t see = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0u;
  if (nt >= 0 && left > 0) see &= word[nt];
  return see >> (4 * half);
}

// A lane's v bits of a channel tile where `expand` masks them: a word for each operand and key
// number % 4 / 2, whose two keys' bits start at bit 10.
__device__ __forceinline__ v4u place_bits(uint32_t vt) { return v4u{vt << 10, vt << 8, vt << 2, vt}; }

// Products' value operands of a channel tile: register i of operand g pairs the lane's keys
// 4g + i and 4g + i + 8, sixteen bits apart.
__device__ __forceinline__ void expand(v4u vt, v8h (&vop)[2]) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    v4u x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = vt[g * 2 + i / 2] & (0x04000400u << i % 2);
    vop[g] = __builtin_bit_cast(v8h, x);
  }
}

template <int NK>
__device__ __forceinline__ v16f scores(const v8i (&kop)[NK], const v8i (&qop)[NK]) {
  v16f a = {};
#pragma unroll
  for (int k = 0; k < NK; ++k)
    a = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kop[k], qop[k], a, 4, 4, 0, 55, 0, 54);
  return a;
}

// A tile's weights: the lane's sixteen table entries.
__device__ __forceinline__ void lookup(uint32_t tab0, const v16f &a, uint32_t (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const uint32_t at = tab0 + 4 * kTabStride * (e & (kTables - 1)) + __float_as_uint(a[e]);
    w[e] = *reinterpret_cast<const SPK_LDS uint32_t *>(static_cast<uintptr_t>(at));
  }
}

// A lane's denominator: sums of high halves by the key's number % 4 and of low halves by its
// number % 2.  Low halves among the high ones would be rounded to the large sums (1.6e-6 of the
// outputs, in the 2-norm, where these lose 4e-7: 2,000 tokens, 140 rows, 128 channels).
struct Sums {
  float high[4] = {0.f, 0.f, 0.f, 0.f}, low[2] = {0.f, 0.f};
  // in the numerators' units
  __device__ __forceinline__ float total() const {
    return ((high[0] + 2.f * high[1]) + (high[2] + 2.f * high[3]) + (low[0] + 2.f * low[1])) * 0x1p-14f;
  }
};

// Adds a tile's weighted values to acc and its weights to l, one by one in fp32: dot products
// of f16 pairs would be half as many instructions, but they take the matrix cores' time (8
// behind each product 78 cycles where 8 additions take 52).
template <int NC, bool MASKED>
__device__ __forceinline__ void products(const uint32_t (&x)[16], uint32_t see, const v8h (&vop)[NC][2],
                                         v16f (&acc)[NC], Sums &l) {
  float one = 1.f;
  asm("" : "+v"(one));  // (kept a register: fma_mix then takes the halves as they are)
  auto keep = [&](int e) {  // the e-th of the lane's sixteen
    if constexpr (MASKED)
      return x[e] & static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(see), 8 * (e >> 2) + (e & 3), 1));
    else return x[e];
  };
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    v4u y[2];  // the weights' halves, two keys a register
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w0 = keep(4 * g + i), w1 = keep(4 * g + i + 8);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t both = __builtin_amdgcn_perm(w1, w0, q ? 0x07060302u : 0x05040100u);
        y[q][i] = both;
        const v2h half = __builtin_bit_cast(v2h, both);  // (of a scalar: an element would give the first)
        float &sum = q ? l.low[i & 1] : l.high[i];
        sum = __builtin_fmaf(static_cast<float>(half[0]), one, sum);
        sum = __builtin_fmaf(static_cast<float>(half[1]), one, sum);
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int c = 0; c < NC; ++c)
        acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vop[c][g], __builtin_bit_cast(v8h, y[q]), acc[c], 0, 0, 0);
  }
}

// Rows of a tile from their sums: kVals of the lane's values of channel tile c (four
// channels 8 * (g0 + k) + 4 * half .. for each k), divided by the row's denominator.
template <int kVals>
__device__ __forceinline__ void store_row(const Params &p, const Seq &s, int t, int kvh, int r, int c, int g0, int half,
                                          const float (&val)[kVals], float den) {
  const float inv = den > 0.f ? 1.f / den : 0.f;  // (a row that sees nothing: zeros)
  const int node = node_of(p, r);
  const int64_t row = t * p.os0 + (s.first + node) * p.os1 + (kvh * p.nrep + r - node * p.nrep) * p.os2;
  if (p.out_vec) {  // D % 4 == 0: four channels lie in or out together
#pragma unroll
    for (int k = 0; k < kVals / 4; ++k) {
      const int ch = 32 * c + 8 * (g0 + k) + 4 * half;
      float o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = val[4 * k + e] * inv;
      if (ch >= p.D) continue;
      if (p.out_dtype == SPK_F32) {
        *reinterpret_cast<v4f *>(static_cast<float *>(p.out) + row + ch) = v4f{o[0], o[1], o[2], o[3]};
        continue;
      }
      uint32_t w2[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint16_t x0, x1;
        if (p.out_dtype == SPK_BF16) {
          x0 = f32_to_bf16_bits(o[2 * e]);
          x1 = f32_to_bf16_bits(o[2 * e + 1]);
        } else {
          x0 = __builtin_bit_cast(uint16_t, static_cast<_Float16>(o[2 * e]));
          x1 = __builtin_bit_cast(uint16_t, static_cast<_Float16>(o[2 * e + 1]));
        }
        w2[e] = x0 | (static_cast<uint32_t>(x1) << 16);
      }
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.out) + row + ch) = make_uint2(w2[0], w2[1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVals; ++j) {
      const int ch = 32 * c + 8 * (g0 + (j >> 2)) + 4 * half + (j & 3);
      if (ch < p.D) store_f32_as(p.out, row + ch, p.out_dtype, val[j] * inv);
    }
  }
}

// A row tile's sums in the workspace: [NC][4][64] vectors of four channels, [32] denominators.
constexpr int tile_sums(int NC) { return NC * 1024 + 32; }
__device__ __forceinline__ float *sums_at(const Params &p, int n, int unit, int part, int rt, int NC) {
  return p.ws + (((static_cast<int64_t>(n) * p.units + unit) * p.parts + part) * p.rtiles + rt) * tile_sums(NC);
}

// The turn-th kPartTiles tiles of a part (the last turn takes what is left).  KW waves a row
// tile; NC = channel tiles of 32.
template <int KW, int NC, typename Smem>
__device__ __forceinline__ void attend(const Params &p, const Seq &s, Smem &sm, int n, int unit, int group, int part,
                                       int turn, int wave, int tid) {
  constexpr int NK = (NC + 1) / 2;   // 64-channel score steps
  constexpr int kWaves = waves_of(NC), kStep = kWaves;
  constexpr int kEach = kStep / KW;  // tiles of a step that a wave takes
  const uint32_t tab0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPK_LDS char *)(void *)sm.tab));
  const int lane = tid & 63, half = lane >> 5, col = lane & 31;
  const int kvh = unit % p.Hkv, t = unit / p.Hkv, rows = s.nodes * p.nrep;
  const int kw = wave % KW, rt = group * kWaves + wave / KW, r = rt * 32 + col;
  const bool live = rt * 32 < rows;  // (without rows of its own a wave prepares tiles)

  const Keys<NK> keys(p, s, n, t, kvh, half, col);
  const int t0 = part * s.ptiles + turn * kPartTiles;
  const int stop = part + 1 < s.parts || (turn + 1) * kPartTiles < s.ptiles ? min(t0 + kPartTiles, s.end) : s.end;
  // The words of this wave's tile of a step are requested a step before they are prepared,
  // their block two.
  uint32_t kwords[NK], vwords[NK], phys = keys.block_of(t0 + wave);
  bool ok;
  auto request = [&](int first) {
    keys.load(first + wave, phys, kwords, vwords, ok);
    phys = keys.block_of(first + kStep + wave);
  };
  request(t0);
  fill_tables(p, sm.tab[0], tid);
  v8i qop[NK];
  load_query<NK>(p, s, t, kvh, min(r, rows - 1), half, qop);
  const uint32_t *mrow = p.masks + (s.first + node_of(p, min(r, rows - 1))) * p.mask_words;
  v16f acc[NC];
  Sums l;
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = v16f{};

  auto prepare = [&](int buf) {
    v8i kop[NK];
    uint32_t vt[2 * NK];
    keys.operands(kwords, vwords, ok, lane, kop, vt);
#pragma unroll
    for (int k = 0; k < NK; ++k)
      sm.k[buf][wave][k][lane] = v4u{static_cast<uint32_t>(kop[k][0]), static_cast<uint32_t>(kop[k][1]),
                                     static_cast<uint32_t>(kop[k][2]), static_cast<uint32_t>(kop[k][3])};
#pragma unroll
    for (int c = 0; c < NC; ++c) sm.v[buf][wave][c][lane] = place_bits(vt[c]);
  };
  prepare(0);
  request(t0 + kStep);
  __syncthreads();
  int buf = 0;
  for (int first = t0; first < stop; first += kStep, buf ^= 1) {
    if (first + kStep < stop) {  // the next step's tile, into the other buffer
      prepare(buf ^ 1);
      request(first + 2 * kStep);
    }
    auto tile = [&](int u, auto masked) {
      v8i kop[NK];
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        const v4u x = sm.k[buf][u][k][lane];
        kop[k] = v8i{static_cast<int>(x[0]), static_cast<int>(x[1]), static_cast<int>(x[2]), static_cast<int>(x[3])};
      }
      uint32_t w[16];
      lookup(tab0, scores<NK>(kop, qop), w);
      v8h vop[NC][2];
#pragma unroll
      for (int c = 0; c < NC; ++c) expand(sm.v[buf][u][c][lane], vop[c]);
      products<NC, decltype(masked)::value>(w, decltype(masked)::value ? seen(s, first + u, mrow, half) : 0u, vop,
                                                 acc, l);
    };
    if (live) {
      if ((first + kStep) * kKeys <= s.ctx) {  // every key counts
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
          tile(kw + u * KW, std::false_type{});
          __builtin_amdgcn_sched_barrier(0);  // tile by tile (several at a time spill)
        }
      } else {
#pragma unroll 1
        for (int u = kw; u < kStep && first + u < stop; u += KW) tile(u, std::true_type{});
      }
    }
    __syncthreads();
  }

  auto done = [&](int c, int quad, const float (&val)[4], float den) {
    if (s.parts > 1) {
      float *to = sums_at(p, n, unit, part, rt, NC), *to_den = to + NC * 1024 + col;
      v4f *at = reinterpret_cast<v4f *>(to + ((c * 4 + quad) * 64 + lane) * 4);
      const v4f sum = {val[0], val[1], val[2], val[3]};
      *at = turn ? *at + sum : sum;  // (the turns before were this lane's too)
      if (c == 0 && quad == 0 && half == 0) *to_den = turn ? *to_den + den : den;
    } else if (r < rows) {
      store_row<4>(p, s, t, kvh, r, c, quad, half, val, den);
    }
  };
  const float mine = l.total();
  if constexpr (KW == 1) {
    const float den = mine + __shfl_xor(mine, 32);
    if (!live) return;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int quad = 0; quad < 4; ++quad) {
        const float val[4] = {acc[c][4 * quad], acc[c][4 * quad + 1], acc[c][4 * quad + 2], acc[c][4 * quad + 3]};
        done(c, quad, val, den);
      }
  } else {
    // The row tile's waves in their order: wave kw finishes four channels of a lane's sixteen
    // (two waves: eight each).
    constexpr int kQuads = KW < 4 ? 4 / KW : 1;
    sm.den[wave][lane] = mine;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (c) __syncthreads();  // (the channel tile before is read)
#pragma unroll
      for (int j = 0; j < 16; ++j) sm.red[wave][j][lane] = acc[c][j];
      __syncthreads();
      if (kw >= 4 || !live) continue;
      float den = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) den += sm.den[wave - kw + w][col] + sm.den[wave - kw + w][col + 32];
#pragma unroll
      for (int x = 0; x < kQuads; ++x) {
        const int quad = kw * kQuads + x;
        float val[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j) val[j] += sm.red[wave - kw + w][quad * 4 + j][lane];
        done(c, quad, val, den);
      }
    }
  }
}

// LONG: parts of several turns (tables of more than 65,536 tokens).  Their loop costs registers:
// 55 us where 54 do without it for 61 nodes on 30,011 tokens, 139.5 for 136 (the 16 contexts
// above), 74.5 for 71.5 (128 channels), captured and replayed.
template <int NC, bool LONG>
__global__ __launch_bounds__(waves_of(NC) * 64) __attribute__((amdgpu_waves_per_eu(NC > 2 ? 2 : 4))) void
tree_attn_kernel(Params p) {
  constexpr int NK = (NC + 1) / 2, kWaves = waves_of(NC), kStep = kWaves;
  struct Smem {
    uint32_t tab[kTables][kTabStride];  // first: a score's accumulator is its entry's LDS address
    float den[kWaves][64];
    union {
      struct {
        v4u k[2][kStep][NK][64];
        v4u v[2][kStep][NC][64];
      };
      float red[kWaves][16][64];
    };
  };
  __shared__ Smem sm;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // (uniform: its branches are scalar)
  const int n = blockIdx.y;
  const int unit = blockIdx.x % p.units, rest = blockIdx.x / p.units;
  const int part = rest % p.parts, group = rest / p.parts;
  const Seq s = sequence(p, n);
  const int rows = s.nodes * p.nrep;
  if (group * kWaves * 32 >= rows || part >= s.parts) return;
  auto take = [&](int turn, int tid) {
    // (one wave a row tile throughout: 54.6 us where these take 51.6 for 32 sequences of
    // 500..5,000 tokens, captured and replayed; 8 nodes on 128 tokens and wide trees the same)
    if (rows > 16 * kWaves) attend<1, NC>(p, s, sm, n, unit, group, part, turn, wave, tid);
    else if (rows > 8 * kWaves) attend<2, NC>(p, s, sm, n, unit, group, part, turn, wave, tid);
    else if (kWaves == 4 || rows > 4 * kWaves) attend<4, NC>(p, s, sm, n, unit, group, part, turn, wave, tid);
    else attend<kWaves, NC>(p, s, sm, n, unit, group, part, turn, wave, tid);
  };
  if constexpr (LONG) {
#pragma unroll 1
    for (int t0 = part * s.ptiles, turn = 0; turn * kPartTiles < s.ptiles && (turn == 0 || t0 < s.end);
         t0 += kPartTiles, ++turn) {
      if (turn) __syncthreads();  // (the turn before has read its sums)
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));  // (nothing of a lane's is kept from turn to turn)
      take(turn, tid);
    }
  } else {
    take(0, threadIdx.x);
  }
}

// Sums of the parts, in their order.  A wave takes four channels of a lane's sixteen of an
// output tile, with kAhead parts' sums on their way at once.  Workgroups of a unit are
// numbered as the attention's are: with 8 units (or a multiple) they run on the XCD whose L2
// has the sums.
__global__ __launch_bounds__(256) void tree_join_kernel(Params p, int NC) {
  constexpr int kAhead = 8;
  const int lane = threadIdx.x & 63, quad = threadIdx.x >> 6, half = lane >> 5, col = lane & 31, n = blockIdx.y;
  const int unit = blockIdx.x % p.units, rest = blockIdx.x / p.units, c = rest % NC, rt = rest / NC;
  const Seq s = sequence(p, n);
  const int rows = s.nodes * p.nrep, r = rt * 32 + col;
  if (rt * 32 >= rows || s.parts <= 1) return;
  const int64_t stride = static_cast<int64_t>(p.rtiles) * tile_sums(NC);  // from part to part
  const float *from = sums_at(p, n, unit, 0, rt, NC);
  const float *at = from + ((c * 4 + quad) * 64 + lane) * 4;
  v4f a = {0.f, 0.f, 0.f, 0.f};
  float den = 0.f;
  for (int part = 0; part < s.parts; part += kAhead) {
    v4f x[kAhead];
    float y[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t to = min(part + u, s.parts - 1) * stride;
      x[u] = *reinterpret_cast<const v4f *>(at + to);
      y[u] = from[to + NC * 1024 + col];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (part + u >= s.parts) break;
      a += x[u];
      den += y[u];
    }
  }
  const float val[4] = {a[0], a[1], a[2], a[3]};
  if (r < rows) store_row<4>(p, s, unit / p.Hkv, unit % p.Hkv, r, c, quad, half, val, den);
}

struct Plan {
  int rtiles, groups, parts;
  size_t bytes;  // workspace
};

inline Plan plan(int T, int N, int Hq, int Hkv, int D, int max_nodes, int block_size, int max_blocks) {
  Plan r;
  const int NC = (D + 31) / 32;
  r.rtiles = static_cast<int>((static_cast<int64_t>(max_nodes) * (Hq / Hkv) + 31) / 32);
  r.groups = (r.rtiles + waves_of(NC) - 1) / waves_of(NC);
  r.parts = most_parts(static_cast<int64_t>(max_blocks) * block_size);
  r.bytes = r.parts > 1 ? static_cast<size_t>(T) * Hkv * N * r.parts * r.rtiles * tile_sums(NC) * sizeof(float) : 0;
  return r;
}

template <int NC>
static int launch(const Params &p, int N, hipStream_t s) {
  const dim3 grid(p.groups * p.parts * p.units, N);
  const int64_t tokens = static_cast<int64_t>(p.max_blocks) << p.bs_log2;
  if (tokens <= int64_t(kPartTiles) * kMaxParts * kKeys) tree_attn_kernel<NC, false><<<grid, waves_of(NC) * 64, 0, s>>>(p);
  else tree_attn_kernel<NC, true><<<grid, waves_of(NC) * 64, 0, s>>>(p);
  const int rc = check_launch("tree_attn");
  if (rc || p.parts == 1) return rc;
  tree_join_kernel<<<dim3(p.units * p.rtiles * NC, N), 256, 0, s>>>(p, NC);
  return check_launch("tree_attn");
}

}  // namespace tree
}  // namespace spk

using namespace spk;

extern "C" size_t spk_tree_attn_workspace_bytes(int T, int N, int Hq, int Hkv, int head_dim, int max_nodes,
                                                int block_size, int max_blocks) {
  if (T <= 0 || N <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0 || head_dim > 128 || max_nodes <= 0 ||
      max_nodes > tree::kMaxNodes || block_size <= 0 || max_blocks < 0)
    return 0;
  return tree::plan(T, N, Hq, Hkv, head_dim, max_nodes, block_size, max_blocks).bytes;
}

extern "C" int spk_tree_attn(const int32_t *q, const int64_t q_strides[3], const int32_t *k_tree,
                             const int32_t *v_tree, const int64_t tree_strides[3], const int32_t *k_cache,
                             const int32_t *v_cache, const int64_t cache_strides[3], int64_t num_slots,
                             const int32_t *block_tables, int64_t bt_stride0, int64_t bt_stride1,
                             const int32_t *context_lens, const int32_t *row_starts, const int64_t *masks,
                             int mask_words, void *out, int out_dtype, const int64_t out_strides[3],
                             int64_t rows, int N, int max_nodes, int T, int Hq, int Hkv, int head_dim,
                             int block_size, int max_blocks, float scale, void *workspace,
                             size_t workspace_bytes, void *stream) {
  if (T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0 || N < 0 || rows < 0 || max_nodes <= 0 ||
      max_blocks < 0 || num_slots < 0)
    return fail(SPK_EINVAL, "tree_attn: bad sizes T=%d Hq=%d Hkv=%d D=%d N=%d rows=%lld max_nodes=%d", T, Hq, Hkv,
                head_dim, N, (long long)rows, max_nodes);
  if (head_dim > 128) return fail(SPK_EUNSUPPORTED, "tree_attn: head_dim=%d (at most 128)", head_dim);
  if (max_nodes > tree::kMaxNodes)
    return fail(SPK_EUNSUPPORTED, "tree_attn: max_nodes=%d (at most %d)", max_nodes, tree::kMaxNodes);
  if (!valid_float_dtype(out_dtype)) return fail(SPK_EINVAL, "tree_attn: out dtype %d not a float type", out_dtype);
  if (!is_pow2(block_size)) return fail(SPK_EINVAL, "tree_attn: block_size=%d is not a power of two", block_size);
  if (mask_words < (max_nodes + 63) / 64)
    return fail(SPK_EINVAL, "tree_attn: %d mask words hold fewer than %d nodes", mask_words, max_nodes);
  if (!(scale > 0.f) || scale * head_dim > 12.f)  // the table's span within f16
    return fail(SPK_EINVAL, "tree_attn: scale=%g outside (0, 12/head_dim]", (double)scale);
  if (static_cast<int64_t>(max_blocks) * block_size > (1 << 30))
    return fail(SPK_EUNSUPPORTED, "tree_attn: block tables of %d x %d tokens (at most 2^30)", max_blocks, block_size);
  if (N == 0 || rows == 0) return SPK_OK;
  if (N > 65535) return fail(SPK_EUNSUPPORTED, "tree_attn: %d sequences (at most 65535)", N);
  if (!q || !k_tree || !v_tree || !context_lens || !row_starts || !masks || !out ||
      (max_blocks > 0 && !block_tables) || (num_slots > 0 && (!k_cache || !v_cache)))
    return fail(SPK_EINVAL, "tree_attn: null pointer");
  if ((T > 1 && !out_strides[0]) || (rows > 1 && !out_strides[1]) || (Hq > 1 && !out_strides[2]))
    return fail(SPK_EINVAL, "tree_attn: rows of out lie on one another");
  const tree::Plan plan = tree::plan(T, N, Hq, Hkv, head_dim, max_nodes, block_size, max_blocks);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
    return fail(SPK_EINVAL, "tree_attn: workspace of %zu bytes, %zu needed", workspace_bytes, plan.bytes);
  const int64_t units = static_cast<int64_t>(T) * Hkv;
  // (a launch has fewer than 2^32 threads along its first axis)
  if (units * plan.rtiles * plan.parts > (1 << 22) || static_cast<int64_t>(max_nodes) * (Hq / Hkv) > (1 << 24))
    return fail(SPK_EUNSUPPORTED, "tree_attn: T=%d Hq=%d Hkv=%d with %d nodes", T, Hq, Hkv, max_nodes);
  if (!tiles::divides_to(static_cast<int64_t>(max_nodes) * (Hq / Hkv), Hq / Hkv))
    return fail(SPK_EUNSUPPORTED, "tree_attn: %d heads a kv head with %d nodes", Hq / Hkv, max_nodes);
  tree::Params p{};
  p.q = reinterpret_cast<const uint32_t *>(q);
  p.qs0 = q_strides[0]; p.qs1 = q_strides[1]; p.qs2 = q_strides[2];
  p.kt = reinterpret_cast<const uint32_t *>(k_tree);
  p.vt = reinterpret_cast<const uint32_t *>(v_tree);
  p.ts0 = tree_strides[0]; p.ts1 = tree_strides[1]; p.ts2 = tree_strides[2];
  p.k = reinterpret_cast<const uint32_t *>(k_cache);
  p.v = reinterpret_cast<const uint32_t *>(v_cache);
  p.ks0 = cache_strides[0]; p.ks1 = cache_strides[1]; p.ks2 = cache_strides[2];
  p.num_slots = num_slots;
  if (num_slots < block_size) {  // no block of a cache: every key is dropped, the loads read q's words
    p.k = p.v = p.q;
    p.ks0 = p.ks1 = p.ks2 = 0;
  }
  p.wide = p.num_slots * p.ks2 > (1ll << 30) || p.ks2 < 0;
  p.bt = block_tables; p.bts0 = bt_stride0; p.bts1 = bt_stride1;
  if (max_blocks == 0) {  // no context: the loads of a table entry read the lengths
    p.bt = context_lens;
    p.bts0 = p.bts1 = 0;
  }
  p.lens = context_lens; p.starts = row_starts;
  p.masks = reinterpret_cast<const uint32_t *>(masks); p.mask_words = 2 * mask_words;
  p.out = out; p.out_dtype = out_dtype;
  p.os0 = out_strides[0]; p.os1 = out_strides[1]; p.os2 = out_strides[2];
  p.out_vec = head_dim % 4 == 0 && p.os0 % 4 == 0 && p.os1 % 4 == 0 && p.os2 % 4 == 0 &&
              (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  p.rows = rows; p.units = static_cast<int>(units); p.Hkv = Hkv; p.nrep = Hq / Hkv; p.D = head_dim;
  p.W = (head_dim + 31) / 32; p.bs_log2 = ilog2(block_size); p.max_blocks = max_blocks; p.max_nodes = max_nodes;
  p.rep_mul = tiles::inverse_of(p.nrep);
  p.rtiles = plan.rtiles; p.groups = plan.groups; p.parts = plan.parts; p.ws = static_cast<float *>(workspace);
  tiles::build_table(scale, head_dim, p.tab);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (p.W) {
    case 1: return tree::launch<1>(p, N, s);
    case 2: return tree::launch<2>(p, N, s);
    case 3: return tree::launch<3>(p, N, s);
    default: return tree::launch<4>(p, N, s);
  }
}
