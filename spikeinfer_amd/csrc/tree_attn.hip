// Attention of drafted token trees over the paged packed cache (head_dim <= 128).
//
// Row r of a sequence (a drafted token) attends, per timestep and query head, to
// the sequence's cached context and to the drafted tokens that its mask names:
//   out = sum_j w_j bits(v_j) / sum_j w_j,  w_j = exp(popc(q & k_j) * scale).
//
// MI355X design, on the tiles of the prefill attention (spike_tiles.hpp):
//   * A workgroup owns 32 * QT rows of one (t, kv head): row r = node r / n_rep, query
//     head r % n_rep.  Its four waves take the 32-key tiles round-robin: first the
//     context's, then the tree's own, which start on a tile of their own, so that a
//     row's mask word is the tile's.
//   * Scores, weights and values as there: one fp4 product per 64 channels leaves the
//     score's table offset in the accumulator's bits, the weight is a look-up, and f16
//     products over two keys a register add bits(v) times the weight.  bf16 outputs take
//     the weights' 11-bit high halves alone (each off by at most 2^-11, and the
//     denominator sums the same halves, where an output's own rounding is 2^-8): half the
//     products.  fp32 and fp16 outputs take both halves, to accumulators of their own,
//     added and divided in fp64.
//   * The context is cut into parts of kPart tokens, the tree's tiles belonging to the
//     last; a part's sums are added over the waves, and parts in their order.  One
//     workgroup takes the parts one after the other, or, where rows are few, a workgroup
//     a part leaves its sums in the workspace and a second launch adds them: the same
//     additions, so a sequence's outputs depend neither on that choice nor on the batch.
#include <type_traits>

#include "spike_tiles.hpp"

namespace spk {
namespace tree {

using namespace tiles;

constexpr int kWaves = 4;
constexpr int kKeys = 32;              // keys per tile
constexpr int kPart = 4096;            // tokens per part
constexpr int kPartTiles = kPart / kKeys;
constexpr int kMaxNodes = 1024;
static_assert(kPartTiles % kWaves == 0, "a wave's tiles go on across parts");

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
  uint32_t rep_mul;         // floor(r / nrep) = r * rep_mul >> 32 for every row
  int units, Hkv, nrep, D, W, bs_log2, max_blocks, max_nodes;
  int groups;               // row groups of a sequence (grid.x = groups * parts * units)
  int parts;                // workgroups along the context: 1, or a part each
  char *ws;                 // with parts > 1: sums of (sequence, group, part, unit)
  uint32_t tab[kTab];
};

// A sequence as the kernels take it: its rows and cached tokens, clamped to the buffers.
struct Seq {
  int64_t first;
  int nodes, ctx, ctiles, parts;
};

__device__ __forceinline__ Seq sequence(const Params &p, int n) {
  Seq s;
  s.first = min<int64_t>(max(p.starts[n], 0), p.rows);
  const int64_t end = min(max<int64_t>(p.starts[n + 1], s.first), p.rows);
  s.nodes = static_cast<int>(min<int64_t>(end - s.first, p.max_nodes));
  s.ctx = min(max(p.lens[n], 0), p.max_blocks << p.bs_log2);
  s.ctiles = (s.ctx + kKeys - 1) / kKeys;
  s.parts = max(1, (s.ctiles + kPartTiles - 1) / kPartTiles);
  return s;
}

// What a workgroup's threads finish: kTiles of its QT x NC output tiles a round, a wave a
// tile, or, of a tile in two parts (fp32), a wave a half.
template <int QT, int NC, bool F32>
struct Shape {
  static constexpr int kUnits = QT * NC;
  static constexpr int kParts = F32 ? 2 : 1;
  static constexpr int kTiles = kWaves / kParts;
  static constexpr int kRounds = (kUnits + kTiles - 1) / kTiles;
  static constexpr int kVals = 16 / kParts;  // values a lane and round
  typedef std::conditional_t<F32, double, float> Sum;
  // one (sequence, group, part, unit) of the workspace: values as the lanes hold them,
  // then the rows' denominators
  static constexpr int kSums = kRounds * kVals * kWaves * 64;
  static constexpr size_t kBytes = sizeof(Sum) * (kSums + 32 * QT);
};

// Rows r0.. of a sequence from their sums: tot as Shape has them, dens in LDS.
template <int QT, int NC, bool F32>
__device__ __forceinline__ void store_rows(const Params &p, const Seq &s, int unit, int r0,
                                           const typename Shape<QT, NC, F32>::Sum (
                                               &tot)[Shape<QT, NC, F32>::kRounds][Shape<QT, NC, F32>::kVals],
                                           const typename Shape<QT, NC, F32>::Sum *dens) {
  typedef Shape<QT, NC, F32> S;
  typedef typename S::Sum Sum;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, col = lane & 31;
  const int kvh = unit % p.Hkv, t = unit / p.Hkv, rows = s.nodes * p.nrep;
#pragma unroll
  for (int rd = 0; rd < S::kRounds; ++rd) {
    const int x = rd * S::kTiles + wave / S::kParts;
    const int i = x / NC, c = x - i * NC, r = r0 + 32 * i + col;
    if (x >= S::kUnits || r >= rows) continue;
    const Sum den = dens[32 * i + col];
    const Sum inv = den > 0 ? Sum(1) / den : Sum(0);  // (a row that sees nothing: zeros)
    const int node = p.nrep == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), p.rep_mul));
    const int64_t row = t * p.os0 + (s.first + node) * p.os1 + (kvh * p.nrep + r - node * p.nrep) * p.os2;
    const int g0 = F32 ? wave % S::kParts * 2 : 0;  // first of the wave's 4-channel groups
    constexpr int kGroups = S::kVals / 4;
    if (p.out_vec) {  // D % 4 == 0: four channels lie in or out together
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        const int ch = 32 * c + 8 * (g0 + k) + 4 * half;
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = static_cast<float>(tot[rd][4 * k + e] * inv);
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
      for (int j = 0; j < S::kVals; ++j) {
        const int ch = 32 * c + 8 * (g0 + (j >> 2)) + 4 * half + (j & 3);
        if (ch < p.D) store_f32_as(p.out, row + ch, p.out_dtype, static_cast<float>(tot[rd][j] * inv));
      }
    }
  }
}

// QT row tiles of 32 rows a workgroup; NC = channel tiles of 32 (ceil(D / 32)).
// F32: weights of two halves (fp32 and fp16 outputs).
template <int QT, int NC, bool F32>
__global__ __launch_bounds__(kWaves * 64) __attribute__((amdgpu_waves_per_eu(2))) void tree_attn_kernel(Params p) {
  typedef Shape<QT, NC, F32> S;
  typedef typename S::Sum Sum;
  constexpr int NK = (NC + 1) / 2;  // 64-channel score steps
  constexpr int kParts = S::kParts;
  struct Smem {
    uint32_t tab[kTab + 3];  // first: a score's accumulator is its entry's LDS address
    Sum dens[32 * QT];
    float lsum[QT][kParts][kWaves][64];
    float red[S::kUnits * kParts < kWaves ? S::kUnits * kParts : kWaves][kWaves][16][64];
  };
  __shared__ Smem sm;
  const uint32_t tab0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((SPK_LDS char *)(void *)sm.tab));

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int half = lane >> 5, col = lane & 31;
  const int n = blockIdx.y;
  const int unit = blockIdx.x % p.units, rest = blockIdx.x / p.units;
  const int part = rest % p.parts, group = rest / p.parts;
  const int kvh = unit % p.Hkv, t = unit / p.Hkv;
  const Seq s = sequence(p, n);
  const int rows = s.nodes * p.nrep, r0 = group * 32 * QT;
  if (r0 >= rows || part >= s.parts) return;
  const int nq = min(QT, (rows - r0 + 31) >> 5);

  if (tid <= p.D) sm.tab[tid] = p.tab[tid];

  // Each lane's rows (clamped to the last): query words as score operands, mask words.
  v8i qop[QT][NK];
  const uint32_t *mrow[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = min(r0 + 32 * i + col, rows - 1);
    const int node = p.nrep == 1 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), p.rep_mul));
    const int h = r - node * p.nrep;
    mrow[i] = p.masks + (s.first + node) * p.mask_words;
    const uint32_t *qp = p.q + t * p.qs0 + (s.first + node) * p.qs1 + (kvh * p.nrep + h) * p.qs2;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int w = 2 * k + half;
      qop[i][k] = fp4_bits(w < p.W ? qp[w] : 0u);
    }
  }

  const int32_t *table = p.bt + n * p.bts0;
  const int bs_mask = (1 << p.bs_log2) - 1;
  const uint32_t nblocks = static_cast<uint32_t>(min<int64_t>(p.num_slots >> p.bs_log2, 0xffffffffll));
  const uint32_t *kbase = p.k + t * p.ks0 + kvh * p.ks1, *vbase = p.v + t * p.ks0 + kvh * p.ks1;
  const uint32_t *ktree = p.kt + t * p.ts0 + s.first * p.ts1 + kvh * p.ts2;
  const uint32_t *vtree = p.vt + t * p.ts0 + s.first * p.ts1 + kvh * p.ts2;
  const int last_block = max(s.ctx - 1, 0) >> p.bs_log2;
  // Loads are unconditional (indices clamped into range, the value dropped where a key
  // is none: zero spikes), so that the wave waits for none of them before its use.
  auto block_of = [&](int kt) -> uint32_t {
    return static_cast<uint32_t>(table[min((kt * kKeys + col) >> p.bs_log2, last_block) * p.bts1]);
  };
  auto load = [&](int kt, uint32_t phys, uint32_t (&kw)[NK], uint32_t (&vw)[NK], bool &ok) {
    const bool own = kt >= s.ctiles;
    const int j = (own ? kt - s.ctiles : kt) * kKeys + col;
    ok = own ? j < s.nodes : j < s.ctx && phys < nblocks;
    const int64_t slot = (static_cast<int64_t>(phys) << p.bs_log2) | (j & bs_mask);
    const int64_t at = ok ? (own ? j * p.ts1 : slot * p.ks2) : 0;
    const uint32_t *kp = (own ? ktree : kbase) + at, *vp = (own ? vtree : vbase) + at;
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const int w = min(2 * k + half, p.W - 1);
      kw[k] = kp[w];
      vw[k] = vp[w];
    }
  };
  auto keep = [&](uint32_t x, int k, bool ok) { return ok && 2 * k + half < p.W ? x : 0u; };

  Sum tot[S::kRounds][S::kVals], dtot = 0;
#pragma unroll
  for (int rd = 0; rd < S::kRounds; ++rd)
#pragma unroll
    for (int j = 0; j < S::kVals; ++j) tot[rd][j] = 0;
  __syncthreads();

  const int p0 = part, p1 = p.parts > 1 ? part + 1 : s.parts;
  const int end = s.ctiles + (s.nodes + kKeys - 1) / kKeys;  // all tiles of the sequence
  uint32_t kw[NK], vw[NK];
  bool ok;
  int kt = p0 * kPartTiles + wave;
  load(kt, block_of(kt), kw, vw, ok);
  uint32_t pnext = block_of(kt + kWaves);
  for (int pt = p0; pt < p1; ++pt) {
    v16f acc[QT][NC * kParts];
    float l[QT][kParts];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
#pragma unroll
      for (int q = 0; q < kParts; ++q) l[i][q] = 0.f;
#pragma unroll
      for (int c = 0; c < NC * kParts; ++c) acc[i][c] = v16f{};
    }
    const int stop = pt + 1 < s.parts ? (pt + 1) * kPartTiles : end;
    for (; kt < stop; kt += kWaves) {
      // Operands of this tile; the next tile's words and the block of the one
      // after are requested before they are used.
      v8i kop[NK];
      uint32_t vt[2 * NK];
#pragma unroll
      for (int k = 0; k < NK; ++k) {
        kop[k] = fp4_bits(keep(kw[k], k, ok));
        const uint32_t x = transpose32(keep(vw[k], k, ok), lane);
        // Both halves of the wave need every channel tile: lanes l and l + 32 take
        // keys 4 * (l / 32) + 0..3 of each eight.
        const auto sw = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        vt[2 * k] = sw[0] >> (4 * half);
        vt[2 * k + 1] = sw[1] >> (4 * half);
      }
      load(kt + kWaves, pnext, kw, vw, ok);
      pnext = block_of(kt + 2 * kWaves);
      // The lane's n-th key of the tile is 8 * (n >> 2) + 4 * half + (n & 3), n < 16.
      // Register e of the operands pairs keys e and e + 8, sixteen bits apart in vt; a
      // bit b at place s <= 3 becomes f16 1.0 by a 24-bit product with 0x3c00 >> s.
      v8h vop[NC][2];
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t b = g ? vt[c] >> 8 : vt[c];
          v4u x;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __umul24(b & (0x00010001u << i), 0x3c00u >> i);
          vop[c][g] = __builtin_bit_cast(v8h, x);
        }
      auto scores = [&](int i) {
        v16f a = {};
#pragma unroll
        for (int k = 0; k < NK; ++k)
          a = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kop[k], qop[i][k], a, 4, 4, 0, 55, 0, 54);
        return a;
      };
      auto lookup = [&](const v16f &a, uint32_t (&w)[16]) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t at = tab0 + __float_as_uint(a[e]);
          w[e] = *reinterpret_cast<const SPK_LDS uint32_t *>(static_cast<uintptr_t>(at));
        }
      };
      auto products = [&](int i, const uint32_t (&w)[16], uint32_t see, auto masked) {
        auto weight = [&](int e) {  // the e-th of the lane's sixteen
          if constexpr (decltype(masked)::value)
            return w[e] & static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(see), 8 * (e >> 2) + (e & 3), 1));
          else return w[e];
        };
        float d[4] = {0.f, 0.f, 0.f, 0.f};  // (a chain of dot2 on one register waits for itself)
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          v4u x[kParts];  // the weights' halves, two keys a register
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t y0 = weight(4 * g + e), y1 = weight(4 * g + e + 8);
#pragma unroll
            for (int q = 0; q < kParts; ++q) {
              const uint32_t y = __builtin_amdgcn_perm(y1, y0, q ? 0x07060302u : 0x05040100u);
              float &dq = d[kParts == 2 ? 2 * (e & 1) + q : e];
              dq = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, y), v2h{1, 1}, dq, false);
              x[q][e] = y;
            }
          }
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int q = 0; q < kParts; ++q) {
              v16f &a = acc[i][kParts * c + q];
              a = __builtin_amdgcn_mfma_f32_32x32x16_f16(vop[c][g], __builtin_bit_cast(v8h, x[q]), a, 0, 0, 0);
            }
        }
        if constexpr (kParts == 2) {
          l[i][0] += d[0] + d[2];
          l[i][1] += d[1] + d[3];
        } else {
          l[i][0] += (d[0] + d[1]) + (d[2] + d[3]);
        }
      };
      if (kt * kKeys + kKeys <= s.ctx && nq == QT) {
        // The next row tile's scores are computed and looked up under this one's
        // products.
        uint32_t w[2][16];
        lookup(scores(0), w[0]);
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          if (i + 1 < QT) lookup(scores(i + 1), w[(i + 1) & 1]);
          products(i, w[i & 1], 0u, std::false_type{});
          __builtin_amdgcn_sched_barrier(0);  // row tile by row tile (several at a time spill)
        }
      } else {
        const int nt = kt - s.ctiles;  // the tree's tile, or the context's last
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          if (i >= nq) continue;
          const int left = (nt < 0 ? s.ctx - kt * kKeys : s.nodes - nt * kKeys);
          uint32_t see = left >= 32 ? ~0u : (1u << left) - 1;
          if (nt >= 0) see &= mrow[i][nt];
          uint32_t w[16];
          lookup(scores(i), w);
          products(i, w, see >> (4 * half), std::true_type{});
        }
      }
    }

    // The part's sums over the waves, in wave order, added to those of the parts before.
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int q = 0; q < kParts; ++q) sm.lsum[i][q][wave][lane] = l[i][q];
#pragma unroll
    for (int rd = 0; rd < S::kRounds; ++rd) {
      if (rd) __syncthreads();
#pragma unroll
      for (int u = 0; u < kWaves; ++u) {
        const int x = rd * S::kTiles + u / kParts;
        if (x < S::kUnits) {
#pragma unroll
          for (int j = 0; j < 16; ++j) sm.red[u][wave][j][lane] = acc[x / NC][x % NC * kParts + u % kParts][j];
        }
      }
      __syncthreads();
      if (rd == 0 && tid < 32 * QT) {
        Sum d = 0;
#pragma unroll
        for (int q = 0; q < kParts; ++q)
#pragma unroll
          for (int w = 0; w < kWaves; ++w)
            d += static_cast<Sum>(sm.lsum[tid >> 5][q][w][tid & 31]) + static_cast<Sum>(sm.lsum[tid >> 5][q][w][(tid & 31) + 32]);
        dtot += d;
      }
      if (rd * S::kTiles + wave / kParts < S::kUnits) {
        const int slot = wave / kParts * kParts, j0 = F32 ? wave % kParts * 8 : 0;
#pragma unroll
        for (int j = 0; j < S::kVals; ++j) {
          Sum a = 0;
#pragma unroll
          for (int q = 0; q < kParts; ++q)
#pragma unroll
            for (int w = 0; w < kWaves; ++w) a += sm.red[slot + q][w][j0 + j][lane];
          tot[rd][j] += a;
        }
      }
    }
    __syncthreads();
  }

  if (p.parts > 1 && s.parts > 1) {
    Sum *to = reinterpret_cast<Sum *>(
        p.ws + (((static_cast<int64_t>(n) * p.groups + group) * p.parts + part) * p.units + unit) * S::kBytes);
#pragma unroll
    for (int rd = 0; rd < S::kRounds; ++rd)
#pragma unroll
      for (int j = 0; j < S::kVals; ++j) to[(rd * S::kVals + j) * (kWaves * 64) + tid] = tot[rd][j];
    if (tid < 32 * QT) to[S::kSums + tid] = dtot;
    return;
  }
  if (tid < 32 * QT) sm.dens[tid] = dtot;
  __syncthreads();
  store_rows<QT, NC, F32>(p, s, unit, r0, tot, sm.dens);
}

// Sums of the parts, in their order.
template <int QT, int NC, bool F32>
__global__ __launch_bounds__(kWaves * 64) void tree_join_kernel(Params p) {
  typedef Shape<QT, NC, F32> S;
  typedef typename S::Sum Sum;
  __shared__ Sum dens[32 * QT];
  const int tid = threadIdx.x, n = blockIdx.y, unit = blockIdx.x % p.units, group = blockIdx.x / p.units;
  const Seq s = sequence(p, n);
  if (group * 32 * QT >= s.nodes * p.nrep || s.parts <= 1) return;
  Sum tot[S::kRounds][S::kVals], dtot = 0;
#pragma unroll
  for (int rd = 0; rd < S::kRounds; ++rd)
#pragma unroll
    for (int j = 0; j < S::kVals; ++j) tot[rd][j] = 0;
  for (int part = 0; part < s.parts; ++part) {
    const Sum *from = reinterpret_cast<const Sum *>(
        p.ws + (((static_cast<int64_t>(n) * p.groups + group) * p.parts + part) * p.units + unit) * S::kBytes);
#pragma unroll
    for (int rd = 0; rd < S::kRounds; ++rd)
#pragma unroll
      for (int j = 0; j < S::kVals; ++j) tot[rd][j] += from[(rd * S::kVals + j) * (kWaves * 64) + tid];
    if (tid < 32 * QT) dtot += from[S::kSums + tid];
  }
  if (tid < 32 * QT) dens[tid] = dtot;
  __syncthreads();
  store_rows<QT, NC, F32>(p, s, unit, group * 32 * QT, tot, dens);
}

// Row tiles a workgroup takes of the `qt` asked for: as many as its sums leave
// registers for.
constexpr int row_tiles(int qt, int NC, bool f32) {
  const int most = NC > 3 ? (f32 ? 1 : 2) : (NC > 2 ? (f32 ? 1 : 2) : (f32 ? 2 : 4));
  return qt < most ? qt : most;
}

struct Plan {
  int qt, groups, parts;  // as asked of row_tiles; of a sequence; along the context
  size_t bytes;           // workspace
};

// The launch of a shape.  Row tiles share a key tile's operands, so four to a workgroup
// while that leaves two workgroups a CU; a workgroup a part of the context where there
// would be fewer than two a CU without.
inline Plan plan(int T, int N, int Hq, int Hkv, int D, int max_nodes, int block_size, int max_blocks, bool f32) {
  Plan r;
  const int NC = (D + 31) / 32;
  const int64_t units = static_cast<int64_t>(T) * Hkv * N;
  const int64_t rtiles = (static_cast<int64_t>(max_nodes) * (Hq / Hkv) + 31) / 32;
  const int64_t parts = (static_cast<int64_t>(max_blocks) * block_size + kPart - 1) / kPart;
  r.qt = 1;
  for (int qt = 4; qt > 1; qt >>= 1) {
    const int used = row_tiles(qt, NC, f32);
    if (used == qt && rtiles > qt / 2 && units * ((rtiles + qt - 1) / qt) * (parts > 1 ? parts : 1) >= 512) {
      r.qt = qt;
      break;
    }
  }
  r.groups = static_cast<int>((rtiles + r.qt - 1) / r.qt);
  r.parts = parts > 1 && units * r.groups < 1024 ? static_cast<int>(parts) : 1;
  r.bytes = 0;
  if (r.parts > 1) {
    const int kParts = f32 ? 2 : 1, tiles = kWaves / kParts, rounds = (r.qt * NC + tiles - 1) / tiles;
    r.bytes = static_cast<size_t>(units) * r.groups * r.parts * (f32 ? 8 : 4) *
              (rounds * (16 / kParts) * kWaves * 64 + 32 * r.qt);
  }
  return r;
}

template <int QT, int NC, bool F32>
static int launch_one(const Params &p, int N, hipStream_t s) {
  if constexpr (row_tiles(QT, NC, F32) == QT) {
    tree_attn_kernel<QT, NC, F32><<<dim3(p.groups * p.parts * p.units, N), kWaves * 64, 0, s>>>(p);
    int rc = check_launch("tree_attn");
    if (rc || p.parts == 1) return rc;
    tree_join_kernel<QT, NC, F32><<<dim3(p.groups * p.units, N), kWaves * 64, 0, s>>>(p);
    return check_launch("tree_attn");
  }
  return fail(SPK_EINVAL, "tree_attn: no kernel of %d row tiles", QT);
}

template <int QT, bool F32>
static int launch(const Params &p, int N, hipStream_t s) {
  switch ((p.D + 31) / 32) {
    case 1: return launch_one<QT, 1, F32>(p, N, s);
    case 2: return launch_one<QT, 2, F32>(p, N, s);
    case 3: return launch_one<QT, 3, F32>(p, N, s);
    default: return launch_one<QT, 4, F32>(p, N, s);
  }
}

}  // namespace tree
}  // namespace spk

using namespace spk;

extern "C" size_t spk_tree_attn_workspace_bytes(int T, int N, int Hq, int Hkv, int head_dim, int max_nodes,
                                                int block_size, int max_blocks) {
  if (T <= 0 || N <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0 || head_dim > 128 || max_nodes <= 0 ||
      max_nodes > tree::kMaxNodes || block_size <= 0 || max_blocks < 0)
    return 0;
  const size_t a = tree::plan(T, N, Hq, Hkv, head_dim, max_nodes, block_size, max_blocks, false).bytes;
  const size_t b = tree::plan(T, N, Hq, Hkv, head_dim, max_nodes, block_size, max_blocks, true).bytes;
  return a > b ? a : b;  // (whatever the outputs' type)
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
  const bool f32 = out_dtype != SPK_BF16;
  const tree::Plan plan = tree::plan(T, N, Hq, Hkv, head_dim, max_nodes, block_size, max_blocks, f32);
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes))
    return fail(SPK_EINVAL, "tree_attn: workspace of %zu bytes, %zu needed", workspace_bytes, plan.bytes);
  const int64_t units = static_cast<int64_t>(T) * Hkv;
  if (units * plan.groups * plan.parts > 0x7fffffffll || static_cast<int64_t>(max_nodes) * (Hq / Hkv) > (1 << 24))
    return fail(SPK_EUNSUPPORTED, "tree_attn: T=%d Hq=%d Hkv=%d with %d nodes", T, Hq, Hkv, max_nodes);
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
  // ceil(2^32 / nrep): its product with r is off by less than r * nrep, below 2^32
  p.rep_mul = static_cast<uint32_t>(((int64_t(1) << 32) + p.nrep - 1) / p.nrep);
  p.groups = plan.groups; p.parts = plan.parts; p.ws = static_cast<char *>(workspace);
  tiles::build_table(scale, head_dim, p.tab);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (f32) return plan.qt >= 2 ? tree::launch<2, true>(p, N, s) : tree::launch<1, true>(p, N, s);
  return plan.qt == 4 ? tree::launch<4, false>(p, N, s)
                      : (plan.qt == 2 ? tree::launch<2, false>(p, N, s) : tree::launch<1, false>(p, N, s));
}
