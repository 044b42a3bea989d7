// Linear layer in 8-bit integers: y = x W^T (+ bias) with a scale for every row of x (a
// token) and every row of W (an output channel),
//   s = max |x| / 127,  q = rint(x / s)  (both quotients rounded to fp32),
//   y[m, n] = s_x[m] s_w[n] sum_k q_x[m, k] q_w[n, k] + bias[n].
// The integer sum is exact (127^2 K < 2^31 for K <= 131,072); its product with the scales
// and the bias are fp32, rounded once to y's type.
//
// Operands lie in the order of the matrix instruction (v_mfma_i32_16x16x64_i8): 16 rows by
// 64 k are one block of 1 KB, lane l's 16 bytes row l % 16 and the k of 8 (l / 16) .. + 7 and
// 32 + 8 (l / 16) .. + 7 (any order will do that is both operands'; in this one four lanes load
// 64 bytes of a row of 16-bit numbers side by side), blocks of a row tile one behind the other.  W is laid out once (spk_linear_int8_pack), x by the
// call's first kernel, with the same code.  W is the instruction's first operand, so a lane
// holds four columns of one row of y; a tile of W has four runs of four of a group of 64
// output channels (tile j of a group: channels 16 q + 4 j + e in row 4 q + e), so that the
// four tiles of a group give a lane 16 columns side by side, and a wave writes whole 128-byte
// lines of y (8,188 x 9,728 of K = 64, nearly all stores: 67 -> 43 us, 44 with any scales).
#include <algorithm>
#include <cmath>

#include "common.hpp"
#include "lif_math.hpp"

namespace spk {
namespace i8 {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;      // k of a block
constexpr int kMaxK = 131072;  // 127^2 kMaxK < 2^31
constexpr int kRowWaves = 16;  // at most, of a tile of rows
constexpr int kKeep = 5;       // blocks a wave keeps between the two passes

inline int row_waves(int KS) { return std::min(kRowWaves, (KS + 1) / 2); }
inline int64_t row_tiles(int64_t rows) { return (rows + 15) / 16; }
inline int64_t k_steps(int64_t K) { return (K + kStep - 1) / kStep; }
inline int64_t packed_bytes(int64_t rows, int64_t K) { return row_tiles(rows) * k_steps(K) * 1024; }
inline int64_t scale_bytes(int64_t rows) { return row_tiles(rows) * 64; }
inline int groups_of(int64_t N) { return static_cast<int>((N + 63) / 64); }  // of 64 output channels

// Sixteen elements of a row, as a block has them in a lane: eight from `k0` on and eight from
// k0 + 32.  What lies behind K is zero.
template <int DT>
struct Block {
  typedef typename Elem<DT>::T E;
  E e[16];

  __device__ __forceinline__ void load(const void *row, int k0, int K) {
    typedef E Eight __attribute__((ext_vector_type(8), aligned(sizeof(E))));  // (rows need no alignment)
    const E *p = static_cast<const E *>(row);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = k0 + 32 * h;
      if (k + 8 <= K) {
        const Eight a = *reinterpret_cast<const Eight *>(p + k);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const E v = a[j];
          e[8 * h + j] = v;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[8 * h + j] = k + j < K ? p[k + j] : static_cast<E>(0);
      }
    }
  }
  // The largest magnitude's bits as fp32 (a NaN's are the largest).
  __device__ __forceinline__ uint32_t most() const {
    uint32_t m = 0;
    if constexpr (DT == SPK_F32) {
#pragma unroll
      for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(e[j]) & 0x7fffffffu);
      return m;
    } else {  // (16-bit numbers of either type are ordered as their bits, infinities and NaN above)
      typedef uint16_t U2 __attribute__((ext_vector_type(2)));
      U2 w = {0, 0};
#pragma unroll
      for (int j = 0; j < 16; j += 2) w = __builtin_elementwise_max(w, U2{static_cast<uint16_t>(e[j] & 0x7fff), static_cast<uint16_t>(e[j + 1] & 0x7fff)});
      m = max(w[0], w[1]);
      return __float_as_uint(elem_to_f32<DT>(static_cast<E>(m)));
    }
  }
};

// A row's scale.  A row that holds an infinity or a NaN (most: the largest magnitude's bits)
// has the scale NaN, so that its products are NaN as those of the numbers themselves would be.
struct Scale {
  float s, inv;
  bool some, tiny;
};
__device__ __forceinline__ Scale scale_of(uint32_t most) {
  const bool finite = most < 0x7f800000u;
  Scale r;
  r.s = finite ? __uint_as_float(most) / 127.f : __uint_as_float(0x7fc00000u);
  r.some = finite && r.s > 0.f;
  r.tiny = !(r.s >= 0x1p-100f);  // 1 / s may have no value
  r.inv = r.tiny ? 0.f : 1.f / r.s;
  return r;
}

// rint(x / s) with the quotient rounded to fp32.  x inv is off by less than two steps of fp32
// (1.5e-5 at 127), so where it lies further than that from a half its rounding is the same
// (adding 1.5 2^23 rounds to an integer in the low bits).  Near a half h = n + 1/2 the quotient rounds to
// h itself where |x - h s| <= s ulp(h) / 2 (h has few bits, a tie is its), and to h's side
// otherwise; x - h s is exact there.  A row whose largest magnitude is 127 times a power of two
// has many halves: 64 rows of 4,864 with one such 5.7 us, 9.6 with divisions.
template <int DT>
__device__ __forceinline__ v4i quantise16(const Block<DT> &b, const Scale &sc) {
  v4i out = {0, 0, 0, 0};
  if (!sc.some) return out;
  constexpr float kMagic = 12582912.f, kNear = 0.5f - 6.2e-5f;
  uint32_t w[16];
  float far = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float x = elem_to_f32<DT>(b.e[j]);
    const float y = __builtin_fmaf(x, sc.inv, kMagic);
    far = fmaxf(far, fabsf(__builtin_fmaf(x, sc.inv, -(y - kMagic))));
    w[j] = __float_as_uint(y);
  }
  if (far > kNear || sc.tiny) {
    const float up = sc.tiny ? 0x1p100f : 1.f, inv = sc.tiny ? 1.f / (sc.s * up) : sc.inv, t = sc.s * up * 0x1p-24f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float x = elem_to_f32<DT>(b.e[j]) * up, y = __builtin_fmaf(x, inv, kMagic) - kMagic;
      const float d = __builtin_fmaf(x, inv, -y);
      if (fabsf(d) > kNear || sc.tiny) {
        const float h = y + copysignf(0.5f, d), r = __builtin_fmaf(-h, sc.s * up, x);
        const float ulp = __uint_as_float(__float_as_uint(h) & 0x7f800000u);  // (over 2^-23)
        const float q = fabsf(r) <= ulp * t ? rintf(h) : h + copysignf(0.5f, r);
        w[j] = __float_as_uint(fminf(fmaxf(q, -127.f), 127.f) + kMagic);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t lo = __builtin_amdgcn_perm(w[4 * q + 1], w[4 * q], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(w[4 * q + 3], w[4 * q + 2], 0x0c0c0400u);
    out[q] = static_cast<int>(lo | hi << 16);
  }
  return out;
}

// A workgroup R rows of a tile (16 or 4): their largest magnitudes, then the integers.  A wave
// takes 16 / R blocks at a time, in all R of their rows; the waves share the row's blocks and keep
// them in registers between the two (kKeep times; longer rows are read again).  WEIGHT: rows in
// the order of the groups of output channels.  Rows that do not exist become zeros.  Bound by
// reading x and by the latency of the two passes: 16,384 rows of 4,864 in bf16 56 us (239 MB read
// and written, 4.3 TB/s), 8,188 of 896 9 us.  Up to 64 tiles by four rows a workgroup: 1,000 rows of 896
// 4.8 us (by 16 rows 8.5), 333 of 777 4.8 (8.9).  The whole call with 896 columns by four and by
// 16 rows, on both sides of that border, us: K = 896, 1,024 rows 12.2 and 12.7, 1,040 11.8 and
// 12.5, 4,096 19.3 and 19.4, 16,384 34.9 and 35.8; K = 4,864, 64 rows 13.9 and 20.8, 1,024 22.0 and 28.2,
// 1,040 22.9 and 28.1, 2,048 36.4 and 39.2, 4,096 53.9 and 52.1, 16,384 143 and 131: from 1,025 to about
// 3,000 long rows the rule's side is the slower one, by up to 5 us.
template <int DT, bool WEIGHT, int R>
__global__ __launch_bounds__(64 * kRowWaves) void rows_kernel(const void *x, int64_t stride, int64_t rows, int K, int KS,
                                                              v4i *packed, float *scales) {
  constexpr int kBlocks = 16 / R;
  __shared__ uint32_t most[kRowWaves][R];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int r16 = static_cast<int>(blockIdx.x % kBlocks) * R + lane % R, kq = lane / R % 4;
  const int64_t tile = blockIdx.x / kBlocks;
  const int64_t row = WEIGHT ? tile / 4 * 64 + 16 * (r16 >> 2) + 4 * (tile & 3) + (r16 & 3) : 16 * tile + r16;
  const bool real = row < rows;
  const char *p = static_cast<const char *>(x) + (real ? row : 0) * stride * static_cast<int64_t>(sizeof(typename Elem<DT>::T));
  const int Kr = real ? K : 0;
  const int first = wave * kBlocks + lane / (4 * R), next = waves * kBlocks;
  v4i *to = packed + tile * KS * 64 + kq * 16 + r16;
  Block<DT> v[kKeep];
#pragma unroll
  for (int q = 0; q < kKeep; ++q)
    if (first + q * next < KS) v[q].load(p, kStep * (first + q * next) + 8 * kq, Kr);
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < kKeep; ++q)
    if (first + q * next < KS) m = max(m, v[q].most());
  for (int ks = first + kKeep * next; ks < KS; ks += next) {
    Block<DT> a;
    a.load(p, kStep * ks + 8 * kq, Kr);
    m = max(m, a.most());
  }
#pragma unroll
  for (int d = R; d < 64; d <<= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), d)));
  if (lane < R) most[wave][lane] = m;
  __syncthreads();
  for (int w = 0; w < waves; ++w) m = max(m, most[w][lane % R]);
  const Scale sc = scale_of(m);
  if (threadIdx.x < R) scales[row] = sc.s;
#pragma unroll
  for (int q = 0; q < kKeep; ++q)
    if (first + q * next < KS) to[(first + q * next) * 64] = quantise16(v[q], sc);
  for (int ks = first + kKeep * next; ks < KS; ks += next) {
    Block<DT> a;
    a.load(p, kStep * ks + 8 * kq, Kr);
    to[ks * 64] = quantise16(a, sc);
  }
}

// Sixteen columns of y from column `col` on, as a lane has them of a group's four tiles: the
// channels' scales and biases, and the store of a row.  Scales are mantissas and exponents: the
// product of two may have no value in fp32 where y has one (large by large with a sum of 0, small by
// small with a large one).  A power of two rounds nothing, so where it has, y's bits are those of sum *
// (s_x * s_w) + bias (8,188 x 9,728 x 896 with x's rows 92 -> 94 us, K = 64 42.8 -> 44.1, others within 2 %).
struct Out {
  const float *ws;
  const void *bias;
  int bias_dtype;
  int N;
};
struct Columns {
  float s[16], b[16];  // mantissas, biases
  int x[16];           // exponents

  __device__ __forceinline__ Columns(const Out &o, int col) {
    typedef float F4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const F4 v = *reinterpret_cast<const F4 *>(o.ws + col + 4 * j);  // (padded to 64)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[4 * j + e] = __builtin_amdgcn_frexp_mantf(v[e]);
        x[4 * j + e] = __builtin_amdgcn_frexp_expf(v[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) b[e] = 0.f;
    if (o.bias) load_bias(o, col);
  }
  __device__ __forceinline__ void load_bias(const Out &o, int col) {
    auto all = [&](auto get) {
#pragma unroll
      for (int e = 0; e < 16; ++e) b[e] = get(min(col + e, o.N - 1));
    };
    if (o.bias_dtype == SPK_F32) all([&](int c) { return static_cast<const float *>(o.bias)[c]; });
    else if (o.bias_dtype == SPK_F16) all([&](int c) { return static_cast<float>(static_cast<const _Float16 *>(o.bias)[c]); });
    else all([&](int c) { return bf16_bits_to_f32(static_cast<const uint16_t *>(o.bias)[c]); });
  }
  template <int OT>
  __device__ __forceinline__ void store(const Out &o, const v4i (&acc)[4], float sx, void *y, int64_t at, int col) const {
    typedef typename Elem<OT>::T E;
    constexpr int W = Elem<OT>::kVec;
    typedef E Some __attribute__((ext_vector_type(W), aligned(sizeof(E))));  // (rows need no alignment)
    typedef float F2 __attribute__((ext_vector_type(2)));
    typedef __bf16 B2 __attribute__((ext_vector_type(2)));
    const float ms = __builtin_amdgcn_frexp_mantf(sx);
    const int xs = __builtin_amdgcn_frexp_expf(sx);
    float f[16];
#pragma unroll
    for (int c = 0; c < 16; ++c)
      f[c] = __builtin_amdgcn_ldexpf(static_cast<float>(acc[c >> 2][c & 3]) * (ms * s[c]), xs + x[c]) + b[c];
    E v[16];
#pragma unroll
    for (int c = 0; c < 16; c += 2) {
      if constexpr (OT == SPK_BF16) {  // (two an instruction)
        const uint32_t two = __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{f[c], f[c + 1]}), B2));
        v[c] = static_cast<E>(two), v[c + 1] = static_cast<E>(two >> 16);
      } else {
        v[c] = f32_to_elem<OT>(f[c]), v[c + 1] = f32_to_elem<OT>(f[c + 1]);
      }
    }
    E *out = static_cast<E *>(y) + at + col;
    if (col + 16 <= o.N) {
#pragma unroll
      for (int h = 0; h < 16 / W; ++h) {
        Some w;
#pragma unroll
        for (int e = 0; e < W; ++e) w[e] = v[W * h + e];
        *reinterpret_cast<Some *>(out + W * h) = w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (col + e < o.N) out[e] = v[e];
    }
  }
};

// ---- few rows -----------------------------------------------------------------------
// A workgroup TM tiles of 16 rows by one group of 64 columns; its eight waves share the steps
// of K, each with its own blocks of both operands from memory, two steps ahead, and their sums
// meet in LDS.  Bound by latency: a wave has few steps (K = 896: two; 333 x 1,001 x 777 5.6 us).
//
// FUSED (at most 16 rows): x is quantised here.  A wave loads the blocks of x that it
// multiplies, the waves exchange the rows' largest magnitudes, and the integers are the
// instruction's operand where they are made; W's first blocks are on their way meanwhile.
// 4 x 1,152 x 896 5.7 us in place of 3.8 and 4.4 in two launches, 16 x 9,728 x 896 5.9 of 4.0 and
// 4.3, 4 x 896 x 4,864 12 of 4.0 and 7.8 (16 rows: 15.6 of 5.8 and 7.8), each with a launch less to
// wait for.  With long rows few columns are few workgroups (14 for 896), which bounds these two.
// Sixteen waves for more than two steps of eight (4 x 896 x 4,864: eight 12.6 where sixteen took 11.4).
constexpr int kSplit = 8;

// Adds up the waves' sums; wave i < TM has row tile i's afterwards.
template <int TM, int WAVES>
__device__ __forceinline__ void join(v4i *sh, const v4i (&acc)[TM][4], v4i (&sum)[4]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sh[((wave * TM + i) * 4 + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  if (wave >= TM) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    sum[j] = sh[(wave * 4 + j) * 64 + lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) sum[j] += sh[((w * TM + wave) * 4 + j) * 64 + lane];
  }
}

template <int TM, int OT>
__global__ __launch_bounds__(64 * kSplit) void split_kernel(const v4i *xq, const float *xs, const v4i *wq, Out o, void *y,
                                                            int64_t ystride, int64_t M, int KS, int64_t MT, int NG) {
  __shared__ v4i sh[kSplit * TM * 4 * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int g = static_cast<int>(blockIdx.x % NG);
  const int64_t m0 = blockIdx.x / NG * TM;
  const v4i *a = wq + static_cast<int64_t>(g) * 4 * KS * 64 + lane, *b[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) b[t] = xq + min(m0 + t, MT - 1) * KS * 64 + lane;
  v4i acc[TM][4], av[2][4], bv[2][TM];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  auto load = [&](int ks, v4i (&av)[4], v4i (&bv)[TM]) {
    const int64_t at = min(ks, KS - 1);  // (steps behind the last are not used)
#pragma unroll
    for (int t = 0; t < 4; ++t) av[t] = a[(t * static_cast<int64_t>(KS) + at) * 64];
#pragma unroll
    for (int t = 0; t < TM; ++t) bv[t] = b[t][at * 64];
  };
  auto products = [&](const v4i (&av)[4], const v4i (&bv)[TM]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[j], bv[i], acc[i][j], 0, 0, 0);
  };
  load(wave, av[0], bv[0]);
  load(wave + kSplit, av[1], bv[1]);
  for (int ks = wave; ks < KS; ks += 2 * kSplit) {
    products(av[0], bv[0]);
    load(ks + 2 * kSplit, av[0], bv[0]);
    if (ks + kSplit >= KS) break;
    products(av[1], bv[1]);
    load(ks + 3 * kSplit, av[1], bv[1]);
  }
  v4i sum[4];
  join<TM, kSplit>(sh, acc, sum);
  const int64_t row = 16 * (m0 + wave) + r16;
  const int col = 64 * g + 16 * kq;
  if (wave < TM && row < M) Columns(o, col).store<OT>(o, sum, xs[row], y, row * ystride, col);
}

// HOLD: blocks of x that a wave holds; those of longer rows are read again.
template <int DT, int WAVES, int HOLD, int OT>
__global__ __launch_bounds__(64 * WAVES) void fused_kernel(const void *x, int64_t stride, const v4i *wq, Out o, void *y,
                                                            int64_t ystride, int M, int K, int KS) {
  __shared__ v4i sh[WAVES * 4 * 64];
  __shared__ uint32_t most[WAVES][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4, g = blockIdx.x;
  const v4i *a = wq + static_cast<int64_t>(g) * 4 * KS * 64 + lane;
  const bool real = r16 < M;
  const char *p = static_cast<const char *>(x) + (real ? r16 : 0) * stride * static_cast<int64_t>(sizeof(typename Elem<DT>::T));
  const int Kr = real ? K : 0;
  v4i av[2][4];
  auto load = [&](int ks, v4i (&av)[4]) {
    const int64_t at = min(ks, KS - 1);
#pragma unroll
    for (int t = 0; t < 4; ++t) av[t] = a[(t * static_cast<int64_t>(KS) + at) * 64];
  };
  Block<DT> v[HOLD];
#pragma unroll
  for (int q = 0; q < HOLD; ++q) v[q].load(p, kStep * (wave + q * WAVES) + 8 * kq, Kr);
  load(wave, av[0]);
  load(wave + WAVES, av[1]);
  uint32_t m = 0;
#pragma unroll
  for (int q = 0; q < HOLD; ++q) m = max(m, v[q].most());
  for (int ks = wave + HOLD * WAVES; ks < KS; ks += WAVES) {
    Block<DT> e;
    e.load(p, kStep * ks + 8 * kq, Kr);
    m = max(m, e.most());
  }
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16)));
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32)));
  if (lane < 16) most[wave][lane] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) m = max(m, most[w][r16]);
  const Scale sc = scale_of(m);
  v4i acc[1][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[0][j] = v4i{0, 0, 0, 0};
  auto products = [&](const v4i (&av)[4], const v4i &b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[0][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[j], b, acc[0][j], 0, 0, 0);
  };
  static_assert(HOLD % 2 == 0, "two buffers of W take turns");
#pragma unroll
  for (int q = 0; q < HOLD; ++q) {
    if (wave + q * WAVES < KS) products(av[q & 1], quantise16(v[q], sc));
    load(wave + (q + 2) * WAVES, av[q & 1]);
  }
  for (int ks = wave + HOLD * WAVES; ks < KS; ks += 2 * WAVES) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (ks + q * WAVES < KS) {
        Block<DT> e;
        e.load(p, kStep * (ks + q * WAVES) + 8 * kq, Kr);
        products(av[q], quantise16(e, sc));
        load(ks + (q + 2) * WAVES, av[q]);
      }
    }
  }
  v4i sum[4];
  join<1, WAVES>(sh, acc, sum);
  const int col = 64 * g + 16 * kq;
  if (wave == 0 && real) Columns(o, col).store<OT>(o, sum, sc.s, y, r16 * ystride, col);
}

// ---- a tile of rows, many columns (the lm_head) -----------------------------------------
// A workgroup's four waves share up to 16 rows of x in LDS, each takes a group of 64 columns
// over the whole K and streams its part of W three steps ahead.  Bound by reading W: 16 x
// 151,936 x 896 24 us with W in the last-level cache and 29 without it (5.9 and 4.9 TB/s; large
// tiles 26 and 31; with more rows in LDS the large tiles are faster: 64 rows 29 and 35 against
// 37 and 43).  Loads that pass the caches by: 26 and 28.
constexpr int kWideWaves = 4;
constexpr int kWideColumns = 512;    // groups of columns from which on
constexpr int kWideLds = 64 * 1024;  // two workgroups a CU
constexpr int kAhead = 3;
template <int OT>
__global__ __launch_bounds__(64 * kWideWaves) void wide_kernel(const v4i *xq, const float *xs, const v4i *wq, Out o, void *y,
                                                               int64_t ystride, int M, int KS, int NG) {
  extern __shared__ v4i shx[];  // [KS][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int g = blockIdx.x * kWideWaves + wave;
  const v4i *a = wq + static_cast<int64_t>(min(g, NG - 1)) * 4 * KS * 64 + lane;
  v4i av[kAhead][4];
  auto load = [&](int ks, v4i (&av)[4]) {
    const int64_t at = min(ks, KS - 1);
#pragma unroll
    for (int t = 0; t < 4; ++t) av[t] = a[(t * static_cast<int64_t>(KS) + at) * 64];
  };
#pragma unroll
  for (int q = 0; q < kAhead; ++q) load(q, av[q]);
  for (int i = threadIdx.x; i < KS * 64; i += 64 * kWideWaves) shx[i] = xq[i];
  __syncthreads();
  if (g >= NG) return;
  v4i acc[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) acc[j] = v4i{0, 0, 0, 0};
  for (int k0 = 0; k0 < KS; k0 += kAhead) {
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (k0 + q < KS) {
        const v4i b = shx[(k0 + q) * 64 + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[q][j], b, acc[j], 0, 0, 0);
        load(k0 + q + kAhead, av[q]);
      }
    }
  }
  const int col = 64 * g + 16 * kq;
  if (r16 < M) Columns(o, col).store<OT>(o, acc, xs[r16], y, r16 * ystride, col);
}

// ---- many rows ----------------------------------------------------------------------
// A workgroup kBM rows by kBN columns, four waves side by side along the columns, 128 x 64
// each (128 accumulator registers); two workgroups a CU, so that one's epilogue runs beside
// the other's products.  The waves share x through LDS (a step's 8 KB, double-buffered, through
// registers so that its loads are two steps ahead); each wave's part of W is its own and
// goes from memory to registers, two steps ahead.  LDS then moves 40 KB a step of 512 cycles
// of products, where both operands through it would take 72.  8,192^3 491 us (2,239 TOP/s), 16,384 x
// 896 x 4,864 69 (2,080), 8,188 x 9,728 x 896 86 (1,650: 14 steps, then 64 KB of stores).
constexpr int kBM = 128, kBN = 256;
constexpr int kTM = kBM / 16, kTN = 4;

template <int OT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void tile_kernel(
    const v4i *xq, const float *xs, const v4i *wq, Out o, void *y, int64_t ystride, int64_t M, int KS, int MT, int NG,
    int mtiles, int ntiles) {
  __shared__ v4i sh[2][kTM * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, kq = lane >> 4;
  // Tiles of one XCD (workgroup b runs on XCD b % 8): a contiguous share of the tiles along
  // the longer side, eight of them at a time against every tile of the other side, so that one
  // operand comes into the XCD's L2 once and the other once for the eight.
  const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
  const bool by_rows = mtiles >= ntiles;
  const int along = by_rows ? mtiles : ntiles, across = by_rows ? ntiles : mtiles;
  const int first = static_cast<int>(static_cast<int64_t>(along) * xcd / 8);
  const int mine = static_cast<int>(static_cast<int64_t>(along) * (xcd + 1) / 8) - first;
  const int group = idx / (8 * across), in = idx - group * 8 * across, some = min(8, mine - 8 * group);
  if (some <= 0 || in >= some * across) return;
  const int u = first + 8 * group + in % some, v = in / some;
  const int mt = by_rows ? u : v, nt = by_rows ? v : u;
  const int m0 = mt * kTM, g = nt * (kBN / 64) + wave;

  // this thread's two 16-byte pieces of a step's x, its wave's four blocks of W
  const v4i *ax[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) ax[p] = xq + static_cast<int64_t>(min(m0 + wave + 4 * p, MT - 1)) * KS * 64 + lane;
  const v4i *bw[kTN];
#pragma unroll
  for (int t = 0; t < kTN; ++t) bw[t] = wq + (4 * static_cast<int64_t>(min(g, NG - 1)) + t) * KS * 64 + lane;

  v4i acc[kTM][kTN];
#pragma unroll
  for (int i = 0; i < kTM; ++i)
#pragma unroll
    for (int j = 0; j < kTN; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  v4i sa[2][2], sb[2][kTN];
  auto load_a = [&](int k, v4i (&r)[2]) {
    const int at = min(k, KS - 1) * 64;  // (steps behind the last are not used)
#pragma unroll
    for (int p = 0; p < 2; ++p) r[p] = ax[p][at];
  };
  auto load_b = [&](int k, v4i (&r)[kTN]) {
    const int at = min(k, KS - 1) * 64;
#pragma unroll
    for (int t = 0; t < kTN; ++t) r[t] = bw[t][at];
  };
  auto put = [&](v4i *to, const v4i (&r)[2]) {
#pragma unroll
    for (int p = 0; p < 2; ++p) to[(wave + 4 * p) * 64 + lane] = r[p];
  };
  load_a(0, sa[0]);
  load_b(0, sb[0]);
  load_a(1, sa[1]);
  load_b(1, sb[1]);
  put(sh[0], sa[0]);
  load_a(2, sa[0]);
  __syncthreads();
  auto step = [&](int k, const v4i *from, v4i *to, v4i (&a)[2], v4i (&b)[kTN]) {
    v4i f[kTM];
#pragma unroll
    for (int i = 0; i < kTM; ++i) f[i] = from[i * 64 + lane];
    put(to, a);
    load_a(k + 3, a);
#pragma unroll
    for (int i = 0; i < kTM; ++i)
#pragma unroll
      for (int j = 0; j < kTN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[j], f[i], acc[i][j], 0, 0, 0);
    load_b(k + 2, b);
    // Half of a step's x is read ahead of its products, the rest between them (and the writes
    // and loads behind): 8,192^3 534 -> 514 us against the compiler's order, two reads ahead.
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);  // LDS reads
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);  // products
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x200, 2, 0);  // LDS writes
    __builtin_amdgcn_sched_group_barrier(0x20, 2, 0);   // loads
    __builtin_amdgcn_sched_group_barrier(0x8, 16, 0);
    __builtin_amdgcn_sched_group_barrier(0x20, 4, 0);
    __syncthreads();
  };
  int k = 0;
  for (; k + 1 < KS; k += 2) {
    step(k, sh[0], sh[1], sa[1], sb[0]);
    step(k + 1, sh[1], sh[0], sa[0], sb[1]);
  }
  if (k < KS) step(k, sh[0], sh[1], sa[1], sb[0]);

  if (g >= NG) return;
  const int col = 64 * g + 16 * kq;
  const Columns cols(o, col);
#pragma unroll
  for (int i = 0; i < kTM; ++i) {
    const int64_t row = 16 * static_cast<int64_t>(m0 + i) + r16;
    if (row < M) cols.store<OT>(o, acc[i], xs[row], y, row * ystride, col);
  }
}

template <int DT>
void launch_rows(const void *x, int64_t stride, int64_t rows, int K, bool weight, void *packed, float *scales,
                 hipStream_t s) {
  const int KS = static_cast<int>(k_steps(K));
  const unsigned tiles = static_cast<unsigned>(weight ? 4 * ((rows + 63) / 64) : row_tiles(rows));
  v4i *to = static_cast<v4i *>(packed);
  if (weight) rows_kernel<DT, true, 16><<<tiles, 64 * row_waves(KS), 0, s>>>(x, stride, rows, K, KS, to, scales);
  else if (tiles > 64) rows_kernel<DT, false, 16><<<tiles, 64 * row_waves(KS), 0, s>>>(x, stride, rows, K, KS, to, scales);
  else rows_kernel<DT, false, 4><<<4 * tiles, 64 * row_waves((KS + 3) / 4), 0, s>>>(x, stride, rows, K, KS, to, scales);
}

void rows(const void *x, int dtype, int64_t stride, int64_t n, int K, bool weight, void *packed, float *scales,
          hipStream_t s) {
  if (dtype == SPK_F32) launch_rows<SPK_F32>(x, stride, n, K, weight, packed, scales, s);
  else if (dtype == SPK_F16) launch_rows<SPK_F16>(x, stride, n, K, weight, packed, scales, s);
  else launch_rows<SPK_BF16>(x, stride, n, K, weight, packed, scales, s);
}

template <int TM, int OT>
void split(const v4i *xq, const float *xs, const v4i *wq, const Out &o, void *y, int64_t ystride, int64_t M, int KS,
           int64_t MT, int NG, hipStream_t s) {
  split_kernel<TM, OT><<<static_cast<unsigned>((MT + TM - 1) / TM * NG), 64 * kSplit, 0, s>>>(xq, xs, wq, o, y, ystride, M,
                                                                                          KS, MT, NG);
}
// The kernel for a size: the least of the times, in us, that fits to measurements give (64 to 2,048
// rows, 512 to 9,728 columns, K = 896 and 4,864; within a fifth, near their borders; other sizes go by
// the same lines, unmeasured).  Measured,
// with one, two, four row tiles a workgroup of the split kernel and with large tiles: 64 x 896 x
// 896 3.6, 4.1, 5.1, 9.1; 256 x 9,728 x 896 16.1, 12.5, 14.0, 12.4; 1,024 x 896 x 4,864 20.5,
// 14.9, 12.9, 32.5; 2,048 x 4,864 x 896 57, 42, 44, 21.  From kWideColumns on large tiles whatever the
// rows: 64 x 33,000 x 896 two row tiles 16, large tiles 12.
enum Way { kSplit1, kSplit2, kSplit4, kTiles };
constexpr double kMostThreads = 4294967295.0;  // of a launch
inline Way way(int64_t M, int N, int KS, int out_bytes) {
  const double ks = KS, ng = groups_of(N), mt = static_cast<double>(row_tiles(M));
  const int64_t tiles = (M + kBM - 1) / kBM * ((N + kBN - 1) / kBN);
  const double t[] = {3.0 + 0.041 * ks + mt * ng * (0.0020 + 0.00025 * ks),
                      3.5 + 0.041 * ks + std::ceil(mt / 2) * ng * (0.0039 + 0.00031 * ks),
                      4.5 + 0.052 * ks + std::ceil(mt / 4) * ng * (0.0108 + 0.00044 * ks),
                      7.0 + 0.33 * ks * static_cast<double>((tiles + 255) / 256) + static_cast<double>(M) * N * out_bytes / 3.7e6};
  return mt * ng * 64 * kSplit > kMostThreads ? kTiles : static_cast<Way>(std::min_element(t, t + 4) - t);
}
// Whether the launches for these sizes have few enough threads.
inline bool launchable(int64_t M, int N, int KS) {
  return static_cast<double>(row_tiles(M)) * 64 * row_waves(KS) <= kMostThreads &&
         (M / kBM + 64.0) * (N / kBN + 64.0) * 256 <= kMostThreads;
}

template <int OT>
void product(const v4i *xq, const float *xs, const v4i *wq, const float *ws, const void *bias, int bias_dtype, void *y,
             int64_t ystride, int64_t M, int N, int KS, hipStream_t s) {
  const int64_t MT = row_tiles(M);
  const int NG = groups_of(N);
  const Out o{ws, bias, bias_dtype, N};
  if (MT <= 1 && NG >= kWideColumns && KS * 1024 <= kWideLds) {
    wide_kernel<OT><<<(NG + kWideWaves - 1) / kWideWaves, 64 * kWideWaves, KS * 1024, s>>>(xq, xs, wq, o, y, ystride,
                                                                                       static_cast<int>(M), KS, NG);
    return;
  }
  switch (NG >= kWideColumns ? kTiles : way(M, N, KS, sizeof(typename Elem<OT>::T))) {
    case kSplit1: split<1, OT>(xq, xs, wq, o, y, ystride, M, KS, MT, NG, s); break;
    case kSplit2: split<2, OT>(xq, xs, wq, o, y, ystride, M, KS, MT, NG, s); break;
    case kSplit4: split<4, OT>(xq, xs, wq, o, y, ystride, M, KS, MT, NG, s); break;
    default: {
      const int64_t mtiles = (M + kBM - 1) / kBM, ntiles = (N + kBN - 1) / kBN;
      const int64_t along = std::max(mtiles, ntiles), across = std::min(mtiles, ntiles);
      const unsigned grid = static_cast<unsigned>(8 * (((along + 7) / 8 + 7) / 8) * 8 * across);
      tile_kernel<OT><<<grid, 256, 0, s>>>(xq, xs, wq, o, y, ystride, M, KS, static_cast<int>(MT), NG, static_cast<int>(mtiles),
                                           static_cast<int>(ntiles));
    }
  }
}

template <int DT, int OT>
void launch_fused(const void *x, int64_t stride, const v4i *wq, const Out &o, void *y, int64_t ystride, int M, int K,
                  hipStream_t s) {
  const int KS = static_cast<int>(k_steps(K)), NG = groups_of(o.N);
  constexpr int kHold = DT == SPK_F32 ? 2 : 6;  // (of what 128 registers hold)
  if (KS <= 2 * kSplit) fused_kernel<DT, kSplit, 2, OT><<<NG, 64 * kSplit, 0, s>>>(x, stride, wq, o, y, ystride, M, K, KS);
  else if (KS <= 2 * 16) fused_kernel<DT, 16, 2, OT><<<NG, 64 * 16, 0, s>>>(x, stride, wq, o, y, ystride, M, K, KS);
  else fused_kernel<DT, 16, kHold, OT><<<NG, 64 * 16, 0, s>>>(x, stride, wq, o, y, ystride, M, K, KS);
}
template <int OT>
void fused(const void *x, int dtype, int64_t stride, const v4i *wq, const float *ws, const void *bias, int bias_dtype,
           void *y, int64_t ystride, int M, int N, int K, hipStream_t s) {
  const Out o{ws, bias, bias_dtype, N};
  if (dtype == SPK_F32) launch_fused<SPK_F32, OT>(x, stride, wq, o, y, ystride, M, K, s);
  else if (dtype == SPK_F16) launch_fused<SPK_F16, OT>(x, stride, wq, o, y, ystride, M, K, s);
  else launch_fused<SPK_BF16, OT>(x, stride, wq, o, y, ystride, M, K, s);
}

}  // namespace i8
}  // namespace spk

using namespace spk;

static int check_sizes(const char *what, int64_t rows, int K) {
  if (rows < 0 || K <= 0) return fail(SPK_EINVAL, "%s: bad sizes rows=%lld K=%d", what, (long long)rows, K);
  if (K > i8::kMaxK || rows > (1ll << 30))
    return fail(SPK_EUNSUPPORTED, "%s: K=%d (at most %d: sums are 32 bits), rows=%lld (at most 2^30)", what, K, i8::kMaxK,
                (long long)rows);
  return SPK_OK;
}

extern "C" size_t spk_linear_int8_packed_bytes(int N, int K) {
  return N > 0 && K > 0 ? static_cast<size_t>(i8::packed_bytes(64ll * i8::groups_of(N), K)) : 0;
}

extern "C" int spk_linear_int8_pack(const void *w, int w_dtype, int64_t w_stride, int N, int K, void *packed,
                                    float *scales, void *stream) {
  if (!valid_float_dtype(w_dtype)) return fail(SPK_EINVAL, "linear_int8_pack: dtype %d is not a float type", w_dtype);
  if (const int rc = check_sizes("linear_int8_pack", N, K)) return rc;
  if (N == 0) return SPK_OK;
  if (!i8::launchable(N, 1, static_cast<int>(i8::k_steps(K))))
    return fail(SPK_EUNSUPPORTED, "linear_int8_pack: more threads than a launch has, N=%d K=%d", N, K);
  if (!w || !packed || !scales) return fail(SPK_EINVAL, "linear_int8_pack: null pointer");
  if (reinterpret_cast<uintptr_t>(packed) & 15) return fail(SPK_EINVAL, "linear_int8_pack: packed must be 16-byte aligned");
  i8::rows(w, w_dtype, w_stride, N, K, true, packed, scales, static_cast<hipStream_t>(stream));
  return check_launch("linear_int8_pack");
}

extern "C" size_t spk_linear_int8_workspace_bytes(int64_t M, int N, int K) {
  return M > 0 && N > 0 && K > 0 ? static_cast<size_t>(i8::packed_bytes(M, K) + i8::scale_bytes(M)) : 0;
}

extern "C" int spk_linear_int8(const void *x, int x_dtype, int64_t x_stride, const void *packed, const float *scales,
                               const void *bias, int bias_dtype, void *y, int y_dtype, int64_t y_stride, int64_t M,
                               int N, int K, void *workspace, size_t workspace_bytes, void *stream) {
  if (!valid_float_dtype(x_dtype) || !valid_float_dtype(y_dtype) || (bias && !valid_float_dtype(bias_dtype)))
    return fail(SPK_EINVAL, "linear_int8: x, y and bias must be of float types");
  if (N <= 0) return fail(SPK_EINVAL, "linear_int8: N=%d", N);
  if (const int rc = check_sizes("linear_int8", M, K)) return rc;
  if (N > (1 << 30)) return fail(SPK_EUNSUPPORTED, "linear_int8: N=%d (at most 2^30)", N);
  if (M > 1 && y_stride < N) return fail(SPK_EINVAL, "linear_int8: rows of y lie on one another");
  if (M == 0) return SPK_OK;
  if (!i8::launchable(M, N, static_cast<int>(i8::k_steps(K))))
    return fail(SPK_EUNSUPPORTED, "linear_int8: more threads than a launch has, M=%lld N=%d K=%d", (long long)M, N, K);
  if (!x || !packed || !scales || !y) return fail(SPK_EINVAL, "linear_int8: null pointer");
  const int64_t yb = y_dtype == SPK_F32 ? 4 : 2, bb = bias_dtype == SPK_F32 ? 4 : 2;
  // (one row in place is fine: a lane writes the columns whose biases it has read)
  if (bias && !(M == 1 && bias == y && bias_dtype == y_dtype) && on_rows(bias, N * bb, y, y_stride * yb, N * yb, M))
    return fail(SPK_EINVAL, "linear_int8: y lies on bias");
  const size_t need = spk_linear_int8_workspace_bytes(M, N, K);
  if (!workspace || workspace_bytes < need)
    return fail(SPK_EINVAL, "linear_int8: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if ((reinterpret_cast<uintptr_t>(packed) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return fail(SPK_EINVAL, "linear_int8: packed and workspace must be 16-byte aligned");
  const int64_t xb = x_dtype == SPK_F32 ? 4 : 2;
  if (on_one_another(x, x_stride * xb, K * xb, y, y_stride * yb, N * yb, M))
    return fail(SPK_EINVAL, "linear_int8: y lies on x");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int KS = static_cast<int>(i8::k_steps(K));
  i8::v4i *xq = static_cast<i8::v4i *>(workspace);
  float *xs = reinterpret_cast<float *>(static_cast<char *>(workspace) + i8::packed_bytes(M, K));
  const i8::v4i *wq = static_cast<const i8::v4i *>(packed);
  if (M <= 16 && i8::groups_of(N) < i8::kWideColumns) {
    if (y_dtype == SPK_F32) i8::fused<SPK_F32>(x, x_dtype, x_stride, wq, scales, bias, bias_dtype, y, y_stride, static_cast<int>(M), N, K, s);
    else if (y_dtype == SPK_F16) i8::fused<SPK_F16>(x, x_dtype, x_stride, wq, scales, bias, bias_dtype, y, y_stride, static_cast<int>(M), N, K, s);
    else i8::fused<SPK_BF16>(x, x_dtype, x_stride, wq, scales, bias, bias_dtype, y, y_stride, static_cast<int>(M), N, K, s);
    return check_launch("linear_int8");
  }
  i8::rows(x, x_dtype, x_stride, M, K, false, xq, xs, s);
  if (y_dtype == SPK_F32) i8::product<SPK_F32>(xq, xs, wq, scales, bias, bias_dtype, y, y_stride, M, N, KS, s);
  else if (y_dtype == SPK_F16) i8::product<SPK_F16>(xq, xs, wq, scales, bias, bias_dtype, y, y_stride, M, N, KS, s);
  else i8::product<SPK_BF16>(xq, xs, wq, scales, bias, bias_dtype, y, y_stride, M, N, KS, s);
  return check_launch("linear_int8");
}
