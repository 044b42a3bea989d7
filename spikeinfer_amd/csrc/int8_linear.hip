// Linear layer in 8-bit integers: y = x W^T (+ bias) with a scale for every row of x (a
// token) and every row of W (an output channel),
//   s = max |x| / 127,  q = rint(x / s)  (both quotients rounded to fp32),
//   y[m, n] = s_x[m] s_w[n] sum_k q_x[m, k] q_w[n, k] + bias[n].
// The integer sum is exact (127^2 K < 2^31 for K <= 131,072); its product with the scales
// and the bias are fp32, rounded once to y's type.
//
// Operands lie in the order of the matrix instruction (v_mfma_i32_16x16x64_i8): 16 rows by
// 64 k are one block of 1 KB, lane l's 16 bytes row l % 16, k 16 (l / 16) .. + 15, blocks of
// a row tile one behind the other.  W is laid out once (spk_linear_int8_pack), x by the
// call's first kernel, with the same code.
#include "common.hpp"
#include "lif_math.hpp"

namespace spk {
namespace i8 {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;      // k of a block
constexpr int kMaxK = 131072;  // 127^2 kMaxK < 2^31
constexpr int kRowWaves = 4;
constexpr int kKeep = 4;       // blocks a wave keeps between the two passes

inline int64_t row_tiles(int64_t rows) { return (rows + 15) / 16; }
inline int64_t k_steps(int64_t K) { return (K + kStep - 1) / kStep; }
inline int64_t packed_bytes(int64_t rows, int64_t K) { return row_tiles(rows) * k_steps(K) * 1024; }
inline int64_t scale_bytes(int64_t rows) { return row_tiles(rows) * 64; }

// rint(x / s) with the quotient rounded to fp32, in -127..127.  x * (1 / s) is off by less
// than two steps of fp32, so where it lies further than that from a half the rounding is
// the same; only near a half is the quotient itself needed (a division is ten instructions),
// or where 1 / s has no value (inv NaN).
__device__ __forceinline__ int quantise(float x, float s, float inv) {
  const float t = x * inv;
  float r = rintf(t);
  if (!(fabsf(fabsf(t - r) - 0.5f) >= 6.2e-5f)) r = rintf(x / s);  // 4 steps at 127
  return static_cast<int>(fminf(fmaxf(r, -127.f), 127.f));
}

// 16 values of a row from k0 on, zeros behind K.
template <int DT, bool VEC>
__device__ __forceinline__ void load16(const void *row, int k0, int K, float (&v)[16]) {
  typedef typename Elem<DT>::T E;
  constexpr int W = Elem<DT>::kVec;
  typedef E Vec __attribute__((ext_vector_type(W)));
  const E *p = static_cast<const E *>(row) + k0;
  if (VEC && k0 + 16 <= K) {
#pragma unroll
    for (int q = 0; q < 16 / W; ++q) {
      const Vec a = reinterpret_cast<const Vec *>(p)[q];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const E e = a[j];
        v[q * W + j] = elem_to_f32<DT>(e);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = k0 + j < K ? elem_to_f32<DT>(p[j]) : 0.f;
  }
}

// A workgroup 16 rows: their largest magnitudes, then the integers.  Rows that do not exist
// become zeros.  A row that holds an infinity or a NaN has the scale NaN, so that its
// products are NaN as those of the numbers themselves would be.
template <int DT, bool VEC>
__global__ __launch_bounds__(64 * kRowWaves) void rows_kernel(const void *x, int64_t stride, int64_t rows, int K, int KS,
                                                              v4i *packed, float *scales) {
  __shared__ uint32_t most[kRowWaves][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int64_t tile = blockIdx.x, row = 16 * tile + r16;
  const bool real = row < rows;
  const char *p = static_cast<const char *>(x) + row * stride * static_cast<int64_t>(sizeof(typename Elem<DT>::T));
  uint32_t m = 0;
  for (int ks = wave; ks < KS; ks += kRowWaves) {
    if (!real) break;
    float v[16];
    load16<DT, VEC>(p, kStep * ks + 16 * kq, K, v);
#pragma unroll
    for (int j = 0; j < 16; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);  // (a NaN's bits are the largest)
  }
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16)));
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32)));
  if (lane < 16) most[wave][lane] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) m = max(m, most[w][r16]);
  const bool finite = m < 0x7f800000u;
  const float s = finite ? __uint_as_float(m) / 127.f : __uint_as_float(0x7fc00000u);
  if (threadIdx.x < 16) scales[row] = s;
  const bool some = finite && s > 0.f;
  const float inv = s >= 0x1p-100f ? 1.f / s : __uint_as_float(0x7fc00000u);
  for (int ks = wave; ks < KS; ks += kRowWaves) {
    v4i out = {0, 0, 0, 0};
    if (real && some) {
      float v[16];
      load16<DT, VEC>(p, kStep * ks + 16 * kq, K, v);
#pragma unroll
      for (int j = 0; j < 16; ++j) out[j >> 2] |= (quantise(v[j], s, inv) & 255) << 8 * (j & 3);
    }
    packed[(tile * KS + ks) * 64 + lane] = out;
  }
}

// A wave TM x TN tiles of 16 rows (of x) by 16 columns (of y), both operands from memory.
// The weight is the instruction's first operand: a lane then holds four columns side by
// side of one row of y.
template <int TM, int TN, int OT>
__global__ __launch_bounds__(256) void product_kernel(const v4i *xq, const float *xs, const v4i *wq, const float *ws,
                                                      const void *bias, int bias_dtype, void *y, int64_t ystride,
                                                      int64_t M, int N, int KS, int64_t MT, int NT) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int cols = (NT + TN - 1) / TN;
  const int64_t m0 = unit / cols * TM;
  const int n0 = static_cast<int>(unit % cols) * TN;
  if (m0 >= MT) return;
  const v4i *a[TN], *b[TM];
#pragma unroll
  for (int t = 0; t < TN; ++t) a[t] = wq + static_cast<int64_t>(min(n0 + t, NT - 1)) * KS * 64 + lane;
#pragma unroll
  for (int t = 0; t < TM; ++t) b[t] = xq + min(m0 + t, MT - 1) * KS * 64 + lane;
  v4i acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  for (int ks = 0; ks < KS; ++ks) {
    v4i av[TN], bv[TM];
#pragma unroll
    for (int t = 0; t < TN; ++t) av[t] = a[t][ks * 64];
#pragma unroll
    for (int t = 0; t < TM; ++t) bv[t] = b[t][ks * 64];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(av[j], bv[i], acc[i][j], 0, 0, 0);
  }
  typedef typename Elem<OT>::T E;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int64_t row = 16 * (m0 + i) + r16;
    if (row >= M) continue;
    const float sx = xs[row];
    E *out = static_cast<E *>(y) + row * ystride;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int col = 16 * (n0 + j) + 4 * kq;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < N) {
          float v = static_cast<float>(acc[i][j][e]) * (sx * ws[col + e]);
          if (bias) v += load_as_f32(bias, col + e, bias_dtype);
          out[col + e] = f32_to_elem<OT>(v);
        }
    }
  }
}

// ---- many rows ----------------------------------------------------------------------
// A workgroup kBM rows by kBN columns, four waves side by side along the columns, 128 x 64
// each (128 accumulator registers); two workgroups a CU, so that one's epilogue runs beside
// the other's products.  The waves share x through LDS (a step's 8 KB, double-buffered, through
// registers so that its loads are two steps ahead); each wave's part of W is its own and
// goes from memory to registers, two steps ahead.  LDS then moves 40 KB a step of 512 cycles
// of products, where both operands through it would take 72.
constexpr int kBM = 128, kBN = 256;
constexpr int kTM = kBM / 16, kTN = 4;

template <int OT, bool BIAS>
__device__ __forceinline__ void store_tile(const v4i &acc, float sx, const float *ws, const void *bias, int bias_dtype,
                                           typename Elem<OT>::T *out, int col, int N, bool vec) {
  typedef typename Elem<OT>::T E;
  typedef E E4 __attribute__((ext_vector_type(4)));
  typedef float F4 __attribute__((ext_vector_type(4)));
  const F4 s = *reinterpret_cast<const F4 *>(ws + col);  // (padded to 16)
  E4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float f = static_cast<float>(acc[e]) * (sx * s[e]);
    if (BIAS) f += col + e < N ? load_as_f32(bias, col + e, bias_dtype) : 0.f;
    v[e] = f32_to_elem<OT>(f);
  }
  if (vec && col + 4 <= N) {
    *reinterpret_cast<E4 *>(out + col) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < N) out[col + e] = v[e];
  }
}

template <int OT, bool BIAS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void tile_kernel(
    const v4i *xq, const float *xs, const v4i *wq, const float *ws, const void *bias, int bias_dtype, void *y,
    int64_t ystride, int64_t M, int N, int KS, int MT, int NT, int mtiles, int ntiles, bool vec) {
  __shared__ v4i sh[2][kTM * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r16 = lane & 15, kq = lane >> 4;
  // Tiles of one XCD (workgroup b runs on XCD b % 8): a contiguous share of the row tiles, eight
  // of them at a time against every column tile, so that x comes into its L2 once and W
  // once for the eight.
  const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
  const int first = static_cast<int>(static_cast<int64_t>(mtiles) * xcd / 8);
  const int mine = static_cast<int>(static_cast<int64_t>(mtiles) * (xcd + 1) / 8) - first;
  const int group = idx / (8 * ntiles), in = idx - group * 8 * ntiles, rows = min(8, mine - 8 * group);
  if (rows <= 0 || in >= rows * ntiles) return;
  const int mt = first + 8 * group + in % rows, nt = in / rows;
  const int m0 = mt * kTM, n0 = nt * (kBN / 16) + wave * kTN;

  // this thread's two 16-byte pieces of a step's x, its wave's four blocks of W
  const v4i *ax[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) ax[p] = xq + static_cast<int64_t>(min(m0 + wave + 4 * p, MT - 1)) * KS * 64 + lane;
  const v4i *bw[kTN];
#pragma unroll
  for (int t = 0; t < kTN; ++t) bw[t] = wq + static_cast<int64_t>(min(n0 + t, NT - 1)) * KS * 64 + lane;

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
    __syncthreads();
  };
  int k = 0;
  for (; k + 1 < KS; k += 2) {
    step(k, sh[0], sh[1], sa[1], sb[0]);
    step(k + 1, sh[1], sh[0], sa[0], sb[1]);
  }
  if (k < KS) step(k, sh[0], sh[1], sa[1], sb[0]);

  typedef typename Elem<OT>::T E;
#pragma unroll
  for (int i = 0; i < kTM; ++i) {
    const int64_t row = 16 * static_cast<int64_t>(m0 + i) + r16;
    if (row >= M) continue;
    const float sx = xs[row];
    E *out = static_cast<E *>(y) + row * ystride;
#pragma unroll
    for (int j = 0; j < kTN; ++j)
      if (n0 + j < NT) store_tile<OT, BIAS>(acc[i][j], sx, ws, bias, bias_dtype, out, 16 * (n0 + j) + 4 * kq, N, vec);
  }
}

template <int DT>
void launch_rows(const void *x, int64_t stride, int64_t rows, int K, void *packed, float *scales, hipStream_t s) {
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (stride * sizeof(typename Elem<DT>::T)) % 16 == 0;
  const int KS = static_cast<int>(k_steps(K));
  const unsigned grid = static_cast<unsigned>(row_tiles(rows));
  if (vec) rows_kernel<DT, true><<<grid, 64 * kRowWaves, 0, s>>>(x, stride, rows, K, KS, static_cast<v4i *>(packed), scales);
  else rows_kernel<DT, false><<<grid, 64 * kRowWaves, 0, s>>>(x, stride, rows, K, KS, static_cast<v4i *>(packed), scales);
}

void rows(const void *x, int dtype, int64_t stride, int64_t n, int K, void *packed, float *scales, hipStream_t s) {
  if (dtype == SPK_F32) launch_rows<SPK_F32>(x, stride, n, K, packed, scales, s);
  else if (dtype == SPK_F16) launch_rows<SPK_F16>(x, stride, n, K, packed, scales, s);
  else launch_rows<SPK_BF16>(x, stride, n, K, packed, scales, s);
}

template <int OT>
void product(const v4i *xq, const float *xs, const v4i *wq, const float *ws, const void *bias, int bias_dtype, void *y,
             int64_t ystride, int64_t M, int N, int KS, hipStream_t s) {
  const int64_t MT = row_tiles(M);
  const int NT = static_cast<int>(row_tiles(N));
  if (M >= 512 && N >= 256) {
    const int mtiles = static_cast<int>((M + kBM - 1) / kBM), ntiles = (N + kBN - 1) / kBN;
    const int most = (mtiles + 7) / 8;  // row tiles of an XCD
    const unsigned grid = 8u * ((most + 7) / 8) * 8 * ntiles;
    typedef typename Elem<OT>::T E;
    const bool vec = (reinterpret_cast<uintptr_t>(y) % (4 * sizeof(E))) == 0 && ystride % 4 == 0;
    if (bias) tile_kernel<OT, true><<<grid, 256, 0, s>>>(xq, xs, wq, ws, bias, bias_dtype, y, ystride, M, N, KS, static_cast<int>(MT), NT, mtiles, ntiles, vec);
    else tile_kernel<OT, false><<<grid, 256, 0, s>>>(xq, xs, wq, ws, bias, bias_dtype, y, ystride, M, N, KS, static_cast<int>(MT), NT, mtiles, ntiles, vec);
    return;
  }
  constexpr int TM = 4, TN = 4;
  const int64_t units = (MT + TM - 1) / TM * ((NT + TN - 1) / TN);
  product_kernel<TM, TN, OT><<<static_cast<unsigned>((units + 3) / 4), 256, 0, s>>>(xq, xs, wq, ws, bias, bias_dtype, y,
                                                                                  ystride, M, N, KS, MT, NT);
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
  return N > 0 && K > 0 ? static_cast<size_t>(i8::packed_bytes(N, K)) : 0;
}

extern "C" int spk_linear_int8_pack(const void *w, int w_dtype, int64_t w_stride, int N, int K, void *packed,
                                    float *scales, void *stream) {
  if (!valid_float_dtype(w_dtype)) return fail(SPK_EINVAL, "linear_int8_pack: dtype %d is not a float type", w_dtype);
  if (const int rc = check_sizes("linear_int8_pack", N, K)) return rc;
  if (N == 0) return SPK_OK;
  if (!w || !packed || !scales) return fail(SPK_EINVAL, "linear_int8_pack: null pointer");
  if (reinterpret_cast<uintptr_t>(packed) & 15) return fail(SPK_EINVAL, "linear_int8_pack: packed must be 16-byte aligned");
  i8::rows(w, w_dtype, w_stride, N, K, packed, scales, static_cast<hipStream_t>(stream));
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
  if (M > 1 && y_stride < N) return fail(SPK_EINVAL, "linear_int8: rows of y lie on one another");
  if (M == 0) return SPK_OK;
  if (!x || !packed || !scales || !y) return fail(SPK_EINVAL, "linear_int8: null pointer");
  const size_t need = spk_linear_int8_workspace_bytes(M, N, K);
  if (!workspace || workspace_bytes < need)
    return fail(SPK_EINVAL, "linear_int8: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
  if ((reinterpret_cast<uintptr_t>(packed) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return fail(SPK_EINVAL, "linear_int8: packed and workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int KS = static_cast<int>(i8::k_steps(K));
  i8::v4i *xq = static_cast<i8::v4i *>(workspace);
  float *xs = reinterpret_cast<float *>(static_cast<char *>(workspace) + i8::packed_bytes(M, K));
  i8::rows(x, x_dtype, x_stride, M, K, xq, xs, s);
  const i8::v4i *wq = static_cast<const i8::v4i *>(packed);
  if (y_dtype == SPK_F32) i8::product<SPK_F32>(xq, xs, wq, scales, bias, bias_dtype, y, y_stride, M, N, KS, s);
  else if (y_dtype == SPK_F16) i8::product<SPK_F16>(xq, xs, wq, scales, bias, bias_dtype, y, y_stride, M, N, KS, s);
  else i8::product<SPK_BF16>(xq, xs, wq, scales, bias, bias_dtype, y, y_stride, M, N, KS, s);
  return check_launch("linear_int8");
}
