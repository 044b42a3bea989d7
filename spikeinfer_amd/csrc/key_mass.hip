// Attention weight that the cached tokens of a sequence get from its last rows.
//
// Row i of a sequence's m rows is the token at position len - m + i and sees the
// positions up to its own:
//   mass[n, g, j] (+)= sum over t, query heads h of kv head g, rows i of
//                      exp(popc(q & k_j) * scale) / sum_j' exp(popc(q & k_j') * scale).
// Two launches: the rows' denominators (a wave a row), then a thread a key.
#include "common.hpp"

namespace spk {
namespace mass {

struct Params {
  const uint32_t *q;
  int64_t qs0, qs1, qs2;
  const uint32_t *k;
  int64_t ks0, ks1, ks2;
  int64_t num_slots;
  const int32_t *bt;
  int64_t bts0, bts1;
  const int32_t *lens, *starts;
  float *mass;
  int64_t ms0, ms1, cap;
  int accumulate;
  int64_t rows;
  int N, max_rows, T, Hq, Hkv, nrep, W, bs_log2, max_blocks;
  float scale;
  float *den;  // [T, rows, Hq]
};

struct Seq {
  int64_t s0;
  int m, len;
};

__device__ __forceinline__ Seq sequence(const Params &p, int n) {
  Seq s;
  s.s0 = p.starts ? min<int64_t>(max(p.starts[n], 0), p.rows) : min<int64_t>(n, p.rows);
  const int64_t e = p.starts ? p.starts[n + 1] : n + 1;
  s.m = static_cast<int>(min(min(max(e, s.s0), s.s0 + p.max_rows), p.rows) - s.s0);
  s.len = min(max(p.lens[n], 0), p.max_blocks << p.bs_log2);
  return s;
}

__device__ __forceinline__ int64_t slot_of(const Params &p, int n, int j, uint32_t nblocks) {
  const uint32_t blk = static_cast<uint32_t>(p.bt[n * p.bts0 + (j >> p.bs_log2) * p.bts1]);
  return blk < nblocks ? (static_cast<int64_t>(blk) << p.bs_log2) | (j & ((1 << p.bs_log2) - 1)) : -1;
}

__global__ __launch_bounds__(256) void den_kernel(Params p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.y;
  const int unit = blockIdx.x * 4 + wave;
  const int h = unit % p.Hq, t = unit / p.Hq % p.T, i = unit / p.Hq / p.T;
  const Seq s = sequence(p, n);
  if (i >= s.m) return;
  const uint32_t nblocks = static_cast<uint32_t>(min<int64_t>(p.num_slots >> p.bs_log2, 0xffffffffll));
  const int see = s.len - s.m + i + 1;
  float l = 0.f;
  for (int j = lane; j < see; j += 64) {
    const int64_t slot = slot_of(p, n, j, nblocks);
    int c = 0;
    for (int w = 0; w < p.W; ++w)
      c += __popc(p.q[t * p.qs0 + (s.s0 + i) * p.qs1 + h * p.qs2 + w] &
                  (slot < 0 ? 0u : p.k[t * p.ks0 + h / p.nrep * p.ks1 + slot * p.ks2 + w]));
    l += expf(c * p.scale);
  }
  for (int x = 32; x; x >>= 1) l += __shfl_xor(l, x);
  if (lane == 0) p.den[(t * p.rows + s.s0 + i) * p.Hq + h] = l;
}

__global__ __launch_bounds__(256) void mass_kernel(Params p) {
  const int g = blockIdx.y % p.Hkv, n = blockIdx.y / p.Hkv;
  const int64_t j = blockIdx.x * 256ll + threadIdx.x;
  if (j >= p.cap) return;
  const Seq s = sequence(p, n);
  float *to = p.mass + n * p.ms0 + g * p.ms1 + j;
  if (j >= s.len) {
    if (!p.accumulate) *to = 0.f;
    return;
  }
  const uint32_t nblocks = static_cast<uint32_t>(min<int64_t>(p.num_slots >> p.bs_log2, 0xffffffffll));
  const int64_t slot = slot_of(p, n, static_cast<int>(j), nblocks);
  float sum = 0.f;
  for (int t = 0; t < p.T; ++t)
    for (int i = max(0, static_cast<int>(j) - (s.len - s.m)); i < s.m; ++i)
      for (int h = g * p.nrep; h < (g + 1) * p.nrep; ++h) {
        int c = 0;
        for (int w = 0; w < p.W; ++w)
          c += __popc(p.q[t * p.qs0 + (s.s0 + i) * p.qs1 + h * p.qs2 + w] &
                      (slot < 0 ? 0u : p.k[t * p.ks0 + g * p.ks1 + slot * p.ks2 + w]));
        sum += expf(c * p.scale) / p.den[(t * p.rows + s.s0 + i) * p.Hq + h];
      }
  *to = p.accumulate ? *to + sum : sum;
}

}  // namespace mass
}  // namespace spk

using namespace spk;

extern "C" size_t spk_key_mass_workspace_bytes(int T, int64_t rows, int Hq, int block_size, int max_blocks) {
  return static_cast<size_t>(T) * rows * Hq * 4;
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
  if (N == 0 || cap == 0) return SPK_OK;
  if (static_cast<int64_t>(N) * Hkv > 65535) return fail(SPK_EUNSUPPORTED, "key_mass: %d sequences of %d heads", N, Hkv);
  if ((rows > 0 && !q) || !seq_lens || !mass || (max_blocks > 0 && !block_tables) || (num_slots > 0 && !k_cache))
    return fail(SPK_EINVAL, "key_mass: null pointer");
  const size_t need = spk_key_mass_workspace_bytes(T, rows, Hq, block_size, max_blocks);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SPK_EINVAL, "key_mass: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  mass::Params p{};
  p.q = reinterpret_cast<const uint32_t *>(q);
  p.qs0 = q_strides[0]; p.qs1 = q_strides[1]; p.qs2 = q_strides[2];
  p.k = reinterpret_cast<const uint32_t *>(k_cache);
  p.ks0 = cache_strides[0]; p.ks1 = cache_strides[1]; p.ks2 = cache_strides[2];
  p.num_slots = num_slots;
  p.bt = block_tables; p.bts0 = bt_stride0; p.bts1 = bt_stride1;
  p.lens = seq_lens; p.starts = row_starts;
  p.mass = mass; p.ms0 = mass_strides[0]; p.ms1 = mass_strides[1]; p.cap = cap;
  p.accumulate = accumulate; p.rows = rows; p.N = N; p.max_rows = max_rows;
  p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.nrep = Hq / Hkv; p.W = (head_dim + 31) / 32;
  p.bs_log2 = ilog2(block_size); p.max_blocks = max_blocks; p.scale = scale;
  p.den = static_cast<float *>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows > 0) {
    const int64_t units = static_cast<int64_t>(max_rows) * T * Hq;
    mass::den_kernel<<<dim3((units + 3) / 4, N), 256, 0, s>>>(p);
  }
  mass::mass_kernel<<<dim3((cap + 255) / 256, N * Hkv), 256, 0, s>>>(p);
  return check_launch("key_mass");
}
