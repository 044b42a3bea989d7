// Attention of drafted token trees over the paged packed cache (head_dim <= 128).
//
// Row r of a sequence (a drafted token) attends, per timestep and query head, to
// the sequence's cached context and to the drafted tokens that its mask names:
//   out = sum_j w_j bits(v_j) / sum_j w_j,  w_j = exp(-popc(q & ~k_j) * scale).
// One wave a (row, timestep, query head): a lane weighs a key, then the wave adds
// the 64 weights to its channels (a lane a channel, two past 64).
#include "common.hpp"

namespace spk {
namespace tree {

struct Params {
  const uint32_t *q;
  int64_t qs0, qs1, qs2;
  const uint32_t *kt, *vt;  // drafted tokens' words (t, row, kv head), the same strides
  int64_t ts0, ts1, ts2;
  const uint32_t *k, *v;    // caches (t, kv head, slot), the same strides
  int64_t ks0, ks1, ks2;
  int64_t num_slots;
  const int32_t *bt;
  int64_t bts0, bts1;
  const int32_t *lens, *starts;
  const uint64_t *masks;
  int mask_words;
  void *out;
  int64_t os0, os1, os2;
  int out_dtype;
  int64_t rows;
  int N, max_nodes, T, Hq, nrep, D, W, bs_log2, max_blocks;
  float scale;
};

__global__ __launch_bounds__(256) void tree_attn_kernel(Params p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int unit = blockIdx.x * 4 + wave;
  const int n = blockIdx.y;
  const int h = unit % p.Hq, t = unit / p.Hq % p.T, node = unit / p.Hq / p.T;
  const int64_t s0 = min<int64_t>(max(p.starts[n], 0), p.rows);
  const int64_t s1 = min<int64_t>(min<int64_t>(max<int64_t>(p.starts[n + 1], s0), s0 + p.max_nodes), p.rows);
  const int nodes = static_cast<int>(s1 - s0);
  if (node >= nodes) return;
  const int ctx = min(max(p.lens[n], 0), p.max_blocks << p.bs_log2);
  const int64_t row = s0 + node;
  const int g = h / p.nrep;
  uint32_t qw[4];
  for (int w = 0; w < 4; ++w) qw[w] = w < p.W ? p.q[t * p.qs0 + row * p.qs1 + h * p.qs2 + w] : 0u;
  const uint32_t nblocks = static_cast<uint32_t>(min<int64_t>(p.num_slots >> p.bs_log2, 0xffffffffll));
  const int bs_mask = (1 << p.bs_log2) - 1;
  float acc[2] = {0.f, 0.f}, l = 0.f;
  const int ctx64 = (ctx + 63) & ~63;
  for (int j0 = 0; j0 < ctx64 + nodes; j0 += 64) {
    const int j = j0 + lane;
    bool see;
    uint32_t kw[4] = {}, vw[4] = {};
    if (j0 < ctx64) {
      see = j < ctx;
      if (see) {
        const uint32_t blk = static_cast<uint32_t>(p.bt[n * p.bts0 + (j >> p.bs_log2) * p.bts1]);
        if (blk < nblocks) {
          const int64_t at = t * p.ks0 + g * p.ks1 + ((static_cast<int64_t>(blk) << p.bs_log2) | (j & bs_mask)) * p.ks2;
          for (int w = 0; w < p.W; ++w) kw[w] = p.k[at + w], vw[w] = p.v[at + w];
        }
      }
    } else {
      const int i = j - ctx64;
      see = i < nodes && ((p.masks[row * p.mask_words + (i >> 6)] >> (i & 63)) & 1);
      if (see) {
        const int64_t at = t * p.ts0 + (s0 + i) * p.ts1 + g * p.ts2;
        for (int w = 0; w < p.W; ++w) kw[w] = p.kt[at + w], vw[w] = p.vt[at + w];
      }
    }
    int d = 0;
    for (int w = 0; w < 4; ++w) d += __popc(qw[w] & ~kw[w]);
    const float wt = see ? expf(-d * p.scale) : 0.f;
    l += wt;
    float part[2] = {0.f, 0.f};
    for (int k = 0; k < 64; ++k) {
      const float x = __shfl(wt, k);
      for (int c = 0; c < 2; ++c) {
        const uint32_t lo = __shfl(vw[2 * c], k), hi = __shfl(vw[2 * c + 1], k);
        part[c] += ((lane < 32 ? lo : hi) >> (lane & 31)) & 1 ? x : 0.f;
      }
    }
    acc[0] += part[0];
    acc[1] += part[1];
  }
  for (int s = 32; s; s >>= 1) l += __shfl_xor(l, s);
  const float inv = l > 0.f ? 1.f / l : 0.f;
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < p.D)
      store_f32_as(p.out, t * p.os0 + row * p.os1 + h * p.os2 + lane + 64 * c, p.out_dtype, acc[c] * inv);
}

}  // namespace tree
}  // namespace spk

using namespace spk;

extern "C" size_t spk_tree_attn_workspace_bytes(int T, int N, int Hq, int Hkv, int head_dim, int max_nodes,
                                                int block_size, int max_blocks) {
  return 0;
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
  if (max_nodes > 1024) return fail(SPK_EUNSUPPORTED, "tree_attn: max_nodes=%d (at most 1024)", max_nodes);
  if (!valid_float_dtype(out_dtype)) return fail(SPK_EINVAL, "tree_attn: out dtype %d not a float type", out_dtype);
  if (!is_pow2(block_size)) return fail(SPK_EINVAL, "tree_attn: block_size=%d is not a power of two", block_size);
  if (mask_words < (max_nodes + 63) / 64)
    return fail(SPK_EINVAL, "tree_attn: %d mask words hold fewer than %d nodes", mask_words, max_nodes);
  if (!(scale > 0.f) || scale * head_dim > 12.f)
    return fail(SPK_EINVAL, "tree_attn: scale=%g outside (0, 12/head_dim]", (double)scale);
  if (static_cast<int64_t>(max_blocks) * block_size > (1 << 30))
    return fail(SPK_EUNSUPPORTED, "tree_attn: block tables of %d x %d tokens (at most 2^30)", max_blocks, block_size);
  if (N == 0 || rows == 0) return SPK_OK;
  if (N > 65535) return fail(SPK_EUNSUPPORTED, "tree_attn: %d sequences (at most 65535)", N);
  if (!q || !k_tree || !v_tree || !context_lens || !row_starts || !masks || !out ||
      (max_blocks > 0 && !block_tables) || (num_slots > 0 && (!k_cache || !v_cache)))
    return fail(SPK_EINVAL, "tree_attn: null pointer");
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
  p.bt = block_tables; p.bts0 = bt_stride0; p.bts1 = bt_stride1;
  p.lens = context_lens; p.starts = row_starts;
  p.masks = reinterpret_cast<const uint64_t *>(masks); p.mask_words = mask_words;
  p.out = out; p.out_dtype = out_dtype;
  p.os0 = out_strides[0]; p.os1 = out_strides[1]; p.os2 = out_strides[2];
  p.rows = rows; p.N = N; p.max_nodes = max_nodes; p.T = T; p.Hq = Hq; p.nrep = Hq / Hkv;
  p.D = head_dim; p.W = (head_dim + 31) / 32; p.bs_log2 = ilog2(block_size); p.max_blocks = max_blocks;
  p.scale = scale;
  const int64_t units = static_cast<int64_t>(max_nodes) * T * Hq;
  tree::tree_attn_kernel<<<dim3((units + 3) / 4, N), 256, 0, static_cast<hipStream_t>(stream)>>>(p);
  return check_launch("tree_attn");
}
