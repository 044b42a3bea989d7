// Trees of drafted tokens: ancestor masks, and the accepted path of a verified tree
// with its words moved from the step's buffers into the paged caches.
//
// A tree's rows are numbered with every parent before its children; row 0 is the
// sequence's last token, the rest hang below it.  Both walks follow that order (a
// parent's number is lower, a child's higher), so they end whatever the numbers are.
#include "common.hpp"
#include "draft_rows.hpp"

namespace spk {
namespace draft {

constexpr int kMaxLayers = 64;  // layers a launch (kernel arguments)
constexpr int kThreads = 256;

// A thread a (row, mask word): it follows the row's parents and keeps the bits of its
// word.  Latency only: depth dependent loads, from the L2 after the first.
__global__ __launch_bounds__(kThreads) void tree_masks_kernel(const int32_t *parents, const int32_t *starts,
                                                              int64_t rows, int N, int max_nodes, uint64_t *masks,
                                                              int words, int32_t *depths) {
  const int64_t id = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x;
  const int64_t row = id / words;
  const int word = static_cast<int>(id - row * words);
  if (row >= rows) return;
  int lo = 0, hi = N;  // the last sequence that starts at or before the row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  const Rows r = rows_of(starts, lo, rows, max_nodes);
  int at = static_cast<int>(row - r.first);
  if (row < r.first || at >= r.count) return;  // no sequence's: left as it was
  uint64_t bits = 0;
  int depth = 0;
  for (;;) {
    if (at >> 6 == word) bits |= 1ull << (at & 63);
    const int up = parents[r.first + at];
    if (up < 0 || up >= at) break;
    at = up;
    ++depth;
  }
  masks[row * words + word] = bits;
  if (word == 0) depths[row] = depth;
}

struct Layer {
  const uint32_t *kn, *vn;  // the step's words (t, row, kv head)
  uint32_t *k, *v;          // the caches (t, kv head, slot)
};

struct Params {
  const int64_t *tokens, *targets;
  const int32_t *parents, *starts;
  int64_t rows;
  int max_nodes;
  int32_t *path, *count;
  int64_t *next;
  int64_t ns0, ns1, ns2;  // strides of the step's words
  int64_t ks0, ks1, ks2;  // of the caches
  int64_t num_slots;
  const int32_t *bt;
  int64_t bts0, bts1;
  const int32_t *lens;
  int T, Hkv, W, bs_log2, max_blocks;
  int first;  // this launch writes path, count and next
  Layer layer[kMaxLayers];
};

// Workgroup (n, layer): its first wave walks tree n, a step a round of 64 candidate
// children, while the others look how many tokens behind the context have a place in the
// cache (a path ends there); then the threads move the path's words of the layer.  Every layer's
// workgroup walks again: the walk takes a few hundred ns a step from LDS, a second
// launch would take more.  Latency only: 24 layers of one tree of 8 rows take 4.1 us, of 64
// trees of 61 rows 7.3.
__global__ __launch_bounds__(kThreads) void accept_kernel(Params p) {
  __shared__ int64_t tok[kMaxNodes], tgt[kMaxNodes];
  __shared__ int32_t par[kMaxNodes], path[kMaxNodes];
  __shared__ int depth, room;
  const int tid = threadIdx.x, lane = tid & 63, n = blockIdx.x;
  const Rows r = rows_of(p.starts, n, p.rows, p.max_nodes);
  for (int i = tid; i < r.count; i += kThreads) {
    tok[i] = p.tokens[r.first + i];
    tgt[i] = p.targets[r.first + i];
    par[i] = p.parents[r.first + i];
  }
  const Layer layer = p.layer[blockIdx.y];
  const int64_t blocks = p.num_slots >> p.bs_log2, ctx = layer.k ? max(p.lens[n], 0) : 0;
  auto slot = [&](int step) -> int64_t {  // of a step's token, below 0: none
    const int64_t pos = ctx + step, blk = pos >> p.bs_log2;
    if (blk >= p.max_blocks) return -1;
    const int64_t phys = p.bt[n * p.bts0 + blk * p.bts1];
    return phys < 0 || phys >= blocks ? -1 : phys << p.bs_log2 | (pos & ((1 << p.bs_log2) - 1));
  };
  if (tid == 0) room = r.count;
  __syncthreads();
  if (tid >= 64) {
    for (int i = tid - 64; layer.k && i < r.count; i += kThreads - 64)
      if (slot(i) < 0) atomicMin(&room, i);
  } else {
    int at = 0, len = r.count > 0 ? 1 : 0;
    if (lane == 0) path[0] = 0;
    while (at < r.count) {
      const int64_t want = tgt[at];
      int found = -1;
      for (int i0 = at + 1; i0 < r.count; i0 += 64) {
        const int i = i0 + lane;
        const uint64_t hits = __ballot(i < r.count && par[i] == at && tok[i] == want);
        if (hits) {
          found = i0 + __builtin_ctzll(hits);
          break;
        }
      }
      if (found < 0) break;
      at = found;
      if (lane == 0) path[len] = at;
      ++len;
    }
    if (lane == 0) depth = len;
  }
  __syncthreads();
  const int len = min(depth, room);
  if (p.first && blockIdx.y == 0) {
    for (int i = tid; i < p.max_nodes; i += kThreads) p.path[n * static_cast<int64_t>(p.max_nodes) + i] = i < len ? path[i] : -1;
    if (tid == 0) {
      p.count[n] = len;
      p.next[n] = len ? tgt[path[len - 1]] : -1;
    }
  }
  if (!layer.k) return;
  const int units = p.T * p.Hkv * p.W;  // words of a token
  for (int i = tid; i < len * units; i += kThreads) {
    const int step = i / units, u = i - step * units;
    const int w = u % p.W, h = u / p.W % p.Hkv, t = u / p.W / p.Hkv;
    const int64_t to = t * p.ks0 + h * p.ks1 + slot(step) * p.ks2 + w;
    const int64_t from = t * p.ns0 + (r.first + path[step]) * p.ns1 + h * p.ns2 + w;
    layer.k[to] = layer.kn[from];
    layer.v[to] = layer.vn[from];
  }
}

}  // namespace draft
}  // namespace spk

using namespace spk;

extern "C" int spk_tree_masks(const int32_t *parents, const int32_t *row_starts, int64_t rows, int N, int max_nodes,
                              int64_t *masks, int mask_words, int32_t *depths, void *stream) {
  if (rows < 0 || N < 0 || max_nodes <= 0 || mask_words < (max_nodes + 63) / 64)
    return fail(SPK_EINVAL, "tree_masks: bad sizes rows=%lld N=%d max_nodes=%d words=%d", (long long)rows, N, max_nodes,
                mask_words);
  if (rows == 0 || N == 0) return SPK_OK;
  const int64_t grid = (rows * mask_words + draft::kThreads - 1) / draft::kThreads;
  if (rows > (1 << 30) || grid > 0x7fffffff) return fail(SPK_EUNSUPPORTED, "tree_masks: %lld rows", (long long)rows);
  if (!parents || !row_starts || !masks || !depths) return fail(SPK_EINVAL, "tree_masks: null pointer");
  draft::tree_masks_kernel<<<grid, draft::kThreads, 0, static_cast<hipStream_t>(stream)>>>(
      parents, row_starts, rows, N, max_nodes, reinterpret_cast<uint64_t *>(masks), mask_words, depths);
  return check_launch("tree_masks");
}

extern "C" int spk_accept_tree(const int64_t *tokens, const int32_t *parents, const int64_t *targets,
                               const int32_t *row_starts, int64_t rows, int N, int max_nodes, int32_t *path,
                               int32_t *count, int64_t *next_tokens, const SpkCommitLayer *layers, int nlayers,
                               const int64_t new_strides[3], const int64_t cache_strides[3], int64_t num_slots,
                               const int32_t *block_tables, int64_t bt_stride0, int64_t bt_stride1,
                               const int32_t *context_lens, int T, int Hkv, int head_dim, int block_size,
                               int max_blocks, void *stream) {
  if (rows < 0 || N < 0 || max_nodes <= 0 || nlayers < 0)
    return fail(SPK_EINVAL, "accept_tree: bad sizes rows=%lld N=%d max_nodes=%d layers=%d", (long long)rows, N,
                max_nodes, nlayers);
  if (max_nodes > draft::kMaxNodes)
    return fail(SPK_EUNSUPPORTED, "accept_tree: max_nodes=%d (at most %d)", max_nodes, draft::kMaxNodes);
  if (nlayers > 0) {
    if (T <= 0 || Hkv <= 0 || head_dim <= 0 || max_blocks < 0 || num_slots < 0)
      return fail(SPK_EINVAL, "accept_tree: bad cache sizes T=%d Hkv=%d D=%d", T, Hkv, head_dim);
    if (head_dim > 512 || static_cast<int64_t>(T) * Hkv > (1 << 16))
      return fail(SPK_EUNSUPPORTED, "accept_tree: T=%d Hkv=%d D=%d", T, Hkv, head_dim);
    if (!is_pow2(block_size)) return fail(SPK_EINVAL, "accept_tree: block_size=%d is not a power of two", block_size);
  }
  if (N == 0) return SPK_OK;
  if (!row_starts || !path || !count || !next_tokens || (rows > 0 && (!tokens || !parents || !targets)))
    return fail(SPK_EINVAL, "accept_tree: null pointer");
  if (nlayers > 0 && (!layers || !context_lens || (max_blocks > 0 && !block_tables)))
    return fail(SPK_EINVAL, "accept_tree: null pointer");
  for (int i = 0; i < nlayers; ++i)
    if (!layers[i].k_cache || !layers[i].v_cache || (rows > 0 && (!layers[i].k_new || !layers[i].v_new)))
      return fail(SPK_EINVAL, "accept_tree: null pointer in layer %d", i);
  if (nlayers > 0 && ((T > 1 && !cache_strides[0]) || (Hkv > 1 && !cache_strides[1]) || (num_slots > 1 && !cache_strides[2])))
    return fail(SPK_EINVAL, "accept_tree: words of a cache lie on one another");
  const int twice = shared_cache(nlayers, [&](int i) { return std::make_pair(layers[i].k_cache, layers[i].v_cache); });
  if (twice >= 0) return fail(SPK_EINVAL, "accept_tree: layer %d has one cache twice, or another layer's", twice);
  draft::Params p{};
  p.tokens = tokens; p.targets = targets; p.parents = parents; p.starts = row_starts;
  p.rows = rows; p.max_nodes = max_nodes; p.path = path; p.count = count; p.next = next_tokens;
  p.num_slots = num_slots;
  p.bt = block_tables; p.bts0 = bt_stride0; p.bts1 = bt_stride1; p.lens = context_lens;
  if (nlayers > 0) {
    p.ns0 = new_strides[0]; p.ns1 = new_strides[1]; p.ns2 = new_strides[2];
    p.ks0 = cache_strides[0]; p.ks1 = cache_strides[1]; p.ks2 = cache_strides[2];
    p.T = T; p.Hkv = Hkv; p.W = (head_dim + 31) / 32; p.bs_log2 = ilog2(block_size); p.max_blocks = max_blocks;
  }
  int i = 0;
  do {
    const int m = nlayers - i < draft::kMaxLayers ? nlayers - i : draft::kMaxLayers;
    for (int k = 0; k < m; ++k)
      p.layer[k] = draft::Layer{reinterpret_cast<const uint32_t *>(layers[i + k].k_new),
                                reinterpret_cast<const uint32_t *>(layers[i + k].v_new),
                                reinterpret_cast<uint32_t *>(layers[i + k].k_cache),
                                reinterpret_cast<uint32_t *>(layers[i + k].v_cache)};
    if (m == 0) p.layer[0] = draft::Layer{};
    p.first = i == 0;
    draft::accept_kernel<<<dim3(N, m > 0 ? m : 1), draft::kThreads, 0, static_cast<hipStream_t>(stream)>>>(p);
    const int rc = check_launch("accept_tree");
    if (rc) return rc;
    i += m;
  } while (i < nlayers);
  return SPK_OK;
}
