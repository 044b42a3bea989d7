// Verification of drafted tokens by given random numbers: which drafted tokens stay, so
// that the tokens that come out are distributed as the target's own samples.
//
// At a row with the target's distribution p and the drafter's q its children are tested in
// order, those drawn from q.  With w = max(p - A q, 0) and c its sum (A = 0, c = 1 at first) the
// child's token x stays if u q(x) c < w(x); if not, A grows by c and the next child is tested
// against what is left.  (Clipping once is the same as after every child: the maximum of
// max(p - a, 0) - b and 0 is that of p - (a + b) and 0.)  Children drawn without replacement
// come from q without the tokens before them, so their c is divided by what those leave; a
// token that did not stay has w = 0 afterwards either way.  Where no child stays, the token
// is the first whose cumulative w exceeds u (row 0's) times the sum.
//
// A test needs two numbers, all trees' of which are loaded at once before the walk; a rejection
// needs the sum over the vocabulary, two rows of it.  These passes are split over workgroups:
// launch r follows each tree up to its r-th sum (the sums before it are there, so every
// workgroup repeats the walk, in LDS), and its slices add up their share.  The last launch,
// one workgroup a tree, follows the walk to its end, sums by itself where a tree needs more, and
// draws.  Many trees are bound by reading the rows (64 chains of up to 8 nodes at 151,936 tokens:
// slices 14.6 us, 5.3 TB/s, the last launch 11), few by latency (one chain 6.3 and 8.4).  Sums and tests are fp64: a decision
// differs from exact arithmetic's only where the numbers are equal to 15 digits.
#include <algorithm>

#include "common.hpp"
#include "draft_rows.hpp"

namespace spk {
namespace verify {

using draft::kMaxNodes;
constexpr int kSliceThreads = 256;
constexpr int kEndThreads = 1024;
constexpr int kMaxSlices = 64;  // a lane each
constexpr int kMaxRounds = 4;

// Launches of slices.  A chain needs one sum, a tree one a rejected sibling, a few as a rule.
// Those that are left to the last launch take one workgroup: 5 to 10 us each at 151,936 tokens,
// 2 at 32,000; a launch that finds every tree done takes 2 to 3.  One launch against four, us (medians
// of five draws, in brackets the slowest), of 5, 8, 9, 12, 16 and 25 nodes alike:
//   151,936 tokens: one chain 14 and 19; one tree with up to 3 siblings 14 (32) and 19 (32); 16 chains
//   16-18 and 20-22, 16 trees 52-55 (73) and 34-37 (46); 64 chains 26-27 and 31-32, 64 trees 57-58
//   (72) and 47-49 (61).
//   32,000 tokens: one chain 14 and 19; 16 chains 15-16 and 20-21, 16 trees 26-27 (38) and 32-35 (48).
// So siblings decide, and only over large vocabularies and in batches.  The host knows nodes alone:
// above 8 it takes trees for granted.  Where that is wrong, batches of smaller trees lose 9 to 18 us,
// longer chains and single trees 5.  Three, four and five launches over 25 draws of 16 trees of 25
// nodes: 39.1, 37.8, 40.5, the slowest 59, 48, 51.
inline int rounds_for(int max_nodes, int V) { return max_nodes > 8 && V >= 65536 ? kMaxRounds : 1; }

struct Params {
  const int64_t *tokens;
  const int32_t *parents, *starts;
  const float *p, *q, *u;
  int64_t ps, qs;  // row strides
  int64_t rows;
  int max_nodes, V, distinct, G, round;
  double *part;   // [round][tree][slice]
  int32_t *done;  // [tree]: the launch behind which its sums are complete (kMaxRounds: not known yet)
  int64_t *out;
};

struct Shared {
  int64_t tok[kMaxNodes], target[kMaxNodes];
  int32_t par[kMaxNodes];
  float u[kMaxNodes], p[kMaxNodes], q[kMaxNodes];  // p and q of each row's token after its parent
  uint8_t stays[kMaxNodes];  // whether it does as its parent's first child
  double part[kMaxSlices], wave[kEndThreads / 64];
  double A;  // the walk's, for the waves that do not follow it
  int at, draw;
  int found, last, token;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
// The sum of the slices' sums, in one order.
__device__ __forceinline__ double total_of(const double *part, int G) {
  const int lane = threadIdx.x & 63;
  return wave_sum(lane < G ? part[lane] : 0.0);
}

// A tree's walk.  The first wave follows it (sixteen would get in each other's way: 0.35 us
// a row against 0.1), the others get the row and A.
struct Walk {
  const Params &P;
  Shared &sh;
  draft::Rows r;
  int at, next;
  double A, mass, before;  // before: what q gives to the children tested so far

  __device__ __forceinline__ const float *prow() const { return P.p + (r.first + at) * P.ps; }
  __device__ __forceinline__ const float *qrow() const { return P.q + (r.first + at) * P.qs; }

  // What c is, divided by what q leaves to a token with qx.
  __device__ __forceinline__ double scaled(double c, double qx) const {
    if (P.distinct) {
      const double left = fmax(1.0 - before, qx);
      if (left > 0.0) c /= left;
    }
    return c;
  }
  __device__ __forceinline__ bool test(double u, double px, double qx, double c) const {
    return u * qx * c < fmax(px - A * qx, 0.0);
  }
  __device__ __forceinline__ void load() {
    go(0);
    for (int i = threadIdx.x; i < r.count; i += blockDim.x) {
      const int64_t x = P.tokens[r.first + i];
      const int up = P.parents[r.first + i];
      const bool child = up >= 0 && up < i && x >= 0 && x < P.V;
      const float u = P.u[r.first + i];
      const float px = child ? P.p[(r.first + up) * P.ps + x] : 0.f;
      const float qx = child ? P.q[(r.first + up) * P.qs + x] : 0.f;
      sh.tok[i] = x;
      sh.par[i] = up;
      sh.u[i] = u;
      sh.p[i] = px;
      sh.q[i] = qx;
      sh.stays[i] = test(u, px, qx, scaled(1.0, qx));
      sh.target[i] = -1;
    }
  }
  __device__ __forceinline__ void go(int row) {
    at = row;
    next = row + 1;
    A = before = 0.0;
    mass = 1.0;
  }
  // The lowest-numbered child of `at` from row `from` on that `ok` takes, or -1.
  template <class Ok>
  __device__ __forceinline__ int child(int from, Ok ok) const {
    const int lane = threadIdx.x & 63;
    for (int i0 = from; i0 < r.count; i0 += 64) {
      const int i = i0 + lane;
      const uint64_t hits = __ballot(i < r.count && sh.par[min(i, kMaxNodes - 1)] == at && ok(i));
      if (hits) return i0 + __builtin_ctzll(hits);
    }
    return -1;
  }
  // tests() for the workgroup.
  __device__ __forceinline__ bool follow() {
    __syncthreads();  // (what the last one wrote is read)
    if (threadIdx.x < 64) {
      const bool draw = tests();
      if (threadIdx.x == 0) sh.at = at, sh.A = A, sh.draw = draw;
    }
    __syncthreads();
    at = sh.at;
    A = sh.A;
    return sh.draw;
  }
  // Tests children until a sum over the vocabulary is needed, for the next test or (true) for
  // the draw.
  __device__ __forceinline__ bool tests() {
    for (;;) {
      const int i = child(next, [](int) { return true; });
      if (i < 0) return true;
      if (A == 0.0 && sh.stays[i]) {  // (a path is mostly first children)
        if (threadIdx.x == 0) sh.target[at] = sh.tok[i];
        go(i);
        continue;
      }
      const double px = sh.p[i], qx = sh.q[i], c = scaled(mass, qx);
      if (A != 0.0 && test(sh.u[i], px, qx, c)) {
        if (threadIdx.x == 0) sh.target[at] = sh.tok[i];
        go(i);
        continue;
      }
      A += c;
      before += qx;
      next = i + 1;
      return false;
    }
  }
  __device__ __forceinline__ int begin(int slice) const {
    return static_cast<int>(static_cast<int64_t>(P.V) * slice / P.G);
  }
  // Weights of the tokens x .. x + 3 that lie below `end`, 0 for the others.
  __device__ __forceinline__ void weights(const float *p, const float *q, int x, int end, double (&w)[4]) const {
    typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
    F4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    if (x + 4 <= end) {
      a = *reinterpret_cast<const F4 *>(p + x);
      if (A != 0.0) b = *reinterpret_cast<const F4 *>(q + x);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x + j < end) {
          a[j] = p[x + j];
          if (A != 0.0) b[j] = q[x + j];
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {  // (a NaN has none; A may be infinite)
      const double v = a[j];
      w[j] = fmax(A == 0.0 ? v : v - A * static_cast<double>(b[j]), 0.0);
    }
  }
  // This thread's share of a slice's sum, `threads` of them from number `me` on.
  __device__ __forceinline__ double share(int slice, int me, int threads) const {
    const float *p = prow(), *q = qrow();
    const int end = begin(slice + 1);
    double s = 0.0;
#pragma unroll 4
    for (int x = begin(slice) + 4 * me; x < end; x += 4 * threads) {
      double w[4];
      weights(p, q, x, end, w);
      s += (w[0] + w[1]) + (w[2] + w[3]);
    }
    return s;
  }
};

__global__ __launch_bounds__(kSliceThreads) void slice_kernel(Params P) {
  __shared__ Shared sh;
  const int n = blockIdx.y, tid = threadIdx.x, N = gridDim.y;
  if (P.round > 0 && P.done[n] < P.round) return;
  Walk w{P, sh, draft::rows_of(P.starts, n, P.rows, P.max_nodes)};
  if (w.r.count == 0) {
    if (tid == 0 && blockIdx.x == 0) P.done[n] = -1;
    return;
  }
  w.load();
  __syncthreads();
  // (a tree whose sums are complete did not get here: the k sums before were not its last)
  bool draw = w.follow();
  for (int k = 0; k < P.round; ++k) {
    w.mass = total_of(P.part + (static_cast<int64_t>(k) * N + n) * P.G, P.G);
    draw = w.follow();
  }
  // Is this the last sum, the draw's or the one behind the last child?  (A child that stays
  // leads on; one whose test the sum decides may.)
  const bool last = draw || w.child(w.next, [](int) { return true; }) < 0;  // (the first wave's)
  double s = wave_sum(w.share(blockIdx.x, tid, kSliceThreads));
  if ((tid & 63) == 0) sh.wave[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < kSliceThreads / 64; ++k) s += sh.wave[k];
    P.part[(static_cast<int64_t>(P.round) * N + n) * P.G + blockIdx.x] = s;
    if (blockIdx.x == 0) P.done[n] = last ? P.round : kMaxRounds;
  }
}

__global__ __launch_bounds__(kEndThreads) void end_kernel(Params P) {
  __shared__ Shared sh;
  const int n = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, N = gridDim.x;
  Walk w{P, sh, draft::rows_of(P.starts, n, P.rows, P.max_nodes)};
  if (w.r.count == 0) return;
  const double first = P.round > 0 && tid < P.G ? P.part[static_cast<int64_t>(n) * P.G + tid] : 0.0;  // (asked for early)
  w.load();
  __syncthreads();
  int taken = 0;  // sums used of the launches before
  auto sum = [&] {  // the slices' sums into sh.part
    __syncthreads();
    if (taken < P.round) {
      const double *part = P.part + (static_cast<int64_t>(taken) * N + n) * P.G;
      if (tid < P.G) sh.part[tid] = taken ? part[tid] : first;
      ++taken;
    } else {
      for (int g = wave; g < P.G; g += kEndThreads / 64) {
        const double s = wave_sum(w.share(g, lane, 64));
        if (lane == 0) sh.part[g] = s;
      }
    }
    __syncthreads();
    return total_of(sh.part, P.G);
  };
  while (true) {
    // the children, one sum a rejection; `fresh`: sh.part is of the weights as they are
    bool fresh = false;
    while (!w.follow()) {
      w.mass = sum();
      fresh = true;
    }
    if (!fresh || w.A == 0.0) w.mass = sum();
    if (!(w.mass > 0.0) && w.A != 0.0) {  // nothing is left of p: p itself
      w.A = 0.0;
      taken = P.round;
      w.mass = sum();
    }
    if (!(w.mass > 0.0)) break;  // no token
    // the slice that holds u times the sum, or the last with any weight, then the token in it
    const double t = static_cast<double>(sh.u[0]) * w.mass;
    const double own = lane < P.G ? sh.part[lane] : 0.0;
    double upto = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(upto, d);
      if (lane >= d) upto += o;
    }
    const uint64_t some = __ballot(own > 0.0), past = __ballot(own > 0.0 && upto > t);
    const int slice = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some | 1);
    double below = __shfl(upto - own, slice);
    const float *p = w.prow(), *q = w.qrow();
    const int b = w.begin(slice), e = w.begin(slice + 1);
    const int each = 4 * ((e - b + 4 * kEndThreads - 1) / (4 * kEndThreads)), x0 = b + tid * each, x1 = min(x0 + each, e);
    double v[4], mine = 0.0;
    for (int x = x0; x < x1; x += 4) {
      w.weights(p, q, x, x1, v);
      mine += (v[0] + v[1]) + (v[2] + v[3]);
    }
    double inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    __syncthreads();  // (the last draw's reads are over)
    if (lane == 63) sh.wave[wave] = inc;
    if (tid == 0) sh.found = kEndThreads, sh.last = -1;
    __syncthreads();
    double waves = lane < kEndThreads / 64 ? sh.wave[lane] : 0.0;
#pragma unroll
    for (int d = 1; d < kEndThreads / 64; d <<= 1) {
      const double o = __shfl_up(waves, d);
      if (lane >= d) waves += o;
    }
    waves = __shfl(waves, max(wave - 1, 0));
    if (wave > 0) below += waves;
    // the first thread whose tokens reach t (rounding may leave t behind them all: the last)
    const uint64_t have = __ballot(mine > 0.0), reach = __ballot(mine > 0.0 && below + inc > t);
    if (lane == 0 && reach) atomicMin(&sh.found, 64 * wave + __builtin_ctzll(reach));
    if (lane == 0 && have) atomicMax(&sh.last, 64 * wave + 63 - __builtin_clzll(have));
    __syncthreads();
    if (tid == (sh.found < kEndThreads ? sh.found : sh.last)) {
      double c = below + (inc - mine);
      int token = -1;
      // (where c is rounded up past t already, the first token with weight)
      for (int x = x0; x < x1 && (token < 0 || !(c > t)); x += 4) {
        if (each > 4) w.weights(p, q, x, x1, v);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (v[j] > 0.0 && (token < 0 || !(c > t))) {
            token = x + j;
            c += v[j];
          }
      }
      sh.token = token;
    }
    __syncthreads();
    const int token = sh.last < 0 ? -1 : sh.token;
    if (token < 0) break;
    if (tid == 0) sh.target[w.at] = token;
    // A drafted token that was not given its weight may be drawn after all: the walk of the
    // accepted path would go there, so this one does.
    const int i = w.child(w.at + 1, [&](int c2) { return sh.tok[c2] == token; });
    if (i < 0) break;
    w.go(i);
    taken = P.round;
  }
  __syncthreads();
  for (int i = tid; i < w.r.count; i += kEndThreads) P.out[w.r.first + i] = sh.target[i];
}

}  // namespace verify
}  // namespace spk

using namespace spk;

static int verify_slices(int N, int V) {
  const int by_size = (V + 4095) / 4096, by_chip = N > 0 ? (1024 + N - 1) / N : 1;
  return std::max(1, std::min(std::min(by_size, by_chip), verify::kMaxSlices));
}

extern "C" size_t spk_verify_tree_workspace_bytes(int N, int V) {
  return N > 0 && V > 0 ? static_cast<size_t>(N) * (verify::kMaxRounds * verify_slices(N, V) * 8 + 8) : 0;
}

extern "C" int spk_verify_tree(const int64_t *tokens, const int32_t *parents, const float *target_probs,
                               int64_t target_stride, const float *draft_probs, int64_t draft_stride,
                               const float *uniforms, const int32_t *row_starts, int64_t rows, int N, int max_nodes,
                               int V, int distinct, int64_t *targets, void *workspace, size_t workspace_bytes,
                               void *stream) {
  if (rows < 0 || N < 0 || max_nodes <= 0 || V <= 0)
    return fail(SPK_EINVAL, "verify_tree: bad sizes rows=%lld N=%d max_nodes=%d V=%d", (long long)rows, N, max_nodes, V);
  if (max_nodes > verify::kMaxNodes || N > 65535)
    return fail(SPK_EUNSUPPORTED, "verify_tree: max_nodes=%d (at most %d), N=%d (at most 65535)", max_nodes,
                verify::kMaxNodes, N);
  if (N == 0 || rows == 0) return SPK_OK;
  if (!tokens || !parents || !target_probs || !draft_probs || !uniforms || !row_starts || !targets)
    return fail(SPK_EINVAL, "verify_tree: null pointer");
  // (in place is fine: a tree's tokens are read before its targets are written)
  if (targets != tokens && on_rows(targets, rows * 8, tokens, 0, rows * 8, 1))
    return fail(SPK_EINVAL, "verify_tree: targets lie on other rows' tokens");
  const size_t need = spk_verify_tree_workspace_bytes(N, V);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))
    return fail(SPK_EINVAL, "verify_tree: workspace of %zu bytes, %zu needed, aligned to 8", workspace ? workspace_bytes : 0,
                need);
  const int G = verify_slices(N, V), rounds = verify::rounds_for(max_nodes, V);
  double *part = static_cast<double *>(workspace);
  verify::Params P{tokens, parents, row_starts, target_probs, draft_probs, uniforms, target_stride, draft_stride, rows,
                   max_nodes, V, distinct, G, 0, part,
                   reinterpret_cast<int32_t *>(part + static_cast<size_t>(verify::kMaxRounds) * N * G), targets};
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (; P.round < rounds; ++P.round)
    verify::slice_kernel<<<dim3(G, N), verify::kSliceThreads, 0, s>>>(P);
  verify::end_kernel<<<N, verify::kEndThreads, 0, s>>>(P);
  return check_launch("verify_tree");
}
