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
// A test needs two numbers, a rejection the sum over the vocabulary (two rows of it).  The
// sums' passes are split over workgroups: launch r of the walk follows each tree up to its
// r-th sum (the sums before it are there, so every workgroup repeats the walk in a few
// dependent loads), and its slices add up their share.  The last launch, one workgroup a
// tree, follows the walk to its end, sums by itself where a tree needs more, and draws.
// Sums and tests are fp64: a decision differs from exact arithmetic's only where the numbers
// are equal to 15 digits.
#include <algorithm>

#include "common.hpp"
#include "draft_rows.hpp"

namespace spk {
namespace verify {

using draft::kMaxNodes;
constexpr int kSliceThreads = 256;
constexpr int kEndThreads = 1024;
constexpr int kMaxSlices = 64;
constexpr int kRounds = 1;

struct Params {
  const int64_t *tokens;
  const int32_t *parents, *starts;
  const float *p, *q, *u;
  int64_t ps, qs;  // row strides
  int64_t rows;
  int max_nodes, V, distinct, G, round;
  double *part;  // [round][tree][slice]
  int64_t *out;
};

struct Shared {
  int64_t tok[kMaxNodes], target[kMaxNodes];
  int32_t par[kMaxNodes];
  float u[kMaxNodes];
  double part[kMaxSlices], wave[kEndThreads / 64];
  int found, last;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

// A tree's walk.  Every thread of a workgroup follows it with the same numbers.
struct Walk {
  const Params &P;
  Shared &sh;
  draft::Rows r;
  int at, next;
  double A, mass, before;  // before: what q gives to the children tested so far

  __device__ __forceinline__ const float *prow() const { return P.p + (r.first + at) * P.ps; }
  __device__ __forceinline__ const float *qrow() const { return P.q + (r.first + at) * P.qs; }

  __device__ __forceinline__ void go(int row) {
    at = row;
    next = row + 1;
    A = before = 0.0;
    mass = 1.0;
  }
  // The lowest-numbered child of `at` from row `next` on that `ok` takes, or -1.
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
  // Tests children until a sum over the vocabulary is needed, for the next test or (true) for
  // the draw.
  __device__ __forceinline__ bool tests() {
    for (;;) {
      const int i = child(next, [](int) { return true; });
      if (i < 0) return true;
      const int64_t x = sh.tok[i];
      double px = 0.0, qx = 0.0;
      if (x >= 0 && x < P.V) px = prow()[x], qx = qrow()[x];
      const double w = fmax(px - A * qx, 0.0);
      double c = mass;
      if (P.distinct) {
        const double left = fmax(1.0 - before, qx);
        if (left > 0.0) c /= left;
      }
      if (static_cast<double>(sh.u[i]) * qx * c < w) {
        if (threadIdx.x == 0) sh.target[at] = x;
        go(i);
        continue;
      }
      A += c;
      before += qx;
      next = i + 1;
      return false;
    }
  }
  __device__ __forceinline__ double weight(const float *p, const float *q, int x) const {
    const double v = p[x];
    return fmax(A == 0.0 ? v : v - A * static_cast<double>(q[x]), 0.0);
  }
  __device__ __forceinline__ int begin(int slice) const {
    return static_cast<int>(static_cast<int64_t>(P.V) * slice / P.G);
  }
};

__device__ __forceinline__ void load_tree(const Params &P, Shared &sh, const draft::Rows &r) {
  for (int i = threadIdx.x; i < r.count; i += blockDim.x) {
    sh.tok[i] = P.tokens[r.first + i];
    sh.par[i] = P.parents[r.first + i];
    sh.u[i] = P.u[r.first + i];
    sh.target[i] = -1;
  }
}

// The sum of the slices' partial sums, in their order.
__device__ __forceinline__ double total_of(const double *part, int G) {
  double s = 0.0;
  for (int g = 0; g < G; ++g) s += part[g];
  return s;
}

__global__ __launch_bounds__(kSliceThreads) void slice_kernel(Params P) {
  __shared__ Shared sh;
  const int n = blockIdx.y, tid = threadIdx.x, N = gridDim.y;
  Walk w{P, sh, draft::rows_of(P.starts, n, P.rows, P.max_nodes)};
  if (w.r.count == 0) return;
  load_tree(P, sh, w.r);
  __syncthreads();
  w.go(0);
  bool draw = w.tests();
  for (int k = 0; k < P.round; ++k) {
    if (draw) return;  // this tree's last sum is there
    w.mass = total_of(P.part + (static_cast<int64_t>(k) * N + n) * P.G, P.G);
    draw = w.tests();
    // (after the last child the sum that was just taken is the draw's)
    if (draw && w.A != 0.0) return;
  }
  const float *p = w.prow(), *q = w.qrow();
  double s = 0.0;
  for (int x = w.begin(blockIdx.x) + tid; x < w.begin(blockIdx.x + 1); x += kSliceThreads) s += w.weight(p, q, x);
  s = wave_sum(s);
  if ((tid & 63) == 0) sh.wave[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < kSliceThreads / 64; ++k) s += sh.wave[k];
    P.part[(static_cast<int64_t>(P.round) * N + n) * P.G + blockIdx.x] = s;
  }
}

__global__ __launch_bounds__(kEndThreads) void end_kernel(Params P) {
  __shared__ Shared sh;
  const int n = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, N = gridDim.x;
  Walk w{P, sh, draft::rows_of(P.starts, n, P.rows, P.max_nodes)};
  if (w.r.count == 0) return;
  load_tree(P, sh, w.r);
  __syncthreads();
  int taken = 0;  // sums used of the launches before
  auto sum = [&] {  // the slices' sums into sh.part
    __syncthreads();
    if (taken < P.round) {
      const double *part = P.part + (static_cast<int64_t>(taken++) * N + n) * P.G;
      if (tid < P.G) sh.part[tid] = part[tid];
    } else {
      const float *p = w.prow(), *q = w.qrow();
      for (int g = wave; g < P.G; g += kEndThreads / 64) {
        double s = 0.0;
        for (int x = w.begin(g) + lane; x < w.begin(g + 1); x += 64) s += w.weight(p, q, x);
        s = wave_sum(s);
        if (lane == 0) sh.part[g] = s;
      }
    }
    __syncthreads();
    return total_of(sh.part, P.G);
  };
  w.go(0);
  while (true) {
    // the children, one sum a rejection; `fresh`: sh.part is of the weights as they are
    bool fresh = false;
    while (!w.tests()) {
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
    // the slice that holds u times the sum, then the token in it
    const double t = static_cast<double>(sh.u[0]) * w.mass;
    double below = 0.0, cum = 0.0;
    int slice = 0;
    for (int g = 0; g < P.G; ++g) {
      const double s = sh.part[g];
      if (s > 0.0) {
        slice = g;
        below = cum;
        if (cum + s > t) break;
      }
      cum += s;
    }
    const float *p = w.prow(), *q = w.qrow();
    const int b = w.begin(slice), e = w.begin(slice + 1), each = (e - b + kEndThreads - 1) / kEndThreads;
    const int x0 = min(b + tid * each, e), x1 = min(x0 + each, e);
    double mine = 0.0;
    for (int x = x0; x < x1; ++x) mine += w.weight(p, q, x);
    double inc = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const double o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 63) sh.wave[wave] = inc;
    if (tid == 0) sh.found = P.V, sh.last = -1;
    __syncthreads();
    for (int k = 0; k < wave; ++k) below += sh.wave[k];
    double c = below + (inc - mine);
    if (mine > 0.0) {
      int last = -1;
      for (int x = x0; x < x1; ++x) {
        const double v = w.weight(p, q, x);
        if (!(v > 0.0)) continue;
        last = x;
        c += v;
        if (c > t) {
          atomicMin(&sh.found, x);
          break;
        }
      }
      atomicMax(&sh.last, last);
    }
    __syncthreads();
    const int token = sh.found < P.V ? sh.found : sh.last;  // (rounding may leave t at the slice's end)
    __syncthreads();
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
  return N > 0 && V > 0 ? static_cast<size_t>(verify::kRounds) * N * verify_slices(N, V) * 8 : 0;
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
  const size_t need = spk_verify_tree_workspace_bytes(N, V);
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))
    return fail(SPK_EINVAL, "verify_tree: workspace of %zu bytes, %zu needed, aligned to 8", workspace ? workspace_bytes : 0,
                need);
  verify::Params P{tokens, parents, row_starts, target_probs, draft_probs, uniforms, target_stride, draft_stride, rows,
                   max_nodes, V, distinct, verify_slices(N, V), 0, static_cast<double *>(workspace), targets};
  hipStream_t s = static_cast<hipStream_t>(stream);
  for (; P.round < verify::kRounds; ++P.round)
    verify::slice_kernel<<<dim3(P.G, N), verify::kSliceThreads, 0, s>>>(P);
  verify::end_kernel<<<N, verify::kEndThreads, 0, s>>>(P);
  return check_launch("verify_tree");
}
