// Which drafts of a speculative tree stand: the step after `spec`, which gives every draft row its logits.  The reference
// verifies attention only (kernels/spec_opus55_v7.py:467-521); the float64 statement lives in oracle/ref64.py (accept_ref64).
//
// Node 0 of a request's tree is the token that is decided already, row c of target_probs is the target's distribution
// after node c, row c of draft_probs the one that c's children were drawn from.  At a node, its children are tried in
// their order; with r_0 = p, a child with token x stands with probability min(1, r(x) / q(x)), and after a refusal the
// target is what the draft left of it, r_{j+1} = max(r_j - q, 0) normalised again.  Kept without normalising:
//     r_j = max(r_{j-1} - M_{j-1} q, 0),  M_j = sum r_j,  M_0 = 1       (M: what the normalised one is divided by)
//         = max(p - S_j q, 0)  with  S_j = M_0 + ... + M_{j-1}          (once an entry is 0 it stays 0)
// so a node's state is two numbers, and a refusal is one pass over a row of p and of q.  A child is taken when
// u M q(x) < r(x).  Without draft_probs the drafts were chosen, not drawn (q = 1 at x): a refusal takes x out of r and
// r(x) off M, which needs no pass.  When no child is left the next token is drawn from r (from p at a leaf, or if r is
// empty) by the inverse of its cumulative sum at the root's number.
//
// Everything is computed in 64 bits or in pairs of fp32 numbers: the answers are whole numbers, and an fp32 sum over a
// vocabulary is off by more than the width of a rare token.  Conversions to fp64 are what a pass over a row is bound by (15 lanes a
// cycle and SM, 6 elements with both operands converted and the difference taken in fp64), so the difference p - S q is
// taken in pairs of fp32 numbers without error: with S = Sh + Sl,
//     t = Sh q rounded, te = Sh q - t (one fused multiply-add), hi = p - t rounded, lo = (p - hi) - t (exact where hi > 0),
//     p - S q = hi + (lo - te - Sl q), the bracket below 2^-23 of p and rounded at 2^-47;
// only hi is converted and summed in fp64, the brackets are summed in fp32 by each thread (n entries).  So M is off by less
// than (2 n + 3) 2^-47 of the row's sum, where fp64 throughout is off by some 2^-53, and twice the error of the M before (it
// is part of S): 2^k (2 n + 3) 2^-47 at the k-th refusal of a node.  Restated in NumPy: below 4e-16 for n of 8 and 256 over five
// refusals, at an M down to 1e-7.  At the first refusal of a node S is 1 and t is q itself: three subtractions.  A pass over a row that L2 holds is bound by its instructions (20 an element took 4.1 us
// for 16384 entries a CTA).  Entries that are NaN, infinite or negative count as 0; a vector that has one is found by one
// comparison of bits and cleaned in a branch of its own.
//
// Of a request's kd rows only those are read at which a draft is refused or the walk ends; the rest of the walk needs
// p and q at (parent, token) of each node, gathered by one thread a node before it begins.  A request is a CLUSTER of
// up to 8 CTAs that walk its tree in step and split the vocabulary between them: partial sums cross through distributed
// shared memory.  Measured: 32 trees of 64 nodes over 131072 entries (fp32) 31 to 34 us, of which the rows that
// have to be read take 5.2; what bounds it is the chain of passes of the request that is refused most often, each 2.5 to 4 us.
// 128 chains over 100003 entries (bf16) 15 us, one chain of 8 over 32768 entries 6.6 us (latency: two dependent gathers, one pass, the
// cluster's barrier, one more look at a warp's range).  Inside a CTA every warp owns a contiguous range of the row, so the drawn position is found by prefix
// over CTAs, then warps, then one warp's range.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <atomic>
#include <cstring>

#include "common.cuh"

namespace vmk {

namespace cg = cooperative_groups;

constexpr int kAcThreads = 512;
constexpr int kAcWarps = kAcThreads / 32;
static_assert(kAcWarps <= 32, "a lane for every warp");
constexpr int kAcNodes = VMK_SPEC_MAX_DRAFTS;
constexpr int kAcCluster = 8;
static_assert(kAcNodes <= kAcThreads, "one thread per node");

struct AcceptParams {
  const void *p, *q;             // (B, kd, V), q null: drafts without probabilities
  const int32_t* tokens;         // (B, kd)
  const uint32_t* bits;          // (B, kd, words)
  const float* u;                // (B, kd)
  int32_t *path, *count, *next;  // (B, kd), (B), (B)
  int kd, words, V;
  int32_t* status;
};

struct AcceptShared {
  float p[kAcNodes], q[kAcNodes], u[kAcNodes];
  int token[kAcNodes], parent[kAcNodes];
  int gone[kAcNodes];            // tokens refused at the current node (drafts without probabilities)
  int path[kAcNodes];
  double warp_sum[kAcWarps];
  double rank_sum[2][kAcCluster];   // every CTA's sum of a pass; alternating, so that one barrier a pass is enough
  double scan[kAcWarps];
  int found, positive;
};

// Sanitised probability: positive and finite, else 0.
__device__ __forceinline__ float ac_clean(float x) {
  return __float_as_uint(x) - 1u < 0x7f7fffffu ? x : 0.f;
}
template <typename T>
__device__ __forceinline__ float ac_float(T x);
template <>
__device__ __forceinline__ float ac_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float ac_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float ac_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
struct AcVec {
  static constexpr int N = 16 / sizeof(T);
  union {
    uint4 raw;
    T e[N];
  };
  __device__ AcVec() {}
};

// N entries as floats that are positive and finite or 0.
template <typename T>
__device__ __forceinline__ void ac_floats(float (&f)[AcVec<T>::N], const AcVec<T>& v) {
  constexpr int N = AcVec<T>::N;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    f[k] = ac_float<T>(v.e[k]);
    top = max(top, __float_as_uint(f[k]));
  }
  if (top > 0x7f7fffffu) {
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = ac_clean(f[k]);
  }
}

// A row of V probabilities as 16-byte vectors: rows of an odd length begin inside one.  Vector i holds the elements
// [i * N - head, (i + 1) * N - head); those outside the row are 0.  `whole`: the vector lies in the row and `row` has the
// alignment that head stands for.
template <typename T>
__device__ __forceinline__ void ac_load(AcVec<T>& v, const T* row, int head, int V, int i, bool whole) {
  constexpr int N = AcVec<T>::N;
  const int e0 = i * N - head;
  if (whole) {
    v.raw = __ldg(reinterpret_cast<const uint4*>(row + e0));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v.e[k] = (e0 + k >= 0 && e0 + k < V) ? row[e0 + k] : T(0.f);
  }
}

struct AcScale {                 // S as two fp32 numbers; 0: q is not taken off
  float hi, lo;
};

// Weights max(p - S q, 0) of one vector, or p without the refused tokens, as hi + lo.
template <typename T, bool HAS_Q>
__device__ __forceinline__ void ac_weights(float (&hi)[AcVec<T>::N], float (&lo)[AcVec<T>::N], const AcVec<T>& p, const AcVec<T>& q,
                                           AcScale S, const int* gone, int n_gone, int e0) {
  constexpr int N = AcVec<T>::N;
  ac_floats<T>(hi, p);
#pragma unroll
  for (int k = 0; k < N; ++k) lo[k] = 0.f;
  if (HAS_Q) {
    if (S.hi != 0.f) {
      float y[N];
      ac_floats<T>(y, q);
      if (S.hi == 1.f && S.lo == 0.f) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float d = __fsub_rn(hi[k], y[k]);
          lo[k] = d > 0.f ? __fsub_rn(__fsub_rn(hi[k], d), y[k]) : 0.f;
          hi[k] = fmaxf(d, 0.f);
        }
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float t = __fmul_rn(S.hi, y[k]), te = __fmaf_rn(S.hi, y[k], -t);
          const float d = __fsub_rn(hi[k], t), e = __fsub_rn(__fsub_rn(hi[k], d), t);
          const float r = __fmaf_rn(-S.lo, y[k], __fsub_rn(e, te));
          const bool some = d + r > 0.f;
          hi[k] = some ? d : 0.f;
          lo[k] = some ? r : 0.f;
        }
      }
    }
  } else {
    for (int g = 0; g < n_gone; ++g) {
      const int k0 = gone[g] - e0;
      if ((unsigned)k0 < (unsigned)N) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (k == k0) hi[k] = 0.f;
      }
    }
  }
}

// Lanes hold sums of consecutive ranges (those beyond the last range 0), `start` is what lies before them.  The first range whose
// running sum exceeds `target`, or the last that has anything; `before`: the running sum where it begins.
__device__ __forceinline__ int ac_pick(double s, double start, double target, double& before) {
  const int lane = threadIdx.x & 31;
  double incl = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  const uint32_t over = __ballot_sync(0xffffffffu, s > 0.0 && start + incl > target), some = __ballot_sync(0xffffffffu, s > 0.0);
  const int i = over != 0u ? __ffs(over) - 1 : some != 0u ? 31 - __clz(some) : 0;
  before = start + __shfl_sync(0xffffffffu, incl - s, i);
  return i;
}

template <typename T, bool HAS_Q>
__global__ void __launch_bounds__(kAcThreads, 2) accept_kernel(const AcceptParams a) {
  constexpr int N = AcVec<T>::N;
  __shared__ AcceptShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  // (waited for before anything is written into a peer's shared memory: the peer runs by then)
  if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int b = blockIdx.x / ranks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kd = a.kd, V = a.V;
  pdl_wait();

  // ---- the tree, and the two probabilities of every node
  const size_t node0 = (size_t)b * kd;
  if (tid < kd) {
    const uint32_t* words = a.bits + (node0 + tid) * a.words;
    const int x = a.tokens[node0 + tid];
    const float u = a.u[node0 + tid];
    uint32_t m[kAcNodes / 32];
#pragma unroll
    for (int w = 0; w < kAcNodes / 32; ++w) m[w] = w < a.words && w * 32 < tid ? words[w] : 0u;
    int parent = -1;
#pragma unroll
    for (int w = 0; w < kAcNodes / 32; ++w) {
      if (w == tid >> 5) m[w] &= (1u << (tid & 31)) - 1u;
      if (m[w] != 0u) parent = w * 32 + 31 - __clz(m[w]);
    }
    const bool inside = x >= 0 && x < V;
    float p = 0.f, q = 0.f;
    if (parent >= 0 && inside) {
      const size_t at = (node0 + parent) * V + x;
      p = ac_clean(ac_float<T>(static_cast<const T*>(a.p)[at]));
      if (HAS_Q) q = ac_clean(ac_float<T>(static_cast<const T*>(a.q)[at]));
    }
    if (tid > 0 && !inside && rank == 0) report(a.status, kStatusBadIndex);
    sh.parent[tid] = parent;
    sh.token[tid] = x;
    sh.p[tid] = p;
    sh.q[tid] = q;
    sh.u[tid] = u;
    sh.path[tid] = tid == 0 ? 0 : -1;
  }
  __syncthreads();
  if (ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  int mine[kAcNodes / 32];                       // every warp: parents of the nodes lane, lane + 32, ...
#pragma unroll
  for (int w = 0; w < kAcNodes / 32; ++w) mine[w] = w * 32 + lane < kd ? sh.parent[w * 32 + lane] : -1;

  int cur = 0, last = 0, n_path = 1, n_gone = 0, passes = 0;   // last: the child tried last
  double S = 0.0, M = 1.0;
  double T_left = 0.0;                           // sum of the weights of the last pass, if it was at this state
  bool have_sum = false;
  const T *prow = nullptr, *qrow = nullptr;
  bool q16 = true;                               // rows of p and q begin at the same place of a 16-byte vector
  int head = 0, nvec = 0, seg = 0;               // every warp of the cluster has `seg` vectors of the row
  AcScale scale{0.f, 0.f};

  // ---- the walk, the same in every thread of the cluster; one turn per child or pass
  for (;;) {
    // the next child of the current node
    int i = -1;
#pragma unroll
    for (int w = kAcNodes / 32 - 1; w >= 0; --w) {
      const uint32_t kids = __ballot_sync(0xffffffffu, mine[w] == cur && w * 32 + lane > last);
      if (kids != 0u) i = w * 32 + __ffs(kids) - 1;
    }
    if (i >= 0) {
      last = i;
      const double p = sh.p[i], q = sh.q[i], u = sh.u[i];
      double r;
      bool yes;
      if (HAS_Q) {
        r = __dsub_rn(p, __dmul_rn(S, q));
        yes = r > 0.0 && __dmul_rn(__dmul_rn(u, M), q) < r;
      } else {
        r = p;
        const int x = sh.token[i];
        for (int g = 0; g < n_gone; ++g)
          if (sh.gone[g] == x) r = 0.0;
        yes = r > 0.0 && __dmul_rn(u, M) < r;
      }
      if (yes) {
        cur = i;
        if (tid == 0) sh.path[n_path] = i;
        ++n_path;
        S = 0.0;
        M = 1.0;
        n_gone = 0;
        have_sum = false;
        continue;
      }
      if (!HAS_Q) {
        M = fmax(__dsub_rn(M, r), 0.0);
        __syncthreads();                         // nobody is still reading the list
        if (tid == 0) sh.gone[n_gone] = sh.token[i];
        ++n_gone;
        __syncthreads();
        continue;
      }
      S += M;
    } else if (have_sum) {
      if (T_left > 0.0 || (S == 0.0 && n_gone == 0)) break;
      S = 0.0;                                   // the residual is empty: the target itself
      n_gone = 0;
    }

    // ---- a pass: the sum of the current weights over the row, every CTA's in rank_sum, every warp's of this CTA in warp_sum
    prow = static_cast<const T*>(a.p) + (node0 + cur) * V;
    qrow = HAS_Q ? static_cast<const T*>(a.q) + (node0 + cur) * V : prow;
    q16 = ((reinterpret_cast<uintptr_t>(prow) ^ reinterpret_cast<uintptr_t>(qrow)) & 15) == 0;
    head = (int)((reinterpret_cast<uintptr_t>(prow) & 15) / sizeof(T));
    nvec = (head + V + N - 1) / N;
    seg = (nvec + ranks * kAcWarps - 1) / (ranks * kAcWarps);
    scale.hi = HAS_Q ? (float)S : 0.f;
    scale.lo = HAS_Q ? (float)(S - (double)scale.hi) : 0.f;
    const bool minus_q = scale.hi != 0.f;
    const int first = (rank * kAcWarps + warp) * seg, end = min(first + seg, nvec);
    double sum[2] = {0.0, 0.0};
    float low = 0.f;
    auto add = [&](const AcVec<T>& p, const AcVec<T>& q, int at) {
      float hi[N], lo[N];
      ac_weights<T, HAS_Q>(hi, lo, p, q, scale, sh.gone, n_gone, at * N - head);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        sum[e & 1] += (double)hi[e];
        if (HAS_Q) low += lo[e];
      }
    };
    // whole vectors first, several in flight; then the row's ends, and rows of q that do not match p's alignment
    constexpr int U = HAS_Q && sizeof(T) == 2 ? 2 : 4;     // what 64 registers hold
    const int w0 = q16 ? max(first, head > 0 ? 1 : 0) : end, w1 = q16 ? min(end, (head + V) / N) : end;
    int v = w0 + lane;
    for (; v + (U - 1) * 32 < w1; v += U * 32) {
      AcVec<T> p[U], q[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        ac_load<T>(p[k], prow, head, V, v + k * 32, true);
        if (HAS_Q && minus_q) ac_load<T>(q[k], qrow, head, V, v + k * 32, true);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) add(p[k], q[k], v + k * 32);
    }
    for (; v < w1; v += 32) {
      AcVec<T> p, q;
      ac_load<T>(p, prow, head, V, v, true);
      if (HAS_Q && minus_q) ac_load<T>(q, qrow, head, V, v, true);
      add(p, q, v);
    }
    for (int x = first + lane; x < end; x += 32) {
      if (x >= w0 && x < w1) {                    // done above: on to the last of them
        x += (w1 - 1 - x) / 32 * 32;
        continue;
      }
      AcVec<T> p, q;
      ac_load<T>(p, prow, head, V, x, false);
      if (HAS_Q && minus_q) ac_load<T>(q, qrow, head, V, x, false);
      add(p, q, x);
    }
    double t = sum[0] + sum[1] + (double)low;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    __syncthreads();                             // readers of the pass before are done with warp_sum
    if (lane == 0) sh.warp_sum[warp] = t;
    __syncthreads();
    double* mine_sum = &sh.rank_sum[passes & 1][0];
    if (warp == 0) {
      double all = lane < kAcWarps ? sh.warp_sum[lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
      if (lane < ranks) *cluster.map_shared_rank(mine_sum + rank, lane) = all;
    }
    if (ranks > 1) cluster.sync(); else __syncthreads();
    double total = 0.0;
    for (int r = 0; r < ranks; ++r) total += mine_sum[r];
    ++passes;
    T_left = M = total;
    have_sum = true;
  }

  // ---- the next token
  if (T_left > 0.0) {
    const double* rank_sum = sh.rank_sum[(passes - 1) & 1];
    const double target = __dmul_rn((double)sh.u[0], T_left);
    // first CTA, then first warp of it, whose running sum exceeds the target; the last one that has anything if none does
    double before, wb;
    const int owner = ac_pick(lane < ranks ? rank_sum[lane] : 0.0, 0.0, target, before);
    if (owner == rank) {
      const int ow = ac_pick(lane < kAcWarps ? sh.warp_sum[lane] : 0.0, before, target, wb);
      // that warp's range, a vector to every thread of the CTA
      const int first = (rank * kAcWarps + ow) * seg, end = min(first + seg, nvec);
      if (tid == 0) {
        sh.found = 0x7fffffff;
        sh.positive = -1;
      }
      double run = wb;
      for (int i0 = first; i0 < end; i0 += kAcThreads) {
        const int i = i0 + tid;
        double w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = 0.0;
        if (i < end) {
          AcVec<T> p, q;
          const bool whole = i * N - head >= 0 && (i + 1) * N - head <= V;
          ac_load<T>(p, prow, head, V, i, whole);
          if (HAS_Q && scale.hi != 0.f) ac_load<T>(q, qrow, head, V, i, whole && q16);
          float hi[N], lo[N];
          ac_weights<T, HAS_Q>(hi, lo, p, q, scale, sh.gone, n_gone, i * N - head);
#pragma unroll
          for (int e = 0; e < N; ++e) w[e] = (double)hi[e] + (double)lo[e];
        }
        double own = 0.0;
#pragma unroll
        for (int e = 0; e < N; ++e) own += w[e];
        double incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        __syncthreads();                         // found is set up; readers of the step before are done with scan
        if (lane == 31) sh.scan[warp] = incl;
        __syncthreads();
        // warps before this one, and all of them: a sum over lanes each
        double part = lane < kAcWarps ? sh.scan[lane] : 0.0, mine_before = lane < warp ? part : 0.0;
#pragma unroll
        for (int o = kAcWarps / 2; o > 0; o >>= 1) {
          part += __shfl_xor_sync(0xffffffffu, part, o);
          mine_before += __shfl_xor_sync(0xffffffffu, mine_before, o);
        }
        part = __shfl_sync(0xffffffffu, part, 0);
        double c = run + __shfl_sync(0xffffffffu, mine_before, 0) + (incl - own);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          c += w[e];
          if (w[e] > 0.0) {
            if (c > target) atomicMin(&sh.found, i * N - head + e);
            atomicMax(&sh.positive, i * N - head + e);
          }
        }
        run += part;
        __syncthreads();
        if (sh.found != 0x7fffffff) break;
      }
      if (tid == 0) a.next[b] = sh.found != 0x7fffffff ? sh.found : sh.positive;
    }
  } else if (rank == 0 && tid == 0) {
    a.next[b] = -1;
  }
  __syncthreads();
  if (rank == 0) {
    if (tid < kd) a.path[node0 + tid] = sh.path[tid];
    if (tid == 0) a.count[b] = n_path;
  }
  // no barrier at the end: what the peers wrote into this CTA's memory was there at the last pass's, and nothing is
  // written or read there after it
}

static void accept_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], int B, int c, cudaStream_t stream) {
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)B * c);
  cfg.blockDim = dim3(kAcThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
}

// CTAs per request: the most (up to 8, with at least 4096 entries each) at which the clusters of all requests are resident
// together, two CTAs an SM.  Measured with at most 8, 4, 2 and 1 (us): 32 trees of 64 nodes over 131072 entries 29.9, 36.1, 57.4,
// 97.2; one chain of 8 over 32768 6.6, 7.0, 8.2, 9.7; 32 chains of 8 over 131072 12.6, 12.1, 16.8, 26; 128 over 100003 in
// bf16 (two are resident) 15.0 with two, 17.0 with one; 64 over 8192 (4, 2, 1) 9.2, 8.2, 7.7: hence the 4096.
static int accept_cluster(int B, int V) {
  if (g_batch_invariant) return V >= 4 * 4096 ? 4 : 1;    // by the row alone: the order of the sums must not follow the batch
  static std::atomic<int> resident[64][4];                 // clusters of 1 << i CTAs that run together, by device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
  for (int i = 3; i > 0; --i) {
    const int c = 1 << i;
    if (V < c * 4096) continue;
    int n = resident[dev][i].load();
    if (n == 0) {
      cudaLaunchConfig_t cfg;
      cudaLaunchAttribute attr[2];
      accept_config(cfg, attr, 1, c, nullptr);
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, accept_kernel<float, true>, &cfg) != cudaSuccess || n < 1) {
        (void)cudaGetLastError();
        n = 1;
      }
      resident[dev][i].store(n);
    }
    if (B <= n) return c;
  }
  return 1;
}

template <typename T>
static int accept_launch(const AcceptParams& a, int B, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  accept_config(cfg, attr, B, accept_cluster(B, a.V), stream);
  return check_launch(a.q != nullptr ? cudaLaunchKernelEx(&cfg, accept_kernel<T, true>, a) : cudaLaunchKernelEx(&cfg, accept_kernel<T, false>, a));
}

}  // namespace vmk

using namespace vmk;

extern "C" int vmk_accept(const void* target_probs, const void* draft_probs, const int32_t* tokens, const uint32_t* bits,
                          int bits_words, const float* u, int32_t* path, int32_t* count, int32_t* next, int B, int kd, int V,
                          int dtype, int32_t* status, void* stream) {
  auto bad = [](const void* x, uintptr_t al) { return x == nullptr || (reinterpret_cast<uintptr_t>(x) & (al - 1)) != 0; };
  if (B < 0 || kd <= 0 || V <= 0 || bits_words <= 0 || dtype < 0 || dtype > 2) return VMK_E_BADARG;
  if (kd > kAcNodes || kd > 32 * bits_words) return VMK_E_UNSUPPORTED;
  if (V > 0x7fffff00 || B > 0x7fffffff / kAcCluster) return VMK_E_TOO_LARGE;
  if (B == 0) return VMK_OK;
  const uintptr_t size = dtype == 0 ? 4 : 2;                // rows of an odd length are not aligned either
  if (bad(target_probs, size) || (draft_probs && bad(draft_probs, size)) || bad(tokens, 4) || bad(bits, 4) || bad(u, 4) || bad(path, 4) ||
      bad(count, 4) || bad(next, 4) || (status && bad(status, 4)))
    return VMK_E_BADARG;
  AcceptParams a;
  memset(&a, 0, sizeof(a));
  a.p = target_probs;
  a.q = draft_probs;
  a.tokens = tokens;
  a.bits = bits;
  a.words = bits_words;
  a.u = u;
  a.path = path;
  a.count = count;
  a.next = next;
  a.kd = kd;
  a.V = V;
  a.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == 0 ? accept_launch<float>(a, B, s) : dtype == 1 ? accept_launch<__half>(a, B, s) : accept_launch<__nv_bfloat16>(a, B, s);
}
