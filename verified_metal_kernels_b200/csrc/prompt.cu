// Attention of whole prompts (or of chunks of prompts over a cache) on the 5th-generation tensor cores: what fills a
// serving engine before the decode kernels of this library take over.  The reference defines decode ops only; the
// float64 statement lives in oracle/ref64.py (prompt_ref64).
//
//   sequence s has the queries [cu_q[s], cu_q[s+1]) (nq of them) and nk keys; query i of it sees the keys
//   j <= nk - nq + i (causal, aligned at the end) or all nk of them:
//       out[i] = sum_j exp(q_i . k_j / sqrt(128) - m_i) v_j / sum_j exp(q_i . k_j / sqrt(128) - m_i)
//   in one pass over the keys with the running maximum m and sum of the softmax in fp32; a query that sees no key
//   gets zeros, and so do rows of `out` outside every sequence.
//
// One UNIT of work = (256-row tile of a sequence, kv head): the rows of a tile are stacked (token, query head of the
// group) pairs, so every K/V tile is read once for the whole group; the tile is two 128-row tiles A and B that share
// the K/V tiles and alternate on the tensor pipe.  A group of G heads puts floor(128 / G) tokens into a tile (the
// rest of its rows is unused).  A planner kernel (one CTA) lists the tiles of all sequences, those with the most key
// blocks first (under a causal mask the last tile of a prompt costs many times its first, and units are handed out
// in that order by an atomic counter, so the short ones fill the end), and a PERSISTENT CTA per SM takes units.
// 384 threads, warp-specialised:
//   warp 8      takes units from the counter, hands them to the other warps through a two-entry ring, and is the TMA
//               producer: Q tiles, and K_0, V_0, K_1, V_1, ... into one ring of five 32 KiB slots, running ahead into
//               the next unit
//   warp 9      owns tensor memory and issues every tcgen05.mma, in the order  P.V of tile t at block j, then Q.K^T of
//               tile t at block j + 1, tiles alternating.  Products of one thread execute in order, so Q.K^T may
//               overwrite the scores of a block as soon as the P.V that reads their P is issued: no wait between the
//               two, and the pipe runs one tile's pair while the other tile's softmax works
//   warps 0-3   softmax of tile A, warps 4-7 of tile B: one thread per row
//   warps 10,11 look for NaN and infinities in the rows of V that not every row of the unit sees; warp 10 zeroes the rows of `out`
//               outside every sequence
// Tensor memory (512 columns): S_A, S_B, O_A, O_B, 128 columns each; P (16-bit pairs, 64 columns) over its scores.
// O is rescaled only when a row's maximum grew by more than 2^8 (P stays below 2^8 and the result is exact); the
// softmax thread does it itself: when the scores of block j are there, the P.V of block j - 1, issued before them,
// has completed.  P is rounded to the tensors' 16-bit type before P.V (the tensor pipe takes 16-bit operands); the
// sum that divides is that of the unrounded P.
//
// Measured (bf16, 32 query heads on 8): 32768 tokens 6.57 ms at 1.965 GHz (1340 TFLOP/s over the visible pairs), 7.57 at the
// power limit (1.54 GHz); 24 prompts of up to 1999 tokens 250 us at 1.965 GHz, 287 at 1.64; 128 tokens 8.8 us; 17 tokens over
// 60001 keys 55 to 58 us (4.2 to 4.5 TB/s).  What bounds the long ones: each tile's softmax and products follow one another, and two tiles
// keep the tensor pipe and the exponential unit at about 60 % each.  A block of 128 keys costs a pair of tiles 3500 cycles
// where the products alone take 2060 and the exponentials 2048.  Tried, and slower: scores of 64 keys in two buffers (N = 64
// products take 48 cycles, not 32), two threads a row, warps of their own for the result, a polynomial for a quarter of the
// exponentials, products cut to the keys that a tile's last block has (the descriptors then leave the uniform registers).
//
// A key that a row does not see has P = 0, but 0 times Inf or NaN is NaN.  In the blocks that the mask cuts, such entries of V
// are cleared in shared memory and added to the results of the rows that see their key (prompt_add_special).  (One short prompt
// 8.67 -> 8.75 us, 24 ragged ones 237 -> 247, a long one the same; one warp a tile instead of two that share the rows 9.27 and 245.)
// Rows of V past the end of a sequence (the next sequence's, or whatever a page holds there) are cleared in shared
// memory before the product: their P is 0, but 0 times Inf would poison the row.
// Every mbarrier wait is bounded; a wait that runs out sets the status word and the CTA winds down through the common
// exit, where tensor memory is freed.
#include <atomic>
#include <cstring>
#include <type_traits>

#include "tcgen05.cuh"

namespace vmk {

constexpr int kPmBK = 128;                       // keys per block
constexpr int kPmD = 128;
constexpr int kPmHalf = 128 * 128;               // [128 rows][128 B] swizzled: one 64-wide half of the head dim
constexpr int kPmTile = 2 * kPmHalf;             // 32 KiB: a Q, K or V tile
constexpr int kPmSlots = 5;
constexpr int kPmTwinSlots = 6;                  // where both tiles read one Q tile (prompt_twin), the other's place is a slot
constexpr int kPmSched = 2;
constexpr int kPmThreads = 384;                // 12 warps x 168 registers; after set-up 2 x 128 threads hold 216, 128 hold 72
constexpr int kPmCols = 512;
constexpr int kPmColS = 0, kPmColO = 256;
constexpr float kPmLazy = 8.f;                   // log2 units
constexpr int kPmPlanThreads = 1024;
// Key blocks that a share holds at least, where 4 CTAs and more share a unit (few rows to merge) and where 2 or 3 do.  (us: 1
// query over 512 keys 10.2 at 2, 11.2 at 4; 32 over 1500 14.1 and 15.5; 512 over 1100 26.2 at 4, 23.3 at 5; 300 over 1500
// 25.7 at 5, 30.8 at 6; 32 heads on 8.)
constexpr int kPmSplitFew = 2, kPmSplitMany = 5;
constexpr int kPmMaxSplit = 32;
constexpr int kPmBins = 256;
constexpr int kPmMaxItems = 1 << 20;             // tiles of a call: 16 million tokens at 16 heads a group, 268 million at one

struct PromptItem {          // one 256-row tile of one sequence
  int tok0;                  // first query token (index into q)
  int ntok;                  // tokens of the tile, 1 .. 2 * tokens per 128-row tile
  int k0;                    // contiguous keys: index of the sequence's first key; paged: the sequence
  int nk;                    // keys of the sequence
  int vis0;                  // keys the tile's first token sees, minus one; token i sees min(nk, vis0 + i + 1)
  int h;                     // kv head (partials only: the merge reads it here)
  int pad[2];
};

struct PromptCtrl {
  int n_items;
  int next;                  // next unit to hand out
};

struct PromptSeqs {            // the sequences of a call, as the planner or (direct) every CTA reads them
  const int32_t *cu_q, *cu_k, *lens;   // lens: paged (keys of each sequence); else cu_k
  int S, Tq, Tk, tpt, causal;
};

struct PromptParams {
  CUtensorMap tmQ, tmK, tmV;
  __half* out;
  PromptItem* items;
  PromptCtrl* ctrl;
  PromptSeqs seqs;
  int direct;                  // one unit (or one split of it) per CTA, found by the CTA itself: no planner
  int nsplit;                  // direct: CTAs that share the keys of a unit; above 1 they emit partials
  int split_min;               // key blocks that a share holds at least
  float *part_ml, *part_o;     // [CTA][256][2], [CTA][256][128]
  const int32_t* page_table;   // paged cache: (S, table_stride); null = packed keys
  int page_size, table_stride, page_groups;
  int Tq, Hq, Hkv, G, tpt;     // tpt = tokens per 128-row tile
  const uint16_t* v;           // as tmV describes it
  long long v_tok, v_head;     // packed: strides in elements
  float sc;                    // log2(e) / sqrt(128)
  int bf16;
  int32_t* status;
};

struct PromptPlanParams {
  PromptSeqs seqs;
  PromptItem* items;
  PromptCtrl* ctrl;
  int max_items, first_units;
  int32_t* status;
};

// Blocks of keys -> 0 .. 255, growing: exact below 16, then four bits of mantissa.
__device__ __forceinline__ int cost_bin(int nblk) {
  if (nblk < 16) return nblk;
  const int e = 31 - __clz(nblk);
  return min(kPmBins - 1, 16 + (e - 4) * 16 + ((nblk >> (e - 4)) & 15));
}

// One sequence's queries and keys, clamped into their tensors.
__device__ __forceinline__ bool prompt_seq(const PromptSeqs& p, int s, int& q0, int& nq, int& k0, int& nk) {
  bool bad = false;
  auto inside = [&](int v, int hi) {
    if (v < 0 || v > hi) bad = true;
    return min(max(v, 0), hi);
  };
  q0 = inside(p.cu_q[s], p.Tq);
  nq = inside(p.cu_q[s + 1], p.Tq) - q0;
  if (p.lens != nullptr) {
    k0 = s;
    nk = inside(p.lens[s], p.Tk);
  } else {
    k0 = inside(p.cu_k[s], p.Tk);
    nk = inside(p.cu_k[s + 1], p.Tk) - k0;
  }
  if (nq < 0 || nk < 0) bad = true;
  nq = max(nq, 0);
  nk = max(nk, 0);
  return bad;
}

// Tile t of a sequence.
__device__ __forceinline__ PromptItem prompt_item(const PromptSeqs& p, int q0, int nq, int k0, int nk, int t) {
  const int per = 2 * p.tpt;
  PromptItem it;
  it.tok0 = q0 + t * per;
  it.ntok = min(per, nq - t * per);
  it.k0 = k0;
  it.nk = nk;
  it.vis0 = p.causal ? nk - nq + t * per : nk;
  it.h = it.pad[0] = it.pad[1] = 0;
  return it;
}

__global__ void __launch_bounds__(kPmPlanThreads, 1) prompt_plan_kernel(const PromptPlanParams p) {
  __shared__ int s_start[kPmPlanThreads + 1];
  __shared__ int s_q0[kPmPlanThreads], s_nq[kPmPlanThreads], s_k0[kPmPlanThreads], s_nk[kPmPlanThreads];
  __shared__ int s_hist[kPmBins];
  __shared__ int s_warp[32];
  __shared__ int s_total;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_release();
  if (tid < kPmBins) s_hist[tid] = 0;
  if (tid == 0) s_total = 0;
  pdl_wait();
  const PromptSeqs& sq = p.seqs;
  const int per = 2 * sq.tpt;
  bool bad = false;
  // Pass 0 counts the tiles of each cost, pass 1 places them, the costly ones first.
  for (int pass = 0; pass < 2; ++pass) {
    int listed = 0;
    for (int base = 0; base < sq.S; base += kPmPlanThreads) {
      const int s = base + tid;
      int q0 = 0, nq = 0, k0 = 0, nk = 0;
      if (s < sq.S) bad |= prompt_seq(sq, s, q0, nq, k0, nk);
      // (sequences that overlap could come to more tiles than the list has room for: sums stay below 2^31 all the same)
      const int tiles = min((nq + per - 1) / per, p.max_items + 1);
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      __syncthreads();                          // the chunk before is done with the shared arrays
      if (lane == 31) s_warp[warp] = incl;
      __syncthreads();
      if (warp == 0) {
        int w = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, w, o);
          if (lane >= o) w += v;
        }
        s_warp[lane] = w;
      }
      __syncthreads();
      incl += warp > 0 ? s_warp[warp - 1] : 0;
      s_start[tid] = incl - tiles;
      s_q0[tid] = q0;
      s_nq[tid] = nq;
      s_k0[tid] = k0;
      s_nk[tid] = nk;
      if (tid == kPmPlanThreads - 1) s_start[kPmPlanThreads] = incl;
      __syncthreads();
      const int room = p.max_items - listed, total = min(s_start[kPmPlanThreads], room);
      if (s_start[kPmPlanThreads] > room) bad = true;
      listed += total;
      for (int i = tid; i < total; i += kPmPlanThreads) {
        int lo = 0, hi = kPmPlanThreads;        // the last sequence whose first tile is at or before i
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (s_start[mid] <= i) lo = mid; else hi = mid;
        }
        const int t = i - s_start[lo];
        const PromptItem it = prompt_item(sq, s_q0[lo], s_nq[lo], s_k0[lo], s_nk[lo], t);
        const int seen = min(it.nk, max(0, it.vis0 + it.ntok));
        const int bin = kPmBins - 1 - cost_bin((seen + kPmBK - 1) / kPmBK);
        if (pass == 0) {
          atomicAdd(&s_hist[bin], 1);
        } else {
          p.items[atomicAdd(&s_hist[bin], 1)] = it;
        }
      }
    }
    __syncthreads();
    if (pass == 0) {
      if (warp == 0) {                          // exclusive scan of the 256 bins by one warp
        int v[kPmBins / 32], sum = 0;
#pragma unroll
        for (int i = 0; i < kPmBins / 32; ++i) {
          v[i] = s_hist[lane * (kPmBins / 32) + i];
          sum += v[i];
        }
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += x;
        }
        int at = incl - sum;
#pragma unroll
        for (int i = 0; i < kPmBins / 32; ++i) {
          s_hist[lane * (kPmBins / 32) + i] = at;
          at += v[i];
        }
        if (lane == 31) s_total = at;
      }
      __syncthreads();
    }
  }
  if (tid == 0) {
    p.ctrl->n_items = s_total;
    p.ctrl->next = p.first_units;
  }
  if (bad) report(p.status, kStatusBadIndex);
}

__device__ __forceinline__ float pm_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void pm_store32(void* dst, const uint32_t (&w)[8]) {      // dst 32-byte aligned
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// 16 lanes x 64 columns of tensor memory: r[4 i .. 4 i + 1] are columns 8 i + 2 (lane % 4) + {0, 1} of row lane / 4, the other two
// those of row lane / 4 + 8.
__device__ __forceinline__ void pm_tmem_ld_16x64(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(taddr));
}
// Four lanes hold four words each: word e of lane l and word l of lane e change places.
__device__ __forceinline__ void pm_quad_transpose(uint32_t (&v)[4], int lane) {
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k & o) continue;
      const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? v[k] : v[k + o], o);
      if (up) v[k] = got; else v[k + o] = got;
    }
  }
}
__device__ __forceinline__ float pm_max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// tcgen05.mma and commit executed by the lanes with `lead` set (one of them) in code that the whole warp runs.
__device__ __forceinline__ void pm_mma_ss(uint32_t lead, uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      ".reg .b64 da, db;\n"
      "setp.ne.b32 p, %6, 0;\n"
      "setp.ne.b32 q, %7, 0;\n"
      "mov.b64 da, {%1, %2};\n"
      "mov.b64 db, {%3, %4};\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n"
      "}\n" ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void pm_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      ".reg .b64 db;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "setp.ne.b32 q, %6, 0;\n"
      "mov.b64 db, {%2, %3};\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n"
      "}\n" ::"r"(d), "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void pm_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.b32 q, %1, 0;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(smem_u32(bar)), "r"(lead)
      : "memory");
}

struct PromptUnit {          // what warp 8 hands to the others
  PromptItem it;
  int h;                     // kv head; -1: no more units
  int j0, na, nb;            // first key block of this CTA's share, and how many of it tiles A and B have to see
  int parts;                 // CTAs that share the unit
  int twin;                  // both tiles hold the same rows, and take the blocks j0, j0 + 2, ... and j0 + 1, j0 + 3, ...
};

// Key blocks that 128-row tile t of an item has to see, and how many tokens it holds.
__device__ __forceinline__ int tile_blocks(const PromptItem& it, int t, int tpt) {
  const int tok = min(it.ntok, (t + 1) * tpt);
  if (tok <= t * tpt) return 0;
  const int seen = min(it.nk, max(0, it.vis0 + tok));
  return (seen + kPmBK - 1) / kPmBK;
}

// Shared units of one 128-row tile: tile B takes every other block of the same rows (one tile alone leaves the tensor pipe
// idle during its softmax and the other way round), and the merge joins the two like shares of their own.  Both read one Q
// tile; the other's place is a sixth slot of the ring.  (17 tokens over 60001 keys: 62.6 us with one tile, 57.0 with two; the
// keys alone take 38 us to read.  Asking for later blocks into L2 ahead of the ring made it 64 to 71.)
__device__ __forceinline__ bool prompt_twin(const PromptItem& it, int tpt, int parts) { return parts > 1 && it.ntok <= tpt; }

// This CTA's share of a unit's key blocks: all of them, or part `sp` of `nsplit` equal ones of at least split_min blocks.
__device__ __forceinline__ int prompt_parts(int nblk, int nsplit, int split_min) { return max(1, min(nsplit, nblk / split_min)); }

__device__ __forceinline__ void prompt_share(PromptUnit& u, int tpt, int nsplit, int split_min, int sp) {
  const int na = tile_blocks(u.it, 0, tpt), nb = tile_blocks(u.it, 1, tpt), nblk = max(na, nb);
  const int parts = prompt_parts(nblk, nsplit, split_min);
  u.parts = parts;
  if (sp >= parts) u.h = -1;
  const int j0 = sp < parts ? (int)((long long)nblk * sp / parts) : nblk, j1 = sp < parts ? (int)((long long)nblk * (sp + 1) / parts) : nblk;
  u.j0 = j0;
  u.na = max(0, min(na, j1) - j0);
  u.nb = max(0, min(nb, j1) - j0);
  u.twin = prompt_twin(u.it, tpt, parts);
  if (u.twin) {
    u.nb = u.na / 2;
    u.na -= u.nb;
  }
}

constexpr int kPmBars = 2 * kPmTwinSlots + 2 * kPmSched + 2 + 2 + 2 + 2 + 2 + 2 + 2;   // (an even number: what follows is 16-byte aligned)
constexpr int kPmSpecial = 4;                    // units that a flag of theirs has to outlive, and more
constexpr int kPmSmem =
    2 * kPmTile + kPmSlots * kPmTile + kPmBars * 8 + kPmSched * (int)sizeof(PromptUnit) + 16 + 2 * kPmSpecial * 4 + 1024;
static_assert(kPmSmem <= 232448, "shared memory of one CTA");

// NaN and infinite, in either 16-bit type.
template <bool BF>
__device__ __forceinline__ bool pm_special(uint32_t h) { return BF ? (h & 0x7f80u) == 0x7f80u : (h & 0x7c00u) == 0x7c00u; }
template <bool BF>
__device__ __forceinline__ float pm_float(uint16_t h) {
  return BF ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
}

template <bool BF>
__device__ __forceinline__ void pm_times_zero(uint32_t& acc, uint32_t x) {
  if (BF) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(0u));
  else asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(x), "r"(0u));
}

// Adds the NaN and infinite entries of V at keys [k0, k1) of a unit's sequence to a row that sees them all: to its result, or to its share.
template <bool BF, bool PART>
__device__ __forceinline__ void prompt_add_special(const PromptParams& p, const PromptItem& it, int h, int k0, int k1, void* row) {
#pragma unroll 1
  for (int x = k0; x < k1; ++x) {
    const uint16_t* v = nullptr;
    if (p.page_table == nullptr) {
      v = p.v + (long long)(it.k0 + x) * p.v_tok + (long long)h * p.v_head;
    } else {
      const int id = x / p.page_size < p.table_stride ? p.page_table[(size_t)it.k0 * p.table_stride + x / p.page_size] : -1;
      if (id >= 0 && id < p.page_groups / p.Hkv) v = p.v + (((size_t)id * p.Hkv + h) * p.page_size + x % p.page_size) * kPmD;
    }
    if (v == nullptr) continue;
#pragma unroll 1
    for (int c = 0; c < kPmD; ++c) {
      const uint16_t e = v[c];
      if (!pm_special<BF>(e)) continue;
      if (PART) {
        static_cast<float*>(row)[c] += pm_float<BF>(e);
      } else {
        uint16_t* o = static_cast<uint16_t*>(row) + c;
        const float sum = pm_float<BF>(*o) + pm_float<BF>(e);
        *o = (uint16_t)pack2(sum, 0.f, BF);
      }
    }
  }
}

// SPLIT: CTAs share units' keys and emit partials (always direct: one unit each).  An instance of its own, so that the
// loops of the others hold nothing of it.
template <bool BF, bool SPLIT>
__global__ void __launch_bounds__(kPmThreads, 1) prompt_kernel(const __grid_constant__ PromptParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                    // [2 tiles][32 KiB]
  uint8_t* sKV = sQ + 2 * kPmTile;                       // [slots][32 KiB]
  uint64_t* full = reinterpret_cast<uint64_t*>(sKV + kPmSlots * kPmTile);   // K or V tile landed (TMA bytes)
  uint64_t* empty = full + kPmTwinSlots;                 // consumed by both tiles' products   (MMA commit)
  uint64_t* sched_full = empty + kPmTwinSlots;           // unit written                       (warp 8)
  uint64_t* sched_empty = sched_full + kPmSched;         // unit read by everybody             (11 warps)
  uint64_t* q_full = sched_empty + kPmSched;             // [tile] Q tile landed               (TMA bytes)
  uint64_t* q_empty = q_full + 2;                        // [tile] last Q.K^T of a unit done   (MMA commit)
  uint64_t* s_full = q_empty + 2;                        // [tile] scores ready                (MMA commit)
  uint64_t* p_part = s_full + 2;                         // [tile] P of the first 96 keys in tensor memory, V looked at (6 warps)
  uint64_t* p_full = p_part + 2;                         // [tile] all of P                    (4 warps)
  uint64_t* o_full = p_full + 2;                         // [tile] last P.V of a unit done     (MMA commit)
  uint64_t* drain = o_full + 2;                          // every product done, after a timeout
  PromptUnit* units = reinterpret_cast<PromptUnit*>(sKV + kPmSlots * kPmTile + kPmBars * 8);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(units + kPmSched);
  uint32_t* special = tmem_slot + 4;                     // [unit % 4][warp 10, 11]: 1 + the unit, if it cleared entries of V

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int s = 0; s < kPmTwinSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < kPmSched; ++s) {
      mbar_init(&sched_full[s], 1);
      mbar_init(&sched_empty[s], 11);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_part[t], 6);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < 2 * kPmSpecial; ++i) special[i] = 0u;
    fence_mbar_init();
  }
  if (warp == 9) tmem_alloc(tmem_slot, kPmCols);
  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&p.tmQ);
    tma_prefetch_desc(&p.tmK);
    tma_prefetch_desc(&p.tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();
  if (p.direct) {
    // This CTA's tile: a scan over the sequences' tile counts by the whole block.  (One CTA of a planner would cost a
    // launch and its own time before any of these begins.)
    const int sp = blockIdx.x % p.nsplit, u = blockIdx.x / p.nsplit, want = u / p.Hkv;
    int* s_warp = reinterpret_cast<int*>(units + 1);
    if (tid == 0) units[0].h = -1;
    int before = 0;
    bool bad = false;
    // (CTA 0 looks at all of them, so that a list that does not ascend is reported wherever it does not)
    for (int base = 0; base < p.seqs.S && (before <= want || blockIdx.x == 0); base += kPmThreads) {
      int q0 = 0, nq = 0, k0 = 0, nk = 0;
      if (base + tid < p.seqs.S) bad |= prompt_seq(p.seqs, base + tid, q0, nq, k0, nk);
      const int tiles = (nq + 2 * p.tpt - 1) / (2 * p.tpt);
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) s_warp[warp] = incl;
      __syncthreads();
      int total = 0;
#pragma unroll
      for (int w = 0; w < kPmThreads / 32; ++w) {
        const int v = s_warp[w];
        if (w < warp) incl += v;
        total += v;
      }
      const int t = want - (before + incl - tiles);
      if (t >= 0 && t < tiles) {
        PromptUnit un;
        un.it = prompt_item(p.seqs, q0, nq, k0, nk, t);
        un.h = un.it.h = u % p.Hkv;
        prompt_share(un, p.tpt, p.nsplit, p.split_min, sp);
        units[0] = un;
        if (p.nsplit > 1 && sp == 0) p.items[u] = un.it;
      }
      before += total;
      __syncthreads();
    }
    if (bad) report(p.status, kStatusBadIndex);
    if (tid == 0 && p.nsplit > 1 && sp == 0 && units[0].h < 0) p.items[u].ntok = 0;
    __syncthreads();
  }

  // The registers of a block are fixed at its launch (384 x 168 = 64512): 256 x 216 + 128 x 72 is the same number.  Each
  // side changes its share as the first thing in its own branch; the branches meet again only at the common exit.
  bool timed_out = false;
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp == 8) {
    // ------------------------------------------------------------------------------ units and TMA producer
    if (lane == 0) {
      const int n_units = p.direct ? 0 : p.ctrl->n_items * p.Hkv;
      const uint32_t q_bytes = (uint32_t)(p.tpt * p.G) * 128u * 2u;
      const int pool_pages = p.page_groups / p.Hkv;
      int u = blockIdx.x;
      uint32_t ring = 0, issued_q[2] = {0, 0}, slots = kPmSlots;
      for (uint32_t n = 0;; ++n) {
        const int sl = n % kPmSched;
        if (n >= kPmSched && !mbar_wait(&sched_empty[sl], (n / kPmSched - 1) & 1)) { timed_out = true; break; }
        PromptUnit un;
        un.h = -1;
        if (p.direct) {
          if (n == 0) un = units[0];                       // found above; there is no second
        } else if (u < n_units) {
          un.it = p.items[u / p.Hkv];
          un.h = u % p.Hkv;
          prompt_share(un, p.tpt, 1, 1, 0);
        }
        units[sl] = un;
        mbar_arrive(&sched_full[sl]);
        if (un.h < 0) break;
        const bool twin = SPLIT && un.twin;
        if (twin) slots = kPmTwinSlots;
        uint8_t* ring0 = twin ? sKV - kPmTile : sKV;
        const int nt0 = un.na, nt1 = un.nb, nblk = twin ? nt0 + nt1 : max(nt0, nt1);
        // Paged keys: a block is two 64-key boxes, each inside one page; page ids are read one block ahead, and positions
        // are kept by counting (a division for each took this thread longer than a block).
        int pg = 0, off = 0, id[2] = {-1, -1}, next_id[2] = {-1, -1}, y[2] = {0, 0}, next_y[2] = {0, 0};
        const int32_t* row = nullptr;
        auto look = [&]() {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            next_id[b] = b == 1 && off != 0 ? next_id[0] : pg < p.table_stride ? row[pg] : -1;
            next_y[b] = off;
            off += 64;
            if (off == p.page_size) {
              off = 0;
              ++pg;
            }
          }
        };
        if (p.page_table != nullptr && nblk > 0) {
          row = p.page_table + (size_t)un.it.k0 * p.table_stride;
          pg = un.j0 * kPmBK / p.page_size;
          off = un.j0 * kPmBK - pg * p.page_size;
          look();
        }
        for (int i = 0; i < 2 * nblk; ++i, ++ring) {
          if (p.page_table != nullptr && (i & 1) == 0) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              id[b] = next_id[b];
              y[b] = next_y[b];
            }
            if (i + 2 < 2 * nblk) look();
          }
          const int s = ring % slots;
          if (ring >= slots && !mbar_wait(&empty[s], (ring / slots - 1) & 1)) { timed_out = true; break; }
          const CUtensorMap* tm = (i & 1) ? &p.tmV : &p.tmK;
          uint8_t* dst = ring0 + s * kPmTile;
          const int kb = (un.j0 + (i >> 1)) * kPmBK;
          mbar_expect_tx(&full[s], kPmTile);
          if (p.page_table == nullptr) {
            tma_load_3d(dst, tm, 0, un.h, un.it.k0 + kb, &full[s]);
            tma_load_3d(dst + kPmHalf, tm, 64, un.h, un.it.k0 + kb, &full[s]);
          } else {
#pragma unroll
            for (int b = 0; b < 2; ++b) {                  // a page id outside the pool reads zeros
              const int z = id[b] >= 0 && id[b] < pool_pages ? id[b] * p.Hkv + un.h : p.page_groups;
              tma_load_3d(dst + b * (kPmHalf / 2), tm, 0, y[b], z, &full[s]);
              tma_load_3d(dst + kPmHalf + b * (kPmHalf / 2), tm, 64, y[b], z, &full[s]);
            }
          }
          if (i == 0) {
            // the queries behind the first keys: the slot of K_0 is free earlier than the Q tiles of the unit before
            for (int t = 0; t < 2 && !timed_out; ++t) {
              if ((t == 0 ? nt0 : twin ? 0 : nt1) == 0) continue;
              if (issued_q[t] > 0 && !mbar_wait(&q_empty[t], (issued_q[t] - 1) & 1)) { timed_out = true; break; }
              ++issued_q[t];
              mbar_expect_tx(&q_full[t], q_bytes);
              tma_load_3d(sQ + t * kPmTile, &p.tmQ, 0, un.h * p.G, un.it.tok0 + t * p.tpt, &q_full[t]);
              tma_load_3d(sQ + t * kPmTile + kPmHalf, &p.tmQ, 64, un.h * p.G, un.it.tok0 + t * p.tpt, &q_full[t]);
            }
            if (timed_out) { ++ring; break; }
          }
        }
        if (timed_out) break;
        if (!p.direct) u = atomicAdd(&p.ctrl->next, 1);
      }
      // no load outlives the CTA: the newest tile of every slot has landed before this warp goes to the exit
      for (uint32_t i = ring > slots ? ring - slots : 0; i < ring; ++i) mbar_wait(&full[i % slots], (i / slots) & 1);
      for (int t = 0; t < 2; ++t)
        if (issued_q[t] > 0) mbar_wait(&q_full[t], (issued_q[t] - 1) & 1);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------------------------ every tcgen05.mma
    // The whole warp runs this code and the instructions themselves are predicated: the descriptors then stay in
    // uniform registers.  (Inside a one-lane branch every one of them was moved there first, at 75 to 85 issue cycles per
    // instruction beside the softmax warps of the same scheduler; one M128 N128 K16 takes the pipe 64.)
    uint32_t lead;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(lead));
    const uint32_t idesc_qk = umma_idesc_16(128, kPmBK, 0, BF), idesc_pv = umma_idesc_16(128, kPmD, 1, BF);
    const uint32_t hi_k = (uint32_t)(umma_desc_sw128(0) >> 32), lo_k = (uint32_t)umma_desc_sw128(0);
    const uint32_t q_lo = lo_k + (smem_u32(sQ) >> 4), k_lo = lo_k + (smem_u32(sKV) >> 4);
    const uint32_t hi_v = (uint32_t)(umma_desc_sw128_mn(0, kPmHalf, 1024) >> 32);
    const uint32_t v_lo = (uint32_t)umma_desc_sw128_mn(0, kPmHalf, 1024) + (smem_u32(sKV) >> 4);
    uint32_t ring = 0, n_q[2] = {0, 0}, n_p[2] = {0, 0};
    auto qk = [&](int t, uint32_t slot) {
      const uint32_t d = tmem_base + kPmColS + t * 128, a = q_lo + t * (kPmTile >> 4), b = k_lo + slot * (kPmTile >> 4);
#pragma unroll
      for (int k = 0; k < 8; ++k)
        pm_mma_ss(lead, d, a + (k >> 2) * (kPmHalf >> 4) + (k & 3) * 2, hi_k, b + (k >> 2) * (kPmHalf >> 4) + (k & 3) * 2, hi_k,
                  idesc_qk, k > 0 ? 1u : 0u);
      pm_commit(lead, &s_full[t]);
    };
    for (uint32_t n = 0;; ++n) {
      const int sl = n % kPmSched;
      if (!mbar_wait(&sched_full[sl], (n / kPmSched) & 1)) timed_out = true;
      // a wait that ran out for one lane ends the unit for it, and here the loop for all
      if (__any_sync(0xffffffffu, timed_out)) { timed_out = true; break; }
      const int h = __shfl_sync(0xffffffffu, units[sl].h, 0);
      const int nt0 = __shfl_sync(0xffffffffu, units[sl].na, 0), nt1 = __shfl_sync(0xffffffffu, units[sl].nb, 0);
      const bool twin = SPLIT && __shfl_sync(0xffffffffu, units[sl].twin, 0) != 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sched_empty[sl]);
      if (h < 0) break;
      const int nblk = max(nt0, nt1);
      if (nblk == 0) continue;
      auto wait_tile = [&](uint32_t i) {
        if (!mbar_wait(&full[i % kPmSlots], (i / kPmSlots) & 1)) timed_out = true;
      };
      if constexpr (SPLIT) {
        if (twin) {                                        // block j belongs to tile j & 1 alone
          const int all = nt0 + nt1;
          const uint32_t k6 = k_lo - (kPmTile >> 4), v6 = v_lo - (kPmTile >> 4);       // six slots, the second Q tile's place among them
          auto landed = [&](uint32_t i) {
            if (!mbar_wait(&full[i % kPmTwinSlots], (i / kPmTwinSlots) & 1)) timed_out = true;
          };
          auto qk_twin = [&](int t, uint32_t slot) {
            const uint32_t d = tmem_base + kPmColS + t * 128, b = k6 + slot * (kPmTile >> 4);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              pm_mma_ss(lead, d, q_lo + (k >> 2) * (kPmHalf >> 4) + (k & 3) * 2, hi_k, b + (k >> 2) * (kPmHalf >> 4) + (k & 3) * 2, hi_k,
                        idesc_qk, k > 0 ? 1u : 0u);
            pm_commit(lead, &s_full[t]);
            pm_commit(lead, &empty[slot]);
          };
          if (!mbar_wait(&q_full[0], 0)) timed_out = true;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= all || timed_out) continue;
            landed(2 * t);
            if (timed_out) continue;
            tc_fence_after();
            qk_twin(t, 2 * t);
          }
          for (int j0 = 0; j0 < all && !timed_out; j0 += 2) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int j = j0 + t;
              if (j >= all || timed_out) continue;
              const uint32_t iv = 2 * j + 1, ik = iv + 3;
              landed(iv);
              const uint32_t o = tmem_base + kPmColO + t * 128, a = tmem_base + kPmColS + t * 128;
              const uint32_t b = v6 + (iv % kPmTwinSlots) * (kPmTile >> 4);
              if (timed_out || !mbar_wait(&p_part[t], n_p[t] & 1)) { timed_out = true; continue; }
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < 6; ++k) pm_mma_ts(lead, o, a + k * 8, b + k * (2048 >> 4), hi_v, idesc_pv, (j0 > 0 || k > 0) ? 1u : 0u);
              if (!mbar_wait(&p_full[t], n_p[t]++ & 1)) { timed_out = true; continue; }
              tc_fence_after();
#pragma unroll
              for (int k = 6; k < 8; ++k) pm_mma_ts(lead, o, a + k * 8, b + k * (2048 >> 4), hi_v, idesc_pv, 1u);
              if (j + 2 >= all) {
                pm_commit(lead, &o_full[t]);
              } else {
                landed(ik);
                if (timed_out) continue;
                qk_twin(t, ik % kPmTwinSlots);
              }
              pm_commit(lead, &empty[iv % kPmTwinSlots]);
            }
          }
          continue;                                        // (a CTA has one such unit)
        }
      }
      wait_tile(ring);                                     // K_0
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int nt = t == 0 ? nt0 : nt1;
        if (nt == 0 || timed_out) continue;
        if (!mbar_wait(&q_full[t], n_q[t]++ & 1)) { timed_out = true; continue; }
        tc_fence_after();
        qk(t, ring % kPmSlots);
        if (nt == 1) pm_commit(lead, &q_empty[t]);
      }
      if (!timed_out) pm_commit(lead, &empty[ring % kPmSlots]);
      for (int j = 0; j < nblk && !timed_out; ++j) {
        const uint32_t iv = ring + 2 * j + 1, ik = iv + 1;
        wait_tile(iv);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int nt = t == 0 ? nt0 : nt1;
          if (j >= nt || timed_out) continue;
          const uint32_t o = tmem_base + kPmColO + t * 128, a = tmem_base + kPmColS + t * 128;
          const uint32_t b = v_lo + (iv % kPmSlots) * (kPmTile >> 4);
          if (!mbar_wait(&p_part[t], n_p[t] & 1)) { timed_out = true; continue; }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < 6; ++k) pm_mma_ts(lead, o, a + k * 8, b + k * (2048 >> 4), hi_v, idesc_pv, (j > 0 || k > 0) ? 1u : 0u);
          if (!mbar_wait(&p_full[t], n_p[t]++ & 1)) { timed_out = true; continue; }
          tc_fence_after();
#pragma unroll
          for (int k = 6; k < 8; ++k) pm_mma_ts(lead, o, a + k * 8, b + k * (2048 >> 4), hi_v, idesc_pv, 1u);
          if (j + 1 == nt) {
            pm_commit(lead, &o_full[t]);
          } else {
            wait_tile(ik);
            if (timed_out) continue;
            qk(t, ik % kPmSlots);
            if (j + 2 == nt) pm_commit(lead, &q_empty[t]);
          }
        }
        if (timed_out) break;
        pm_commit(lead, &empty[iv % kPmSlots]);
        if (j + 1 < nblk) pm_commit(lead, &empty[ik % kPmSlots]);
      }
      ring += 2 * nblk;
    }
    if (timed_out) {                                       // the products in flight end before tensor memory is freed
      pm_commit(lead, drain);
      mbar_wait(drain, 0);
    }
  } else {
    // ------------------------------------------------------------------------------ NaN and infinities in V
    const int mine = warp - 10;                            // the two share a block's rows
    uint32_t ring = 0, n_p[2] = {0, 0};
    for (uint32_t n = 0; !timed_out; ++n) {
      const int sl = n % kPmSched;
      if (!__all_sync(0xffffffffu, mbar_wait(&sched_full[sl], (n / kPmSched) & 1))) { timed_out = true; break; }
      const int h = units[sl].h, j0 = units[sl].j0, na = units[sl].na, nb = units[sl].nb, nk = units[sl].it.nk, vis0 = units[sl].it.vis0;
      const bool twin = SPLIT && units[sl].twin;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sched_empty[sl]);
      if (h < 0) break;
      const int nblk = twin ? na + nb : max(na, nb);
      const int vis_all = min(nk, max(0, vis0 + 1));       // keys that the unit's first token sees
      for (int j = 0; j < nblk && !timed_out; ++j) {
        const int kb = (j0 + j) * kPmBK, r0 = max(0, vis_all - kb), r1 = min(kPmBK, nk - kb);
        if (r0 < r1) {
          const uint32_t iv = ring + 2 * j + 1, slots = twin ? kPmTwinSlots : kPmSlots;
          if (!__all_sync(0xffffffffu, mbar_wait(&full[iv % slots], (iv / slots) & 1))) { timed_out = true; break; }
          uint8_t* v = sKV + (iv % slots) * kPmTile - (twin ? kPmTile : 0);
          // 0 x + 0 is NaN where x is NaN or infinite, and 0 or -0 elsewhere: one packed product for two entries
          uint32_t acc[4] = {0u, 0u, 0u, 0u};
          const uint8_t* col = v + ((lane & 15) >> 3) * kPmHalf;
          const int first = r0 + 2 * mine + (lane >> 4);
#pragma unroll 8
          for (int r = first; r < r1; r += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(col + swz128(r, lane & 7));
            pm_times_zero<BF>(acc[0], x.x);
            pm_times_zero<BF>(acc[1], x.y);
            pm_times_zero<BF>(acc[2], x.z);
            pm_times_zero<BF>(acc[3], x.w);
          }
          if (__any_sync(0xffffffffu, ((acc[0] | acc[1] | acc[2] | acc[3]) & 0x7fff7fffu) != 0u)) {
            if (lane == 0) *reinterpret_cast<volatile uint32_t*>(special + (n % kPmSpecial) * 2 + mine) = n + 1;
#pragma unroll 1
            for (int r = first; r < r1; r += 4)
#pragma unroll 1
              for (int c = 0; c < 8; ++c) {
                uint16_t* x = reinterpret_cast<uint16_t*>(v + ((lane & 15) >> 3) * kPmHalf + swz128(r, lane & 7)) + c;
                if (pm_special<BF>(*x)) *x = 0;
              }
          }
          fence_proxy_async();
          __syncwarp();
        }
        // each tile that the block belongs to; an arrival counts for the phase after the one that is complete
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (twin ? (j & 1) != t : j >= (t == 0 ? na : nb)) continue;
          if (n_p[t] > 0 && !__all_sync(0xffffffffu, mbar_wait(&p_part[t], (n_p[t] - 1) & 1))) { timed_out = true; continue; }
          if (lane == 0) mbar_arrive(&p_part[t]);
          ++n_p[t];
        }
      }
      ring += 2 * nblk;
    }
    if (warp == 10) {
      // ------------------------------------------------------------------------------ rows outside every sequence
      const int lo = min(max(p.seqs.cu_q[0], 0), p.Tq);
      const int hi = max(lo, min(max(p.seqs.cu_q[p.seqs.S], 0), p.Tq));
      const size_t row16 = (size_t)p.Hq * (kPmD / 8);       // 16-byte chunks of one token's row
      const size_t n = (size_t)(lo + (p.Tq - hi)) * row16;
      for (size_t e = (size_t)blockIdx.x * 32 + lane; e < n; e += (size_t)gridDim.x * 32) {
        const size_t at = e < (size_t)lo * row16 ? e : e - (size_t)lo * row16 + (size_t)hi * row16;
        reinterpret_cast<uint4*>(p.out)[at] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------------------------ softmax
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;               // row of the tile = tensor-memory lane
    const uint32_t lane_base = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tS = lane_base + kPmColS + t * 128, tO = lane_base + kPmColO + t * 128;
    const int tok = row / p.G;                            // token of the row inside its 128-row tile
    const int g = row - tok * p.G;
    uint32_t ring = 0, n_s = 0, n_o = 0;
    for (uint32_t n = 0; !timed_out; ++n) {
      const int sl = n % kPmSched;
      if (!__all_sync(0xffffffffu, mbar_wait(&sched_full[sl], (n / kPmSched) & 1))) { timed_out = true; break; }
      const PromptItem it = units[sl].it;
      const int h = units[sl].h, j0 = units[sl].j0, na = units[sl].na, nb = units[sl].nb;
      const bool twin = SPLIT && units[sl].twin, part = SPLIT && units[sl].parts > 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sched_empty[sl]);
      if (h < 0) break;
      const int nblk = twin ? na + nb : max(na, nb), mine = t == 0 ? na : nb;
      const int tile0 = twin ? 0 : t * p.tpt;             // the tile's first token inside the item
      const int tk = tile0 + tok;                         // that of the row
      const bool valid = tok < p.tpt && tk < it.ntok;
      const int vis = valid ? min(it.nk, max(0, it.vis0 + tk + 1)) : 0;
      // keys that every row of this tile sees (its first token's)
      const int vis_all = min(it.nk, max(0, it.vis0 + tile0 + 1));

      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < mine; ++j) {
        if (!__all_sync(0xffffffffu, mbar_wait(&s_full[t], n_s++ & 1))) { timed_out = true; break; }
        tc_fence_after();
        const int blk = twin ? 2 * j + t : j, kb = (j0 + blk) * kPmBK;
        uint32_t sv[128];
        tmem_ld32(tS, *reinterpret_cast<uint32_t(*)[32]>(sv));
        tmem_ld32(tS + 32, *reinterpret_cast<uint32_t(*)[32]>(sv + 32));
        tmem_ld32(tS + 64, *reinterpret_cast<uint32_t(*)[32]>(sv + 64));
        tmem_ld32(tS + 96, *reinterpret_cast<uint32_t(*)[32]>(sv + 96));
        tmem_ld_wait();
        const bool edge = kb + kPmBK > vis_all;
        if (edge) {
          // a block that the mask or the end of the keys cuts: hidden scores become -inf whatever they were
          const int lim = vis - kb;
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (i >= lim) sv[i] = 0xff800000u;
        }
        // P = 2^(score * scale - m) (exactly 0 for a hidden key: -inf stays -inf) and its sum, 32 keys at a time
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[16];
        auto chunk = [&](int c, float mu, float (&add)[4]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float a = pm_exp2(fmaf(__uint_as_float(sv[c * 32 + 2 * i]), p.sc, -mu));
            const float b = pm_exp2(fmaf(__uint_as_float(sv[c * 32 + 2 * i + 1]), p.sc, -mu));
            add[(i & 1) * 2] += a;
            add[(i & 1) * 2 + 1] += b;
            pk[i] = BF ? pack_bf16x2(a, b) : pack_half2(a, b);
          }
        };
        // The first 32 keys go by the maximum of the blocks before: their exponentials need not wait for this block's maximum.
        // Only where a row's maximum has grown by more than 2^8 (or at a row's first block) they are done again.
        float mu = (m == -INFINITY) ? 0.f : m;
        chunk(0, mu, sum);
        float mx[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) mx[i] = fmaxf(__uint_as_float(sv[i]), __uint_as_float(sv[i + 8]));
#pragma unroll
        for (int i = 16; i < 128; i += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k) mx[k] = pm_max3(mx[k], __uint_as_float(sv[i + k]), __uint_as_float(sv[i + k + 8]));
        mx[0] = pm_max3(mx[0], mx[1], mx[2]);
        mx[3] = pm_max3(mx[3], mx[4], mx[5]);
        mx[0] = pm_max3(mx[0], mx[6], mx[7]);
        const float bm = fmaxf(mx[0], mx[3]) * p.sc;         // the scale is positive: max commutes with it
        const bool grown = bm > m + kPmLazy;                 // (m is -inf before a row's first visible key)
        if (__any_sync(0xffffffffu, grown)) {
          float alpha = 1.f;
          if (grown) {
            if (m != -INFINITY) alpha = pm_exp2(m - bm);
            m = bm;
          }
          l *= alpha;
          if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(tO + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(tO + c * 16, o);
            }
          }
          mu = (m == -INFINITY) ? 0.f : m;
          sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
          chunk(0, mu, sum);
        }
        if (kb + kPmBK > it.nk && (twin || t == 0 || j >= na)) {
          // rows of V past the sequence's end are cleared by the tile whose product comes first
          const uint32_t iv = ring + 2 * blk + 1, slots = twin ? kPmTwinSlots : kPmSlots;
          if (!__all_sync(0xffffffffu, mbar_wait(&full[iv % slots], (iv / slots) & 1))) { timed_out = true; break; }
          uint8_t* v = sKV + (iv % slots) * kPmTile - (twin ? kPmTile : 0);
          const int r0 = it.nk - kb;
          for (int e = row; e < (kPmBK - r0) * 16; e += 128) {
            const int r = r0 + (e >> 4), c = e & 15;
            *reinterpret_cast<uint4*>(v + (c >> 3) * kPmHalf + swz128(r, c & 7)) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async();
        }
        tmem_st16(tS, pk);
#pragma unroll
        for (int c = 1; c < 4; ++c) {
          chunk(c, mu, sum);
          tmem_st16(tS + c * 16, pk);
          if (c == 2) {                                   // the product of the first 96 keys may begin
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_part[t]);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
      if (timed_out) break;
      ring += 2 * nblk;

      // ---- the row's result
      if (mine > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(&o_full[t], n_o++ & 1))) { timed_out = true; break; }
        tc_fence_after();
      }
      // entries of V that were cleared, at keys that this row sees: those behind the first that not all rows of the unit see
      const volatile uint32_t* sp = special + (n % kPmSpecial) * 2;
      const bool add = sp[0] == n + 1 || sp[1] == n + 1;
      const int add0 = max(min(it.nk, max(0, it.vis0 + 1)), j0 * kPmBK), add1 = min(vis, (j0 + nblk) * kPmBK);
      if (part) {
        // a share of the keys: the row's maximum, sum and unnormalised output, for the merge
        const size_t at = (size_t)blockIdx.x * 256 + t * 128 + row;
        if (valid) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mine > 0 ? m : -INFINITY, l);
        if (mine > 0) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_ld_wait();
            if (!valid) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = o[8 * i + e];
              pm_store32(p.part_o + at * kPmD + c * 32 + i * 8, w);
            }
          }
        }
        if (add && valid && mine > 0) prompt_add_special<BF, true>(p, it, h, add0, add1, p.part_o + at * kPmD);
        tc_fence_before();
        continue;
      }
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;           // 0: the row saw no key (a NaN stays one)
      const unsigned long long dst =
          valid ? (unsigned long long)(p.out + ((size_t)(it.tok0 + tk) * p.Hq + (size_t)h * p.G + g) * kPmD) : 0ull;
      // Whole 128-byte lines: a quad of lanes has 64 columns of a row (8 rows a store).  With a row to each thread (32 sectors of as
      // many lines a store) the load/store unit was busy with a unit's stores for 2 us, now for 1.4 (24 ragged prompts 244.6 ->
      // 238.8 us).  Loading more of O at a time spills.
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int la = half * 16 + (lane >> 2);
        const float ia = __shfl_sync(0xffffffffu, inv, la), ib = __shfl_sync(0xffffffffu, inv, la + 8);
        const unsigned long long da = __shfl_sync(0xffffffffu, dst, la), db = __shfl_sync(0xffffffffu, dst, la + 8);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t o[32], wa[8], wb[8];
          if (mine > 0) {
            pm_tmem_ld_16x64(tO + ((uint32_t)(half * 16) << 16) + c * 64, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t ta[4], tb[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = 4 * (2 * e + x);
              ta[e] = mine > 0 && ia != 0.f ? pack2(__uint_as_float(o[i]) * ia, __uint_as_float(o[i + 1]) * ia, BF) : 0u;
              tb[e] = mine > 0 && ib != 0.f ? pack2(__uint_as_float(o[i + 2]) * ib, __uint_as_float(o[i + 3]) * ib, BF) : 0u;
            }
            pm_quad_transpose(ta, lane);
            pm_quad_transpose(tb, lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              wa[4 * x + e] = ta[e];
              wb[4 * x + e] = tb[e];
            }
          }
          const int at = (c * 64 + (lane & 3) * 16) * 2;
          if (da != 0ull) pm_store32(reinterpret_cast<uint8_t*>(da) + at, wa);
          if (db != 0ull) pm_store32(reinterpret_cast<uint8_t*>(db) + at, wb);
        }
      }
      if (add) {
        __syncwarp();
        if (valid && mine > 0) prompt_add_special<BF, false>(p, it, h, add0, add1, reinterpret_cast<void*>(dst));
      }
      tc_fence_before();                                  // these loads before the p_full of the next unit
    }
  }
  if (timed_out) report(p.status, kStatusTimeout);

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_free(tmem_base, kPmCols);
  }
}

// Merge of a unit's shares: one warp per row, four columns per lane; K shares (of two tiles each, where both hold the row) are
// loaded at a time: many where few rows have many shares, few where many rows need the registers.
template <int K>
__global__ void __launch_bounds__(256, K > 2 ? 2 : 6) prompt_merge_kernel(const PromptParams p) {
  const int lane = threadIdx.x & 31;
  const int u = blockIdx.x >> 5, r = (blockIdx.x & 31) * 8 + (threadIdx.x >> 5);       // row of the 256
  pdl_wait();
  const PromptItem it = p.items[u];
  const int t = r >> 7, tok = (r & 127) / p.G, g = (r & 127) - tok * p.G, tk = t * p.tpt + tok;
  if (tok >= p.tpt || tk >= it.ntok) return;
  const int parts = prompt_parts(max(tile_blocks(it, 0, p.tpt), tile_blocks(it, 1, p.tpt)), p.nsplit, p.split_min);
  if (parts == 1) return;                                // it has its result
  const int tiles = prompt_twin(it, p.tpt, parts) ? 2 : 1;     // of a share that hold this row
  const size_t at0 = (size_t)u * p.nsplit * 256 + r;
  float2 ml[2];
  float m = -INFINITY;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    ml[s] = make_float2(-INFINITY, 0.f);
    if (lane < parts && s < tiles) ml[s] = *reinterpret_cast<const float2*>(p.part_ml + (at0 + (size_t)lane * 256 + s * 128) * 2);
    // the maximum leaves a NaN share out of m, but its l is NaN and reaches the sum
    m = fmaxf(m, ml[s].x);
  }
  m = warp_max(m);
  float w[2], l = 0.f;
  uint32_t seen[2];                                      // shares in which the row saw a key: all of these are read
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    seen[s] = __ballot_sync(0xffffffffu, ml[s].x != -INFINITY);
    w[s] = ml[s].x == -INFINITY ? 0.f : pm_exp2(ml[s].x - m);
    l += ml[s].x == -INFINITY && ml[s].y == 0.f ? 0.f : w[s] * ml[s].y;
  }
  l = warp_sum(l);
  const float scale = l > 0.f || l != l ? 1.f / l : 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < parts; i += K) {                   // (loads under predicates: all of them in flight)
    float4 v[K][2];
    float wi[K][2];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        wi[k][s] = __shfl_sync(0xffffffffu, w[s], (i + k) & 31);
        const bool read = i + k < parts && (seen[s] >> (i + k) & 1u) != 0u;
        v[k][s] = make_float4(0.f, 0.f, 0.f, 0.f);
        // a share that this row sees nothing of may not have been written; one whose weight comes to 0 is read all the same: a NaN
        // or infinity in it reaches the row, as it does where one CTA takes all keys
        if (read) v[k][s] = *reinterpret_cast<const float4*>(p.part_o + (at0 + (size_t)(i + k) * 256 + s * 128) * kPmD + lane * 4);
      }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        o.x += wi[k][s] * v[k][s].x;
        o.y += wi[k][s] * v[k][s].y;
        o.z += wi[k][s] * v[k][s].z;
        o.w += wi[k][s] * v[k][s].w;
      }
  }
  uint2 out = make_uint2(0u, 0u);
  if (scale != 0.f) out = make_uint2(pack2(o.x * scale, o.y * scale, p.bf16), pack2(o.z * scale, o.w * scale, p.bf16));
  *reinterpret_cast<uint2*>(p.out + ((size_t)(it.tok0 + tk) * p.Hq + (size_t)it.h * p.G + g) * kPmD + lane * 4) = out;
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
static int prompt_tiles_bound(int Tq, int S, int tpt) {
  // ceil(n / per) <= (n - 1) / per + 1 for every sequence that is not empty
  const long long s = S < Tq ? S : Tq, n = ((long long)Tq - s) / (2 * tpt) + s;
  return n > kPmMaxItems ? -1 : (int)n;
}

// How a call is cut.  Up to one unit per SM, every CTA finds its unit itself (one prompt of 128 tokens 9.3 us, with the planner
// 12.4; of 1000 tokens 22.8 and 25.3), and where that leaves half of the SMs or more without one, several CTAs share a unit's
// keys: few rows over a long cache are bound by how many SMs read it (17 queries over 9000 keys 17.8 us, not shared 108.8;
// 1 over 1000 10.4 and 17.4; 512 over 4000 44.4 and 61.5; where no unit turns out to be worth sharing, the merge's launch is lost: four
// of 64 over 700 22.3 and 19.2).  Else the planner's list and persistent CTAs.  The batch-invariant mode never shares: how
// many CTAs do depends on the batch.
struct PromptPlan {
  int max_items, direct, nsplit, split_min, grid;
  size_t items_bytes, ws_bytes;
};

static bool prompt_plan(PromptPlan& pl, int S, int Tq, long long keys, int Hkv, int tpt) {
  pl.max_items = prompt_tiles_bound(Tq, S, tpt);
  if (pl.max_items < 0 || (long long)pl.max_items * Hkv > 0x3fffffffll) return false;
  const long long units = (long long)pl.max_items * Hkv;
  const int sms = sm_count();
  pl.direct = units <= sms;
  pl.nsplit = pl.split_min = 1;
  if (pl.direct && !g_batch_invariant && units > 0) {
    // what prompt_parts can come to for a sequence of all the keys: the bound changes no result, only the scratch
    pl.nsplit = (int)(sms / units);
    pl.split_min = pl.nsplit >= 4 ? kPmSplitFew : kPmSplitMany;
    const long long most = (keys + kPmBK - 1) / kPmBK / pl.split_min;
    if (pl.nsplit > most) pl.nsplit = (int)most;
    if (pl.nsplit > kPmMaxSplit) pl.nsplit = kPmMaxSplit;
    if (pl.nsplit < 2) pl.nsplit = 1;
  }
  pl.grid = (int)(units < 1 ? 1 : pl.direct ? units * pl.nsplit : sms);
  const long long listed = pl.direct ? (pl.nsplit > 1 ? units : 0) : pl.max_items;
  pl.items_bytes = 256 + ((size_t)listed * sizeof(PromptItem) + 255) / 256 * 256;
  pl.ws_bytes = pl.items_bytes + (pl.nsplit > 1 ? (size_t)pl.grid * 256 * (kPmD + 2) * sizeof(float) : 0);
  return true;
}

struct PromptStrides {
  long long tok, head;       // elements
};

static int prompt_impl(const void* q, const void* k, const void* v, const int32_t* cu_q, const int32_t* cu_k,
                       const int32_t* lens, const int32_t* page_table, int pages, int page_size, int table_stride,
                       PromptStrides sq, PromptStrides sk, PromptStrides sv, void* out, int S, int Tq, int Tk, int Hq, int Hkv,
                       int D, int causal, int bf16, void* ws, size_t ws_bytes, int32_t* status, cudaStream_t stream) {
  auto bad_ptr = [](const void* x, uintptr_t a) { return x == nullptr || (reinterpret_cast<uintptr_t>(x) & (a - 1)) != 0; };
  const bool paged = lens != nullptr;
  if (S < 0 || Tq < 0 || Tk < 0 || Hq <= 0 || Hkv <= 0 || (bf16 != 0 && bf16 != 1) || (causal != 0 && causal != 1)) return VMK_E_BADARG;
  if (D != kPmD || Hq % Hkv != 0 || Hq / Hkv > 16) return VMK_E_UNSUPPORTED;
  if (Tq == 0) return VMK_OK;
  if (bad_ptr(q, 16) || bad_ptr(out, 32) || bad_ptr(cu_q, 4) || (status && bad_ptr(status, 4))) return VMK_E_BADARG;
  const bool keys = paged ? pages > 0 : Tk > 0;
  if (keys && (bad_ptr(k, 16) || bad_ptr(v, 16))) return VMK_E_BADARG;
  if (paged) {
    if (bad_ptr(page_table, 4) || bad_ptr(lens, 4) || pages < 0 || page_size <= 0 || page_size % 64 != 0 || table_stride <= 0) return VMK_E_BADARG;
    if ((long long)pages * Hkv > 0x7fffffffll) return VMK_E_TOO_LARGE;
  } else if (bad_ptr(cu_k, 4)) {
    return VMK_E_BADARG;
  }
  if (Tk > 0x7fff0000 || Tq > 0x7fff0000) return VMK_E_TOO_LARGE;
  const int G = Hq / Hkv, tpt = 128 / G;
  PromptPlan pl;
  if (!prompt_plan(pl, S, Tq, paged ? (long long)table_stride * page_size : Tk, Hkv, tpt)) return VMK_E_TOO_LARGE;
  if (bad_ptr(ws, 256)) return VMK_E_BADARG;
  if (ws_bytes < pl.ws_bytes) return VMK_E_WORKSPACE;

  PromptParams p;
  memset(&p, 0, sizeof(p));
  int rc = make_tmap_strided(&p.tmQ, q, (uint64_t)Hq, (uint64_t)Tq, sq.head, sq.tok, 64, G, tpt);
  if (rc != VMK_OK) return rc;
  if (keys) {
    if (paged) {
      rc = make_tmap_3d(&p.tmK, k, kPmD, page_size, (uint64_t)pages * Hkv, 64, 64);
      if (rc == VMK_OK) rc = make_tmap_3d(&p.tmV, v, kPmD, page_size, (uint64_t)pages * Hkv, 64, 64);
    } else {
      rc = make_tmap_strided(&p.tmK, k, (uint64_t)Hkv, (uint64_t)Tk, sk.head, sk.tok, 64, 1, kPmBK);
      if (rc == VMK_OK) rc = make_tmap_strided(&p.tmV, v, (uint64_t)Hkv, (uint64_t)Tk, sv.head, sv.tok, 64, 1, kPmBK);
    }
    if (rc != VMK_OK) return rc;
  } else {
    p.tmK = p.tmV = p.tmQ;                                 // valid descriptors that no load uses
  }
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return VMK_E_LAUNCH;
  if (dev >= 64 || !(configured.load() >> dev & 1)) {
    cudaError_t e = cudaSuccess;
    for (auto kernel : {prompt_kernel<false, false>, prompt_kernel<false, true>, prompt_kernel<true, false>, prompt_kernel<true, true>})
      if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPmSmem);
    if (e != cudaSuccess) return check_launch(e);
    if (dev < 64) configured.fetch_or(1ull << dev);
  }
  p.out = static_cast<__half*>(out);
  p.ctrl = static_cast<PromptCtrl*>(ws);
  p.items = reinterpret_cast<PromptItem*>(static_cast<uint8_t*>(ws) + 256);
  p.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + pl.items_bytes);
  p.part_o = p.part_ml + (size_t)pl.grid * 256 * 2;
  p.direct = pl.direct;
  p.nsplit = pl.nsplit;
  p.split_min = pl.split_min;
  p.page_table = paged ? page_table : nullptr;
  p.page_size = page_size;
  p.v = static_cast<const uint16_t*>(v);
  p.v_tok = sv.tok;
  p.v_head = sv.head;
  p.table_stride = table_stride;
  p.page_groups = paged ? pages * Hkv : 0;
  p.Tq = Tq;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.G = G;
  p.tpt = tpt;
  p.sc = kLog2e * 0.08838834764831845f;                    // log2(e) / sqrt(128)
  p.bf16 = bf16;
  p.status = status;
  const long long cap = (long long)table_stride * page_size;
  p.seqs = PromptSeqs{cu_q, cu_k, lens, S, Tq, !keys ? 0 : paged ? (int)(cap > 0x7fff0000ll ? 0x7fff0000ll : cap) : Tk, tpt, causal};

  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!pl.direct) {
    PromptPlanParams pp;
    memset(&pp, 0, sizeof(pp));
    pp.seqs = p.seqs;
    pp.items = p.items;
    pp.ctrl = p.ctrl;
    pp.max_items = pl.max_items;
    pp.first_units = pl.grid;
    pp.status = status;
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(kPmPlanThreads);
    rc = check_launch(cudaLaunchKernelEx(&cfg, prompt_plan_kernel, pp));
    if (rc != VMK_OK) return rc;
  }
  cfg.gridDim = dim3(pl.grid);
  cfg.blockDim = dim3(kPmThreads);
  cfg.dynamicSmemBytes = kPmSmem;
  const auto kernel = pl.nsplit > 1 ? (bf16 ? prompt_kernel<true, true> : prompt_kernel<false, true>)
                                    : (bf16 ? prompt_kernel<true, false> : prompt_kernel<false, false>);
  rc = check_launch(cudaLaunchKernelEx(&cfg, kernel, p));
  if (rc != VMK_OK || pl.nsplit == 1) return rc;
  // (17 queries over 60001 keys 51.6 us with eight shares at a time, 54.2 with two; 512 over 2000 48.8 and 31.8)
  cfg.gridDim = dim3(pl.grid / pl.nsplit * 32);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = 0;
  return check_launch(cudaLaunchKernelEx(&cfg, pl.nsplit >= 4 ? prompt_merge_kernel<8> : prompt_merge_kernel<2>, p));
}

}  // namespace vmk

using namespace vmk;

extern "C" size_t vmk_prompt_workspace_bytes(int S, int Tq, long long keys, int Hq, int Hkv, int D) {
  if (S < 0 || Tq < 0 || keys < 0 || Hq <= 0 || Hkv <= 0 || D != kPmD || Hq % Hkv != 0 || Hq / Hkv > 16) return 0;
  PromptPlan pl;
  return prompt_plan(pl, S, Tq, keys, Hkv, 128 / (Hq / Hkv)) ? pl.ws_bytes : 0;
}

extern "C" int vmk_prompt(const void* q, const void* k, const void* v, const int32_t* cu_q, const int32_t* cu_k,
                          const int64_t* strides, void* out, int S, int Tq, int Tk, int Hq, int Hkv, int D, int causal,
                          int bf16, void* ws, size_t ws_bytes, int32_t* status, void* stream) {
  const long long dq = (long long)Hq * D, dk = (long long)Hkv * D;
  PromptStrides sq{dq, D}, sk{dk, D}, sv{dk, D};
  if (strides != nullptr) {
    sq = {strides[0], strides[1]};
    sk = {strides[2], strides[3]};
    sv = {strides[4], strides[5]};
  }
  return prompt_impl(q, k, v, cu_q, cu_k, nullptr, nullptr, 0, 0, 0, sq, sk, sv, out, S, Tq, Tk, Hq, Hkv, D, causal, bf16, ws,
                     ws_bytes, status, static_cast<cudaStream_t>(stream));
}

extern "C" int vmk_prompt_paged(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table, int pages,
                                int page_size, int table_stride, const int32_t* cu_q, const int32_t* lens,
                                const int64_t* strides, void* out, int S, int Tq, int Hq, int Hkv, int D, int causal,
                                int bf16, void* ws, size_t ws_bytes, int32_t* status, void* stream) {
  if (lens == nullptr) return VMK_E_BADARG;
  PromptStrides sq{(long long)Hq * D, D};
  if (strides != nullptr) sq = {strides[0], strides[1]};
  return prompt_impl(q, k_pages, v_pages, cu_q, nullptr, lens, page_table, pages, page_size, table_stride, sq, sq, sq, out, S,
                     Tq, 0, Hq, Hkv, D, causal, bf16, ws, ws_bytes, status, static_cast<cudaStream_t>(stream));
}
