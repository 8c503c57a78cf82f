// The pages of a paged cache: giving them to growing requests, filling them, copying them, sharing them between forked
// requests, closing up a verified draft tail, taking them back.  The reference names the paged cache as the variant it
// leaves out (README.md:141-142); the paged attention calls of this library read the tables that these operators keep.
//
// State: page_table (R, T) int32 (slot i of row r: the page of its positions [i * page_size, (i+1) * page_size), -1
// behind them), lens (R) int32, refs (pages) int32: how many slots name a page.  A page is free when refs is 0, and the
// lowest free page is given first, to rows in their order: the result does not depend on timing, and there is no free
// list that could go out of step with the counts.  A row gets all the pages that it asks for or none.
//
// Pools are any number (up to 8) of tensors (layers, pages, heads, page_size, row bytes), so one call moves the pages of
// every layer, of keys and values, or of dsa's latent rows and index keys.  The operators that move data are bound by
// the bytes they read and write; those that only keep the tables by latency: one launch each, the giving of pages by ONE
// CTA (a scan over the counts that stops at the last page needed), so that nothing waits for another CTA.
//
// Measured: copying 256 pages of 16 KiB x 8 heads in 8 layers, K and V (1.07 GB moved) 171 us = 6.3 TB/s; 48 rows of up to
// 1500 positions freed, reserved and filled 56 us = 5.3 TB/s, 128 forks of 32 rows 51 us = 5.5 TB/s; the five launches of
// one step after a verification (free, reserve, append, compact with its free) 18.3 to 19.7 us.  Before reserve looked at the
// counts of last pages it was 17.8 on the same GPU (16.3 on another); letting a launch begin while the one before runs
// (launch_dependents at the top) made those 16.3 17.7.
//
// A row grows only into positions of its own: where its last page is partly used and shared, reserve refuses it, and
// compact moves a row's drafts all together or not at all.
#include <cstring>

#include "common.cuh"

namespace vmk {

constexpr int kPgPools = 8;
constexpr int kPgThreads = 1024;
constexpr int kPgPer = 8;                        // page counts per thread and step of the scan

struct PagePool {
  uint8_t* base;
  long long layers;
  int heads, row_bytes;                          // row_bytes a multiple of 16
};

struct PagePools {
  PagePool pool[kPgPools];
  int n, pages, page_size;
};

struct PageTables {
  int32_t *table, *lens, *refs;
  int R, T, pages, page_size;
  int32_t* status;
};

__device__ __forceinline__ int pg_ceil(int a, int b) { return (int)(((long long)a + b - 1) / b); }

// Inclusive prefix sum over the block's threads (1024); every thread calls it.
__device__ __forceinline__ int block_scan(int v, int* s_warp) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();                               // readers of the scan before are done
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += x;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  return v + (warp > 0 ? s_warp[warp - 1] : 0);
}

// The lowest `want` free pages into list[0..); returns how many there are (at most want).  One CTA.
__device__ int find_free(const int32_t* refs, int pages, int want, int* list, int* s_warp) {
  int found = 0;
  for (int base = 0; base < pages && found < want; base += kPgThreads * kPgPer) {
    const int first = base + threadIdx.x * kPgPer;
    uint32_t mask = 0;
    if (first + kPgPer <= pages) {               // refs is 16-byte aligned, first a multiple of 8
      int4 v[kPgPer / 4];
#pragma unroll
      for (int i = 0; i < kPgPer / 4; ++i) v[i] = reinterpret_cast<const int4*>(refs + first)[i];
#pragma unroll
      for (int i = 0; i < kPgPer / 4; ++i)
        mask |= ((v[i].x == 0 ? 1u : 0u) | (v[i].y == 0 ? 2u : 0u) | (v[i].z == 0 ? 4u : 0u) | (v[i].w == 0 ? 8u : 0u)) << (4 * i);
    } else {
      for (int i = 0; i < kPgPer && first + i < pages; ++i) mask |= (refs[first + i] == 0 ? 1u : 0u) << i;
    }
    const int n = __popc(mask), incl = block_scan(n, s_warp);
    int at = found + incl - n;
    for (uint32_t m = mask; m != 0u && at < want; m &= m - 1u, ++at) list[at] = first + __ffs(m) - 1;
    __syncthreads();
    found += s_warp[31];
  }
  __syncthreads();                               // the list is complete for the whole block
  return min(found, want);
}

// ------------------------------------------------------------------------------------------------ reserve
struct ReserveParams {
  PageTables t;
  const int32_t* extra;
  int32_t* granted;                              // nullable
  int *list, *start;                             // pages, R; start -1: refused, its last page is shared
};

__device__ __forceinline__ bool reserve_need(const ReserveParams& p, int r, int& have, int& need, int& len, int& more) {
  len = max(p.t.lens[r], 0);
  more = p.extra[r];
  have = pg_ceil(len, p.t.page_size);
  need = 0;
  if (more <= 0) return more == 0;
  const long long want = ((long long)len + more + p.t.page_size - 1) / p.t.page_size;
  if (want > p.t.T || have > p.t.T || (long long)len + more > 0x7fffffffll) return false;
  need = (int)want - have;
  return true;
}

// Whether the row's last page is partly used and other slots name it too (a forked row that was cut inside a shared page, or
// the row that it was forked from): the positions behind lens are theirs, so the row must not grow into them.
__device__ __forceinline__ bool reserve_shared(const PageTables& t, int r, int have, int len) {
  if (len % t.page_size == 0) return false;
  const int id = t.table[(size_t)r * t.T + have - 1];
  return id >= 0 && id < t.pages && t.refs[id] > 1;
}

__global__ void __launch_bounds__(kPgThreads, 1) pages_reserve_kernel(const ReserveParams p) {
  __shared__ int s_warp[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  // No more than every page can be given, whatever the rows ask for: sums saturate just above that (a row asks for at
  // most 2^20 pages, the width of a table, so a block's sum stays below 2^31).
  const int cap = p.t.pages + 1;
  int total = 0;
  for (int base = 0; base < p.t.R; base += kPgThreads) {
    const int r = base + tid;
    int have, need = 0, len, more;
    bool shared = false;
    if (r < p.t.R && reserve_need(p, r, have, need, len, more) && more > 0) shared = reserve_shared(p.t, r, have, len);
    const int capped = shared ? 0 : min(need, cap);
    const int incl = block_scan(capped, s_warp);
    if (r < p.t.R) p.start[r] = shared ? -1 : (int)min((long long)total + incl - capped, (long long)cap);
    __syncthreads();
    total = (int)min((long long)total + s_warp[31], (long long)cap);
  }
  const int found = find_free(p.t.refs, p.t.pages, min(total, p.t.pages), p.list, s_warp);
  for (int r = warp; r < p.t.R; r += kPgThreads / 32) {
    int have, need, len, more;
    const bool valid = reserve_need(p, r, have, need, len, more);
    const int start = p.start[r];
    const bool ok = valid && start >= 0 && (long long)start + need <= (need > 0 ? found : 0x7fffffff);
    if (ok) {
      for (int i = lane; i < need; i += 32) {
        const int id = p.list[start + i];
        p.t.table[(size_t)r * p.t.T + have + i] = id;
        p.t.refs[id] = 1;
      }
    }
    __syncwarp();
    if (lane == 0) {
      if (ok) p.t.lens[r] = len + more;
      if (p.granted != nullptr) p.granted[r] = ok ? 1 : 0;
      if (!ok) report(p.t.status, valid ? kStatusPages : (more < 0 ? kStatusBadIndex : kStatusPages));
    }
  }
}

// ------------------------------------------------------------------------------------------------ free
struct FreeParams {
  PageTables t;
  const int32_t* keep;                           // tokens that row r keeps; null: lens - kd + count (after compact)
  const int32_t *count, *granted;                // granted nullable: a row with 0 has no drafts
  int kd;
};

// One warp per row.
__global__ void __launch_bounds__(256) pages_free_kernel(const FreeParams p) {
  const int r = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  if (r >= p.t.R) return;
  const int marked = p.t.lens[r], len = max(marked, 0);
  __syncwarp();                                  // every lane has read lens before lane 0 writes it
  if (p.keep == nullptr && marked < 0) {         // compact refused the row: length and pages as they were
    if (lane == 0) p.t.lens[r] = ~marked;
    return;
  }
  int keep;
  bool bad = false;
  if (p.keep != nullptr) {
    keep = p.keep[r];
    if (keep < 0) { bad = true; keep = len; }    // refused: the row stays as it is
  } else {
    const int c = p.granted != nullptr && p.granted[r] == 0 ? -1 : p.count[r];
    keep = c < 0 || len < p.kd ? len : len - p.kd + min(c, p.kd);
  }
  keep = min(keep, len);
  const int first = pg_ceil(keep, p.t.page_size), last = min(pg_ceil(len, p.t.page_size), p.t.T);
  int32_t* row = p.t.table + (size_t)r * p.t.T;
  for (int i = first + lane; i < last; i += 32) {
    const int id = row[i];
    if (id >= 0 && id < p.t.pages) {
      if (atomicSub(&p.t.refs[id], 1) <= 0) {    // nobody held it: the count stays at zero
        atomicAdd(&p.t.refs[id], 1);
        bad = true;
      }
    } else {
      bad = true;
    }
    row[i] = -1;
  }
  __syncwarp();
  if (lane == 0) p.t.lens[r] = keep;
  if (bad) report(p.t.status, kStatusBadIndex);
}

// ------------------------------------------------------------------------------------------------ fork
struct ForkJob {
  int src, dst, rows;                            // copy the first `rows` rows of page src to page dst
  int pad;
};

struct ForkParams {
  PageTables t;
  const int32_t *parents, *children;
  int F;
  int *list, *owner;                             // F (at most one page each), R
  int *start, *len;                              // F each; len < 0: refused
  ForkJob* jobs;                                 // F
};

__global__ void __launch_bounds__(kPgThreads, 1) pages_fork_kernel(const ForkParams p) {
  __shared__ int s_warp[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const PageTables& t = p.t;
  pdl_wait();
  // the same child named twice: the first entry has it
  for (int f = tid; f < p.F; f += kPgThreads) {
    const int c = p.children[f];
    if (c >= 0 && c < t.R) p.owner[c] = 0x7fffffff;
  }
  __syncthreads();
  for (int f = tid; f < p.F; f += kPgThreads) {
    const int c = p.children[f];
    if (c >= 0 && c < t.R && p.parents[f] >= 0) atomicMin(&p.owner[c], f);
  }
  __syncthreads();
  int total = 0;
  bool bad = false;
  for (int base = 0; base < p.F; base += kPgThreads) {
    const int f = base + tid;
    int need = 0, n = -1;
    if (f < p.F) {
      const int par = p.parents[f], c = p.children[f];
      if (par >= 0) {                            // a negative parent: an entry that does nothing
        const bool ok = par < t.R && c >= 0 && c < t.R && t.lens[c] == 0 && p.owner[c] == f;
        if (ok) n = max(t.lens[par], 0);
        if (!ok || pg_ceil(n, t.page_size) > t.T) { bad = true; n = -1; }
      }
      need = n > 0 && n % t.page_size != 0 ? 1 : 0;
    }
    const int incl = block_scan(need, s_warp);
    if (f < p.F) {
      p.start[f] = total + incl - need;
      p.len[f] = n;
    }
    __syncthreads();
    total += s_warp[31];
  }
  const int found = find_free(t.refs, t.pages, min(total, t.pages), p.list, s_warp);
  for (int f = warp; f < p.F; f += kPgThreads / 32) {
    int n = p.len[f];
    const int start = p.start[f];
    ForkJob job{0, 0, 0, 0};
    if (n > 0) {
      const int par = p.parents[f], c = p.children[f];
      const int32_t* from = t.table + (size_t)par * t.T;
      int32_t* to = t.table + (size_t)c * t.T;
      const int full = n / t.page_size, rest = n - full * t.page_size;
      if (rest > 0 && start >= found) {
        if (lane == 0) report(t.status, kStatusPages);
      } else {
        for (int i = lane; i < full; i += 32) {
          const int id = from[i];
          to[i] = id;
          if (id >= 0 && id < t.pages) atomicAdd(&t.refs[id], 1); else bad = true;
        }
        if (rest > 0) {
          const int src = from[full], dst = p.list[start];
          if (src >= 0 && src < t.pages) job = ForkJob{src, dst, rest, 0}; else bad = true;
          if (lane == 0) {
            to[full] = dst;
            t.refs[dst] = 1;
          }
        }
        if (lane == 0) t.lens[c] = n;
      }
    }
    if (lane == 0) p.jobs[f] = job;
  }
  if (bad) report(t.status, kStatusBadIndex);
}

// A warp copies n 16-byte chunks, eight loads in flight per lane.
__device__ __forceinline__ void warp_copy(uint4* dst, const uint4* src, int n, int lane) {
  for (int i = lane; i < n; i += 8 * 32) {
    uint4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k * 32 < n) v[k] = src[i + k * 32];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i + k * 32 < n) dst[i + k * 32] = v[k];
  }
}

// One warp per (entry, layer, head): the rows of a head are contiguous inside a page.
__global__ void __launch_bounds__(256) pages_fork_copy_kernel(const PagePools pools, const ForkJob* jobs, int F, int per_entry) {
  const int lane = threadIdx.x & 31;
  pdl_wait();
  const long long n = (long long)F * per_entry;
  for (long long w = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; w < n; w += (long long)gridDim.x * 8) {
    const ForkJob job = jobs[w / per_entry];
    if (job.rows == 0) continue;
    int k = (int)(w % per_entry), i = 0;
    for (; k >= (int)pools.pool[i].layers * pools.pool[i].heads; ++i) k -= (int)pools.pool[i].layers * pools.pool[i].heads;
    const PagePool& pl = pools.pool[i];
    const int layer = k / pl.heads, head = k - layer * pl.heads;
    const size_t head_bytes = (size_t)pools.page_size * pl.row_bytes;
    uint8_t* at = pl.base + ((size_t)layer * pools.pages * pl.heads + head) * head_bytes;
    warp_copy(reinterpret_cast<uint4*>(at + (size_t)job.dst * pl.heads * head_bytes),
              reinterpret_cast<const uint4*>(at + (size_t)job.src * pl.heads * head_bytes), job.rows * (pl.row_bytes / 16), lane);
  }
}

// ------------------------------------------------------------------------------------------------ copy
// One warp per 8 KiB of a page (a whole page of one layer is contiguous).
constexpr int kPgChunk = 8192;

__global__ void __launch_bounds__(256) pages_copy_kernel(const PagePools pools, const int32_t* src, const int32_t* dst, int n,
                                                         long long per_entry, int32_t* status) {
  const int lane = threadIdx.x & 31;
  pdl_wait();
  const long long total = (long long)n * per_entry;
  for (long long w = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; w < total; w += (long long)gridDim.x * 8) {
    const int e = (int)(w / per_entry);
    long long k = w - (long long)e * per_entry;
    const int s = src[e], d = dst[e];
    if (s < 0 || s >= pools.pages || d < 0 || d >= pools.pages) {
      if (k == 0 && lane == 0) report(status, kStatusBadIndex);
      continue;
    }
    if (s == d) continue;
    int i = 0;
    for (;; ++i) {
      const long long bytes = (long long)pools.pool[i].heads * pools.page_size * pools.pool[i].row_bytes;
      const long long chunks = (bytes + kPgChunk - 1) / kPgChunk * pools.pool[i].layers;
      if (k < chunks) break;
      k -= chunks;
    }
    const PagePool& pl = pools.pool[i];
    const long long bytes = (long long)pl.heads * pools.page_size * pl.row_bytes, chunks = (bytes + kPgChunk - 1) / kPgChunk;
    const long long layer = k / chunks, at = (k - layer * chunks) * kPgChunk;
    uint8_t* page0 = pl.base + (size_t)layer * pools.pages * bytes + at;
    warp_copy(reinterpret_cast<uint4*>(page0 + (size_t)d * bytes), reinterpret_cast<const uint4*>(page0 + (size_t)s * bytes),
              (int)(min((long long)kPgChunk, bytes - at) / 16), lane);
  }
}

// ------------------------------------------------------------------------------------------------ append
struct AppendSource {
  const uint8_t* src;                            // (tokens, heads, row)
  long long tok, head;                           // strides in bytes
};

struct AppendParams {
  PagePools pools;
  AppendSource from[2];
  const int32_t *table, *cu, *lens;
  const int32_t *refs, *granted;                 // both nullable; granted 0: the row did not get the positions of its tokens
  int S, T, tokens;
  int32_t* status;
};

// One warp per token: its position is the row's length minus what is left of the row's new tokens.
__global__ void __launch_bounds__(256) pages_append_kernel(const AppendParams p) {
  const int lane = threadIdx.x & 31;
  pdl_wait();
  const int t = (blockIdx.x * 256 + threadIdx.x) >> 5;
  if (t >= p.tokens) return;
  // the last sequence that begins at or before t: 32-ary search (cu ascending)
  int lo = 0, n = p.S + 1;                       // cu[lo] <= t < cu[lo + n), if any is
  if (t < p.cu[0] || t >= p.cu[p.S]) return;     // behind the last sequence: nothing is written
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i = lo + lane * step;
    const bool le = i < lo + n && p.cu[i] <= t;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, le) | 1u);
    lo += last * step;
    n = min(step, n - last * step);
  }
  if (p.granted != nullptr && lo < p.S && p.granted[lo] == 0) return;      // lens does not count them: they would fall on older ones
  const int end = p.cu[min(lo + 1, p.S)];
  const long long pos = (long long)p.lens[min(lo, p.S - 1)] - (end - t);
  const long long slot = pos >= 0 ? pos / p.pools.page_size : -1;
  const int id = lo < p.S && slot >= 0 && slot < p.T ? p.table[(size_t)lo * p.T + slot] : -1;
  if (id < 0 || id >= p.pools.pages) {
    if (lane == 0) report(p.status, kStatusBadIndex);
    return;
  }
  if (p.refs != nullptr && p.refs[id] > 1) {     // other rows' positions too
    if (lane == 0) report(p.status, kStatusPages);
    return;
  }
  const int row = (int)(pos - slot * p.pools.page_size);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const PagePool& pl = p.pools.pool[i];
    const int c = pl.row_bytes / 16, all = c * pl.heads;
    const uint8_t* src = p.from[i].src + (size_t)t * p.from[i].tok;
    uint8_t* dst = pl.base + (((size_t)id * pl.heads) * p.pools.page_size + row) * pl.row_bytes;
    for (int e = lane; e < all; e += 4 * 32) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int x = e + k * 32, h = x / c;
        if (x < all) v[k] = *reinterpret_cast<const uint4*>(src + (size_t)h * p.from[i].head + (size_t)(x - h * c) * 16);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int x = e + k * 32, h = x / c;
        if (x < all) *reinterpret_cast<uint4*>(dst + (size_t)h * p.pools.page_size * pl.row_bytes + (size_t)(x - h * c) * 16) = v[k];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ compact
struct CompactParams {
  PagePools pools;
  int32_t* lens;
  const int32_t *table, *refs, *path, *count, *granted;
  int R, T, kd, per_row;                         // per_row: 16-byte columns of one position over all pools
  int32_t* status;
};

// A thread owns one 16-byte column of a row's positions and moves it down the path: entry j goes from base + path[j] to
// base + j with path[j] >= j ascending, so a source is never a destination of an earlier entry, and reads of eight
// entries may go before their writes.
//
// A row moves as a whole or not at all: where one of its entries cannot move (its new place is in a page that others share, the
// path does not ascend) nothing is written and the row stays as it is, or its positions would hold other drafts than the
// accepted ones.  Every CTA of the row comes to that by itself; its first one tells the free that follows by the one word that
// both see, lens, which it turns negative (~lens) until then.  A CTA that reads lens after that knows the same.
__global__ void __launch_bounds__(256) pages_compact_kernel(const CompactParams p) {
  extern __shared__ int s_at[];                  // [kd] source page * page_size + row, [kd] destination; -1: nothing to move
  int* s_from = s_at;
  int* s_to = s_at + p.kd;
  const int r = blockIdx.x, tid = threadIdx.x;
  pdl_wait();
  const int len = *const_cast<const volatile int32_t*>(p.lens + r), base = len - p.kd;
  const int n = p.granted != nullptr && p.granted[r] == 0 ? -1 : min(p.count[r], p.kd);
  const int ps = p.pools.page_size;
  bool refused = false;
  for (int j = tid; j < p.kd; j += 256) {
    int from = -1, to = -1;
    bool bad = false, shared = false;
    if (j < n) {
      const int x = p.path[(size_t)r * p.kd + j];
      if (base < 0 || x < j || x >= p.kd || (j > 0 && x <= p.path[(size_t)r * p.kd + j - 1])) {
        bad = true;
      } else if (x > j) {
        const int sf = (base + x) / ps, st = (base + j) / ps;
        const int a = sf < p.T ? p.table[(size_t)r * p.T + sf] : -1, b = st < p.T ? p.table[(size_t)r * p.T + st] : -1;
        if (a < 0 || a >= p.pools.pages || b < 0 || b >= p.pools.pages) {
          bad = true;
        } else if (p.refs[b] > 1) {
          shared = true;
        } else {
          from = (base + x) - sf * ps;
          to = (base + j) - st * ps;
          s_from[j] = a;
          s_to[j] = b;
        }
      }
    }
    if (blockIdx.y == 0 && bad) report(p.status, kStatusBadIndex);
    if (blockIdx.y == 0 && shared) report(p.status, kStatusPages);
    refused |= bad || shared;
    s_at[2 * p.kd + j] = from;
    s_at[3 * p.kd + j] = to;
  }
  refused = __syncthreads_or(refused);
  if (blockIdx.y == 0 && tid == 0 && (refused || len < 0)) p.lens[r] = ~max(len, 0);      // (len < 0: no length, it becomes 0)
  if (n <= 0 || refused) return;
  for (int c0 = blockIdx.y * 256 + tid; c0 < p.per_row; c0 += gridDim.y * 256) {
    int c = c0, i = 0;
    for (;; ++i) {
      const int cols = (int)p.pools.pool[i].layers * p.pools.pool[i].heads * (p.pools.pool[i].row_bytes / 16);
      if (c < cols) break;
      c -= cols;
    }
    const PagePool& pl = p.pools.pool[i];
    const int w = pl.row_bytes / 16;
    const int lh = c / w, layer = lh / pl.heads, head = lh - layer * pl.heads;
    uint8_t* col = pl.base + (((size_t)layer * p.pools.pages * pl.heads + head) * ps) * pl.row_bytes + (size_t)(c - lh * w) * 16;
    const size_t page_bytes = (size_t)pl.heads * ps * pl.row_bytes;
    for (int j0 = 0; j0 < n; j0 += 8) {
      uint4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = j0 + k;
        if (j < n && s_at[2 * p.kd + j] >= 0)
          v[k] = *reinterpret_cast<const uint4*>(col + (size_t)s_from[j] * page_bytes + (size_t)s_at[2 * p.kd + j] * pl.row_bytes);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = j0 + k;
        if (j < n && s_at[2 * p.kd + j] >= 0)
          *reinterpret_cast<uint4*>(col + (size_t)s_to[j] * page_bytes + (size_t)s_at[3 * p.kd + j] * pl.row_bytes) = v[k];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
static bool pg_bad(const void* x, uintptr_t a) { return x == nullptr || (reinterpret_cast<uintptr_t>(x) & (a - 1)) != 0; }

// pools: 4 numbers each (address, layers, heads, bytes of one position of one head).  Returns a VMK_E_* code.
static int read_pools(PagePools& out, const int64_t* pools, int n, int pages, int page_size, int max_pools) {
  memset(&out, 0, sizeof(out));
  if (pools == nullptr || n <= 0 || pages <= 0 || page_size <= 0) return VMK_E_BADARG;
  if (n > max_pools) return VMK_E_UNSUPPORTED;
  long long columns = 0;
  for (int i = 0; i < n; ++i) {
    const int64_t* d = pools + 4 * i;
    if (d[0] == 0 || (d[0] & 15) != 0 || d[1] <= 0 || d[2] <= 0 || d[3] <= 0 || d[3] % 16 != 0) return VMK_E_BADARG;
    if (d[1] > (1 << 20) || d[2] > (1 << 20) || d[3] > (1 << 24)) return VMK_E_TOO_LARGE;
    // a page of one head and a page of one layer fit 31 bits of 16-byte chunks
    if ((long long)page_size * d[3] > 0x7fffffffll || (long long)page_size * d[3] / 16 * d[2] > 0x7fffffffll) return VMK_E_TOO_LARGE;
    columns += d[1] * d[2] * (d[3] / 16);
    if (columns > 0x7fffffffll) return VMK_E_TOO_LARGE;
    out.pool[i].base = reinterpret_cast<uint8_t*>(static_cast<uintptr_t>(d[0]));
    out.pool[i].layers = d[1];
    out.pool[i].heads = (int)d[2];
    out.pool[i].row_bytes = (int)d[3];
  }
  out.n = n;
  out.pages = pages;
  out.page_size = page_size;
  return VMK_OK;
}

static int read_tables(PageTables& t, int32_t* table, int R, int T, int32_t* lens, int32_t* refs, int pages, int page_size,
                       int32_t* status) {
  if (R < 0 || T <= 0 || pages <= 0 || page_size <= 0) return VMK_E_BADARG;
  if (R > 0 && (pg_bad(table, 4) || pg_bad(lens, 4) || pg_bad(refs, 16))) return VMK_E_BADARG;
  if (status && pg_bad(status, 4)) return VMK_E_BADARG;
  if (R > (1 << 26) || pages > 0x7fff0000 || T > (1 << 20)) return VMK_E_TOO_LARGE;
  t = PageTables{table, lens, refs, R, T, pages, page_size, status};
  return VMK_OK;
}

// Every kernel here is a programmatic dependent (its pdl_wait comes before its first read): in a chain of page operators
// a launch is set up while the one before runs.
template <typename K, typename... A>
static int pg_launch(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_launch(cudaLaunchKernelEx(&cfg, kernel, args...));
}

static int blocks_for(long long warps, int per_sm) {
  const long long b = (warps + 7) / 8, cap = (long long)sm_count() * per_sm;
  return (int)(b < 1 ? 1 : b < cap ? b : cap);
}

}  // namespace vmk

using namespace vmk;

extern "C" int vmk_pages_copy(const int64_t* pools, int n_pools, int pages, int page_size, const int32_t* src,
                              const int32_t* dst, int n, int32_t* status, void* stream) {
  PagePools pl;
  const int rc = read_pools(pl, pools, n_pools, pages, page_size, kPgPools);
  if (rc != VMK_OK) return rc;
  if (n < 0) return VMK_E_BADARG;
  if (n == 0) return VMK_OK;
  if (pg_bad(src, 4) || pg_bad(dst, 4) || (status && pg_bad(status, 4))) return VMK_E_BADARG;
  long long per = 0;
  for (int i = 0; i < n_pools; ++i)
    per += ((long long)pl.pool[i].heads * page_size * pl.pool[i].row_bytes + kPgChunk - 1) / kPgChunk * pl.pool[i].layers;
  return pg_launch(pages_copy_kernel, dim3(blocks_for((long long)n * per, 8)), 256, 0, static_cast<cudaStream_t>(stream), pl, src, dst,
                   n, per, status);
}

extern "C" int vmk_pages_append(const int64_t* pools, const int64_t* sources, int pages, int page_size, const int32_t* page_table,
                                int table_stride, const int32_t* cu, const int32_t* lens, int S, int tokens, int32_t* status,
                                void* stream) {
  return vmk_pages_append_granted(pools, sources, pages, page_size, page_table, table_stride, cu, lens, nullptr, nullptr, S, tokens,
                                  status, stream);
}

extern "C" int vmk_pages_append_granted(const int64_t* pools, const int64_t* sources, int pages, int page_size,
                                        const int32_t* page_table, int table_stride, const int32_t* cu, const int32_t* lens,
                                        const int32_t* refs, const int32_t* granted, int S, int tokens, int32_t* status,
                                        void* stream) {
  AppendParams p;
  memset(&p, 0, sizeof(p));
  const int rc = read_pools(p.pools, pools, 2, pages, page_size, 2);
  if (rc != VMK_OK) return rc;
  if (sources == nullptr || S < 0 || tokens < 0 || table_stride <= 0) return VMK_E_BADARG;
  if (p.pools.pool[0].layers != 1 || p.pools.pool[1].layers != 1) return VMK_E_UNSUPPORTED;
  if (S == 0 || tokens == 0) return VMK_OK;
  if (pg_bad(page_table, 4) || pg_bad(cu, 4) || pg_bad(lens, 4) || (refs && pg_bad(refs, 4)) || (granted && pg_bad(granted, 4)) ||
      (status && pg_bad(status, 4)))
    return VMK_E_BADARG;
  if (tokens > 0x7fffffff / 32 - 256) return VMK_E_TOO_LARGE;
  for (int i = 0; i < 2; ++i) {
    const int64_t* d = sources + 3 * i;
    if (d[0] == 0 || (d[0] & 15) != 0 || d[1] < 0 || d[1] % 16 != 0 || d[2] < 0 || d[2] % 16 != 0) return VMK_E_BADARG;
    p.from[i] = AppendSource{reinterpret_cast<const uint8_t*>(static_cast<uintptr_t>(d[0])), d[1], d[2]};
  }
  p.table = page_table;
  p.cu = cu;
  p.lens = lens;
  p.refs = refs;
  p.granted = granted;
  p.S = S;
  p.T = table_stride;
  p.tokens = tokens;
  p.status = status;
  return pg_launch(pages_append_kernel, dim3((tokens + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream), p);
}

extern "C" size_t vmk_pages_workspace_bytes(int R, int F, int pages) {
  if (R < 0 || F < 0 || pages < 0) return 0;
  // reserve: list (pages) + start (R); fork: jobs (F) + list (F) + owner (R) + start (F) + len (F)
  const size_t reserve = 4 * ((size_t)pages + R), fork = (sizeof(ForkJob) + 12) * (size_t)F + 4 * (size_t)R;
  return (reserve > fork ? reserve : fork) + 256;
}

extern "C" int vmk_pages_reserve(int32_t* page_table, int R, int table_stride, int32_t* lens, int32_t* refs, int pages,
                                 int page_size, const int32_t* extra, int32_t* granted, void* ws, size_t ws_bytes,
                                 int32_t* status, void* stream) {
  ReserveParams p;
  memset(&p, 0, sizeof(p));
  const int rc = read_tables(p.t, page_table, R, table_stride, lens, refs, pages, page_size, status);
  if (rc != VMK_OK) return rc;
  if (R == 0) return VMK_OK;
  if (pg_bad(extra, 4) || (granted && pg_bad(granted, 4)) || pg_bad(ws, 16)) return VMK_E_BADARG;
  if (ws_bytes < vmk_pages_workspace_bytes(R, 0, pages)) return VMK_E_WORKSPACE;
  p.extra = extra;
  p.granted = granted;
  p.list = static_cast<int*>(ws);
  p.start = p.list + pages;
  return pg_launch(pages_reserve_kernel, dim3(1), kPgThreads, 0, static_cast<cudaStream_t>(stream), p);
}

extern "C" int vmk_pages_free(int32_t* page_table, int R, int table_stride, int32_t* lens, int32_t* refs, int pages, int page_size,
                              const int32_t* keep, int32_t* status, void* stream) {
  FreeParams p;
  memset(&p, 0, sizeof(p));
  const int rc = read_tables(p.t, page_table, R, table_stride, lens, refs, pages, page_size, status);
  if (rc != VMK_OK) return rc;
  if (R == 0) return VMK_OK;
  if (pg_bad(keep, 4)) return VMK_E_BADARG;
  p.keep = keep;
  return pg_launch(pages_free_kernel, dim3((R + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream), p);
}

extern "C" int vmk_pages_fork(const int64_t* pools, int n_pools, int32_t* page_table, int R, int table_stride, int32_t* lens,
                              int32_t* refs, int pages, int page_size, const int32_t* parents, const int32_t* children, int F,
                              void* ws, size_t ws_bytes, int32_t* status, void* stream) {
  ForkParams p;
  memset(&p, 0, sizeof(p));
  PagePools pl;
  int rc = read_pools(pl, pools, n_pools, pages, page_size, kPgPools);
  if (rc == VMK_OK) rc = read_tables(p.t, page_table, R, table_stride, lens, refs, pages, page_size, status);
  if (rc != VMK_OK) return rc;
  if (F < 0) return VMK_E_BADARG;
  if (F == 0 || R == 0) return VMK_OK;
  if (pg_bad(parents, 4) || pg_bad(children, 4) || pg_bad(ws, 16)) return VMK_E_BADARG;
  if (F > (1 << 26)) return VMK_E_TOO_LARGE;
  if (ws_bytes < vmk_pages_workspace_bytes(R, F, 0)) return VMK_E_WORKSPACE;
  p.parents = parents;
  p.children = children;
  p.F = F;
  p.jobs = static_cast<ForkJob*>(ws);
  p.list = reinterpret_cast<int*>(p.jobs + F);
  p.start = p.list + F;
  p.len = p.start + F;
  p.owner = p.len + F;
  long long per = 0;
  for (int i = 0; i < n_pools; ++i) per += pl.pool[i].layers * pl.pool[i].heads;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = pg_launch(pages_fork_kernel, dim3(1), kPgThreads, 0, s, p);
  if (rc != VMK_OK) return rc;
  return pg_launch(pages_fork_copy_kernel, dim3(blocks_for((long long)F * per, 8)), 256, 0, s, pl, (const ForkJob*)p.jobs, F, (int)per);
}

extern "C" int vmk_pages_compact(const int64_t* pools, int n_pools, int32_t* page_table, int R, int table_stride, int32_t* lens,
                                 int32_t* refs, int pages, int page_size, const int32_t* path, const int32_t* count, int kd,
                                 int32_t* status, void* stream) {
  return vmk_pages_compact_granted(pools, n_pools, page_table, R, table_stride, lens, refs, pages, page_size, path, count, nullptr, kd,
                                   status, stream);
}

extern "C" int vmk_pages_compact_granted(const int64_t* pools, int n_pools, int32_t* page_table, int R, int table_stride,
                                         int32_t* lens, int32_t* refs, int pages, int page_size, const int32_t* path,
                                         const int32_t* count, const int32_t* granted, int kd, int32_t* status, void* stream) {
  CompactParams p;
  FreeParams f;
  memset(&p, 0, sizeof(p));
  memset(&f, 0, sizeof(f));
  int rc = read_pools(p.pools, pools, n_pools, pages, page_size, kPgPools);
  if (rc == VMK_OK) rc = read_tables(f.t, page_table, R, table_stride, lens, refs, pages, page_size, status);
  if (rc != VMK_OK) return rc;
  if (kd <= 0) return VMK_E_BADARG;
  if (kd > VMK_SPEC_MAX_DRAFTS) return VMK_E_UNSUPPORTED;
  if (R == 0) return VMK_OK;
  if (pg_bad(path, 4) || pg_bad(count, 4) || (granted && pg_bad(granted, 4))) return VMK_E_BADARG;
  p.table = page_table;
  p.lens = lens;
  p.refs = refs;
  p.path = path;
  p.count = count;
  p.granted = f.granted = granted;
  p.R = R;
  p.T = table_stride;
  p.kd = kd;
  for (int i = 0; i < n_pools; ++i) p.per_row += (int)(pools[4 * i + 1] * pools[4 * i + 2] * (pools[4 * i + 3] / 16));
  p.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int ny = (p.per_row + 255) / 256;
  rc = pg_launch(pages_compact_kernel, dim3(R, ny < 65535 ? ny : 65535), 256, (size_t)4 * kd * sizeof(int), s, p);
  if (rc != VMK_OK) return rc;
  f.count = count;
  f.kd = kd;
  return pg_launch(pages_free_kernel, dim3((R + 7) / 8), 256, 0, s, f);
}
