// Pages of a paged K/V cache on the device: requests grow, shrink and leave
// (dsb_resize_requests), start from another request's tokens without a copy
// of its whole pages (dsb_fork_requests), the live pages move to the front of
// the pool (dsb_compact_pages), and pages are copied (dsb_copy_pages).
//
// State: ref_counts[N] (rows that hold the page; 0: free), block_tables
// [R, C] (entry -1: none) and held[R] (pages each row holds, its first
// entries).  Pages are handed out lowest id first, rows in call order, so a
// call's result depends on its arguments alone.
#include <algorithm>

#include "tma_umma.cuh"

namespace dsb {
namespace {

// A planning CTA has 256 threads when they see its pages in one turn (and the
// call's rows are few), else 1024: what such a call takes is the latency of its
// barriers and dependent reads (512 pages to compact: 13 us with 1024 threads,
// 6.5 with 256).
constexpr int kPgThreads = 1024, kPgFew = 256;
constexpr int kPgPages = 16;        // pages a thread looks at in a turn
constexpr int kPgTurn = kPgThreads * kPgPages;
// The planning CTAs are a cluster, each with a stretch of the pool: one CTA as
// long as it sees the pool in one turn, else eight (40000 pages, 64 children:
// 19 us by one, 15 by eight; a turn's masks are kept in registers from the
// count to the pages handed out).
constexpr int kPgCluster = 8;
constexpr int kPgMaxRows = 4096;    // rows of one call
constexpr int kPgMaxCaches = 128;   // caches of one launch
// Rows x table columns up to which one CTA lets the pages go by itself; beyond
// it a kernel over the GPU does first (524288 entries of 64 rows: 497 us by
// one CTA; 8192 entries of 8 rows: one launch less is worth 2 us).
constexpr int64_t kPgAlone = 16384;

struct Pool {
  int32_t *refs;
  int64_t pages;
  int32_t *tables;
  int64_t rows, stride, cols;
  int32_t *held;
  int bs;
  int32_t *status;  // [2]: rows left without pages, free pages after the call
  int32_t *err;
};

struct Caches {
  void *p[kPgMaxCaches];
  int n;
};

// Sums of counts; with SAT they end at INT32_MAX (what rows ask for may pass it).
template <bool SAT> __device__ __forceinline__ int add_counts(int a, int b) {
  return SAT ? (int)min((unsigned)a + (unsigned)b, (unsigned)INT32_MAX) : a + b;
}

// Sum of the warps' values before this warp's; `total` gets the sum of all.
template <int T, bool SAT = false> __device__ int warps_before(int mine, int32_t *warp_tot, int &total) {
  if ((threadIdx.x & 31) == 0) warp_tot[threadIdx.x >> 5] = mine;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < T / 32; ++w) {
    if (w == (int)(threadIdx.x >> 5)) before = total;
    total = add_counts<SAT>(total, warp_tot[w]);
  }
  __syncthreads();
  return before;
}

// Inclusive prefix sum over the CTA's threads.
template <int T, bool SAT = false> __device__ int block_scan(int v, int32_t *warp_tot, int &total) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = add_counts<SAT>(v, x);
  }
  return add_counts<SAT>(warps_before<T, SAT>(__shfl_sync(0xffffffffu, v, 31), warp_tot, total), v);
}

// a[0..n) in shared memory becomes its inclusive prefix sum, at most INT32_MAX.
template <int T> __device__ int scan_rows(int32_t *a, int n, int32_t *warp_tot) {
  int run = 0;
  for (int base = 0; base < n; base += T) {
    const int i = base + threadIdx.x;
    int total;
    const int s = block_scan<T, true>(i < n ? a[i] : 0, warp_tot, total);
    if (i < n) a[i] = add_counts<true>(s, run);
    run = add_counts<true>(run, total);
  }
  __syncthreads();
  return run;
}

// This CTA's stretch of the pool, and what the CTAs of the cluster tell each
// other (every CTA of it calls these together).
struct Stretch {
  int64_t from, till;
  int rank, ranks;
  int32_t *told;  // [kPgCluster] in shared memory
  __device__ Stretch(int64_t pages, int ranks_, int32_t *told_) : ranks(ranks_), told(told_) {
    rank = ranks > 1 ? (int)cluster_rank() : 0;
    const int64_t per = (pages + ranks - 1) / ranks;
    from = min(pages, rank * per);
    till = min(pages, from + per);
    if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  }
  // Every CTA of the cluster has begun (its shared memory may not be written
  // before): once, in front of the first sync or gather.
  __device__ void begun() const {
    if (ranks > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
  }
  __device__ void sync() const {
    __syncthreads();
    if (ranks > 1) cluster_sync_all();
  }
  // Sum of `mine` over the CTAs, and over those before this one.
  __device__ int gather(int mine, int &before) const {
    if (ranks == 1) {
      before = 0;
      return mine;
    }
    __syncthreads();
    if ((int)threadIdx.x < ranks)
      st_cluster(cluster_map(smem_u32(told + rank), threadIdx.x), __int_as_float(mine));
    cluster_sync_all();
    int total = 0;
    before = 0;
    for (int r = 0; r < ranks; ++r) {
      if (r == rank) before = total;
      total += told[r];
    }
    cluster_sync_all();  // (the places are written again by the next gather)
    return total;
  }
};

// The CTA's stretch in turns of 16 pages a thread: look(j, page, count) for
// each page of a thread, side by side in a warp (a warp has 512 pages in a row,
// a thread every 32nd of them), with the loads of a turn all on their way at
// once.
__device__ __forceinline__ int64_t warp_page(int64_t base, int j) {
  return base + (int64_t)(threadIdx.x >> 5) * 32 * kPgPages + 32 * j;
}
template <typename F> __device__ __forceinline__ void read_turn(const Pool &p, int64_t base, int64_t till, F look) {
  int v[kPgPages];
  const int64_t first = warp_page(base, 0) + (threadIdx.x & 31);
#pragma unroll
  for (int j = 0; j < kPgPages; ++j) v[j] = first + 32 * j < till ? __ldcg(p.refs + first + 32 * j) : -1;
#pragma unroll
  for (int j = 0; j < kPgPages; ++j) look(j, first + 32 * j, v[j]);  // (behind `till`: -1)
}

// The free pages of the CTA's stretch: their number, and of its last turn
// (`whole`: its only one) a mask for each 32 pages of the warp and the free
// ones before the warp.
template <int T> struct Free {
  unsigned mask[kPgPages];
  int before, total;
  bool whole;
  __device__ __forceinline__ int read(const Pool &p, const Stretch &s, int64_t base) {
    int mine = 0;
    read_turn(p, base, s.till, [&](int j, int64_t, int v) {
      mask[j] = __ballot_sync(0xffffffffu, v == 0);
      mine += __popc(mask[j]);
    });
    return mine;
  }
  // Counts below zero (pages let go more often than they were held) are
  // flagged and cleared.
  __device__ __forceinline__ void count(const Pool &p, const Stretch &s, int32_t *warp_tot) {
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kPgPages; ++j) mask[j] = 0;
    for (int64_t base = s.from; base < s.till; base += T * kPgPages)
      read_turn(p, base, s.till, [&](int j, int64_t page, int v) {
        if (v < 0 && page < s.till) {
          p.refs[page] = 0;
          flag_error(p.err, DSB_FLAG_BLOCK);
          v = 0;
        }
        mask[j] = __ballot_sync(0xffffffffu, v == 0);
        mine += __popc(mask[j]);
      });
    before = warps_before<T>(mine, warp_tot, total);
    whole = s.till - s.from <= T * kPgPages;
  }
};
// The lowest x of 32 bits.
__device__ __forceinline__ unsigned low_bits(int x) {
  return x <= 0 ? 0u : x >= 32 ? ~0u : (1u << x) - 1;
}

// Drop `n` references to `page`.  More than there are leave a negative count,
// which the pass over the pool that follows flags and clears: an atomic that
// returns nothing is half the time of one that tells.
__device__ __forceinline__ void release(const Pool &p, int page, int n) {
  if (page < 0 || page >= p.pages)
    flag_error(p.err, DSB_FLAG_BLOCK);
  else
    atomicSub(p.refs + page, n);
}

// Changes of reference counts that a thread meets one after another, joined
// while they name one of the last four pages: the rows of a call share most
// of their pages, and an atomic a page is what they cost.
struct PageCounts {
  int page[4], n[4], next;
  __device__ PageCounts() : next(0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) page[i] = -1, n[i] = 0;
  }
  template <typename F> __device__ void add(int x, F flush) {
    bool found = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!found && n[i] > 0 && page[i] == x) {
        ++n[i];
        found = true;
      }
    if (found) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i == next) {
        if (n[i] > 0) flush(page[i], n[i]);
        page[i] = x;
        n[i] = 1;
      }
    next = (next + 1) & 3;
  }
};

// Hand the lowest free pages out: want[] is the inclusive prefix sum of the
// rows' needs, `granted` the pages given in all, `run` the free pages before
// this CTA's stretch; give(i, k, page) stores row i's k-th new page.
template <int T, typename F>
__device__ void allot(const Pool &p, const Stretch &s, Free<T> &free, const int32_t *want, int n, int granted,
                      int run, int32_t *warp_tot, F give) {
  const int lane = threadIdx.x & 31;
  for (int64_t base = s.from; base < s.till && run < granted; base += T * kPgPages) {
    if (!free.whole) free.before = warps_before<T>(free.read(p, s, base), warp_tot, free.total);
    int rank = run + free.before;
#pragma unroll
    for (int j = 0; j < kPgPages; ++j) {
      const unsigned mask = free.mask[j];
      const int k = rank + __popc(mask & ((1u << lane) - 1));
      rank += __popc(mask);
      if (!(mask >> lane & 1) || k >= granted) continue;
      int lo = 0, hi = n - 1;  // first row whose prefix sum passes the rank
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (want[mid] > k) hi = mid;
        else lo = mid + 1;
      }
      const int page = (int)warp_page(base, j) + lane;
      p.refs[page] = 1;
      give(lo, k - (lo > 0 ? want[lo - 1] : 0), page);
    }
    run += free.total;
  }
}

// Rows given twice in one call: the first counts, the others are flagged.
// again[i] for rows[0..n) in shared memory, a warp a row.
template <int T> __device__ void find_repeats(const int32_t *rows, int32_t *again, int n) {
  for (int i = threadIdx.x >> 5; i < n; i += T / 32) {
    bool hit = false;
    for (int j = threadIdx.x & 31; j < i; j += 32) hit |= rows[j] == rows[i];
    hit = __any_sync(0xffffffffu, hit);
    if ((threadIdx.x & 31) == 0) again[i] = hit;
  }
}

// Pages of row r: those it has, and those `len` tokens need (-1: the table
// cannot hold them).
__device__ __forceinline__ int pages_held(const Pool &p, int r) {
  return min(max(p.held[r], 0), (int)min(p.cols, (int64_t)INT32_MAX));
}
__device__ __forceinline__ int pages_needed(const Pool &p, int len) {
  const int64_t need = ((int64_t)len + p.bs - 1) / p.bs;
  return len < 0 || need > p.cols ? -1 : (int)need;
}

// The surplus pages of 16 rows of the call in 256 table columns: a thread has
// a column, so that a warp reads a row's entries side by side.
constexpr int kPgRows = 16;
__global__ void __launch_bounds__(256)
    release_kernel(const Pool p, const int32_t *__restrict__ rows, const int32_t *__restrict__ lens,
                   int n) {
  __shared__ int32_t s_row[kPgRows], s_keep[kPgRows], s_held[kPgRows];
  pdl_begin();
  const int i0 = blockIdx.y * kPgRows, m = min(kPgRows, n - i0);
  if (threadIdx.x < kPgRows) {
    int r = -1, keep = 0, held = 0;
    if (threadIdx.x < m) {
      r = rows[i0 + threadIdx.x];
      if (r < 0 || r >= p.rows) r = -1;
      if (r >= 0) {
        held = pages_held(p, r);
        keep = pages_needed(p, lens[i0 + threadIdx.x]);
        if (keep < 0 || keep >= held) r = -1;  // nothing to let go
      }
    }
    s_row[threadIdx.x] = r, s_keep[threadIdx.x] = keep, s_held[threadIdx.x] = held;
  }
  __syncthreads();
  // a row named before in the call is not this one's to change
  for (int j = threadIdx.x; j < i0 + m; j += 256) {
    const int r = rows[j];
#pragma unroll
    for (int k = 0; k < kPgRows; ++k)
      if (k < m && j < i0 + k && r == rows[i0 + k]) s_row[k] = -1;
  }
  __syncthreads();
  const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int entry[kPgRows];  // (every read on its way before the first is used)
  unsigned mine = 0;
#pragma unroll
  for (int k = 0; k < kPgRows; ++k)
    if (k < m && s_row[k] >= 0 && j >= s_keep[k] && j < s_held[k]) {
      mine |= 1u << k;
      entry[k] = p.tables[(int64_t)s_row[k] * p.stride + j];
    }
  PageCounts counts;
#pragma unroll
  for (int k = 0; k < kPgRows; ++k)
    if (mine >> k & 1) {
      p.tables[(int64_t)s_row[k] * p.stride + j] = -1;
      counts.add(entry[k], [&](int page, int count) { release(p, page, count); });
    }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (counts.n[i] > 0) release(p, counts.page[i], counts.n[i]);
}

// Every CTA of the cluster has the rows' needs; the first one changes what
// they hold and reports.
template <int T> __global__ void __launch_bounds__(T)
    resize_kernel(const Pool p, const int32_t *__restrict__ rows, const int32_t *__restrict__ lens,
                  int n, int alone, int ranks) {
  extern __shared__ int32_t pg_smem[];
  int32_t *want = pg_smem, *row = want + n, *has = row + n, *target = has + n;
  int32_t *last = target + n;  // the page it has that its new length ends inside, or -1
  __shared__ int32_t warp_tot[T / 32], told[kPgCluster];
  __shared__ int lacking, granted;
  pdl_begin();
  const Stretch s(p.pages, ranks, told);
  const int tid = threadIdx.x;
  if (tid == 0) lacking = granted = 0;
  for (int i = tid; i < n; i += T) row[i] = rows[i], target[i] = lens[i];
  __syncthreads();
  find_repeats<T>(row, want, n);
  __syncthreads();
  for (int i = tid; i < n; i += T) {
    const int r = row[i];
    int have = 0, need = -1, ends_in = -1;
    if (r < 0 || r >= p.rows || want[i]) {
      if (s.rank == 0) flag_error(p.err, DSB_FLAG_SLOT);
    } else {
      need = pages_needed(p, target[i]);
      if (need > 0 && target[i] % p.bs != 0) ends_in = p.tables[(int64_t)r * p.stride + need - 1];
      have = pages_held(p, r);
      if (need > have) ends_in = -1;
      if (need < 0 && s.rank == 0) flag_error(p.err, DSB_FLAG_POSITION);
    }
    last[i] = ends_in;
    has[i] = have;
    target[i] = need;
    want[i] = max(0, need - have);
  }
  __syncthreads();
  s.begun();
  // releases first, a warp a row (unless release_kernel has let them go)
  if (alone) {
    for (int i = tid >> 5; i < n && s.rank == 0; i += T / 32) {
      if (target[i] < 0) continue;
      int32_t *t = p.tables + (int64_t)row[i] * p.stride;
      for (int j = target[i] + (tid & 31); j < has[i]; j += 32) {
        release(p, t[j], 1);
        t[j] = -1;
      }
    }
    s.sync();
  }
  Free<T> free;
  free.count(p, s, warp_tot);
  // a length inside a page that other rows hold, too: what the row writes behind
  // it would be theirs as well
  for (int i = tid; i < n && s.rank == 0; i += T)
    if (last[i] >= 0 && last[i] < p.pages && __ldcg(p.refs + last[i]) > 1)
      flag_error(p.err, DSB_FLAG_POSITION);
  int before;
  const int nfree = s.gather(free.total, before);
  scan_rows<T>(want, n, warp_tot);
  // rows in order until the first that does not fit
  for (int i = tid; i < n; i += T) {
    const bool needs = target[i] > has[i];
    if (want[i] <= nfree && want[i] < INT32_MAX) {
      if (needs) atomicMax(&granted, want[i]);
    } else if (needs) {
      atomicAdd(&lacking, 1);
      continue;
    }
    if (s.rank == 0 && target[i] >= 0) p.held[row[i]] = target[i];
  }
  __syncthreads();
  allot(p, s, free, want, n, granted, before, warp_tot, [&](int i, int k, int page) {
    p.tables[(int64_t)row[i] * p.stride + has[i] + k] = page;
  });
  if (tid == 0 && s.rank == 0 && p.status != nullptr) {
    p.status[0] = lacking;
    p.status[1] = nfree - granted;
  }
  s.sync();  // (held has been read by every CTA before one of them ends)
}

// Per child: parent row, child row (-1: not forked), whole pages, the started
// page's source, its copy and the tokens in it.
struct ForkPlan {
  int32_t parent, child, full, src, dst, tokens;
};

// As in resize_kernel, every CTA has the children's needs, the first one
// writes the plan.
template <int T> __global__ void __launch_bounds__(T)
    fork_plan_kernel(const Pool p, const int32_t *__restrict__ parents,
                     const int32_t *__restrict__ children, const int32_t *__restrict__ lens, int n,
                     ForkPlan *__restrict__ plan, int ranks) {
  extern __shared__ int32_t pg_smem[];
  int32_t *want = pg_smem, *kid = want + n, *par = kid + n;
  int32_t *full = par + n;  // the length, then the whole pages, -1 not forked
  __shared__ int32_t warp_tot[T / 32], told[kPgCluster];
  __shared__ int lacking, granted;
  pdl_begin();
  const Stretch s(p.pages, ranks, told);
  const int tid = threadIdx.x;
  if (tid == 0) lacking = granted = 0;
  // (the first T children and the pool are read at the same time)
  const int c0 = tid < n ? children[tid] : 0, up0 = tid < n ? parents[tid] : 0;
  const int len0 = tid < n ? lens[tid] : 0;
  Free<T> free;
  free.count(p, s, warp_tot);
  for (int i = tid; i < n; i += T) {
    kid[i] = i < T ? c0 : children[i];
    par[i] = i < T ? up0 : parents[i];
    full[i] = i < T ? len0 : lens[i];
  }
  __syncthreads();
  find_repeats<T>(kid, want, n);
  __syncthreads();
  for (int i = tid; i < n; i += T) {
    const int up = par[i], c = kid[i], len = full[i];
    const bool inside = up >= 0 && up < p.rows && c >= 0 && c < p.rows;
    const int parent_has = inside ? p.held[up] : 0, child_has = inside ? p.held[c] : 0;
    ForkPlan f{up, -1, -1, -1, -1, 0};
    int flag = 0;
    if (!inside || want[i] || child_has != 0) {
      flag = DSB_FLAG_SLOT;
    } else if (len < 0 || (int64_t)len > (int64_t)parent_has * p.bs ||
               (int64_t)len > p.cols * p.bs) {
      flag = DSB_FLAG_POSITION;
    } else {
      f.child = c;
      f.full = len / p.bs;
      f.tokens = len % p.bs;
      if (f.tokens > 0) {
        f.src = p.tables[(int64_t)up * p.stride + f.full];
        if (f.src < 0 || f.src >= p.pages) {
          flag = DSB_FLAG_BLOCK;
          f.child = f.full = -1;
          f.tokens = 0;
        }
      }
    }
    want[i] = f.tokens > 0;
    full[i] = f.full;
    if (s.rank == 0) {
      plan[i] = f;
      if (flag != 0) flag_error(p.err, flag);
    }
  }
  __syncthreads();
  s.begun();
  int before;
  const int nfree = s.gather(free.total, before);
  scan_rows<T>(want, n, warp_tot);
  for (int i = tid; i < n; i += T) {
    const bool started = want[i] > (i > 0 ? want[i - 1] : 0);
    if (started && want[i] > nfree) {  // no page for it: not forked
      atomicAdd(&lacking, 1);
      if (s.rank == 0) plan[i].child = -1;
    } else if (full[i] >= 0) {
      if (started) atomicMax(&granted, want[i]);
      if (s.rank == 0) p.held[kid[i]] = full[i] + (started ? 1 : 0);
    }
  }
  __syncthreads();
  allot(p, s, free, want, n, granted, before, warp_tot, [&](int i, int, int page) {
    plan[i].dst = page;
    p.tables[(int64_t)kid[i] * p.stride + full[i]] = page;
  });
  if (tid == 0 && s.rank == 0 && p.status != nullptr) {
    p.status[0] = lacking;
    p.status[1] = nfree - granted;
  }
  s.sync();
}

// `bytes` (a multiple of 16) from src to dst by a CTA of 256 threads, four
// pieces of a thread on their way at once.
__device__ __forceinline__ void copy_bytes(char *dst, const char *src, int64_t bytes) {
  const int64_t n = bytes / 16;
  const uint4 *from = reinterpret_cast<const uint4 *>(src);
  uint4 *to = reinterpret_cast<uint4 *>(dst);
  for (int64_t i = threadIdx.x; i < n; i += 4 * 256) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + 256 * j < n) v[j] = from[i + 256 * j];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + 256 * j < n) to[i + 256 * j] = v[j];
  }
}

// blockIdx.y: 16 children.  The first blocks along x name their whole pages (a
// reference more for each), 256 table columns a block; the others copy the
// started pages' tokens, a (child, cache) at a time.
__global__ void __launch_bounds__(256)
    fork_apply_kernel(const Pool p, const ForkPlan *__restrict__ plan, int n, const Caches caches,
                      int64_t token_bytes, int table_blocks) {
  __shared__ ForkPlan s_plan[kPgRows];
  pdl_begin();
  const int i0 = blockIdx.y * kPgRows, m = min(kPgRows, n - i0);
  if (threadIdx.x < m) s_plan[threadIdx.x] = plan[i0 + threadIdx.x];
  __syncthreads();
  if ((int)blockIdx.x < table_blocks) {
    auto flush = [&](int page, int count) {
      if (page >= 0 && page < p.pages)
        atomicAdd(p.refs + page, count);
      else
        flag_error(p.err, DSB_FLAG_BLOCK);
    };
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < p.cols; j += table_blocks * 256) {
      int page[kPgRows];  // (every read on its way before the first is used)
      unsigned mine = 0;
#pragma unroll
      for (int k = 0; k < kPgRows; ++k)
        if (k < m && s_plan[k].child >= 0 && j < s_plan[k].full) {
          mine |= 1u << k;
          page[k] = p.tables[(int64_t)s_plan[k].parent * p.stride + j];
        }
      PageCounts counts;
#pragma unroll
      for (int k = 0; k < kPgRows; ++k)
        if (mine >> k & 1) {
          p.tables[(int64_t)s_plan[k].child * p.stride + j] = page[k];
          counts.add(page[k], flush);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (counts.n[i] > 0) flush(counts.page[i], counts.n[i]);
    }
    return;
  }
  const int64_t page_bytes = p.bs * token_bytes;
  for (int u = blockIdx.x - table_blocks; u < m * caches.n; u += gridDim.x - table_blocks) {
    const ForkPlan &f = s_plan[u / caches.n];
    if (f.child < 0 || f.tokens <= 0) continue;
    char *base = static_cast<char *>(caches.p[u % caches.n]);
    copy_bytes(base + f.dst * page_bytes, base + f.src * page_bytes, f.tokens * token_bytes);
  }
}

// scratch: [0] pages to move, then sources[N], targets[N], new names[N]
template <int T> __global__ void __launch_bounds__(T)
    compact_plan_kernel(const Pool p, int32_t *__restrict__ scratch, int ranks) {
  __shared__ int32_t warp_tot[T / 32], told[kPgCluster];
  pdl_begin();
  const Stretch s(p.pages, ranks, told);
  const int tid = threadIdx.x, lane = tid & 31;
  const unsigned below = (1u << lane) - 1;
  Free<T> free;
  free.count(p, s, warp_tot);
  s.begun();
  int before;
  const int nfree = s.gather(free.total, before);
  const int64_t live = p.pages - nfree;
  int32_t *src = scratch + 1, *dst = src + p.pages, *name = dst + p.pages;
  // Holes are the free pages below `live`, and as many pages move: in all, and
  // before this stretch.  (One CTA with one turn finds them in its masks.)
  int holes = 0, moved = 0;
  const bool once = ranks == 1 && free.whole;
  if (!once) {
    int h = 0, total;  // free pages of the stretch below `live`
    for (int64_t base = s.from; base < min(s.till, live); base += T * kPgPages)
      read_turn(p, base, min(s.till, live), [&](int, int64_t, int v) { h += v == 0; });
    block_scan<T>(h, warp_tot, total);
    moved = s.gather(total, holes);
  }
  // live pages at or behind `live` and before this stretch: those before the
  // stretch less those before `live`
  int at = s.from <= live ? 0 : (int)(s.from - before) - (int)(live - moved);
  int hole_at = holes;
  for (int64_t base = s.from; base < s.till; base += T * kPgPages) {
    if (!free.whole) free.read(p, s, base);
    int mine = 0, total;  // holes, and pages to move, in 16 bits each
    // pages of the warp below `live`, and within the stretch
    auto ahead = [&](int64_t x) {
      return (int)max((int64_t)0, min((int64_t)32 * kPgPages, x - warp_page(base, 0)));
    };
    const int front = ahead(live), all = ahead(s.till);
    auto hole = [&](int j) { return free.mask[j] & low_bits(front - 32 * j); };
    auto move = [&](int j) {
      return ~free.mask[j] & ~low_bits(front - 32 * j) & low_bits(all - 32 * j);
    };
#pragma unroll
    for (int j = 0; j < kPgPages; ++j) mine += __popc(hole(j)) + (__popc(move(j)) << 16);
    const int b = warps_before<T>(mine, warp_tot, total);
    int h = hole_at + (b & 0xffff), m = at + (b >> 16);
#pragma unroll
    for (int j = 0; j < kPgPages; ++j) {
      const unsigned hm = hole(j), mm = move(j);
      const int page = (int)warp_page(base, j) + lane;
      if (hm >> lane & 1) dst[h + __popc(hm & below)] = page;
      else if (mm >> lane & 1) src[m + __popc(mm & below)] = page;
      else if (free.mask[j] >> lane & 1) name[page] = -1;  // no row holds it
      h += __popc(hm);
      m += __popc(mm);
    }
    hole_at += total & 0xffff;
    at += total >> 16;
    if (once) moved = total & 0xffff;
  }
  s.sync();
#pragma unroll 4
  for (int k = s.rank * T + tid; k < moved; k += ranks * T) {
    const int a = __ldcg(src + k), t = __ldcg(dst + k);
    name[a] = t;
    p.refs[t] = p.refs[a];
    p.refs[a] = 0;
  }
  if (tid == 0 && s.rank == 0) {
    scratch[0] = moved;
    p.status[0] = 0;
    p.status[1] = nfree;
  }
}

// Pages src[k] -> dst[k] of every cache, k < *count (or `n` when null);
// negative entries are skipped, bad ones flagged.  A CTA takes one page of one
// cache at a time.
__device__ void copy_pairs(const Caches &caches, int64_t page_bytes, int64_t pages,
                           const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                           int64_t count, int32_t *err, int64_t first, int64_t step) {
  for (int64_t u = first; u < count * caches.n; u += step) {
    const int64_t k = u / caches.n;
    const int s = src[k], t = dst[k];
    if (s < 0 || t < 0) continue;
    if (s >= pages || t >= pages) {
      if (threadIdx.x == 0) flag_error(err, DSB_FLAG_BLOCK);
      continue;
    }
    char *base = static_cast<char *>(caches.p[u % caches.n]);
    copy_bytes(base + t * page_bytes, base + s * page_bytes, page_bytes);
  }
}

__global__ void __launch_bounds__(256)
    copy_pages_kernel(const Caches caches, int64_t page_bytes, int64_t pages,
                      const int32_t *__restrict__ src, const int32_t *__restrict__ dst, int n,
                      int32_t *err) {
  pdl_begin();
  copy_pairs(caches, page_bytes, pages, src, dst, n, err, blockIdx.x, gridDim.x);
}

// The first `rename_blocks` blocks name the moved pages' new places in the
// rows' tables, the others move the pages.
__global__ void __launch_bounds__(256)
    compact_apply_kernel(const Pool p, const Caches caches, int64_t page_bytes,
                         const int32_t *__restrict__ scratch, int rename_blocks) {
  pdl_begin();
  if ((int)blockIdx.x >= rename_blocks) {
    copy_pairs(caches, page_bytes, p.pages, scratch + 1, scratch + 1 + p.pages, scratch[0], p.err,
               blockIdx.x - rename_blocks, gridDim.x - rename_blocks);
    return;
  }
  const int32_t *name = scratch + 1 + 2 * p.pages;
  // live pages are in front now: an entry that points behind them was moved
  const int64_t live = p.pages - p.status[1];
  for (int64_t row = blockIdx.x; row < p.rows; row += rename_blocks) {
    const int held = pages_held(p, (int)row);
    int32_t *t = p.tables + row * p.stride;
#pragma unroll 4
    for (int j = threadIdx.x; j < held; j += 256) {
      const int page = t[j];
      if (page < 0 || page >= p.pages)
        flag_error(p.err, DSB_FLAG_BLOCK);
      else if (page >= live)
        t[j] = name[page];
    }
  }
}

// f(threads, CTAs) with the planners of a pool: the variant's threads as a type.
template <typename F> void with_planners(int64_t pages, int n, F f) {
  const int ranks = pages <= kPgFew * kPgPages ? 1 : kPgCluster;
  if (pages <= (int64_t)ranks * kPgFew * kPgPages && n <= kPgFew)
    f(std::integral_constant<int, kPgFew>{}, ranks);
  else
    f(std::integral_constant<int, kPgThreads>{}, pages <= kPgTurn ? 1 : kPgCluster);
}

int check_pool(const Pool &p, int n) {
  if (p.pages <= 0 || p.pages > INT32_MAX || p.rows <= 0 || p.rows > INT32_MAX || p.cols <= 0 ||
      p.stride < p.cols)
    return fail(DSB_ERR_INVALID, "bad pool or block-table geometry");
  if (p.bs <= 0) return fail(DSB_ERR_INVALID, "block_size must be positive");
  if (n < 0 || n > kPgMaxRows)
    return fail(DSB_ERR_INVALID, "the rows of one call must be in [0, 4096]");
  if (!p.refs || !p.tables || !p.held) return fail(DSB_ERR_INVALID, "null pointer argument");
  return DSB_OK;
}

int check_caches(const void *const *caches, int num_caches, int64_t unit_bytes) {
  if (num_caches < 0 || (num_caches > 0 && !caches))
    return fail(DSB_ERR_INVALID, "null pointer argument");
  if (unit_bytes <= 0 || unit_bytes % 16)
    return fail(DSB_ERR_UNSUPPORTED, "a token's K (or V) row must be a multiple of 16 bytes");
  for (int i = 0; i < num_caches; ++i)
    if (!caches[i] || reinterpret_cast<uintptr_t>(caches[i]) % 16)
      return fail(DSB_ERR_INVALID, "caches must be non-null and 16-byte aligned");
  return DSB_OK;
}

// f(part) for runs of at most kPgMaxCaches caches.
template <typename F> void each_part(void *const *caches, int n, F f) {
  for (int base = 0; base < n; base += kPgMaxCaches) {
    Caches part{};
    part.n = std::min(n - base, kPgMaxCaches);
    for (int i = 0; i < part.n; ++i) part.p[i] = caches[base + i];
    f(part);
  }
}

}  // namespace
}  // namespace dsb

using namespace dsb;

extern "C" int dsb_resize_requests(int32_t *ref_counts, int64_t num_pages, int32_t *block_tables,
                                   int64_t table_rows, int64_t table_stride, int64_t table_cols,
                                   int32_t *held, const int32_t *rows, const int32_t *lens,
                                   int32_t n, int32_t block_size, int32_t *status,
                                   int32_t *error_flag, void *stream) {
  const Pool p{ref_counts, num_pages, block_tables, table_rows, table_stride, table_cols,
               held,       block_size, status,      error_flag};
  if (int e = check_pool(p, n)) return e;
  if (n > 0 && (!rows || !lens)) return fail(DSB_ERR_INVALID, "null pointer argument");
  const cudaStream_t st = as_stream(stream);
  const bool alone = (int64_t)n * table_cols <= kPgAlone;
  if (!alone) {
    launch_kernel(release_kernel,
                  dim3((unsigned)((table_cols + 255) / 256), (unsigned)((n + kPgRows - 1) / kPgRows)),
                  dim3(256), 0, st, p, rows, lens, (int)n);
    if (int e = check_launch("release_kernel")) return e;
  }
  const size_t smem = (size_t)n * 5 * sizeof(int32_t);
  int e = DSB_OK;
  with_planners(num_pages, n, [&](auto threads, int ranks) {
    auto kern = resize_kernel<threads()>;
    if ((e = ensure_smem((const void *)kern, smem)) != DSB_OK) return;
    launch_kernel_cluster(kern, dim3(ranks), dim3(threads()), smem, st, ranks, p, rows, lens, (int)n,
                          alone ? 1 : 0, ranks);
  });
  return e != DSB_OK ? e : check_launch("resize_kernel");
}

extern "C" int64_t dsb_fork_scratch_ints(int32_t n) { return n > 0 ? 6 * (int64_t)n : 0; }

extern "C" int dsb_fork_requests(int32_t *ref_counts, int64_t num_pages, int32_t *block_tables,
                                 int64_t table_rows, int64_t table_stride, int64_t table_cols,
                                 int32_t *held, const int32_t *parents, const int32_t *children,
                                 const int32_t *lens, int32_t n, int32_t block_size,
                                 void *const *caches, int32_t num_caches, int64_t token_bytes,
                                 int32_t *status, int32_t *scratch, int64_t scratch_ints,
                                 int32_t *error_flag, void *stream) {
  const Pool p{ref_counts, num_pages, block_tables, table_rows, table_stride, table_cols,
               held,       block_size, status,      error_flag};
  if (int e = check_pool(p, n)) return e;
  if (int e = check_caches(caches, num_caches, token_bytes)) return e;
  if (n > 0 && (!parents || !children || !lens || !scratch))
    return fail(DSB_ERR_INVALID, "null pointer argument");
  if (scratch_ints < dsb_fork_scratch_ints(n))
    return fail(DSB_ERR_INVALID, "scratch smaller than dsb_fork_scratch_ints");
  const cudaStream_t st = as_stream(stream);
  ForkPlan *plan = reinterpret_cast<ForkPlan *>(scratch);
  const size_t smem = (size_t)n * 4 * sizeof(int32_t);
  int e = DSB_OK;
  with_planners(num_pages, n, [&](auto threads, int ranks) {
    auto kern = fork_plan_kernel<threads()>;
    if ((e = ensure_smem((const void *)kern, smem)) != DSB_OK) return;
    launch_kernel_cluster(kern, dim3(ranks), dim3(threads()), smem, st, ranks, p, parents, children, lens,
                          (int)n, plan, ranks);
  });
  if (e != DSB_OK) return e;
  if (int err = check_launch("fork_plan_kernel")) return err;
  if (n == 0) return DSB_OK;
  const int table_blocks = (int)std::min<int64_t>(64, (table_cols + 255) / 256);
  const unsigned gy = (unsigned)((n + kPgRows - 1) / kPgRows);
  bool first = true;
  auto apply = [&](const Caches &part) {
    const int tb = first ? table_blocks : 0;  // the tables once
    first = false;
    launch_kernel(fork_apply_kernel, dim3(tb + std::min(kPgRows * part.n, 128), gy), dim3(256), 0, st,
                  p, (const ForkPlan *)plan, (int)n, part, token_bytes, tb);
  };
  each_part(caches, num_caches, apply);
  if (num_caches == 0) apply(Caches{});
  return check_launch("fork_apply_kernel");
}

extern "C" int64_t dsb_compact_scratch_ints(int64_t num_pages) {
  return num_pages > 0 ? 1 + 3 * num_pages : 0;
}

extern "C" int dsb_compact_pages(int32_t *ref_counts, int64_t num_pages, int32_t *block_tables,
                                 int64_t table_rows, int64_t table_stride, int64_t table_cols,
                                 int32_t *held, int32_t block_size, void *const *caches,
                                 int32_t num_caches, int64_t token_bytes, int32_t *status,
                                 int32_t *scratch, int64_t scratch_ints, int32_t *error_flag,
                                 void *stream) {
  const Pool p{ref_counts, num_pages, block_tables, table_rows, table_stride, table_cols,
               held,       block_size, status,      error_flag};
  if (int e = check_pool(p, 0)) return e;
  if (int e = check_caches(caches, num_caches, token_bytes)) return e;
  if (!status || !scratch) return fail(DSB_ERR_INVALID, "null pointer argument");
  if (scratch_ints < dsb_compact_scratch_ints(num_pages))
    return fail(DSB_ERR_INVALID, "scratch smaller than dsb_compact_scratch_ints");
  const cudaStream_t st = as_stream(stream);
  with_planners(num_pages, 0, [&](auto threads, int ranks) {
    launch_kernel_cluster(compact_plan_kernel<threads()>, dim3(ranks), dim3(threads()), 0, st, ranks, p,
                          scratch, ranks);
  });
  if (int e = check_launch("compact_plan_kernel")) return e;
  bool first = true;
  auto apply = [&](const Caches &part) {
    const int rb = first ? (int)std::min<int64_t>(table_rows, 64) : 0;  // the tables once
    first = false;
    const int64_t units = (num_pages / 2 + 1) * part.n;  // at most half of the pages move
    const unsigned cb = (unsigned)std::min<int64_t>(units, 8L * sm_count());
    launch_kernel(compact_apply_kernel, dim3(rb + cb), dim3(256), 0, st, p, part,
                  token_bytes * block_size, (const int32_t *)scratch, rb);
  };
  each_part(caches, num_caches, apply);
  if (num_caches == 0) apply(Caches{});
  return check_launch("compact_apply_kernel");
}

extern "C" int dsb_copy_pages(void *const *caches, int32_t num_caches, int64_t num_pages,
                              int64_t page_bytes, const int32_t *src, const int32_t *dst,
                              int32_t n, int32_t *error_flag, void *stream) {
  if (n < 0 || num_pages <= 0 || num_pages > INT32_MAX)
    return fail(DSB_ERR_INVALID, "bad page counts");
  if (int e = check_caches(caches, num_caches, page_bytes)) return e;
  if (n == 0 || num_caches == 0) return DSB_OK;
  if (!src || !dst) return fail(DSB_ERR_INVALID, "null pointer argument");
  each_part(caches, num_caches, [&](const Caches &part) {
    const int64_t units = (int64_t)n * part.n;
    launch_kernel(copy_pages_kernel, dim3((unsigned)std::min<int64_t>(units, 8L * sm_count())),
                  dim3(256), 0, as_stream(stream), part, page_bytes, num_pages, src, dst, (int)n,
                  error_flag);
  });
  return check_launch("copy_pages_kernel");
}
