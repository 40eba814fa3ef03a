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

#include "common.cuh"

namespace dsb {
namespace {

constexpr int kPgThreads = 1024;
constexpr int kPgMaxRows = 4096;    // rows of one call
constexpr int kPgMaxCaches = 128;   // caches of one launch

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

// Inclusive prefix sum over the block's threads; `total` gets the sum.
__device__ int block_scan(int v, int32_t *warp_tot, int &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  __syncthreads();
  if (lane == 31) warp_tot[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = warp_tot[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += x;
    }
    warp_tot[lane] = w;
  }
  __syncthreads();
  total = warp_tot[31];
  return incl + (warp > 0 ? warp_tot[warp - 1] : 0);
}

// a[0..n) in shared memory becomes its inclusive prefix sum.
__device__ int scan_rows(int32_t *a, int n, int32_t *warp_tot) {
  int run = 0;
  for (int base = 0; base < n; base += kPgThreads) {
    const int i = base + threadIdx.x;
    int total;
    const int s = block_scan(i < n ? a[i] : 0, warp_tot, total) + run;
    if (i < n) a[i] = s;
    run += total;
  }
  __syncthreads();
  return run;
}

__device__ int free_pages(const Pool &p, int32_t *warp_tot) {
  int mine = 0, total;
  for (int64_t i = threadIdx.x; i < p.pages; i += kPgThreads) mine += __ldcg(p.refs + i) == 0;
  block_scan(mine, warp_tot, total);
  return total;
}

// Drop one reference to `page`; a page that nothing holds is flagged.
__device__ __forceinline__ void release(const Pool &p, int page) {
  if (page < 0 || page >= p.pages) {
    flag_error(p.err, DSB_FLAG_BLOCK);
    return;
  }
  if (atomicSub(p.refs + page, 1) <= 0) {
    atomicAdd(p.refs + page, 1);
    flag_error(p.err, DSB_FLAG_BLOCK);
  }
}

// Hand the lowest free pages out: want[] is the inclusive prefix sum of the
// rows' needs, `granted` the pages given in all; give(i, k, page) stores row
// i's k-th new page.
template <typename F>
__device__ void allot(const Pool &p, const int32_t *want, int n, int granted, int32_t *warp_tot,
                      F give) {
  int run = 0;
  for (int64_t base = 0; base < p.pages && run < granted; base += kPgThreads) {
    const int64_t page = base + threadIdx.x;
    const bool is_free = page < p.pages && __ldcg(p.refs + page) == 0;
    int total;
    const int rank = run + block_scan(is_free, warp_tot, total) - 1;
    if (is_free && rank < granted) {
      int lo = 0, hi = n - 1;  // first row whose prefix sum passes the rank
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (want[mid] > rank) hi = mid;
        else lo = mid + 1;
      }
      p.refs[page] = 1;
      give(lo, rank - (lo > 0 ? want[lo - 1] : 0), (int)page);
    }
    run += total;
  }
}

// Rows given twice in one call: the first counts, the others are flagged.
__device__ bool repeated(const int32_t *rows, int i) {
  for (int j = 0; j < i; ++j)
    if (rows[j] == rows[i]) return true;
  return false;
}

__global__ void __launch_bounds__(kPgThreads)
    resize_kernel(const Pool p, const int32_t *__restrict__ rows, const int32_t *__restrict__ lens,
                  int n) {
  extern __shared__ int32_t pg_smem[];
  int32_t *want = pg_smem, *row = want + n, *has = row + n, *target = has + n;
  __shared__ int32_t warp_tot[32];
  __shared__ int lacking;
  pdl_begin();
  const int tid = threadIdx.x;
  if (tid == 0) lacking = 0;
  for (int i = tid; i < n; i += kPgThreads) row[i] = rows[i];
  __syncthreads();
  for (int i = tid; i < n; i += kPgThreads) {
    const int r = row[i], len = lens[i];
    int have = 0, need = 0;
    bool ok = true;
    if (r < 0 || r >= p.rows || repeated(row, i)) {
      ok = false;
      flag_error(p.err, DSB_FLAG_SLOT);
    } else {
      have = min(max(p.held[r], 0), (int)min(p.cols, (int64_t)INT32_MAX));
      need = len < 0 ? -1 : (int)(((int64_t)len + p.bs - 1) / p.bs);
      if (need < 0 || need > p.cols) {
        ok = false;
        flag_error(p.err, DSB_FLAG_POSITION);
      }
    }
    has[i] = have;
    target[i] = ok ? need : -1;
    want[i] = ok ? max(0, need - have) : 0;
  }
  __syncthreads();
  // releases first: a warp a row
  for (int i = tid >> 5; i < n; i += kPgThreads / 32) {
    if (target[i] < 0 || target[i] >= has[i]) continue;
    int32_t *t = p.tables + (int64_t)row[i] * p.stride;
    for (int j = target[i] + (tid & 31); j < has[i]; j += 32) {
      release(p, t[j]);
      t[j] = -1;
    }
    if ((tid & 31) == 0) p.held[row[i]] = target[i];
  }
  __syncthreads();
  const int nfree = free_pages(p, warp_tot);
  scan_rows(want, n, warp_tot);
  __shared__ int granted;
  if (tid == 0) granted = 0;
  __syncthreads();
  // rows in order until the first that does not fit
  for (int i = tid; i < n; i += kPgThreads) {
    const int need = want[i] - (i > 0 ? want[i - 1] : 0);
    if (need == 0) continue;
    if (want[i] <= nfree) {
      atomicMax(&granted, want[i]);
      p.held[row[i]] = target[i];
    } else {
      atomicAdd(&lacking, 1);
    }
  }
  __syncthreads();
  allot(p, want, n, granted, warp_tot, [&](int i, int k, int page) {
    p.tables[(int64_t)row[i] * p.stride + has[i] + k] = page;
  });
  if (tid == 0 && p.status != nullptr) {
    p.status[0] = lacking;
    p.status[1] = nfree - granted;
  }
}

// Per child: parent row, child row (-1: not forked), whole pages, the started
// page's source, its copy and the tokens in it.
struct ForkPlan {
  int32_t parent, child, full, src, dst, tokens;
};

__global__ void __launch_bounds__(kPgThreads)
    fork_plan_kernel(const Pool p, const int32_t *__restrict__ parents,
                     const int32_t *__restrict__ children, const int32_t *__restrict__ lens, int n,
                     ForkPlan *__restrict__ plan) {
  extern __shared__ int32_t pg_smem[];
  int32_t *want = pg_smem, *kid = want + n;
  __shared__ int32_t warp_tot[32];
  __shared__ int lacking, granted;
  pdl_begin();
  const int tid = threadIdx.x;
  if (tid == 0) lacking = granted = 0;
  for (int i = tid; i < n; i += kPgThreads) kid[i] = children[i];
  __syncthreads();
  for (int i = tid; i < n; i += kPgThreads) {
    const int up = parents[i], c = kid[i], len = lens[i];
    ForkPlan f{up, -1, 0, -1, -1, 0};
    if (up < 0 || up >= p.rows || c < 0 || c >= p.rows || repeated(kid, i) || p.held[c] != 0) {
      flag_error(p.err, DSB_FLAG_SLOT);
    } else if (len < 0 || (int64_t)len > (int64_t)p.held[up] * p.bs ||
               (int64_t)len > p.cols * p.bs) {
      flag_error(p.err, DSB_FLAG_POSITION);
    } else {
      f.child = c;
      f.full = len / p.bs;
      f.tokens = len % p.bs;
      if (f.tokens > 0) {
        f.src = p.tables[(int64_t)up * p.stride + f.full];
        if (f.src < 0 || f.src >= p.pages) {
          flag_error(p.err, DSB_FLAG_BLOCK);
          f.child = -1;
          f.tokens = 0;
        }
      }
    }
    want[i] = f.tokens > 0;
    plan[i] = f;
  }
  __syncthreads();
  const int nfree = free_pages(p, warp_tot);
  scan_rows(want, n, warp_tot);
  for (int i = tid; i < n; i += kPgThreads) {
    ForkPlan &f = plan[i];
    if (f.tokens > 0 && want[i] > nfree) {  // no page for it: not forked
      atomicAdd(&lacking, 1);
      f.child = -1;
      f.tokens = 0;
    } else if (f.child >= 0) {
      if (f.tokens > 0) atomicMax(&granted, want[i]);
      p.held[f.child] = f.full + (f.tokens > 0);
    }
  }
  __syncthreads();
  allot(p, want, n, granted, warp_tot, [&](int i, int, int page) {
    plan[i].dst = page;
    p.tables[(int64_t)kid[i] * p.stride + plan[i].full] = page;
  });
  if (tid == 0 && p.status != nullptr) {
    p.status[0] = lacking;
    p.status[1] = nfree - granted;
  }
}

// blockIdx.y: child.  The first blocks along x rename its whole pages (each a
// reference more), the others copy the started page's tokens of the caches.
__global__ void __launch_bounds__(256)
    fork_apply_kernel(const Pool p, const ForkPlan *__restrict__ plan, const Caches caches,
                      int64_t token_bytes, int table_blocks) {
  pdl_begin();
  const ForkPlan f = plan[blockIdx.y];
  if (f.child < 0) return;
  if ((int)blockIdx.x < table_blocks) {
    const int32_t *up = p.tables + (int64_t)f.parent * p.stride;
    int32_t *to = p.tables + (int64_t)f.child * p.stride;
    for (int j = blockIdx.x * 256 + threadIdx.x; j < f.full; j += table_blocks * 256) {
      const int page = up[j];
      to[j] = page;
      if (page >= 0 && page < p.pages)
        atomicAdd(p.refs + page, 1);
      else
        flag_error(p.err, DSB_FLAG_BLOCK);
    }
    return;
  }
  if (f.tokens <= 0) return;
  const int64_t bytes = f.tokens * token_bytes, page_bytes = p.bs * token_bytes;
  for (int c = blockIdx.x - table_blocks; c < caches.n; c += gridDim.x - table_blocks) {
    const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const char *>(caches.p[c]) +
                                                       f.src * page_bytes);
    uint4 *dst = reinterpret_cast<uint4 *>(static_cast<char *>(caches.p[c]) + f.dst * page_bytes);
    for (int64_t i = threadIdx.x; i < bytes / 16; i += 256) dst[i] = src[i];
  }
}

// scratch: [0] pages to move, then sources[N], targets[N], new names[N]
__global__ void __launch_bounds__(kPgThreads)
    compact_plan_kernel(const Pool p, int32_t *__restrict__ scratch) {
  __shared__ int32_t warp_tot[32];
  pdl_begin();
  const int tid = threadIdx.x;
  const int nfree = free_pages(p, warp_tot);
  const int64_t live = p.pages - nfree;
  int32_t *src = scratch + 1, *dst = src + p.pages, *name = dst + p.pages;
  int holes = 0, moved = 0;
  for (int64_t base = 0; base < p.pages; base += kPgThreads) {
    const int64_t page = base + tid;
    const bool in = page < p.pages;
    const bool used = in && p.refs[page] != 0;
    const bool hole = in && !used && page < live, move = used && page >= live;
    int total;
    const int h = holes + block_scan(hole, warp_tot, total) - 1;
    holes += total;
    const int m = moved + block_scan(move, warp_tot, total) - 1;
    moved += total;
    if (hole) dst[h] = (int)page;
    if (move) src[m] = (int)page;
    if (in && !used && page >= live) name[page] = -1;  // no row holds it
  }
  __syncthreads();
  for (int k = tid; k < moved; k += kPgThreads) {
    const int s = src[k], t = dst[k];
    name[s] = t;
    p.refs[t] = p.refs[s];
    p.refs[s] = 0;
  }
  if (tid == 0) {
    scratch[0] = moved;
    if (p.status != nullptr) {
      p.status[0] = 0;
      p.status[1] = nfree;
    }
  }
}

__global__ void __launch_bounds__(256)
    rename_kernel(const Pool p, const int32_t *__restrict__ scratch) {
  pdl_begin();
  const int32_t *name = scratch + 1 + 2 * p.pages;
  const int row = blockIdx.y;
  const int held = min(max(p.held[row], 0), (int)min(p.cols, (int64_t)INT32_MAX));
  int32_t *t = p.tables + (int64_t)row * p.stride;
  // live pages are in front now: an entry that points behind them was moved
  const int64_t live = p.pages - p.status[1];
  for (int j = blockIdx.x * 256 + threadIdx.x; j < held; j += gridDim.x * 256) {
    const int page = t[j];
    if (page < 0 || page >= p.pages)
      flag_error(p.err, DSB_FLAG_BLOCK);
    else if (page >= live)
      t[j] = name[page];
  }
}

// Pages src[k] -> dst[k] of every cache, k < *count (or `n` when null);
// negative entries are skipped, bad ones flagged.
__global__ void __launch_bounds__(256)
    copy_pages_kernel(const Caches caches, int64_t page_bytes, int64_t pages,
                      const int32_t *__restrict__ src, const int32_t *__restrict__ dst,
                      const int32_t *__restrict__ count, int n, int32_t *err) {
  pdl_begin();
  const int64_t total = (int64_t)(count != nullptr ? *count : n) * caches.n;
  for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
    const int64_t k = u / caches.n;
    const int c = (int)(u % caches.n);
    const int s = src[k], t = dst[k];
    if (s < 0 || t < 0) continue;
    if (s >= pages || t >= pages) {
      if (threadIdx.x == 0) flag_error(err, DSB_FLAG_BLOCK);
      continue;
    }
    const uint4 *from = reinterpret_cast<const uint4 *>(static_cast<const char *>(caches.p[c]) +
                                                        s * page_bytes);
    uint4 *to = reinterpret_cast<uint4 *>(static_cast<char *>(caches.p[c]) + t * page_bytes);
    for (int64_t i = threadIdx.x; i < page_bytes / 16; i += 256) to[i] = from[i];
  }
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
  const size_t smem = (size_t)n * 4 * sizeof(int32_t);
  if (int e = ensure_smem((const void *)resize_kernel, smem)) return e;
  launch_kernel(resize_kernel, dim3(1), dim3(kPgThreads), smem, as_stream(stream), p, rows, lens,
                (int)n);
  return check_launch("resize_kernel");
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
  const size_t smem = (size_t)n * 2 * sizeof(int32_t);
  if (int e = ensure_smem((const void *)fork_plan_kernel, smem)) return e;
  launch_kernel(fork_plan_kernel, dim3(1), dim3(kPgThreads), smem, st, p, parents, children, lens,
                (int)n, plan);
  if (int e = check_launch("fork_plan_kernel")) return e;
  if (n == 0) return DSB_OK;
  const int table_blocks = (int)std::min<int64_t>(32, (table_cols + 255) / 256);
  bool first = true;
  auto apply = [&](const Caches &part) {
    const int tb = first ? table_blocks : 0;  // the tables once
    first = false;
    if (tb + part.n > 0)
      launch_kernel(fork_apply_kernel, dim3(tb + part.n, n), dim3(256), 0, st, p,
                    (const ForkPlan *)plan, part, token_bytes, tb);
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
  if (table_rows > 65535) return fail(DSB_ERR_UNSUPPORTED, "grid too large");
  const cudaStream_t st = as_stream(stream);
  launch_kernel(compact_plan_kernel, dim3(1), dim3(kPgThreads), 0, st, p, scratch);
  if (int e = check_launch("compact_plan_kernel")) return e;
  const unsigned gx = (unsigned)std::min<int64_t>(32, (table_cols + 255) / 256);
  launch_kernel(rename_kernel, dim3(gx, (unsigned)table_rows), dim3(256), 0, st, p,
                (const int32_t *)scratch);
  if (int e = check_launch("rename_kernel")) return e;
  each_part(caches, num_caches, [&](const Caches &part) {
    const int64_t units = (num_pages / 2 + 1) * part.n;  // at most half of the pages move
    launch_kernel(copy_pages_kernel, dim3((unsigned)std::min<int64_t>(units, 8L * sm_count())),
                  dim3(256), 0, st, part, token_bytes * block_size, num_pages,
                  (const int32_t *)(scratch + 1), (const int32_t *)(scratch + 1 + num_pages),
                  (const int32_t *)scratch, 0, error_flag);
  });
  return check_launch("copy_pages_kernel");
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
                  dim3(256), 0, as_stream(stream), part, page_bytes, num_pages, src, dst,
                  (const int32_t *)nullptr, (int)n, error_flag);
  });
  return check_launch("copy_pages_kernel");
}
