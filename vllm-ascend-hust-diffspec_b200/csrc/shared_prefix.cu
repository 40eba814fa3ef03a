// Target paged decode attention, with the softmax LSE, for requests that
// share a prefix of their tokens (forked from one prompt, or on one system
// prompt): rows [group_starts[i], group_starts[i + 1]) hold the same tokens
// at positions [0, prefix_lens[i]).
//   out[r, h] = sum_t softmax_t(scale * q[r, h] . k_t) v_t,  t < seq_lens[r]
//   lse[r, h] = log sum_t exp(scale * q[r, h] . k_t)          (natural log)
//
// The work is cut into segments, a run of tokens that a set of query rows
// reads through one table row:
//   * the prefix of a group, with up to 256 of its query rows (rows x the G
//     query heads of a kv head);
//   * the tokens behind it of consecutive rows on one table row (the verify
//     rows of a request), with up to 128 query rows.
// A K/V tile read from HBM thus serves every query row that sees it.  Three
// launches: a plan of the segments (one CTA), the partial sums (one
// persistent CTA an SM, each with an equal share of the work), and the merge
// of the pieces in order.  Which CTA computes what depends on the lengths
// alone, and the pieces are merged in token order: the same call gives the
// same bits.  Back to back: 16 rows on one prefix of 40800 tokens (32/4 heads)
// 37 us, 80 on 32777 90, 64 on two of 65536 (64/8 heads) 244 (0.34 of the
// measured bf16 rate before the second term of the weights is counted).
#include <type_traits>

#include "paged_split.cuh"
#include "tma_umma.cuh"

namespace dsb {
namespace {

constexpr int kSpTile = 32768;      // 128 rows x 128 dims, 16-bit
constexpr int kSpHalf = 16384;      // (queries: 64 dims of all rows, then the other 64)
constexpr int kSpTok = 128;
constexpr int kSpSlots = 5;         // K / V tiles in flight
constexpr int kSpThreads = 384;
constexpr int kSpSmem = 1024 + (2 + kSpSlots) * kSpTile + 256;  // queries, ring, barriers
constexpr int kSpStage = 144;       // bytes: 32 columns of a row, and 16 more for the banks
constexpr float kSpGrow = 8.f;      // log2 of the growth that rescales O
// log2 of what the weights are multiplied by: fp16 has no steps below 2^-24, and
// with the growth above this takes the weights to its upper end, 2^15.
template <typename T> constexpr float kSpUp = std::is_same<T, __half>::value ? 7.f : 0.f;
// The shares are counted in units of 2300 clocks: a tile is one of them, or two
// when both streams take it, and a piece's queries, first loads and sums are
// five.  (640 query rows of a kv head are tiles of both kinds: 88 us against
// 98 with a unit for every tile; 64 rows with 512 tokens of their own behind
// two prefixes of 65536: 191 us with five, 214 with three.)
struct SpCost {
  static constexpr int start = 5;
  int tile;
  __device__ explicit SpCost(int nq) : tile(nq > 128 ? 2 : 1) {}
  __device__ int units(int tiles) const { return tiles * tile + start; }
  // tiles that begin before unit x of a segment's kv head
  __device__ int before(int x) const { return (max(x - start, 0) + tile - 1) >> (tile - 1); }
};

// Tokens [tok0, tok1) for query rows m < nq: (row0 + (q0 + m) / G, head
// (q0 + m) % G).  Tiles start at `base`, tok0 rounded down to a TMA box.
struct alignas(16) SpSeg {
  int32_t row0, q0, nq, trow, tok0, tok1, base;
  int32_t len;     // units of one kv head, 0: nothing to do
  int64_t unit0;   // units before this segment
  int64_t acc;     // first row of its partial sums
  int32_t maxp;    // pieces that one kv head may be cut into
  int32_t pad[3];
};
static_assert(sizeof(SpSeg) == 64, "one segment per 64 bytes");

// The units' even shares, floor and remainder of units / CTAs, and the segment
// that a CTA's first unit is in.
struct alignas(16) SpBegin {
  int64_t share;
  int32_t rest, seg;
};

// Where a row's partial sums are: its group's first prefix segment and row,
// its own segment and its place in it (-1: none).
struct alignas(16) SpRow {
  int32_t row0, pseg, sseg, srow;
};

struct SpArgs {
  TaArgs a;
  const int32_t *prefix_lens, *group_starts;  // (group_starts null: one group)
  int groups, ctas;
  int box;             // tokens of a TMA box: 8 .. 128, dividing the page
  int64_t token_rows;  // num_blocks * block_size
  SpBegin *begin;      // [ctas]
  SpSeg *segs;
  SpRow *rows;
  int32_t *gseg;       // [groups] first prefix segment of each
  int32_t *pieces;     // [segs, kv heads] pieces of a segment, 0 until its last one is there
  float *acc;          // [rows of partial sums, D]
  float2 *ml;          // [rows of partial sums]: maximum (log2), sum
};

// A CTA's first unit, floor(cta * units / ctas), and the CTA that owns unit u
// (64-bit divisions cost more than the loads they wait for).
__device__ __forceinline__ int64_t sp_first(int cta, const SpBegin &x, int ctas) {
  return cta * x.share + (unsigned)(cta * x.rest) / (unsigned)ctas;
}
__device__ __forceinline__ int sp_owner(int64_t u, const SpBegin &x, int ctas) {
  const float units = (float)x.share * (float)ctas + (float)x.rest;
  // floor(((u + 1) * ctas - 1) / units), right to one
  int b = min((int)(((float)(u + 1) * (float)ctas - 1.f) / units), ctas - 1);
  while (b > 0 && sp_first(b, x, ctas) > u) --b;
  while (b + 1 < ctas && sp_first(b + 1, x, ctas) <= u) ++b;
  return b;
}

// Tokens that a table row can address; a few tiles short of 2^31, so that the
// places of a tile that reaches behind them are whole numbers of 32 bits, too.
__device__ __forceinline__ int64_t sp_cap(const TaArgs &a) {
  return min(a.bt_cols * a.bs, (int64_t)INT32_MAX - 4 * kSpTok);
}
// Tokens that a row of L tokens on table row `trow` may see, 0 for a row
// without a valid table row.
__device__ __forceinline__ int sp_sees(const TaArgs &a, int L, int64_t trow, bool report) {
  if (L <= 0) return 0;
  if (trow < 0 || trow >= a.bt_rows) {
    if (report) flag_error(a.err, DSB_FLAG_SLOT);
    return 0;
  }
  const int64_t cap = sp_cap(a);
  if (L > cap) {
    if (report) flag_error(a.err, DSB_FLAG_POSITION);
    return (int)cap;
  }
  return L;
}
__device__ __forceinline__ int64_t sp_table_row(const TaArgs &a, int r) {
  return a.trows != nullptr ? a.trows[r] : r;
}

// ------------------------------------------------------------------- plan
// One CTA of 256 threads: the plan's time is the latency of its dependent
// reads and of its barriers (1024 threads: 1200 clocks a scan; 9 us in all
// for 16 rows).  What it reads again is kept in shared memory: the first
// kPlanKeep groups and segments, and the rows of a turn of the loop.
constexpr int kPlanThreads = 256, kPlanKeep = 1024;

// Inclusive scan over the block (sum, or maximum); the last value in `total`.
template <typename V, bool MAX> __device__ V plan_scan(V v, V *warp_v, V &total) {
  constexpr int kWarps = kPlanThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto join = [](V x, V y) { return MAX ? (x > y ? x : y) : x + y; };
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = join(x, v);
  }
  if (lane == 31) warp_v[warp] = v;
  __syncthreads();
  V before = v;
  total = warp_v[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) {
    if (w == warp) before = join(total, v);
    total = join(total, warp_v[w]);
  }
  __syncthreads();  // (warp_v is written again by the next scan)
  return warp > 0 ? before : v;
}

__global__ void __launch_bounds__(kPlanThreads) shared_prefix_plan_kernel(const SpArgs s) {
  __shared__ int32_t warp_i[kPlanThreads / 32];
  __shared__ int64_t warp_l[kPlanThreads / 32];
  __shared__ int32_t s_start[kPlanKeep + 1], s_prefix[kPlanKeep], s_gseg[kPlanKeep];
  __shared__ int32_t s_trow[kPlanThreads + 128], s_seen[kPlanThreads + 128];
  __shared__ int32_t s_len[kPlanKeep], s_nq[kPlanKeep];
  __shared__ int64_t s_unit0[kPlanKeep];
  const TaArgs &a = s.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.hq / a.hk, run_rows = 128 / G;
  const int64_t cap = sp_cap(a);
  pdl_begin();

  // The rows of a turn: what each sees, and its table row (-1: none).  A run
  // may reach into the rows of the next turn.
  auto read_rows = [&](int base, int L, int64_t t) {  // (of the thread's first row)
    for (int i = tid; i < kPlanThreads + run_rows && base + i < a.rows; i += kPlanThreads) {
      if (i >= kPlanThreads) L = a.seq[base + i], t = sp_table_row(a, base + i);
      s_seen[i] = sp_sees(a, L, t, i < kPlanThreads);
      s_trow[i] = t >= 0 && t < a.bt_rows ? (int)t : -1;
    }
  };
  // what the first turns need is read at the same time
  const int L0 = tid < a.rows ? a.seq[tid] : 0;
  const int64_t t0 = tid < a.rows ? sp_table_row(a, tid) : -1;
  const bool first_groups = tid <= s.groups, starts_given = s.group_starts != nullptr;
  const int at0 = first_groups && starts_given ? s.group_starts[tid] : 0;
  const int before0 = first_groups && starts_given && tid > 0 ? s.group_starts[tid - 1] : 0;
  const int prefix0 = tid < s.groups ? s.prefix_lens[tid] : 0;
  read_rows(0, L0, t0);
  // the groups; if they do not ascend within the rows, nothing is shared
  bool bad = false;
  for (int i = tid; i <= s.groups; i += kPlanThreads) {
    const bool mine = i == tid;
    const int at = !starts_given ? (i == 0 ? 0 : a.rows) : mine ? at0 : s.group_starts[i];
    if (i <= kPlanKeep) s_start[i] = at;
    if (i < s.groups && i < kPlanKeep) s_prefix[i] = mine ? prefix0 : s.prefix_lens[i];
    bad |= at < 0 || at > a.rows ||
           (i > 0 && starts_given && (mine ? before0 : s.group_starts[i - 1]) > at);
  }
  for (int r = tid; r < a.rows; r += kPlanThreads) s.rows[r] = SpRow{0, -1, -1, 0};
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) flag_error(a.err, DSB_FLAG_SLOT);
  const int groups = bad ? 0 : s.groups;
  auto start_of = [&](int i) { return i <= kPlanKeep ? s_start[i] : s.group_starts[i]; };
  auto prefix_of = [&](int i) {
    const int p = i < kPlanKeep ? s_prefix[i] : s.prefix_lens[i];
    return (int)min((int64_t)max(p, 0), cap);
  };
  auto gseg_of = [&](int i) { return i < kPlanKeep ? s_gseg[i] : s.gseg[i]; };
  auto keep = [&](int i, const SpSeg &g) {
    s.segs[i] = g;
    if (i < kPlanKeep) s_len[i] = g.len, s_nq[i] = g.nq;
  };

  // prefix segments: each group's query rows, 256 at a time
  int nprefix = 0;
  for (int base = 0; base < groups; base += kPlanThreads) {
    const int i = base + tid;
    int tiles = 0, total, cum;
    if (i < groups) tiles = (int)(((int64_t)(start_of(i + 1) - start_of(i)) * G + 255) / 256);
    if (groups == 1) {
      cum = tiles;
      total = (int)(((int64_t)(start_of(1) - start_of(0)) * G + 255) / 256);
    } else {
      cum = plan_scan<int32_t, false>(tiles, warp_i, total);
    }
    if (i < groups) {
      s.gseg[i] = nprefix + cum - tiles;
      if (i < kPlanKeep) s_gseg[i] = nprefix + cum - tiles;
    }
    nprefix += total;
  }
  __syncthreads();

  // the prefix segments, a warp each (the last ones first: the first warps have
  // the rows): as far as any of their rows sees, through the table row of one
  // that sees as far (a shorter one's need not name the pages behind it)
  for (int p = kPlanThreads / 32 - 1 - warp; p < nprefix; p += kPlanThreads / 32) {
    int x = 0, y = groups;
    while (x < y) {
      const int mid = (x + y) / 2;
      if (gseg_of(mid) <= p) x = mid + 1;
      else y = mid;
    }
    // (groups without rows share their segment's number with the next one)
    const int gi = x - 1, lo = start_of(gi), prefix = prefix_of(gi);
    SpSeg g{};
    g.row0 = lo, g.q0 = (p - gseg_of(gi)) * 256;
    g.nq = (int)min((int64_t)256, (int64_t)(start_of(gi + 1) - lo) * G - g.q0);
    const int r0 = lo + g.q0 / G, r1 = lo + (g.q0 + g.nq - 1) / G;
    int most = 0, trow = 0;  // of the lane's rows, its first that sees most
    for (int r = r0 + lane; r <= r1; r += 32) {
      int64_t t;
      int L;
      if (r < kPlanThreads) {
        L = s_seen[r], t = s_trow[r];
      } else {
        t = sp_table_row(a, r);
        L = sp_sees(a, a.seq[r], t, false);
      }
      L = min(L, prefix);
      if (L > most) most = L, trow = (int)t;
    }
    const int lane_most = most;
    most = __reduce_max_sync(0xffffffffu, most);
    const unsigned whole = __ballot_sync(0xffffffffu, lane_most == most);
    trow = __shfl_sync(0xffffffffu, trow, __ffs(whole) - 1);
    g.trow = trow;
    g.tok1 = most;
    g.len = most > 0 ? SpCost(g.nq).units((most + kSpTok - 1) / kSpTok) : 0;
    if (lane == 0) keep(p, g);
  }

  // segments of the rows' own tokens: rows of a group on one table row
  int nown = 0, carry = -1;
  for (int base = 0; base < a.rows; base += kPlanThreads) {
    if (base > 0) {
      __syncthreads();
      const bool mine = base + tid < a.rows;
      read_rows(base, mine ? a.seq[base + tid] : 0, mine ? sp_table_row(a, base + tid) : -1);
      __syncthreads();
    }
    const int r = base + tid;
    int gi = -1, lo = 0, hi = a.rows, prefix = 0, trow = -1;
    bool starts = false;
    if (r < a.rows) {
      if (groups > 0) {  // the last group that begins at or before the row
        int x = 0, y = groups;
        while (x < y) {
          const int mid = (x + y) / 2;
          if (start_of(mid) <= r) x = mid + 1;
          else y = mid;
        }
        gi = x - 1;
        if (gi >= 0) lo = start_of(gi), hi = start_of(gi + 1);
        if (gi < 0 || r >= hi) {  // outside every group: no shared prefix
          lo = gi < 0 ? 0 : hi;
          hi = gi < 0 ? start_of(0) : a.rows;
          gi = -1;
        }
      }
      if (gi >= 0) {
        prefix = prefix_of(gi);
        s.rows[r].row0 = lo;
        s.rows[r].pseg = gseg_of(gi);
      }
      trow = s_trow[tid];
      int before = -1;
      if (r > lo) {
        if (tid > 0) {
          before = s_trow[tid - 1];
        } else {
          const int64_t t = sp_table_row(a, r - 1);
          before = t >= 0 && t < a.bt_rows ? (int)t : -1;
        }
      }
      starts = r == lo || before != trow;
    }
    int total;
    const int first = max(carry, plan_scan<int32_t, true>(starts ? r : -1, warp_i, total));
    carry = max(carry, total);
    // a run is taken run_rows rows at a time, by the first of them
    const bool leads = trow >= 0 && (r - first) % run_rows == 0;
    int nrows = 0, most = 0;
    if (leads)
      for (; nrows < run_rows && r + nrows < hi && s_trow[tid + nrows] == trow; ++nrows)
        most = max(most, s_seen[tid + nrows]);
    const bool has = leads && most > prefix;
    const int at = nprefix + nown + plan_scan<int32_t, false>(has ? 1 : 0, warp_i, total) - 1;
    nown += total;
    if (has) {
      SpSeg g{};
      g.row0 = r, g.q0 = 0, g.nq = nrows * G, g.trow = trow;
      g.tok0 = prefix, g.tok1 = most;
      g.base = prefix / s.box * s.box;
      g.len = SpCost(g.nq).units((most - g.base + kSpTok - 1) / kSpTok);
      keep(at, g);
      for (int j = 0; j < nrows; ++j) {
        s.rows[r + j].sseg = at;
        s.rows[r + j].srow = j;
      }
    }
  }
  __syncthreads();

  // units before each segment, then the places of their partial sums
  const int nseg = nprefix + nown;
  auto len_of = [&](int i) { return i < kPlanKeep ? s_len[i] : s.segs[i].len; };
  auto nq_of = [&](int i) { return i < kPlanKeep ? s_nq[i] : s.segs[i].nq; };
  int64_t units = 0, total = 0;
  for (int base = 0; base < nseg; base += kPlanThreads) {
    const int i = base + tid;
    const int64_t mine = i < nseg ? (int64_t)len_of(i) * a.hk : 0;
    const int64_t u0 = units + plan_scan<int64_t, false>(mine, warp_l, total) - mine;
    units += total;
    if (i < nseg) {
      s.segs[i].unit0 = u0;
      if (i < kPlanKeep) s_unit0[i] = u0;
    }
  }
  const float share = units > 0 ? (float)s.ctas / (float)units : 0.f;
  int64_t sums = 0;
  for (int base = 0; base < nseg; base += kPlanThreads) {
    const int i = base + tid;
    const int len = i < nseg ? len_of(i) : 0;
    // pieces that a kv head's `len` units can fall into: two more than its
    // share of the CTAs (one more again for the rounding of the share)
    const int maxp = len > 0 ? (int)((float)len * share) + 3 : 0;
    const int64_t rows = len > 0 ? (int64_t)a.hk * maxp * nq_of(i) : 0;
    const int64_t acc = sums + plan_scan<int64_t, false>(rows, warp_l, total) - rows;
    sums += total;
    if (i < nseg) {
      s.segs[i].acc = acc;
      s.segs[i].maxp = maxp;
    }
  }
  // no pieces yet: a CTA that gives up on a wait leaves its segments without
  for (int64_t i = tid; i < (int64_t)nseg * a.hk; i += kPlanThreads) s.pieces[i] = 0;
  // where each CTA begins: the last segment that starts at or before its first
  // unit (an empty one starts where the next does)
  SpBegin shares{units / s.ctas, (int)(units % s.ctas), 0};
  for (int b = tid; b < s.ctas; b += kPlanThreads) {
    const int64_t u = sp_first(b, shares, s.ctas);
    int x = 0, y = nseg;
    while (x < y) {
      const int mid = (x + y) / 2;
      if ((mid < kPlanKeep ? s_unit0[mid] : s.segs[mid].unit0) <= u) x = mid + 1;
      else y = mid;
    }
    shares.seg = max(x - 1, 0);
    s.begin[b] = shares;
  }
}

// ---------------------------------------------------------- partial sums
// A few tries before the bounded wait, whose timer reads cost more than a try.
__device__ __forceinline__ bool sp_wait(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
  }
  return mbar_wait(bar, parity);
}

// Slots of the ring are taken in turn by both loaders and used by both streams,
// so one of them may come to a slot before the turn ahead of its own has ended,
// or even begun, and a wait on a parity alone would be satisfied by the turn
// before that.  `turns[slot]` counts the loads that were asked for; whoever
// needs load i waits for it first.
__device__ __forceinline__ bool sp_wait_turn(const volatile int *turns, int i, int count) {
  uint64_t t0 = 0;
  for (int k = 0; turns[i % kSpSlots] < count; ++k) {  // (bounded as mbar_wait)
    if (k == kWaitSpins) return false;
    if ((k & 63) == 63) {
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > kWaitNs) return false;
    }
  }
  return true;
}
// Load i has landed; its slot may be filled with load i.
__device__ __forceinline__ bool sp_wait_load(const volatile int *turns, uint32_t full, int i) {
  return sp_wait_turn(turns, i, i / kSpSlots + 1) &&
         sp_wait(full + 8 * (i % kSpSlots), (uint32_t)(i / kSpSlots) & 1u);
}
__device__ __forceinline__ bool sp_wait_slot(const volatile int *turns, uint32_t empty, int i) {
  return i < kSpSlots || (sp_wait_turn(turns, i, i / kSpSlots) &&
                          sp_wait(empty + 8 * (i % kSpSlots), (uint32_t)(i / kSpSlots - 1) & 1u));
}

__device__ __forceinline__ float sp_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

#define SP_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), \
                    "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define SP_U8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), \
                    "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of this thread's tensor-memory row; the caller waits.
__device__ __forceinline__ void sp_ld32(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : SP_R8(r, 0), SP_R8(r, 8), SP_R8(r, 16), SP_R8(r, 24)
      : "r"(addr));
}
__device__ __forceinline__ void sp_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::SP_U8(r, 0),
      SP_U8(r, 8), SP_U8(r, 16), SP_U8(r, 24), "r"(addr)
      : "memory");
}
#define SP_M8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), \
                    "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
// The loads are done: `r` holds its columns (named as an operand, so that
// nothing that reads it moves before the wait).
__device__ __forceinline__ void sp_wait_ld(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : SP_M8(r, 0), SP_M8(r, 8), SP_M8(r, 16), SP_M8(r, 24)::"memory");
}
__device__ __forceinline__ void sp_ld16(uint32_t addr, uint32_t *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : SP_R8(r, 0), SP_R8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void sp_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15};" ::SP_U8(r, 0),
      SP_U8(r, 8), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void sp_wait_ld16(uint32_t *r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : SP_M8(r, 0), SP_M8(r, 8)::"memory");
}
__device__ __forceinline__ void sp_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// A box of a head's tokens: x (64 dims, two halves), 8-token rows from `row8`.
// It lands as [8 tokens][half][8 rows of 128 bytes] (swizzled atoms of 1 KB):
// one box a page, with both halves of the head's 256 bytes.
__device__ __forceinline__ void sp_load(uint32_t dst, const CUtensorMap *map, int row8, int head,
                                        uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %2, %2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(row8), "r"(head), "r"(bar)
      : "memory");
}
// D[tmem] (+)= A[smem] . B[smem], and A[tmem] . B[smem], by the one thread
// whose `one` is set; descriptors as words.  The whole warp comes here with the
// same values, so they stay in the registers that the products are issued from:
// under a branch on the lane a tile's products were issued in 1180 clocks, in
// 955 this way.
__device__ __forceinline__ void sp_umma_ss(uint32_t one, uint32_t d, uint32_t a_lo, uint32_t a_hi,
                                           uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                                           bool accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 a, b;\n setp.ne.b32 p, %6, 0;\n setp.ne.b32 e, %7, 0;\n"
      " mov.b64 a, {%1, %2};\n mov.b64 b, {%3, %4};\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n}" ::"r"(d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(one)
      : "memory");
}
__device__ __forceinline__ void sp_umma_ts(uint32_t one, uint32_t d, uint32_t a, uint32_t b_lo,
                                           uint32_t b_hi, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n .reg .b64 b;\n setp.ne.b32 p, %5, 0;\n setp.ne.b32 e, %6, 0;\n"
      " mov.b64 b, {%2, %3};\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(one)
      : "memory");
}
__device__ __forceinline__ void sp_commit(uint32_t one, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
      "r"(one)
      : "memory");
}
__device__ __forceinline__ void sp_arrive(uint32_t one, uint32_t bar) {
  asm volatile(
      "{\n .reg .pred e;\n setp.ne.b32 e, %1, 0;\n @e mbarrier.arrive.shared::cta.b64 _, [%0];\n}" ::"r"(
          bar),
      "r"(one)
      : "memory");
}
// one lane of a warp
__device__ __forceinline__ uint32_t sp_elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}" : "=r"(one));
  return one;
}

// d = max(a, b, c)
__device__ __forceinline__ float sp_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 32 bytes of a row (32-byte aligned)
__device__ __forceinline__ void sp_st_global8(float *p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]),
               "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// A CTA's share of a segment's kv head: tiles [t0, t0 + n) from `base`, those
// whose first units it has, and the index-th of the shares that have tiles.
struct SpPiece {
  SpSeg g;
  int seg, h, t0, n, index;
};

// The pieces of this CTA, in order; every role walks them for itself.
struct SpWalk {
  int64_t u, end;
  SpBegin share;
  int seg;
  __device__ void begin(const SpArgs &s) {
    share = s.begin[blockIdx.x];
    seg = share.seg;
    u = sp_first(blockIdx.x, share, s.ctas);
    end = sp_first(blockIdx.x + 1, share, s.ctas);
  }
  __device__ bool next(const SpArgs &s, SpPiece &p) {
    while (u < end) {
      p.g = s.segs[seg];
      if (u >= p.g.unit0 + (int64_t)p.g.len * s.a.hk) {
        ++seg;
        continue;
      }
      const int64_t off = u - p.g.unit0;
      p.h = (int)((float)off / (float)p.g.len);  // right to one
      if (p.h * (int64_t)p.g.len > off) --p.h;
      if ((p.h + 1) * (int64_t)p.g.len <= off) ++p.h;
      const int a = (int)(off - (int64_t)p.h * p.g.len);
      const int b = (int)min((int64_t)p.g.len, a + (end - u));
      u += b - a;
      const SpCost cost(p.g.nq);
      p.t0 = cost.before(a);
      p.n = cost.before(b) - p.t0;
      if (p.n <= 0) continue;
      p.seg = seg;
      // (shares below a tile: every tile is a piece; else every share between
      // the first and the last that have tiles has some)
      p.index = share.share < cost.tile
                    ? p.t0
                    : (int)blockIdx.x -
                          sp_owner(p.g.unit0 + (int64_t)p.h * p.g.len + cost.start, share, s.ctas);
      return true;
    }
    return false;
  }
};

// Warps 0-3 and 4-7 are two softmax streams; warps 8 and 10 load keys and
// values, warps 9 and 11 issue the products of a stream each (the waits of one
// pass beside the products of the other).  A stream takes a 128-token tile in
// two halves, which alternate between two places of its tensor memory:
//   S[128 x 64] = Q . K^T                 (tensor memory, fp32)
//   P = exp2(scale S - m), m the row's running maximum; a thread has a row
//   O[128 x 128] += P . V                 (A = P from tensor memory)
// While the exponentials of one half are taken, the other half's P . V and
// next Q . K^T run, so a stream's softmax hardly waits for its own products
// (4700 clocks for a tile of each stream; whole tiles, whose products take a
// quarter less of the tensor pipe, 4900, two fifths of it that wait).
// P takes S's place as two 16-bit terms, hi + lo (the weights keep ~16 bits;
// one term alone costs the output half a step more), so P . V is two
// products.  O is rescaled only when a row's maximum has grown by more than
// 2^8 since the last time: until then P stays below 2^8, in fp32 sums.  In fp16,
// whose steps end at 2^-24, P is 2^7 times that: a weight is then off by at most
// 2^-17 of itself or 2^-32 of the row's largest (without, 2^-25 of it, and the
// tokens 17 nats below one that dominates a piece were lost to the output and
// not to the sum: 4e-5 of 1.7e-4 for 7000 such tokens).
//   up to 128 query rows in the segment: the streams take its even and odd
//   tiles, and their sums are joined at the piece's end;
//   more: each stream has 128 of the query rows, and takes every tile.
// K and V tiles pass through one ring of 32 KB slots in the order of use; the
// loads of a piece begin while the one before it is still being computed.
template <typename T>
__global__ void __launch_bounds__(kSpThreads, 1)
    shared_prefix_kernel(const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const SpArgs s) {
  const TaArgs &a = s.a;
  extern __shared__ uint8_t sp_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(sp_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t s_q = smem_u32(smem), s_kv = s_q + 2 * kSpTile;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + (2 + kSpSlots) * kSpTile);
  const uint32_t full = smem_u32(bars), empty = full + 8 * kSpSlots, s_full = empty + 8 * kSpSlots,
                 p_ready = s_full + 32, o_done = p_ready + 32, q_ready = o_done + 8,
                 joint = q_ready + 8, drain = joint + 8,
                 pv_done = drain + 8;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_turns[kSpSlots];
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int G = a.hq / a.hk;

  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tk)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tv)) : "memory");
    for (int i = 0; i < kSpSlots; ++i) {
      mbar_init(full + 8 * i);
      mbar_init_count(empty + 8 * i, 2);  // both streams, or one of them twice
    }
    for (int i = 0; i < 4; ++i) mbar_init(s_full + 8 * i);  // [stream][half]
    for (int i = 0; i < 4; ++i) mbar_init_count(p_ready + 8 * i, 128);
    mbar_init_count(o_done, 2);
    mbar_init_count(q_ready, 256);
    mbar_init_count(joint, 256);
    mbar_init_count(drain, 2);
    for (int i = 0; i < 4; ++i) mbar_init(pv_done + 8 * i);  // [stream][half]
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
    for (int i = 0; i < kSpSlots; ++i) s_turns[i] = 0;
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&s_tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  SpWalk walk;
  auto stop = [&]() {
    atomicExch(&s_abort, 1);
    flag_error(a.err, DSB_FLAG_TIMEOUT);
  };
  int pieces = 0;
  SpPiece p;

  if (warp == 8 || warp == 10) {  // the keys, and the values
    pdl_begin();
    walk.begin(s);
    const bool is_v = warp == 10;
    const CUtensorMap *map = is_v ? &tv : &tk;
    const int boxes = kSpTok / s.box;  // of a tile, at most 16: a lane each
    int i0 = 0;  // loads of the pieces before
    bool bad = false, ok = true;
    while (ok && walk.next(s, p)) {
      const int32_t *bt = a.bt + (int64_t)p.g.trow * a.bt_stride;
      const bool two = p.g.nq > 128;
      // where lane's box of tile j begins, in 8-token rows of the cache
      auto place = [&](int j) {
        const int tok = p.g.base + (p.t0 + j) * kSpTok + lane * s.box;
        if (lane >= boxes || tok >= p.g.tok1) return (int)(s.token_rows / 8);  // out of range: zeros
        const int64_t page = bt[tok / a.bs];
        if (page < 0 || page >= a.nblocks) {
          bad = true;
          return (int)(s.token_rows / 8);
        }
        return (int)((page * a.bs + tok % a.bs) / 8);
      };
      int at = place(0);
      for (int j = 0; j < p.n; ++j) {
        // loads in the order of use: K0 V0 K1 V1 ..., or K0 K1 V0 K2 V1 ...
        const int i = i0 + (is_v ? (two ? 2 * j + 1 : min(2 * j + 2, 2 * p.n - 1))
                                 : (two ? 2 * j : (j < 2 ? j : 2 * j - 1)));
        const int slot = i % kSpSlots;
        ok = sp_wait_slot(s_turns, empty, i);
        ok = __all_sync(0xffffffffu, ok && !*reinterpret_cast<volatile int *>(&s_abort));
        if (!ok) break;
        const uint32_t bar = full + 8 * slot;
        if (lane == 0) {
          mbar_expect_tx(bar, kSpTile);
          *reinterpret_cast<volatile int *>(s_turns + slot) = i / kSpSlots + 1;
        }
        __syncwarp();
        if (lane < boxes) sp_load(s_kv + slot * kSpTile + lane * s.box * 256, map, at, p.h, bar);
        if (j + 1 < p.n) at = place(j + 1);
      }
      i0 += 2 * p.n;
    }
    if (bad) flag_error(a.err, DSB_FLAG_BLOCK);
    if (!ok && lane == 0) stop();
  } else if (warp == 9 || warp == 11) {
    const int st = warp == 11;
    const uint32_t qk = umma_idesc<T, 64>(false);
    const uint32_t pv = umma_idesc<T, 128>(false) | (1u << 16);  // V is dim-contiguous
    // Operand descriptors as two words; only the address (16-byte units, in
    // the low word) changes, so a product costs two additions to issue.
    constexpr uint32_t kHi = (1u << 14) | (2u << 29);  // version, 128-byte swizzle
    constexpr uint32_t kHiQ = kHi | 1024 / 16, kHiKv = kHi | 2048 / 16;
    const uint32_t one = sp_elect(), ts = __reduce_max_sync(0xffffffffu, tmem) + st * 128;
    int i0 = 0, tiles = 0;  // loads, and this stream's tiles, of the pieces before
    bool ok = true, rehearsal = true;
    // S of the halves of a stream's first tile, then O of a half and S of the
    // same half of its next tile in turn, the streams taking turns.  `e` counts
    // the tiles of both, a stream's are those of its parity.
    while (ok) {
      bool two = false;
      int n = 2;
      if (!rehearsal) {
        if (!__any_sync(0xffffffffu, walk.next(s, p))) break;
        n = __reduce_max_sync(0xffffffffu, p.n);
        two = __reduce_max_sync(0xffffffffu, p.g.nq) > 128;
        ok = __all_sync(0xffffffffu, sp_wait(q_ready, (uint32_t)pieces & 1u));
        if (!ok) break;
      }
      const int all = two ? 2 * n : n;
      for (int u = 0; ok && u < 2 * ((all - st + 1) / 2 + 1); ++u) {
        const int half = u & 1, k = (u >> 1) - 1, e = 2 * k + st;
        const uint32_t th = ts + half * 64;
        if (k >= 0) {  // O, this half of the stream's tile k
          const int v = i0 + (two ? e | 1 : min(2 * e + 2, 2 * n - 1));  // the load of its V
          const uint32_t slot = (uint32_t)v % kSpSlots;
          const uint32_t b0 =
              ((s_kv + slot * kSpTile + half * (kSpTile / 2)) >> 4) | (1024 / 16) << 16;
          if (!rehearsal) {
            ok = (half == 1 || sp_wait_load(s_turns, full, v)) &&
                 sp_wait(p_ready + 16 * st + 8 * half, (uint32_t)(tiles + k) & 1u);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
          }
          tc_fence_after();
#pragma unroll
          for (int x = 0; x < 8; ++x) {  // 16 tokens, the hi terms, then the lo ones
            const int c = x >> 1;
            sp_umma_ts(one, ts + 256, th + (c >> 1) * 32 + (c & 1) * 8 + (x & 1) * 16,
                       b0 + c * (4096 / 16), kHiKv, pv, x + half + k > 0);
          }
          if (!rehearsal) {
            sp_commit(one, pv_done + 16 * st + 8 * half);
            if (half == 1) {
              sp_commit(one, empty + 8 * slot);
              if (!two) sp_arrive(one, empty + 8 * slot);
            }
          }
        }
        if (e + 2 < all) {  // S, this half of its next tile
          const int kl = i0 + (two ? (e + 2) & ~1 : (k < 0 ? e + 2 : 2 * e + 3));  // the load of its K
          const uint32_t slot = (uint32_t)kl % kSpSlots;
          const uint32_t b0 = ((s_kv + slot * kSpTile + half * (kSpTile / 2)) >> 4) | 1u << 16;
          // one query tile alternates between the two places
          const uint32_t a0 = ((s_q + (two ? st : pieces & 1) * kSpTile) >> 4) | 1u << 16;
          if (!rehearsal) {
            ok = __all_sync(0xffffffffu, half == 1 || sp_wait_load(s_turns, full, kl));
            if (!ok) break;
          }
          tc_fence_after();
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const uint32_t d = (x & 3) * (32 / 16);
            sp_umma_ss(one, th, a0 + (x >> 2) * (kSpHalf / 16) + d, kHiQ,
                       b0 + (x >> 2) * (1024 / 16) + d, kHiKv, qk, x > 0);
          }
          if (!rehearsal) {
            sp_commit(one, s_full + 16 * st + 8 * half);
            if (half == 1) {
              sp_commit(one, empty + 8 * slot);
              if (!two) sp_arrive(one, empty + 8 * slot);
            }
          }
        }
      }
      if (!ok) break;
      if (rehearsal) {  // (on whatever shared memory holds; the sums are not used)
        rehearsal = false;
        sp_commit(one, drain);
        ok = __all_sync(0xffffffffu, sp_wait(drain, 0));
        pdl_begin();
        walk.begin(s);
        continue;
      }
      i0 += 2 * n;
      tiles += (all - st + 1) / 2;
      sp_commit(one, o_done);
      ++pieces;
    }
    if (!ok && lane == 0) stop();
  } else if (warp < 8) {
    const int stream = warp >> 2, m128 = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + stream * 128, to = ts + 256;
    int i0 = 0, kt = 0;  // loads and this stream's tiles of the pieces before
    int joints = 0;
    bool ok = true;
    auto both = [&]() {  // all 256 threads are here (a bounded wait, unlike bar.sync)
      mbar_arrive(joint);
      ok = __all_sync(0xffffffffu, sp_wait(joint, (uint32_t)joints++ & 1u));
    };
    // A piece's queries, swizzled as the operand wants them, 16 rows at a time
    // (places behind nq keep what they hold: a query row meets only its own
    // sums).  One query tile alternates between the two places.
    const int step_row = 16 / G, step_head = 16 - step_row * G;
    auto fetch = [&](const SpPiece &x, int place) {
      const bool pair = x.g.nq > 128;
      const int c = tid & 15, first = x.g.q0 + (tid >> 4);
      int row = first / G, head = first - row * G;
#pragma unroll 1
      for (int r = tid >> 4; r - (tid >> 4) < x.g.nq; r += 16) {
        const uint32_t dst = s_q + (pair ? r >> 7 : place & 1) * kSpTile;
        const T *src = static_cast<const T *>(a.q) +
                       ((int64_t)(x.g.row0 + row) * a.hq + x.h * G + head) * kTaD + c * 8;
        if (r < x.g.nq)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           dst + (c >> 3) * kSpHalf + (r & 127) * 128 + (((c & 7) ^ (r & 7)) * 16)),
                       "l"(src)
                       : "memory");
        row += step_row, head += step_head;
        if (head >= G) head -= G, ++row;
      }
      cp_async_commit();
    };
    auto fetched = [&]() {
      cp_async_wait<0>();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(q_ready);
    };
    // The first turn of the loop is a rehearsal on whatever the tensor memory
    // holds, stores nothing and brings the instructions in (~7000 clocks of
    // misses) while the plan is still being made.
    bool rehearsal = true, has_next = false, early = false;
    SpPiece after;
    p = SpPiece{};
    p.n = 1;
    p.g.nq = 128;
    p.g.tok1 = kSpTok;
    // this thread's query row of a piece; the tokens [tok0, sees) are what it sees
    auto query_row = [&](const SpPiece &x) { return (x.g.nq > 128 ? stream * 128 : 0) + m128; };
    auto sees = [&](const SpPiece &x) {
      if (query_row(x) >= x.g.nq) return 0;
      const int row = x.g.row0 + (x.g.q0 + query_row(x)) / G;
      return min(sp_sees(a, a.seq[row], sp_table_row(a, row), false), x.g.tok1);
    };
    int lim = kSpTok;
    while (ok) {
      const int n = p.n, nq = p.g.nq;
      const bool two = nq > 128;
      const int m = query_row(p);
      const bool mine = m < nq && !rehearsal;
      if (!rehearsal && !early) {
        fetch(p, pieces);
        lim = sees(p);  // (beside the copies)
        fetched();
      }
      const bool works = __any_sync(0xffffffffu, m < nq);
      const int count = rehearsal ? 1 : two ? n : (n - stream + 1) / 2;
      float m_ref = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int u = 0; u < 2 * count; ++u) {
        const int k = u >> 1, half = u & 1, j = two ? k : 2 * k + stream;
        const int T0 = p.g.base + (p.t0 + j) * kSpTok;
        const uint32_t th = ts + half * 64;
        if (!rehearsal) {
          ok = __all_sync(0xffffffffu, sp_wait(s_full + 16 * stream + 8 * half, (uint32_t)(kt + k) & 1u));
          if (!ok) break;
          tc_fence_after();
          // What a page holds behind the segment's end has weights of zero, but
          // zero times what lies there may not be: those values become zeros
          // (two streams write theirs both, each before its own products).
          if (half == 0 && T0 + kSpTok > p.g.tok1) {
            const int i = i0 + (two ? 2 * j + 1 : min(2 * j + 2, 2 * n - 1));
            ok = __all_sync(0xffffffffu, sp_wait_load(s_turns, full, i));
            if (!ok) break;
            const uint32_t v = s_kv + (i % kSpSlots) * kSpTile;
            for (int z = (p.g.tok1 - T0) * 8 + m128; z < kSpTok * 8; z += 128) {
              const uint32_t at = v + (z >> 6) * 2048 + (z & 63) * 16;
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at + 1024), "r"(0u)
                           : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        if (works) {
          uint32_t x0[32], x1[32];
          sp_ld32(th, x0);
          sp_ld32(th + 32, x1);
          // columns of this half that the row sees
          const int from = min(max(p.g.tok0 - T0 - half * 64, 0), 64);
          const int till = min(max((rehearsal ? kSpTok : lim - T0) - half * 64, 0), 64);
          sp_wait_ld(x0);
          sp_wait_ld(x1);
          if (!__all_sync(0xffffffffu, from <= 0 && till >= 64)) {
            const uint64_t seen = (till < 64 ? (1ull << till) - 1 : ~0ull) &
                                  (from < 64 ? ~((1ull << from) - 1) : 0ull);
            const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (!(s0 >> i & 1)) x0[i] = __float_as_uint(-INFINITY);
              if (!(s1 >> i & 1)) x1[i] = __float_as_uint(-INFINITY);
            }
          }
          float t0 = -INFINITY, t1 = -INFINITY, t2 = -INFINITY, t3 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            t0 = sp_max3(t0, __uint_as_float(x0[i]), __uint_as_float(x0[i + 1]));
            t1 = sp_max3(t1, __uint_as_float(x0[i + 2]), __uint_as_float(x0[i + 3]));
            t2 = sp_max3(t2, __uint_as_float(x1[i]), __uint_as_float(x1[i + 1]));
            t3 = sp_max3(t3, __uint_as_float(x1[i + 2]), __uint_as_float(x1[i + 3]));
          }
          const float top = fmaxf(sp_max3(t0, t1, t2), t3) * a.scale_log2;
          if (__any_sync(0xffffffffu, top > m_ref + kSpGrow)) {
            const float now = fmaxf(m_ref, top);
            const float f = now == -INFINITY ? 1.f : sp_exp2(m_ref - now);
            m_ref = now;
            l *= f;
            if (u > 0 && !rehearsal) {
              // O is whole once the half before this one has been added
              ok = __all_sync(0xffffffffu, sp_wait(pv_done + 16 * stream + 8 * (half ^ 1),
                                                   (uint32_t)(kt + ((u - 1) >> 1)) & 1u));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < 128; c += 16) {
                uint32_t o[16];
                sp_ld16(to + c, o);
                sp_wait_ld16(o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                sp_st16(to + c, o);
              }
            }
          }
          const float neg = (m_ref == -INFINITY ? 0.f : -m_ref) + kSpUp<T>;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          auto weights = [&](const uint32_t(&x)[32], int c) {
            uint32_t w[32];  // 16 pairs of hi terms, 16 of lo terms
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float p0 = sp_exp2(fmaf(__uint_as_float(x[2 * i]), a.scale_log2, neg));
              const float p1 = sp_exp2(fmaf(__uint_as_float(x[2 * i + 1]), a.scale_log2, neg));
              sum[(2 * i) & 3] += p0;
              sum[(2 * i + 1) & 3] += p1;
              pack2_split<T>(p0, p1, w[i], w[16 + i]);
            }
            sp_st32(th + c, w);
          };
          weights(x0, 0);
          weights(x1, 32);
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          sp_wait_st();
        }
        tc_fence_before();
        if (!rehearsal) mbar_arrive(p_ready + 16 * stream + 8 * half);
      }
      if (!ok) break;
      if (!rehearsal) {
        kt += count;
        i0 += 2 * n;
        // the next piece's queries, while the last products run; its first ones
        // run beside the sums
        has_next = walk.next(s, after);
        early = has_next && !two && after.g.nq <= 128;
        if (early) {
          fetch(after, pieces + 1);
          lim = sees(after);
        }

        // the piece's sums (its products are done): [nq][D], and (maximum, sum)
        ok = __all_sync(0xffffffffu, sp_wait(o_done, (uint32_t)pieces & 1u));
        if (!ok) break;
        if (early) fetched();
      }
      tc_fence_after();
      const int64_t at = p.g.acc + ((int64_t)p.h * p.g.maxp + p.index) * nq + m;
      float *part = s.acc + at * kTaD;
      if (tid == 0 && mine && p.t0 + n == SpCost(nq).before(p.g.len))
        s.pieces[(int64_t)p.seg * a.hk + p.h] = p.index + 1;
      if (two) {
        // 32 columns of the warp's rows at a time pass through where the
        // queries were, so that a store writes 128 bytes of four rows (each
        // lane its own row: 8000 clocks for the sums of 256 rows)
        const uint32_t stage = s_q + warp * (32 * kSpStage);
        float *rows = part - (int64_t)lane * kTaD;
        const int left = nq - (m - lane);  // rows of this warp that there are
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t o[32];
          sp_ld32(to + c, o);
          sp_wait_ld(o);
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * kSpStage + i * 4),
                         "r"(o[i]), "r"(o[i + 1]), "r"(o[i + 2]), "r"(o[i + 3])
                         : "memory");
          __syncwarp();
#pragma unroll
          for (int r = lane >> 3; r < 32; r += 4) {
            float4 v;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(stage + r * kSpStage + (lane & 7) * 16)
                         : "memory");
            if (r < left) *reinterpret_cast<float4 *>(rows + (int64_t)r * kTaD + c + (lane & 7) * 4) = v;
          }
          __syncwarp();
        }
        if (mine) s.ml[at] = make_float2(l != l ? 0.f : m_ref - kSpUp<T>, l);  // (NaN is no empty sum)
        tc_fence_before();
        both();  // all of it is read before the next piece's queries
      } else {
        // both streams' sums of a row lie in the same lane: each stream joins
        // half of the columns (maxima and sums pass where the queries were)
        float2 *ml = reinterpret_cast<float2 *>(smem + (pieces & 1) * kSpTile);
        ml[stream * 128 + m128] = make_float2(m_ref, l);
        both();
        if (!ok) break;
        const float2 x0 = ml[m128], x1 = ml[128 + m128];
        const float M = fmaxf(x0.x, x1.x);
        const float f0 = M == -INFINITY ? 0.f : sp_exp2(x0.x - M);
        const float f1 = M == -INFINITY ? 0.f : sp_exp2(x1.x - M);
        const uint32_t t0 = tmem + lanes + 256 + stream * 64;
        if (works)
#pragma unroll 1
          for (int c = 0; c < 64; c += 32) {
            uint32_t o0[32], o1[32];
            sp_ld32(t0 + c, o0);
            sp_ld32(t0 + 128 + c, o1);
            sp_wait_ld(o0);
            sp_wait_ld(o1);
            if (mine)
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  y[e] = __uint_as_float(o0[i + e]) * f0;
                  if (n > 1) y[e] = fmaf(__uint_as_float(o1[i + e]), f1, y[e]);
                }
                sp_st_global8(part + stream * 64 + c + i, y);
              }
          }
        const float sum = x0.y * f0 + x1.y * f1;
        if (mine && stream == 0) s.ml[at] = make_float2(sum != sum ? 0.f : M - kSpUp<T>, sum);
        // all of it is read before the next piece's queries and products
        tc_fence_before();
        both();
      }
      if (rehearsal) {
        rehearsal = false;
        pdl_begin();
        walk.begin(s);
        if (!walk.next(s, p)) break;
        continue;
      }
      ++pieces;
      if (!has_next) break;
      p = after;
    }
    cp_async_wait<0>();
    if (!ok && lane == 0) stop();
  }
  tc_fence_before();
  __syncthreads();
  if (s_abort) {
    // A wait ran out: let the copies land and the products end before the
    // shared and tensor memory go.
    if (tid < kSpSlots && s_turns[tid] > 0)  // (the last load of each slot)
      mbar_wait(full + 8 * tid, (uint32_t)(s_turns[tid] - 1) & 1u);
    if (warp == 9 || warp == 11) {
      sp_commit(sp_elect(), drain);
      mbar_wait(drain, 1);
    }
    __syncthreads();
  }
  if (warp == 9)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ------------------------------------------------------------------ merge
constexpr int kMergeWarps = 4;

// A CTA a (row, query head), a lane four of its dims: warp w takes pieces w,
// w + 4, ... of the prefix and, behind them, of the row's own tokens, eight
// loads on their way, and the warps' sums are joined in order.  One warp a
// (row, head) instead (SPREAD false) when they alone fill the GPU (a call with
// 7680 of a few pieces each: 54 us against 67; 512 of 38 pieces: 50 against 46).
template <typename T, bool SPREAD>
__global__ void __launch_bounds__(kMergeWarps * 32) shared_prefix_merge_kernel(const SpArgs s) {
  __shared__ float4 s_acc[kMergeWarps][32];
  __shared__ float2 s_ml[kMergeWarps];
  pdl_begin();
  const TaArgs &a = s.a;
  constexpr int kStep = SPREAD ? kMergeWarps : 1;
  const int lane = threadIdx.x & 31, G = a.hq / a.hk;
  const int warp = SPREAD ? threadIdx.x >> 5 : 0;
  const int64_t rh = SPREAD ? blockIdx.x : (int64_t)blockIdx.x * kMergeWarps + (threadIdx.x >> 5);
  if (rh >= (int64_t)a.rows * a.hq) return;  // (whole warps, none of SPREAD's)
  const int row = (int)(rh / a.hq), head = (int)(rh - (int64_t)row * a.hq), h = head / G;
  const SpRow at = s.rows[row];
  const int m = (row - at.row0) * G + head % G;  // query row in the group
  // the two segments: pieces, first place, places between pieces
  int count[2] = {0, 0}, stride[2] = {0, 0};
  int64_t place[2] = {0, 0};
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int seg = part == 0 ? (at.pseg < 0 ? -1 : at.pseg + m / 256) : at.sseg;
    if (seg < 0) continue;
    const SpSeg &g = s.segs[seg];
    count[part] = min(s.pieces[(int64_t)seg * a.hk + h], g.maxp);  // (0 of 0 without tokens)
    stride[part] = g.nq;
    place[part] = g.acc + (int64_t)h * g.maxp * g.nq + (part == 0 ? m % 256 : at.srow * G + head % G);
  }
  const int all = count[0] + count[1];
  float M = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int base = warp; base < all; base += 8 * kStep) {
    float4 v[8];
    float2 x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = base + j * kStep;
      v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      x[j] = make_float2(-INFINITY, 0.f);
      if (i < all) {
        const bool own = i >= count[0];
        const int64_t src = (own ? place[1] : place[0]) +
                            (int64_t)(own ? i - count[0] : i) * (own ? stride[1] : stride[0]);
        x[j] = s.ml[src];
        v[j] = *reinterpret_cast<const float4 *>(s.acc + src * kTaD + 4 * lane);
      }
    }
    float now = M;
#pragma unroll
    for (int j = 0; j < 8; ++j) now = fmaxf(now, x[j].x);
    if (now == -INFINITY) continue;
    const float f = sp_exp2(M - now);
    M = now;
    sum *= f, acc.x *= f, acc.y *= f, acc.z *= f, acc.w *= f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (x[j].x == -INFINITY) continue;  // (nothing seen: its sums are nothing, too)
      const float w = sp_exp2(x[j].x - now);
      sum = fmaf(x[j].y, w, sum);
      acc.x = fmaf(v[j].x, w, acc.x);
      acc.y = fmaf(v[j].y, w, acc.y);
      acc.z = fmaf(v[j].z, w, acc.z);
      acc.w = fmaf(v[j].w, w, acc.w);
    }
  }
  float top = M;
  if (SPREAD) {
    s_acc[warp][lane] = acc;
    if (lane == 0) s_ml[warp] = make_float2(M, sum);
    __syncthreads();
    if (warp != 0) return;
    top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) top = fmaxf(top, s_ml[w].x);
    sum = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kMergeWarps; ++w) {
      if (s_ml[w].x == -INFINITY) continue;
      const float f = sp_exp2(s_ml[w].x - top);
      const float4 v = s_acc[w][lane];
      sum = fmaf(s_ml[w].y, f, sum);
      acc.x = fmaf(v.x, f, acc.x);
      acc.y = fmaf(v.y, f, acc.y);
      acc.z = fmaf(v.z, f, acc.z);
      acc.w = fmaf(v.w, f, acc.w);
    }
  }
  // nothing seen: zeros and -inf (a sum that is NaN says so)
  const bool none = top == -INFINITY;
  const float inv = none ? 0.f : 1.f / sum;
  uint2 out;
  out.x = pack2<T>(acc.x * inv, acc.y * inv);
  out.y = pack2<T>(acc.z * inv, acc.w * inv);
  T *dst = static_cast<T *>(a.out) + rh * kTaD + 4 * lane;
  if (reinterpret_cast<uintptr_t>(dst) % 8 == 0) {
    *reinterpret_cast<uint2 *>(dst) = out;
  } else {  // rows that begin off an 8-byte boundary (a view of a wider buffer)
    const T *y = reinterpret_cast<const T *>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = y[i];
  }
  if (lane == 0) a.lse[rh] = none ? -INFINITY : (top + log2f(sum)) * kTaLn2;
}

// ------------------------------------------------------------------- host
// The paged cache as (64 dims, 8 tokens, 2 halves, rows of 8 tokens, heads);
// a box holds `box` tokens of one head.
bool sp_encode_map(CUtensorMap *map, const void *base, int64_t token_rows, int heads, int dtype,
                   int box) {
  auto fn = tensor_map_encoder();
  if (fn == nullptr) return false;
  const cuuint64_t token = (cuuint64_t)heads * kTaD * 2;
  cuuint64_t dims[5] = {64, 8, 2, (cuuint64_t)token_rows / 8, (cuuint64_t)heads};
  cuuint64_t strides[4] = {token, 128, 8 * token, kTaD * 2};
  cuuint32_t boxes[5] = {64, 8, 2, (cuuint32_t)box / 8, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(map, dtype == DSB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
            5, const_cast<void *>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct SpPlan {
  int box;             // 0: pages that no TMA box fits (every row for itself)
  int64_t splits;      // of a row, without boxes
  // scratch, in floats (every part a multiple of 16 bytes)
  int64_t begin, segs, rows, gseg, pieces, acc, ml, total;
};

SpPlan plan_for(int rows, int hq, int hk, int groups, int bs, int max_prefix, int max_suffix) {
  SpPlan p{};
  // The tiles are copied in boxes of whole 8-row swizzle atoms inside a page;
  // pages that are no multiple of 8 tokens take a pass of every row by
  // itself (one row of 40960 tokens by itself costs what all rows do here).
  p.box = kSpTok;
  while (p.box >= 8 && bs % p.box) p.box /= 2;
  if (p.box < 8) {
    p.box = 0;
    // splits that give the GPU four CTAs an SM, of 64 to 1024 tokens
    const int64_t most = (int64_t)max_prefix + max_suffix;
    const int64_t ctas = std::max<int64_t>(1, 4LL * sm_count() / ((int64_t)rows * hk));
    p.splits = std::max<int64_t>(std::min<int64_t>(ctas, (most + 63) / 64), (most + 1023) / 1024);
    p.splits = std::max<int64_t>(p.splits, 1);
    p.total = (int64_t)rows * hq * p.splits * (kTaD + 2);
    return p;
  }
  const int64_t g = hq / hk, ctas = sm_count();
  const int64_t segs = ((int64_t)rows * g + 255) / 256 + groups + rows;
  // pieces x query rows: each (row, head) is in two segments, each of which
  // has places for three pieces more than its share of the CTAs
  const int64_t sums = 6 * (int64_t)rows * hq + 257 * ctas;
  auto round = [](int64_t n) { return (n + 7) / 8 * 8; };
  p.begin = 0;
  p.segs = ctas * 4;
  p.rows = p.segs + segs * 16;
  p.gseg = p.rows + (int64_t)rows * 4;
  p.pieces = round(p.gseg + groups);
  p.ml = round(p.pieces + segs * hk);
  p.acc = round(p.ml + 2 * sums);
  p.total = p.acc + sums * kTaD;
  return p;
}

template <typename T> int run_typed(SpArgs &s, const SpPlan &p, float *scratch, int dtype, cudaStream_t st) {
  TaArgs &a = s.a;
  const int64_t rh = (int64_t)a.rows * a.hq;
  if (p.box == 0) {
    a.splits = (int)p.splits;
    a.part = scratch;
    a.page_tiles = 0;
    auto kern = paged_decode_split_kernel<T, 16, true>;
    constexpr size_t smem = TaSmem<16>::kBytes;
    if (int e = ensure_smem((const void *)kern, smem); e != DSB_OK) return e;
    launch_kernel(kern, dim3(a.hk, a.splits, a.rows), dim3(kTaWarps * 32), smem, st, a);
    if (int e = check_launch("paged_decode_split_kernel")) return e;
    launch_kernel(paged_decode_merge_kernel<T, true>, dim3((unsigned)rh), dim3(kTaD), 0, st, a);
    return check_launch("paged_decode_merge_kernel");
  }
  s.box = p.box;
  s.ctas = sm_count();
  s.begin = reinterpret_cast<SpBegin *>(scratch + p.begin);
  s.segs = reinterpret_cast<SpSeg *>(scratch + p.segs);
  s.rows = reinterpret_cast<SpRow *>(scratch + p.rows);
  s.gseg = reinterpret_cast<int32_t *>(scratch + p.gseg);
  s.pieces = reinterpret_cast<int32_t *>(scratch + p.pieces);
  s.ml = reinterpret_cast<float2 *>(scratch + p.ml);
  s.acc = scratch + p.acc;
  auto kern = shared_prefix_kernel<T>;
  if (int e = ensure_smem((const void *)kern, kSpSmem); e != DSB_OK) return e;
  CUtensorMap tk, tv;
  if (!sp_encode_map(&tk, a.k, s.token_rows, a.hk, dtype, p.box) ||
      !sp_encode_map(&tv, a.v, s.token_rows, a.hk, dtype, p.box))
    return fail(DSB_ERR_CUDA, "tensor map of the paged cache");
  launch_kernel(shared_prefix_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, s);
  if (int e = check_launch("shared_prefix_plan_kernel")) return e;
  launch_kernel(kern, dim3(s.ctas), dim3(kSpThreads), kSpSmem, st, tk, tv, s);
  if (int e = check_launch("shared_prefix_kernel")) return e;
  if (rh < 8L * s.ctas)
    launch_kernel(shared_prefix_merge_kernel<T, true>, dim3((unsigned)rh), dim3(kMergeWarps * 32), 0,
                  st, s);
  else
    launch_kernel(shared_prefix_merge_kernel<T, false>,
                  dim3((unsigned)((rh + kMergeWarps - 1) / kMergeWarps)), dim3(kMergeWarps * 32), 0,
                  st, s);
  return check_launch("shared_prefix_merge_kernel");
}

}  // namespace
}  // namespace dsb

using namespace dsb;

extern "C" int64_t dsb_shared_prefix_scratch_floats(int32_t query_rows, int32_t num_query_heads,
                                                    int32_t num_kv_heads, int32_t num_groups,
                                                    int32_t block_size, int32_t max_prefix_len,
                                                    int32_t max_suffix_len) {
  if (query_rows <= 0 || num_query_heads <= 0 || num_kv_heads <= 0 || num_groups <= 0 ||
      block_size <= 0 || max_prefix_len < 0 || max_suffix_len < 0)
    return 0;
  const SpPlan p = plan_for(query_rows, num_query_heads, num_kv_heads, num_groups, block_size,
                            max_prefix_len, max_suffix_len);
  return p.total;
}

extern "C" int dsb_shared_prefix_attention_lse(
    const void *query, int32_t query_rows, int32_t num_query_heads, int32_t num_kv_heads,
    int32_t head_dim, const void *key_cache, const void *value_cache, int64_t num_blocks,
    int32_t block_size, const int32_t *block_table, int64_t block_table_stride,
    int64_t block_table_rows, int64_t block_table_cols, const int32_t *seq_lens,
    const int32_t *table_rows, const int32_t *prefix_lens, const int32_t *group_starts,
    int32_t num_groups, int32_t max_prefix_len, int32_t max_suffix_len, float scale,
    int32_t dtype, void *out, float *lse, float *scratch, int64_t scratch_floats,
    int32_t *error_flag, void *stream) {
  if (query_rows < 0) return fail(DSB_ERR_INVALID, "negative query_rows");
  if (query_rows == 0) return DSB_OK;
  if (dtype != DSB_BF16 && dtype != DSB_F16)
    return fail(DSB_ERR_INVALID, "query and caches must be BF16 or FP16");
  if (num_query_heads <= 0 || num_kv_heads <= 0 || num_query_heads % num_kv_heads)
    return fail(DSB_ERR_INVALID, "query heads must be a positive multiple of kv heads");
  if (head_dim != kTaD) return fail(DSB_ERR_UNSUPPORTED, "head_dim must be 128");
  if (num_query_heads / num_kv_heads > 16)
    return fail(DSB_ERR_UNSUPPORTED, "at most 16 query heads per kv head");
  if (num_blocks <= 0 || block_size <= 0 || block_table_rows <= 0 || block_table_cols <= 0 ||
      block_table_stride < block_table_cols || max_prefix_len < 0 || max_suffix_len < 0)
    return fail(DSB_ERR_INVALID, "bad cache or block-table geometry");
  if (num_groups <= 0 || num_groups > query_rows || (!group_starts && num_groups != 1))
    return fail(DSB_ERR_INVALID,
                "num_groups must be in [1, query_rows]; one group when group_starts is null");
  if (!(scale > 0.f)) return fail(DSB_ERR_INVALID, "scale must be positive");
  if (!query || !key_cache || !value_cache || !block_table || !seq_lens || !prefix_lens || !out ||
      !lse || !scratch)
    return fail(DSB_ERR_INVALID, "null pointer argument");
  const SpPlan p = plan_for(query_rows, num_query_heads, num_kv_heads, num_groups, block_size,
                            max_prefix_len, max_suffix_len);
  if (p.splits > 65535 || num_kv_heads > 65535 || query_rows > 65535 ||
      (int64_t)query_rows * num_query_heads > INT32_MAX)
    return fail(DSB_ERR_UNSUPPORTED, "grid too large");
  if (num_blocks * block_size >= INT32_MAX)
    return fail(DSB_ERR_UNSUPPORTED, "the cache must hold fewer than 2^31 - 1 tokens");
  if (scratch_floats < p.total)
    return fail(DSB_ERR_INVALID, "scratch smaller than dsb_shared_prefix_scratch_floats");
  if (reinterpret_cast<uintptr_t>(query) % 16 || reinterpret_cast<uintptr_t>(key_cache) % 16 ||
      reinterpret_cast<uintptr_t>(value_cache) % 16 || reinterpret_cast<uintptr_t>(scratch) % 32)
    return fail(DSB_ERR_UNSUPPORTED,
                "query and caches must be 16-byte aligned, scratch 32-byte");
  SpArgs s{};
  TaArgs &a = s.a;
  a.q = query;
  a.k = key_cache;
  a.v = value_cache;
  a.bt = block_table;
  a.seq = seq_lens;
  a.trows = table_rows;
  a.bt_stride = block_table_stride;
  a.bt_cols = block_table_cols;
  a.bt_rows = block_table_rows;
  a.nblocks = num_blocks;
  a.bs = block_size;
  a.hq = num_query_heads;
  a.hk = num_kv_heads;
  a.rows = query_rows;
  a.scale_log2 = scale * kTaLog2e;
  a.out = out;
  a.lse = lse;
  a.err = error_flag;
  s.prefix_lens = prefix_lens;
  s.group_starts = group_starts;
  s.groups = num_groups;
  s.token_rows = num_blocks * block_size;
  cudaStream_t st = as_stream(stream);
  return dtype == DSB_BF16 ? run_typed<__nv_bfloat16>(s, p, scratch, dtype, st)
                           : run_typed<__half>(s, p, scratch, dtype, st);
}
