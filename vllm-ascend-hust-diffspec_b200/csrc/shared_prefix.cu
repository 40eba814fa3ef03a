// Target paged decode attention, with the softmax LSE, for requests that
// share a prefix of their tokens (forked from one prompt, or on one system
// prompt): rows [group_starts[i], group_starts[i + 1]) hold the same tokens
// at positions [0, prefix_lens[i]).
//   out[r, h] = sum_t softmax_t(scale * q[r, h] . k_t) v_t,  t < seq_lens[r]
//   lse[r, h] = log sum_t exp(scale * q[r, h] . k_t)          (natural log)
//
// Two partial passes and a merge, all on the framework's split-KV pattern:
//  * the prefix, once for the group: the queries of all its rows that read
//    one kv head (rows x G of them) are the M = 128 rows of tensor-core
//    tiles, so a K/V tile read from HBM serves all of them.  Bound by that
//    stream up to ~200 query rows (K + V of 128 tokens are 64 KB, ~2800 SM
//    clocks of the measured copy bandwidth, against ~1540 of products), by
//    the products beyond;
//  * each row's own tokens behind it: the split kernel of the plain decode
//    attention (paged_split.cuh);
//  * the merge of both, in a fixed order.
#include "paged_split.cuh"
#include "tma_umma.cuh"

namespace dsb {
namespace {

// ------------------------------------------------------------ prefix pass
// CTA (kv head, split, tile of query rows): warps 0-3 and 4-7 are two softmax
// streams, warp 8 loads, warp 9 issues the products.  Per 128-token tile of
// a stream:
//   S[128 x 128] = Q . K^T                (tensor memory, fp32)
//   P = exp2(scale S - m), m the row's running maximum; a thread has a row
//   O[128 x 128] += P . V                 (A = P from tensor memory)
// P overwrites S as two 16-bit terms, hi + lo (the weights keep ~16 bits; one
// term alone costs half an output step more), so P . V is two products.  O
// is rescaled only when a row's maximum has grown by more than 2^8 since the
// last time: until then P stays below 2^8 and sums in fp32 as well.
//   one query tile a CTA (up to 128 query rows in a group): the streams take
//   the split's even and odd token tiles and are merged at its end;
//   two (more rows): each stream has 128 query rows of its own, and a K/V
//   tile serves 256.
// K and V tiles pass through one ring of 32 KB slots in the order of use.
constexpr int kSpTile = 32768;      // 128 tokens x 128 dims, 16-bit: two 64-dim halves
constexpr int kSpHalf = 16384;
constexpr int kSpTok = 128;
constexpr int kSpThreads = 320;
constexpr int kSpSmem = 1024 + 7 * kSpTile + 256;  // query tiles + ring, barriers
constexpr float kSpGrow = 8.f;      // log2 of the growth that rescales O

struct SpArgs {
  TaArgs a;
  int psplits;
  float *acc;    // [rows * hq, psplits, D]: sums of the prefix's splits
  float2 *ml;    // [rows * hq, psplits]: (maximum, sum)
  int64_t token_rows;  // num_blocks * block_size
  int box;       // tokens of a TMA box: 8 .. 128, dividing the page
};

// One try first: most waits are over when they begin, and the bounded wait
// reads the timer.
__device__ __forceinline__ bool sp_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done || mbar_wait(bar, parity);
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
__device__ __forceinline__ void sp_st16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15};" ::SP_U8(r, 0),
      SP_U8(r, 8), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void sp_st32(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::SP_U8(r, 0),
      SP_U8(r, 8), SP_U8(r, 16), SP_U8(r, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void sp_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void sp_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// D[tmem] (+)= A[tmem] . B[smem]
__device__ __forceinline__ void sp_umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                           bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}

// What a CTA works on.
struct SpTask {
  int row0, nrows;   // the group's rows
  int tile;          // query tile of the group
  int prefix;        // its tokens
  int64_t trow;      // the table row that they are read through
};

// The CTA's (group, query tile) from blockIdx.z, by one warp; false: none.
__device__ bool sp_find(const SpArgs &s, int per_tile, int heads, SpTask &task) {
  const TaArgs &a = s.a;
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < a.groups; base += 32) {
    const int i = base + lane;
    int lo = 0, hi = 0;
    if (i < a.groups) {
      lo = a.group_starts != nullptr ? a.group_starts[i] : 0;
      hi = a.group_starts != nullptr ? a.group_starts[i + 1] : a.rows;
      if ((hi < lo || lo < 0 || hi > a.rows) && blockIdx.x + blockIdx.y + blockIdx.z == 0)
        flag_error(a.err, DSB_FLAG_SLOT);
      lo = min(max(lo, 0), a.rows);
      hi = min(max(hi, lo), a.rows);
    }
    const int tiles = (int)(((int64_t)(hi - lo) * heads + per_tile - 1) / per_tile);
    int cum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, cum, o);
      if (lane >= o) cum += x;
    }
    const int z = (int)blockIdx.z - before;
    const unsigned hit = __ballot_sync(0xffffffffu, cum > z);
    if (hit) {
      const int src = __ffs(hit) - 1;
      task.row0 = __shfl_sync(0xffffffffu, lo, src);
      task.nrows = __shfl_sync(0xffffffffu, hi - lo, src);
      task.tile = z - __shfl_sync(0xffffffffu, cum - tiles, src);
      task.prefix = 0;
      task.trow = 0;
      // the first row of the group that sees anything
      for (int r0 = 0; r0 < task.nrows; r0 += 32) {
        const int r = task.row0 + r0 + lane;
        int64_t trow = -1;
        if (r0 + lane < task.nrows && a.seq[r] > 0) trow = a.trows != nullptr ? a.trows[r] : r;
        const unsigned ok = __ballot_sync(0xffffffffu, trow >= 0 && trow < a.bt_rows);
        if (ok) {
          task.trow = __shfl_sync(0xffffffffu, trow, __ffs(ok) - 1);
          const int p = a.prefix_lens[base + src];
          task.prefix = (int)min((int64_t)max(p, 0), a.bt_cols * a.bs);
          break;
        }
      }
      return true;
    }
    before += __shfl_sync(0xffffffffu, cum, 31);
  }
  return false;
}

template <typename T, int MT>  // MT query tiles a CTA
__global__ void __launch_bounds__(kSpThreads, 1)
    shared_prefix_kernel(const __grid_constant__ CUtensorMap tk,
                         const __grid_constant__ CUtensorMap tv, const SpArgs s) {
  constexpr int kSlots = MT == 1 ? 6 : 5;
  const TaArgs &a = s.a;
  extern __shared__ uint8_t sp_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(sp_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t s_q = smem_u32(smem), s_kv = s_q + MT * kSpTile;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + 7 * kSpTile);
  const uint32_t full = smem_u32(bars), empty = full + 8 * kSlots, s_full = empty + 8 * kSlots,
                 p_ready = s_full + 16, done = p_ready + 16, tail = done + 8;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_found, s_issued, s_seen;
  __shared__ SpTask s_task;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.hq / a.hk, h = blockIdx.x, split = blockIdx.y;

  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tk)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tv)) : "memory");
    for (int i = 0; i < 2 * kSlots; ++i) mbar_init(full + 8 * i);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i);
      mbar_init_count(p_ready + 8 * i, 128);
    }
    mbar_init(done);
    mbar_init(tail);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_abort = 0;
    s_issued = 0;
    s_seen = 0;
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_u32(&s_tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_begin();
  if (warp == 8) {
    SpTask t{0, 0, 0, 0, 0};  // (no task: no rows)
    const bool found = sp_find(s, 128 * MT, G, t);
    if (lane == 0) {
      s_task = t;
      s_found = found;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const SpTask task = s_task;
  const int heads = s_found ? task.nrows * G : 0;  // query rows of the group for this kv head

  // this thread's query row: (row, query head), or none
  const int stream = warp >> 2;
  const int m = task.tile * 128 * MT + (MT == 2 ? stream * 128 : 0) + (tid & 127);
  const bool mine = warp < 8 && m < heads;
  const int row = mine ? task.row0 + m / G : 0;
  const int64_t rh = (int64_t)row * a.hq + h * G + (mine ? m % G : 0);
  int lim = 0;  // the prefix tokens that it sees
  if (mine) {
    const int64_t trow = a.trows != nullptr ? a.trows[row] : row;
    lim = trow >= 0 && trow < a.bt_rows ? min(max(a.seq[row], 0), task.prefix) : 0;
  }
  if (warp < 8) {
    const int most = __reduce_max_sync(0xffffffffu, lim);
    if (lane == 0) atomicMax(&s_seen, most);
    // query tiles, swizzled as the operand wants them; rows past the group are zero
    for (int i = tid; i < MT * 128 * 16; i += 256) {
      const int q = i >> 4, c = i & 15;  // query row of the CTA, 16-byte piece of its 256 bytes
      const int mm = task.tile * 128 * MT + q;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (mm < heads)
        v = *reinterpret_cast<const uint4 *>(
            static_cast<const T *>(a.q) +
            ((int64_t)(task.row0 + mm / G) * a.hq + h * G + mm % G) * kTaD + c * 8);
      const int r = q & 127;
      *reinterpret_cast<uint4 *>(smem + (q >> 7) * kSpTile + (c >> 3) * kSpHalf + r * 128 +
                                 (((c & 7) ^ (r & 7)) * 16)) = v;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  const int seen = s_seen;  // prefix tokens that any of these query rows sees
  const int ntok = (seen + kSpTok - 1) / kSpTok;
  const int t0 = (int)((int64_t)split * ntok / s.psplits);
  const int n = (int)((int64_t)(split + 1) * ntok / s.psplits) - t0;  // token tiles of this CTA

  if (n > 0) {
    // index of a tile's load in the order of use
    auto k_index = [&](int j) { return MT == 2 ? 2 * j : (j < 2 ? j : 2 * j - 1); };
    auto v_index = [&](int j) { return MT == 2 ? 2 * j + 1 : min(2 * j + 2, 2 * n - 1); };

    if (warp == 8) {
      const int32_t *bt = a.bt + task.trow * a.bt_stride;
      int i = 0;
      bool bad = false, ok = true;
      auto load = [&](int j, bool is_v) {
        if (!ok) return;
        const int slot = i % kSlots;
        if (i >= kSlots) ok = sp_wait(empty + 8 * slot, (uint32_t)(i / kSlots - 1) & 1u);
        ok = __all_sync(0xffffffffu, ok && !*reinterpret_cast<volatile int *>(&s_abort));
        if (!ok) return;
        const int T0 = (t0 + j) * kSpTok;
        const uint32_t dst = s_kv + slot * kSpTile;
        // the values behind the last token seen are zeroed once they are here
        // (their weights are zero, but zero times what lies there may not be)
        const bool cut = is_v && T0 + kSpTok > seen;
        const uint32_t bar = cut ? tail : full + 8 * slot;
        if (lane == 0) mbar_expect_tx(bar, kSpTile);
        __syncwarp();
        const int boxes = kSpTok / s.box;
        for (int b = lane; b < 2 * boxes; b += 32) {
          const int half = b / boxes, first = (b % boxes) * s.box, tok = T0 + first;
          int y = (int)s.token_rows;  // out of range: zeros
          if (tok < seen) {
            const int64_t page = bt[tok / a.bs];
            if (page >= 0 && page < a.nblocks)
              y = (int)(page * a.bs + tok % a.bs);
            else
              bad = true;
          }
          tma_load_3d(dst + half * kSpHalf + first * 128, is_v ? &tv : &tk, half * 64, h, y, bar);
        }
        __syncwarp();
        if (lane == 0) s_issued = i + 1;
        if (cut) {
          ok = __all_sync(0xffffffffu, sp_wait(tail, 0));
          if (ok) {
            const int keep = seen - T0;
            for (int z = keep * 8 + lane; z < kSpTok * 8; z += 32) {
              const uint32_t p = dst + (z >> 3) * 128 + (z & 7) * 16;
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(p), "r"(0u) : "memory");
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(p + kSpHalf), "r"(0u)
                           : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * slot);
          }
        }
        ++i;
      };
      load(0, false);
      if (MT == 1 && n > 1) load(1, false);
      for (int j = 0; j < n; ++j) {
        load(j, true);
        if (j + MT % 2 + 1 < n) load(j + MT % 2 + 1, false);
      }
      if (bad) flag_error(a.err, DSB_FLAG_BLOCK);
      if (!ok && lane == 0) {
        atomicExch(&s_abort, 1);
        flag_error(a.err, DSB_FLAG_TIMEOUT);
      }
    } else if (tid == 9 * 32) {
      const uint32_t qk = umma_idesc<T, 128>(false), pv = qk | (1u << 16);  // V is dim-contiguous
      auto slot_of = [&](int i) { return s_kv + (i % kSlots) * kSpTile; };
      auto filled = [&](int i) {
        const bool got = sp_wait(full + 8 * (i % kSlots), (uint32_t)(i / kSlots) & 1u);
        tc_fence_after();
        return got;
      };
      auto product_s = [&](int st, int j) {  // S of stream st
        const uint32_t q = s_q + (MT == 2 ? st * kSpTile : 0), k = slot_of(k_index(j));
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const uint32_t off = (x >> 2) * kSpHalf + (x & 3) * 32;
          umma(tmem + st * 128, umma_desc(q + off, 16, 1024), umma_desc(k + off, 16, 1024), qk, x > 0);
        }
        umma_commit(s_full + 8 * st);
      };
      auto product_o = [&](int st, int j, bool first) {  // O of stream st
        const uint32_t v = slot_of(v_index(j)), p = tmem + st * 128, o = tmem + 256 + st * 128;
#pragma unroll
        for (int x = 0; x < 16; ++x)  // the hi terms, then the lo ones
          sp_umma_ts(o, p + x * 8, umma_desc(v + (x & 7) * 2048, kSpHalf, 1024), pv, !(first && x == 0));
      };
      auto freed = [&](int i) { umma_commit(empty + 8 * (i % kSlots)); };
      bool ok = filled(k_index(0));
      if (ok) {
        product_s(0, 0);
        if (MT == 2) product_s(1, 0);
        freed(k_index(0));
      }
      if (MT == 1 && n > 1 && ok) {
        ok = filled(k_index(1));
        if (ok) {
          product_s(1, 1);
          freed(k_index(1));
        }
      }
      for (int j = 0; j < n && ok; ++j) {
        ok = filled(v_index(j));
        if (MT == 2) {
          for (int st = 0; st < 2 && ok; ++st) {
            ok = sp_wait(p_ready + 8 * st, (uint32_t)j & 1u);
            if (!ok) break;
            tc_fence_after();
            product_o(st, j, j == 0);
            if (st == 1) freed(v_index(j));
            if (j + 1 < n) {
              if (st == 0) ok = filled(k_index(j + 1));
              if (!ok) break;
              product_s(st, j + 1);
              if (st == 1) freed(k_index(j + 1));
            }
          }
        } else if (ok) {
          const int st = j & 1;
          ok = sp_wait(p_ready + 8 * st, (uint32_t)(j >> 1) & 1u);
          if (!ok) break;
          tc_fence_after();
          product_o(st, j, j < 2);
          freed(v_index(j));
          if (j + 2 < n) {
            ok = filled(k_index(j + 2));
            if (!ok) break;
            product_s(st, j + 2);
            freed(k_index(j + 2));
          }
        }
      }
      if (!ok) {
        atomicExch(&s_abort, 1);
        flag_error(a.err, DSB_FLAG_TIMEOUT);
      }
      umma_commit(done);  // arrives once every issued product is done
    }

    float m_ref = -INFINITY, l = 0.f;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = tmem + lanes + stream * 128, to = ts + 256;
    const int count = warp >= 8 ? 0 : (MT == 2 ? n : (n - stream + 1) / 2);
    for (int k = 0; k < count; ++k) {
      const int T0 = (t0 + (MT == 2 ? k : 2 * k + stream)) * kSpTok;
      if (!__all_sync(0xffffffffu, sp_wait(s_full + 8 * stream, (uint32_t)k & 1u))) {
        if (lane == 0) {
          atomicExch(&s_abort, 1);
          flag_error(a.err, DSB_FLAG_TIMEOUT);
        }
        break;
      }
      tc_fence_after();
      uint32_t x[128];
      sp_ld32(ts, x);
      sp_ld32(ts + 32, x + 32);
      sp_ld32(ts + 64, x + 64);
      sp_ld32(ts + 96, x + 96);
      sp_wait_ld();
      const int vis = lim - T0;
      if (vis < kSpTok) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= vis) x[i] = __float_as_uint(-INFINITY);
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(x[i]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
      if (__any_sync(0xffffffffu, top > m_ref + kSpGrow)) {
        const float now = fmaxf(m_ref, top);
        const float f = now == -INFINITY ? 1.f : sp_exp2(m_ref - now);
        m_ref = now;
        l *= f;
        if (k > 0) {
#pragma unroll
          for (int c = 0; c < 128; c += 32) {
            uint32_t o[32];
            sp_ld32(to + c, o);
            sp_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            sp_st32(to + c, o);
          }
        }
      }
      const float base = m_ref == -INFINITY ? 0.f : m_ref;
      float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p0 = sp_exp2(fmaf(__uint_as_float(x[c + 2 * i]), a.scale_log2, -base));
          const float p1 = sp_exp2(fmaf(__uint_as_float(x[c + 2 * i + 1]), a.scale_log2, -base));
          ls[(2 * i) & 3] += p0;
          ls[(2 * i + 1) & 3] += p1;
          pack2_split<T>(p0, p1, hi[i], lo[i]);
        }
        sp_st16(ts + c / 2, hi);
        sp_st16(ts + 64 + c / 2, lo);
      }
      l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
      sp_wait_st();
      tc_fence_before();
      mbar_arrive(p_ready + 8 * stream);
    }

    // every product done, every load landed: the partial sums
    bool good = true;
    if (warp < 8 || tid == 9 * 32) good = sp_wait(done, 0);
    good = __syncthreads_and(good) && !s_abort;
    if (!good) {
      if (tid == 0) flag_error(a.err, DSB_FLAG_TIMEOUT);
      if (tid == 8 * 32)  // (the copies in flight land, or their waits run out)
        for (int i = max(0, s_issued - kSlots); i < s_issued; ++i)
          mbar_wait(full + 8 * (i % kSlots), (uint32_t)(i / kSlots) & 1u);
      if (tid == 0) mbar_wait(done, 0);
      __syncthreads();
      m_ref = -INFINITY;
      l = 0.f;
    }
    tc_fence_after();
    float *stage = reinterpret_cast<float *>(smem + MT * kSpTile);  // [128][132], the ring's place
    float *part = s.acc + (rh * s.psplits + split) * kTaD;
    if (MT == 2) {
      if (warp < 8) {
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t o[32];
          sp_ld32(to + c, o);
          sp_wait_ld();
          if (mine)
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4 *>(part + c + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
        if (mine) s.ml[rh * s.psplits + split] = make_float2(m_ref, l);
      }
    } else {
      __shared__ float2 s_ml[128];
      if (stream == 1 && warp < 8) {
        s_ml[tid & 127] = make_float2(m_ref, l);
        if (n > 1) {
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            uint32_t o[32];
            sp_ld32(to + c, o);
            sp_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<uint4 *>(stage + (tid & 127) * 132 + c + i) =
                  make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      __syncthreads();
      if (stream == 0) {
        const float2 other = s_ml[tid];
        const float M = fmaxf(m_ref, other.x);
        const float f0 = M == -INFINITY ? 0.f : sp_exp2(m_ref - M);
        const float f1 = M == -INFINITY ? 0.f : sp_exp2(other.x - M);
#pragma unroll 1
        for (int c = 0; c < 128; c += 32) {
          uint32_t o[32];
          sp_ld32(to + c, o);
          sp_wait_ld();
          if (mine)
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
              if (n > 1) w = *reinterpret_cast<const float4 *>(stage + tid * 132 + c + i);
              float4 y;
              y.x = __uint_as_float(o[i]) * f0 + w.x * f1;
              y.y = __uint_as_float(o[i + 1]) * f0 + w.y * f1;
              y.z = __uint_as_float(o[i + 2]) * f0 + w.z * f1;
              y.w = __uint_as_float(o[i + 3]) * f0 + w.w * f1;
              *reinterpret_cast<float4 *>(part + c + i) = y;
            }
        }
        if (mine) s.ml[rh * s.psplits + split] = make_float2(M, l * f0 + other.y * f1);
      }
    }
  } else if (mine && (MT == 2 || stream == 0)) {
    s.ml[rh * s.psplits + split] = make_float2(-INFINITY, 0.f);  // no tokens for this split
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// One CTA per (row, query head), thread = output element: the prefix's
// splits, then the row's own, in order.
template <typename T>
__global__ void __launch_bounds__(kTaD) shared_prefix_merge_kernel(const SpArgs s) {
  pdl_begin();
  const TaArgs &a = s.a;
  const int64_t rh = blockIdx.x;
  const int row = (int)(rh / a.hq), d = threadIdx.x;
  const int np = ta_group_of(row, a.group_starts, a.groups) >= 0 ? s.psplits : 0;
  const float2 *ml = s.ml + rh * s.psplits;
  const float *own = a.part + rh * a.splits * (kTaD + 2);
  float M = -INFINITY;
  for (int i = 0; i < np; ++i) M = fmaxf(M, ml[i].x);
  for (int i = 0; i < a.splits; ++i) M = fmaxf(M, own[i * (kTaD + 2) + kTaD]);
  float sum = 0.f, ac = 0.f;
  if (M != -INFINITY) {
    for (int i = 0; i < np; ++i) {
      const float2 x = ml[i];
      if (x.x == -INFINITY) continue;  // (its sums were not written)
      const float f = exp2f(x.x - M);
      sum = fmaf(x.y, f, sum);
      ac = fmaf(s.acc[(rh * s.psplits + i) * kTaD + d], f, ac);
    }
    for (int i = 0; i < a.splits; ++i) {
      const float *q = own + i * (kTaD + 2);
      const float f = exp2f(q[kTaD] - M);
      sum = fmaf(q[kTaD + 1], f, sum);
      ac = fmaf(q[d], f, ac);
    }
  }
  const float y = sum > 0.f ? ac / sum : 0.f;
  static_cast<T *>(a.out)[rh * kTaD + d] = Elem<T>::from_f(y);
  if (d == 0) a.lse[rh] = sum > 0.f ? (M + log2f(sum)) * kTaLn2 : -INFINITY;
}

// ------------------------------------------------------------------- host
// Tokens of a split of the rows' own range: long ones when the rows alone
// fill the GPU, else shorter ones for more CTAs (a multiple of the tile).
int own_tokens_per_split(int64_t own, int rows, int hk) {
  const int64_t ctas = 4LL * 148 / std::max<int64_t>(1, (int64_t)rows * hk);  // splits wanted
  const int64_t tps = (own + std::max<int64_t>(ctas, 1) - 1) / std::max<int64_t>(ctas, 1);
  return (int)std::min<int64_t>(1024, std::max<int64_t>(64, (tps + 15) / 16 * 16));
}

struct SpPlan {
  bool shared;         // the prefix pass runs (else every row reads its whole sequence)
  int box, query_tiles, psplits, ztiles;
  int64_t own, splits; // tokens and splits of the rows' own range
  int tps;
  int64_t acc_floats, ml_floats, own_floats;
};

SpPlan plan_for(int rows, int hq, int hk, int groups, int bs, int max_prefix, int max_suffix) {
  SpPlan p{};
  // The prefix is copied in boxes of whole 8-row swizzle atoms inside a page;
  // pages that are no multiple of 8 tokens take the rows' own pass alone.
  p.box = kSpTok;
  while (p.box >= 8 && bs % p.box) p.box /= 2;
  p.shared = p.box >= 8 && max_prefix > 0;
  if (p.shared) {
    const int g = hq / hk;
    const int64_t each = ((int64_t)rows + groups - 1) / groups * g;  // query rows of a group
    p.query_tiles = each > 128 ? 2 : 1;
    const int per = 128 * p.query_tiles;
    p.ztiles = (int)((int64_t)rows * g / per) + groups;
    // splits of the prefix: the fewest rounds of 148 CTAs, each with ~3 tiles'
    // worth of start and end
    const int64_t columns = hk * groups * ((each + per - 1) / per);
    const int64_t tiles = ((int64_t)max_prefix + kSpTok - 1) / kSpTok;
    int64_t best = -1;
    for (int64_t k = 1; k <= std::min<int64_t>(tiles, 148); ++k) {
      const int64_t rounds = (columns * k + 147) / 148, cost = rounds * ((tiles + k - 1) / k + 3);
      if (best < 0 || cost < best) {
        best = cost;
        p.psplits = (int)k;
      }
    }
    p.acc_floats = (int64_t)rows * hq * p.psplits * kTaD;
    p.ml_floats = (int64_t)rows * hq * p.psplits * 2;
  }
  // the rows' own range starts on a tile of 16 tokens at or before its first
  p.own = p.shared ? (int64_t)max_suffix + kTaTile - 1 : (int64_t)max_prefix + max_suffix;
  p.tps = own_tokens_per_split(p.own, rows, hk);
  p.splits = std::max<int64_t>(1, (p.own + p.tps - 1) / p.tps);
  p.own_floats = (int64_t)rows * hq * p.splits * (kTaD + 2);
  return p;
}

template <typename T, int MT> int run_prefix(const SpArgs &s, const SpPlan &p, int dtype, cudaStream_t st) {
  auto kern = shared_prefix_kernel<T, MT>;
  if (int e = ensure_smem((const void *)kern, kSpSmem); e != DSB_OK) return e;
  CUtensorMap tk, tv;
  if (!encode_paged_map(&tk, s.a.k, s.token_rows, s.a.hk, kTaD, dtype, p.box) ||
      !encode_paged_map(&tv, s.a.v, s.token_rows, s.a.hk, kTaD, dtype, p.box))
    return fail(DSB_ERR_CUDA, "tensor map of the paged cache");
  launch_kernel(kern, dim3(s.a.hk, p.psplits, p.ztiles), dim3(kSpThreads), kSpSmem, st, tk, tv, s);
  return check_launch("shared_prefix_kernel");
}

template <typename T> int run_typed(const SpArgs &s, const SpPlan &p, int dtype, cudaStream_t st) {
  if (p.shared) {
    const int e = p.query_tiles == 1 ? run_prefix<T, 1>(s, p, dtype, st)
                                     : run_prefix<T, 2>(s, p, dtype, st);
    if (e != DSB_OK) return e;
  }
  const TaArgs &a = s.a;
  auto kern = paged_decode_split_kernel<T, 16, true>;
  constexpr size_t smem = TaSmem<16>::kBytes;
  if (int e = ensure_smem((const void *)kern, smem); e != DSB_OK) return e;
  launch_kernel(kern, dim3(a.hk, a.splits, a.rows), dim3(kTaWarps * 32), smem, st, a);
  if (int e = check_launch("paged_decode_split_kernel (own range)")) return e;
  const dim3 grid((unsigned)((int64_t)a.rows * a.hq));
  if (p.shared)
    launch_kernel(shared_prefix_merge_kernel<T>, grid, dim3(kTaD), 0, st, s);
  else
    launch_kernel(paged_decode_merge_kernel<T>, grid, dim3(kTaD), 0, st, a);
  return check_launch("merge kernel");
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
  return p.acc_floats + p.ml_floats + p.own_floats;
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
  if (p.splits > 65535 || num_kv_heads > 65535 || query_rows > 65535 || p.ztiles > 65535 ||
      (int64_t)query_rows * num_query_heads > INT32_MAX)
    return fail(DSB_ERR_UNSUPPORTED, "grid too large");
  if (num_blocks * block_size >= INT32_MAX)
    return fail(DSB_ERR_UNSUPPORTED, "the cache must hold fewer than 2^31 - 1 tokens");
  if (scratch_floats < p.acc_floats + p.ml_floats + p.own_floats)
    return fail(DSB_ERR_INVALID, "scratch smaller than dsb_shared_prefix_scratch_floats");
  if (reinterpret_cast<uintptr_t>(query) % 16 || reinterpret_cast<uintptr_t>(key_cache) % 16 ||
      reinterpret_cast<uintptr_t>(value_cache) % 16 || reinterpret_cast<uintptr_t>(scratch) % 16)
    return fail(DSB_ERR_UNSUPPORTED, "query, caches and scratch must be 16-byte aligned");
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
  a.splits = (int)p.splits;
  a.tps = p.tps;
  a.page_tiles = block_size % kTaTile == 0 ? 1 : 0;
  a.scale_log2 = scale * kTaLog2e;
  a.out = out;
  a.lse = lse;
  a.err = error_flag;
  if (p.shared) {
    a.prefix_lens = prefix_lens;
    a.group_starts = group_starts;
    a.groups = num_groups;
  }
  s.acc = scratch;
  s.ml = reinterpret_cast<float2 *>(scratch + p.acc_floats);
  a.part = scratch + p.acc_floats + p.ml_floats;
  s.psplits = p.psplits;
  s.token_rows = num_blocks * block_size;
  s.box = p.box;
  cudaStream_t st = as_stream(stream);
  return dtype == DSB_BF16 ? run_typed<__nv_bfloat16>(s, p, dtype, st)
                           : run_typed<__half>(s, p, dtype, st);
}
