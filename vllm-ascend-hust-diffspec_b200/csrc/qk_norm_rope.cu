// RMSNorm of every query and key head with the position rotation in the same
// pass, and the step's K/V rows written where the next kernels read them.
//
// With x a head of the projection (fp32 math throughout):
//   y   = x * rsqrt(mean(x^2) + eps) * w
//   out = rotate(y, cos, sin of the token's position)
// rounded once, when a value is stored.  The draft layer takes the rotated
// keys and the values as contiguous rows for its attention, and the raw
// cache the normed keys before the rotation (the working-cache rebuild
// rotates them at their local positions); the target's step writes rotated
// keys and values into its pages.
#include <algorithm>

#include "common.cuh"

namespace dsb {
namespace {

enum { kDestNone = 0, kDestRaw = 1, kDestPaged = 2 };

struct QkArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;  // k_out / v_out: contiguous rows, or null
  int64_t q_stride, qo_stride, k_stride, v_stride;  // elements between tokens
  const void *qw, *kw;
  float eps;
  const void *cos_sin;
  int64_t cs_stride;
  const int32_t *positions;
  int pos_offset, rotary_rows;
  int tokens, hq, hk, d, rot, neox;
  // K/V destination: raw caches [dst_rows slots, max_len, hk, d] at
  // [index[t], abs_pos[t]], or pages of table row index[t] (t when null)
  int dest;
  void *dst_k, *dst_v;
  const int32_t *index;
  const int64_t *abs_pos;
  int64_t dst_rows, max_len;
  const int32_t *bt;
  int64_t bt_stride, bt_cols, nblocks;
  int bs;
  int32_t *err;
};

// Row (in units of hk * d elements) of the destination caches that token t's
// K/V go to; -1: none (a padding token, or a bad index, which is flagged).
__device__ __forceinline__ int64_t dest_row(const QkArgs &a, int t, int pos, bool report) {
  if (a.dest == kDestRaw) {
    const int slot = a.index[t];
    if (slot < 0) return -1;
    const int64_t p = a.abs_pos[t];
    if (slot >= a.dst_rows || p < 0 || p >= a.max_len) {
      if (report) flag_error(a.err, slot >= a.dst_rows ? DSB_FLAG_SLOT : DSB_FLAG_POSITION);
      return -1;
    }
    return slot * a.max_len + p;
  }
  const int row = a.index != nullptr ? a.index[t] : t;
  if (row < 0) return -1;
  if (row >= a.dst_rows || pos < 0 || pos / a.bs >= a.bt_cols) {
    if (report) flag_error(a.err, row >= a.dst_rows ? DSB_FLAG_SLOT : DSB_FLAG_POSITION);
    return -1;
  }
  const int64_t page = a.bt[row * a.bt_stride + pos / a.bs];
  if (page < 0 || page >= a.nblocks) {
    if (report) flag_error(a.err, DSB_FLAG_BLOCK);
    return -1;
  }
  return page * a.bs + pos % a.bs;
}

// ---------------------------------------------------------------- any head
// One warp per (token, head), heads in the order q, k, v, for head sizes,
// partial rotations and alignments that the kernel below does not take.
// Element pairs that rotate together are read and written by one lane, so
// q_out may be q.
template <typename T, typename CS>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(const QkArgs a) {
  pdl_begin();
  const int64_t warp = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int heads = a.hq + 2 * a.hk;
  if (warp >= (int64_t)a.tokens * heads) return;
  const int t = (int)(warp / heads), h = (int)(warp % heads);
  const int d = a.d;
  const int pos = a.positions[t] + a.pos_offset;
  const bool is_q = h < a.hq;
  const int kh = is_q ? 0 : (h - a.hq) % a.hk;
  int64_t row = -1;
  if (!is_q && a.dest != kDestNone)
    row = dest_row(a, t, pos, lane == 0 && h == a.hq);
  T *dst_v = nullptr, *dst_k = nullptr;
  if (row >= 0) {
    dst_k = static_cast<T *>(a.dst_k) + (row * a.hk + kh) * d;
    dst_v = static_cast<T *>(a.dst_v) + (row * a.hk + kh) * d;
  }
  const int64_t out_row = ((int64_t)t * a.hk + kh) * d;
  if (h >= a.hq + a.hk) {  // value head: copied
    const T *src = static_cast<const T *>(a.v) + t * a.v_stride + (int64_t)kh * d;
    T *out = a.v_out != nullptr ? static_cast<T *>(a.v_out) + out_row : nullptr;
    for (int i = lane; i < d; i += 32) {
      const T x = src[i];
      if (out != nullptr) out[i] = x;
      if (dst_v != nullptr) dst_v[i] = x;
    }
    return;
  }
  const T *src = is_q ? static_cast<const T *>(a.q) + t * a.q_stride + (int64_t)h * d
                      : static_cast<const T *>(a.k) + t * a.k_stride + (int64_t)kh * d;
  T *out = is_q ? static_cast<T *>(a.q_out) + t * a.qo_stride + (int64_t)h * d
                : (a.k_out != nullptr ? static_cast<T *>(a.k_out) + out_row : nullptr);
  const T *w = static_cast<const T *>(is_q ? a.qw : a.kw);
  float ss = 0.f;
  for (int i = lane; i < d; i += 32) {
    const float x = Elem<T>::to_f(src[i]);
    ss = fmaf(x, x, ss);
  }
  const float inv = rsqrtf(warp_sum(ss) / static_cast<float>(d) + a.eps);
  bool turn = true;
  if (pos < 0 || pos >= a.rotary_rows) {  // no such row of the table: normed only
    if (lane == 0 && h == 0) flag_error(a.err, DSB_FLAG_POSITION);
    turn = false;
  }
  const CS *cs = static_cast<const CS *>(a.cos_sin) + (turn ? pos : 0) * a.cs_stride;
  const int half = a.rot / 2;
  auto put = [&](int i, float y, float rotated) {
    if (out != nullptr) out[i] = Elem<T>::from_f(rotated);
    if (dst_k != nullptr) dst_k[i] = Elem<T>::from_f(a.dest == kDestRaw ? y : rotated);
  };
  for (int i = lane; i < half; i += 32) {
    const int i1 = a.neox ? i : 2 * i, i2 = a.neox ? i + half : 2 * i + 1;
    const float y1 = Elem<T>::to_f(src[i1]) * inv * Elem<T>::to_f(w[i1]);
    const float y2 = Elem<T>::to_f(src[i2]) * inv * Elem<T>::to_f(w[i2]);
    const float c = turn ? Elem<CS>::to_f(cs[i]) : 1.f;
    const float s = turn ? Elem<CS>::to_f(cs[i + half]) : 0.f;
    put(i1, y1, turn ? y1 * c - y2 * s : y1);
    put(i2, y2, turn ? y2 * c + y1 * s : y2);
  }
  for (int i = a.rot + lane; i < d; i += 32) {
    const float y = Elem<T>::to_f(src[i]) * inv * Elem<T>::to_f(w[i]);
    put(i, y, y);
  }
}

// ------------------------------------------------------------- whole heads
// Heads of D = 64, 128 or 256 rotated in full, 16-byte aligned rows: D / 16
// lanes a head, a lane 16 of its elements in two 16-byte pieces that rotate
// with each other (NeoX: elements 8 l .. and D / 2 + 8 l ..; pairs: 16 l ..),
// so the rotation needs no exchange and the norm a few shuffles.  A thread
// takes kQkHeads heads of one token at once: its loads are all on their way
// before the first is used, and one row of cosines and sines serves them.
constexpr int kQkHeads = 4;

template <typename T> __device__ __forceinline__ void qk_unpack(const uint4 &w, float (&v)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(u[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T> __device__ __forceinline__ uint4 qk_pack(const float (&v)[8]) {
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                    pack2<T>(v[6], v[7]));
}
// 8 consecutive entries of the table
template <typename CS> __device__ __forceinline__ void qk_table(const CS *p, float (&v)[8]) {
  qk_unpack<CS>(*reinterpret_cast<const uint4 *>(p), v);
}
template <> __device__ __forceinline__ void qk_table<float>(const float *p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// 16 bytes that no other thread reads, kept out of L1 (not through the
// read-only path: the queries may be rotated in place).
__device__ __forceinline__ uint4 qk_load(const void *p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// A lane's two pieces of a head: the mean of the head's squares.
template <int D>
__device__ __forceinline__ float qk_mean_square(const float (&v1)[8], const float (&v2)[8]) {
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = fmaf(v1[j], v1[j], fmaf(v2[j], v2[j], ss));
#pragma unroll
  for (int o = D / 32; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  return ss * (1.f / D);
}

// What turns a head's pieces: out = inv * (v1 * c1 - v2' * s2 ...), the weight
// and the cosines and sines of the token in one factor each, shared by the
// heads that a thread takes.  A lane's 16 elements make 8 pairs (x, y):
// NeoX (v1[j], v2[j]), else neighbours.
struct QkTurn {
  float xc[8], ys[8], yc[8], xs[8];  // wx c, wy s, wy c, wx s
};

template <typename T, typename CS, int D, bool NEOX>
__device__ __forceinline__ void qk_factors(QkTurn &f, const T *w, const CS *cs, int l, bool turn) {
  float c[8], n[8], w1[8], w2[8];
  qk_table<CS>(cs + 8 * l, c);
  qk_table<CS>(cs + D / 2 + 8 * l, n);
  qk_unpack<T>(*reinterpret_cast<const uint4 *>(w + (NEOX ? 8 * l : 16 * l)), w1);
  qk_unpack<T>(*reinterpret_cast<const uint4 *>(w + (NEOX ? D / 2 + 8 * l : 16 * l + 8)), w2);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float wx = NEOX ? w1[j] : (j < 4 ? w1[2 * j] : w2[2 * j - 8]);
    const float wy = NEOX ? w2[j] : (j < 4 ? w1[2 * j + 1] : w2[2 * j - 7]);
    const float cj = turn ? c[j] : 1.f, sj = turn ? n[j] : 0.f;
    f.xc[j] = wx * cj, f.ys[j] = wy * sj;
    f.yc[j] = wy * cj, f.xs[j] = wx * sj;
  }
}

template <bool NEOX>
__device__ __forceinline__ void qk_turn(const QkTurn &f, float inv, const float (&v1)[8],
                                        const float (&v2)[8], float (&o1)[8], float (&o2)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = NEOX ? v1[j] : (j < 4 ? v1[2 * j] : v2[2 * j - 8]);
    const float y = NEOX ? v2[j] : (j < 4 ? v1[2 * j + 1] : v2[2 * j - 7]);
    const float a = inv * (x * f.xc[j] - y * f.ys[j]), b = inv * (y * f.yc[j] + x * f.xs[j]);
    if (NEOX) {
      o1[j] = a, o2[j] = b;
    } else if (j < 4) {
      o1[2 * j] = a, o1[2 * j + 1] = b;
    } else {
      o2[2 * j - 8] = a, o2[2 * j - 7] = b;
    }
  }
}

// A warp takes kPer query heads of one token, or kPer of its key and value
// heads.  Bound by memory, by way of the loads in flight and of how soon a
// finished warp's place is taken: 65536 tokens of 32/4 heads of 128 into
// pages (1.35 GB) take 281 us with 16 warps of 123 registers an SM in CTAs of
// 256 threads, 247 with 24 warps of 80 (every instance then spills, 116 to 200
// bytes stored and 360 to 532 read again a thread), 235 with stores that do not
// stay in the way in L2, 227 in CTAs of 64 (one launch by itself, 5.9 TB/s; 242
// in a run of calls, 5.6 TB/s, 0.85 of the measured copy).  Two or six heads a
// thread are slower (268 and 286), and so is asking later rows into L2 ahead of
// their warps (243 for 235).
constexpr int kQkThreads = 64;

// With fewer query heads (keys and values) than half of what a warp takes, it
// takes 2, 4 or 8 tokens side by side (QSIDE, KSIDE).  400000 tokens of 8/1
// heads of 64: 705 us with one token a warp, 234 so; 60000 of 32/4 heads of 64:
// 135 and 123.  Not the keys and values of D = 256, two of whose heads are a
// warp's width (47725 tokens of 12/2 heads: 174 and 186).
__host__ __device__ __forceinline__ int qk_side(int heads, int per, int groups) {
  int n = 1;
  while (2 * n <= groups && per / (2 * n) >= heads) n *= 2;
  return n;
}
// The warps of a run of tokens: those of the query heads, then those of the
// keys and values.
struct QkWarps {
  int qside, kside, tokens, qchunks, kchunks, q, all;
  __host__ __device__ QkWarps(int hq, int hk, int groups, bool qs, bool ks) {
    const int per = groups * kQkHeads;
    qside = qs ? qk_side(hq, per, groups) : 1;
    kside = ks ? qk_side(2 * hk, per, groups) : 1;
    tokens = qside > kside ? qside : kside;
    qchunks = (hq + per / qside - 1) / (per / qside);
    kchunks = (2 * hk + per / kside - 1) / (per / kside);
    q = tokens / qside * qchunks;
    all = q + tokens / kside * kchunks;
  }
};

template <typename T, typename CS, int D, bool NEOX, bool QSIDE, bool KSIDE>
__global__ void __launch_bounds__(kQkThreads, 12) qk_norm_rope_heads_kernel(const QkArgs a) {
  constexpr int kLanes = D / 16;  // of a head
  pdl_begin();
  const QkWarps w(a.hq, a.hk, 32 / kLanes, QSIDE, KSIDE);
  const int64_t warp = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31, l = lane % kLanes;
  const int64_t run = warp / w.all;
  const int of_run = (int)(warp - run * w.all);
  const bool queries = of_run < w.q;
  const int u = queries ? of_run : of_run - w.q, chunks = queries ? w.qchunks : w.kchunks;
  const int side = queries ? (QSIDE ? w.qside : 1) : (KSIDE ? w.kside : 1);
  const int kGroups = 32 / kLanes / side;  // heads of a token that a warp has side by side
  const int group = lane / kLanes % kGroups;
  int chunk = u, turn_of = 0;  // of the run's tokens
  if (QSIDE || KSIDE) {
    turn_of = chunks == 1 ? u : u / chunks;
    chunk = u - turn_of * chunks;
  }
  const int64_t token0 = run * w.tokens + turn_of * side;
  if (token0 >= a.tokens) return;
  const int64_t mine = token0 + (QSIDE || KSIDE ? lane / kLanes / kGroups : 0);
  const bool live = !(QSIDE || KSIDE) || mine < a.tokens;  // (else its lanes only take part)
  const int t = (int)(live ? mine : a.tokens - 1);
  const bool first = QSIDE || KSIDE ? live && lane % (kLanes * kGroups) == 0 : lane == 0;
  const int e1 = NEOX ? 8 * l : 16 * l, e2 = NEOX ? D / 2 + 8 * l : 16 * l + 8;
  const int pos = a.positions[t] + a.pos_offset;
  const bool turn = pos >= 0 && pos < a.rotary_rows;  // else: normed, not rotated
  const CS *cs = static_cast<const CS *>(a.cos_sin) + (turn ? pos : 0) * a.cs_stride;
  uint4 x1[kQkHeads], x2[kQkHeads];
  QkTurn f;

  if (queries) {
    const int h0 = chunk * kGroups * kQkHeads + group;
    const T *src = static_cast<const T *>(a.q) + t * a.q_stride + (int64_t)h0 * D;
#pragma unroll
    for (int i = 0; i < kQkHeads; ++i) {  // (a head past the last: zeros, not stored)
      const bool in = live && h0 + i * kGroups < a.hq;
      x1[i] = in ? qk_load(src + i * kGroups * D + e1) : make_uint4(0, 0, 0, 0);
      x2[i] = in ? qk_load(src + i * kGroups * D + e2) : make_uint4(0, 0, 0, 0);
    }
    if (!turn && first && chunk == 0) flag_error(a.err, DSB_FLAG_POSITION);
    qk_factors<T, CS, D, NEOX>(f, static_cast<const T *>(a.qw), cs, l, turn);
    T *out = static_cast<T *>(a.q_out) + t * a.qo_stride + (int64_t)h0 * D;
#pragma unroll
    for (int i = 0; i < kQkHeads; ++i) {
      float v1[8], v2[8], o1[8], o2[8];
      qk_unpack<T>(x1[i], v1);
      qk_unpack<T>(x2[i], v2);
      const float inv = rsqrtf(qk_mean_square<D>(v1, v2) + a.eps);
      qk_turn<NEOX>(f, inv, v1, v2, o1, o2);
      if (live && h0 + i * kGroups < a.hq) {
        __stcs(reinterpret_cast<uint4 *>(out + i * kGroups * D + e1), qk_pack<T>(o1));
        __stcs(reinterpret_cast<uint4 *>(out + i * kGroups * D + e2), qk_pack<T>(o2));
      }
    }
    return;
  }

  const int k0 = chunk * kGroups * kQkHeads, h0 = k0 + group;  // keys, then values
  const T *key = static_cast<const T *>(a.k) + t * a.k_stride;
  const T *value = static_cast<const T *>(a.v) + t * a.v_stride;
#pragma unroll
  for (int i = 0; i < kQkHeads; ++i) {
    const int h = h0 + i * kGroups;
    const T *src = h < a.hk ? key + h * D : value + (h - a.hk) * D;
    const bool in = live && h < 2 * a.hk;
    x1[i] = in ? qk_load(src + e1) : make_uint4(0, 0, 0, 0);
    x2[i] = in ? qk_load(src + e2) : make_uint4(0, 0, 0, 0);
  }
  const int64_t row = a.dest != kDestNone ? dest_row(a, t, pos, first) : -1;
  if (k0 < a.hk) qk_factors<T, CS, D, NEOX>(f, static_cast<const T *>(a.kw), cs, l, turn);
#pragma unroll
  for (int i = 0; i < kQkHeads; ++i) {
    const int h = h0 + i * kGroups;
    uint4 r1 = x1[i], r2 = x2[i], y1 = x1[i], y2 = x2[i];
    if (k0 + i * kGroups < a.hk) {  // some of the warp's heads are keys
      float v1[8], v2[8], o1[8], o2[8];
      qk_unpack<T>(x1[i], v1);
      qk_unpack<T>(x2[i], v2);
      const float inv = rsqrtf(qk_mean_square<D>(v1, v2) + a.eps);
      if (h < a.hk) {
        qk_turn<NEOX>(f, inv, v1, v2, o1, o2);
        r1 = qk_pack<T>(o1), r2 = qk_pack<T>(o2);
        if (a.dest == kDestRaw) {  // the raw cache holds them before the rotation
          float w1[8], w2[8];
          const T *w = static_cast<const T *>(a.kw);
          qk_unpack<T>(*reinterpret_cast<const uint4 *>(w + e1), w1);
          qk_unpack<T>(*reinterpret_cast<const uint4 *>(w + e2), w2);
#pragma unroll
          for (int j = 0; j < 8; ++j) v1[j] *= inv * w1[j], v2[j] *= inv * w2[j];
          y1 = qk_pack<T>(v1), y2 = qk_pack<T>(v2);
        }
      }
    }
    if (!live || h >= 2 * a.hk) continue;
    const bool is_key = h < a.hk;
    const int kh = is_key ? h : h - a.hk;
    T *out = static_cast<T *>(is_key ? a.k_out : a.v_out);
    if (out != nullptr) {
      out += ((int64_t)t * a.hk + kh) * D;
      __stcs(reinterpret_cast<uint4 *>(out + e1), r1);
      __stcs(reinterpret_cast<uint4 *>(out + e2), r2);
    }
    if (row >= 0) {
      T *dst = static_cast<T *>(is_key ? a.dst_k : a.dst_v) + (row * a.hk + kh) * D;
      const bool raw = a.dest == kDestRaw;
      __stcs(reinterpret_cast<uint4 *>(dst + e1), raw ? y1 : r1);
      __stcs(reinterpret_cast<uint4 *>(dst + e2), raw ? y2 : r2);
    }
  }
}

// Whether the whole-head kernel takes the call: its pieces are 16 bytes.
bool whole_heads(const QkArgs &a, int cos_sin_dtype) {
  auto ok = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const int64_t cs_step = cos_sin_dtype == DSB_F32 ? 4 : 8;
  return (a.d == 64 || a.d == 128 || a.d == 256) && a.rot == a.d && ok(a.q) && ok(a.q_out) &&
         ok(a.k) && ok(a.v) && ok(a.k_out) && ok(a.v_out) && ok(a.dst_k) && ok(a.dst_v) && ok(a.qw) &&
         ok(a.kw) && ok(a.cos_sin) && a.q_stride % 8 == 0 && a.qo_stride % 8 == 0 &&
         a.k_stride % 8 == 0 && a.v_stride % 8 == 0 && a.cs_stride % cs_step == 0;
}

template <typename T, typename CS, int D> void launch_heads(const QkArgs &a, cudaStream_t st) {
  const QkWarps w(a.hq, a.hk, 32 / (D / 16), true, D < 256);
  const int64_t warps = ((int64_t)a.tokens + w.tokens - 1) / w.tokens * w.all;
  constexpr int kWarps = kQkThreads / 32;
  const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps)), block(kQkThreads);
  auto with = [&](auto neox, auto qside, auto kside) {
    launch_kernel(qk_norm_rope_heads_kernel<T, CS, D, neox(), qside(), kside()>, grid, block, 0, st, a);
  };
  auto sides = [&](auto neox) {
    using Yes = std::true_type;
    using No = std::false_type;
    if constexpr (D < 256) {
      if (w.kside > 1) return w.qside > 1 ? with(neox, Yes(), Yes()) : with(neox, No(), Yes());
    }
    w.qside > 1 ? with(neox, Yes(), No()) : with(neox, No(), No());
  };
  a.neox ? sides(std::true_type()) : sides(std::false_type());
}

int launch(const QkArgs &a, int cos_sin_dtype, int dtype, cudaStream_t st) {
  const int64_t warps = (int64_t)a.tokens * (a.hq + 2 * a.hk);
  if ((warps + 7) / 8 > INT32_MAX) return fail(DSB_ERR_UNSUPPORTED, "grid too large");
  const dim3 grid((unsigned)((warps + 7) / 8)), block(256);
  const bool whole = whole_heads(a, cos_sin_dtype);
  auto with = [&](auto tag, auto table) {
    using T = decltype(tag);
    using CS = decltype(table);
    if (!whole)
      launch_kernel(qk_norm_rope_kernel<T, CS>, grid, block, 0, st, a);
    else if (a.d == 64)
      launch_heads<T, CS, 64>(a, st);
    else if (a.d == 128)
      launch_heads<T, CS, 128>(a, st);
    else
      launch_heads<T, CS, 256>(a, st);
  };
  auto go = [&](auto tag) {
    if (cos_sin_dtype == DSB_F32)
      with(tag, 0.f);
    else if (cos_sin_dtype == DSB_BF16)
      with(tag, __nv_bfloat16());
    else
      with(tag, __half());
  };
  if (dtype == DSB_BF16)
    go(__nv_bfloat16());
  else
    go(__half());
  return check_launch("qk_norm_rope_kernel");
}

// What both entry points check; fills the common arguments.
int prepare(QkArgs &a, const void *query, int64_t query_row_stride, void *query_out,
            int64_t query_out_row_stride, int num_query_heads, const void *key,
            int64_t key_row_stride, const void *value, int64_t value_row_stride, int num_kv_heads,
            int head_dim, int rotary_dim, int is_neox, const void *q_weight, const void *k_weight,
            float eps, const int32_t *positions, int position_offset, int tokens,
            const void *cos_sin, int64_t cos_sin_row_stride, int rotary_rows, int cos_sin_dtype,
            int dtype, int32_t *error_flag) {
  if (dtype != DSB_BF16 && dtype != DSB_F16)
    return fail(DSB_ERR_INVALID, "queries and keys must be BF16 or FP16");
  if (cos_sin_dtype != DSB_BF16 && cos_sin_dtype != DSB_F16 && cos_sin_dtype != DSB_F32)
    return fail(DSB_ERR_INVALID, "cos_sin must be BF16, FP16 or FP32");
  if (num_query_heads <= 0 || num_kv_heads <= 0)
    return fail(DSB_ERR_INVALID, "head counts must be positive");
  if (head_dim <= 0 || rotary_dim < 0 || rotary_dim % 2 || rotary_dim > head_dim ||
      rotary_rows <= 0 || cos_sin_row_stride < rotary_dim)
    return fail(DSB_ERR_INVALID,
                "rotary_dim must be even and at most head_dim; cos_sin rows hold [cos | sin] of it");
  if (!(eps >= 0.f)) return fail(DSB_ERR_INVALID, "eps must be >= 0");
  if (!query || !query_out || !key || !value || !q_weight || !k_weight || !positions || !cos_sin)
    return fail(DSB_ERR_INVALID, "null pointer argument");
  const int64_t q_row = (int64_t)num_query_heads * head_dim, kv_row = (int64_t)num_kv_heads * head_dim;
  if (query_row_stride < q_row || query_out_row_stride < q_row || key_row_stride < kv_row ||
      value_row_stride < kv_row)
    return fail(DSB_ERR_INVALID, "row stride shorter than its heads");
  if (query_out == query && query_out_row_stride != query_row_stride)
    return fail(DSB_ERR_INVALID, "in-place queries need one row stride");
  a.q = query, a.k = key, a.v = value;
  a.q_out = query_out;
  a.q_stride = query_row_stride, a.qo_stride = query_out_row_stride;
  a.k_stride = key_row_stride, a.v_stride = value_row_stride;
  a.qw = q_weight, a.kw = k_weight, a.eps = eps;
  a.cos_sin = cos_sin, a.cs_stride = cos_sin_row_stride;
  a.positions = positions, a.pos_offset = position_offset, a.rotary_rows = rotary_rows;
  a.tokens = tokens, a.hq = num_query_heads, a.hk = num_kv_heads, a.d = head_dim;
  a.rot = rotary_dim, a.neox = is_neox ? 1 : 0;
  a.err = error_flag;
  return DSB_OK;
}

}  // namespace
}  // namespace dsb

using namespace dsb;

extern "C" int dsb_qk_norm_rope(
    const void *query, int64_t query_row_stride, void *query_out, int64_t query_out_row_stride,
    int32_t num_query_heads, const void *key, int64_t key_row_stride, void *key_out,
    const void *value, int64_t value_row_stride, void *value_out, int32_t num_kv_heads,
    int32_t head_dim, int32_t rotary_dim, int32_t is_neox, const void *q_weight,
    const void *k_weight, float eps, const int32_t *positions, int32_t position_offset,
    int32_t tokens, const void *cos_sin, int64_t cos_sin_row_stride, int32_t rotary_rows,
    int32_t cos_sin_dtype, int32_t dtype, void *raw_key, void *raw_value, const int32_t *slots,
    const int64_t *abs_positions, int32_t num_slots, int64_t max_model_len, int32_t *error_flag,
    void *stream) {
  if (tokens < 0) return fail(DSB_ERR_INVALID, "negative token count");
  if (tokens == 0) return DSB_OK;
  QkArgs a{};
  if (int e = prepare(a, query, query_row_stride, query_out, query_out_row_stride, num_query_heads,
                      key, key_row_stride, value, value_row_stride, num_kv_heads, head_dim,
                      rotary_dim, is_neox, q_weight, k_weight, eps, positions, position_offset,
                      tokens, cos_sin, cos_sin_row_stride, rotary_rows, cos_sin_dtype, dtype,
                      error_flag))
    return e;
  if (!key_out || !value_out) return fail(DSB_ERR_INVALID, "null pointer argument");
  a.k_out = key_out, a.v_out = value_out;
  if (raw_key != nullptr || raw_value != nullptr) {
    if (!raw_key || !raw_value || !slots || !abs_positions)
      return fail(DSB_ERR_INVALID, "the raw caches come together, with slots and positions");
    if (num_slots <= 0 || max_model_len <= 0)
      return fail(DSB_ERR_INVALID, "raw cache geometry must be positive");
    a.dest = kDestRaw;
    a.dst_k = raw_key, a.dst_v = raw_value;
    a.index = slots, a.abs_pos = abs_positions;
    a.dst_rows = num_slots, a.max_len = max_model_len;
  }
  return launch(a, cos_sin_dtype, dtype, as_stream(stream));
}

extern "C" int dsb_qk_norm_rope_paged(
    const void *query, int64_t query_row_stride, void *query_out, int64_t query_out_row_stride,
    int32_t num_query_heads, const void *key, int64_t key_row_stride, const void *value,
    int64_t value_row_stride, int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim,
    int32_t is_neox, const void *q_weight, const void *k_weight, float eps,
    const int32_t *positions, int32_t tokens, const void *cos_sin, int64_t cos_sin_row_stride,
    int32_t rotary_rows, int32_t cos_sin_dtype, int32_t dtype, void *key_cache, void *value_cache,
    int64_t num_blocks, int32_t block_size, const int32_t *block_table, int64_t block_table_stride,
    int64_t block_table_rows, int64_t block_table_cols, const int32_t *table_rows,
    int32_t *error_flag, void *stream) {
  if (tokens < 0) return fail(DSB_ERR_INVALID, "negative token count");
  if (tokens == 0) return DSB_OK;
  QkArgs a{};
  if (int e = prepare(a, query, query_row_stride, query_out, query_out_row_stride, num_query_heads,
                      key, key_row_stride, value, value_row_stride, num_kv_heads, head_dim,
                      rotary_dim, is_neox, q_weight, k_weight, eps, positions, 0, tokens, cos_sin,
                      cos_sin_row_stride, rotary_rows, cos_sin_dtype, dtype, error_flag))
    return e;
  if (!key_cache || !value_cache || !block_table)
    return fail(DSB_ERR_INVALID, "null pointer argument");
  if (num_blocks <= 0 || block_size <= 0 || block_table_rows <= 0 || block_table_cols <= 0 ||
      block_table_stride < block_table_cols)
    return fail(DSB_ERR_INVALID, "bad cache or block-table geometry");
  a.dest = kDestPaged;
  a.dst_k = key_cache, a.dst_v = value_cache;
  a.index = table_rows, a.dst_rows = block_table_rows;
  a.bt = block_table, a.bt_stride = block_table_stride, a.bt_cols = block_table_cols;
  a.nblocks = num_blocks, a.bs = block_size;
  return launch(a, cos_sin_dtype, dtype, as_stream(stream));
}
