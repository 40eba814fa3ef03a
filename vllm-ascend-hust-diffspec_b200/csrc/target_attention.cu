// Target-model paged decode attention that also exports the softmax LSE.
//
// Reference: the target verifier's attention runs as FIA with
// softmax_lse_flag forced on (diffspec/ascend_patch.py:191-240) so that
// capture_target_attention (diffspec/runtime.py:841-894) can keep the LSE
// for the chunk-retrieval scores (kernels.py:11-150 divides by exp(lse)).
// On B200 the LSE falls out of a flash-decode epilogue: this kernel computes
//   out[r, h]  = sum_t softmax_t(scale * q[r, h] . k_t) v_t
//   lse[r, h]  = log sum_t exp(scale * q[r, h] . k_t)          (natural log)
// over the first seq_lens[r] tokens of the row's paged K/V, so retrieval
// can score chunks with it instead of running its own LSE pass.
//
// B200 design: decode attention is bound by the K/V stream (2 * D * 2 bytes
// per token and kv head).  Split-KV: CTA (split, kv head, row) streams
// tokens_per_split tokens of one kv head for all G = Hq / Hk query heads of
// the group (the K/V rows are read once per group, not once per query
// head); each warp takes every fourth 16-token tile and runs it through the
// tensor cores (S = Q K^T and O += P V with mma.sync, base-2 online softmax
// on the accumulators, P split into hi + lo 16-bit terms).  The warps'
// states merge in shared memory and each CTA writes one (max, sum, acc[D])
// partial per query head; a second launch merges the splits in order
// (deterministic) and writes out and lse.  No waits on other CTAs.
#include "paged_split.cuh"

namespace dsb {
namespace {

template <typename T, int G> int launch_group(const TaArgs &a, cudaStream_t st) {
  auto kern = paged_decode_split_kernel<T, G, false>;
  constexpr size_t smem = TaSmem<G>::kBytes;
  if (int e = ensure_smem((const void *)kern, smem); e != DSB_OK) return e;
  launch_kernel(kern, dim3(a.hk, a.splits, a.rows), dim3(kTaWarps * 32), smem, st, a);
  return DSB_OK;
}

template <typename T> int launch_typed(const TaArgs &a, int group, cudaStream_t st) {
  int e = DSB_OK;
  switch (group) {
    case 1: e = launch_group<T, 1>(a, st); break;
    case 2: e = launch_group<T, 2>(a, st); break;
    case 4: e = launch_group<T, 4>(a, st); break;
    case 8: e = launch_group<T, 8>(a, st); break;
    case 16: e = launch_group<T, 16>(a, st); break;
    default: return fail(DSB_ERR_UNSUPPORTED, "query heads per kv head must be 1, 2, 4, 8 or 16");
  }
  if (e != DSB_OK) return e;
  if (int e2 = check_launch("paged_decode_split_kernel")) return e2;
  launch_kernel(paged_decode_merge_kernel<T, false>, dim3((unsigned)(a.rows * a.hq)), dim3(kTaD), 0, st,
                a);
  return check_launch("paged_decode_merge_kernel");
}

// The split length when the caller passes <= 0: 1024 tokens for long
// contexts (max_seq_len >= 16384: fewer CTA ramp-ups and a smaller merge;
// 266 us against 313 us at 16 rows x 40960 tokens), 512 otherwise (more
// splits to fill the GPU when the rows are short).
int32_t default_tokens_per_split(int32_t max_seq_len) {
  return max_seq_len >= 16384 ? 1024 : 512;
}

int64_t splits_for(int32_t max_seq_len, int32_t tokens_per_split) {
  return std::max<int64_t>(1, ((int64_t)max_seq_len + tokens_per_split - 1) / tokens_per_split);
}

}  // namespace
}  // namespace dsb

using namespace dsb;

extern "C" int64_t dsb_paged_decode_scratch_floats(int32_t query_rows, int32_t num_query_heads,
                                                    int32_t max_seq_len, int32_t tokens_per_split) {
  if (query_rows <= 0 || num_query_heads <= 0 || max_seq_len < 0) return 0;
  if (tokens_per_split <= 0) tokens_per_split = default_tokens_per_split(max_seq_len);
  return (int64_t)query_rows * num_query_heads * splits_for(max_seq_len, tokens_per_split) *
         (kTaD + 2);
}

extern "C" int dsb_paged_decode_attention_lse(
    const void *query, int32_t query_rows, int32_t num_query_heads, int32_t num_kv_heads,
    int32_t head_dim, const void *key_cache, const void *value_cache, int64_t num_blocks,
    int32_t block_size, const int32_t *block_table, int64_t block_table_stride,
    int64_t block_table_rows, int64_t block_table_cols, const int32_t *seq_lens,
    const int32_t *table_rows, int32_t max_seq_len, float scale, int32_t dtype,
    int32_t tokens_per_split, void *out, float *lse, float *scratch, int64_t scratch_floats,
    int32_t *error_flag, void *stream) {
  if (query_rows < 0) return fail(DSB_ERR_INVALID, "negative query_rows");
  if (query_rows == 0) return DSB_OK;
  if (dtype != DSB_BF16 && dtype != DSB_F16)
    return fail(DSB_ERR_INVALID, "query and caches must be BF16 or FP16");
  if (num_query_heads <= 0 || num_kv_heads <= 0 || num_query_heads % num_kv_heads)
    return fail(DSB_ERR_INVALID, "query heads must be a positive multiple of kv heads");
  if (head_dim != kTaD) return fail(DSB_ERR_UNSUPPORTED, "head_dim must be 128");
  if (num_blocks <= 0 || block_size <= 0 || block_table_rows <= 0 || block_table_cols <= 0 ||
      block_table_stride < block_table_cols || max_seq_len < 0)
    return fail(DSB_ERR_INVALID, "bad cache or block-table geometry");
  if (tokens_per_split <= 0) tokens_per_split = default_tokens_per_split(max_seq_len);
  if (!(scale > 0.f)) return fail(DSB_ERR_INVALID, "scale must be positive");
  if (!query || !key_cache || !value_cache || !block_table || !seq_lens || !out || !lse || !scratch)
    return fail(DSB_ERR_INVALID, "null pointer argument");
  const int64_t splits = splits_for(max_seq_len, tokens_per_split);
  if (splits > 65535 || num_kv_heads > 65535 || query_rows > 65535)
    return fail(DSB_ERR_UNSUPPORTED, "grid too large");
  if (scratch_floats < dsb_paged_decode_scratch_floats(query_rows, num_query_heads, max_seq_len,
                                                       tokens_per_split))
    return fail(DSB_ERR_INVALID, "scratch smaller than dsb_paged_decode_scratch_floats");
  if (reinterpret_cast<uintptr_t>(query) % 16 || reinterpret_cast<uintptr_t>(key_cache) % 16 ||
      reinterpret_cast<uintptr_t>(value_cache) % 16)
    return fail(DSB_ERR_UNSUPPORTED, "query and caches must be 16-byte aligned");
  TaArgs a{};
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
  a.splits = (int)splits;
  a.tps = tokens_per_split;
  a.page_tiles = (block_size % kTaTile == 0 && tokens_per_split % kTaTile == 0) ? 1 : 0;
  a.scale_log2 = scale * kTaLog2e;
  a.part = scratch;
  a.out = out;
  a.lse = lse;
  a.err = error_flag;
  const int group = num_query_heads / num_kv_heads;
  cudaStream_t st = as_stream(stream);
  return dtype == DSB_BF16 ? launch_typed<__nv_bfloat16>(a, group, st)
                           : launch_typed<__half>(a, group, st);
}
