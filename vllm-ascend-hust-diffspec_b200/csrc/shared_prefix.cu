// Target paged decode attention, with the softmax LSE, for requests that
// share a prefix of their tokens (forked from one prompt, or on one system
// prompt): rows [group_starts[i], group_starts[i + 1]) hold the same tokens
// at positions [0, prefix_lens[i]).
//   out[r, h] = sum_t softmax_t(scale * q[r, h] . k_t) v_t,  t < seq_lens[r]
//   lse[r, h] = log sum_t exp(scale * q[r, h] . k_t)          (natural log)
#include "paged_split.cuh"

namespace dsb {
namespace {

// Tokens of a split of the rows' own range: long ones when the rows alone
// fill the GPU, else shorter ones for more CTAs (a multiple of the tile).
int own_tokens_per_split(int64_t own, int rows, int hk) {
  const int64_t ctas = 4LL * 148 / std::max<int64_t>(1, (int64_t)rows * hk);  // splits wanted
  const int64_t tps = (own + std::max<int64_t>(ctas, 1) - 1) / std::max<int64_t>(ctas, 1);
  return (int)std::min<int64_t>(1024, std::max<int64_t>(64, (tps + 15) / 16 * 16));
}

struct SpPlan {
  int64_t own, splits;  // tokens and splits of the rows' own range
  int tps;
};

SpPlan plan_for(int rows, int hk, int max_prefix, int max_suffix) {
  SpPlan p;
  p.own = (int64_t)max_prefix + max_suffix;
  p.tps = own_tokens_per_split(p.own, rows, hk);
  p.splits = std::max<int64_t>(1, (p.own + p.tps - 1) / p.tps);
  return p;
}

template <typename T> int run_typed(const TaArgs &a, cudaStream_t st) {
  auto kern = paged_decode_split_kernel<T, 16, true>;
  constexpr size_t smem = TaSmem<16>::kBytes;
  if (int e = ensure_smem((const void *)kern, smem); e != DSB_OK) return e;
  launch_kernel(kern, dim3(a.hk, a.splits, a.rows), dim3(kTaWarps * 32), smem, st, a);
  if (int e = check_launch("paged_decode_split_kernel (own range)")) return e;
  launch_kernel(paged_decode_merge_kernel<T>, dim3((unsigned)(a.rows * a.hq)), dim3(kTaD), 0, st,
                a);
  return check_launch("paged_decode_merge_kernel");
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
  const SpPlan p = plan_for(query_rows, num_kv_heads, max_prefix_len, max_suffix_len);
  return (int64_t)query_rows * num_query_heads * p.splits * (kTaD + 2);
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
  const SpPlan p = plan_for(query_rows, num_kv_heads, max_prefix_len, max_suffix_len);
  if (p.splits > 65535 || num_kv_heads > 65535 || query_rows > 65535)
    return fail(DSB_ERR_UNSUPPORTED, "grid too large");
  if (scratch_floats < dsb_shared_prefix_scratch_floats(query_rows, num_query_heads, num_kv_heads,
                                                        num_groups, block_size, max_prefix_len,
                                                        max_suffix_len))
    return fail(DSB_ERR_INVALID, "scratch smaller than dsb_shared_prefix_scratch_floats");
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
  a.splits = (int)p.splits;
  a.tps = p.tps;
  a.page_tiles = block_size % kTaTile == 0 ? 1 : 0;
  a.scale_log2 = scale * kTaLog2e;
  a.part = scratch;
  a.out = out;
  a.lse = lse;
  a.err = error_flag;
  cudaStream_t st = as_stream(stream);
  return dtype == DSB_BF16 ? run_typed<__nv_bfloat16>(a, st) : run_typed<__half>(a, st);
}
