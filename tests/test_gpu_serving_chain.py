"""Pages, norms and shared-prefix attention as a serving step uses them
together, and inside the framework's own paths: requests forked from a prompt,
their new tokens normed, rotated and written into pages, the target's
attention over the shared prefix with its LSE, the retrieval that divides by
it, the pool compacted; the draft layer whose heads are normed; the runtime's
target attention with shared prefixes."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from conftest import close_bf16

pytestmark = pytest.mark.gpu

_BF = torch.bfloat16


def _table(rows, d, cuda, base=1e6):
    angle = torch.arange(rows, device=cuda, dtype=torch.float64)[:, None] * (
        base ** (-torch.arange(0, d, 2, device=cuda, dtype=torch.float64) / d))[None]
    return torch.cat((angle.cos(), angle.sin()), 1)


def _plain_heads(x, w, cos_sin, eps):
    """RMSNorm of heads and NeoX rotation in fp64."""
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    c, s = cos_sin.double()[:, None].chunk(2, -1)
    a, b = y.chunk(2, -1)
    return y, torch.cat((a * c - b * s, b * c + a * s), -1)


def test_forked_requests_decode_together(dsb, cuda):
    """Eight requests forked from one prompt of 999 tokens, five steps of one
    token each through pages, norms and attention; every step against fp64 over
    a dense copy of each request's keys and values."""
    hq, hk, d, page, pages, n, prompt, steps = 16, 2, 128, 16, 160, 8, 999, 5
    g = torch.Generator(device=cuda).manual_seed(5)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    refs = torch.zeros(pages, dtype=torch.int32, device=cuda)
    tables = torch.full((n + 1, 70), -1, dtype=torch.int32, device=cuda)
    held = torch.zeros(n + 1, dtype=torch.int32, device=cuda)
    cache = [torch.full((pages, page, hk, d), float("nan"), dtype=_BF, device=cuda) for _ in range(2)]
    cs = _table(1100, d, cuda).to(_BF)
    wq, wk = (1 + 0.2 * torch.randn(d, generator=g, device=cuda) for _ in range(2))
    wq, wk, eps = wq.to(_BF), wk.to(_BF), 1e-6

    def project(tokens):
        return torch.randn((tokens, (hq + 2 * hk) * d), generator=g, device=cuda).to(_BF)

    def write(qkv, positions, rows):
        out = torch.empty((qkv.shape[0], hq * d), dtype=_BF, device=cuda)
        return dsb.kernels.qk_norm_rope_write_paged(
            qkv[:, : hq * d], qkv[:, hq * d:], positions, cs, *cache, tables, wq, wk, eps,
            table_rows=rows, query_out=out)

    # the prompt in row 0, then its children in rows 1..8; the parent leaves
    dsb.pages.resize_requests(refs, tables, held, ints([0]), ints([prompt]), block_size=page)
    qkv = project(prompt)
    at = torch.arange(prompt, device=cuda, dtype=torch.int32)
    write(qkv, at, torch.zeros_like(at))
    dense = [(_plain_heads(qkv[:, hq * d: (hq + hk) * d].view(-1, hk, d), wk, cs[:prompt], eps)[1],
              qkv[:, (hq + hk) * d:].view(-1, hk, d).double())] * n
    children = list(range(1, n + 1))
    dsb.pages.fork_requests(refs, tables, held, ints([0] * n), ints(children), ints([prompt] * n), cache)
    dsb.pages.resize_requests(refs, tables, held, ints([0]), ints([0]), block_size=page)
    for step in range(steps):
        length = prompt + step + 1
        st = dsb.pages.resize_requests(refs, tables, held, ints(children), ints([length] * n),
                                       block_size=page)
        qkv = project(n)
        rows, pos = ints(children), ints([length - 1] * n)
        query = write(qkv, pos, rows)
        out, lse = dsb.kernels.shared_prefix_attention_lse(
            query.view(n, hq, d), *cache, tables, ints([length] * n), ints([prompt]), scale=d ** -0.5,
            max_prefix_len=prompt, max_suffix_len=step + 1, table_rows=rows)
        plain, plain_lse = dsb.kernels.paged_decode_attention_lse(
            query.view(n, hq, d), *cache, tables, ints([length] * n), scale=d ** -0.5,
            max_seq_len=length, table_rows=rows)
        close_bf16(out.float().cpu().numpy(), plain.float().cpu().numpy(), max_rel=2.0 ** -7)
        np.testing.assert_allclose(lse.cpu().numpy(), plain_lse.cpu().numpy(), atol=2e-5)
        new_k = _plain_heads(qkv[:, hq * d: (hq + hk) * d].view(n, hk, d), wk, cs[pos.long()], eps)[1]
        new_v = qkv[:, (hq + hk) * d:].view(n, hk, d).double()
        dense = [(torch.cat((k, new_k[i: i + 1])), torch.cat((v, new_v[i: i + 1])))
                 for i, (k, v) in enumerate(dense)]
        q = _plain_heads(qkv[:, : hq * d].view(n, hq, d), wq, cs[pos.long()], eps)[1]
        for i, (k, v) in enumerate(dense):
            s = torch.einsum("kgd,tkd->kgt", q[i].view(hk, hq // hk, d), k) * d ** -0.5
            ref = torch.einsum("kgt,tkd->kgd", torch.softmax(s, -1), v).reshape(hq, d)
            # the query and key are rounded to bf16 on the way: the path's tolerance
            close_bf16(out[i].float().cpu().numpy(), ref.cpu().numpy(), mean_rel=2e-2)
        assert st[0] == 0
    # the exported LSE in the retrieval scores, against the ones they compute
    kw = dict(chunk_size=32, max_seq_len=length, scale=d ** -0.5)
    table = tables[1:].contiguous()
    args = (query.view(n, hq, d), cache[0])
    with_lse = dsb.kernels.paged_chunk_attention_scores(*args, lse, table, ints([length] * n), **kw)
    alone = dsb.kernels.paged_chunk_attention_scores(*args, None, table, ints([length] * n), **kw)
    np.testing.assert_allclose(with_lse.cpu().numpy(), alone.cpu().numpy(), rtol=1e-3, atol=1e-7)
    # some leave, the pool is compacted, the others see the same tokens
    dsb.pages.resize_requests(refs, tables, held, ints([1, 3, 6]), ints([0] * 3), block_size=page)
    live = int((refs > 0).sum())
    dsb.pages.compact_pages(refs, tables, held, cache)
    assert int((refs[:live] > 0).sum()) == live and not refs[live:].any()
    stay = [2, 4, 5, 7, 8]
    keep = torch.tensor([i - 1 for i in stay], device=cuda)
    again, again_lse = dsb.kernels.shared_prefix_attention_lse(
        query.view(n, hq, d)[keep], *cache, tables, ints([length] * 5), ints([prompt]),
        scale=d ** -0.5, max_prefix_len=prompt, max_suffix_len=steps, table_rows=ints(stay))
    close_bf16(again.float().cpu().numpy(), out[keep].float().cpu().numpy(), max_rel=2.0 ** -7)
    np.testing.assert_allclose(again_lse.cpu().numpy(), lse[keep].cpu().numpy(), atol=2e-5)
    torch.cuda.synchronize()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("groups", [([300], [4]), ([300, 0, 130], [2, 3, 4]), ([0], [4])])
def test_runtime_target_attention_with_shared_prefixes(dsb, cuda, groups):
    """DiffSpecDraftCache.run_target_attention with shared_prefix: the plain
    call's outputs and LSE, and a retrieval driven by them."""
    g = torch.Generator(device=cuda).manual_seed(len(groups[0]))
    hq, hk, d, page = 16, 2, 128, 16
    seq_lens, span = [340, 301, 333, 420], 3
    cols = 30
    table = torch.arange(4 * cols, device=cuda, dtype=torch.int32).view(4, cols)
    begin = 0
    cache = [torch.randn((4 * cols, page, hk, d), generator=g, device=cuda).to(_BF) for _ in range(2)]
    for prefix, end in zip(*groups):
        table[begin:end, : prefix // page] = table[begin, : prefix // page].clone()
        if prefix % page:
            for r in range(begin, end):
                for c in cache:
                    c[table[r, prefix // page].long(), : prefix % page] = c[
                        table[begin, prefix // page].long(), : prefix % page].clone()
        begin = end
    query = torch.randn((4 * span, hq, d), generator=g, device=cuda).to(_BF)
    meta = SimpleNamespace(actual_seq_lengths_q=[3, 6, 9, 12], seq_lens_list=seq_lens,
                           block_tables=table, num_prefills=0)
    got = []
    for shared in (None, groups):
        cache_ = dsb.runtime.DiffSpecDraftCache(
            dsb.runtime.DiffSpecSettings(16, 128, 1, 4, 3, 0.7, False), max_num_reqs=4,
            max_model_len=512, num_kv_heads=hk, head_dim=d, target_num_layers=2, dtype=_BF,
            device=cuda, cos_sin_cache=torch.zeros((128, d), device=cuda).to(_BF))
        cache_.begin_target_forward(["a", "b", "c", "d"])
        kw = {} if shared is None else dict(shared_prefix=shared)
        out = cache_.run_target_attention(query, *cache, meta, d ** -0.5, **kw)
        lse = cache_._target["lse"].clone()
        cache_.accept_target_queries(torch.tensor([2, 3, 1, 3], device=cuda), is_prefill=False)
        assert cache_.retrieval_status()["retrieval_count"] == 1
        got.append((out, lse, cache_.sel_chunks.clone(), cache_.sel_count.clone()))
    close_bf16(got[1][0].float().cpu().numpy(), got[0][0].float().cpu().numpy(), max_rel=2.0 ** -7)
    np.testing.assert_allclose(got[1][1].cpu().numpy(), got[0][1].cpu().numpy(), atol=2e-5)
    assert torch.equal(got[1][3], got[0][3])
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_runtime_selects_the_same_chunks(dsb, cuda):
    """The retrieval driven by the LSE of the shared-prefix call selects the
    chunks that the plain call's LSE selects: chunks of one request whose scores
    lie far apart (its keys there point along the query, more or less)."""
    g = torch.Generator(device=cuda).manual_seed(8)
    hq, hk, d, page, n, prefix = 16, 2, 128, 16, 3, 304
    seq_lens, cols = [340, 420, 460], 30
    table = torch.arange(n * cols, device=cuda, dtype=torch.int32).view(n, cols)
    table[1:, : prefix // page] = table[0, : prefix // page].clone()
    query = torch.randn((1, 1, d), generator=g, device=cuda)
    keys, value = (torch.randn((n * cols, page, hk, d), generator=g, device=cuda) for _ in range(2))
    # each 32 tokens have their own share of the query, half a nat apart and in no order
    step = torch.randperm(n * cols // 2, generator=g, device=cuda).repeat_interleave(2) / 2
    keys = 0.01 * keys + (step[:, None, None, None] % 8) * query / query.square().sum() * d ** 0.5
    cache = [keys.to(_BF), value.to(_BF)]
    query = query.expand(n, hq, d).to(_BF).contiguous()
    meta = SimpleNamespace(actual_seq_lengths_q=[1, 2, 3], seq_lens_list=seq_lens, block_tables=table,
                           num_prefills=0)
    got = []
    for kw in ({}, dict(shared_prefix=([prefix], [n]))):
        state = dsb.runtime.DiffSpecDraftCache(
            dsb.runtime.DiffSpecSettings(32, 160, 1, 4, 3, 0.7, False), max_num_reqs=n,
            max_model_len=512, num_kv_heads=hk, head_dim=d, target_num_layers=2, dtype=_BF,
            device=cuda, cos_sin_cache=torch.zeros((160, d), device=cuda).to(_BF))
        state.begin_target_forward(["a", "b", "c"])
        state.run_target_attention(query, *cache, meta, d ** -0.5, **kw)
        state.accept_target_queries(torch.tensor([1, 1, 1], device=cuda), is_prefill=False)
        got.append([sorted(row[:k]) for row, k in zip(state.sel_chunks.tolist(), state.sel_count.tolist())])
    assert got[0] == got[1] and all(len(row) > 1 for row in got[0][:n])
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("query_ends", [[1, 1, 2, 3], [0, 0, 2, 2], [3, 3, 3, 3], [0, 0, 0, 0]])
def test_runtime_groups_without_query_rows(dsb, cuda, query_ends):
    """Requests without query rows this step, each a group of its own (more
    groups than rows): the plain call's outputs and LSE."""
    g = torch.Generator(device=cuda).manual_seed(sum(query_ends))
    hq, hk, d, page = 8, 2, 128, 16
    cache = [torch.randn((40, page, hk, d), generator=g, device=cuda).to(_BF) for _ in range(2)]
    query = torch.randn((query_ends[-1], hq, d), generator=g, device=cuda).to(_BF)
    meta = SimpleNamespace(actual_seq_lengths_q=query_ends, seq_lens_list=[30, 40, 50, 60],
                           block_tables=torch.arange(40, device=cuda, dtype=torch.int32).view(4, 10),
                           num_prefills=0)
    got = []
    for kw in ({}, dict(shared_prefix=([10, 0, 5, 7], [1, 2, 3, 4])), dict(shared_prefix=([0, 9], [3, 4]))):
        state = dsb.runtime.DiffSpecDraftCache(
            dsb.runtime.DiffSpecSettings(16, 128, 1, 4, 3, 0.7, False), max_num_reqs=4,
            max_model_len=512, num_kv_heads=hk, head_dim=d, target_num_layers=2, dtype=_BF,
            device=cuda, cos_sin_cache=torch.zeros((128, d), device=cuda).to(_BF))
        state.begin_target_forward(["a", "b", "c", "d"])
        got.append((state.run_target_attention(query, *cache, meta, d ** -0.5, **kw),
                    state._target["lse"].clone()))
    for out, lse in got[1:]:
        assert out.shape == got[0][0].shape
        close_bf16(out.float().cpu().numpy(), got[0][0].float().cpu().numpy(), max_rel=2.0 ** -7)
        np.testing.assert_allclose(lse.cpu().numpy(), got[0][1].cpu().numpy(), atol=2e-5)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_draft_layer_with_head_norms(dsb, cuda):
    """Eagle3DraftLayer(qk_norm=True): the pieces of its step against the layer
    computed from the projection by hand, the raw cache's keys normed and not
    rotated, the rebuilt working cache the one that the steps wrote; a shard of
    one rank gives the same layer."""
    dl = dsb.draft_layer
    hidden, qkv_in, hq, hk, d, n, slots_n, max_len, budget = 256, 512, 8, 2, 128, 5, 7, 600, 256
    layer = dl.Eagle3DraftLayer(cuda, hidden=hidden, qkv_in=qkv_in, num_heads=hq, num_kv_heads=hk,
                                head_dim=d, intermediate=512, seed=3, qk_norm=True)
    g = torch.Generator(device=cuda).manual_seed(1)
    layer.q_norm.copy_(1 + 0.3 * torch.randn(d, generator=g, device=cuda))
    layer.k_norm.copy_(1 + 0.3 * torch.randn(d, generator=g, device=cuda))
    x_in = torch.randn((n, qkv_in), generator=g, device=cuda).to(_BF)
    residual = torch.randn((n, hidden), generator=g, device=cuda).to(_BF)
    slots = torch.randperm(slots_n, generator=g, device=cuda)[:n].int()
    at = torch.randint(0, max_len, (n,), generator=g, device=cuda)
    local = torch.randint(2, budget - 4, (n,), generator=g, device=cuda).int()
    cs = _table(budget, d, cuda).to(_BF)
    raw = [torch.zeros((slots_n, max_len, hk, d), dtype=_BF, device=cuda) for _ in range(2)]
    work = [torch.randn((slots_n, hk, budget, d), generator=g, device=cuda).to(_BF) for _ in range(2)]
    before = [w.clone() for w in work]
    step = dict(slots=slots, abs_positions=at, local_positions=local - 2, position_offset=2,
                raw_key=raw[0], raw_value=raw[1], cos_sin=cs)
    out = layer.step(x_in, residual, working_key=work[0], working_value=work[1], **step)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    # by hand, from the layer's own projection
    h = dl.rms_norm(x_in, layer.in_norm, layer.eps)
    qkv = dl.draft_linear(h, layer.p_qkv, packed=True)
    heads = qkv.view(n, hq + 2 * hk, d)
    cos = cs[local.long()]
    qy, qr = _plain_heads(heads[:, :hq], layer.q_norm, cos, layer.eps)
    ky, kr = _plain_heads(heads[:, hq: hq + hk], layer.k_norm, cos, layer.eps)
    s, p = slots.long(), local.long()
    close_bf16(raw[0][s, at].float().cpu().numpy(), ky.cpu().numpy(), max_rel=2.0 ** -8)
    assert torch.equal(raw[1][s, at], heads[:, hq + hk:])
    close_bf16(work[0][s, :, p].float().cpu().numpy(), kr.cpu().numpy(), max_rel=2.0 ** -8)
    assert torch.equal(work[1][s, :, p], heads[:, hq + hk:])
    attn = dsb.attention.draft_decode_attention(
        qr.to(_BF), kr.to(_BF), heads[:, hq + hk:].contiguous(), *[w.clone() for w in before], slots,
        local, d ** -0.5)
    x = dl.draft_linear(attn.view(n, hq * d), layer.p_o, "residual", residual, packed=True)
    act = dl.draft_linear(dl.rms_norm(x, layer.post_norm, layer.eps), layer.p_gate_up, "swiglu",
                          packed=True)
    ref = dl.draft_linear(act, layer.p_down, "residual", x, packed=True)
    close_bf16(out.float().cpu().numpy(), ref.float().cpu().numpy())
    # one tensor-parallel rank is the layer
    shard = dl.Eagle3DraftLayerTP(layer, 0, 1)
    raw2, work2 = [torch.zeros_like(c) for c in raw], [w.clone() for w in before]
    got = shard.step(x_in, residual, working_key=work2[0], working_value=work2[1],
                     **{**step, "raw_key": raw2[0], "raw_value": raw2[1]})
    assert torch.equal(got, out) and torch.equal(raw2[0], raw[0]) and torch.equal(work2[0], work[0])
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
