"""Per-head RMSNorm of queries and keys with RoPE in one pass
(draft_layer.qk_norm_rope, kernels.qk_norm_rope_write_paged) against the fp64
oracle, with the raw-cache and page writes.

Tolerance: fp32 arithmetic, one rounding.  With u = 2^-24 the sum of D squares
is off by at most D u relative (its root's inverse by half of that), rsqrt by
4 u, the products by 3 u and the rotation by 3 u of |y1| + |y2|; the store adds
half a step of the result."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import diffspec_oracle as O

pytestmark = pytest.mark.gpu

_T = {"bf16": torch.bfloat16, "f16": torch.float16}


def _inputs(cuda, tokens, hq, hk, d, rot, dtype, cs_dtype, rows, seed, neox=True):
    g = torch.Generator(device=cuda).manual_seed(seed)
    size = torch.exp(torch.randn((1, hq + 2 * hk, 1), generator=g, device=cuda))
    qkv = (torch.randn((tokens, hq + 2 * hk, d), generator=g, device=cuda) * size).to(_T[dtype])
    w = [(1 + 0.3 * torch.randn(d, generator=g, device=cuda)).to(_T[dtype]) for _ in range(2)]
    angle = torch.rand((rows, max(rot // 2, 1)), generator=g, device=cuda, dtype=torch.float64) * 6.3
    cs = torch.cat((angle.cos(), angle.sin()), 1)[:, : max(rot, 2)].to(cs_dtype).contiguous()
    pos = torch.randint(0, rows, (tokens,), generator=g, device=cuda).int()
    return qkv, w, cs, pos


def _close(got, ref, other, d, dtype):
    """|got - ref| within the bound of the module's text; `other`: |y1| + |y2|."""
    got = got.double().cpu().numpy()
    step = torch.finfo(_T[dtype]).eps / 2
    e = (d / 2 + 16) * 2.0 ** -24 * other
    tol = step * (np.abs(ref) + e) + e + torch.finfo(_T[dtype]).smallest_normal * step
    assert (np.abs(got - ref) <= tol).all(), float((np.abs(got - ref) / tol).max())


def _expect(qkv, w, cs, pos, hq, hk, rot, neox, eps):
    x = qkv.double().cpu().numpy()
    rows = cs.double().cpu().numpy()[pos.cpu().numpy()]
    q = O.qk_norm_rope(x[:, :hq], w[0].double().cpu().numpy(), eps, rows, rot, neox)
    k = O.qk_norm_rope(x[:, hq: hq + hk], w[1].double().cpu().numpy(), eps, rows, rot, neox)
    return q, k


def _both(y):
    """An upper bound of |y1| + |y2| of each element's pair."""
    return np.abs(y) + np.abs(y).max(-1, keepdims=True)


CASES = [
    # tokens, hq, hk, d, rot, dtype, table dtype, neox
    (1, 32, 4, 128, 128, "bf16", torch.bfloat16, True),
    (16, 32, 4, 128, 128, "bf16", torch.float32, True),
    (37, 64, 8, 128, 128, "f16", torch.float16, True),
    (5, 8, 1, 64, 64, "bf16", torch.float32, True),
    (9, 12, 2, 256, 256, "f16", torch.float32, False),
    (7, 16, 16, 128, 128, "bf16", torch.bfloat16, False),
    (6, 5, 1, 128, 64, "bf16", torch.float32, True),    # part of the head rotated
    (6, 3, 3, 64, 20, "f16", torch.float32, False),
    (4, 4, 2, 96, 96, "bf16", torch.float32, True),     # head sizes off the powers of two
    (4, 2, 1, 30, 30, "f16", torch.float32, True),
    (3, 2, 1, 512, 512, "bf16", torch.float32, True),
    (3, 4, 2, 128, 0, "bf16", torch.float32, True),     # norms alone
    (2, 7, 1, 33, 32, "bf16", torch.float32, False),    # an odd head
    (513, 32, 4, 128, 128, "bf16", torch.bfloat16, True),
]


@pytest.mark.parametrize("tokens,hq,hk,d,rot,dtype,cs_dtype,neox", CASES)
def test_rows_and_raw_caches(dsb, cuda, tokens, hq, hk, d, rot, dtype, cs_dtype, neox):
    rows, slots_n, max_len = 300, tokens + 2, 11
    qkv, w, cs, pos = _inputs(cuda, tokens, hq, hk, d, rot, dtype, cs_dtype, rows, d + tokens)
    flat = qkv.view(tokens, -1)
    slots = torch.randperm(slots_n, device=cuda)[:tokens].int()
    slots[0] = -1  # padding: nothing written
    at = torch.randint(0, max_len, (tokens,), device=cuda)
    raw = [torch.full((slots_n, max_len, hk, d), 7.0, dtype=_T[dtype], device=cuda) for _ in range(2)]
    out = torch.empty((tokens, hq * d), dtype=_T[dtype], device=cuda)
    q, k, v = dsb.draft_layer.qk_norm_rope(
        flat[:, : hq * d], flat[:, hq * d:], pos - 3, cs, hk, w[0], w[1], 1e-6, query_out=out,
        position_offset=3, rotary_dim=rot, is_neox_style=neox, raw=(*raw, slots, at))
    torch.cuda.synchronize()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    (qy, qr), (ky, kr) = _expect(qkv, w, cs, pos, hq, hk, rot, neox, 1e-6)
    assert q is out
    _close(q.view(tokens, hq, d), qr, _both(qy), d, dtype)
    _close(k, kr, _both(ky), d, dtype)
    assert torch.equal(v, qkv[:, hq + hk:])
    s, a = slots[1:].long(), at[1:]
    _close(raw[0][s, a], ky[1:], _both(ky[1:]), d, dtype)
    assert torch.equal(raw[1][s, a], v[1:])
    for cache in raw:  # rows of no token are as they were
        cache[s, a] = 7.0
        assert (cache == 7.0).all()


@pytest.mark.parametrize("tokens,hq,hk,d,rot,dtype,cs_dtype,neox", CASES)
@pytest.mark.parametrize("page", [1, 5, 16])
def test_pages(dsb, cuda, tokens, hq, hk, d, rot, dtype, cs_dtype, neox, page):
    rows = 40 * 5
    qkv, w, cs, _ = _inputs(cuda, tokens, hq, hk, d, rot, dtype, cs_dtype, rows, d + tokens + page)
    flat = qkv.view(tokens, -1)
    per = 40  # tokens of a request
    pos = (torch.arange(tokens, device=cuda) % per).int()
    trow = (torch.arange(tokens, device=cuda) // per).int()
    cols = -(-per // page)
    n = int(trow.max()) + 1
    pages = n * cols + 3
    table = torch.randperm(pages, device=cuda)[: n * cols].int().view(n, cols)
    trow[0] = -1
    caches = [torch.full((pages, page, hk, d), 7.0, dtype=_T[dtype], device=cuda) for _ in range(2)]
    query = flat[:, : hq * d].clone()  # in place
    got = dsb.kernels.qk_norm_rope_write_paged(
        query, flat[:, hq * d:], pos, cs, *caches, table, w[0], w[1], 1e-5, table_rows=trow,
        rotary_dim=rot, is_neox_style=neox)
    torch.cuda.synchronize()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    (qy, qr), (ky, kr) = _expect(qkv, w, cs, pos, hq, hk, rot, neox, 1e-5)
    assert got is query
    _close(query.view(tokens, hq, d), qr, _both(qy), d, dtype)
    p = pos[1:].long()
    at = (table[trow[1:].long(), p // page].long(), p % page)
    _close(caches[0][at], kr[1:], _both(ky[1:]), d, dtype)
    assert torch.equal(caches[1][at], qkv[1:, hq + hk:])
    for cache in caches:
        cache[at] = 7.0
        assert (cache == 7.0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_strides_and_values(dsb, cuda, dtype):
    """Rows of a wider buffer at offsets that are not 16-byte aligned; heads of
    zeros, tiny and huge values (the norm's sum must not overflow); a NaN head
    leaves the others alone."""
    tokens, hq, hk, d = 6, 4, 2, 128
    heads = hq + 2 * hk
    qkv, w, cs, pos = _inputs(cuda, tokens, hq, hk, d, d, dtype, torch.float32, 64, 5)
    qkv[0, 0] = 0
    qkv[1, 1] = 6e4 if dtype == "f16" else 1e15
    qkv[2, 2] = 6e-6 if dtype == "f16" else 1e-30
    qkv[3, 3, 5] = float("nan")
    for shift in (1, 4):
        wide = torch.zeros((tokens, heads * d + 13), dtype=_T[dtype], device=cuda)
        wide[:, shift: shift + heads * d] = qkv.view(tokens, -1)
        flat = wide[:, shift: shift + heads * d]
        out = torch.full((tokens, hq * d + 9), 3.0, dtype=_T[dtype], device=cuda)
        q, k, v = dsb.draft_layer.qk_norm_rope(flat[:, : hq * d], flat[:, hq * d:], pos, cs, hk,
                                               w[0], w[1], 1e-6, query_out=out[:, 2: 2 + hq * d])
        torch.cuda.synchronize()
        (qy, qr), (ky, kr) = _expect(qkv, w, cs, pos, hq, hk, d, True, 1e-6)
        got = q.reshape(tokens, hq, d)
        assert torch.isnan(got[3, 3]).all()
        qr[3, 3] = qy[3, 3] = 0
        got[3, 3] = 0
        _close(got, qr, _both(qy), d, dtype)
        _close(k, kr, _both(ky), d, dtype)
        assert torch.equal(v, qkv[:, hq + hk:])
        assert (out[:, :2] == 3).all() and (out[:, 2 + hq * d:] == 3).all()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_bad_indices_are_flagged_and_skipped(dsb, cuda):
    tokens, hq, hk, d = 5, 4, 2, 128
    qkv, w, cs, _ = _inputs(cuda, tokens, hq, hk, d, d, "bf16", torch.float32, 32, 9)
    flat = qkv.view(tokens, -1)
    take = lambda: dsb._lib.read_and_clear_error_flag(cuda)  # noqa: E731
    ints = lambda *x, t=torch.int32: torch.tensor(x, dtype=t, device=cuda)  # noqa: E731
    caches = lambda n, m: [torch.zeros((n, m, hk, d), dtype=torch.bfloat16, device=cuda)  # noqa: E731
                           for _ in range(2)]
    out = torch.empty_like(flat[:, : hq * d])
    args = (flat[:, : hq * d], flat[:, hq * d:])
    # a position outside the table: normed, not rotated
    pos = ints(0, 32, -1, 3, 4)
    q, k, _ = dsb.draft_layer.qk_norm_rope(*args, pos, cs, hk, *w, 1e-6, query_out=out)
    assert take() == dsb._lib.DSB_FLAG_POSITION
    (qy, _), (ky, _) = _expect(qkv, w, cs, pos.clamp(0, 31), hq, hk, d, True, 1e-6)
    for t in (1, 2):
        _close(q.view(tokens, hq, d)[t], qy[t], _both(qy[t]), d, "bf16")
        _close(k[t], ky[t], _both(ky[t]), d, "bf16")
    # raw cache: slot and position out of range
    good = ints(0, 1, 2, 3, 4)
    for slots, at, flag in ((ints(0, 1, 2, 3, 9), (0, 1, 2, 3, 4), dsb._lib.DSB_FLAG_SLOT),
                            (good, (0, 1, 2, 3, 6), dsb._lib.DSB_FLAG_POSITION),
                            (good, (0, 1, 2, 3, -1), dsb._lib.DSB_FLAG_POSITION)):
        raw = caches(5, 6)
        dsb.draft_layer.qk_norm_rope(*args, good, cs, hk, *w, 1e-6, query_out=out,
                                     raw=(*raw, slots, ints(*at, t=torch.int64)))
        assert take() == flag
        assert sum(int((raw[1][s, p] != 0).any()) for s in range(5) for p in range(6)) == 4
    # pages: table row, column and page out of range
    table = ints(0, 1, 2, 3, 4).view(5, 1)
    for rows, pos, bad, flag in ((ints(0, 1, 2, 3, 5), good, table, dsb._lib.DSB_FLAG_SLOT),
                                 (good, ints(0, 1, 2, 3, 8), table, dsb._lib.DSB_FLAG_POSITION),
                                 (good, good, ints(0, 1, 2, 3, 5).view(5, 1), 4),
                                 (good, good, ints(0, 1, 2, 3, -1).view(5, 1), 4)):
        cache = caches(5, 8)
        dsb.kernels.qk_norm_rope_write_paged(*args, pos, cs, *cache, bad, *w, 1e-6, table_rows=rows,
                                             query_out=out)
        assert take() == flag
        assert sum(int((cache[1][s, p] != 0).any()) for s in range(5) for p in range(8)) == 4


def test_no_tokens(dsb, cuda):
    qkv, w, cs, pos = _inputs(cuda, 0, 4, 2, 64, 64, "bf16", torch.float32, 8, 1)
    flat = qkv.view(0, 8 * 64)
    q, k, v = dsb.draft_layer.qk_norm_rope(flat[:, :256], flat[:, 256:], pos, cs, 2, *w, 1e-6)
    assert q.shape == (0, 256) and k.shape == v.shape == (0, 2, 64)


def test_captured_and_on_another_stream(dsb, cuda):
    """Two graphs of the call and an eager one give the same rows."""
    tokens, hq, hk, d = 33, 32, 4, 128
    qkv, w, cs, pos = _inputs(cuda, tokens, hq, hk, d, d, "bf16", torch.bfloat16, 64, 3)
    flat = qkv.view(tokens, -1)
    outs = [torch.zeros((tokens, hq * d), dtype=torch.bfloat16, device=cuda) for _ in range(4)]
    call = lambda o: dsb.draft_layer.qk_norm_rope(  # noqa: E731
        flat[:, : hq * d], flat[:, hq * d:], pos, cs, hk, *w, 1e-6, query_out=o)
    call(outs[0])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        call(outs[1])
    torch.cuda.synchronize()
    graphs = []
    for o in outs[2:]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kv = call(o)[1:]
        graphs.append((g, kv))
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 1), (3, 3), (4, 2), (5, 1), (8, 1), (8, 8), (16, 2), (17, 9)])
def test_heads_on_both_sides_of_a_warp(dsb, cuda, hq, hk, d):
    """Head counts around what a warp takes (tokens side by side, the last ones
    of a run missing), raw and paged; a bad slot in a run harms no neighbour."""
    for tokens, neox in ((1, True), (13, False), (38, True)):
        test_rows_and_raw_caches(dsb, cuda, tokens, hq, hk, d, d, "bf16", torch.float32, neox)
        test_pages(dsb, cuda, tokens, hq, hk, d, d, "f16", torch.bfloat16, neox, 16)
    tokens, n = 11, 6
    qkv, w, cs, pos = _inputs(cuda, tokens, hq, hk, d, d, "bf16", torch.float32, 50, d + hq)
    flat = qkv.view(tokens, -1)
    slots = torch.arange(tokens, device=cuda).int()
    at = torch.zeros(tokens, dtype=torch.int64, device=cuda)
    raw = [torch.full((tokens, 2, hk, d), 7.0, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    slots[n], pos[n + 2] = tokens, 50  # a slot and a position outside
    out = torch.empty((tokens, hq * d), dtype=torch.bfloat16, device=cuda)
    q, k, v = dsb.draft_layer.qk_norm_rope(
        flat[:, : hq * d], flat[:, hq * d:], pos, cs, hk, w[0], w[1], 1e-6, query_out=out,
        raw=(*raw, slots, at))
    assert dsb._lib.read_and_clear_error_flag(cuda) == dsb._lib.DSB_FLAG_SLOT | dsb._lib.DSB_FLAG_POSITION
    pos[n + 2] = 0
    (qy, qr), (ky, kr) = _expect(qkv, w, cs, pos, hq, hk, d, True, 1e-6)
    qr[n + 2], kr[n + 2] = qy[n + 2], ky[n + 2]  # normed, not rotated
    _close(q.view(tokens, hq, d), qr, _both(qy), d, "bf16")
    _close(k, kr, _both(ky), d, "bf16")
    keep = [i for i in range(tokens) if i != n]
    _close(raw[0][keep, 0], ky[keep], _both(ky[keep]), d, "bf16")
    assert torch.equal(raw[1][keep, 0], v[keep])
    assert (raw[0][n] == 7.0).all() and (raw[0][:, 1] == 7.0).all()


@pytest.mark.parametrize("d", [128, 96])
def test_offsets_past_32_bits(dsb, cuda, d):
    """Rows of the projection, of the raw caches and of the pages whose offsets
    pass 2^31 elements and 2^32 bytes (both kernels)."""
    hq, hk, n, page, rows = 32, 4, 37, 16, 64
    width = (hq + 2 * hk) * d
    tokens = 2 ** 31 // width + 100
    small, w, cs, pos_n = _inputs(cuda, n, hq, hk, d, d, "bf16", torch.float32, rows, d)
    (qy, qr), (ky, kr) = _expect(small, w, cs, pos_n, hq, hk, d, True, 1e-6)
    qkv = torch.zeros((tokens, width), dtype=torch.bfloat16, device=cuda)
    qkv[-n:] = small.view(n, width)
    pos = torch.zeros(tokens, dtype=torch.int32, device=cuda)
    pos[-n:] = pos_n
    slots = torch.full((tokens,), -1, dtype=torch.int32, device=cuda)  # (the others: padding)
    at = torch.zeros(tokens, dtype=torch.int64, device=cuda)
    max_len = 2 ** 31 // (2 * hk * d) + 50
    raw = [torch.zeros((3, max_len, hk, d), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    slots[-n:], at[-n:] = 2, torch.arange(max_len - n, max_len, device=cuda)
    q, k, v = dsb.draft_layer.qk_norm_rope(
        qkv[:, : hq * d], qkv[:, hq * d:], pos, cs, hk, *w, 1e-6, raw=(*raw, slots, at))  # in place
    _close(q[-n:].reshape(n, hq, d), qr, _both(qy), d, "bf16")
    _close(k[-n:], kr, _both(ky), d, "bf16")
    assert torch.equal(v[-n:], small[:, hq + hk:])
    _close(raw[0][2, -n:], ky, _both(ky), d, "bf16")
    assert torch.equal(raw[1][2, -n:], small[:, hq + hk:])
    del raw, q, k, v, qkv
    # the last pages of a cache
    pages = 2 ** 31 // (page * hk * d) + 400
    caches = [torch.zeros((pages, page, hk, d), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    table = torch.arange(pages - 4, pages, device=cuda).int()[None].expand(1, 4).contiguous()
    pos = torch.randperm(4 * page, device=cuda)[:n].int()
    flat = small.view(n, width)
    out = torch.empty((n, hq * d), dtype=torch.bfloat16, device=cuda)
    dsb.kernels.qk_norm_rope_write_paged(
        flat[:, : hq * d], flat[:, hq * d:], pos, cs, *caches, table, *w, 1e-6,
        table_rows=torch.zeros(n, dtype=torch.int32, device=cuda), query_out=out)
    (qy, qr), (ky, kr) = _expect(small, w, cs, pos, hq, hk, d, True, 1e-6)
    _close(out.view(n, hq, d), qr, _both(qy), d, "bf16")
    place = (pages - 4 + pos.long() // page, pos.long() % page)
    _close(caches[0][place], kr, _both(ky), d, "bf16")
    assert torch.equal(caches[1][place], small[:, hq + hk:])
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
