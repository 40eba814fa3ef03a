"""Attention of requests that share a prefix, with the softmax LSE
(kernels.shared_prefix_attention_lse), against a plain fp64 form that gives
every row its own full sequence.

Tolerances, from the arithmetic (u = 2^-24): a logit sums 128 products in
fp32, off by at most dS = 128 u scale max(sum |q k|); the weights carry 16
bits (two 16-bit terms, 2^-17 relative) and sum over L tokens in fp32; the
exponential is good to 2^-22.  So an output is off by at most
(2 dS + 2^-17 + 2^-22 + (L / 32 + 256) u) max|v| before its rounding (half a
step), where partial sums of 32 or more lanes and splits bound the chain of
additions, and the LSE by dS + 2^-22 + (L / 32 + 256) u + 2 u |lse|."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

_T = {"bf16": torch.bfloat16, "f16": torch.float16}
_D = 128


def _case(cuda, groups, hq, hk, page, dtype, seed, scale_q=2.0):
    """groups: [(prefix, [request lengths], span), ...].  Shared whole pages,
    the started one copied for each request; rows in group order."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    tables, seq, trow, starts, prefix = [], [], [], [0], []
    used, reqs = 0, 0
    cols = max(max(1, -(-max(p, max(lens)) // page)) for p, lens, _ in groups)
    copies = []
    for p, lens, span in groups:
        shared = list(range(used, used + p // page))
        used += p // page
        first = None
        for n in lens:
            n_pages = -(-max(n, p) // page)
            own = list(range(used, used + n_pages - len(shared)))
            used += len(own)
            tables.append(shared + own + [-1] * (cols - n_pages))
            if p % page:
                if first is None:
                    first = own[0]
                copies.append((first, own[0], p % page))
            for j in range(span):
                seq.append(max(0, n - (span - 1 - j)))
                trow.append(reqs)
            reqs += 1
        starts.append(len(seq))
        prefix.append(p)
    total = used + 3
    perm = torch.randperm(total, generator=g, device=cuda)
    table = torch.tensor(tables, device=cuda)
    table = torch.where(table >= 0, perm[table.clamp(min=0)], table).int()
    key, value = (torch.randn((total, page, hk, _D), generator=g, device=cuda).to(_T[dtype])
                  for _ in range(2))
    for s, t, n in copies:
        for c in (key, value):
            c[perm[t], :n] = c[perm[s], :n].clone()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    query = (torch.randn((len(seq), hq, _D), generator=g, device=cuda) * scale_q).to(_T[dtype])
    return dict(query=query, key=key, value=value, table=table, seq=ints(seq), trow=ints(trow),
                starts=ints(starts), prefix=ints(prefix), max_prefix=max(prefix),
                max_suffix=max(max(0, s - p) for s, p in zip(
                    seq, [prefix[i] for i in range(len(groups)) for _ in range(starts[i + 1] - starts[i])])))


def _run(dsb, c, **kw):
    kw = {**dict(max_prefix_len=c["max_prefix"], max_suffix_len=c["max_suffix"],
                 group_starts=c["starts"], table_rows=c["trow"], scale=_D ** -0.5), **kw}
    return dsb.kernels.shared_prefix_attention_lse(c["query"], c["key"], c["value"], c["table"],
                                                   c["seq"], c["prefix"], **kw)


def _check(c, out, lse, seq=None, scale=_D ** -0.5):
    seq = c["seq"].tolist() if seq is None else seq
    hk, page = c["key"].shape[2], c["key"].shape[1]
    rows, hq, _ = c["query"].shape
    u = 2.0 ** -24
    step = torch.finfo(c["query"].dtype).eps / 2
    tiny = torch.finfo(c["query"].dtype).smallest_normal * step
    for r in range(rows):
        if seq[r] <= 0:
            assert (out[r] == 0).all() and torch.isneginf(lse[r]).all(), r
            continue
        entry = c["table"][c["trow"][r].long(), : -(-seq[r] // page)].long()
        k = c["key"][entry].reshape(-1, hk, _D)[: seq[r]].double()
        v = c["value"][entry].reshape(-1, hk, _D)[: seq[r]].double()
        q = c["query"][r].double().view(hk, hq // hk, _D)
        s = torch.einsum("kgd,tkd->kgt", q, k) * scale
        ref_lse = torch.logsumexp(s, -1).reshape(hq)
        ref = torch.einsum("kgt,tkd->kgd", torch.softmax(s, -1), v).reshape(hq, _D)
        ds = 128 * u * scale * float(torch.einsum("kgd,tkd->kgt", q.abs(), k.abs()).max())
        chain = (seq[r] / 32 + 256) * u
        e = (2 * ds + 2.0 ** -17 + 2.0 ** -22 + chain) * float(v.abs().max())
        off = (out[r].double() - ref).abs()
        tol = step * (ref.abs() + e) + e + tiny
        assert bool((off <= tol).all()), (r, float((off / tol).max()))
        tol = ds + 2.0 ** -22 + chain + 2 * u * ref_lse.abs()
        off = (lse[r].double() - ref_lse).abs()
        assert bool((off <= tol).all()), (r, float((off / tol).max()))


CASES = {
    "one row": ([(40, [41], 1)], 8, 1, 16, "bf16"),
    "two short": ([(500, [503, 537], 1)], 8, 1, 16, "bf16"),
    "no prefix": ([(0, [33, 1, 200], 1)], 32, 4, 16, "bf16"),
    "prefix alone": ([(256, [256, 256, 256], 1)], 32, 4, 16, "f16"),
    "prefix of one token": ([(1, [1, 2, 70], 1)], 4, 2, 16, "bf16"),
    "sixteen samples": ([(1000, [1001 + 13 * i for i in range(16)], 1)], 32, 4, 16, "bf16"),
    "verify spans": ([(777, [790, 800, 1200], 5)], 32, 4, 16, "f16"),
    "verify spans over two tiles": ([(650, [660 + i for i in range(5)], 5)], 64, 8, 32, "bf16"),
    "many rows": ([(384, [400 + i for i in range(70)], 1)], 64, 8, 16, "bf16"),
    "three groups": ([(130, [140, 131], 1), (0, [50], 1), (513, [600, 514, 700, 513], 1)],
                     8, 2, 16, "f16"),
    "groups of many rows": ([(300, [310 + i for i in range(20)], 3), (260, [270] * 11, 2)],
                            32, 4, 16, "bf16"),
    "rows shorter than the prefix": ([(300, [300, 120, 0, 310, 1], 1)], 16, 2, 16, "bf16"),
    "empty rows": ([(64, [0, 0], 1), (40, [0, 60], 1)], 8, 1, 16, "bf16"),
    "one head each": ([(200, [210, 260], 1)], 8, 8, 16, "f16"),
    "sixteen heads a group": ([(200, [210, 260, 201], 2)], 32, 2, 16, "bf16"),
    "heads off the powers of two": ([(333, [340, 400, 334], 1)], 12, 2, 16, "bf16"),
    "five heads a group": ([(150, [160, 151], 3)], 15, 3, 8, "f16"),
    "pages of 8": ([(203, [210, 280], 1)], 8, 1, 8, "bf16"),
    "pages of 24": ([(500, [510, 600, 501], 1)], 8, 2, 24, "f16"),
    "pages of 128": ([(1000, [1010, 1300], 1)], 8, 2, 128, "bf16"),
    "pages of 256": ([(700, [710, 1300], 1)], 8, 2, 256, "f16"),
    "runs of one table row longer than a tile": ([(90, [400], 40), (0, [300], 33)], 32, 4, 16, "f16"),
    "prefix off the boxes": ([(129, [140, 300], 2), (15, [20, 400], 1)], 8, 1, 128, "bf16"),
    "pages of 5": ([(203, [210, 280], 1)], 8, 1, 5, "bf16"),
    "pages of one": ([(97, [100, 98], 1)], 8, 2, 1, "f16"),
    "long": ([(20000, [20100, 22000, 20001], 1)], 32, 4, 16, "bf16"),
    "long, one row's tail": ([(131, [9000, 132], 1)], 8, 1, 16, "bf16"),
}


@pytest.mark.parametrize("name", list(CASES))
def test_matches_fp64(dsb, cuda, name):
    groups, hq, hk, page, dtype = CASES[name]
    c = _case(cuda, groups, hq, hk, page, dtype, seed=len(name))
    out, lse = _run(dsb, c)
    torch.cuda.synchronize()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    _check(c, out, lse)
    # the bounds are bounds: larger ones give the same answer to rounding
    out2, lse2 = _run(dsb, c, max_prefix_len=4 * c["max_prefix"] + 999,
                      max_suffix_len=3 * c["max_suffix"] + 700)
    _check(c, out2, lse2)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    # run again: the same bits
    again, lse3 = _run(dsb, c)
    assert torch.equal(out, again) and torch.equal(lse, lse3)


def test_defaults_and_outputs(dsb, cuda):
    """One group without group_starts, rows on their own table rows, outputs
    and 64-bit indices of the caller's."""
    c = _case(cuda, [(100, [120, 101, 133], 1)], 8, 2, 16, "bf16", 3)
    out, lse = torch.empty_like(c["query"]), torch.empty((3, 8), device=cuda)
    got = dsb.kernels.shared_prefix_attention_lse(
        c["query"], c["key"], c["value"], c["table"].long(), c["seq"].long(), c["prefix"].long(),
        scale=0.3, max_prefix_len=100, max_suffix_len=33, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    _check(c, out, lse, scale=0.3)
    none = dsb.kernels.shared_prefix_attention_lse(
        c["query"][:0], c["key"], c["value"], c["table"], c["seq"], c["prefix"], scale=0.3,
        max_prefix_len=100, max_suffix_len=33)
    assert none[0].shape == (0, 8, _D)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_what_lies_behind_the_sequences_is_not_read(dsb, cuda):
    """NaN and infinities in the pages behind every length, and in free pages,
    leave the results alone."""
    for page, dtype in ((16, "bf16"), (128, "f16"), (5, "bf16")):
        c = _case(cuda, [(203, [203, 230, 204], 1), (70, [71, 90], 2)], 16, 2, page, dtype, 4)
        seen = torch.zeros(c["key"].shape[:2], dtype=torch.bool, device=cuda)
        for r in range(c["seq"].numel()):
            t = torch.arange(int(c["seq"][r]), device=cuda)
            seen[c["table"][c["trow"][r].long(), t // page].long(), t % page] = True
        for cache, bad in ((c["key"], float("nan")), (c["value"], float("inf"))):
            cache[~seen] = bad
        out, lse = _run(dsb, c)
        _check(c, out, lse)
        c["value"][~seen] = float("nan")
        out, lse = _run(dsb, c)
        _check(c, out, lse)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_sharp_and_flat_softmax(dsb, cuda, dtype):
    """Logits that span hundreds (one token takes all, and the running maximum
    grows late), and logits that are all equal."""
    c = _case(cuda, [(900, [910, 1000, 901], 1)], 32, 4, 16, dtype, 6, scale_q=1.0)
    c["query"].mul_(16)
    # keys grow along the sequence, so the maximum keeps moving
    for r in range(3):
        t = torch.arange(int(c["seq"][r]), device=cuda)
        at = (c["table"][r, t // 16].long(), t % 16)
        grown = c["key"][at].float() * (0.2 + 2.0 * t[:, None, None] / 1000)
        c["key"][at] = grown.to(_T[dtype])
    for s in range(1, 3):  # the copies of the started page stay copies
        a, b = c["table"][0, 56].long(), c["table"][s, 56].long()
        c["key"][b, :4] = c["key"][a, :4]
    out, lse = _run(dsb, c)
    _check(c, out, lse)
    c["query"].zero_()
    out, lse = _run(dsb, c)
    _check(c, out, lse)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_bad_indices_are_flagged(dsb, cuda):
    P = dsb._lib
    c = _case(cuda, [(200, [230, 260, 201], 1)], 8, 2, 16, "bf16", 8)
    take = lambda: P.read_and_clear_error_flag(cuda)  # noqa: E731
    # the two lengths of the call size its launches alone
    out, lse = _run(dsb, c, max_prefix_len=3, max_suffix_len=10)
    _check(c, out, lse)
    assert take() == 0
    # a table row outside the table: nothing for that row, the others right
    c["trow"][1] = 9
    out, lse = _run(dsb, c)
    assert take() == P.DSB_FLAG_SLOT
    c["trow"][1] = 1
    seq = c["seq"].tolist()
    for r in (0, 2):
        one = {**c, "query": c["query"][r:r + 1], "trow": c["trow"][r:r + 1]}
        _check(one, out[r:r + 1], lse[r:r + 1], seq=[seq[r]])
    # pages outside the cache, in the prefix and behind it
    for col in (3, 14):
        bad = {**c, "table": c["table"].clone()}
        bad["table"][0, col] = 10 ** 6 if col == 3 else -5
        _run(dsb, bad)
        assert take() == 4
    # lengths that no table row holds (whose unused entries, -1, are no pages either)
    long = {**c, "seq": c["seq"] + 10 ** 6}
    _run(dsb, long)
    assert take() in (P.DSB_FLAG_POSITION, P.DSB_FLAG_POSITION | 4)
    # a prefix beyond the table is cut to it (the rows' own tokens are then read
    # through the first row, which has no pages for the longest)
    cut = {**c, "prefix": c["prefix"] + 10 ** 6}
    _run(dsb, cut)
    assert take() in (0, 4)
    # groups that leave rows out: those rows have no shared prefix
    part = {**c, "starts": torch.tensor([1, 3], dtype=torch.int32, device=cuda)}
    out, lse = _run(dsb, part)
    assert take() == 0
    _check(c, out, lse)
    # groups that do not ascend within the rows: flagged, and nothing shared
    for starts in ([0, 2, 1, 3], [0, 3, 3, 4], [-1, 3, 3, 3], [2, 0, 3, 3]):
        part = {**c, "starts": torch.tensor(starts, dtype=torch.int32, device=cuda),
                "prefix": c["prefix"].repeat(3)}
        out, lse = _run(dsb, part)
        assert take() == P.DSB_FLAG_SLOT
        _check(c, out, lse)


def test_two_streams_and_two_graphs(dsb, cuda):
    c = _case(cuda, [(1000, [1001 + 13 * i for i in range(16)], 1)], 32, 4, 16, "bf16", 2)
    ref, ref_lse = _run(dsb, c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_run(dsb, c))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(_run(dsb, c))
        graphs.append(g)
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    for out, lse in got:
        assert torch.equal(out, ref) and torch.equal(lse, ref_lse)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_a_cache_past_32_bits(dsb, cuda):
    """Pages whose byte and element offsets pass 2^32 and 2^31."""
    page, hk, hq = 16, 8, 64
    pages = 2 ** 31 // (page * hk * _D) + 600
    key, value = (torch.zeros((pages, page, hk, _D), dtype=torch.bfloat16, device=cuda)
                  for _ in range(2))
    c = _case(cuda, [(500, [530, 600], 1)], hq, hk, page, "bf16", 12)
    n = c["key"].shape[0]
    key[-n:], value[-n:] = c["key"], c["value"]
    c["table"] = torch.where(c["table"] >= 0, c["table"] + (pages - n), c["table"])
    c |= dict(key=key, value=value)
    out, lse = _run(dsb, c)
    torch.cuda.synchronize()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    _check(c, out, lse)


@pytest.mark.parametrize("own", [0, 1, 150])
@pytest.mark.parametrize("prefix", [127, 1000, 9000, 12000, 19000, 38000])
def test_shares_of_a_few_units(dsb, cuda, prefix, own):
    """160 query rows of one kv head on a prefix whose tiles are fewer, as many
    and a few times as many as the CTAs: shares below a tile, of one and of
    several."""
    c = _case(cuda, [(prefix, [prefix + own * (i % 3 > 0) for i in range(20)], 1)], 8, 1, 16, "bf16",
              prefix + own)
    out, lse = _run(dsb, c)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    _check(c, out, lse)
    again, lse2 = _run(dsb, c)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_what_lies_behind_many_rows_is_not_read(dsb, cuda):
    """The same with more query rows than one operand holds (two streams read
    the tile that the prefix ends inside), and with row counts on both sides."""
    for requests, hq, hk, prefix in ((20, 8, 1, 203), (33, 16, 2, 75), (17, 8, 1, 129)):
        c = _case(cuda, [(prefix, [prefix + i % 4 for i in range(requests)], 1)], hq, hk, 16, "bf16",
                  requests)
        seen = torch.zeros(c["key"].shape[:2], dtype=torch.bool, device=cuda)
        for r in range(requests):
            t = torch.arange(int(c["seq"][r]), device=cuda)
            seen[c["table"][c["trow"][r].long(), t // 16].long(), t % 16] = True
        c["key"][~seen] = float("inf")
        c["value"][~seen] = float("nan")
        for _ in range(5):
            out, lse = _run(dsb, c)
            _check(c, out, lse)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("rows", [4, 40])
def test_loads_that_arrive_out_of_order(dsb, cuda, rows):
    """Pages scattered over a cache of several GB, each read for the first time:
    some loads then take microseconds longer than the ones behind them.  The
    cold run gives what the warm one does."""
    page, hk, tokens, n = 32, 8, 45718, 24
    per = -(-(tokens + 100) // page)
    key, value = (torch.empty((n * per, page, hk, _D), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    for cache in (key, value):
        for part in cache.chunk(n):
            part.normal_()
    g = torch.Generator(device=cuda).manual_seed(1)
    order = torch.randperm(n * per, generator=g, device=cuda).int()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    query = torch.randn((rows, 32, _D), generator=g, device=cuda).bfloat16()
    trow, prefix, seq = ints(*[0] * rows), ints(tokens), ints(*[tokens + 10 + i for i in range(rows)])
    for i in range(n):
        call = lambda: dsb.kernels.shared_prefix_attention_lse(  # noqa: E731
            query, key, value, order[i * per:(i + 1) * per].view(1, per), seq, prefix, scale=_D ** -0.5,
            max_prefix_len=tokens, max_suffix_len=100, table_rows=trow)
        cold, cold_lse = call()
        for _ in range(2):
            warm, warm_lse = call()
        assert torch.equal(cold, warm) and torch.equal(cold_lse, warm_lse), i
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_scratch_that_holds_other_numbers(dsb, cuda):
    """The merge walks as many pieces as the scratch says.  The counts of
    segments that no CTA writes (without tokens here; those of a CTA whose wait
    ran out) are zeros after the call, whatever the scratch held."""
    lens, hq, hk, page, groups = [33, 1, 200], 32, 4, 16, 1
    c = _case(cuda, [(0, lens, 1)], hq, hk, page, "bf16", 1)
    rows, P = len(lens), dsb._lib
    floats = P.load().dsb_shared_prefix_scratch_floats(rows, hq, hk, groups, page, 0, 200)
    scratch = torch.full((floats,), 0x7f7f7f7f, dtype=torch.int32, device=cuda)
    out, lse = torch.empty_like(c["query"]), torch.empty((rows, hq), device=cuda)
    P.call("dsb_shared_prefix_attention_lse", P.ptr(c["query"]), rows, hq, hk, _D, P.ptr(c["key"]),
           P.ptr(c["value"]), c["key"].shape[0], page, P.ptr(c["table"]), c["table"].stride(0),
           *c["table"].shape, P.ptr(c["seq"]), P.ptr(c["trow"]), P.ptr(c["prefix"]),
           P.ptr(c["starts"]), groups, 0, 200, _D ** -0.5, P.dtype_code(torch.bfloat16), P.ptr(out),
           P.ptr(lse), P.ptr(scratch), floats, P.ptr(P.error_flag(cuda)), P.stream_ptr(cuda))
    _check(c, out, lse)
    # scratch: 4 words a CTA, 16 a segment, 4 a row, 1 a group, then the counts [segments, kv heads]
    segments = -(-rows * (hq // hk) // 256) + groups + rows
    at = -(-(P.sm_count(cuda) * 4 + segments * 16 + rows * 4 + groups) // 8) * 8
    counts = scratch[at: at + (1 + rows) * hk].view(-1, hk)
    assert counts.tolist() == [[0] * hk, [1] * hk, [1] * hk, [2] * hk]
    assert P.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("requests,page", [(3, 16), (40, 16), (3, 5)])
@pytest.mark.parametrize("shift", [1, 2, 6])
def test_outputs_at_an_offset(dsb, cuda, requests, page, shift):
    """``out`` and ``lse`` that are views into wider buffers, at any element."""
    c = _case(cuda, [(100, [101 + i for i in range(requests)], 1)], 32, 4, page, "bf16", shift)
    rows, hq = c["query"].shape[:2]
    wide = torch.full((rows * hq * _D + 16,), 7.0, dtype=torch.bfloat16, device=cuda)
    wide_lse = torch.full((rows * hq + 16,), 7.0, device=cuda)
    out = wide[shift: shift + rows * hq * _D].view(rows, hq, _D)
    lse = wide_lse[shift: shift + rows * hq].view(rows, hq)
    got = _run(dsb, c, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    _check(c, out, lse)
    plain, plain_lse = _run(dsb, c)
    assert torch.equal(out, plain) and torch.equal(lse, plain_lse)
    for w, n in ((wide, rows * hq * _D), (wide_lse, rows * hq)):
        assert (w[:shift] == 7).all() and (w[shift + n:] == 7).all()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("behind", ["none", "others"])
@pytest.mark.parametrize("page", [16, 128, 5])
def test_a_short_row_in_front(dsb, cuda, behind, page):
    """Rows that see less of the prefix than the ones behind them, in one
    segment and in several, whose table rows have no pages, or pages of
    something else, behind their own lengths."""
    for lens, hq, hk in (([120, 0, 300, 310], 16, 2), ([0, 1, 299, 300], 8, 1),
                         ([7, *[290] * 8, 300, 301] * 8, 16, 1), ([33, 120], 8, 1)):
        c = _case(cuda, [(300, lens, 1)], hq, hk, page, "bf16", page + len(lens))
        c["prefix"].fill_(max(min(300, n) for n in lens))
        other = c["table"].max() if behind == "others" else -1
        for r, n in enumerate(lens):
            c["table"][r, -(-n // page):] = other
        out, lse = _run(dsb, c)
        assert dsb._lib.read_and_clear_error_flag(cuda) == 0
        _check(c, out, lse)
    # a prefix beyond the table is cut to it, and no row's missing pages are read
    c["prefix"].fill_(10 ** 6)
    _run(dsb, c)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("span", [1, 30])
def test_weights_far_below_the_largest(dsb, cuda, dtype, page, span):
    """One token takes nearly all of the weight and has a value of zero; 7000
    others, 15 to 18 nats below it, make the output by themselves.  With one
    product a logit, dS is the rounding of the scale, of the logit times it and
    of the difference from the maximum (4 u of 26 bits); the rest as above, of
    the output itself, as all of its terms are of one sign.  A weight is off by
    2^-32 of the largest at most in fp16, and never by more than 2^-17 of itself
    in bf16."""
    n, requests = 7000, 20
    lens = [n - i for i in range(requests)]
    c = _case(cuda, [(0, lens, span)], 8, 8, page, dtype, 3)  # each request reads its own tokens
    low = torch.tensor([12.375, 10.75, 11.5, 12.0, 12.75, 10.625, 11.0, 12.625], device=cuda)
    c["query"].zero_()
    c["query"][..., 0] = 16
    c["key"].zero_()
    c["key"][..., 0] = -low.to(_T[dtype])
    c["value"].fill_(1.0)
    for r in range(requests):
        first = c["table"][r, 0].long()
        c["key"][first, 0, :, 0] = 0
        c["value"][first, 0] = 0
    scale = _D ** -0.5
    out, lse = _run(dsb, c, max_prefix_len=0, max_suffix_len=0)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    u, step = 2.0 ** -24, torch.finfo(_T[dtype]).eps / 2
    far = torch.exp(-16 * low.to(_T[dtype]).double() * scale)
    for r, seen in enumerate(c["seq"].tolist()):
        w = far * (seen - 1)
        ref = (w / (1 + w))[:, None]
        chain = (seen / 32 + 256) * u
        e = ref * (4 * 26 * u + 2.0 ** -17 + 2.0 ** -22 + chain)
        if dtype == "f16":
            e = e + (seen - 1) * 2.0 ** -32
        tol = step * (ref + e) + e + torch.finfo(_T[dtype]).smallest_normal * step
        off = (out[r].double() - ref).abs()
        assert bool((off <= tol).all()), (r, float((off / tol).max()))
        tol = 4 * 26 * u + 2.0 ** -22 + chain + u
        assert bool(((lse[r].double() - torch.log1p(w)).abs() <= tol).all()), r


@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_nan_among_what_a_row_sees(dsb, cuda, page, dtype):
    """A key that is not a number among a request's own tokens, every key of a
    request, a value: the rows that see it say so, whatever the page size, and
    the others are right."""
    def case():
        return _case(cuda, [(90, [100, 95, 97], 2)], 8, 1, page, dtype, 5)

    def alone(c, rows, out, lse):
        part = {**c, "query": c["query"][rows], "trow": c["trow"][rows]}
        _check(part, out[rows], lse[rows], seq=[c["seq"].tolist()[r] for r in rows])

    c = case()
    at = c["table"][0, 98 // page].long(), 98 % page
    c["key"][at] = float("nan")  # behind all that the others see
    out, lse = _run(dsb, c)
    for r in (0, 1):
        assert torch.isnan(out[r]).all() and torch.isnan(lse[r]).all(), r
    alone(c, [2, 3, 4, 5], out, lse)
    c = case()
    c["value"][at[0], at[1], 0, 3] = float("nan")
    out, lse = _run(dsb, c)
    assert torch.isnan(out[:2, :, 3]).all() and not torch.isnan(out[:2, :, 4:]).any()
    assert torch.isfinite(lse).all()
    alone(c, [2, 3, 4, 5], out, lse)
    c = case()
    c["key"].fill_(float("nan"))
    c["seq"][4] = 0
    out, lse = _run(dsb, c)
    for r in (0, 1, 2, 3, 5):
        assert torch.isnan(out[r]).all() and torch.isnan(lse[r]).all(), r
    assert (out[4] == 0).all() and torch.isneginf(lse[4]).all()
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("prefix", [0, 2 ** 31 - 1])
def test_lengths_up_to_31_bits(dsb, cuda, prefix):
    """A table row that names one page again and again holds 2^31 tokens and
    more; what a row sees is cut a few tiles below that and flagged.  Logits of
    zero and values of one: every sum is a whole number that fp32 holds until
    the merge (a piece has 2^24 tokens a stream at most)."""
    page = 2 ** 16
    key, value = (torch.ones((1, page, 1, _D), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    query = torch.zeros((1, 8, _D), dtype=torch.bfloat16, device=cuda)
    table = torch.zeros((1, 2 ** 15 + 3), dtype=torch.int32, device=cuda)
    out, lse = dsb.kernels.shared_prefix_attention_lse(
        query, key, value, table, ints(2 ** 31 - 1), ints(prefix), scale=_D ** -0.5,
        max_prefix_len=prefix, max_suffix_len=0)
    assert dsb._lib.read_and_clear_error_flag(cuda) == dsb._lib.DSB_FLAG_POSITION
    assert (out == 1).all()
    # 148 pieces joined in fp32, and the logarithm
    np.testing.assert_allclose(lse.cpu().numpy(), np.log(2.0 ** 31 - 1 - 512), rtol=0,
                               atol=(148 + 4 * 22) * 2.0 ** -24)


@pytest.mark.parametrize("rows,groups,hq,hk", [(5000, 3000, 8, 2), (5000, 1, 8, 1), (700, 300, 32, 2),
                                               (65535, 1500, 1, 1)])
def test_many_rows_and_groups(dsb, cuda, rows, groups, hq, hk):
    """More rows, groups and segments than the plan keeps beside it, against the
    attention of every row by itself (the module's bounds on both sides, with
    sum |q k| at most |q| |k|, and two roundings of the output)."""
    g = torch.Generator(device=cuda).manual_seed(rows)
    page, prefix, requests = 16, 35, 12
    cols = 8
    table = torch.arange(requests * cols, device=cuda, dtype=torch.int32).view(requests, cols)
    key, value = (torch.randn((requests * cols, page, hk, _D), generator=g, device=cuda).bfloat16()
                  for _ in range(2))
    table[:, :2] = table[0, :2].clone()
    for c in (key, value):
        c[table[1:, 2].long(), : prefix % page] = c[table[0, 2].long(), : prefix % page]
    seq = torch.randint(0, cols * page + 1, (rows,), generator=g, device=cuda).int()
    trow = torch.sort(torch.randint(0, requests, (rows,), generator=g, device=cuda))[0].int()
    cuts = torch.sort(torch.randint(0, rows + 1, (groups - 1,), generator=g, device=cuda))[0].int()
    starts = torch.cat((torch.zeros_like(seq[:1]), cuts, torch.full_like(seq[:1], rows)))
    lens = torch.randint(0, prefix + 1, (groups,), generator=g, device=cuda).int()
    query = torch.randn((rows, hq, _D), generator=g, device=cuda).bfloat16()
    out, lse = dsb.kernels.shared_prefix_attention_lse(
        query, key, value, table, seq, lens, scale=_D ** -0.5, max_prefix_len=prefix,
        max_suffix_len=cols * page, group_starts=starts, table_rows=trow)
    ref, ref_lse = dsb.kernels.paged_decode_attention_lse(
        query, key, value, table, seq, scale=_D ** -0.5, max_seq_len=cols * page, table_rows=trow)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0
    u = 2.0 ** -24
    ds = 128 * u * _D ** -0.5 * float(query.double().norm(dim=-1).max() * key.double().norm(dim=-1).max())
    chain = (cols * page / 32 + 256) * u
    e = 2 * (2 * ds + 2.0 ** -17 + 2.0 ** -22 + chain) * float(value.abs().max())
    off = (out.double() - ref.double()).abs()
    step = torch.finfo(torch.bfloat16).eps / 2
    assert bool((off <= 2 * step * (ref.double().abs() + e) + e).all()), float(off.max())
    assert torch.equal(torch.isneginf(lse), torch.isneginf(ref_lse))
    seen = seq > 0
    tol = 2 * (ds + 2.0 ** -22 + chain + 2 * u * ref_lse[seen].double().abs())
    assert bool(((lse - ref_lse)[seen].double().abs() <= tol).all())
