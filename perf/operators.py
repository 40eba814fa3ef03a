"""Workloads of three operator families, each in a plain form and as this package's calls.

* ``qk``     - the norms of queries and keys for each head with the position
               rotation, writing K/V where the next step reads them: the draft
               layer's contiguous rows and raw cache, or the target's pages.
* ``prefix`` - the target's decode attention (with the softmax LSE) for
               requests that share a prefix of their pages.
* ``fork`` / ``compact`` - pages of the target's cache: finished requests
               freed, new ones forked from a parent with its started page
               copied; the live pages moved to the front of the pool.

Layouts are the package's: paged K/V ``[pages, page, Hk, D]``, raw draft K/V
``[slots, max_len, Hk, D]``, int32 block tables.
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

_DEV = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_PACKAGE = "vllm-ascend-hust-diffspec_b200"


# ------------------------------------------------------------------- cases
def _qk(tokens, hq, hk, d, dtype, dest, neox=True, page=16):
    return dict(op="qk", tokens=tokens, hq=hq, hk=hk, d=d, dtype=dtype, dest=dest, neox=neox, page=page)


def _prefix(requests, span, groups, hq, hk, prefix, suffix, page, dtype):
    return dict(op="prefix", requests=requests, span=span, groups=groups, hq=hq, hk=hk,
                prefix=prefix, suffix=suffix, page=page, dtype=dtype)


def _fork(parents, children, length, pages, page, hk, layers, dtype):
    return dict(op="fork", parents=parents, children=children, length=length, pages=pages, page=page,
                hk=hk, layers=layers, dtype=dtype)


def _compact(requests, length, pages, page, hk, layers, dtype):
    return dict(op="compact", requests=requests, length=length, pages=pages, page=page, hk=hk,
                layers=layers, dtype=dtype)


def listed():
    cases = {
        # one request's draft step: latency
        "qk 1 token, draft": _qk(1, 32, 4, 128, "bf16", "raw"),
        # a ragged batch's draft step, other head layout and type
        "qk 77 tokens, draft f16": _qk(77, 64, 8, 128, "f16", "raw"),
        # a verify pass or a short prompt of the target, into its pages
        "qk 2047 tokens, pages": _qk(2047, 64, 8, 128, "bf16", "pages"),
        # prompts of a whole batch
        "qk 65536 tokens, pages": _qk(65536, 32, 4, 128, "bf16", "pages"),
        # two samples of a short prompt: latency
        "prefix 2 x 500": _prefix(2, 1, 1, 8, 1, 500, 37, 16, "bf16"),
        # sixteen samples of one 40k prompt, one token each
        "prefix 16 x 40800": _prefix(16, 1, 1, 32, 4, 40800, 160, 16, "bf16"),
        # the same verifying four drafted tokens and the root, own contexts longer
        "prefix 16 x 5 x 32777 f16": _prefix(16, 5, 1, 32, 4, 32777, 2048, 32, "f16"),
        # two system prompts, many requests, 64 heads
        "prefix 2 groups, 64 x 65536": _prefix(64, 1, 2, 64, 8, 65536, 512, 16, "bf16"),
        # a few samples of one prompt
        "fork 8 of 1 x 1003": _fork(1, 8, 1003, 1024, 16, 4, 1, "bf16"),
        # many samples of long prompts, several layers
        "fork 64 of 4 x 131061": _fork(4, 64, 131061, 40000, 16, 4, 2, "bf16"),
        # a small pool after some requests have left
        "compact 512 pages f16": _compact(8, 470, 512, 16, 2, 1, "f16"),
        # a large one
        "compact 32768 pages": _compact(16, 16000, 32768, 16, 4, 1, "bf16"),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "f16"])
    op = rng.choice(["qk", "qk", "prefix", "prefix", "prefix", "fork", "compact"])
    hq, hk = rng.choice([(8, 1), (32, 4), (64, 8), (32, 8), (16, 16), (12, 2)])
    page = rng.choice([8, 16, 32, 128])
    if op == "qk":
        d = rng.choice([64, 128, 128, 256])
        most = 65536 * 40 * 128 // ((hq + 2 * hk) * d)
        return _qk(_log(rng, 1, most), hq, hk, d, dtype, rng.choice(["raw", "pages"]),
                   rng.random() < 0.7, page)
    if op == "prefix":
        groups = rng.choice([1, 1, 1, 2, 3])
        requests, span = groups * _log(rng, 1, 24), rng.choice([1, 1, 4, 5])
        most = max(32, min(65536, 2_000_000_000 // (hq * requests * span * 16)))
        return _prefix(requests, span, groups, hq, hk, _log(rng, 16, most), _log(rng, span, 1500),
                       page, dtype)
    if op == "fork":
        parents, children = rng.randint(1, 4), _log(rng, 4, 64)
        length = _log(rng, 5, 60000)
        need = parents * (length // page + 1) + children
        return _fork(parents, children, length, need + rng.randint(1, 500), page, rng.choice([1, 2, 4]),
                     rng.randint(1, 2), dtype)
    requests, length = _log(rng, 1, 32), _log(rng, 40, 8000)
    need = requests * (length // page + 1)
    return _compact(requests, length, need + _log(rng, 10, 2 * need + 20), page, rng.choice([1, 2, 4]), 1,
                    dtype)


# --------------------------------------------------------------- quantities
def _prefix_lens(c):
    """Prefix tokens of each group, and each request's own tokens behind it."""
    p = [c["prefix"] - 17 * g if c["prefix"] > 17 * g + 1 else c["prefix"] for g in range(c["groups"])]
    s = [c["span"] + (c["suffix"] - c["span"]) * ((7 * r + 3) % 11) // 10 for r in range(c["requests"])]
    return p, s


def _lengths(c):
    """Tokens of each request of a compacted pool: ragged around `length`."""
    return [max(1, c["length"] * (5 + (3 * r) % 7) // 11) for r in range(c["requests"])]


def _parent_lengths(c):
    """Tokens of each parent: the first has `length`, the others a little less."""
    return [max(1, c["length"] - 37 * p) for p in range(c["parents"])]


def work(case):
    c, e = case, 2
    if c["op"] == "qk":
        t, heads = c["tokens"], c["hq"] + 2 * c["hk"]
        row = t * c["d"] * e
        written = heads + (2 * c["hk"] if c["dest"] == "raw" else 0)
        index = t * (4 + (12 if c["dest"] == "raw" else 4))
        return {"bytes": row * (heads + written) + min(t, _positions(c)) * c["d"] * e + index,
                "flops": t * (c["hq"] + c["hk"]) * c["d"] * 7}
    if c["op"] == "prefix":
        p, s = _prefix_lens(c)
        rows, d = c["requests"] * c["span"], 128
        each = c["requests"] // c["groups"]
        seen = sum((p[r // each] + s[r]) * c["span"] for r in range(c["requests"]))
        kv = (sum(p) + sum(s)) * c["hk"] * d * 2 * e
        pages = sum(-(-x // c["page"]) for x in p) + sum(x // c["page"] + 1 for x in s)
        return {"bytes": kv + rows * c["hq"] * (2 * d * e + 4) + 4 * pages + 8 * rows,
                "flops": 4 * seen * c["hq"] * d}
    token = c["hk"] * 128 * e * 2 * c["layers"]
    if c["op"] == "fork":
        n, lens = c["children"], _parent_lengths(c)
        entries = sum(-(-x // c["page"]) for x in lens) / len(lens)
        rest = sum(x % c["page"] for x in lens) / len(lens)
        # tables: the parents' rows read, the children's read (to free) and written
        tables = 4 * entries * (c["parents"] + 2 * n)
        return {"bytes": 2 * n * rest * token + tables + 2 * 4 * c["pages"], "flops": 0}
    held = [-(-x // c["page"]) for x in _lengths(c)]
    live = sum(held)
    moved = live * (c["pages"] - live) // c["pages"]
    return {"bytes": 2 * moved * c["page"] * token + 2 * 4 * c["pages"] + 2 * 4 * live, "flops": 0}


# ------------------------------------------------------------------- inputs
def _positions(c):
    return 40960 if c["tokens"] > 256 else 4096


def _generator(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=_DEV) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def prepare(case, seed):
    c, g = case, _generator(seed)
    return {"qk": _prepare_qk, "prefix": _prepare_prefix, "fork": _prepare_fork,
            "compact": _prepare_compact}[c["op"]](c, g, _DTYPES[c["dtype"]])


def _prepare_qk(c, g, dtype):
    t, hq, hk, d, most = c["tokens"], c["hq"], c["hk"], c["d"], _positions(c)
    width = (hq + 2 * hk) * d
    # heads of a projection differ in size by orders of magnitude before the norm
    size = torch.exp(torch.randn((1, hq + 2 * hk, 1), generator=g, device=_DEV))
    qkv = (torch.randn((t, hq + 2 * hk, d), generator=g, device=_DEV) * size).to(dtype).view(t, width)
    weight = [1 + 0.2 * torch.randn(d, generator=g, device=_DEV) for _ in range(2)]
    angle = torch.arange(most, device=_DEV, dtype=torch.float64)[:, None] * (
        1e6 ** (-torch.arange(0, d, 2, device=_DEV, dtype=torch.float64) / d))[None]
    s = dict(c=c, qkv=qkv, query=qkv[:, : hq * d], kv=qkv[:, hq * d:], q_weight=weight[0].to(dtype),
             k_weight=weight[1].to(dtype), eps=1e-6,
             cos_sin=torch.cat((angle.cos(), angle.sin()), 1).to(dtype),
             query_out=torch.empty((t, hq * d), dtype=dtype, device=_DEV))
    if c["dest"] == "raw":
        # draft step: each token is a request with a slot of its own
        slots = torch.randperm(t + 3, generator=g, device=_DEV)[:t]
        length = max(3, min(most, 65536 // (t + 3)))
        s |= dict(slots=slots.int(), abs_positions=torch.randint(0, length, (t,), generator=g, device=_DEV),
                  positions=torch.randint(0, most, (t,), generator=g, device=_DEV).int(),
                  raw_key=torch.zeros((t + 3, length, hk, d), dtype=dtype, device=_DEV),
                  key_out=torch.empty((t, hk, d), dtype=dtype, device=_DEV),
                  value_out=torch.empty((t, hk, d), dtype=dtype, device=_DEV))
        s["raw_value"] = torch.zeros_like(s["raw_key"])
        return s
    # prompts: runs of consecutive positions, several requests' one after another
    request = max(1, min(most, 5 * t // 12 + 1))
    at = torch.arange(t, device=_DEV)
    rows, page = -(-t // request), c["page"]
    cols = -(-request // page)
    pages = rows * cols + 5
    s |= dict(positions=(at % request).int(), table_rows=(at // request).int(),
              block_table=torch.randperm(pages, generator=g, device=_DEV)[: rows * cols].int().view(rows, cols),
              key_cache=torch.zeros((pages, page, hk, d), dtype=dtype, device=_DEV))
    s["value_cache"] = torch.zeros_like(s["key_cache"])
    return s


def _prepare_prefix(c, g, dtype):
    p, own_tokens = _prefix_lens(c)
    n, span, groups, page, hk = c["requests"], c["span"], c["groups"], c["page"], c["hk"]
    each = n // groups
    seq = [p[r // each] + own_tokens[r] for r in range(n)]
    cols = max(-(-x // page) for x in seq)
    shared = [x // page for x in p]  # whole pages; the started one is each request's own copy
    pages = sum(shared) + sum(-(-x // page) - shared[r // each] for r, x in enumerate(seq)) + 7
    ids = torch.randperm(pages, generator=g, device=_DEV).int()
    table = torch.full((n, cols), -1, dtype=torch.int32, device=_DEV)
    used = 0
    for k in range(groups):
        table[k * each:(k + 1) * each, : shared[k]] = ids[used: used + shared[k]]
        used += shared[k]
    for r in range(n):
        k = -(-seq[r] // page) - shared[r // each]
        table[r, shared[r // each]: shared[r // each] + k] = ids[used: used + k]
        used += k
    key = _normal(g, (pages, page, hk, 128), dtype)
    value = _normal(g, (pages, page, hk, 128), dtype)
    for k in range(groups):  # the copies hold what was copied
        if p[k] % page:
            last = table[k * each:(k + 1) * each, shared[k]].long()
            for cache in (key, value):
                cache[last, : p[k] % page] = cache[last[0], : p[k] % page][None]
    visible = [x - (span - 1 - j) for x in seq for j in range(span)]
    rows = [r for r in range(n) for _ in range(span)]
    return dict(c=c, query=_normal(g, (n * span, c["hq"], 128), dtype, 2.0), key_cache=key, value_cache=value,
                block_table=table, seq_lens=_ints(visible), prefix_lens=_ints(p), table_rows=_ints(rows),
                group_starts=_ints([k * each * span for k in range(groups + 1)]), scale=128 ** -0.5,
                max_prefix_len=max(p), max_suffix_len=max(own_tokens),
                out=torch.empty((n * span, c["hq"], 128), dtype=dtype, device=_DEV),
                lse=torch.empty((n * span, c["hq"]), dtype=torch.float32, device=_DEV))


def _pool(c, g, dtype):
    shape = (c["pages"], c["page"], c["hk"], 128)
    return [_normal(g, shape, dtype) for _ in range(2 * c["layers"])]


def _prepare_fork(c, g, dtype):
    parents, n, page, lens = c["parents"], c["children"], c["page"], _parent_lengths(c)
    count = [-(-x // page) for x in lens]
    ids = torch.randperm(c["pages"], generator=g, device=_DEV).int()
    table = torch.full((parents + n, max(count) + 2), -1, dtype=torch.int32, device=_DEV)
    used = 0
    for p, k in enumerate(count):
        table[p, :k] = ids[used: used + k]
        used += k
    # the children of an earlier step, which leave as the new ones come
    of = torch.randint(0, parents, (n,), generator=g, device=_DEV)
    started = _ints([x % page > 0 for x in lens])[of]
    table[parents:] = table[of]
    rows = torch.arange(parents, parents + n, device=_DEV)
    last = (_ints(count)[of] - 1).long()
    table[rows, last] = torch.where(started > 0, ids[used: used + n], table[rows, last])
    refs = torch.zeros(c["pages"], dtype=torch.int32, device=_DEV)
    refs.index_add_(0, table[table >= 0].long(), torch.ones_like(table[table >= 0]))
    new = torch.randint(0, parents, (n,), generator=g, device=_DEV)
    return dict(c=c, ref_counts=refs, block_tables=table,
                held=torch.cat((_ints(count), _ints(count)[of])), parents=new.int(),
                children=(parents + torch.randperm(n, generator=g, device=_DEV)).int(),
                lens=_ints(lens)[new], none=torch.zeros(n, dtype=torch.int32, device=_DEV),
                caches=_pool(c, g, dtype))


def _prepare_compact(c, g, dtype):
    count = [-(-x // c["page"]) for x in _lengths(c)]
    ids = torch.randperm(c["pages"], generator=g, device=_DEV).int()
    table = torch.full((len(count), max(count) + 1), -1, dtype=torch.int32, device=_DEV)
    used = 0
    for r, k in enumerate(count):
        table[r, :k] = ids[used: used + k]
        used += k
    refs = torch.zeros(c["pages"], dtype=torch.int32, device=_DEV)
    refs[ids[:used].long()] = 1
    return dict(c=c, ref_counts=refs.clone(), block_tables=table.clone(), held=_ints(count),
                refs_before=refs, tables_before=table, caches=_pool(c, g, dtype))


# --------------------------------------------------------------------- runs
def run(state):
    s, c = state, state["c"]
    if own:
        return _run_own(s, c)
    return {"qk": _plain_qk, "prefix": _plain_prefix, "fork": _plain_fork,
            "compact": _plain_compact}[c["op"]](s, c)


def _run_own(s, c):
    package = importlib.import_module(_PACKAGE)
    if c["op"] == "qk" and c["dest"] == "raw":
        package.draft_layer.qk_norm_rope(
            s["query"], s["kv"], s["positions"], s["cos_sin"], c["hk"], s["q_weight"], s["k_weight"],
            s["eps"], query_out=s["query_out"], key_out=s["key_out"], value_out=s["value_out"],
            is_neox_style=c["neox"], raw=(s["raw_key"], s["raw_value"], s["slots"], s["abs_positions"]))
        return [s[k] for k in ("query_out", "key_out", "value_out", "raw_key", "raw_value")]
    if c["op"] == "qk":
        package.kernels.qk_norm_rope_write_paged(
            s["query"], s["kv"], s["positions"], s["cos_sin"], s["key_cache"], s["value_cache"],
            s["block_table"], s["q_weight"], s["k_weight"], s["eps"], table_rows=s["table_rows"],
            query_out=s["query_out"], is_neox_style=c["neox"])
        return [s[k] for k in ("query_out", "key_cache", "value_cache")]
    if c["op"] == "prefix":
        package.kernels.shared_prefix_attention_lse(
            s["query"], s["key_cache"], s["value_cache"], s["block_table"], s["seq_lens"], s["prefix_lens"],
            scale=s["scale"], max_prefix_len=s["max_prefix_len"], max_suffix_len=s["max_suffix_len"],
            group_starts=s["group_starts"], table_rows=s["table_rows"], out=s["out"], lse=s["lse"])
        return [s["out"], s["lse"]]
    pool = (s["ref_counts"], s["block_tables"], s["held"])
    if c["op"] == "fork":
        package.pages.resize_requests(*pool, s["children"], s["none"], block_size=c["page"])
        package.pages.fork_requests(*pool, s["parents"], s["children"], s["lens"], s["caches"])
        return [*pool, *s["caches"]]
    # the pool as it was, so that each pass has the same pages to move
    s["ref_counts"].copy_(s["refs_before"])
    s["block_tables"].copy_(s["tables_before"])
    package.pages.compact_pages(*pool, s["caches"])
    return [*pool, *s["caches"]]


# -------------------------------------------------------------- plain forms
def _norm(x, weight, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight


def _rotate(x, cos, sin, neox):
    if neox:
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)


def _plain_qk(s, c):
    t, hq, hk, d = c["tokens"], c["hq"], c["hk"], c["d"]
    query = _norm(s["query"].float().reshape(t, hq, d), s["q_weight"].float(), s["eps"])
    key = _norm(s["kv"][:, : hk * d].float().reshape(t, hk, d), s["k_weight"].float(), s["eps"])
    value = s["kv"][:, hk * d:].reshape(t, hk, d)
    cos, sin = s["cos_sin"][s["positions"].long()].float()[:, None].chunk(2, -1)
    rotated = _rotate(key, cos, sin, c["neox"])
    s["query_out"].copy_(_rotate(query, cos, sin, c["neox"]).view(t, hq * d))
    if c["dest"] == "raw":
        s["key_out"].copy_(rotated)
        s["value_out"].copy_(value)
        at = (s["slots"].long(), s["abs_positions"])
        s["raw_key"][at] = key.to(s["raw_key"].dtype)
        s["raw_value"][at] = value
        return [s[k] for k in ("query_out", "key_out", "value_out", "raw_key", "raw_value")]
    pos = s["positions"].long()
    at = (s["block_table"][s["table_rows"].long(), pos // c["page"]].long(), pos % c["page"])
    s["key_cache"][at] = rotated.to(s["key_cache"].dtype)
    s["value_cache"][at] = value
    return [s[k] for k in ("query_out", "key_cache", "value_cache")]


def _paged(cache, table, start, count, page):
    """``[rows, count, Hk, D]`` of tokens start.. of each table row, in 32 bits."""
    at = start[:, None] + torch.arange(count, device=cache.device)
    entry = torch.gather(table.long(), 1, (at // page).clamp(max=table.shape[1] - 1)).clamp(min=0)
    return cache[entry, at % page].float()


def _plain_prefix(s, c):
    groups, page, hk, d = c["groups"], c["page"], c["hk"], 128
    rows, hq = s["query"].shape[:2]
    each, g = rows // groups, hq // hk
    q = s["query"].float().reshape(groups, each, hk, g, d) * s["scale"]
    group = torch.arange(rows, device=q.device) // each
    start = s["prefix_lens"][group].long()
    seq = s["seq_lens"].long()
    # the prefix: every query of a group against one copy of its keys
    first = s["block_table"][s["table_rows"][::each].long()]
    p = s["max_prefix_len"]
    kp, vp = (_paged(x, first, torch.zeros_like(first[:, 0]).long(), p, page).transpose(1, 2)
              for x in (s["key_cache"], s["value_cache"]))
    sp = q.permute(0, 2, 1, 3, 4).reshape(groups, hk, each * g, d) @ kp.transpose(-1, -2)
    at = torch.arange(p, device=q.device)
    hidden = at[None] >= torch.minimum(start, seq)[:, None]
    sp = sp.reshape(groups, hk, each, g, p).masked_fill_(
        hidden.reshape(groups, 1, each, 1, p), float("-inf"))
    # each row's own tokens behind it
    n = s["max_suffix_len"]
    own_table = s["block_table"][s["table_rows"].long()]
    ks, vs = (_paged(x, own_table, start, n, page).transpose(1, 2) for x in (s["key_cache"], s["value_cache"]))
    ss = q.reshape(rows, hk, g, d) @ ks.transpose(-1, -2)
    hidden = start[:, None] + torch.arange(n, device=q.device) >= seq[:, None]
    ss.masked_fill_(hidden[:, None, None], float("-inf"))
    # one softmax over both
    mp = sp.amax(-1).transpose(1, 2).reshape(rows, hk, g)
    top = torch.maximum(mp, ss.amax(-1)).clamp(min=-3e38)
    sp = sp.sub_(top.reshape(groups, each, hk, g).transpose(1, 2)[..., None]).exp_()
    ss = ss.sub_(top[..., None]).exp_()
    total = sp.sum(-1).transpose(1, 2).reshape(rows, hk, g) + ss.sum(-1)
    out = (sp.reshape(groups, hk, each * g, p) @ vp).reshape(groups, hk, each, g, d).transpose(1, 2)
    out = out.reshape(rows, hk, g, d) + ss @ vs
    out = torch.where(total[..., None] > 0, out / total[..., None], torch.zeros_like(out))
    s["out"].copy_(out.reshape(rows, hq, d))
    s["lse"].copy_((top + total.log()).reshape(rows, hq))
    return [s["out"], s["lse"]]


def _plain_fork(s, c):
    refs, table, held = s["ref_counts"], s["block_tables"], s["held"]
    page, cols = c["page"], torch.arange(table.shape[1], device=table.device)
    # the old children's pages go back
    kids = s["children"].long()
    old = table[kids]
    refs.index_add_(0, old.clamp(min=0).flatten().long(), -(old >= 0).int().flatten())
    # the new ones share whole pages and copy the started one
    up, lens = s["parents"].long(), s["lens"]
    full, rest = lens // page, lens % page
    started = rest > 0
    shared = torch.where(cols < full[:, None], table[up], -1)
    refs.index_add_(0, shared.clamp(min=0).flatten().long(), (shared >= 0).int().flatten())
    rank = torch.cumsum(started, 0)
    fresh = torch.searchsorted(torch.cumsum(refs == 0, 0), rank).clamp(max=refs.shape[0] - 1)
    source = torch.gather(table[up], 1, full[:, None].long()).flatten()[started].long()
    table[kids] = torch.where((cols == full[:, None]) & started[:, None], fresh[:, None].int(), shared)
    held[kids] = full + started.int()
    fresh = fresh[started]
    refs[fresh] = 1
    copied = torch.arange(page, device=table.device) < rest[started][:, None]
    for cache in s["caches"]:
        cache[fresh] = torch.where(copied[:, :, None, None], cache[source], cache[fresh])
    return [refs, table, held, *s["caches"]]


def _plain_compact(s, c):
    s["ref_counts"].copy_(s["refs_before"])
    s["block_tables"].copy_(s["tables_before"])
    refs, table = s["ref_counts"], s["block_tables"]
    live = refs > 0
    front = torch.arange(refs.shape[0], device=refs.device) < live.sum()
    source, target = torch.nonzero(live & ~front).flatten(), torch.nonzero(~live & front).flatten()
    name = torch.arange(refs.shape[0], device=refs.device, dtype=torch.int32)
    name[source] = target.int()
    table.copy_(torch.where(table >= 0, name[table.clamp(min=0).long()], table))
    refs[target] = refs[source]
    refs[source] = 0
    for cache in s["caches"]:
        cache[target] = cache[source]
    return [refs, table, s["held"], *s["caches"]]


# ------------------------------------------------------------- 64-bit values
def exact(case, seed):
    c = case
    if c["op"] not in ("qk", "prefix"):
        return None  # whole numbers, and copies
    s = prepare(case, seed)
    return _exact_qk(s, c) if c["op"] == "qk" else _exact_prefix(s, c)


def _exact_qk(s, c):
    t, hq, hk, d, half = c["tokens"], c["hq"], c["hk"], c["d"], c["d"] // 2
    table = s["cos_sin"].double()[s["positions"].long()]
    # element i of a head is paired with partner[i]; its sine has a sign
    i = torch.arange(d, device=table.device)
    if c["neox"]:
        partner, freq, first = (i + half) % d, i % half, i < half
    else:
        partner, freq, first = i ^ 1, i // 2, i % 2 == 0
    cos, sin = table[:, None, freq], table[:, None, half + freq] * torch.where(first, -1.0, 1.0).double()

    def normed(x, weight):
        x = x.double()
        return x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + s["eps"]) * weight.double()

    heads = s["qkv"].view(t, hq + 2 * hk, d)
    q = normed(heads[:, :hq], s["q_weight"])
    q = (q * cos + q[..., partner] * sin).reshape(t, hq * d)
    k = normed(heads[:, hq: hq + hk], s["k_weight"])
    rotated, v = k * cos + k[..., partner] * sin, heads[:, hq + hk:].double()
    if c["dest"] == "raw":
        raw_key, raw_value = s["raw_key"].double(), s["raw_value"].double()
        flat = s["slots"].long() * raw_key.shape[1] + s["abs_positions"]
        raw_key.view(-1, hk, d)[flat] = k
        raw_value.view(-1, hk, d)[flat] = v
        return [q, rotated, v, raw_key, raw_value]
    pos = s["positions"].long()
    flat = s["block_table"][s["table_rows"].long(), pos // c["page"]].long() * c["page"] + pos % c["page"]
    key, value = s["key_cache"].double(), s["value_cache"].double()
    key.view(-1, hk, d)[flat] = rotated
    value.view(-1, hk, d)[flat] = v
    return [q, key, value]


def _exact_prefix(s, c):
    hq, hk, d, page = c["hq"], c["hk"], 128, c["page"]
    g, rows = hq // hk, s["query"].shape[0]
    out = torch.zeros((rows, hq, d), dtype=torch.float64, device=_DEV)
    lse = torch.full((rows, hq), float("-inf"), dtype=torch.float64, device=_DEV)
    seq, of = s["seq_lens"].tolist(), s["table_rows"].tolist()
    for r in range(rows):  # every row by itself, over its own table
        if seq[r] <= 0:
            continue
        entry = s["block_table"][of[r], : -(-seq[r] // page)].long()
        k = s["key_cache"][entry].reshape(-1, hk, d)[: seq[r]].double()
        v = s["value_cache"][entry].reshape(-1, hk, d)[: seq[r]].double()
        logits = torch.einsum("kgd,tkd->kgt", s["query"][r].double().view(hk, g, d), k) * s["scale"]
        lse[r] = torch.logsumexp(logits, -1).flatten()
        out[r] = torch.einsum("kgt,tkd->kgd", torch.softmax(logits, -1), v).reshape(hq, d)
    return [out, lse]
