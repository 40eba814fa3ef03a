"""Refusals of the page calls, the shared-prefix attention and the query/key
norms: before any launch, on the host, and CPU tensors (there is no CPU
path)."""

from __future__ import annotations

import ctypes

import pytest
import torch


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_pages_validation(dsb):
    pg = dsb.pages
    refs, tables, held = _i(8), _i(4, 3), _i(4)
    caches = [torch.zeros((8, 16, 2, 8), dtype=torch.bfloat16)] * 2
    resize = lambda *a, bs=16, **k: pg.resize_requests(*a, block_size=bs, **k)  # noqa: E731
    with pytest.raises(ValueError, match="block_size"):
        resize(refs, tables, held, _i(1), _i(1), bs=0)
    with pytest.raises(ValueError, match="one entry per block-table row"):
        resize(refs, tables, _i(3), _i(1), _i(1))
    with pytest.raises(ValueError, match="int32"):
        resize(refs.long(), tables, held, _i(1), _i(1))
    with pytest.raises(ValueError, match=r"\[rows, cols\]"):
        resize(refs, tables[0], held, _i(1), _i(1))
    with pytest.raises(ValueError, match="contiguous"):
        resize(refs, _i(3, 4).t(), held, _i(1), _i(1))
    with pytest.raises(ValueError, match="one entry per request"):
        resize(refs, tables, held, _i(2), _i(1))
    with pytest.raises(ValueError, match="whole numbers"):
        resize(refs, tables, held, _i(1), torch.zeros(1))
    with pytest.raises(ValueError, match="need CUDA tensors"):
        resize(refs, tables, held, _i(1), _i(1))
    fork = lambda *a, **k: pg.fork_requests(refs, tables, held, *a, **k)  # noqa: E731
    with pytest.raises(ValueError, match="at least one tensor"):
        fork(_i(1), _i(1), _i(1), [])
    with pytest.raises(ValueError, match="one shape and dtype"):
        fork(_i(1), _i(1), _i(1), [caches[0], caches[0].half()])
    with pytest.raises(ValueError, match="one page per reference count"):
        fork(_i(1), _i(1), _i(1), [caches[0][:5]])
    with pytest.raises(ValueError, match="one entry per request"):
        fork(_i(1), _i(2), _i(1), caches)
    with pytest.raises(ValueError, match="need CUDA tensors"):
        fork(_i(1), _i(1), _i(1), caches)
    with pytest.raises(ValueError, match=r"\[pages, block_size"):
        pg.compact_pages(refs, tables, held, [torch.zeros(8, 16)])
    with pytest.raises(ValueError, match="need CUDA tensors"):
        pg.compact_pages(refs, tables, held, caches)
    with pytest.raises(ValueError, match=r"\[pages, block_size"):
        pg.copy_pages([], _i(1), _i(1))
    with pytest.raises(ValueError, match="one entry per request"):
        pg.copy_pages(caches, _i(2), _i(1))
    with pytest.raises(ValueError, match="need CUDA tensors"):
        pg.copy_pages(caches, _i(1), _i(1))


def test_shared_prefix_validation(dsb):
    f = dsb.kernels.shared_prefix_attention_lse
    q = torch.zeros((3, 8, 128), dtype=torch.bfloat16)
    kc = torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16)
    bt, seq, pre = _i(3, 4), _i(3), _i(1)
    kw = dict(scale=0.1, max_prefix_len=16, max_suffix_len=16)
    with pytest.raises(ValueError, match="query must be"):
        f(q[0], kc, kc, bt, seq, pre, **kw)
    with pytest.raises(ValueError, match="query must be"):
        f(q, kc, kc[:2], bt, seq, pre, **kw)
    with pytest.raises(ValueError, match="head dims"):
        f(q[:, :7], kc, kc, bt, seq, pre, **kw)
    with pytest.raises(ValueError, match="share a dtype"):
        f(q.half(), kc, kc, bt, seq, pre, **kw)
    with pytest.raises(ValueError, match="seq_lens"):
        f(q, kc, kc, bt, seq[:2], pre, **kw)
    with pytest.raises(ValueError, match="one row per query row"):
        f(q, kc, kc, bt[:2], seq, pre, **kw)
    with pytest.raises(ValueError, match="table_rows"):
        f(q, kc, kc, bt, seq, pre, table_rows=_i(2), **kw)
    with pytest.raises(ValueError, match="without group_starts"):
        f(q, kc, kc, bt, seq, _i(2), **kw)
    with pytest.raises(ValueError, match="one entry more"):
        f(q, kc, kc, bt, seq, _i(2), group_starts=_i(2), **kw)
    with pytest.raises(ValueError, match="must be >= 0"):
        f(q, kc, kc, bt, seq, pre, **{**kw, "max_suffix_len": -1})
    with pytest.raises(ValueError, match="need CUDA tensors"):
        f(q, kc, kc, bt, seq, pre, **kw)


def test_qk_norm_rope_validation(dsb):
    f = dsb.draft_layer.qk_norm_rope
    bf = torch.bfloat16
    q, kv = torch.zeros((3, 512), dtype=bf), torch.zeros((3, 512), dtype=bf)
    pos, cs, w = _i(3), torch.zeros((8, 128)), torch.ones(128, dtype=bf)
    with pytest.raises(ValueError, match="query must be"):
        f(q, kv[:, :500], pos, cs, 2, w, w, 1e-6)
    with pytest.raises(ValueError, match=r"query must be \[T"):
        f(q[:, :500], kv, pos, cs, 2, w, w, 1e-6)
    with pytest.raises(ValueError, match=r"must be \[head_dim\]"):
        f(q, kv, pos, cs, 2, w, w[:64], 1e-6)
    with pytest.raises(ValueError, match="share a dtype"):
        f(q, kv, pos, cs, 2, w, w.half(), 1e-6)
    with pytest.raises(ValueError, match="rotary_dim"):
        f(q, kv, pos, cs, 2, w, w, 1e-6, rotary_dim=130)
    with pytest.raises(ValueError, match="cos_sin"):
        f(q, kv, pos, cs[:, :64], 2, w, w, 1e-6)
    with pytest.raises(ValueError, match="positions"):
        f(q, kv, pos.long(), cs, 2, w, w, 1e-6)
    with pytest.raises(ValueError, match="query_out"):
        f(q, kv, pos, cs, 2, w, w, 1e-6, query_out=q[:2])
    raw = torch.zeros((4, 6, 2, 128), dtype=bf)
    with pytest.raises(ValueError, match="raw key/value"):
        f(q, kv, pos, cs, 2, w, w, 1e-6, raw=(raw, raw[:2], _i(3), pos.long()))
    with pytest.raises(ValueError, match="slots must be int32"):
        f(q, kv, pos, cs, 2, w, w, 1e-6, raw=(raw, raw, _i(3), pos))
    with pytest.raises(ValueError, match="need CUDA tensors"):
        f(q, kv, pos, cs, 2, w, w, 1e-6)
    g = dsb.kernels.qk_norm_rope_write_paged
    cache = torch.zeros((4, 16, 2, 128), dtype=bf)
    with pytest.raises(ValueError, match="matching"):
        g(q, kv, pos, cs, cache, cache[:2], _i(3, 2), w, w, 1e-6)
    with pytest.raises(ValueError, match="head_dim and dtype"):
        g(q, kv, pos, cs, cache.half(), cache.half(), _i(3, 2), w, w, 1e-6)
    with pytest.raises(ValueError, match="row for every token"):
        g(q, kv, pos, cs, cache, cache, _i(2, 2), w, w, 1e-6)
    with pytest.raises(ValueError, match="map every token"):
        g(q, kv, pos, cs, cache, cache, _i(3, 2), w, w, 1e-6, table_rows=_i(2))
    with pytest.raises(ValueError, match="need CUDA tensors"):
        g(q, kv, pos, cs, cache, cache, _i(3, 2), w, w, 1e-6)


def test_abi_rejects_before_any_launch(dsb):
    L, P = dsb._lib.load(), dsb._lib
    fake = ctypes.c_void_p(256)
    odd = ctypes.c_void_p(8)

    def attention(**k):
        a = dict(q=fake, rows=4, hq=32, hk=4, d=128, kc=fake, vc=fake, blocks=100, bs=16, bt=fake,
                 stride=8, trows=4, cols=8, seq=fake, tr=None, pre=fake, gs=None, groups=1, mp=64,
                 ms=64, scale=0.1, dt=0, out=fake, lse=fake, scratch=fake, floats=1 << 40, err=None,
                 st=None)
        return L.dsb_shared_prefix_attention_lse(*{**a, **k}.values())

    for k in (dict(rows=-1), dict(hq=30), dict(hk=0), dict(dt=2), dict(blocks=0), dict(bs=0),
              dict(stride=4), dict(mp=-1), dict(ms=-1), dict(groups=0), dict(groups=2),
              dict(groups=9, gs=fake), dict(scale=0.0), dict(pre=None), dict(lse=None),
              dict(floats=0)):
        assert attention(**k) == P.DSB_ERR_INVALID, k
    for k in (dict(d=64), dict(hq=68), dict(q=odd), dict(rows=70000)):
        assert attention(**k) == P.DSB_ERR_UNSUPPORTED, k
    assert attention(rows=0) == P.DSB_OK
    assert L.dsb_shared_prefix_scratch_floats(0, 8, 1, 1, 16, 10, 10) == 0

    def resize(**k):
        a = dict(refs=fake, pages=8, bt=fake, rows=4, stride=3, cols=3, held=fake, r=fake, n=fake,
                 k=2, bs=16, status=None, err=None, st=None)
        return L.dsb_resize_requests(*{**a, **k}.values())

    for k in (dict(pages=0), dict(rows=0), dict(stride=2), dict(k=-1), dict(k=5000), dict(bs=0),
              dict(refs=None), dict(r=None)):
        assert resize(**k) == P.DSB_ERR_INVALID, k

    ptrs = (ctypes.c_void_p * 2)(256, 512)
    null = (ctypes.c_void_p * 2)(256, None)

    def fork(**k):
        a = dict(refs=fake, pages=8, bt=fake, rows=4, stride=3, cols=3, held=fake, up=fake, c=fake,
                 n=fake, k=2, bs=16, caches=ptrs, m=2, token=64, status=None, scratch=fake, ints=12,
                 err=None, st=None)
        return L.dsb_fork_requests(*{**a, **k}.values())

    for k in (dict(k=4097), dict(caches=None), dict(caches=null), dict(ints=11), dict(up=None),
              dict(held=None)):
        assert fork(**k) == P.DSB_ERR_INVALID, k
    assert fork(token=24) == P.DSB_ERR_UNSUPPORTED

    def compact(**k):
        a = dict(refs=fake, pages=8, bt=fake, rows=4, stride=3, cols=3, held=fake, bs=16,
                 caches=ptrs, m=2, token=64, status=fake, scratch=fake, ints=1 << 20, err=None,
                 st=None)
        return L.dsb_compact_pages(*{**a, **k}.values())

    for k in (dict(pages=0), dict(status=None), dict(scratch=None), dict(ints=3), dict(caches=null)):
        assert compact(**k) == P.DSB_ERR_INVALID, k
    assert L.dsb_copy_pages(ptrs, 2, 8, 64, None, fake, 1, None, None) == P.DSB_ERR_INVALID
    assert L.dsb_copy_pages(ptrs, 2, 8, 60, fake, fake, 1, None, None) == P.DSB_ERR_UNSUPPORTED
    assert L.dsb_copy_pages(ptrs, 2, 8, 64, None, None, 0, None, None) == P.DSB_OK

    def norm(**k):
        a = dict(q=fake, qs=512, qo=fake, qos=512, hq=4, k=fake, ks=512, ko=fake, v=fake, vs=512,
                 vo=fake, hk=2, d=128, rot=128, neox=1, qw=fake, kw=fake, eps=1e-6, pos=fake, off=0,
                 tokens=3, cs=fake, css=128, rows=8, csdt=2, dt=0, rk=None, rv=None, slots=None,
                 abs=None, ns=0, ml=0, err=None, st=None)
        return L.dsb_qk_norm_rope(*{**a, **k}.values())

    for k in (dict(tokens=-1), dict(dt=2), dict(csdt=7), dict(hq=0), dict(rot=3), dict(rot=130),
              dict(css=64), dict(eps=-1.0), dict(qs=256), dict(ks=100), dict(qos=640, qo=fake),
              dict(ko=None), dict(qw=None), dict(rk=fake), dict(rk=fake, rv=fake, slots=fake),
              dict(rk=fake, rv=fake, slots=fake, abs=fake)):
        assert norm(**k) == P.DSB_ERR_INVALID, k
    assert norm(tokens=0) == P.DSB_OK


def test_prefix_groups(dsb):
    f = dsb.runtime.prefix_groups
    assert f([300], [4], [3, 6, 9, 12], [340, 301, 333, 420]) == ([300], [0, 12], 120)
    assert f([300, 0, 130], [2, 2, 4], [1, 2, 3, 4], [340, 301, 200, 131]) == (
        [300, 0, 130], [0, 2, 2, 4], 70)
    assert f([7], [0], [], []) == ([7], [0, 0], 0)
    for lens, ends in (([], []), ([1], [3, 4]), ([-1], [4]), ([1, 1], [3, 2]), ([1], [5]), ([1], [3])):
        with pytest.raises(ValueError, match="shared_prefix"):
            f(lens, ends, [1, 2, 3, 4], [5, 5, 5, 5])


def test_scratch_is_sized_on_the_tensors_device(dsb, monkeypatch):
    """Two devices of other SM counts: each call's scratch has the size that
    the device of its tensors needs, whatever is current and whatever came
    before."""
    kernels, lib = dsb.kernels, dsb._lib
    current, sizes, asked = [0], {0: 1000, 1: 3000}, []

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.before

    class Library:
        @staticmethod
        def dsb_shared_prefix_scratch_floats(*sizes_):
            return sizes[current[0]]

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(lib, "load", Library)
    monkeypatch.setattr(lib, "error_flag_ptr", lambda device: 0)
    monkeypatch.setattr(lib, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(lib, "call_on", lambda device, name, *a: asked.append((device.index, a[-3])))
    q = torch.zeros((3, 8, 128), dtype=torch.bfloat16)
    kc = torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16)
    kernels._shared_prefix_floats.cache_clear()
    for index in (1, 0, 1, 0):
        monkeypatch.setattr(lib, "device_of", lambda *_: torch.device("cuda", index))
        kernels.shared_prefix_attention_lse(q, kc, kc, _i(3, 4), _i(3), _i(1), scale=0.1,
                                            max_prefix_len=16, max_suffix_len=16)
    kernels._shared_prefix_floats.cache_clear()
    assert asked == [(1, 3000), (0, 1000), (1, 3000), (0, 1000)]


def test_a_tokens_bytes_go_by_the_shape(dsb):
    """One token a page, or one page: contiguous tensors whose strides of those
    dimensions are anything."""
    for cache in (torch.zeros((1, 8, 2, 8)).transpose(0, 1), torch.zeros((8, 2, 8)).unsqueeze(1),
                  torch.zeros((8, 1, 2, 8)), torch.zeros((5, 1, 2, 8)).transpose(0, 1)):
        assert cache.is_contiguous()
        addresses, block_size, token_bytes = dsb.pages._caches([cache], cache.shape[0])
        assert list(addresses) == [cache.data_ptr()]
        assert (block_size, token_bytes) == (cache.shape[1], 2 * 8 * 4)


def test_the_stride_of_a_single_row_is_not_read(dsb):
    """One token, one table row, one row of cosines: transposed columns are
    contiguous rows, too."""
    column = lambda n, **k: torch.zeros((n, 1), **k).t()  # noqa: E731
    bf = dict(dtype=torch.bfloat16)
    q, kv, out, cs, w = column(512, **bf), column(512, **bf), column(512, **bf), column(128), torch.ones(128, **bf)
    got = dsb.kernels._qk_norm_inputs(q, kv, _i(1), cs, 2, w, w, None, out)
    assert got[5] == (q.data_ptr(), 512, out.data_ptr(), 512, 4, kv.data_ptr(), 512)
    assert got[7][:3] == (cs.data_ptr(), 128, 1)
    got = dsb.kernels._qk_norm_inputs(q, kv, _i(1), cs, 2, w, w, None, None)
    assert got[5] == (q.data_ptr(), 512, q.data_ptr(), 512, 4, kv.data_ptr(), 512)
    table = column(7, dtype=torch.int32)
    assert dsb.pages._pool(_i(8), table, _i(1))[3:6] == (1, 7, 7)
    assert dsb.kernels._row_stride(table) == 7 and dsb.kernels._row_stride(_i(3, 9)[:, :7]) == 9
    assert dsb.pages._pool(_i(8), _i(1, 3).t(), _i(3))[3:6] == (3, 1, 1)


def test_rows_and_lengths_beyond_32_bits_stay_out_of_range(dsb):
    """2^32 + 5 tokens are not five, and row 2^32 is not row zero."""
    got = dsb.pages._row(torch.tensor([5, 2 ** 32 + 5, 2 ** 31, -2 ** 40, -1]), 5, "lens")
    assert got.dtype == torch.int32 and got.tolist() == [5, 2 ** 31 - 1, 2 ** 31 - 1, -1, -1]
    assert dsb.pages._row(torch.tensor([5, 200], dtype=torch.uint8), 2, "rows").tolist() == [5, 200]


def test_scratch_of_the_page_calls(dsb):
    """The sizes that the Python calls work out themselves are the C side's."""
    L = dsb._lib.load()
    for n in (1, 7, 4096):
        assert L.dsb_fork_scratch_ints(n) == 6 * n
        assert L.dsb_compact_scratch_ints(n) == 1 + 3 * n
