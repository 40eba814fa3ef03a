"""Pages of a paged cache on the device (pages.resize_requests, fork_requests,
compact_pages, copy_pages) against the oracle's plain pool: tables, reference
counts, pages held, the status words and the cache contents, all exact."""

from __future__ import annotations

import random

import pytest
import torch

from oracle import diffspec_oracle as O

pytestmark = pytest.mark.gpu


class _Pool:
    """The device state beside the oracle's, with caches whose values say
    where they were written."""

    def __init__(self, dsb, cuda, pages, rows, cols, bs, layers=1, hk=2, d=8, dtype=torch.bfloat16,
                 wide=0):
        self.dsb, self.cuda, self.bs = dsb, cuda, bs
        self.ref = O.PagePool(pages, rows, cols, bs)
        ints = dict(dtype=torch.int32, device=cuda)
        self.refs = torch.zeros(pages, **ints)
        self.tables = torch.full((rows, cols + wide), -1, **ints)[:, :cols]
        self.held = torch.zeros(rows, **ints)
        g = torch.Generator(device=cuda).manual_seed(pages)
        self.caches = [torch.randn((pages, bs, hk, d), generator=g, device=cuda).to(dtype)
                       for _ in range(2 * layers)]
        self.copy = [c.clone() for c in self.caches]

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.cuda)

    @property
    def state(self):
        return self.refs, self.tables, self.held

    def resize(self, rows, lens):
        st = self.dsb.pages.resize_requests(*self.state, self.ints(rows), self.ints(lens),
                                            block_size=self.bs)
        self.ref.resize(rows, lens)
        self.check(st)

    def fork(self, parents, children, lens):
        st = self.dsb.pages.fork_requests(*self.state, self.ints(parents), self.ints(children),
                                          self.ints(lens), self.caches)
        for s, t, n in self.ref.fork(parents, children, lens):
            for c in self.copy:
                c[t, :n] = c[s, :n]
        self.check(st)

    def compact(self):
        st = self.dsb.pages.compact_pages(*self.state, self.caches)
        self.ref.lacking = 0
        moves = self.ref.compact()
        if moves:
            s, t = (torch.tensor(x, device=self.cuda) for x in zip(*moves))
            for c in self.copy:
                c[t] = c[s]
        self.check(st)

    def check(self, status):
        assert status.tolist() == [self.ref.lacking, len(self.ref.free())]
        assert self.refs.tolist() == self.ref.refs
        assert self.held.tolist() == self.ref.held
        assert self.tables.tolist() == self.ref.tables
        for a, b in zip(self.caches, self.copy):
            assert torch.equal(a, b)
        want = set()
        for name, bit in (("slot", 1), ("position", 2)):
            if name in self.ref.flags:
                want.add(bit)
        self.ref.flags.clear()
        assert self.dsb._lib.read_and_clear_error_flag(self.cuda) == sum(want)


@pytest.mark.parametrize("pages,rows,cols,bs,layers,dtype", [
    (64, 8, 10, 16, 1, torch.bfloat16),
    (40, 12, 9, 1, 2, torch.float16),      # one token a page
    (3000, 40, 100, 5, 1, torch.float32),  # several passes over the pool, odd pages
    (1, 2, 1, 16, 1, torch.bfloat16),      # a single page
    (9000, 16, 700, 8, 3, torch.bfloat16),
    (20011, 24, 900, 2, 1, torch.bfloat16),
    (70001, 24, 3500, 1, 1, torch.bfloat16),  # several CTAs plan
])
def test_random_histories(dsb, cuda, pages, rows, cols, bs, layers, dtype):
    rng = random.Random(pages)
    p = _Pool(dsb, cuda, pages, rows, cols, bs, layers, dtype=dtype, wide=3)
    longest = cols * bs
    for step in range(60):
        what = rng.random()
        if what < 0.5:
            n = rng.randint(0, rows)
            who = rng.sample(range(rows), n)
            p.resize(who, [rng.choice([0, 1, rng.randint(0, longest), rng.randint(0, bs)])
                           for _ in who])
        elif what < 0.85:
            empty = [r for r in range(rows) if not p.ref.held[r]]
            full = [r for r in range(rows) if p.ref.held[r]] or [0]
            kids = rng.sample(empty, rng.randint(0, len(empty)))
            ups = [rng.choice(full) for _ in kids]
            p.fork(ups, kids, [rng.randint(0, p.ref.held[u] * bs) for u in ups])
        else:
            p.compact()


def test_a_batch_forked_from_one_prompt_and_freed(dsb, cuda):
    p = _Pool(dsb, cuda, 600, 66, 200, 16, layers=2)
    p.resize([0], [2999])
    p.fork([0] * 64, list(range(65, 1, -1)), [2999] * 64)
    assert int(p.refs.max()) == 65
    p.resize(list(range(2, 66)), [3000 + r for r in range(64)])  # each writes on
    p.resize([0], [0])  # the parent leaves, its pages stay
    assert int(p.refs.max()) == 64
    p.resize(list(range(2, 66)), [0] * 64)
    assert int(p.refs.sum()) == 0


def test_exhaustion(dsb, cuda):
    """Rows in order until the first that does not fit; a smaller one behind
    it waits too; what is let go in the call can be given in it."""
    p = _Pool(dsb, cuda, 10, 6, 10, 4)
    p.resize([0, 1, 2, 3], [16, 12, 16, 4])  # 4 + 3 fit; 4 do not, nor does the 1 behind
    assert p.ref.lacking == 2
    p.resize([2, 0], [16, 0])
    assert p.ref.lacking == 0
    p.fork([1] * 4, [3, 4, 5, 0], [9, 8, 9, 9])  # three started pages, three free ones
    assert p.ref.lacking == 0 and not p.ref.free()
    p.resize([3, 4, 5, 0], [0] * 4)
    p.resize([5], [8])
    p.fork([1, 1, 1], [3, 4, 0], [9, 11, 8])  # one page left: the second finds none
    assert p.ref.lacking == 1 and p.ref.held[:5] == [2, 3, 4, 3, 0]


def test_compact_full_empty_and_settled_pools(dsb, cuda):
    p = _Pool(dsb, cuda, 50, 4, 50, 2)
    p.compact()  # nothing live
    p.resize([0, 1], [60, 40])
    p.compact()  # nothing free
    p.resize([0], [0])
    p.compact()  # all live pages move
    p.compact()  # settled
    p.fork([1], [2], [39])
    p.resize([1], [0])
    p.compact()


def test_bad_rows_are_flagged_and_left_alone(dsb, cuda):
    p = _Pool(dsb, cuda, 30, 5, 6, 4)
    p.resize([0, 0, 1, 7, -1, 2], [8, 24, 99, 4, 4, -1])  # twice, too long, outside, negative
    p.fork([0, 0, 0, 9, 0, 0], [1, 1, 0, 2, 8, 3], [5, 5, 5, 1, 1, 9])
    p.fork([4, 3], [3, 4], [0, 0])  # of nothing
    assert p.ref.held == [2, 2, 0, 0, 0]


def test_bad_pages_are_flagged(dsb, cuda):
    """Entries that are no page, and a page let go twice."""
    p = _Pool(dsb, cuda, 8, 4, 4, 4)
    take = lambda: dsb._lib.read_and_clear_error_flag(cuda)  # noqa: E731
    p.resize([0, 1], [16, 8])
    p.tables[0, 1] = 99
    p.tables[0, 2] = p.tables[0, 3]
    st = dsb.pages.resize_requests(*p.state, p.ints([0]), p.ints([0]), block_size=4)
    assert take() == 4 and st.tolist() == [0, 4]
    assert p.refs.tolist()[:4] == [0, 1, 1, 0]
    p.tables[1, 1] = -1
    dsb.pages.fork_requests(*p.state, p.ints([1, 1]), p.ints([2, 3]), p.ints([7, 3]), p.caches)
    assert take() == 4 and p.held.tolist() == [0, 2, 0, 1]
    p.tables[1, 1] = 77
    dsb.pages.compact_pages(*p.state, p.caches)
    assert take() == 4 and int(p.tables[1, 1]) == 77


def test_copy_pages(dsb, cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    for layers, bs, hk, d, n in ((1, 16, 4, 128, 13), (3, 1, 1, 8, 500), (70, 2, 1, 8, 3)):
        pages = 3 * n + 5
        caches = [torch.randn((pages, bs, hk, d), generator=g, device=cuda).bfloat16()
                  for _ in range(2 * layers)]
        want = [c.clone() for c in caches]
        perm = torch.randperm(pages, generator=g, device=cuda)
        src, dst = perm[:n].int(), perm[n:2 * n].int()
        for c in want:
            c[dst.long()[1:]] = c[src.long()[1:]]
        src[0] = -1
        dsb.pages.copy_pages(caches, src, dst)
        assert all(torch.equal(a, b) for a, b in zip(caches, want))
        assert dsb._lib.read_and_clear_error_flag(cuda) == 0
        dst[1] = pages
        dsb.pages.copy_pages(caches, src[:2], dst[:2])
        assert dsb._lib.read_and_clear_error_flag(cuda) == 4
        assert all(torch.equal(a, b) for a, b in zip(caches, want))
        dsb.pages.copy_pages(caches, src[:0], dst[:0])


def test_captured(dsb, cuda):
    """A step of freeing, forking and compacting replayed from a graph does
    what the calls did."""
    a, b = (_Pool(dsb, cuda, 100, 10, 20, 16) for _ in range(2))
    kids, ups = a.ints([3, 4, 5]), a.ints([0, 1, 0])
    none, lens = a.ints([0, 0, 0]), a.ints([37, 64, 40])

    def step(p):
        dsb.pages.resize_requests(*p.state, kids, none, block_size=16)
        dsb.pages.fork_requests(*p.state, ups, kids, lens, p.caches)
        return dsb.pages.compact_pages(*p.state, p.caches)

    for p in (a, b):
        p.resize([0, 1], [100, 64])
        step(p)  # (and loads the kernels)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for _ in range(3):
        step(a)
        graph.replay()
    torch.cuda.synchronize()
    for x, y in zip((*a.state, *a.caches), (*b.state, *b.caches)):
        assert torch.equal(x, y)
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("pages", [1900, 4096, 4097, 30000])
def test_many_rows_in_a_call(dsb, cuda, pages):
    """More rows than a small planner has threads, pools on both sides of what
    it sees in one turn."""
    rows = 700
    p = _Pool(dsb, cuda, pages, rows, 9, 4)
    rng = random.Random(pages)
    who = rng.sample(range(rows), 300)
    p.resize(who, [rng.randint(0, 20) for _ in who])
    kids = [r for r in range(rows) if not p.ref.held[r]][:390]
    ups = [rng.choice(who) for _ in kids]
    p.fork(ups, kids, [rng.randint(0, p.ref.held[u] * 4) for u in ups])
    p.resize(who + kids, [rng.choice([0, 3, 36]) for _ in who + kids])
    p.compact()
    p.resize(kids, [rng.randint(0, 36) for _ in kids])


def test_pools_beyond_a_turn_of_the_planners(dsb, cuda):
    """More pages than the planning CTAs hold in registers."""
    pages, cols = 300001, 40000
    p = _Pool(dsb, cuda, pages, 12, cols, 1, hk=1)
    p.resize([3, 1, 7], [30000, 39999, 12345])
    p.fork([1, 3, 1], [0, 2, 9], [39999, 29999, 77])
    p.resize([5, 6, 8, 10, 11], [40000] * 5)
    p.resize([3, 2, 5], [0, 17, 100])
    p.resize([4], [40000])
    p.compact()
    p.resize([1, 6], [0, 0])
    p.compact()
    p.resize([1, 3, 6], [39000, 5, 40000])


@pytest.mark.parametrize("pages,cols", [(64, 9), (64, 9000), (5000, 9), (40000, 9000)])
def test_a_row_cut_back_into_a_shared_page_is_flagged(dsb, cuda, pages, cols):
    """What the row would write next is in a page of its siblings.  Cut to a
    page's end, into a page of its own, or as the others leave, it is not
    (tables on both sides of what one CTA lets go by itself; one planner and
    several)."""
    def take():
        return dsb._lib.read_and_clear_error_flag(cuda)

    def resize(rows, lens):
        dsb.pages.resize_requests(*p.state, p.ints(rows), p.ints(lens), block_size=4)
        flag = take()
        p.ref.resize(rows, lens)
        p.ref.flags.clear()
        p.check(p.ints([p.ref.lacking, len(p.ref.free())]))
        return flag

    p = _Pool(dsb, cuda, pages, 5, cols, 4)
    p.resize([0], [18])
    p.fork([0, 0], [1, 2], [16, 18])  # four shared pages, and two tokens of its own for row 2
    assert resize([1], [15]) == dsb._lib.DSB_FLAG_POSITION
    assert resize([1], [15]) == dsb._lib.DSB_FLAG_POSITION  # still so
    assert resize([1, 2, 0], [12, 17, 17]) == 0  # whole pages, pages of their own
    assert resize([0, 1, 2], [3, 4, 20]) == dsb._lib.DSB_FLAG_POSITION
    assert resize([0, 1, 2], [0, 0, 7]) == 0  # the others leave in the same call
    p.fork([2], [1], [7])
    assert resize([1], [5]) == 0  # the fork's copy
    assert p.ref.held == [0, 2, 2, 0, 0]


def test_needs_whose_sum_passes_32_bits(dsb, cuda):
    """Rows that ask for more pages together than a 32-bit count holds find
    none, and the ones in front of them are served."""
    cols, pages = 1_100_000_000, 100
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    refs, held = torch.zeros(pages, dtype=torch.int32, device=cuda), ints(0, 0, 0)
    tables = torch.full((3, cols), -1, dtype=torch.int32, device=cuda)
    st = dsb.pages.resize_requests(refs, tables, held, ints(1, 0, 2), ints(60, cols, cols), block_size=1)
    assert st.tolist() == [2, 40] and held.tolist() == [0, 60, 0]
    assert refs.tolist() == [1] * 60 + [0] * 40 and tables[1, :61].tolist() == [*range(60), -1]
    st = dsb.pages.resize_requests(refs, tables, held, ints(0, 2, 1), ints(cols, cols, 3), block_size=1)
    assert st.tolist() == [2, 97] and held.tolist() == [0, 3, 0]  # the surplus goes all the same
    assert int((tables >= 0).sum()) == 3
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


def test_caches_past_32_bits(dsb, cuda):
    """Pages whose offsets pass 2^31 elements and 2^32 bytes: copied, forked
    into and compacted."""
    page, hk, d = 16, 4, 128
    pages = 2 ** 31 // (page * hk * d) + 400
    cache = torch.zeros((pages, page, hk, d), dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    cache[-60:] = torch.randn((60, page, hk, d), generator=g, device=cuda).bfloat16()
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    want = cache[-60:].clone()
    top = pages - 60
    dsb.pages.copy_pages([cache], ints(top, top + 1, 7), ints(top + 40, 3, top + 41))
    want[40], want[41] = want[0], 0
    assert torch.equal(cache[-60:], want) and torch.equal(cache[3], want[1])
    # every page but the last twenty is someone else's
    refs = torch.ones(pages, dtype=torch.int32, device=cuda)
    refs[-20:] = 0
    tables = torch.full((3, 4), -1, dtype=torch.int32, device=cuda)
    held = torch.zeros(3, dtype=torch.int32, device=cuda)
    dsb.pages.resize_requests(refs, tables, held, ints(0), ints(40), block_size=page)
    st = dsb.pages.fork_requests(refs, tables, held, ints(0), ints(1), ints(40), [cache])
    assert tables[:2].tolist() == [[pages - 20, pages - 19, pages - 18, -1],
                                   [pages - 20, pages - 19, pages - 17, -1]]
    want[43, :8] = want[42, :8]
    assert st.tolist() == [0, 16] and torch.equal(cache[-60:], want)
    # the low half becomes free: the live pages move down, those of the rows among them
    refs[: pages - 100] = 0
    st = dsb.pages.compact_pages(refs, tables, held, [cache])
    live = 100 - 16
    assert st.tolist() == [0, pages - live] and tables[1].tolist() == [live - 4, live - 3, live - 1, -1]
    assert torch.equal(cache[live - 44: live], want[:44])
    assert dsb._lib.read_and_clear_error_flag(cuda) == 0


@pytest.mark.parametrize("pages", [3000, 20000])
def test_the_most_rows_that_a_call_takes(dsb, cuda, pages):
    """4096 rows a call, one CTA's pool and a cluster's; one more is refused."""
    rows = 9000
    p = _Pool(dsb, cuda, pages, rows, 5, 4)
    rng = random.Random(pages)
    who = rng.sample(range(rows), 4096)
    p.resize(who, [rng.randint(0, 12) for _ in who])
    kids = [r for r in range(rows) if not p.ref.held[r]][:4096]
    ups = [rng.choice(who) for _ in kids]
    p.fork(ups, kids, [rng.randint(0, p.ref.held[u] * 4) for u in ups])
    p.resize(kids, [rng.choice([0, 3, 20]) for _ in kids])
    p.compact()
    many = p.ints([0] * 4097)
    for call in (lambda: dsb.pages.resize_requests(*p.state, many, many, block_size=4),
                 lambda: dsb.pages.fork_requests(*p.state, many, many, many, p.caches)):
        with pytest.raises(ValueError, match="4096"):
            call()
