"""Pages that sequences share against a pool in plain Python: the pages each call takes, the table, the counts and every row of the caches."""
import random

import pytest
import torch

I32 = torch.int32


class Plain:
    """What a pool holds, with a cache as a list of rows per page."""

    def __init__(self, pages, page_tokens, slots, max_pages, rows):
        self.n, self.pt, self.P = pages, page_tokens, max_pages
        self.table, self.lengths = [[-1] * max_pages for _ in range(slots)], [0] * slots
        self.rows = rows                               # [pages][page_tokens] of anything

    def refs(self):
        r = [0] * self.n
        for row in self.table:
            for p in row:
                if p >= 0:
                    r[p] += 1
        return r

    def free_pages(self):
        return [p for p, r in enumerate(self.refs()) if r == 0]

    def extend(self, slots, tokens):
        if len(set(slots)) < len(slots) or any(not 0 <= s < len(self.table) for s in slots) or any(not 0 <= t <= self.P * self.pt for t in tokens):
            return "index"
        need = [(s, j) for s, t in zip(slots, tokens) for j in range(-(-self.lengths[s] // self.pt), -(-t // self.pt))]
        free = self.free_pages()
        if len(free) < len(need):
            return "pages"
        for (s, j), p in zip(need, free):
            self.table[s][j] = p
        for s, t in zip(slots, tokens):
            self.lengths[s] = max(self.lengths[s], t)

    def fork(self, src, dst):
        if len(set(dst)) < len(dst) or any(not 0 <= s < len(self.table) for s in src + dst):
            return "index"
        table, lengths = [list(r) for r in self.table], list(self.lengths)
        for a, b in zip(src, dst):
            self.table[b], self.lengths[b] = list(table[a]), lengths[a]
        copies = [i for i, a in enumerate(src) if lengths[a] % self.pt and (a not in dst or a in src[:i])]
        free = self.free_pages()
        if len(free) < len(copies):
            self.table, self.lengths = table, lengths
            return "pages"
        for i, p in zip(copies, free):
            j, used = divmod(lengths[src[i]], self.pt)
            self.rows[p][:used] = self.rows[self.table[dst[i]][j]][:used]
            self.table[dst[i]][j] = p

    def free(self, slots, below=None):
        for i, s in enumerate(slots):
            if not 0 <= s < len(self.table) or (below and below[i] < 0):
                continue
            end = self.P if below is None else min(below[i], self.lengths[s]) // self.pt
            self.table[s][:end] = [-1] * end
            if below is None:
                self.lengths[s] = 0

    def compact(self):
        r = self.refs()
        live = sum(v > 0 for v in r)
        at, to = [p for p in range(live, self.n) if r[p]], [p for p in range(live) if not r[p]]
        for a, b in zip(at, to):
            self.rows[b] = list(self.rows[a])
        m = dict(zip(at, to))
        self.table = [[m.get(p, p) for p in row] for row in self.table]
        return live


# -- refusals, on any machine -----------------------------------------------------------------------------------------------
def test_refusals_without_a_device():
    from ironpangu_b200.ops import pages as P

    c = torch.zeros(4, 16, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no caches"):
        P.PageSet([])
    with pytest.raises(ValueError, match="on one device"):
        P.PageSet([c])                                 # not on a device


def test_plain_pool_by_hand():
    """The model of these tests itself, on cases that a reader can follow."""
    p = Plain(8, 4, 4, 4, [[(i, r) for r in range(4)] for i in range(8)])
    assert p.extend([0], [10]) is None and p.table[0] == [0, 1, 2, -1]
    assert p.fork([0, 0], [1, 2]) is None                 # 10 % 4 = 2 rows of page 2, which slot 0 keeps
    assert p.table[1] == [0, 1, 3, -1] and p.table[2] == [0, 1, 4, -1] and p.refs()[:5] == [3, 3, 1, 1, 1] and p.rows[3] == [(2, 0), (2, 1), (3, 2), (3, 3)]
    assert p.fork([2, 1, 1], [1, 2, 3]) is None           # both replaced: their first children go on with their pages
    assert p.table[1] == [0, 1, 4, -1] and p.table[2] == [0, 1, 3, -1] and p.table[3] == [0, 1, 5, -1]
    p.free([1, 1, 0])
    assert p.refs() == [2, 2, 0, 1, 0, 1, 0, 0] and p.compact() == 4 and p.table[3] == [0, 1, 2, -1]
    assert p.extend([0], [17]) == "index" and p.extend([0, 1], [16, 4]) == "pages" and p.extend([0, 0], [4, 4]) == "index" and p.lengths == [0, 0, 10, 10]


# -- on the device ----------------------------------------------------------------------------------------------------------
def _pool(pages, pt, slots, max_pages, widths, seed=0):
    from ironpangu_b200.ops import pages as P

    g = torch.Generator(device="cuda").manual_seed(seed)
    caches = []
    for width, dtype in widths:
        c = torch.randint(-120, 120, (pages, pt, width), generator=g, device="cuda", dtype=torch.int8)
        caches.append(c.to(dtype) if dtype.is_floating_point else c)
    return P.PagePool(caches, slots=slots, max_pages=max_pages), Plain(pages, pt, slots, max_pages, [[(p, r) for r in range(pt)] for p in range(pages)]), [c.clone() for c in caches]


def _same(pool, plain, before):
    assert pool.table.tolist() == plain.table and pool.lengths.tolist() == plain.lengths and pool.refs.tolist() == plain.refs()
    bits = [int(w) >> i & 1 for w in pool._bits.tolist() for i in range(32)][:plain.n]
    assert bits == [int(r == 0) for r in plain.refs()]
    p = torch.tensor([[a for a, _ in page] for page in plain.rows], device="cuda")
    r = torch.tensor([[b for _, b in page] for page in plain.rows], device="cuda")
    for now, then in zip(pool.pages.caches, before):
        assert torch.equal(now, then[p, r])


def _tell(pool, got):
    want = {None: None, "index": IndexError, "pages": OverflowError}[got]
    if want is None:
        pool.check()
    else:
        with pytest.raises(want):
            pool.check()
        pool.check()


def _list(v):
    return torch.tensor(v, dtype=I32, device="cuda")


WIDTHS = [[(8, torch.bfloat16)], [(656, torch.int8), (16, torch.int8), (64, torch.float32)], [(128, torch.bfloat16)] * 5]


@pytest.mark.gpu
@pytest.mark.parametrize("seed,pages,pt,slots,max_pages,kind", [(0, 33, 4, 6, 9, 0), (1, 64, 1, 5, 30, 1), (2, 200, 16, 24, 20, 2), (3, 31, 7, 3, 40, 1), (4, 1100, 2, 70, 60, 0),
                                                              (5, 10, 8, 40, 4, 0), (6, 1, 16, 2, 1, 2)])
def test_runs_of_calls(seed, pages, pt, slots, max_pages, kind):
    rng = random.Random(seed)
    pool, plain, before = _pool(pages, pt, slots, max_pages, WIDTHS[kind], seed)
    for step in range(60):
        what = rng.choice(("extend", "extend", "fork", "fork", "free", "below", "compact"))
        pick = rng.sample(range(slots), rng.randint(1, min(slots, 8)))
        if what == "extend":
            tokens = [min(max_pages * pt, plain.lengths[s] + rng.randint(0, 3 * pt)) for s in pick]
            if rng.random() < 0.1:
                tokens[0] = rng.choice((-1, max_pages * pt + 1))
            if rng.random() < 0.1:
                pick[0] = rng.choice((slots, -1, pick[-1]))
            pool.extend(_list(pick), _list(tokens))
            got = plain.extend(pick, tokens)
        elif what == "fork":
            src = [rng.choice(pick + [rng.randrange(slots)]) for _ in pick]
            if rng.random() < 0.1:
                (src if rng.random() < 0.5 else pick)[0] = rng.choice((slots, -5))
            pool.fork(_list(src), _list(pick))
            got = plain.fork(src, pick)
        elif what == "compact":
            pool.compact()
            assert int(pool.live) == plain.compact()
            got = None
        else:
            pick = pick[:3] + pick[:1]                   # one of them twice
            below = [rng.randint(0, max_pages * pt) for _ in pick] if what == "below" else None
            pool.free(_list(pick), None if below is None else _list(below))
            plain.free(pick, below)
            got = None
        _tell(pool, got)
        _same(pool, plain, before)


@pytest.mark.gpu
def test_a_pool_without_room_stays_as_it_was():
    pool, plain, before = _pool(12, 4, 8, 6, WIDTHS[0])
    for slots, tokens in (([0], [22]), ([1, 2], [9, 13])):
        pool.extend(_list(slots), _list(tokens))
        assert plain.extend(slots, tokens) is (None if slots == [0] else "pages")
    _tell(pool, "pages")
    src, dst = [0] * 7, [1, 2, 3, 4, 5, 6, 7]              # seven copies of a partly filled page, six free pages
    pool.fork(_list(src), _list(dst))
    assert plain.fork(src, dst) == "pages"
    _tell(pool, "pages")
    _same(pool, plain, before)
    pool.fork(_list([0] * 8), _list([0] + dst))            # the parent is replaced too, by its first child
    assert plain.fork([0] * 8, [0] + dst) == "pages"
    pool.fork(_list(src[:6]), _list(dst[:6]))
    assert plain.fork(src[:6], dst[:6]) is None
    _tell(pool, "pages")
    _same(pool, plain, before)
    pool.fork(_list([3, 2, 1]), _list([1, 2, 3]))          # no page is free, none is needed
    assert plain.fork([3, 2, 1], [1, 2, 3]) is None
    _tell(pool, None)
    _same(pool, plain, before)


@pytest.mark.gpu
def test_copy_of_pages():
    from ironpangu_b200.ops import pages as P

    g = torch.Generator(device="cuda").manual_seed(0)
    make = lambda n: [torch.randint(-120, 120, (n, 6, w), generator=g, device="cuda", dtype=torch.int8) for w in (16, 48, 4096)]
    a, b = make(9), make(70)
    want = [t.clone() for t in b]
    src, dst, rows = [8, 0, 3, 3, 9, -1, 2, 2], [1, 69, 5, 6, 7, 8, 70, 9], [6, 1, 0, 5, 6, 6, 6, 7]
    for s, d, r in zip(src[:4], dst[:4], rows[:4]):
        for x, y in zip(want, a):
            x[d, :r] = y[s, :r]
    A, B = P.PageSet(a), P.PageSet(b)
    P.copy(A, B, _list(src), _list(dst), _list(rows))
    assert all(torch.equal(x, y) for x, y in zip(b, want))
    with pytest.raises(IndexError):
        B.check()
    P.copy(B, B, _list([1, 69]), _list([2, 3]))
    assert all(torch.equal(t[2], t[1]) and torch.equal(t[3], t[69]) for t in b)
    P.copy(A, B, _list([]), _list([]))
    B.check()
    with pytest.raises(ValueError, match="not alike"):
        P.copy(P.PageSet(a[:2]), B, _list([0]), _list([0]))
    with pytest.raises(ValueError, match="beside"):
        P.copy(A, B, _list([0, 1]), _list([0]))
    with pytest.raises(ValueError, match="int32"):
        P.copy(A, B, torch.zeros(1, dtype=torch.int64, device="cuda"), _list([0]))
    with pytest.raises(ValueError, match="multiple of 16"):
        P.PageSet([torch.zeros(2, 4, 12, dtype=torch.int8, device="cuda")])
    with pytest.raises(ValueError, match="contiguous"):
        P.PageSet([torch.zeros(2, 4, 32, dtype=torch.int8, device="cuda")[..., :16]])


@pytest.mark.gpu
def test_a_step_in_a_graph():
    """Fork, extend and free captured once and replayed with lists that change on the device."""
    pool, plain, before = _pool(90, 4, 6, 12, WIDTHS[2])
    pool.extend(_list([0]), _list([13]))
    plain.extend([0], [13])
    src, dst, tokens = _list([0] * 4), _list([1, 2, 3, 4]), _list([14, 15, 16, 17])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pool.fork(src, dst)
        pool.extend(dst, tokens)
        pool.compact()
    for step in range(6):
        parents = [0] * 4 if step == 0 else [random.Random(step + i).randint(1, 4) for i in range(4)]
        want = [14 + 2 * step + i for i in range(4)]
        src.copy_(_list(parents))
        tokens.copy_(_list(want))
        g.replay()
        assert plain.fork(parents, [1, 2, 3, 4]) is None and plain.extend([1, 2, 3, 4], want) is None
        plain.compact()
        _tell(pool, None)
        _same(pool, plain, before)
    pool.free(_list(list(range(6))))
    assert int(pool.refs.sum()) == 0 and bool((pool.table == -1).all())


@pytest.mark.gpu
def test_positions_fit_32_bits_with_a_page_to_spare():
    from ironpangu_b200.ops import pages as P

    cache = torch.zeros(2, 1 << 19, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="not supported"):
        P.PagePool([cache], slots=1, max_pages=(1 << 12) - 1)
    pool = P.PagePool([cache], slots=1, max_pages=(1 << 12) - 2)
    i32 = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")
    pool.extend(i32(0), i32(((1 << 12) - 2) << 19))
    with pytest.raises(OverflowError):
        pool.check()
    pool.extend(i32(0), i32(1 << 20))
    pool.check()
    assert pool.table[0, :3].tolist() == [0, 1, -1]


@pytest.mark.gpu
def test_pages_beyond_4_gb_of_a_cache():
    """Offsets that pass 32 bits: a page near the end of a cache of 5 GB is shared, copied, moved and copied out."""
    from ironpangu_b200.ops import pages as P

    n, pt = 5120, 16
    cache = torch.zeros(n, pt, 1 << 15, dtype=torch.bfloat16, device="cuda")
    pool = P.PagePool([cache], slots=3, max_pages=n)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    pool.extend(i32(0, 1), i32((n - 3) * pt, pt + 5))
    assert pool.table[1, :2].tolist() == [n - 3, n - 2]
    cache[n - 3], cache[n - 2] = 3.0, 5.0
    pool.fork(i32(1), i32(2))
    pool.check()
    assert pool.table[2, :2].tolist() == [n - 3, n - 1] and bool((cache[n - 1, :5] == 5).all()) and not bool(cache[n - 1, 5:].any())
    out = torch.zeros(2, pt, 1 << 15, dtype=torch.bfloat16, device="cuda")
    store = P.PageSet([out])
    P.copy(pool.pages, store, i32(n - 1), i32(1), i32(5))
    assert bool((out[1, :5] == 5).all()) and not bool(out[0].any()) and not bool(out[1, 5:].any())
    pool.free(i32(0))
    pool.compact()
    pool.check()
    assert int(pool.live) == 3 and pool.table[2, :2].tolist() == [0, 2] and pool.table[1, :2].tolist() == [0, 1]
    assert bool((cache[0] == 3).all()) and bool((cache[1] == 5).all()) and bool((cache[2, :5] == 5).all())
    del cache, pool
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("slots,below", [([-1], None), ([2, -1], [9, 9]), ([-1, -1], [5, 5]), ([-1] * 20, [5] * 20), ([0, 1, 0, -1], [9, 9, 9, 9]), ([0, 0, -1, -1, 0], None),
                                         ([1, 6], None), ([2 ** 31 - 1, 1], [8, 8]), ([-2 ** 31, 1, -1, -2 ** 31], [8, 8, 8, 8]), ([1, 2], [8, -1]), ([3] * 9 + [-1], [8] * 10)])
def test_free_refuses_a_bad_list_as_a_whole(slots, below):
    """A slot out of range, or a negative position, wherever it stands in the list and however often: no page is given back, no length changes, and check says so once."""
    pool, plain, before = _pool(40, 4, 6, 9, WIDTHS[0])
    lists = ([0, 1, 2, 3], [22, 9, 36, 13])
    pool.extend(*map(_list, lists))
    plain.extend(*lists)
    pool.free(_list(slots), None if below is None else _list(below))
    _tell(pool, "index")
    _same(pool, plain, before)
    pool.free(_list([0, 1, 0]), _list([4, 9, 17]))
    plain.free([0, 1, 0], [4, 9, 17])
    _tell(pool, None)
    _same(pool, plain, before)


@pytest.mark.gpu
def test_entries_of_a_table_fit_32_bits():
    from ironpangu_b200.ops import _lib, pages as P

    cache = torch.zeros(2, 1, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="not supported"):
        P.PagePool([cache], slots=8192, max_pages=1 << 18)
    pool = P.PagePool([cache], slots=2, max_pages=2)
    i32 = lambda v: torch.tensor([v], dtype=I32, device="cuda")
    where = [i32(0), i32(1)]
    for slots, most in ((8192, 1 << 18), (1, (1 << 31) - 1)):          # nothing is launched for a pool that the kernels cannot count
        pool.desc.slots, pool.desc.max_pages = slots, most
        for call, args in (("extend", where), ("fork", where), ("free", where[:1]), ("compact", ())):
            with pytest.raises(RuntimeError):
                getattr(pool, call)(*args)
    pool.desc.slots, pool.desc.max_pages = 2, 2
    pool.extend(*where)
    pool.check()
    assert pool.table.tolist() == [[0, -1], [-1, -1]]


@pytest.mark.gpu
def test_check_raises_for_every_kind_of_refusal():
    """A bad list and a lack of pages between two checks: neither hides the other, whichever came first."""
    for calls in (([0, 0], [4]), ([4], [0, 0])):
        pool, plain, before = _pool(3, 4, 5, 6, WIDTHS[0])
        for pick in calls:
            pool.extend(_list(pick), _list([17] * len(pick)))
        _ = [pytest.raises(e, pool.check) for e in (IndexError, OverflowError)]
        _tell(pool, None)
        _same(pool, plain, before)
