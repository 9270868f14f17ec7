"""Attention of rows that share a prefix, against the definition in 64 bits."""
import random

import pytest
import torch

from ironpangu_b200.ops import decode as K
from ironpangu_b200.ops import shared_prefix as S

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
BAD_INDEX = 4
gpu = pytest.mark.gpu


class Batch:
    """Rows of sequences in groups. ``groups``: (rows, shared positions, own positions of each row behind them - or less than none: so many before the prefix's end); rows outside: (rows, None, positions)."""

    def __init__(self, groups, *, heads=8, kv=2, dim=128, page=16, seed=0, each=1, spare=3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = random.Random(seed)
        self.heads, self.kv, self.dim, self.page = heads, kv, dim, page
        tables, slots, positions, listed, taken = [], [], [], [], 0

        def pages_for(n):
            nonlocal taken
            count = -(-n // page)
            taken += count
            return list(range(taken - count, taken))

        for rows, shared, own in groups:
            if shared is not None:
                listed.append([len(slots), rows * each, shared, len(tables)])
                front = pages_for(shared)
                tables.append(front)
            for _ in range(rows):
                mine = own() if callable(own) else own
                last = (shared or 0) + mine - 1
                tables.append((front[:shared // page] if shared is not None else []))
                tables[-1] = tables[-1] + pages_for(last + 1 - page * len(tables[-1]) if last + 1 > page * len(tables[-1]) else 0)
                for e in range(each):
                    slots.append(len(tables) - 1)
                    positions.append(last - each + 1 + e)
        most = max(1, max(len(t) for t in tables))
        n = taken + spare
        where = torch.randperm(n, generator=g, device="cuda").tolist()
        self.table = torch.tensor([[where[p] for p in t] + [-1] * (most - len(t)) for t in tables], dtype=I32, device="cuda")
        dev = lambda v: torch.tensor(v, dtype=I32, device="cuda")
        self.slots, self.positions, self.groups = dev(slots), dev(positions), dev(listed).view(-1, 4)
        randn = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.k = (randn(n, page, kv, dim) + 0.5 * randn(kv, dim)).to(BF16)
        self.v = (randn(n, page, kv, dim) + 0.5 * randn(kv, dim)).to(BF16)
        self.q = randn(len(slots), heads * dim).to(BF16)
        self.scale = dim ** -0.5
        self.status = torch.zeros(1, dtype=I32, device="cuda")

    def run(self, **kw):
        args = dict(heads=self.heads, kv_heads=self.kv, head_dim=self.dim, scale=self.scale, status_ptr=self.status.data_ptr())
        return S.attention(kw.pop("q", self.q), self.k, self.v, self.positions, self.slots, self.table, kw.pop("groups", self.groups), **{**args, **kw})

    def rows_of(self, t):
        """(page, row in it) of every position that row t sees, those that are not there left out."""
        pos, groups = int(self.positions[t]), self.groups.tolist()
        shared, front = next(((n, s) for first, rows, n, s in groups if first <= t < first + rows), (0, None))
        found = []
        for j in range(min(pos + 1, self.table.shape[1] * self.page)):
            slot = front if j < shared else int(self.slots[t])
            page = int(self.table_list[slot][j // self.page]) if 0 <= slot < len(self.table_list) else -1
            if 0 <= page < self.k.shape[0]:
                found.append((page, j % self.page))
        return found

    def want(self, rows=None):
        """(result, what its error may be): a row is rounded once (2^-8), its weights have 15 bits and come from scores and sums in f32 (together 2^-14 of the sum of w |v|)."""
        self.table_list = self.table.tolist()
        out, room = {}, {}
        for t in range(self.q.shape[0]) if rows is None else rows:
            at = self.rows_of(t)
            if not at:
                out[t] = room[t] = torch.zeros(self.heads * self.dim, dtype=F64, device="cuda")
                continue
            pages, inside = (torch.tensor(x, device="cuda") for x in zip(*at))
            k, v = (x[pages, inside].to(F64).repeat_interleave(self.heads // self.kv, 1) for x in (self.k, self.v))
            w = torch.softmax(torch.einsum("hd,jhd->hj", self.q[t, :self.heads * self.dim].view(self.heads, self.dim).to(F64), k) * self.scale, 1)
            out[t] = torch.einsum("hj,jhd->hd", w, v).reshape(-1)
            room[t] = out[t].abs() * 2 ** -8 + torch.einsum("hj,jhd->hd", w, v.abs()).reshape(-1) * 2 ** -14
        return out, room

    def check(self, rows=None, got=None, status=0, **kw):
        got = self.run(**kw) if got is None else got
        out, room = self.want(rows)
        for t in out:
            off = (got[t].to(F64) - out[t]).abs()
            assert bool((off <= room[t]).all()), f"row {t}: {float((off - room[t]).max())} too far off"
        assert int(self.status) == status
        return got


@gpu
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 4, 64), (7, 1, 64), (16, 1, 128), (12, 2, 128)])
@pytest.mark.parametrize("page", [1, 5, 16, 64])
def test_one_group(heads, kv, dim, page):
    for rows, shared, own in ((1, 1, 1), (2, 0, 3), (3, 15, 1), (5, 64, 2), (2, 65, 0), (4, 200, 70), (9, 333, 17)):
        b = Batch([(rows, shared, own)], heads=heads, kv=kv, dim=dim, page=page, seed=rows * 100 + shared)
        b.check()


@gpu
@pytest.mark.parametrize("rows", [1, 2, 4, 7, 8, 9, 15, 16, 17, 31, 33, 64, 130])
def test_rows_of_one_prompt(rows):
    rng = random.Random(rows)
    b = Batch([(rows, 517, lambda: rng.randint(1, 200))], heads=8, kv=2, dim=128, seed=rows)
    b.check()


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_groups_and_rows_outside(dim):
    rng = random.Random(1)
    own = lambda: rng.randint(1, 90)
    b = Batch([(3, None, 77), (5, 300, own), (1, 1000, 5), (2, None, own), (20, 130, own), (4, 0, own), (1, 16, 16)], heads=8, kv=2, dim=dim, seed=5)
    b.check()


@gpu
def test_a_long_prefix_and_long_own_parts():
    b = Batch([(6, 20011, lambda: 3000)], heads=8, kv=2, dim=128, seed=2)
    b.check(rows=[0, 5])
    b = Batch([(40, 9000, lambda: 2100)], heads=4, kv=2, dim=64, seed=3)
    b.check(rows=[0, 17, 39])


@gpu
def test_positions_within_the_prefix():
    """A row that lies before its prefix's end sees it up to its own position, whatever lies behind."""
    b = Batch([(12, 300, lambda: 5)], heads=8, kv=2, dim=128, seed=4)
    b.positions[:6] = torch.tensor([0, 1, 63, 298, 299, 300], dtype=I32)
    b.k[b.table[0, 299 // 16].long(), 299 % 16] = float("nan")       # the prefix's last position
    got = b.run()
    seen = b.positions >= 299
    assert bool(got[seen].isnan().all()) and not bool(got[~seen].isnan().any())
    b.check(rows=[0, 1, 2, 3], got=got)


@gpu
def test_questions_of_several_rows():
    for each, rows, shared in ((3, 5, 100), (40, 4, 513), (128, 2, 1000)):
        b = Batch([(rows, shared, each + 7)], heads=8, kv=2, dim=128, each=each, seed=each)
        b.check(rows=range(0, rows * each, max(1, each // 5)))


@gpu
def test_what_no_row_sees_does_not_matter():
    b = Batch([(5, 100, lambda: 9), (2, None, 50)], heads=8, kv=2, dim=128, seed=6)
    plain = b.run()
    seen = {}
    b.table_list = b.table.tolist()
    for t in range(7):
        for at in b.rows_of(t):
            seen[at] = True
    for value in (float("nan"), float("inf"), -float("inf"), torch.finfo(BF16).min):
        k, v = b.k.clone(), b.v.clone()
        keep = torch.zeros(b.k.shape[:2], dtype=torch.bool, device="cuda")
        for page, row in seen:
            keep[page, row] = True
        b.k[~keep], b.v[~keep] = value, value
        assert torch.equal(b.run(), plain)
        b.k, b.v = k, v
    assert int(b.status) == 0


@gpu
def test_nobodys_rows_are_left_as_they_are():
    b = Batch([(9, 100, lambda: 9)], heads=8, kv=2, dim=128, seed=7)
    b.positions[torch.tensor([0, 4, 8], device="cuda")] = -1
    b.slots[4], b.slots[8] = 1 << 30, -5
    out = torch.full((11, 8 * 128), 7.0, dtype=BF16, device="cuda")
    got = b.run(out=out[1:10])
    assert bool((out[[0, 10, 1, 5, 9]] == 7).all())
    b.check(rows=[1, 2, 3, 5, 6, 7], got=got)
    b.positions.fill_(-1)
    out.fill_(3.0)
    b.run(out=out[1:10])
    assert bool((out == 3).all()) and int(b.status) == 0


@gpu
def test_infinite_values_that_are_seen():
    b = Batch([(3, 70, lambda: 5)], heads=8, kv=2, dim=128, seed=8)
    page = b.table[0, 2].long()
    b.v[page, 3, 0, 5] = float("inf")
    b.v[page, 4, 1, 6] = -float("inf")
    b.k[b.table[1, 70 // 16].long(), 70 % 16, 1] = float("nan")      # own key of row 0
    got = b.run().view(3, 8, 128)
    assert bool((got[:, :4, 5] == float("inf")).all()) and bool((got[1:, 4:, 6] == -float("inf")).all())
    assert bool(got[0, 4:].isnan().all()) and not bool(got[1:].isnan().any()) and not bool(got[0, :4].isnan().any())


@gpu
def test_large_scores():
    b = Batch([(6, 400, lambda: 40)], heads=8, kv=2, dim=128, seed=9)
    b.q *= 30                                      # scores of hundreds: all weight on one key
    b.scale = 1.0
    got = b.run()
    out, _ = b.want()
    # scores of about 500 that are off by 2^-20 of the sum of their terms' sizes, so weights by 2^-9: beside rounding, 2^-8 of the values' spread
    for t in out:
        assert float((got[t].to(F64) - out[t]).abs().max()) <= 2 ** -8 * 5 + float(out[t].abs().max()) * 2 ** -8
    assert bool(got.isfinite().all())


@gpu
def test_pages_slots_and_groups_that_are_not_there():
    b = Batch([(4, 100, lambda: 40), (3, 50, lambda: 20)], heads=8, kv=2, dim=128, seed=10)
    table = b.table.clone()
    b.table[0, 2], b.table[1, 7], b.table[2, 8] = -1, 1 << 29, -7      # of the prefix, of two rows' own
    b.check(status=BAD_INDEX)
    b.table.copy_(table)
    b.status.zero_()
    b.slots[1] = 99
    b.check(status=BAD_INDEX)
    b.slots[1] = -1
    b.check(status=BAD_INDEX)
    b.slots[1] = 2
    b.status.zero_()
    b.positions[2] = b.table.shape[1] * 16 + 1000
    b.check(status=BAD_INDEX)
    b.positions[2] = 120
    good = b.groups.clone()
    for bad in ([-1, 4, 100, 0], [0, 4, -1, 0], [0, 4, 100, 99], [0, 4, 100, -1], [0, 8, 100, 0], [0, 4, 1 << 30, 0], [0, 1 << 31 - 1, 5, 0], [3, -1, 5, 0]):
        b.status.zero_()
        listed = good.clone()
        listed[0] = torch.tensor(bad, dtype=torch.int64).to(I32)
        got = b.run(groups=listed)
        assert int(b.status) == BAD_INDEX
        b.status.zero_()
        kept, b.groups = b.groups, good[1:]        # its rows see everything through their own slots
        b.check(got=got, rows=[4, 5, 6])
        b.groups = kept
    b.status.zero_()
    listed = torch.stack([good[1], good[0]])       # not in the order of their rows: the second one counts as none
    b.run(groups=listed)
    assert int(b.status) == BAD_INDEX
    b.status.zero_()
    empty = torch.tensor([[0, 0, 0, 0], good[0].tolist(), [4, 0, 7, 99], good[1].tolist()], dtype=I32, device="cuda")
    assert torch.equal(b.run(groups=empty), b.run()) and int(b.status) == 0


@gpu
def test_a_row_that_sees_nothing():
    b = Batch([(3, 40, lambda: 3)], heads=8, kv=2, dim=64, seed=11)
    b.table[0], b.table[2] = -1, -1
    got = b.run()
    assert bool((got[1] == 0).all()) and int(b.status) == BAD_INDEX
    b.check(rows=[0, 2], got=got, status=BAD_INDEX)


@gpu
def test_strides_and_given_buffers():
    b = Batch([(5, 90, lambda: 11)], heads=8, kv=2, dim=64, seed=12)
    wide = torch.full((5, 1000), 9.0, dtype=BF16, device="cuda")
    wide[:, :512] = b.q
    out = torch.full((5, 640), 4.0, dtype=BF16, device="cuda")
    scratch = torch.empty(S.scratch_bytes(5, 8, 2, 64), dtype=torch.uint8, device="cuda")
    plain = b.run()
    b.run(q=wide[:, :512], out=out[:, 64:576], scratch=scratch)
    assert torch.equal(out[:, 64:576], plain) and bool((out[:, :64] == 4).all()) and bool((out[:, 576:] == 4).all())
    b.run(q=wide, out=wide[:, :512])               # in the queries' place
    assert torch.equal(wide[:, :512], plain) and bool((wide[:, 512:] == 9).all())
    assert S.attention(b.q[:0], b.k, b.v, b.positions[:0], b.slots[:0], b.table, b.groups, heads=8, kv_heads=2, head_dim=64, scale=1.0).shape == (0, 512)
    b.groups = b.groups[:0]                        # every row sees what its own slot holds
    b.check()


@gpu
def test_captured_on_another_stream_and_twice():
    b, c = (Batch([(6, 400, lambda: 30)], heads=8, kv=2, dim=128, seed=s) for s in (13, 14))
    want_b, want_c = b.run(), c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got_b = b.run()
    with torch.cuda.stream(side):
        got_c = c.run()
    torch.cuda.synchronize()
    assert torch.equal(got_b, want_b) and torch.equal(got_c, want_c)
    out = torch.empty_like(want_b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(out=out)
    graph.replay()
    assert torch.equal(out, want_b)
    b.q.copy_(c.q)                                 # other queries, a shorter prefix, other positions
    b.groups[0, 2] = 112
    b.positions -= 200
    graph.replay()
    b.check(got=out)


@gpu
def test_caches_beyond_32_bits():
    pages, pt, kv, dim = (1 << 31) // (16 * 8 * 128) + 40, 16, 8, 128       # more than 2^31 elements
    b = Batch([(3, 200, lambda: 40)], heads=16, kv=kv, dim=dim, seed=15)
    small, n = (b.k, b.v), b.k.shape[0]
    b.k, b.v = (torch.empty(pages, pt, kv, dim, dtype=BF16, device="cuda") for _ in range(2))
    for big, s in zip((b.k, b.v), small):
        big[pages - n:] = s
    b.table = torch.where(b.table >= 0, b.table + (pages - n), b.table)
    b.check()


@gpu
def test_beside_the_kernel_that_reads_the_prefix_for_every_row():
    b = Batch([(8, 1000, lambda: 64)], heads=16, kv=4, dim=128, seed=16)
    own = b.table.clone()
    for t in range(8):                             # the partly filled page of the prefix, as a fork copies it
        b.k[own[1 + t, 62].long(), :8] = b.k[own[0, 62].long(), :8]
        b.v[own[1 + t, 62].long(), :8] = b.v[own[0, 62].long(), :8]
    other = K.gqa_decode_attention(b.q, b.k, b.v, b.positions, b.slots, b.table, heads=16, kv_heads=4, head_dim=128, scale=b.scale)
    got = b.check()
    assert float((other.float() - got.float()).abs().max()) <= 2 ** -7 * float(got.float().abs().max())


def stale(b):
    """A scratch that a call has to fill by itself: NaN wherever it reads what it did not write."""
    return torch.full((S.scratch_bytes(b.q.shape[0], b.heads, b.kv, b.dim, b.groups.shape[0]),), 255, dtype=torch.uint8, device="cuda")


# From 400 rows by kv heads on, prefixes are read by tiles of 256 pairs on tcgen05 and own positions by four warps each, from 1184 on by one warp; groups of 128 pairs at most have streams of keys
@gpu
@pytest.mark.parametrize("rows,heads,kv,dim,page", [(200, 8, 2, 128, 16), (201, 8, 2, 64, 8), (100, 4, 4, 64, 64), (407, 7, 1, 128, 128), (601, 8, 2, 128, 16), (1200, 16, 1, 64, 24), (301, 12, 4, 128, 256)])
def test_many_rows(rows, heads, kv, dim, page):
    for shared, own in ((1, 1), (0, 3), (127, 0), (128, 1), (129, 2), (500, 130), (1300, 17)):
        b = Batch([(rows, shared, own)], heads=heads, kv=kv, dim=dim, page=page, seed=rows + shared)
        b.check(rows=[0, 1, 31, 32, 64, rows // 2, rows - 1], scratch=stale(b))


@gpu
@pytest.mark.parametrize("rows,heads,kv,dim", [(208, 128, 8, 128), (400, 128, 8, 64), (1024, 8, 4, 64), (900, 14, 2, 128), (640, 64, 16, 64), (1030, 16, 16, 64), (2500, 32, 8, 64)])
def test_stretches_that_fill_the_chip(rows, heads, kv, dim):
    for groups in (1, 3):
        each = rows // groups
        for shared in (130, 1300, 6500):
            b = Batch([(each, shared - 16 * i, 3) for i in range(groups)], heads=heads, kv=kv, dim=dim, page=16, seed=rows)
            b.check(rows=[0, each // 2, each - 1, each * groups - 1], scratch=stale(b))


@gpu
@pytest.mark.parametrize("kv,dim", [(2, 128), (8, 64)])
def test_many_rows_in_groups(kv, dim):
    rng = random.Random(kv)
    own = lambda: rng.randint(1, 60)
    b = Batch([(3, None, 77), (15, 300, own), (1, 2000, 5), (32, 129, own), (2, None, own), (33, 1030, own), (64, 700, own), (65, 128, own), (4, 0, own), (1, 16, 16)], heads=4 * kv, kv=kv, dim=dim, seed=5)
    b.check(rows=[0, 2, 3, 10, 17, 18, 19, 50, 51, 52, 53, 85, 86, 100, 149, 150, 214, 215, 218, 219], scratch=stale(b))


@gpu
def test_many_rows_within_the_prefix_and_nobodys():
    b = Batch([(220, 700, lambda: 5)], heads=8, kv=2, dim=128, seed=20)
    b.positions[:7] = torch.tensor([0, 1, 127, 128, 698, 699, 700], dtype=I32)
    b.positions[100:110] = -1
    b.slots[105] = 1 << 30
    b.k[b.table[0, 699 // 16].long(), 699 % 16] = float("nan")       # the prefix's last position
    out = torch.full((220, 8 * 128), 7.0, dtype=BF16, device="cuda")
    got = b.run(out=out, scratch=stale(b))
    assert bool((got[100:110] == 7).all())
    seen = b.positions >= 699
    assert bool(got[seen].isnan().all()) and not bool(got[~seen].isnan().any())
    b.check(rows=[0, 1, 2, 3, 4], got=got)


@gpu
@pytest.mark.parametrize("rows,page", [(220, 16), (25, 8)])
def test_many_rows_and_pages_that_are_not_there(rows, page):
    b = Batch([(rows, 900, lambda: 40), (220, 400, lambda: 3)], heads=8, kv=2, dim=128, page=page, seed=21)
    at = 1 + rows
    b.table[0, 2], b.table[0, 899 // page], b.table[1, 920 // page], b.table[at, :] = -1, 1 << 29, -7, -1
    b.check(rows=[0, 1, 17, rows - 1, rows, rows + 219], status=BAD_INDEX, scratch=stale(b))


@gpu
@pytest.mark.parametrize("shared", [300, 400])
def test_many_rows_and_what_none_sees(shared):
    b = Batch([(30, shared, lambda: 9), (190, shared, lambda: 9), (2, None, 50)], heads=8, kv=2, dim=128, seed=22)
    plain = b.run(scratch=stale(b))
    b.table_list = b.table.tolist()
    keep = torch.zeros(b.k.shape[:2], dtype=torch.bool, device="cuda")
    for t in range(222):
        pages, inside = (torch.tensor(x, device="cuda") for x in zip(*b.rows_of(t)))
        keep[pages, inside] = True
    for value in (float("nan"), float("inf"), -float("inf"), torch.finfo(BF16).min):
        k, v = b.k.clone(), b.v.clone()
        b.k[~keep], b.v[~keep] = value, value
        assert torch.equal(b.run(), plain)
        b.k, b.v = k, v
    page = b.table[0, 2].long()                    # of the first group's prefix
    b.v[page, 3, 0, 5], b.v[page, 4, 1, 6] = float("inf"), -float("inf")
    got = b.run().view(222, 8, 128)
    assert bool((got[:30, :4, 5] == float("inf")).all()) and bool((got[:30, 4:, 6] == -float("inf")).all()) and torch.equal(got[30:].reshape(192, -1), plain[30:])
    assert not bool(got.isnan().any()) and int(b.status) == 0


@gpu
def test_many_rows_and_large_scores():
    b = Batch([(210, 600, lambda: 40)], heads=8, kv=2, dim=128, seed=23)
    b.q *= 30
    b.scale = 1.0
    got = b.run()
    out, _ = b.want(rows=[0, 100, 209])
    for t in out:                                  # as for few rows
        assert float((got[t].to(F64) - out[t]).abs().max()) <= 2 ** -8 * 5 + float(out[t].abs().max()) * 2 ** -8
    assert bool(got.isfinite().all())


@gpu
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (64, 8, 64)])
def test_the_work_of_a_prefix_decides(heads, kv, dim):
    """16 rows over a few thousand positions: below and from 3.5 million pairs by positions on (7 million of 64 columns), replayed from one graph."""
    b = Batch([(16, 7168, lambda: 33)], heads=heads, kv=kv, dim=dim, page=64, seed=24)
    edge = 3500000 * 128 // dim // kv // (16 * heads // kv)
    scratch = stale(b)
    out = torch.empty_like(b.q)
    b.run(out=out, scratch=scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(out=out, scratch=scratch)
    for shared in (7168, 1, edge // 64 * 64, (edge // 64 + 1) * 64, 0, 6000, 7168):
        b.groups[0, 2] = shared
        b.positions.fill_(shared + 20)
        out.fill_(9.0)
        graph.replay()
        b.check(rows=[0, 15], got=out)


@gpu
def test_a_long_prefix_of_two_groups_and_rows_within_it():
    b = Batch([(18, 9001, lambda: 30), (3, 100, lambda: 10), (30, 5000, lambda: 300)], heads=32, kv=8, dim=128, page=16, seed=25)
    b.positions[3:6] = torch.tensor([0, 5000, 8999], dtype=I32)
    b.positions[19] = -1
    b.check(rows=[0, 3, 4, 5, 17, 18, 20, 21, 50], scratch=stale(b))


@gpu
def test_many_rows_over_caches_beyond_32_bits():
    pages, pt, kv, dim = (1 << 31) // (16 * 8 * 128) + 40, 16, 8, 128       # more than 2^31 elements
    b = Batch([(60, 200, lambda: 4)], heads=16, kv=kv, dim=dim, seed=26)
    small, n = (b.k, b.v), b.k.shape[0]
    b.k, b.v = (torch.empty(pages, pt, kv, dim, dtype=BF16, device="cuda") for _ in range(2))
    for big, s in zip((b.k, b.v), small):
        big[pages - n:] = s
    b.table = torch.where(b.table >= 0, b.table + (pages - n), b.table)
    b.check(rows=[0, 30, 59], scratch=stale(b))


@gpu
def test_many_rows_captured_and_on_two_streams():
    b, c = (Batch([(205, 600, lambda: 30)], heads=8, kv=2, dim=128, seed=s) for s in (27, 28))
    want_b, want_c = b.run(), c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got_b = b.run()
    with torch.cuda.stream(side):
        got_c = c.run()
    torch.cuda.synchronize()
    assert torch.equal(got_b, want_b) and torch.equal(got_c, want_c)
    out = torch.empty_like(want_b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run(out=out)
    graph.replay()
    assert torch.equal(out, want_b)
    b.groups[0, 2] = 112
    b.positions -= 400
    graph.replay()
    b.check(rows=[0, 100, 204], got=out)


@gpu
@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 128), (16, 8, 64), (24, 8, 128), (32, 8, 128), (40, 8, 128), (64, 8, 64), (112, 8, 128), (128, 8, 128), (16, 4, 128), (21, 3, 64), (16, 1, 128)])
def test_questions_of_many_rows(heads, kv, dim):
    """Rows of one sequence that read their own keys together, four by four, wherever their question begins and ends."""
    for each, count in ((4, -(-1184 // kv) // 4), (37, 1 + 1184 // kv // 37), (130, 1 + 1184 // kv // 130)):
        b = Batch([(count, 70, each + 60), (2, None, each)], heads=heads, kv=kv, dim=dim, each=each, seed=each)
        b.positions[1], b.positions[each + 2] = -1, -1
        out = torch.full_like(b.q, 7.0)
        got = b.run(out=out, scratch=stale(b))
        assert bool((got[[1, each + 2]] == 7).all())
        b.check(rows=[0, 2, 3, each - 1, each, each + 1, count * each // 2, count * each - 1, count * each, (count + 2) * each - 1], got=got)


@gpu
def test_questions_whose_later_rows_see_what_is_not_finite():
    b = Batch([(10, 70, 40)], heads=32, kv=8, dim=128, each=16, seed=31)
    plain = b.run()
    lowest = torch.finfo(BF16).min
    def cell(t, back):                             # where row t's key `back` positions before its own lies
        pos = int(b.positions[t]) - back
        return b.table[int(b.slots[t]), pos // 16].long(), pos % 16
    for row, change in ((5, float("nan")), (22, float("inf")), (39, lowest), (54, -float("inf"))):
        page, at = cell(row, 0)
        b.v[page, at] = change
    page, at = cell(70, 0)
    b.k[page, at] = float("nan")
    page, at = cell(86, 0)
    b.k[page, at, 3] = lowest                      # scores of 1e38 times a sum of either sign
    inplace = b.q.clone()
    got = b.run(out=inplace, q=inplace)
    assert torch.equal(got.view(torch.int16), b.run().view(torch.int16))
    for t in range(160):
        first = {0: 5, 1: 22, 2: 39, 3: 54, 4: 70, 5: 86}.get(t // 16, 1 << 30)
        if t < first:
            assert torch.equal(got[t], plain[t]) or bool(((got[t].to(F64) - plain[t].to(F64)).abs() <= 2 ** -7 * plain[t].to(F64).abs() + 2 ** -13 * 8).all())
    b.check(rows=[0, 4, 16, 21, 32, 38, 48, 53, 64, 69, 80, 85, 100, 159], got=got)
    assert bool(got[5:16].isnan().all()) and bool((got[22:32] == float("inf")).all()) and bool((got[54:64] == -float("inf")).all()) and bool(got[70:80].isnan().all())
    assert bool(got[39:48].isfinite().all())


@gpu
def test_the_same_row_many_times():
    b = Batch([(3, 100, 40), (1, None, 33)], heads=32, kv=8, dim=128, seed=32)
    again = torch.arange(4, device="cuda").repeat_interleave(50)
    b.q, b.positions, b.slots = b.q[again].contiguous(), b.positions[again].contiguous(), b.slots[again].contiguous()
    b.groups[0, 1] = 150
    got = b.check(rows=[0, 49, 50, 149, 150, 199])
    for first in range(0, 200, 50):
        assert float((got[first:first + 50].float() - got[first].float()).abs().max()) <= 2 ** -7 * float(got[first].float().abs().max())


@gpu
def test_a_great_many_rows():
    b = Batch([(500, 300, 75), (500, 333, 71)], heads=4, kv=1, dim=64, each=70, seed=41)
    b.check(rows=[0, 69, 70, 34999, 35000, 35001, 50000, 69999], scratch=stale(b))


@gpu
@pytest.mark.parametrize("page", [1, 5, 12, 1000])
def test_many_rows_over_pages_of_any_size(page):
    rng = random.Random(page)
    b = Batch([(3, None, 40), (200, 450, lambda: rng.randint(1, 80)), (20, 131, 5)], heads=8, kv=2, dim=128, page=page, seed=42)
    b.check(rows=[0, 2, 3, 100, 202, 203, 222], scratch=stale(b))


@gpu
@pytest.mark.parametrize("most", [7, 40])
def test_as_many_groups_as_there_may_be(most):
    rng = random.Random(most)
    own = lambda: rng.randint(1, 30)
    b = Batch([(1 + i % most, 17 * i, own) for i in range(64)], heads=8, kv=2, dim=64, seed=43)
    T = b.q.shape[0]
    b.check(rows=[0, 1, 2, T // 3, T // 2, T - 2, T - 1], scratch=stale(b))


@gpu
def test_many_rows_in_the_queries_place():
    b = Batch([(220, 300, lambda: 11)], heads=8, kv=2, dim=64, seed=44)
    plain = b.run()
    wide = torch.full((220, 1000), 9.0, dtype=BF16, device="cuda")
    wide[:, 8:520] = b.q
    b.run(q=wide[:, 8:], out=wide[:, 8:520])
    assert torch.equal(wide[:, 8:520], plain) and bool((wide[:, :8] == 9).all()) and bool((wide[:, 520:] == 9).all())
    b.check(rows=[0, 219], got=plain)


def test_refused_on_the_host():
    q, c, i = torch.zeros(2, 512, dtype=BF16), torch.zeros(4, 16, 2, 64, dtype=BF16), torch.zeros(2, dtype=I32)
    with pytest.raises(ValueError, match="on the host"):
        S.attention(q, c, c, i, i, i.view(1, 2), torch.zeros(1, 4, dtype=I32), heads=8, kv_heads=2, head_dim=64, scale=1.0)
    with pytest.raises(ValueError, match="bf16"):
        S.attention(q.float(), c, c, i, i, i.view(1, 2), torch.zeros(1, 4, dtype=I32), heads=8, kv_heads=2, head_dim=64, scale=1.0)


def test_scratch_refused_and_enough():
    for bad in ((-1, 8, 2, 64), (1 << 21, 8, 2, 64), (4, 7, 2, 64), (4, 8, 0, 64), (4, 34, 2, 64), (4, 8, 2, 0), (4, 8, 2, 32), (4, 8, 2, 64, 65), (4, 8, 2, 64, -1), (4, 0, 2, 64)):
        with pytest.raises(ValueError, match="not supported"):
            S.scratch_bytes(*bad)
    for heads, kv, dim, groups in ((8, 2, 128, 1), (16, 1, 64, 3), (32, 8, 64, 64), (128, 8, 128, 0)):
        most = 0
        for rows in range(1, 700):
            most = max(most, S._scratch(rows, heads, kv, dim, groups))
            if rows % 97 == 0:
                assert S.scratch_bytes(rows, heads, kv, dim, groups) == most
    assert S.scratch_bytes(0, 8, 2, 64) == 0 and S.scratch_bytes(1 << 20, 8, 2, 64) > 1 << 32


@gpu
def test_heads_of_no_columns_are_refused():
    z = lambda *s: torch.zeros(s, dtype=BF16, device="cuda")
    i = torch.zeros(2, dtype=I32, device="cuda")
    with pytest.raises(ValueError, match="columns"):
        S.attention(z(2, 8), z(4, 16, 2, 0), z(4, 16, 2, 0), i, i, i.view(1, 2), i[:0].view(0, 4), heads=8, kv_heads=2, head_dim=0, scale=1.0)


@gpu
def test_refused():
    b = Batch([(4, 20, 3)], heads=8, kv=2, dim=64, seed=1)
    good = dict(q=b.q, k_cache=b.k, v_cache=b.v, positions=b.positions, slots=b.slots, page_table=b.table, groups=b.groups, heads=8, kv_heads=2, head_dim=64, scale=1.0)
    shifted = torch.zeros(4 * 512 + 8, dtype=BF16, device="cuda")[1:2049].view(4, 512)
    for bad, what in ((dict(heads=7), "heads"), (dict(heads=34, kv_heads=2), "heads"), (dict(head_dim=32), "columns"), (dict(heads=16), "queries of"), (dict(kv_heads=4), "keys"), (dict(q=b.q.float()), "bf16"),
                      (dict(q=b.q.T), "bf16"), (dict(q=shifted), "16 bytes"), (dict(v_cache=b.v[:1]), "values"), (dict(k_cache=b.k.transpose(1, 2)), "keys"), (dict(k_cache=b.k.cpu()), "keys"),
                      (dict(positions=b.positions.long()), "positions"), (dict(slots=b.slots[:3]), "slots"), (dict(page_table=b.table.cpu()), "page_table"), (dict(groups=b.groups.long()), "groups"),
                      (dict(groups=b.groups[:, :3].contiguous()), "groups"), (dict(groups=b.groups.expand(65, 4).contiguous()), "groups"), (dict(out=torch.empty(4, 511, dtype=BF16, device="cuda")), "output"),
                      (dict(out=torch.empty(1, 512, dtype=BF16, device="cuda").expand(4, 512)), "output"), (dict(scratch=torch.empty(8, dtype=torch.uint8, device="cuda")), "scratch")):
        with pytest.raises(ValueError, match=what):
            S.attention(**{**good, **bad})
