"""What is left of continuations when a call was refused on the device: nothing goes on from positions that were never written, a start that fails leaves none, and what an
ended run could not do is not said of the next one. The order of calls on the host against a pool and a decoder in plain Python; the rest on the device."""
import pytest
import torch

I32 = torch.int32
NO_PAGES, MBAR_TIMEOUT = 8, 2


class FakePool:
    """A pool that counts pages of 16 positions per slot and shares nothing."""

    def __init__(self, slots, pages):
        self.status, self.lengths, self.page_tokens, self.pages = torch.zeros(1, dtype=I32), torch.zeros(slots, dtype=I32), 16, pages

    def held(self, lengths):
        return int((-(-lengths // 16)).sum())

    def extend(self, slots, tokens):
        now = self.lengths.clone()
        now[slots.long()] = torch.maximum(now[slots.long()], tokens)
        if self.held(now) > self.pages:
            self.status |= NO_PAGES
        else:
            self.lengths = now

    def fork(self, src, dst):
        now = self.lengths.clone()
        now[dst.long()] = self.lengths[src.long()]
        if self.held(now) > self.pages:
            self.status |= NO_PAGES
        else:
            self.lengths = now

    def free(self, slots):
        self.lengths[slots.long()] = 0

    def check(self):
        if int(self.status):
            self.status.zero_()
            raise OverflowError("pages")


class FakeFabric:
    word = 0

    def status(self):
        return self.word

    def clear_status(self):
        self.word = 0


class FakeDecoder:
    T, num_slots, max_context = 4, 5, 200

    def __init__(self, pages):
        self.pool, self.fabric, self.logits = FakePool(5, pages), FakeFabric(), torch.zeros(4, 50)
        self.tokens, self.positions, self.slots = (torch.zeros(4, dtype=I32) for _ in range(3))
        self.k_cache = self.v_cache = []

    def forward(self, n):
        short = self.pool.lengths[self.slots[:n].long()] <= self.positions[:n]
        if bool(short.any()):
            self.fabric.word |= 4              # kernels skip pages that are not there and say so


class Replay:
    """A step without a graph."""

    def __init__(self, c, n):
        self.replay = lambda: c._step(n)


@pytest.fixture
def faked(monkeypatch):
    from ironpangu_b200.runtime import continuations as C

    monkeypatch.setattr(C.K, "sample_topk", lambda logits, *a, out_ids, **k: out_ids.fill_(1))

    def make(pages):
        c = C.Continuations(FakeDecoder(pages))
        c._graphs = {(n, k): Replay(c, n) for n in range(1, 5) for k in (1, 50)}
        return c

    return make


def _refused(c, error, *, word=0):
    with pytest.raises(error):
        c.check()
    for call in (c.step, c.check, lambda: c.resample(torch.zeros(c.n, dtype=I32)), lambda: c.set_aside(0)):
        with pytest.raises(RuntimeError, match="have to be ended"):
            call()


def test_nothing_goes_on_behind_a_refused_step(faked):
    c = faked(12)
    c.start(list(range(30)), 4)                    # two pages each, for the prompt too: ten
    for _ in range(2):
        c.step()
    c.check()
    c.step()                                       # position 32
    _refused(c, OverflowError)
    c.end()
    assert int(c.pool.lengths.sum()) == 0 and c.dec.fabric.word == 0
    c.start(list(range(30)), 2)
    for _ in range(5):
        c.step()
    c.check()


def test_a_refused_step_that_was_not_asked_about(faked):
    c = faked(12)
    c.start(list(range(32)), 4)
    c.step()
    with pytest.raises(OverflowError):             # it has positions that it holds no pages for
        c.set_aside(1)
    c.end()
    c.start(list(range(32)), 4)
    c.step()
    c.end()
    c.start(list(range(32)), 2)                    # not refused for what the ended ones lacked
    c.step()
    c.check()


def test_a_start_without_room_leaves_nothing(faked):
    for pages in (1, 5):                           # not enough for the prompt; not enough for its copies
        c = faked(pages)
        with pytest.raises(OverflowError):
            c.start(list(range(20)), 4)
        assert c.n == 0 and int(c.pool.lengths.sum()) == 0 and c.dec.fabric.word == 0
        with pytest.raises(RuntimeError, match="start"):
            c.step()
        if pages > 1:
            c.start(list(range(20)), 1)
            c.step()
            c.check()


def test_a_resampling_without_room_is_not_gone_on_from(faked):
    c = faked(20)
    c.start(list(range(20)), 4)
    c.pool.pages = 0
    c.resample(torch.tensor([0, 0, 1, 1], dtype=I32))
    _refused(c, OverflowError)


def test_kernels_that_gave_up_show(faked):
    c = faked(20)
    c.dec.fabric.word = MBAR_TIMEOUT
    with pytest.raises(RuntimeError, match="status word = 2"):
        c.start(list(range(20)), 2)
    assert c.n == 0
    c.start(list(range(20)), 2)
    c.step()
    c.dec.fabric.word = MBAR_TIMEOUT
    _refused(c, RuntimeError)
    c.start(list(range(20)), 2)
    c.step()
    c.check()


def test_generate_ends_what_it_started(faked):
    for pages, length, tokens, error in ((12, 30, 40, OverflowError), (1000, 190, 20, OverflowError), (1000, 20, 0, ValueError), (1000, 20, -3, ValueError)):
        c = faked(pages)
        with pytest.raises(error):                 # no pages; past the context; no tokens wanted
            c.generate(list(range(length)), 4, tokens)
        assert c.n == 0 and int(c.pool.lengths.sum()) == 0
        assert c.generate(list(range(20)), 2, 3) == [[1, 1, 1]] * 2 and c.generate(list(range(20)), 2, 1) == [[1]] * 2


def test_generate_refused_for_its_arguments_ends_nothing(faked):
    c = faked(100)
    c.start(list(range(20)), 2)
    for args in (([], 2, 3), ([1], 9, 3), ([1], 2, 0)):
        with pytest.raises(ValueError):
            c.generate(*args)
    assert c.n == 2
    c.step()
    c.check()


def test_seeds_of_any_size(faked):
    c = faked(100)
    for seed in (0, 5, -7, (1 << 32) - 1, 1 << 32, (1 << 63) - 1, (1 << 64) - 1, -(1 << 63), 1 << 100):
        c.start([1, 2, 3], 4, seed=seed)
        assert [int(v) % (1 << 64) for v in c.seeds] == [(seed * 0x9E3779B1 + i) % (1 << 64) for i in range(4)]


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [False, True])
def test_on_the_device(int4):
    """A pool of seven pages: a step that lacks pages, starts that lack them for the prompt and for its copies; and then what a decoder that met none of it gives."""
    from ironpangu_b200.runtime.continuations import Continuations
    from test_continuations import _decoder

    _, fab, dec = _decoder(int4, pages=7)
    _, _, fresh = _decoder(int4, pages=7)
    want = Continuations(fresh).generate(list(range(20)), 3, 12, seed=3)
    c = Continuations(dec)
    c.start(list(range(40)), 4)
    for _ in range(9):
        c.step()
    _refused(c, OverflowError)
    with pytest.raises(OverflowError):
        c.start(list(range(95)), 3)                # six pages, and three copies of the last one
    assert c.n == 0 and int(dec.pool.refs.sum()) == 0 and fab.status() == 0
    c.start(list(range(40)), 4)
    for _ in range(12):
        c.step()
    c.end()                                        # without asking
    assert c.generate(list(range(20)), 3, 12, seed=3) == want and fab.status() == 0 and int(dec.pool.status) == 0
    fab.close()
