"""Continuations that read their prompt once for all and draw from the whole vocabulary: every step's attention and tokens against the definitions."""
import numpy as np
import pytest
import torch

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
gpu = pytest.mark.gpu


def _decoder(*, slots=14, rows=12, context=256, pages=None, int4=False):
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric

    cfg = G.DenseConfig.tiny(2)
    w = G.shard_weights(cfg, G.random_full_weights(cfg, 3), 0, 1, "cuda")
    w["lm_head"] *= 6                              # logits with something to choose
    if int4:
        w = G.quantise_weights(w, group=64)
    return cfg, G.DenseDecoder(cfg, w, Fabric(0, 1), max_tokens=rows, max_context=context, num_slots=slots, keep_logits=True, page_pool=True, num_pages=pages)


def _attention(dec, n):
    """The last layer's attention of the step's rows, from its queries and caches in 64 bits, each sequence through its own pages; and what the result may be off (2^-8 for its rounding, 2^-14 of
    the sum of weights times values for 15-bit weights of f32 scores)."""
    c, hd, g = dec.cfg, dec.cfg.head_dim, dec.hq // dec.hk
    out, room = [], []
    for t in range(n):
        at = torch.arange(int(dec.positions[t]) + 1, device="cuda")
        pages = dec.page_table[int(dec.slots[t])].long()[at // c.page_tokens]
        k, v = (x[-1][pages, at % c.page_tokens].to(F64).repeat_interleave(g, 1) for x in (dec.k_cache, dec.v_cache))
        w = torch.softmax(torch.einsum("hd,jhd->hj", dec.qkv[t, :dec.hq * hd].view(dec.hq, hd).to(F64), k) / hd ** 0.5, 1)
        out.append(torch.einsum("hj,jhd->hd", w, v).reshape(-1))
        room.append(out[-1].abs() * 2 ** -8 + torch.einsum("hj,jhd->hd", w, v.abs()).reshape(-1) * 2 ** -14)
    return torch.stack(out), torch.stack(room)


def _right(c, n):
    want, room = _attention(c.dec, n)
    assert bool(((c.dec.attn[:n].to(F64) - want).abs() <= room).all())


def _drawn(logits, u, it, top_k, top_p, min_p):
    x = logits.double().cpu().numpy()
    w = np.exp(x * it - x.max() * it)
    order = np.argsort(-x, kind="stable")
    n = top_k if 1 <= top_k < len(x) else len(x)
    if min_p > 0:
        n = min(n, max(1, int((w[order] >= min_p).sum())))
    if top_p < 1:
        mass = np.cumsum(w[order[:n]])
        n = max(1, int((np.concatenate([[0.0], mass[:-1]]) < top_p * mass[-1]).sum()))
    ids = np.sort(order[:n])
    run = np.cumsum(w[ids])
    return int(ids[int((run > u * run[-1]).argmax())])


@gpu
@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("length", [1, 16, 37, 150])
@pytest.mark.parametrize("prefill", [False, True])
def test_every_step_is_what_it_says(length, prefill, int4):
    from ironpangu_b200.models.dense_prefill import DensePrefill
    from ironpangu_b200.runtime.continuations import Continuations

    cfg, dec = _decoder(int4=int4)
    c = Continuations(dec, prefill=DensePrefill(dec, max_rows=64, attn_rows=32) if prefill else None, store_pages=24, shared_prefix=True)
    prompt = torch.randint(0, cfg.vocab, (length,), generator=torch.Generator().manual_seed(length)).tolist()
    n, (it, k, p, m) = 10, (np.float32(1 / 0.9), 200, np.float32(0.95), np.float32(0.001))
    ids = c.start(prompt, n, temperature=0.9, top_k=200, top_p=0.95, min_p=0.001, seed=7)

    def tokens(step):
        u = c._table[step, :n].tolist()
        # the table's temperature is a float of 1 / 0.9
        assert ids.tolist() == [_drawn(dec.logits[t], u[t], float(c.inv_temp[t]), k, float(p), float(m)) for t in range(n)]

    tokens(0)
    for step in range(1, 30):                      # the first one is run, the others are replayed
        if step == 12:
            c.resample(torch.tensor([3, 3, 0, 9, 3, 5, 6, 7, 8, 9], dtype=I32, device="cuda"))
        if step == 20:
            held = c.set_aside(4)
            c.pack()
            c.take_up(4, held)
        before = dec.positions[:n].clone()
        c.step()
        dec.positions[:n].copy_(before)            # where the step's rows were
        _right(c, n)
        dec.positions[:n].add_(1)
        tokens(step)
    c.check()
    assert len(set(ids.tolist())) > 1
    c.end()
    assert dec.prefix_groups is None and int(dec.pool.refs.sum()) == 0


@gpu
def test_another_start_with_the_same_graphs():
    """A longer prompt and other wishes through graphs that were captured before, and rows that share nothing afterwards."""
    from ironpangu_b200.runtime.continuations import Continuations

    cfg, dec = _decoder()
    c = Continuations(dec, shared_prefix=True)
    got = {}
    for seed in (1, 2, 1):
        for length, top_k in ((40, 0), (100, 70), (9, 20)):
            prompt = torch.randint(0, cfg.vocab, (length,), generator=torch.Generator().manual_seed(length)).tolist()
            rows = c.generate(prompt, 6, 15, top_k=top_k, seed=seed, temperature=1.3)
            assert got.setdefault((seed, length), rows) == rows and len({tuple(r) for r in rows}) > 1
    fresh_cfg, fresh = _decoder()
    for (seed, length), rows in got.items():
        prompt = torch.randint(0, cfg.vocab, (length,), generator=torch.Generator().manual_seed(length)).tolist()
        assert Continuations(fresh, shared_prefix=True).generate(prompt, 6, 15, top_k={40: 0, 100: 70, 9: 20}[length], seed=seed, temperature=1.3) == rows


@gpu
def test_greedy_with_and_without():
    """Greedy continuations differ only where two logits are as near as the two roundings of the attention leave them."""
    from ironpangu_b200.runtime.continuations import Continuations

    cfg, dec = _decoder()
    prompt = list(range(50))
    a = Continuations(dec, shared_prefix=True).generate(prompt, 3, 10, temperature=0.0, top_k=0)
    assert a[0] == a[1] == a[2]
    _, other = _decoder()
    c = Continuations(other)
    token = c.start(prompt, 1, temperature=0.0)
    for t in a[0]:
        logits = other.logits[0]
        assert float(logits.max() - logits[t]) <= 0.05 * float(logits.abs().max())
        other.tokens[:1].fill_(t)                  # the same tokens in both
        token = c.step()


@gpu
def test_heads_that_share_no_prefix():
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric
    from ironpangu_b200.runtime.continuations import Continuations

    cfg = G.DenseConfig(layers=1, hidden=512, heads=2, kv_heads=1, head_dim=256, ffn=512, vocab=256)
    dec = G.DenseDecoder(cfg, G.random_rank_weights(cfg, 0, 1, "cuda"), Fabric(0, 1), max_tokens=4, max_context=64, num_slots=5, keep_logits=True, page_pool=True)
    with pytest.raises(ValueError, match="share no prefix"):
        Continuations(dec, shared_prefix=True)


class _Fabric:
    world = 2

    def status(self):
        return 0


class _Decoder:
    T, num_slots, max_context = 4, 5, 200
    pool = object()
    fabric = _Fabric()

    def __init__(self):
        self.logits, self.tokens = torch.zeros(4, 50), torch.zeros(4, dtype=I32)
        self.k_cache = self.v_cache = []


def test_refused():
    from ironpangu_b200.runtime.continuations import Continuations

    c = Continuations(_Decoder())
    for kw, what in ((dict(top_k=-1), "top_k"), (dict(top_k=1 << 31), "top_k"), (dict(min_p=-0.1), "min_p"), (dict(min_p=1.5), "min_p"), (dict(min_p=float("nan")), "min_p"), (dict(top_k=0), "several ranks"),
                     (dict(top_k=65), "several ranks"), (dict(top_k=20, min_p=0.1), "several ranks")):
        with pytest.raises(ValueError, match=what):
            c.start([1, 2], 2, **kw)
