"""Continuations of one prompt over shared pages, with bf16 and with 4-bit weights: against the same sequences run one by one, drawn again, set aside and packed."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32


def _decoder(int4, *, slots=6, pool=True, rows=5, context=96, pages=None):
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric

    cfg = G.DenseConfig.tiny(2)
    w = G.shard_weights(cfg, G.random_full_weights(cfg, 3), 0, 1, "cuda")
    fab = Fabric(0, 1)
    if int4:
        w = G.quantise_weights(w, group=64)
    return cfg, fab, G.DenseDecoder(cfg, w, fab, max_tokens=rows, max_context=context, num_slots=slots, keep_logits=True, page_pool=pool, num_pages=pages)


def _row(dec, token, position, slot):
    dec.tokens[:1].fill_(token)
    dec.positions[:1].fill_(position)
    dec.slots[:1].fill_(slot)
    dec.forward(1)
    return dec.logits[0].clone()


def test_a_decoder_with_4_bit_weights_is_one_with_their_values():
    """Logits of the 4-bit decoder against the bf16 one whose weights are the 4-bit values: decode rows, a prompt of many rows, batched rows."""
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.models.dense_prefill import DensePrefill
    from ironpangu_b200.parallel.fabric import Fabric

    cfg, fab, four = _decoder(True, pool=False, rows=8, context=256)
    values = {k: (v.dequantise() if hasattr(v, "dequantise") else v) for k, v in four.w.items()}
    full = G.DenseDecoder(cfg, values, Fabric(0, 1), max_tokens=8, max_context=256, num_slots=6, keep_logits=True)
    prompt = torch.randint(0, cfg.vocab, (150,), generator=torch.Generator().manual_seed(1), dtype=I32).cuda()
    pre = [DensePrefill(d, max_rows=100, attn_rows=32) for d in (four, full)]
    got = []
    for d, p in zip((four, full), pre):
        for at in (0, 100):
            p.forward(prompt[at:at + 100], at, 2)
        got.append([d.logits[0].clone(), _row(d, 7, 150, 2)])
        rows = torch.tensor([5, 9, 11, 900] * 5, dtype=I32, device="cuda")
        slots = torch.tensor([2, 3, 4, 5] * 5, dtype=I32, device="cuda")
        pos = torch.cat([torch.tensor([151, 0, 0, 0]) + i for i in range(5)]).to(I32).cuda()
        got[-1].append(p.forward_rows(rows, pos, slots, torch.arange(20, device="cuda")).clone())
    # the same values but for rounding: weights of bf16(s (q - z)) there, a unit's gate and up rounded there
    for a, b in zip(*got):
        torch.testing.assert_close(a, b, rtol=2e-2, atol=2e-2)
    assert four.fabric.status() == 0 and sum(w.nbytes for w in four.w.values() if hasattr(w, "nbytes") and hasattr(w, "units")) < 0.33 * sum(
        values[k].numel() * 2 for k, w in four.w.items() if hasattr(w, "units"))


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("length", [1, 15, 16, 37])
def test_continuations_are_the_sequences_run_alone(int4, length):
    from ironpangu_b200.runtime.continuations import Continuations

    cfg, fab, dec = _decoder(int4)
    c = Continuations(dec)
    prompt = torch.randint(0, cfg.vocab, (length,), generator=torch.Generator().manual_seed(length)).tolist()
    got = c.generate(prompt, 4, 20, temperature=0.8, top_k=20, seed=5)
    assert len({tuple(r) for r in got}) > 1 and all(len(r) == 20 for r in got) and int(dec.pool.refs.sum()) == 0
    # each continuation's tokens through a slot of its own: the same sampling, logits of rows that stand alone
    from ironpangu_b200.ops import decode as K

    _, _, one = _decoder(int4, pool=False)
    for i, row in enumerate(got):
        for p, t in enumerate(prompt):
            logits = _row(one, t, p, 0)
        f = lambda v, dt=torch.float32: torch.tensor([v], dtype=dt, device="cuda")
        counter, seed = f(0, torch.int64), f(i + 5 * 0x9E3779B1, torch.int64)
        for k, t in enumerate(row):
            want = K.sample_topk(logits[None].contiguous(), one.fabric, top_k=20, inv_temperature=f(1 / 0.8), top_p=f(1.0), seeds=seed, counters=counter)
            if int(want) != t:               # two candidates whose draw lies at their border: the batch rounds a sum another way
                probs = torch.softmax(logits / 0.8, -1)
                assert probs[t] > 0.5 * probs.topk(20).values[-1], (i, k)
                break
            logits = _row(one, t, length + k, 0)
    fab.close()


@pytest.mark.parametrize("int4", [False, True])
def test_drawn_again_set_aside_and_packed(int4):
    from ironpangu_b200.models.dense_prefill import DensePrefill
    from ironpangu_b200.runtime.continuations import Continuations

    cfg, fab, dec = _decoder(int4)
    c = Continuations(dec, prefill=DensePrefill(dec, max_rows=64, attn_rows=32), store_pages=12)
    prompt = torch.randint(0, cfg.vocab, (37,), generator=torch.Generator().manual_seed(0)).tolist()
    c.start(prompt, 5, temperature=1.0, top_k=30, seed=1)
    for _ in range(6):
        c.step()

    def caches(i):
        n = int(dec.pool.lengths[1 + i])
        pages = dec.pool.table[1 + i, :-(-n // 16)].long()
        return torch.stack([t[pages].flatten(0, 1)[:n] for t in dec.k_cache + dec.v_cache])

    before, tokens = [caches(i) for i in range(5)], dec.tokens[:5].clone()
    c.resample(torch.tensor([3, 0, 0, 3, 1], dtype=I32, device="cuda"))
    c.check()
    for i, j in enumerate((3, 0, 0, 3, 1)):
        assert torch.equal(caches(i), before[j]) and int(dec.tokens[i]) == int(tokens[j])
    now = [caches(i) for i in range(5)]
    held = c.set_aside(2)
    assert int(dec.pool.lengths[3]) == 0
    live = c.pack()
    assert live == int((dec.pool.refs > 0).sum()) and bool((dec.pool.refs[:live] > 0).all())
    for i in (0, 1, 3, 4):
        assert torch.equal(caches(i), now[i])
    c.take_up(2, held)
    assert torch.equal(caches(2), now[2])
    alike = torch.tensor([0, 3], device="cuda")       # drawn from the same parent, with different seeds from here on
    first = c.step().clone()
    logits = dec.logits[:5].clone()
    assert torch.equal(logits[alike[0]], logits[alike[1]])
    for _ in range(4):
        c.step()
    c.check()
    c.end()
    assert int(dec.pool.refs.sum()) == 0 and first.shape == (5,)
    fab.close()


def test_refusals():
    from ironpangu_b200.runtime.continuations import Continuations

    _, fab, dec = _decoder(False, pool=False)
    with pytest.raises(ValueError, match="page_pool"):
        Continuations(dec)
    cfg, fab, dec = _decoder(False, pages=7)
    c = Continuations(dec)
    for args, what in (((range(5), 6), "takes 1 to 5"), (([], 2), "prompt of 0"), ((range(97), 2), "prompt of 97")):
        with pytest.raises(ValueError, match=what):
            c.start(list(args[0]), args[1])
    with pytest.raises(RuntimeError, match="start"):
        c.step()
    c.start(list(range(40)), 4)                       # three pages, and four copies of the last one
    for _ in range(8):
        c.step()
    c.check()
    c.step()                                          # position 48: a page more for each, and none left
    with pytest.raises(OverflowError):
        c.check()
    c.end()
    c.start(list(range(20)), 2)
    assert c.generate(list(range(20)), 2, 3, temperature=0.0)[0] == c.generate(list(range(20)), 1, 3, temperature=0.0)[0]


def test_set_aside_once_and_taken_up_as_itself():
    """While a continuation is set aside no step is taken and nothing is drawn; it comes back once, from what it was set aside as, or goes with the end."""
    from ironpangu_b200.runtime.continuations import Continuations

    _, fab, dec = _decoder(False)
    c = Continuations(dec, store_pages=4)
    c.start(list(range(20)), 3, seed=2)
    held = c.set_aside(1)
    for call, what in ((c.step, "set aside"), (lambda: c.resample(torch.zeros(3, dtype=I32, device="cuda")), "set aside")):
        with pytest.raises(RuntimeError, match=what):
            call()
    other = c.set_aside(0)
    for call in (lambda: c.set_aside(1), lambda: c.take_up(1, other), lambda: c.take_up(2, held)):
        with pytest.raises(ValueError):
            call()
    c.take_up(1, held)
    with pytest.raises(ValueError):
        c.take_up(1, held)
    c.take_up(0, other)
    c.step()
    c.check()
    c.set_aside(2)
    c.end()
    assert sorted(c._store_free) == [0, 1, 2, 3] and int(dec.pool.refs.sum()) == 0
    fab.close()


def test_parents_out_of_range_change_nothing():
    from ironpangu_b200.runtime.continuations import Continuations

    _, fab, dec = _decoder(False)
    c = Continuations(dec)
    c.start(list(range(20)), 3, seed=2)
    table, tokens = dec.pool.table.clone(), dec.tokens.clone()
    for bad in ([0, -1, 1], [0, 1, 3], [2, 2, 2 ** 31 - 1]):
        c.resample(torch.tensor(bad, dtype=I32, device="cuda"))
        with pytest.raises(IndexError):
            c.check()
        assert torch.equal(dec.pool.table, table) and torch.equal(dec.tokens, tokens)
    c.resample(torch.tensor([2, 2, 0], dtype=I32, device="cuda"))
    c.check()
    assert torch.equal(dec.tokens[:3], tokens[:3][[2, 2, 0]])
    fab.close()


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("length,prompt_kernels", [(1, False), (15, False), (16, True), (37, True)])
def test_logits_are_those_of_sequences_that_share_nothing(int4, length, prompt_kernels):
    """Every step's logits, bit for bit, against a decoder whose slots have pages of their own and which runs the same launches with the tokens that were drawn: over ends of pages,
    draws with repeats (whose caches are copied whole there), packing, and a continuation that was away."""
    from ironpangu_b200.models.dense_prefill import DensePrefill
    from ironpangu_b200.runtime.continuations import Continuations

    n = 4
    cfg, fab, dec = _decoder(int4)
    _, _, own = _decoder(int4, pool=False)
    pre = [DensePrefill(d, max_rows=24, attn_rows=32) if prompt_kernels else None for d in (dec, own)]
    c = Continuations(dec, prefill=pre[0], store_pages=8)
    prompt = torch.randint(0, cfg.vocab, (length,), generator=torch.Generator().manual_seed(length)).to(I32)
    tokens = c.start(prompt.tolist(), n, temperature=1.2, top_k=40, seed=9).clone()
    for slot in range(1, n + 1):                      # the prompt, in each slot
        for p in range(0, length, 24 if prompt_kernels else own.T):
            part = prompt[p:p + (24 if prompt_kernels else own.T)].cuda()
            if prompt_kernels:
                pre[1].forward(part, p, slot)
            else:
                m = part.numel()
                own.tokens[:m].copy_(part)
                own.positions[:m].copy_(torch.arange(p, p + m, dtype=I32))
                own.slots[:m].fill_(slot)
                own.forward(m)
        last = 0 if prompt_kernels else part.numel() - 1
        assert torch.equal(own.logits[last], dec.logits[slot - 1])
    parents = {3: [1, 1, 3, 0], 18: [2, 2, 2, 2], 33: [3, 0, 1, 0]}
    for k in range(40):
        own.tokens[:n].copy_(tokens)
        own.positions[:n].fill_(length + k)
        own.slots[:n].copy_(torch.arange(1, n + 1, dtype=I32))
        own.forward(n)
        want = own.logits[:n].clone()
        tokens = c.step().clone()
        assert torch.equal(dec.logits[:n], want), k
        if k in parents:
            at = torch.tensor(parents[k], device="cuda")
            c.resample(at.to(I32))
            tokens = tokens[at]
            of = own.page_table.long()
            for t in own.k_cache + own.v_cache:
                t[of[1:n + 1]] = t[of[1 + at]]
        if k % 10 == 4:
            c.pack()
        if k % 10 == 7:
            c.take_up(2, c.set_aside(2))
    c.check()
    c.end()
    assert int(dec.pool.refs.sum()) == 0 and own.fabric.status() == 0
    fab.close()


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("n", [9, 16, 20])
def test_more_rows_than_the_head_takes(int4, n):
    """Steps of more than eight continuations - with 4-bit weights of more than sixteen, whose rows are operands made in a launch ahead - in a captured graph: every step's logits against the
    same launches over slots that share nothing."""
    from ironpangu_b200.runtime.continuations import Continuations

    cfg, fab, dec = _decoder(int4, slots=22, rows=20)
    _, _, own = _decoder(int4, pool=False, slots=22, rows=20)
    c = Continuations(dec)
    prompt = torch.randint(0, cfg.vocab, (25,), generator=torch.Generator().manual_seed(n)).to(I32)
    tokens = c.start(prompt.tolist(), n, temperature=1.2, top_k=40, seed=4).clone()
    for slot in range(1, n + 1):
        for p in range(0, 25, 20):
            m = min(20, 25 - p)
            own.tokens[:m].copy_(prompt[p:p + m])
            own.positions[:m].copy_(torch.arange(p, p + m, dtype=I32))
            own.slots[:m].fill_(slot)
            own.forward(m)
        assert torch.equal(own.logits[4], dec.logits[slot - 1])
    for k in range(12):
        own.tokens[:n].copy_(tokens)
        own.positions[:n].fill_(25 + k)
        own.slots[:n].copy_(torch.arange(1, n + 1, dtype=I32))
        ids = own.forward(n)
        tokens = c.step().clone()
        assert torch.equal(dec.logits[:n], own.logits[:n]), k
        assert torch.equal(ids.long(), own.logits[:n].argmax(-1))
    c.check()
    c.end()
    assert own.fabric.status() == 0
    fab.close()


def test_more_rows_than_the_sampling_takes():
    """130 continuations: drawn with seeds of their own, from logits that are alike for a prompt's first token; each row's tokens are those of the sampling of that row alone."""
    from ironpangu_b200.ops import decode as K
    from ironpangu_b200.runtime.continuations import Continuations

    n = 130
    cfg, fab, dec = _decoder(True, slots=n + 1, rows=n)
    c = Continuations(dec, store_pages=8)
    for k in range(8):
        ids = c.start(list(range(20)), n, temperature=1.1, top_k=30, seed=6).clone() if k == 0 else c.step().clone()
        for i in (0, 63, 64, 100, 127, 128, 129):
            f = lambda v, dt=torch.float32: torch.tensor([v], dtype=dt, device="cuda")
            want = K.sample_topk(dec.logits[i:i + 1].contiguous(), fab, top_k=30, inv_temperature=f(1 / 1.1), top_p=f(1.0), seeds=f(i + 6 * 0x9E3779B1, torch.int64),
                                 counters=f(k, torch.int64))
            assert int(ids[i]) == int(want), (k, i)
    c.resample(torch.arange(n, dtype=I32, device="cuda") // 2)
    c.step()
    c.pack()
    c.take_up(n - 1, c.set_aside(n - 1))
    c.step()
    c.check()
    c.end()
    assert int(dec.pool.refs.sum()) == 0 and fab.status() == 0
    fab.close()
