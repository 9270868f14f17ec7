"""Which rows of a decoder go by which groups: those of continuations by their own, whatever else uses the decoder between their steps."""
import pytest
import torch

BF16, I32 = torch.bfloat16, torch.int32
pytestmark = pytest.mark.gpu
PROMPT, N = list(range(3, 60)), 6


def _decoder(slots=12, rows=10):
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric

    cfg = G.DenseConfig.tiny(2)
    w = G.shard_weights(cfg, G.random_full_weights(cfg, 3), 0, 1, "cuda")
    w["lm_head"] *= 6                              # logits with something to choose
    return G.DenseDecoder(cfg, w, Fabric(0, 1), max_tokens=rows, max_context=160, num_slots=slots, keep_logits=True, page_pool=True)


def _steps(dec, c, between=lambda step: None, steps=6):
    """Tokens and the last layer's attention of each step."""
    ids, got = c.start(PROMPT, N, temperature=1.2, top_k=40, seed=5), []
    tokens = [ids.clone()]
    for i in range(steps):
        between(i)
        tokens.append(c.step().clone())
        got.append(dec.attn[:N].clone())
    c.check()
    c.end()
    return torch.stack(tokens), torch.stack(got)


def _same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.fixture(scope="module")
def alone():
    """With and without a shared prefix; the two round differently, so that a step of the other kind shows."""
    from ironpangu_b200.runtime.continuations import Continuations

    found = {}
    for shared in (False, True):
        dec = _decoder()
        found[shared] = _steps(dec, Continuations(dec, shared_prefix=shared))
        assert dec.prefix_groups is None
    assert not torch.equal(found[False][1], found[True][1])
    return found


def test_another_object_between_the_steps(alone):
    """Made, or ended, between a start and the first step, which is captured then, and between later ones."""
    from ironpangu_b200.runtime.continuations import Continuations

    for at in (0, 1, 3):
        dec = _decoder()
        c = Continuations(dec, shared_prefix=True)
        assert _same(_steps(dec, c, lambda i: Continuations(dec, shared_prefix=True) if i == at else None), alone[True])
        # the graphs that were captured then
        assert _same(_steps(dec, c), alone[True])


def test_rows_of_others_between_the_steps():
    """A sequence of its own in a slot that no continuation has, while continuations with a longer prompt live: it sees its own pages."""
    from ironpangu_b200.runtime.continuations import Continuations

    def row(dec, token, position, slot):
        dec.pool.extend(torch.tensor([slot], dtype=I32, device="cuda"), torch.tensor([position + 1], dtype=I32, device="cuda"))
        kept = [x[:1].clone() for x in (dec.tokens, dec.positions, dec.slots)]
        for x, v in zip((dec.tokens, dec.positions, dec.slots), (token, position, slot)):
            x[:1].fill_(v)
        dec.forward(1)
        for x, v in zip((dec.tokens, dec.positions, dec.slots), kept):
            x[:1].copy_(v)
        return dec.logits[0].clone()

    dec = _decoder()
    want = [row(dec, 7 + i, i, N + 3) for i in range(6)]
    dec = _decoder()
    got = []
    _steps(dec, Continuations(dec, shared_prefix=True), lambda i: got.append(row(dec, 7 + i, i, N + 3)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert dec.prefix_groups is None


def test_groups_that_the_decoder_was_given(alone):
    """They are for other rows: continuations do not go by them, and leave them."""
    from ironpangu_b200.runtime.continuations import Continuations

    for shared in (False, True):
        dec = _decoder()
        mine = torch.tensor([[0, 4, 48, 11]], dtype=I32, device="cuda")
        dec.share_prefix(mine)
        assert _same(_steps(dec, Continuations(dec, shared_prefix=shared)), alone[shared])
        assert dec.prefix_groups is mine


def test_a_step_that_raises_leaves_the_groups():
    from ironpangu_b200.runtime.continuations import Continuations

    dec = _decoder()
    c = Continuations(dec, shared_prefix=True)
    c.start(PROMPT, N, top_k=40, seed=1)
    forward = dec.forward
    dec.forward = lambda *a: (_ for _ in ()).throw(RuntimeError("no"))
    with pytest.raises(RuntimeError, match="no"):
        c.step()
    dec.forward = forward
    assert dec.prefix_groups is None
    c.end()
