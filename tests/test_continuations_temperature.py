"""Continuations drawn from the whole vocabulary at the ends of what a temperature may be."""
import math

import pytest
import torch

I32 = torch.int32


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [math.inf, 1e39, 1e300])
def test_endless_temperatures_make_all_kept_tokens_alike(temperature):
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric
    from ironpangu_b200.runtime.continuations import Continuations

    cfg = G.DenseConfig.tiny(2)
    dec = G.DenseDecoder(cfg, G.shard_weights(cfg, G.random_full_weights(cfg, 3), 0, 1, "cuda"), Fabric(0, 1), max_tokens=10, max_context=64, num_slots=12, keep_logits=True, page_pool=True)
    c = Continuations(dec)
    for top_k in (0, 100):
        ids = c.start([1, 2, 3], 10, temperature=temperature, top_k=top_k, seed=4)
        for step in range(4):
            for t, (u, got) in enumerate(zip(c._table[step, :10].double().tolist(), ids.tolist())):
                order = torch.argsort(dec.logits[t], descending=True, stable=True)
                kept = order[:top_k or cfg.vocab].sort().values.tolist()
                assert got == kept[int(u * len(kept))]
            c.step()
        c.check()
        c.end()


class _Fabric:
    world = 1

    def status(self):
        return 0


class _Decoder:
    T, num_slots, max_context = 4, 5, 200
    pool = object()
    fabric = _Fabric()

    def __init__(self):
        self.logits, self.tokens = torch.zeros(4, 50), torch.zeros(4, dtype=I32)
        self.k_cache = self.v_cache = []


def test_a_temperature_that_is_no_number():
    """Also where it had let top_k 0 through to the sampler of 64 at most."""
    from ironpangu_b200.runtime.continuations import Continuations

    c = Continuations(_Decoder())
    for kw in (dict(top_k=0), dict(top_k=65), dict(min_p=0.1)):
        with pytest.raises(ValueError, match="no number"):
            c.start([1, 2], 2, temperature=math.nan, **kw)
