"""Kernels that a call of the attention over shared prefixes launches, and a decoder's count of its own."""
import pytest
import torch

from ironpangu_b200.ops import shared_prefix as S

BF16, I32 = torch.bfloat16, torch.int32
CASES = [((4, 8, 2, 64, 1, 16, 10), 2), ((4, 8, 2, 64, 0, 16, 10000), 2), ((24, 32, 8, 128, 1, 16, 100), 2), ((24, 32, 8, 128, 1, 16, 300), 3), ((24, 32, 8, 128, 1, 12, 400), 2),
         ((200, 8, 2, 64, 1, 16, 10), 2), ((200, 8, 2, 64, 1, 12, 10), 2), ((600, 8, 2, 64, 3, 16, 10), 2)]


@pytest.mark.parametrize("call,want", CASES)
def test_launches(call, want):
    assert S.launches(*call) == want


def test_refused():
    for bad in ((0, 8, 2, 64, 1, 16, 10), (4, 7, 2, 64, 1, 16, 10), (4, 8, 2, 32, 1, 16, 10), (4, 8, 2, 64, -1, 16, 10), (4, 8, 2, 64, 1, 0, 10)):
        with pytest.raises(ValueError, match="not supported"):
            S.launches(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("call,want", CASES)
def test_launches_of_a_call(call, want):
    """Kernels of a captured call, by the graph's own account."""
    from cuda.bindings import runtime

    rows, heads, kv, dim, groups, page, pages = call
    z = lambda *s, dt=I32: torch.zeros(*s, dtype=dt, device="cuda")
    args = (z(rows, heads * dim, dt=BF16), z(3, page, kv, dim, dt=BF16), z(3, page, kv, dim, dt=BF16), z(rows), z(rows), z(1, pages), z(groups, 4))
    kw = dict(heads=heads, kv_heads=kv, head_dim=dim, scale=1.0, out=z(rows, heads * dim, dt=BF16), scratch=z(S.scratch_bytes(rows, heads, kv, dim, groups), dt=torch.uint8))
    S.attention(*args, **kw)
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        S.attention(*args, **kw)
    error, _, n = runtime.cudaGraphGetNodes(runtime.cudaGraph_t(graph.raw_cuda_graph()), 64)
    assert int(error) == 0 and n == want


@pytest.mark.gpu
def test_a_decoder_counts_them():
    from ironpangu_b200.models import dense_gqa as G
    from ironpangu_b200.parallel.fabric import Fabric

    cfg = G.DenseConfig.tiny(2)
    dec = G.DenseDecoder(cfg, G.random_rank_weights(cfg, 0, 1, "cuda"), Fabric(0, 1), max_tokens=6, max_context=64, num_slots=8)
    plain = dec.launches_per_forward
    dec.share_prefix(torch.zeros(1, 4, dtype=I32, device="cuda"))
    assert dec.launches_per_forward == plain + cfg.layers
    dec.share_prefix(None)
    assert dec.launches_per_forward == plain
