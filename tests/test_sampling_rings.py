"""Sampling of more rows than shared memory holds: they are read again, pass by pass, through rings of each thread. Against the definition in 64 bits, in both types, with every cut."""
import pytest
import torch

from ironpangu_b200.ops import sampling
from test_sampling import CUTS, SHARES, plain

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
pytestmark = pytest.mark.gpu
NAMES = ("inv_temperature", "top_k", "top_p", "min_p")


def rows(T, V, pitch, dtype, seed, spread=2.0, offset=0):
    """Logits in rows that lie `pitch` elements apart, from 16 bytes and `offset` elements on; what lies between them is larger than any of them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.full((T * pitch + offset,), 90.0, device="cuda", dtype=dtype)
    x = base[offset:].as_strided((T, V), (pitch, 1))
    v = torch.randn(T, V, generator=g, device="cuda") * spread
    v.scatter_add_(1, torch.randint(0, V, (T, 20), generator=g, device="cuda"), torch.rand(T, 20, generator=g, device="cuda") * 12 * min(1.0, spread))
    x.copy_(v)
    return x, torch.rand(T, generator=g, device="cuda")


def check(x, u, some, **cuts):
    """`some`: the rows that are compared. Probabilities are rounded once to f32 (2^-24 of themselves), of sums of weights that are off by 2^-28 of themselves and 2^-45 each, of at least 1 in all."""
    T, V = x.shape
    given = {k: torch.tensor(v, device="cuda", dtype=I32 if k == "top_k" else F32) for k, v in cuts.items()}
    ids, probs = sampling.sample(x, u, probs=True, **given)
    f = lambda k, t, other: other if k not in given else given[k][t].item()
    for t in some:
        want, p = plain(x[t].float().cpu().numpy(), u[t].item(), f("inv_temperature", t, 1.0), f("top_k", t, 0), f("top_p", t, 1.0), f("min_p", t, 0.0))
        assert ids[t].item() == want, f"row {t}: {ids[t].item()}, {want} wanted"
        assert abs(probs[t].item() - p) <= p * (2 ** -24 + V * 2 ** -45 + 2 ** -28), f"row {t}: probability {probs[t].item()}, {p} wanted"
    return ids, probs


# four CTAs a row, two, one; rings to the end; rings and a tail; no rings, as the rows lie on 16 bytes by chance only
SHAPES = [(40, 100000, 100000, 0), (64, 151936, 151936, 0), (100, 60000, 60000, 0), (150, 100008, 100008, 0), (297, 40000, 40000, 0), (40, 100003, 100008, 0), (297, 33333, 33336, 0), (40, 100003, 100003, 0),
          (150, 100000, 100001, 3), (19, 1 << 18, 1 << 18, 0)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,pitch,offset", SHAPES)
def test_definition(T, V, pitch, offset, dtype):
    x, u = rows(T, V, pitch, dtype, T + V, offset=offset)
    some = sorted({0, 1, T // 3, T // 2, T - 2, T - 1})
    for name, cut in CUTS.items():
        check(x, u, some, inv_temperature=[0.5 + 0.3 * (t % 5) for t in range(T)], **{k: [v] * T for k, v in cut.items()})
    # every row its own
    check(x, u, range(min(T, 24)), inv_temperature=[(0.0, 1.0, -1.0, 0.6, 1e-3, 1e4, 0.7, 1.3)[t % 8] for t in range(T)], top_k=[(0, 1, 5, 64, 1000, V - 1, V, 20000)[(t + t // 8) % 8] for t in range(T)],
          top_p=[(1.0, 0.5, 0.0, 0.999999, 2.0, 0.9, 0.97, 0.3)[(t + t // 5) % 8] for t in range(T)], min_p=[(0.0, 0.0, 0.3, 1.0, 2.0, 0.01, 1e-5, 0.0)[t * 3 % 8] for t in range(T)])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,spread,it", [(40, 100000, 0.5, 1.0), (40, 100003, 2.0, 0.05), (40, 151936, 0.1, 1.0), (150, 100000, 2.0, 8.0), (150, 100000, 0.02, 1.0), (150, 60000, 1e-6, 1.0), (150, 60000, 1e4, 1.0),
                                           (19, 1 << 18, 0.5, 1.0)])
def test_shares_that_end_among_many_tokens(T, V, spread, it, dtype):
    """Where the mass reaches the share, more tokens lie close than a list takes: stretches of a bin, then bits of values and ids."""
    x, u = rows(T, V, (V + 7) // 8 * 8, dtype, V, spread)
    some = sorted(set(range(8)) | {T - 1})
    share = [SHARES[t % 8] for t in range(T)]
    temper = [it] * T
    check(x, u, some, inv_temperature=temper, top_p=share)
    check(x, u, some, inv_temperature=temper, top_p=share[::-1], top_k=[(V // 2, V // 3, 2000, 1500, 0, V - 1, V, 3)[t % 8] for t in range(T)])
    check(x, u, some, inv_temperature=temper, top_p=share, min_p=[(0.9, 0.5, 0.1, 0.01, 1e-4, 0.99, 0.2, 0.0)[t % 8] for t in range(T)])


def test_values_that_are_nearly_equal():
    T, V = 150, 60000
    g = torch.Generator(device="cuda").manual_seed(9)
    x = 1 + torch.randint(0, 40, (T, V), generator=g, device="cuda").float() * 2 ** -23         # forty values side by side, 1500 tokens each
    u = torch.rand(T, generator=g, device="cuda")
    share = [SHARES[t % 8] for t in range(T)]
    check(x, u, range(8), top_p=share)
    x[:, ::2] -= 30                                # half of them weigh nothing
    check(x, u, range(8), top_p=share)
    x[:, 5] = 4.0
    check(x, u, range(8), top_p=share, top_k=[20000] * T)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_and_masked_logits(dtype):
    T, V, inf = 150, 60000, float("inf")
    x = torch.full((T, V), 1.5, device="cuda", dtype=dtype)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999] * 30, device="cuda")
    check(x, u, range(5))
    check(x, u, range(5), top_k=[1, 2, 3, V // 2, V - 1] * 30)
    check(x, u, range(5), top_p=[0.5, 0.25, 0.125, 0.9, 0.0] * 30)
    x[:] = -inf
    x[1, 59999] = 3.0
    x[2] = torch.finfo(dtype).min
    x[3] = torch.finfo(dtype).min
    x[3, [5, 600, 19999]] = torch.tensor([1.0, 2.0, 0.5], device="cuda", dtype=dtype)
    x[4] = float("nan")
    x[5] = float("nan")
    x[5, 1::7] = torch.randn(len(range(1, V, 7)), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    x[6, [17, 4000, 59992]] = inf
    for kw in ({}, dict(top_k=[3] * T), dict(top_p=[0.9] * T), dict(min_p=[0.2] * T), dict(inv_temperature=[1e-38] * T, top_p=[0.7] * T), dict(inv_temperature=[0.0] * T)):
        ids, probs = check(x, u, range(8), **kw)
        assert ids[[0, 4, 7, 149]].tolist() == [-1] * 4 and probs[[0, 4, 7, 149]].tolist() == [0.0] * 4


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_as_rows_that_are_held(dtype):
    """A row of many, and the same row by itself: one form each, and the same token and probability, bit for bit."""
    x, u = rows(150, 100003, 100008, dtype, 3, 0.7)
    kw = dict(inv_temperature=torch.full((150,), 1.1, device="cuda"), top_k=torch.full((150,), 60000, dtype=I32, device="cuda"), top_p=torch.full((150,), 0.95, device="cuda"))
    ids, probs = sampling.sample(x, u, probs=True, **kw)
    for t in range(0, 150, 7):
        one, p = sampling.sample(x[t:t + 1], u[t:t + 1], probs=True, **{k: v[t:t + 1] for k, v in kw.items()})
        assert one.item() == ids[t].item() and p.item() == probs[t].item()
