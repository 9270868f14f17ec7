"""How far a weight may be off, by the tokens that are drawn next to a border of two."""
import pytest
import torch

from ironpangu_b200.ops import sampling

F32, F64, I32 = torch.float32, torch.float64, torch.int32


@pytest.mark.gpu
@pytest.mark.parametrize("depth", [0.1, 2.0, 11.0, 25.0])
@pytest.mark.parametrize("it", [1.0, 0.37, 3.1, 1e-3])
def test_borders_of_two_tokens(it, depth):
    """Token 0 weighs w, token 1 is the largest. 0 is drawn where w exceeds u (1 + w): with a weight that is off by 2^-28 of itself and 2^-45, and a border that is rounded down to units of 2^-44, always where
    w (1 - u) / u is further than 2^-28 + 2^-43 / w from 1 on that side."""
    T = 1 << 18
    g = torch.Generator(device="cuda").manual_seed(int(depth * 10))
    rand = lambda: torch.rand(T, generator=g, device="cuda", dtype=F64)
    it = float(torch.tensor(it, dtype=F32))
    x = torch.empty(T, 2, device="cuda")
    x[:, 1] = (rand() * 60 - 30) / it
    x[:, 0] = (x[:, 1].double() - rand() * depth / it).float()
    w = torch.exp((x[:, 0].double() - x[:, 1].double()) * it)
    near = (w / (1 + w)).float()
    for side in (-1, 0, 1):
        u = (near.view(I32) + side).view(F32)
        ids = sampling.sample(x, u, inv_temperature=torch.full((T,), it, device="cuda"))
        over = w * (1 - u.double()) / u.double() - 1
        room = 2 ** -28 + 2 ** -43 / w
        assert bool((ids[over > room] == 0).all()) and bool((ids[over < -room] == 1).all())
        if depth < 12 and not side:
            assert int(((over.abs() > room) & (over.abs() < 2 ** -26)).sum()) > 1000
    # weights of one value are the same
    x[:, 0] = x[:, 1]
    half = torch.full((T,), 0.5, device="cuda")
    below = (half.view(I32) - 1).view(F32)
    assert bool((sampling.sample(x, half) == 1).all()) and bool((sampling.sample(x, below) == 0).all())
