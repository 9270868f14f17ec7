"""As many rows as a call takes."""
import pytest
import torch

from ironpangu_b200.ops import sampling, shared_prefix

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32
pytestmark = pytest.mark.gpu
MOST = 1 << 20


def test_sampling():
    g = torch.Generator(device="cuda").manual_seed(1)
    x, u = torch.randn(MOST, 3, generator=g, device="cuda"), torch.rand(MOST, generator=g, device="cuda")
    ids, probs = sampling.sample(x, u, probs=True)
    p = torch.softmax(x.double(), 1)
    # borders apart by what weights may be off (2^-28 of themselves) and the definition's own rounding here
    low, high = (torch.cumsum(p, 1) - p).gather(1, ids.long()[:, None])[:, 0], torch.cumsum(p, 1).gather(1, ids.long()[:, None])[:, 0]
    assert bool(((u.double() >= low - 2 ** -27) & (u.double() <= high + 2 ** -27)).all())
    assert bool(((probs.double() - p.gather(1, ids.long()[:, None])[:, 0]).abs() <= 2 ** -23 * probs.double()).all())
    with pytest.raises(ValueError, match="not supported"):
        sampling.sample(torch.zeros(MOST + 1, 1, device="cuda"), torch.zeros(MOST + 1, device="cuda"))


def test_attention():
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(9, 16, 1, 64, generator=g, device="cuda").to(BF16) for _ in range(2))
    q = torch.randn(MOST, 64, generator=g, device="cuda").to(BF16)
    positions = torch.randint(99, 144, (MOST,), generator=g, device="cuda").to(I32)
    i32 = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    args = (k, v, positions, torch.zeros(MOST, dtype=I32, device="cuda"), torch.arange(9, dtype=I32, device="cuda").view(1, 9))
    kw = dict(heads=1, kv_heads=1, head_dim=64, scale=0.125)
    out = shared_prefix.attention(q, *args, i32([[0, MOST, 100, 0]]), **kw)
    keys, values = k.view(-1, 64).double(), v.view(-1, 64).double()
    for rows in (slice(0, 2000), slice(MOST // 2, MOST // 2 + 2000), slice(MOST - 2000, MOST)):
        z = (q[rows].double() @ keys.T * 0.125).masked_fill(torch.arange(144, device="cuda") > positions[rows, None], -torch.inf)
        w = torch.softmax(z, 1)
        # rounded once, 15-bit weights
        assert bool(((out[rows].double() - w @ values).abs() <= (w @ values).abs() * 2 ** -8 + w @ values.abs() * 2 ** -14).all())
    del out
    with pytest.raises(ValueError, match="not supported"):
        shared_prefix.scratch_bytes(MOST + 1, 1, 1, 64)
