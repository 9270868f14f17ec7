"""Scales of the attention over shared prefixes at the ends of what f32 holds."""
import math

import pytest
import torch

from ironpangu_b200.ops import shared_prefix as S

BF16, I32 = torch.bfloat16, torch.int32


@pytest.mark.gpu
def test_scales():
    i32 = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(*s, generator=g, device="cuda").to(BF16) for s in ((3, 512), (2, 16, 2, 64), (2, 16, 2, 64)))
    args = (k, v, i32([19, 20, 24]), i32([0, 0, 0]), i32([[0, 1]]), i32([[0, 3, 18, 0]]))
    run = lambda scale, q=q: S.attention(q, *args, heads=8, kv_heads=2, head_dim=64, scale=scale)
    for scale in (0.0, -1.0, math.nan, math.inf, -math.inf, 1e39, 2.4e38, 3e38, 1e-46, 1e-300):
        with pytest.raises(ValueError, match="a scale of"):
            run(scale)
    # the largest one that is taken: nothing but the largest score weighs; the smallest: all weigh alike
    hot = run(2.35e38, q * 2.0 ** -120)
    assert torch.equal(hot, run(2.35e38 * 2.0 ** -120))
    rows = torch.cat([v[0], v[1]]).double()
    for t, n in enumerate((20, 21, 25)):
        want = rows[:n].mean(0).repeat_interleave(4, 0).reshape(-1)
        assert bool(((run(1.5e-45)[t].double() - want).abs() <= want.abs() * 2 ** -8 + rows[:n].abs().mean(0).repeat_interleave(4, 0).reshape(-1) * 2 ** -14).all())
