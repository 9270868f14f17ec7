"""Outputs of the attention over shared prefixes that lie over what it reads."""
import pytest
import torch

from ironpangu_b200.ops import shared_prefix as S

BF16, I32 = torch.bfloat16, torch.int32
gpu = pytest.mark.gpu


def _case(rows, heads=8, kv=2, dim=64, shared=100, page=16):
    g = torch.Generator(device="cuda").manual_seed(rows)
    n = -(-(shared + 4) // page)
    k, v = (torch.randn(n, page, kv, dim, generator=g, device="cuda").to(BF16) for _ in range(2))
    i32 = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    rest = (k, v, torch.full((rows,), shared + 3, dtype=I32, device="cuda"), i32([0] * rows), torch.arange(n, dtype=I32, device="cuda").view(1, n), i32([[0, rows, shared, 0]]))
    return torch.randn(rows, heads * dim, generator=g, device="cuda").to(BF16), rest, dict(heads=heads, kv_heads=kv, head_dim=dim, scale=dim ** -0.5)


@gpu
@pytest.mark.parametrize("rows", [5, 230, 700])
def test_over_the_queries(rows):
    q, rest, kw = _case(rows)
    want = S.attention(q, *rest, **kw)
    wide = torch.zeros(rows + 1, 1600, dtype=BF16, device="cuda")
    for first, ok in ((0, True), (512, True), (1088, True), (8, False), (504, False), (511, False)):
        wide[:rows, :512] = q
        out = wide[:rows, first:first + 512]
        if not ok:
            with pytest.raises(ValueError, match="overlap"):
                S.attention(wide[:rows, :512], *rest, out=out, **kw)
            assert torch.equal(wide[:rows, :512], q)
            continue
        S.attention(wide[:rows], *rest, out=out, **kw)
        assert torch.equal(out, want)
    for out in (wide[1:, :512], wide[1:, 504:1016], wide.view(-1)[512:].as_strided((rows, 512), (512, 1))):
        wide[:rows, :512] = q
        with pytest.raises(ValueError, match="overlap"):
            S.attention(wide[:rows, :512], *rest, out=out, **kw)
        assert torch.equal(wide[:rows, :512], q)


@gpu
def test_over_the_rest():
    rows = 4
    q, rest, kw = _case(rows)
    k, v = rest[0], rest[1]
    ints = torch.zeros(4096, dtype=I32, device="cuda")
    ints[:4] = rest[2]
    scratch = torch.zeros(S.scratch_bytes(rows, 8, 2, 64) + 8192, dtype=torch.uint8, device="cuda")
    cover = lambda t: t.view(-1).view(BF16)[:rows * 512].view(rows, 512)
    for bad in (dict(out=cover(k)), dict(out=cover(v)), dict(out=cover(scratch), scratch=scratch[:-8192]), dict(out=cover(scratch[-8192:]), scratch=scratch)):
        with pytest.raises(ValueError, match="overlap"):
            S.attention(q, *rest, **bad, **kw)
    with pytest.raises(ValueError, match="overlap"):
        S.attention(q, k, v, ints[:4], *rest[3:], out=cover(ints), **kw)
    want = S.attention(q, *rest, **kw)
    assert torch.equal(S.attention(q, *rest, out=cover(scratch[-8192:]), scratch=scratch[:-8192], **kw), want)
