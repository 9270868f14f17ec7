"""Results of sampling in the place of what it reads, and over it."""
import pytest
import torch

from ironpangu_b200.ops import sampling

F32, I32 = torch.float32, torch.int32
gpu = pytest.mark.gpu


def _case(T, V, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, V, generator=g, device="cuda") * 2
    return x, torch.rand(T, generator=g, device="cuda"), torch.randint(1, 500, (T,), generator=g, device="cuda").to(I32), torch.rand(T, generator=g, device="cuda") * 0.5 + 0.45


@gpu
@pytest.mark.parametrize("T,V", [(1, 151936), (16, 151936), (37, 40000), (300, 3001)])
def test_in_the_place_of_the_rows_values(T, V):
    """Eight CTAs a row read its random number, and one of them writes."""
    x, u, k, p = _case(T, V, T)
    ids, probs = sampling.sample(x, u, top_k=k, top_p=p, probs=True)
    for _ in range(50):
        a, b, c = u.clone(), k.clone(), p.clone()
        sampling.sample(x, a, top_k=b, top_p=c, out_ids=b, out_probs=a)
        assert torch.equal(b, ids) and torch.equal(a, probs) and torch.equal(c, p)
        a, b = u.clone(), k.clone()
        sampling.sample(x, a, top_k=b, top_p=p, out_ids=a.view(I32))
        assert torch.equal(a.view(I32), ids) and torch.equal(b, k)
        c = p.clone()
        sampling.sample(x, u, top_k=k, top_p=c, out_probs=c)
        assert torch.equal(c, probs)


@gpu
def test_refused_over_what_is_read_or_written():
    T, V = 6, 1000
    x, u, k, p = _case(T, V, 5)
    both = torch.zeros(3 * T, device="cuda")
    both[1:T + 1] = u
    shifted, ints = both[1:T + 1], both.view(I32)
    wide = torch.zeros(T, V + T, device="cuda")
    wide[:, :V] = x
    for kw in (dict(uniforms=shifted, out_probs=both[:T]), dict(uniforms=shifted, out_probs=both[2:T + 2]), dict(uniforms=shifted, out_ids=ints[T:2 * T]), dict(uniforms=u, top_p=shifted, out_ids=ints[:T]),
               dict(uniforms=u, out_ids=ints[:T], out_probs=both[:T]), dict(uniforms=u, out_ids=ints[:T], out_probs=both[T - 1:2 * T - 1]), dict(uniforms=u, out_probs=x[2, 10:10 + T]),
               dict(uniforms=u, out_ids=x[T - 1].view(I32)[V - T:])):
        with pytest.raises(ValueError, match="overlap"):
            sampling.sample(x, **kw)
    for kw in (dict(out_probs=wide[0, V - 1:V + T - 1]), dict(out_probs=wide.view(-1)[V + 1:V + T + 1]), dict(out_ids=wide[1].view(I32)[:T])):
        with pytest.raises(ValueError, match="overlap"):
            sampling.sample(wide[:, :V], u, **kw)
    want = sampling.sample(x, u, probs=True)
    for out_ids, out_probs in ((ints[:T], both[T:2 * T]), (wide[0, V:].view(I32), wide[3, V:]), (ints[2 * T:], None), (None, both[T:2 * T])):
        got = sampling.sample(wide[:, :V], u, out_ids=out_ids, out_probs=out_probs, probs=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(wide[:, :V], x)


@gpu
def test_refused_over_rows_that_are_one():
    x, u, _, _ = _case(1, 64, 2)
    one = x.expand(3, 64)
    with pytest.raises(ValueError, match="lie apart"):
        sampling.sample(one, u.expand(3).contiguous(), out_probs=x[0, :3])
