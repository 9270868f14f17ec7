"""Sampling from the whole vocabulary with given random numbers, against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from ironpangu_b200.ops import sampling

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
gpu = pytest.mark.gpu


def plain(logits, u, it=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Id and probability of one row: the documented definition, a token at a time where that matters."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64)) + 0.0
    if x.max() == -np.inf:
        return -1, 0.0
    if not (it > 0) or math.isinf(it):
        return int(x.argmax()), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp(x * it - x.max() * it)) if np.isfinite(x.max()) else (x == x.max()).astype(np.float64)
    order = np.argsort(-x, kind="stable")
    n = len(x)
    if 1 <= top_k < n:
        n = top_k
    if min_p > 0:
        n = min(n, max(1, int((w[order] >= min_p).sum())))
    if top_p < 1:
        mass = np.cumsum(w[order[:n]])
        ahead = np.concatenate([[0.0], mass[:-1]])
        n = max(1, int((ahead < top_p * mass[-1]).sum()))
    ids = np.sort(order[:n])
    run = np.cumsum(w[ids])
    past = run > (u * run[-1] if u > 0 else 0.0)
    at = int(past.argmax()) if past.any() else int(np.flatnonzero(w[ids])[-1])
    return int(ids[at]), float(w[ids[at]] / run[-1])


def check(logits, u, it=None, top_k=None, top_p=None, min_p=None):
    """`logits` on the device; the others lists or None. Probabilities: rounded once to f32 (2^-24 relative), of sums that are off by 2^-45 a token (V 2^-45 of at least 1)
    and 2^-30 of each weight, so of themselves."""
    T, V = logits.shape
    dev = lambda v, dt: None if v is None else torch.tensor(v, dtype=dt, device="cuda")
    args = dict(inv_temperature=dev(it, F32), top_k=dev(top_k, I32), top_p=dev(top_p, F32), min_p=dev(min_p, F32))
    ids, probs = sampling.sample(logits, dev(u, F32), probs=True, **args)
    ids, probs, x = ids.tolist(), probs.tolist(), logits.float().cpu().numpy()
    f = lambda v, t, other: other if v is None else float(np.float32(v[t]))
    for t in range(T):
        want, p = plain(x[t], f(u, t, 0), f(it, t, 1.0), 0 if top_k is None else top_k[t], f(top_p, t, 1.0), f(min_p, t, 0.0))
        assert ids[t] == want, f"row {t}: {ids[t]}, {want} wanted"
        assert abs(probs[t] - p) <= p * (2 ** -24 + V * 2 ** -45 + 2 ** -30), f"row {t}: probability {probs[t]}, {p} wanted"
    return ids


def some(T, V, seed, dtype=F32, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, V, generator=g, device="cuda") * spread
    x.scatter_add_(1, torch.randint(0, V, (T, 20), generator=g, device="cuda"), torch.rand(T, 20, generator=g, device="cuda") * 12)
    return x.to(dtype), torch.rand(T, generator=g, device="cuda").tolist()


CUTS = {"none": {}, "top_k": dict(top_k=50), "top_p": dict(top_p=0.9), "min_p": dict(min_p=0.05), "all": dict(top_k=300, top_p=0.8, min_p=0.01)}


@gpu
@pytest.mark.parametrize("cut", list(CUTS))
@pytest.mark.parametrize("T,V,dtype", [(1, 1, F32), (2, 2, BF16), (3, 7, F32), (5, 1000, BF16), (4, 1025, F32), (2, 8193, BF16), (3, 32000, F32), (9, 50257, BF16), (33, 151936, F32),
                                       (2, 1 << 18, F32)])
def test_definition(T, V, dtype, cut):
    x, u = some(T, V, T * 31 + V, dtype)
    check(x, u, it=[0.5 + 0.3 * (t % 5) for t in range(T)], **{k: [v] * T for k, v in CUTS[cut].items()})


@gpu
def test_rows_with_wishes_of_their_own():
    T = 24
    x, u = some(T, 40000, 5)
    check(x, u, it=[0.0, 1.0, -1.0, float("inf"), float("nan"), 1e-3, 1e4, 0.7] * 3, top_k=[0, 1, 5, 64, 65, 1000, 39999, 40000] * 3, top_p=[1.0, 0.5, 0.0, -1.0, 0.999999, 2.0, float("nan"), 0.9] * 3,
          min_p=[0.0, 0.0, 0.3, 1.0, 2.0, -1.0, float("nan"), 1e-30] * 3)


@gpu
@pytest.mark.parametrize("V", [5, 3000, 151936])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_equal_logits_go_by_rising_ids(V, dtype):
    u = [0.0, 0.25, 0.5, 0.75, 0.999]
    T = len(u)
    x = torch.full((T, V), 1.5, device="cuda", dtype=dtype)
    check(x, u)
    check(x, u, top_k=[1, 2, 3, V // 2, V - 1])
    check(x, u, top_p=[0.5, 0.25, 0.125, 0.9, 0.0])
    x[:, V // 2] = 1.75                            # one ahead of a great many
    check(x, u, top_k=[1, 2, 3, V // 2, V - 1], top_p=[0.5, 0.25, 0.125, 0.9, 0.0])
    check(x, u, min_p=[0.7, 0.78, 0.7788, 0.779, 1.0], it=[1.0] * T)


@gpu
def test_a_few_values_many_times():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-3, 4, (6, 60000), generator=g, device="cuda").float()
    check(x, [0.1, 0.3, 0.5, 0.7, 0.9, 0.99], top_k=[0, 10, 8571, 8600, 30000, 59999], top_p=[0.5, 1.0, 0.99, 0.6, 0.95, 0.3])


@gpu
def test_masked_and_infinite_logits():
    V, low, inf = 20000, torch.finfo(F32).min, float("inf")
    x = torch.full((9, V), -inf, device="cuda")
    x[1, 777] = 3.0                                # all but one masked
    x[2] = low                                     # masks of the type's lowest value, everywhere
    x[3] = low
    x[3, [5, 600, 19999]] = torch.tensor([1.0, 2.0, 0.5], device="cuda")
    x[4] = float("nan")
    x[5, ::7] = float("nan")
    x[5, 1::7] = torch.randn(len(range(1, V, 7)), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x[6] = torch.linspace(-1, 1, V)
    x[6, [17, 4000, 4001]] = inf
    x[7] = torch.linspace(low, torch.finfo(F32).max, V, dtype=torch.float64).float()
    x[8, 3], x[8, 9], x[8, 12] = 0.0, -0.0, 0.0
    u = [0.3, 0.4, 0.5, 0.6, 0.1, 0.7, 0.5, 0.9, 0.5]
    for kw in ({}, dict(top_k=[3] * 9), dict(top_k=[2] * 9), dict(top_p=[0.9] * 9), dict(min_p=[0.2] * 9), dict(it=[1e-38] * 9, top_p=[0.7] * 9), dict(it=[1e30] * 9)):
        check(x, u, **kw)
    assert sampling.sample(x, torch.rand(9, device="cuda"))[[0, 4]].tolist() == [-1, -1]
    with_low = x.to(BF16)
    check(with_low[:6], u[:6], top_p=[0.9] * 6)


@gpu
@pytest.mark.parametrize("T,V", [(3000, 61), (700, 1500), (297, 4096)])
def test_a_great_many_rows(T, V):
    x, u = some(T, V, T)
    check(x, u, it=[0.4 + 0.2 * (t % 7) for t in range(T)], top_k=[t % 50 for t in range(T)], top_p=[0.3 + 0.1 * (t % 9) for t in range(T)], min_p=[0.02 * (t % 3) for t in range(T)])


SHARES = [0.05, 0.3, 0.5, 0.8, 0.9, 0.99, 0.9999, 0.99999]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,spread,it", [(1 << 18, 0.5, 1.0), (1 << 18, 2.0, 0.05), (151936, 0.1, 1.0), (32000, 3.0, 0.01), (5000, 0.02, 1.0), (1 << 18, 2.0, 8.0), (40000, 1e-6, 1.0), (40000, 1e4, 1.0)])
def test_shares_that_end_among_many_tokens(V, spread, it, dtype):
    """Where the mass reaches the share, thousands of tokens lie close: more than one list takes, in f32 with values of their own."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(8, V, generator=g, device="cuda") * spread).to(dtype)
    u = torch.rand(8, generator=g, device="cuda").tolist()
    check(x, u, it=[it] * 8, top_p=SHARES)
    check(x, u, it=[it] * 8, top_p=SHARES[::-1], top_k=[V // 2, V // 3, 2000, 1500, 0, V - 1, V, 3])
    check(x, u, it=[it] * 8, top_p=SHARES, min_p=[0.9, 0.5, 0.1, 0.01, 1e-4, 0.99, 0.2, 0.0])


@gpu
def test_shares_of_values_that_are_nearly_equal():
    g = torch.Generator(device="cuda").manual_seed(9)
    steps = torch.randint(0, 40, (8, 60000), generator=g, device="cuda").float()
    x = 1 + steps * 2 ** -23                       # forty values side by side, 1500 tokens each
    check(x, [0.1, 0.2, 0.3, 0.4, 0.5, 0.6, 0.7, 0.999], top_p=SHARES)
    x[:, ::2] -= 30                                # half of them weigh nothing
    check(x, [0.1, 0.2, 0.3, 0.4, 0.5, 0.6, 0.7, 0.999], top_p=SHARES)
    x[:, 5] = 4.0
    check(x, [0.1, 0.2, 0.3, 0.4, 0.5, 0.6, 0.7, 0.999], top_p=SHARES, top_k=[20000] * 8)


@gpu
def test_random_numbers_at_and_beyond_their_ends():
    x, _ = some(6, 5000, 11)
    last = 1 - 2 ** -24
    check(x, [0.0, last, 1.0, 2.0, -1.0, float("inf")], top_p=[0.95] * 6)
    assert sampling.sample(x[:1], torch.tensor([float("nan")], device="cuda")).item() == sampling.sample(x[:1], torch.zeros(1, device="cuda")).item()


@gpu
def test_every_share_is_drawn():
    """Random numbers in the middle of each token's share draw that token."""
    V = 1000
    x = torch.randn(1, V, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    p = torch.softmax(x[0].double(), 0)
    middle = (torch.cumsum(p, 0) - p / 2).float()
    assert torch.equal(sampling.sample(x.expand(V, V).contiguous(), middle), torch.arange(V, device="cuda", dtype=I32))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_lie_anywhere(dtype):
    T, V = 4, 5003
    base = torch.full((T * 6001 + 5,), 50.0, device="cuda", dtype=dtype)          # what lies between the rows is not theirs
    for offset, pitch in ((1, 6001), (0, 6000), (3, 5003), (0, 5008)):
        x = base[offset:offset + T * pitch].as_strided((T, V), (pitch, 1))
        keep = base.clone()
        v, u = some(T, V, pitch, dtype)
        x.copy_(v)
        check(x, u, top_p=[0.9] * T)
        base.copy_(keep)


@gpu
def test_outputs_that_are_given_and_no_rows():
    x, u = some(3, 700, 1)
    ids, probs = torch.full((5,), -7, dtype=I32, device="cuda"), torch.full((5,), -7.0, device="cuda")
    a, b = sampling.sample(x, torch.tensor(u, device="cuda"), out_ids=ids[1:4], out_probs=probs[1:4])
    assert a.data_ptr() == ids[1:4].data_ptr() and b.data_ptr() == probs[1:4].data_ptr()
    assert ids[[0, 4]].tolist() == [-7, -7] and probs[[0, 4]].tolist() == [-7, -7] and int(ids[1:4].min()) >= 0
    assert sampling.sample(x[:0], torch.empty(0, device="cuda")).shape == (0,)


@gpu
def test_captured_and_on_another_stream():
    T, V = 5, 32000
    x, u = some(T, V, 7)
    u = torch.tensor(u, device="cuda")
    p = torch.full((T,), 0.9, device="cuda")
    ids = torch.empty(T, dtype=I32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = sampling.sample(x, u, top_p=p)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling.sample(x, u, top_p=p, out_ids=ids)
    graph.replay()
    assert torch.equal(ids, want) and torch.equal(sampling.sample(x, u, top_p=p), want)
    y, v = some(T, V, 8)
    x.copy_(y)
    u.copy_(torch.tensor(v))
    graph.replay()
    assert torch.equal(ids, sampling.sample(y, torch.tensor(v, device="cuda"), top_p=p))


@gpu
def test_results_do_not_change_from_call_to_call():
    x, u = some(40, 100003, 13, spread=0.5)
    u = torch.tensor(u, device="cuda")
    p = torch.full((40,), 0.97, device="cuda")
    first = sampling.sample(x, u, top_p=p, probs=True)
    for _ in range(5):
        again = sampling.sample(x, u, top_p=p, probs=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refused_on_the_host():
    x, u = torch.zeros(2, 8), torch.zeros(2)
    with pytest.raises(ValueError, match="on the host"):
        sampling.sample(x, u)
    with pytest.raises(ValueError, match="f32 or bf16"):
        sampling.sample(x.double(), u)
    with pytest.raises(ValueError, match="f32 or bf16"):
        sampling.sample(x[0], u)


@gpu
def test_refused():
    x, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    for bad, what in ((dict(logits=x.half()), "f32 or bf16"), (dict(logits=x.T), "one behind the other"), (dict(logits=x[:1].expand(2, 8)), "lie apart"),
                      (dict(logits=torch.empty(1, (1 << 18) + 1, device="cuda"), uniforms=u[:1]), "not supported"), (dict(uniforms=u[:1]), "uniforms"), (dict(uniforms=u.double()), "uniforms"),
                      (dict(uniforms=u.cpu()), "uniforms"), (dict(uniforms=None), "uniforms"), (dict(top_k=u), "top_k"), (dict(top_p=torch.zeros(2, 2, device="cuda")[:, 0]), "top_p"), (dict(min_p=u.int()), "min_p"),
                      (dict(inv_temperature=u[:1]), "inv_temperature"), (dict(out_ids=u), "out_ids"), (dict(out_probs=u.int()), "out_probs")):
        with pytest.raises(ValueError, match=what):
            sampling.sample(**{**dict(logits=x, uniforms=u), **bad})
