"""Linears with 4-bit weights against 64 bits: groups, zero points, scales in both types, gated matrices, norms, residuals; widths and lengths that no tile divides; rows
that no launch holds at once. Beyond sixteen rows a weight has the 11 bits of f16, and the reference rounds it too. Bounds: products of a group are exact in f32 and added by tensor cores that cut off, at worst 17 addends a product and 8 products a group at
2^-23 of the group's sum of magnitudes: 2^-16 of it (a whole row of K in one chain: 2^-23 of it a product, K / 16 of them); the result's rounding to bf16 is 2^-8 of the value."""
import pytest
import torch

BF16, F16 = torch.bfloat16, torch.float16
CUT = 2.0 ** -16


def _codes(rows, k, group, zeros, seed, f16=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-k // group)
    q = torch.randint(0, 16, (rows, k), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand(rows, groups, generator=g, device="cuda") * 0.01 + 0.001).to(F16 if f16 else BF16)
    z = torch.randint(0, 16, (rows, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return q, s, z


def _values(q, s, z, group):
    at = torch.arange(q.shape[1], device=q.device) // group
    return (q.double() - (8 if z is None else z.double()[:, at])) * s.double()[:, at]


def _operands(v, x):
    """Weights as the products have them, and the bound of their sums."""
    if x.shape[0] > 16:
        m, e = torch.frexp(v)                            # scales of a row are within a factor of 16 here: no weight is below f16's normal range
        v = torch.ldexp(torch.round(m * 2 ** 11) / 2 ** 11, e)
    return v, (x.double().abs() @ v.abs().T) * (CUT if x.shape[0] <= 16 else max(CUT, 17 * x.shape[1] / 16 * 2.0 ** -23))


def _rows(T, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, k + 8, generator=g, device="cuda").to(BF16)[:, :k]


def _close(out, want, bound):
    bad = ~((out.double() - want).abs() <= bound)
    assert not bool(bad.any()), (int(bad.sum()), float(((out.double() - want).abs() - bound).max()))


# -- refusals, on any machine -----------------------------------------------------------------------------------------------
def test_refusals_without_a_device():
    from ironpangu_b200.ops import int4

    w = torch.zeros(16, 64, dtype=BF16)
    with pytest.raises(ValueError, match="on the device"):
        int4.quantise(w)
    for rows, k, kw, what in ((16, 60, {}, "eights"), (0, 64, {}, "not supported"), (16, 64, dict(group=48), "groups of 48"), (15, 64, dict(gated=True), "gate and up")):
        with pytest.raises(ValueError, match=what):
            int4.Int4Weight(rows, k, device="cpu", **kw)
    h = int4.Int4Weight(33, 136, group=64, zeros=True, device="cpu")
    assert h.nbytes == 3 * (2 * (1024 + 2 * 48) + 64) and h.n == 33
    x = torch.zeros(2, 136, dtype=BF16)
    for bad, kw, what in ((x.float(), {}, "rows must be bf16"), (x[:, :128], {}, "rows must be bf16"), (torch.zeros(2, 140, dtype=BF16)[:, :136], {}, "16 bytes"),
                          (torch.zeros(9, 136, dtype=BF16), dict(norm_w=torch.ones(136, dtype=BF16)), "a launch of its own"), (x, dict(norm_w=torch.ones(136)), "gains"),
                          (x, dict(residual=torch.zeros(2, 32, dtype=BF16)), "residual"), (x, dict(out=torch.zeros(2, 33, dtype=F16)), "output")):
        with pytest.raises(ValueError, match=what):
            int4.linear(bad, h, **kw)
    with pytest.raises(ValueError, match="no residual"):
        int4.linear(torch.zeros(1, 64, dtype=BF16), int4.Int4Weight(32, 64, gated=True, device="cpu"), residual=torch.zeros(1, 16, dtype=BF16))
    assert int4.linear(torch.zeros(0, 136, dtype=BF16), h).shape == (0, 33)
    q, s = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 1, dtype=BF16)
    with pytest.raises(ValueError, match="on the device"):
        int4.pack(q, s)


# -- on the device ----------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,k,gated", [(1, 8, False), (17, 72, False), (40, 136, False), (64, 256, True), (70, 1000, True)])
def test_pack_and_back(rows, k, gated, zeros, group):
    from ironpangu_b200.ops import int4

    for f16 in (False, True):
        q, s, z = _codes(rows, k, group, zeros, rows + k, f16)
        w = int4.pack(q, s, z, group=group, gated=gated)
        assert w.nbytes == w.units.numel() and w.rows == rows
        out = torch.full((rows + 1, k + 8), 7.0, dtype=BF16, device="cuda")
        w.dequantise(out[:rows, :k])
        assert torch.equal(out[:rows, :k], _values(q, s, z, group).to(BF16))         # 4 bits by 8 or 11: exact in f32, rounded once
        assert bool((out[rows:] == 7).all()) and bool((out[:, k:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,k,gated", [(3, 24, False), (130, 264, True), (257, 2048, False)])
def test_quantise(rows, k, gated, zeros, group):
    from ironpangu_b200.ops import int4

    g = torch.Generator(device="cuda").manual_seed(rows)
    w = (torch.randn(rows, k + 8, generator=g, device="cuda") * 0.02).to(BF16)[:, :k]
    w[0] = 0                                             # a group of zeros
    w[1] = torch.arange(k, device="cuda") % 15 - 7.0     # symmetric: s = 1; without ties
    w[2] = (torch.arange(k, device="cuda") % 2) * 0.5 + 0.25        # of one sign
    f = torch.nn.functional.pad(w.double(), (0, -k % group)).view(rows, -1, group)
    if zeros:
        lo, hi = f.amin(-1).clamp(max=0), f.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).float().to(BF16).double()
    else:
        s = (f.abs().amax(-1) / 7).float().to(BF16).double()
    s = torch.where(s == 0, 1.0, s)[..., None]
    z = torch.round(-lo[..., None] / s).clamp(0, 15) if zeros else 8
    q = (torch.round(f / s) + z).clamp(0, 15)
    want = ((q - z) * s).reshape(rows, -1)[:, :k].to(BF16)
    h = int4.quantise(w, group=group, zeros=zeros, gated=gated)
    assert torch.equal(h.dequantise(), want)
    # within half a step of the matrix, but for what the scale's rounding to bf16 clips at the ends
    if group == 128 and not zeros:
        step = s.expand_as(f).reshape(rows, -1)[:, :k]
        assert bool(((want.double() - w.double()).abs() <= step * (0.5 + 7 * 2.0 ** -8) + want.double().abs() * 2.0 ** -8).all())


@pytest.mark.gpu
def test_quantise_groups_without_a_value():
    from ironpangu_b200.ops import int4

    w = torch.randn(20, 256, device="cuda").to(BF16)
    w[3, 5], w[4, 200], w[7, 130] = float("nan"), float("inf"), float("-inf")
    for zeros in (False, True):
        back = int4.quantise(w, group=128, zeros=zeros).dequantise()
        nan = torch.zeros(20, 2, dtype=torch.bool, device="cuda")
        nan[3, 0] = nan[4, 1] = nan[7, 1] = True
        assert torch.equal(back.isnan().view(20, 2, 128).all(-1), nan) and torch.equal(back.isnan().view(20, 2, 128).any(-1), nan)
        y = int4.linear(torch.ones(1, 256, device="cuda", dtype=BF16), int4.quantise(w, group=128, zeros=zeros))
        assert torch.equal(y[0].isnan(), nan.any(-1))


SHAPES = [(1, 8, 1), (16, 128, 1), (17, 72, 2), (1, 4096, 3), (300, 1032, 5), (1024, 1024, 1), (2741, 2056, 3), (2368, 264, 8), (5000, 136, 7), (64, 16392, 8), (200, 9000, 2),
          (48, 640, 9), (333, 2056, 16), (70, 9000, 13), (130, 520, 21), (40, 264, 67), (1, 8, 17), (1237, 1032, 129), (5000, 136, 203), (333, 9000, 40), (129, 4096, 255), (300, 640, 1000), (5000, 520, 700), (2741, 1032, 1501), (9500, 136, 300), (18000, 72, 140)]


@pytest.mark.gpu
@pytest.mark.parametrize("group,zeros,f16", [(128, False, False), (128, True, False), (64, False, True), (64, True, False), (32, False, False), (32, True, True)])
@pytest.mark.parametrize("N,K,T", SHAPES)
def test_linear(N, K, T, group, zeros, f16):
    from ironpangu_b200.ops import int4

    q, s, z = _codes(N, K, group, zeros, N + K, f16)
    w, x = int4.pack(q, s, z, group=group), _rows(T, K, T)
    v, scale = _operands(_values(q, s, z, group), x)
    want = x.double() @ v.T
    out = torch.full((T + 1, N + 3), 7.0, device="cuda")
    int4.linear(x, w, out=out[:T, :N])
    _close(out[:T, :N], want, scale + 1e-30)
    assert bool((out[T:] == 7).all()) and bool((out[:, N:] == 7).all())
    y = _rows(T, N + (-N) % 8, 3)[:, :N].contiguous()
    res = y.double()
    int4.linear(x, w, residual=y, out=y)                 # in place
    _close(y, want + res, scale + 2.0 ** -8 * (want + res).abs() + 1e-30)
    assert int4.linear(x, w).dtype == BF16 and int4.linear(x, w, out_f32=True).dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("group,zeros", [(128, False), (64, True), (32, True)])
@pytest.mark.parametrize("F,K,T", [(1, 8, 1), (17, 264, 3), (150, 1544, 8), (3000, 512, 1), (16, 4096, 11), (1237, 1032, 5), (96, 520, 33), (1, 8, 17), (1237, 1032, 130), (65, 9000, 20), (200, 2048, 600), (1237, 520, 1101), (5000, 264, 333), (2736, 1160, 500)])
def test_gated(F, K, T, group, zeros):
    from ironpangu_b200.ops import int4

    q, s, z = _codes(2 * F, K, group, zeros, F + K)
    w, x = int4.pack(q, s, z, group=group, gated=True), _rows(T, K, T)
    v, scale = _operands(_values(q, s, z, group), x)
    y = x.double() @ v.T
    gate, up, a, b = y[:, :F], y[:, F:], scale[:, :F], scale[:, F:]
    want = gate * torch.sigmoid(gate) * up
    out = torch.full((T + 1, F + 3), 7.0, dtype=BF16, device="cuda")
    int4.linear(x, w, out=out[:T, :F])
    # the unit's slope is at most 1.1; its exponential and quotient are off by a few steps of f32
    _close(out[:T, :F], want, (2.0 ** -8 + 2.0 ** -20) * want.abs() + 1.1 * a * (up.abs() + b) + (gate.abs() + a) * b + 1e-30)
    assert bool((out[T:] == 7).all()) and bool((out[:, F:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,T", [(33, 8, 1), (1024, 1024, 1), (300, 1032, 8), (130, 9000, 3), (64, 20000, 8)])
def test_norm_ahead(N, K, T):
    from ironpangu_b200.ops import int4

    q, s, z = _codes(N, K, 64, True, N + K)
    w, v, x = int4.pack(q, s, z, group=64), _values(q, s, z, 64), _rows(T, K, T)
    gain = (torch.randn(K, device="cuda") * 0.1 + 1).to(BF16)
    xn = (x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-6) * gain.double()).to(BF16).double()
    want, scale = xn @ v.T, xn.abs() @ v.abs().T
    out = int4.linear(x, w, norm_w=gain, eps=1e-6, out_f32=True)
    # an f32 norm rounds to the other bf16 value (2^-7 of it) where it ends within some 2^-21 of their border: one operand of 2^13, four more allowed
    flips = (4 + K // 1024) * 2.0 ** -7 * float((xn.abs().amax() * v.abs().amax()))
    _close(out, want, CUT * scale + flips)
    alone = torch.cat([int4.linear(x[t:t + 1], w, norm_w=gain, eps=1e-6, out_f32=True) for t in range(T)])
    assert torch.equal(out, alone)                       # the bits that a row has alone


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(500, 1160), (300, 4104), (100, 20000)])
def test_rows_beside_a_row_change_nothing(N, K):
    from ironpangu_b200.ops import int4

    q, s, z = _codes(N, K, 128, False, 5)
    w, x = int4.pack(q, s, z, group=128), _rows(16, K, 1)
    alone = torch.cat([int4.linear(x[t:t + 1], w) for t in range(16)])
    for T in (2, 8, 9, 16):
        assert torch.equal(int4.linear(x[:T], w), alone[:T])
    x[1] = float("nan")
    x[2, 7] = float("inf")
    y = int4.linear(x, w)
    assert torch.equal(y[0], alone[0]) and torch.equal(y[3:], alone[3:]) and bool(y[1].isnan().all()) and not bool(y[2].isfinite().any())


@pytest.mark.gpu
def test_streams_and_graphs():
    """A captured linear, replayed on other rows; the matrix packed on another stream; the row ahead of it written by a kernel of the same stream."""
    from ironpangu_b200.ops import int4

    q, s, z = _codes(600, 2048, 128, True, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w = int4.pack(q, s, z, group=128)
        x = _rows(4, 2048, 1).contiguous()
        first = int4.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(int4.linear(x, w), first)
    out = torch.empty(4, 600, dtype=BF16, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        int4.linear(x * 2, w, out=out)
    for seed in (3, 4):
        x.copy_(_rows(4, 2048, seed))
        g.replay()
        assert torch.equal(out, int4.linear(x * 2, w))
    for _ in range(20):                                  # a matrix that the launch ahead has just packed
        m = torch.randn(600, 2048, device="cuda").to(BF16)
        h = int4.quantise(m)
        got = int4.linear(x, h)
        torch.cuda.synchronize()
        assert torch.equal(got, int4.linear(x, h))


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,gated", [(300, 700, False), (1300, 4100, False), (1300, 2052, True)])
def test_a_wait_that_runs_out(T, N, gated):
    """With a limit of no polls every warp gives up at its first wait: the status word says so, the result is NaN and the next call is right."""
    from ironpangu_b200.ops import _lib, int4

    K = 2048
    q, s, z = _codes(N * (1 + gated), K, 128, False, 1)
    w, x = int4.pack(q, s, z, group=128, gated=gated), _rows(T, K, 1).contiguous()
    want = int4.linear(x, w)
    scratch = torch.empty(_lib.load().ifab_int4_gemm_scratch(T, K), dtype=torch.uint8, device="cuda")
    status, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(T, N, dtype=BF16, device="cuda")
    _lib.check(_lib.load().ifab_int4_gemm(w.ref, x.data_ptr(), K, None, 0, out.data_ptr(), N, 0, T, scratch.data_ptr(), 0, status.data_ptr(), torch.cuda.current_stream().cuda_stream),
               "gemm")
    torch.cuda.synchronize()
    assert int(status) == 2 and bool(out.isnan().all())
    status.zero_()
    assert torch.equal(int4.linear(x, w, status_ptr=status.data_ptr()), want) and int(status) == 0


@pytest.mark.gpu
def test_ranges_of_rows_and_scales():
    """Many rows: scales and rows of x of any magnitude, an infinity or NaN in one row of x, a scale of NaN in one row of the matrix."""
    from ironpangu_b200.ops import int4

    g = torch.Generator(device="cuda").manual_seed(4)
    N, K, T = 150, 520, 40
    q, s, z = _codes(N, K, 64, True, 7)
    rowwise, token = torch.linspace(-30, 30, N, device="cuda"), torch.linspace(-60, 60, T, device="cuda")
    s = (s.double() * torch.exp2(rowwise.round().double())[:, None]).to(BF16)
    x = (torch.randn(T, K, generator=g, device="cuda").double() * torch.exp2(token.round().double())[:, None]).to(BF16)
    x[:, 7] *= 2.0 ** -20                                # far below its row's largest
    v = _values(q, s, z, 64)
    w = int4.pack(q, s, z, group=64)
    out = int4.linear(x, w, out_f32=True)
    v, bound = _operands(v, x)
    _close(out, x.double() @ v.T, bound)
    s[5, 3] = float("nan")
    x[3, 9], x[4, 10], x[6] = float("inf"), float("nan"), 0
    bad = int4.linear(x, int4.pack(q, s, z, group=64), out_f32=True)
    keep_n, keep_t = torch.ones(N, dtype=torch.bool, device="cuda"), torch.ones(T, dtype=torch.bool, device="cuda")
    keep_n[5], keep_t[3], keep_t[4], keep_t[6] = False, False, False, False
    assert torch.equal(bad[keep_t][:, keep_n], out[keep_t][:, keep_n]) and bool(bad[:, 5].isnan().all())
    assert not bool(bad[3].isfinite().any()) and bool(bad[4].isnan().all()) and bool((bad[6, keep_n] == 0).all())
    tiny = torch.full((20, K), 2.0 ** -133, dtype=BF16, device="cuda")
    y, scale = int4.linear(tiny, w, out_f32=True), tiny.double().abs() @ v[:20].abs().T
    # the smallest bf16 numbers: a result below f32's normal range has steps of 2^-149
    _close(y, tiny.double() @ v.T, _operands(v, tiny)[1] + 2.0 ** -148)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [20, 140, 250])
@pytest.mark.parametrize("N", [260, 2100, 3300, 4500, 5800, 7700, 12100])
def test_shares_of_k_of_any_number(N, T):
    """Widths whose tiles leave K to one, two, three ... CTAs of a cluster."""
    test_linear(N, 2056, T, 64, True, False)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,gated", [(60, 300, False), (128, 9000, True), (129, 300, True), (250, 9000, False)])
def test_a_wait_that_runs_out_of_fewer_rows(T, N, gated):
    test_a_wait_that_runs_out(T, N, gated)


@pytest.mark.gpu
def test_where_matrices_and_rows_lie():
    """Rows that lie too near, off 16 bytes or over one another are refused before anything is launched; of a single row the stride says nothing."""
    from ironpangu_b200.ops import int4

    m = torch.randn(40, 272, device="cuda").to(BF16)
    for bad in (m[:, :268].reshape(-1)[:40 * 268].view(40, 268)[:, :264], m[:, 4:268], m[:1, :264].expand(40, 264), m[:0, :264]):
        with pytest.raises(ValueError, match="rows must lie|not supported"):
            int4.quantise(bad)
    w = int4.quantise(m[:, :264])
    one = torch.as_strided(m, (1, 264), (3, 1))
    assert torch.equal(int4.quantise(one).dequantise(), w.dequantise()[:1])
    with pytest.raises(ValueError, match="rows must lie"):
        w.dequantise(torch.empty(40, 268, dtype=BF16, device="cuda")[:, :264])
    q, s, z = _codes(40, 264, 64, False, 0)
    for args, group, what in (((q[:1].expand(40, 264), s), 64, "one behind the other"), ((q, s), 0, "groups of 0"), ((q, s), 48, "groups of 48")):
        with pytest.raises(ValueError, match=what):
            int4.pack(*args, group=group)
    x = torch.randn(4, 272, device="cuda").to(BF16)
    with pytest.raises(ValueError, match="16 bytes"):
        int4.linear(x[:, 1:265], w)
    with pytest.raises(ValueError, match="16 bytes"):
        int4.linear(x.reshape(-1)[:4 * 268].view(4, 268)[:, :264], w)
    assert torch.equal(int4.linear(torch.as_strided(x, (1, 264), (3, 1)), w), int4.linear(x[:1, :264], w))
    square = int4.quantise(torch.randn(264, 264, device="cuda").to(BF16))
    y = x[:, :264].contiguous()
    with pytest.raises(ValueError, match="overlap"):
        int4.linear(y, square, out=y)
    assert torch.equal(int4.linear(y, square, residual=(r := y.clone()), out=r), int4.linear(y, square, residual=y))


def test_weights_on_the_host_multiply_nothing():
    from ironpangu_b200.ops import int4

    with pytest.raises(ValueError, match="on the host"):
        int4.linear(torch.zeros(1, 64, dtype=BF16), int4.Int4Weight(16, 64, device="cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K,norm,gated", [(1, 64, 1024, False, False), (1, 9000, 4104, True, True), (3, 300, 16392, False, False), (8, 30000, 2056, True, False), (16, 5000, 9000, False, True), (11, 100, 520, False, False)])
def test_a_copy_that_does_not_land_in_time(T, N, K, norm, gated):
    """Few rows, with a limit of no polls: every warp gives up at its first wait, the copies under way are waited for, the status word says so, the result is NaN and the next
    call is right."""
    from ironpangu_b200.ops import _lib, int4

    q, s, z = _codes(N * (1 + gated), K, 32, True, 1)
    w, x, gain = int4.pack(q, s, z, group=32, gated=gated), _rows(T, K, 1).contiguous(), torch.ones(K, dtype=BF16, device="cuda")
    want = int4.linear(x, w, norm_w=gain if norm else None)
    for _ in range(3):
        status, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(T, N, dtype=BF16, device="cuda")
        _lib.check(_lib.load().ifab_int4_rows(w.ref, x.data_ptr(), K, gain.data_ptr() if norm else None, 1e-5, None, 0, out.data_ptr(), N, 0, T, 0, status.data_ptr(),
                                              torch.cuda.current_stream().cuda_stream), "rows")
        torch.cuda.synchronize()
        assert int(status) == 2 and bool(out.isnan().all())
        status.zero_()
        assert torch.equal(int4.linear(x, w, norm_w=gain if norm else None, status_ptr=status.data_ptr()), want) and int(status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,gated", [(1300, 4100, False), (1300, 2052, True), (700, 9500, False)])
def test_launches_right_behind_one_that_gave_up(T, N, gated):
    """Pairs of SMs whose waits run out, and products of other rows behind them without the host between: nothing that was signalled or copied for the first meets the second."""
    from ironpangu_b200.ops import _lib, int4

    K = 1160
    q, s, z = _codes(N * (1 + gated), K, 64, True, 1)
    w, x, few = int4.pack(q, s, z, group=64, gated=gated), _rows(T, K, 1).contiguous(), _rows(200, K, 2).contiguous()
    want, want_few = int4.linear(x, w), int4.linear(few, w)
    scratch = torch.empty(_lib.load().ifab_int4_gemm_scratch(T, K), dtype=torch.uint8, device="cuda")
    status, out = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(T, N, dtype=BF16, device="cuda")
    for _ in range(3):
        _lib.check(_lib.load().ifab_int4_gemm(w.ref, x.data_ptr(), K, None, 0, out.data_ptr(), N, 0, T, scratch.data_ptr(), 0, status.data_ptr(),
                                              torch.cuda.current_stream().cuda_stream), "gemm")
        a, b = int4.linear(few, w), int4.linear(x, w)
        assert torch.equal(a, want_few) and torch.equal(b, want) and int(status) == 2 and bool(out.isnan().all())
        status.zero_()


def test_weights_on_the_host_have_no_values():
    from ironpangu_b200.ops import int4

    w = int4.Int4Weight(16, 64, device="cpu")
    for out in (None, torch.zeros(16, 64, dtype=BF16)):
        with pytest.raises(ValueError, match="on the host"):
            w.dequantise(out)


EXACT = [(200, 16392, 1), (333, 9000, 3), (64, 16392, 8), (48, 9000, 16), (130, 9000, 17), (333, 9000, 40), (1237, 4104, 64), (300, 16392, 129), (129, 4096, 255), (1000, 9000, 300), (2741, 4104, 700),
         (9500, 4104, 300), (5000, 2056, 1101)]


@pytest.mark.gpu
@pytest.mark.parametrize("group,zeros", [(128, True), (64, False), (32, True)])
@pytest.mark.parametrize("N,K,T", EXACT)
def test_sums_without_any_rounding(N, K, T, group, zeros):
    """Small integers and scales of 1/2, 1 and 2: products are multiples of 1/2 and the sums of their magnitudes stay below 16392 x 4 x 31 x 2 < 2^22 (with the offset of 16 that up
    to sixteen rows have), so every order of f32 sums is exact, and a column that is left out, taken twice or met by another's weight shows."""
    from ironpangu_b200.ops import int4

    g = torch.Generator(device="cuda").manual_seed(N + K + T)
    q, s, z = _codes(N, K, group, zeros, N + K)
    s = torch.exp2(torch.randint(-1, 2, s.shape, generator=g, device="cuda").float()).to(BF16)
    x = torch.randint(-4, 5, (T, K + 8), generator=g, device="cuda").to(BF16)[:, :K]
    want = x.double() @ _values(q, s, z, group).T
    assert torch.equal(int4.linear(x, int4.pack(q, s, z, group=group), out_f32=True).double(), want)
    if N % 2 == 0:
        y = int4.linear(x, int4.pack(q, s, z, group=group, gated=True), out_f32=True).double()
        gate, up = want[:, :N // 2], want[:, N // 2:]
        unit = gate * torch.sigmoid(gate) * up
        # CUDA's fast exponential is documented to be off by up to 2 + floor(1.173 |a|) steps of f32, 2^-23 of it each; 1 + it, the quotient or reciprocal and two products take
        # six more at most. Below e^-87 the unit is less than 87 e^-87 2^19 < 1e-30
        steps = 8 + 1.173 * gate.abs().clamp(max=90)
        assert bool(((y - unit).abs() <= 2.0 ** -23 * steps * unit.abs() + 1e-30).all())


@pytest.mark.gpu
@pytest.mark.parametrize("group,zeros,f16", [(128, False, False), (64, True, True), (32, True, False)])
@pytest.mark.parametrize("N,K,T", [(333, 520, 17), (130, 9000, 40), (1237, 1032, 129), (129, 4096, 255), (5000, 520, 700), (2741, 1032, 1501)])
def test_many_rows_against_the_matrix_that_was_packed(N, K, T, group, zeros, f16):
    """Without the rounding of weights in the reference: half a step of f16, 2^-11 of a weight, beside the bound of the sums."""
    from ironpangu_b200.ops import int4

    q, s, z = _codes(N, K, group, zeros, N + K, f16)
    x, v = _rows(T, K, T), _values(q, s, z, group)
    bound = _operands(v, x)[1] + 2.0 ** -11 * (x.double().abs() @ v.abs().T)
    _close(int4.linear(x, int4.pack(q, s, z, group=group), out_f32=True), x.double() @ v.T, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("group,zeros,f16", [(128, False, False), (64, True, True), (32, True, False)])
@pytest.mark.parametrize("N,K,T", [(300, 1032, 1), (70, 520, 3), (5000, 136, 8), (64, 16392, 2), (333, 2056, 16), (130, 520, 21), (333, 1032, 140), (300, 640, 600)])
def test_infinities_and_rows_near_the_end_of_the_range(N, K, T, group, zeros, f16):
    """An infinity in a row of x gives infinities of the weights' signs, and NaN where the weight is 0 or two of them meet with opposite signs, whatever the number of rows; rows whose
    products with 16 + q pass f32's range give the finite results that they have."""
    from ironpangu_b200.ops import int4

    q, s, z = _codes(N, K, group, zeros, N + K, f16)
    x, v = _rows(T, K, T), _values(q, s, z, group)
    w = int4.pack(q, s, z, group=group)
    x[0, 5] = float("inf")
    if T > 1:
        x[1, K - 1], x[1, 3] = float("-inf"), 0
    if T > 2:
        x[2] *= 2.0 ** 124
    if T > 3:
        x[3, 0], x[3, K // 2] = float("inf"), float("inf")
    want = x.double() @ v.T
    out = int4.linear(x, w, out_f32=True)
    fine = want.isfinite()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf() & ~fine, want.isinf()) and torch.equal(out[want.isinf()].double(), want[want.isinf()])
    bound = (x.double().abs() @ v.abs().T)[fine] * (max(CUT, 17 * K / 16 * 2.0 ** -23) + (2.0 ** -11 if T > 16 else 0)) + 1e-30
    assert bool(((out.double() - want)[fine].abs() <= bound).all())
    both = int4.linear(x, w, residual=torch.ones(T, N, dtype=BF16, device="cuda"))
    assert torch.equal(both.isnan(), want.isnan()) and torch.equal(both[want.isinf()].double(), want[want.isinf()])


@pytest.mark.gpu
def test_infinite_gains_and_gated_units():
    from ironpangu_b200.ops import int4

    F, K = 90, 520
    q, s, z = _codes(2 * F, K, 64, True, 5)
    w, v = int4.pack(q, s, z, group=64, gated=True), _values(q, s, z, 64)
    for T in (1, 5):
        x, gain = _rows(T, K, T), torch.ones(K, dtype=BF16, device="cuda")
        gain[17] = float("inf")
        xn = (x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-5)).to(BF16).double()
        xn[:, 17] = torch.where(xn[:, 17] > 0, float("inf"), float("-inf"))
        y = xn @ v.T
        gate, up = y[:, :F], y[:, F:]
        want = gate / (1 + torch.exp(-gate)) * up
        out = int4.linear(x, w, norm_w=gain, eps=1e-5, out_f32=True)
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf()) and torch.equal(out[want.isinf()].double(), want[want.isinf()])


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("power", [-133, -126, -120, -60, 96, 104, 115, 122, 124, 126, 127])
def test_quantise_at_the_ends_of_the_range(power, zeros):
    """Matrices near bf16's smallest and largest numbers, quotients halfway between two codes among them: codes, scales and zero points are the definition's, also where the largest
    less the smallest passes f32's range."""
    from ironpangu_b200.ops import int4

    g = torch.Generator(device="cuda").manual_seed(power + 200)
    w = (torch.randn(70, 264, generator=g, device="cuda").clamp(-1.9, 1.9).double() * 2.0 ** power)
    w[1] = (torch.arange(264, device="cuda") % 31 - 15).double() / 2 * 2.0 ** (power - 3)        # halves of a scale of 2^(power - 3)
    w[2] = torch.where(torch.arange(264, device="cuda") % 2 == 0, 1.99, -1.99).double() * 2.0 ** power
    w = w.to(BF16)
    assert bool(w.isfinite().all())
    f = torch.nn.functional.pad(w.double(), (0, -264 % 128)).view(70, -1, 128)
    lo, hi = f.amin(-1).clamp(max=0), f.amax(-1).clamp(min=0)
    # f32 and then bf16, as it is defined; a quotient by 15 or 7 is rounded to f32 first (f32's subnormals have steps of 2^-149)
    exact = (hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7
    s = exact.float().to(BF16).double()
    s = torch.where(s == 0, 1.0, s)[..., None]
    z = torch.round(-lo[..., None] / s).clamp(0, 15) if zeros else 8
    q = (torch.round(f / s) + z).clamp(0, 15)
    want = ((q - z) * s).reshape(70, -1)[:, :264].float().to(BF16)
    assert torch.equal(int4.quantise(w, group=128, zeros=zeros).dequantise(), want)


def test_outputs_that_overlap_are_refused():
    """Rows of an output over one another, over the rows that are read or over a residual that is another matrix; side by side in one buffer is no overlap. On the host, where what
    is not refused for this is refused for the weights' place."""
    from ironpangu_b200.ops import int4

    w, F32 = int4.Int4Weight(64, 64, device="cpu"), torch.float32
    buffer = torch.zeros(40, 256, dtype=BF16)
    flat = buffer.view(-1)
    x, apart, wide = buffer[:9, :64], buffer[:9, 64:128], torch.zeros(9, 128, dtype=F32)
    rows = lambda at, pitch: torch.as_strided(flat, (9, 64), (pitch, 1), at)
    for out, what in ((torch.zeros(1, 64, dtype=BF16).expand(9, 64), "lie apart"), (rows(5000, 32), "lie apart"), (x, "overlap"), (buffer[:9, 32:96], "overlap"), (buffer[8:17, :64], "overlap"),
                      (buffer[:9, 200:][:, :56].new_zeros(0), "output must be"), (rows(0, 512), "overlap"), (rows(256 - 8, 256), "overlap"), (buffer.view(F32)[:9, 16:80], "overlap"),
                      (rows(64, 264), "overlap")):
        with pytest.raises(ValueError, match=what):
            int4.linear(x, w, out=out)
    for residual in (buffer[:9, 128:192], buffer[:9, 64:128].clone(), buffer[1:10, 64:128], rows(64, 512), buffer[:9, 100:164]):
        with pytest.raises(ValueError, match="the output or lie apart|on the host") as e:
            int4.linear(x, w, out=apart, residual=residual)
        meet = residual.data_ptr() in (buffer[1:10, 64:128].data_ptr(), rows(64, 512).data_ptr(), buffer[:9, 100:164].data_ptr()) and residual.untyped_storage().data_ptr() == flat.data_ptr()
        assert ("lie apart" in str(e.value)) == meet
    for call in (dict(out=apart, residual=apart), dict(out=apart, residual=buffer[:9, 64:128]), dict(out=wide[:, :64]), dict(out=buffer[9:18, :64]), dict(out=buffer[20:29, 7:71]),
                 dict(residual=x), dict(out=apart, residual=x)):
        with pytest.raises(ValueError, match="on the host"):
            int4.linear(x, w, **call)
    one = torch.zeros(1, 64, dtype=BF16)
    with pytest.raises(ValueError, match="on the host"):
        int4.linear(one, w, out=torch.zeros(2, 64, dtype=BF16)[:1].as_strided((1, 64), (0, 1)))
    with pytest.raises(ValueError, match="overlap"):
        int4.linear(flat[:64].view(1, 64), w, out=flat[63:127].view(1, 64))
