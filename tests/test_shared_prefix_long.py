"""Attention of rows that share a prefix over long stretches of keys with values of one sign, whose sums grow with every key: nothing of them may be lost on the way."""
import pytest
import torch

from ironpangu_b200.ops import shared_prefix as S

BF16, F64, I32 = torch.bfloat16, torch.float64, torch.int32
gpu = pytest.mark.gpu


def _error(rows, heads, kv, dim, page, shared, own, checked, *, slots=1, groups=1, rising=0.0):
    """Relative errors of the checked rows: all sequences lie on the same pages, the first `shared` positions of them a prefix of every group. `rising`: by how much scores grow from the first to the last key."""
    g = torch.Generator(device="cuda").manual_seed(shared + own)
    n = shared + own
    pages = -(-n // page)
    k = torch.randn(pages, page, kv, dim, generator=g, device="cuda")
    q = torch.randn(rows, heads, dim, generator=g, device="cuda") * 0.3
    if rising:
        q[..., 0] = dim ** 0.25
        k.view(-1, kv, dim)[:, :, 0] = (torch.arange(pages * page, device="cuda") / n * rising * dim ** 0.25)[:, None]
    k, q = k.to(BF16), q.to(BF16).view(rows, -1)
    # columns of sizes of their own, so that roundings of the results do not all go one way
    v = ((torch.randn(pages, page, kv, dim, generator=g, device="cuda").abs() + 0.5) * (1 + torch.rand(kv, dim, generator=g, device="cuda"))).to(BF16)
    table = torch.arange(pages, device="cuda", dtype=I32).expand(slots, -1).contiguous()
    each = rows // groups
    listed = torch.tensor([[i * each, each, shared, 0] for i in range(groups)] if shared else [], dtype=I32, device="cuda").view(-1, 4)
    status = torch.zeros(1, dtype=I32, device="cuda")
    slot_of = (torch.arange(rows, device="cuda") % slots).to(I32)
    scratch = torch.full((S.scratch_bytes(rows, heads, kv, dim, listed.shape[0]),), 255, dtype=torch.uint8, device="cuda")
    out = S.attention(q, k, v, torch.full((rows,), n - 1, dtype=I32, device="cuda"), slot_of, table, listed, heads=heads, kv_heads=kv, head_dim=dim, scale=dim ** -0.5, scratch=scratch,
                      status_ptr=status.data_ptr())
    assert int(status) == 0
    errors = []
    keys, values = (x.view(-1, kv, dim)[:n] for x in (k, v))
    for t in checked:
        for h in range(heads):
            j = h // (heads // kv)
            w = torch.softmax(keys[:, j].to(F64) @ q[t, h * dim:(h + 1) * dim].to(F64) * dim ** -0.5, 0)
            want = w @ values[:, j].to(F64)
            errors.append((out[t, h * dim:(h + 1) * dim].to(F64) - want) / want)
    return torch.cat(errors)


def _check(errors):
    """A result is rounded once: by 2^-8 of itself at most. Its weights have 15 bits (2^-15), its scores are f32 sums of 128 products (2^-18 of a weight), and a sum that the tensor core adds up loses 1.1e-8 of
    itself a key, 4096 keys 2^-14.4: together 2^-13.5. The mean of N roundings is within five times 2^-8 / sqrt(3 N) of 0."""
    assert float(errors.abs().max()) <= 2 ** -8 + 2 ** -13.5
    assert abs(float(errors.mean())) <= 2 ** -13.5 + 5 * 2 ** -8 / (3 * errors.numel()) ** 0.5


@gpu
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (8, 2, 64)])
def test_a_prefix_in_one_stretch(heads, kv, dim):
    """148 tiles of 256 pairs: an SM each, whatever the prefix's length. Also lengths about the ends of a sum."""
    _check(_error(4736, heads, kv, dim, 16, 131072, 4, [0, 2000, 4735]))
    for shared in (4096, 4097, 8192, 8320, 12289):
        _check(_error(4736, heads, kv, dim, 16, shared, 1, [0, 255, 4735]))


@gpu
def test_a_prefix_of_scores_that_rise():
    """Maxima that move while sums go on, and behind their ends."""
    for rising in (10.0, 40.0, 200.0):
        _check(_error(4736, 8, 2, 128, 16, 40000, 4, [0, 2000, 4735], rising=rising))


@gpu
def test_a_prefix_in_streams_of_keys():
    """64 groups of a row: two streams of a tile's keys, a prefix in one stretch."""
    _check(_error(64, 16, 4, 128, 16, 131072, 4, [0, 31, 63], groups=64))
    _check(_error(64, 16, 4, 128, 16, 16500, 4, [0, 31, 63], groups=64, rising=30.0))


@gpu
def test_a_prefix_over_pages_that_the_tensor_maps_do_not_take():
    _check(_error(1200, 8, 2, 128, 12, 131064, 4, [0, 500, 1199]))
    _check(_error(600, 8, 2, 64, 12, 65532, 4, [0, 300, 599], rising=40.0))


@gpu
@pytest.mark.parametrize("rows,heads,kv,shared,own,slots", [(600, 8, 2, 16, 65536, 600), (600, 8, 2, 16, 262144, 1), (600, 32, 2, 16, 65536, 1), (210, 8, 2, 16, 262144, 210), (150, 8, 1, 0, 262144, 150)])
def test_long_own_positions(rows, heads, kv, shared, own, slots):
    """A warp a row; four rows of a sequence together; the same of more heads; four warps a row; rows that no group names."""
    _check(_error(rows, heads, kv, 128, 16, shared, own, [0, rows // 2, rows - 1], slots=slots))
    _check(_error(rows, heads, kv, 128, 16, shared, 20000, [0, rows // 2, rows - 1], slots=slots, rising=25.0))


@gpu
@pytest.mark.parametrize("page,most", [(1, (1 << 31) - 257), (8, ((1 << 31) - 257) // 8)])
def test_prefixes_to_the_end_of_32_bits(page, most):
    """The last positions that there may be, of pages that are all the same but for the last: all weight lies there. Stretches of whole tiles would end behind 2^31."""
    g = torch.Generator(device="cuda").manual_seed(page)
    k, v = torch.zeros(2, page, 1, 64, dtype=BF16, device="cuda"), torch.randn(2, page, 1, 64, generator=g, device="cuda").to(BF16)
    k[1] = 5.0
    table = torch.zeros(1, most, dtype=I32, device="cuda")
    table[0, -1] = 1
    n = most * page
    i32 = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    status = torch.zeros(1, dtype=I32, device="cuda")
    out = S.attention(torch.full((1, 64), 5.0, dtype=BF16, device="cuda"), k, v, i32([n - 1]), i32([0]), table, i32([[0, 1, n, 0]]), heads=1, kv_heads=1, head_dim=64, scale=0.125, status_ptr=status.data_ptr())
    want = v[1, :, 0].double().mean(0)             # the other 2^31 keys weigh e^-200 each
    assert bool(((out[0].double() - want).abs() <= want.abs() * 2 ** -8 + v[1, :, 0].double().abs().mean(0) * 2 ** -13.5).all()) and int(status) == 0
