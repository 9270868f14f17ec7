"""Groups that cannot be: their rows see everything through their own slots, by every kernel that has rows of groups."""
import pytest
import torch

from ironpangu_b200.ops import shared_prefix as S
from test_shared_prefix import BAD_INDEX, Batch, stale

I32 = torch.int32
pytestmark = pytest.mark.gpu
MOST = (1 << 31) - 1


def _listed(groups):
    return torch.tensor(groups, dtype=torch.int64).to(I32).cuda()


def _refused(b, groups, valid, rows, status=BAD_INDEX):
    """A call by `groups` is one by `valid`, those of them that can be; every checked row is what the definition says."""
    b.status.zero_()
    got = b.run(groups=_listed(groups), scratch=torch.full((S.scratch_bytes(b.q.shape[0], b.heads, b.kv, b.dim, len(groups)),), 255, dtype=torch.uint8, device="cuda"))
    assert int(b.status) == status
    b.status.zero_()
    kept, b.groups = b.groups, _listed(valid) if valid else b.groups[:0]
    b.check(got=got, rows=rows)
    b.groups = kept


# few rows: parts and merge; 400 rows by kv heads: tiles and four warps a row; 1184: one warp
@pytest.mark.parametrize("first,second,heads,kv", [(4, 3, 8, 2), (150, 60, 8, 2), (420, 200, 8, 2)])
def test_groups_that_cannot_be(first, second, heads, kv):
    b = Batch([(first, 100, lambda: 40), (second, 50, lambda: 20)], heads=heads, kv=kv, dim=128, seed=10)
    # what the groups' own slots hold and what the rows' hold differ from here on: a row that took the wrong one shows
    T, rows = first + second, sorted({0, 1, 2, first - 1, first, first + 1, first + second // 2, first + second - 1})
    one, two = b.groups.tolist()
    for bad in ([-1, first, 100, 0], [-MOST - 1, first, 100, 0], [0, first, -1, 0], [0, first, 100, b.table.shape[0]], [0, first, 100, -1], [0, first, 100, MOST], [0, first + second + 1, 100, 0], [0, first, 1 << 30, 0],
                [0, first, MOST, 0], [0, MOST, 5, 0], [0, 1 << 30, 5, 0], [1, MOST, 5, 0], [MOST, 1, 5, 0], [MOST, MOST, 5, 0], [T, 1, 5, 0], [3, -1, 5, 0], [0, -MOST - 1, 5, 0]):
        _refused(b, [bad, two], [two], rows)
        _refused(b, [bad], [], rows)
    _refused(b, [two, one], [two], rows)           # not in the order of their rows
    _refused(b, [one, [first - 1, second, 50, two[3]]], [one], rows)                      # rows of another group
    _refused(b, [one, one, two], [one, two], rows)
    _refused(b, [one, [first, 0, 50, 99], two, [0, 0, 0, 0]], [one, two], rows, status=0)      # of no rows: counts as none
    everyone = [[0, T, 0, 0]]                      # nothing shared
    _refused(b, everyone, [], rows, status=0)
    assert torch.equal(b.run(groups=_listed([one, two]), scratch=stale(b)), b.run())
