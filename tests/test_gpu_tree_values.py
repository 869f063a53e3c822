"""Infinities and NaNs that the rows of a tree see."""
import pytest
import torch

from test_gpu_tree import make, run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (256, 16), (64, 5), (128, 5), (256, 6)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_of_cached_positions_reach_every_row(rt, D, bs, bad):
    """One cached position's V row holds `bad` in some columns: the first or the last cached position of the 32 that the
    tree begins in, or one well before them. Every row sees it: those columns are `bad`, the others keep their bits."""
    for at in (lambda c: c & ~31, lambda c: c - 1, lambda c: 2):
        lens, clens = [6, 40, 3], [21, 85, 747]
        clean, dirty = (make(9, lens, clens, 4, 2, D, bs, BF) for _ in range(2))
        for i, c in enumerate(clens):
            b = int(dirty["tables"][i * dirty["mb"] + at(c) // bs])
            dirty["v"][b, at(c) % bs, :, 3::7] = bad
        a, b = run(rt, clean)[:sum(lens)].view(-1, 4, D), run(rt, dirty)[:sum(lens)].view(-1, 4, D)
        x = b[:, :, 3::7].float()
        assert (x != x).all() if bad != bad else (x == bad).all()
        rest = [d for d in range(D) if d % 7 != 3]
        assert torch.equal(a[:, :, rest], b[:, :, rest])


def test_values_that_some_rows_see_beside_values_that_all_see(rt):
    """A cached +infinity and a node's -infinity in the same columns: a NaN for the rows that see both."""
    for D in (64, 128, 256):
        w = make(10, [6], [21], 4, 2, D, 16, BF)
        pos = lambda p: (int(w["tables"][p // 16]), p % 16)  # noqa: E731
        w["v"][pos(20)][:, 5] = float("inf")
        w["v"][pos(21 + 2)][:, 5] = -float("inf")
        x = run(rt, w)[:6].view(6, 4, D)[:, :, 5].float()
        for r in range(6):
            if int(w["mask"][r, 0]) >> 2 & 1:
                assert (x[r] != x[r]).all()
            else:
                assert (x[r] == float("inf")).all()
