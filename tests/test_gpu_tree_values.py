"""What does not have ordinary values: infinities and NaNs that the rows of a tree see, queries that are NaN, and V scales
of a cache of bytes from nothing to the largest."""
import pytest
import torch

from gvirt_amd import workloads as W
from test_gpu_tree import check, make, run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16


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


@pytest.mark.parametrize("cache", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (64, 1)])     # (blocks of one: through the 16-bit copy)
def test_queries_that_are_nan_over_caches_of_bytes(rt, D, bs, dtype, cache):
    clean, dirty = (make(12, [9, 40], [70, 5], 4, 2, D, bs, dtype, cache) for _ in range(2))
    dirty["qkv"].view(-1, 8, D)[11, 1, 7] = float("nan")
    a, b = run(rt, clean).view(-1, 4, D), run(rt, dirty).view(-1, 4, D)
    assert (b[11, 1] != b[11, 1]).all()
    b[11, 1] = a[11, 1]
    assert torch.equal(a, b)


def test_queries_that_are_nan_in_the_causal_kernel(rt):
    """The same conversion of queries serves chunks over a cache of bytes."""
    from gvirt_amd._C import attention
    for limit in (None, 64):     # through the 16-bit copy, and read on the fly
        w = make(12, [40], [70], 4, 2, 128, 16, BF, "int8", spare=0)
        w["qkv"].view(-1, 8, 128)[11, 1, 7] = float("nan")
        d = W.to_device({k: v for k, v in w.items() if isinstance(v, torch.Tensor)}, DEV)
        out = torch.zeros(40, 4 * 128, dtype=BF, device=DEV)
        attention(rt, d["qkv"], d["k"], d["v"], out, d["qsl"], d["lens"], d["clens"], d["tables"], 4, 2, 128, 16, 1, w["mb"], k_scale=d["ks"],
                  v_scale=d["vs"], workspace_limit=limit)
        bad = torch.isnan(out.float().view(40, 4, 128)).cpu()
        assert bad[11, 1].all() and bad.sum() == 128


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache", ["int8", "fp8"])
def test_v_scales_that_are_nan_reach_the_rows_that_see_them(rt, D, cache):
    for node in (2, -3):     # a node, a cached position of the tile that the tree begins in
        clean, dirty = (make(13, [6], [21], 4, 2, D, 16, FP, cache) for _ in range(2))
        p = 21 + node
        dirty["vs"][int(dirty["tables"][p // 16]), p % 16, 1] = float("nan")
        a, b = run(rt, clean).view(-1, 4, D), run(rt, dirty).view(-1, 4, D)
        for r in range(6):
            sees = node < 0 or int(clean["mask"][r, 0]) >> node & 1
            assert torch.isnan(b[r, 2:]).all() if sees else torch.equal(a[r], b[r])
            assert torch.equal(a[r, :2], b[r, :2])     # (the other kv head's)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache", ["int8", "fp8"])
def test_v_scales_from_nothing_to_the_largest(rt, D, cache):
    """Positions of scale zero keep their weight in the normaliser beside positions of scale 2^50."""
    w = make(14, [9, 3], [300, 40], 4, 2, D, 16, BF, cache)
    g = torch.Generator().manual_seed(2)
    w["vs"] = torch.full(w["vs"].shape, 2.0 ** 50)
    w["vs"][torch.rand(w["vs"].shape, generator=g) < 0.5] = 0.0
    check(run(rt, w), w)
    w["vs"] *= 2.0 ** -80     # and of small ones
    check(run(rt, w), w)
