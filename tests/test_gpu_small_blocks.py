"""Caches of blocks of one and two positions: the operators on drafted trees and on caches kept to a budget against the same
plain implementations, and within the same tolerances, as over larger blocks."""
import pytest
import torch

from test_gpu_evict import BF, FP, compact_case, i32, paged, plain_select, slots, weights_case
from test_gpu_tree import check, make, run

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bs", [1, 2])
@pytest.mark.parametrize("D,dtype,cache", [(64, BF, "same"), (128, FP, "same"), (256, BF, "same"), (64, FP, "int8"), (128, BF, "int8"), (64, BF, "fp8")])
def test_trees(rt, D, dtype, cache, bs):
    w = make(31, [9, 1, 0, 33], [70, 33, 5, 0], 4, 2, D, bs, dtype, cache)
    check(run(rt, w), w)


@pytest.mark.parametrize("bs", [1, 2])
@pytest.mark.parametrize("D,dtype,cache", [(64, BF, "same"), (128, FP, "same"), (256, BF, "same"), (64, FP, "int8"), (128, BF, "fp8")])
def test_weights(rt, D, dtype, cache, bs):
    for lens, clens in (([1, 0, 1, 2], [70, 4, 0, 300]), ([40, 3], [65, 9])):    # scores stored, scores formed twice
        got, want, tol = weights_case(rt, lens, clens, 4, 2, D, bs, dtype, cache=cache)
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("bs", [1, 2])
@pytest.mark.parametrize("lens,budget,recent,sink", [([300, 17, 64], 64, 16, 4), ([5000, 1], 700, 0, 0)])
def test_select(rt, lens, budget, recent, sink, bs):
    from gvirt_amd._C import select_kept
    KV = 2
    tables, mb, NB, g = paged(budget, lens, bs)
    w = torch.rand(NB, bs, KV, generator=g)
    kept, kept_lens = i32([[[9] * budget] * KV] * len(lens)), i32([9] * len(lens))
    select_kept(rt, w.to(DEV), kept, kept_lens, i32(lens), tables.to(DEV), KV, bs, len(lens), mb, budget, recent, sink)
    assert kept_lens.tolist() == [min(n, budget) for n in lens]
    for i, n in enumerate(lens):
        for h in range(KV):
            want = plain_select(w.view(-1, KV)[slots(tables[i], n, bs), h].tolist(), n, budget, recent, sink)
            assert kept[i, h].tolist() == want + [-1] * (budget - len(want)), (i, h)


@pytest.mark.parametrize("bs", [1, 2])
@pytest.mark.parametrize("dtype", [BF, torch.int8])
def test_compact(rt, dtype, bs):
    compact_case(rt, 1, [300, 41, 1, 900], None, 2, 64, bs, dtype, True, [128, 41, 1, 700], 700)
    compact_case(rt, 3, [120, 9, 33, 64], [100, 0, 30, 63], 3, 64, bs, dtype, False, [6, 9, 1, 0], 9)
