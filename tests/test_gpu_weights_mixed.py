"""`attention_weights` of batches that mix a few long chunks with many short sequences, and of block tables that are much wider
than the contexts, against the same plain implementation as ordinary batches."""
import pytest
import torch

from test_gpu_evict import BF, FP, i32, paged, weights_case

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("lens", [[70] + [1] * 40 + [0], [1] * 30 + [0, 150, 2] + [1] * 60, [1] * 66 + [0] * 5 + [90] + [1] * 30 + [67],
                                  [64, 65] + [1] * 60, [70] + [0] * 80])
@pytest.mark.parametrize("H,KV,D,bs,cache", [(28, 4, 128, 16, "same"), (8, 2, 64, 7, "same"), (16, 4, 256, 24, "same"), (14, 2, 64, 16, "fp8"),
                                             (4, 1, 128, 24, "int8")])
def test_long_chunks_beside_short_sequences(rt, H, KV, D, bs, cache, lens):
    clens = [(37 * i) % 90 for i in range(len(lens))]
    got, want, tol = weights_case(rt, lens, clens, H, KV, D, bs, BF if len(lens) % 2 else FP, cache=cache)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
    assert (got == want.float().double())[tol == 0].all()      # slots of no visible position


@pytest.mark.parametrize("window", [40, 80])
def test_windows_of_long_chunks(rt, window):
    lens = [100, 90, 0] + [1] * 60
    got, want, tol = weights_case(rt, lens, [(11 * i) % 50 for i in range(len(lens))], 16, 2, 128, 16, BF, window=window)
    assert ((got - want).abs() <= tol).all()


def test_the_same_in_every_run(rt):
    lens = [70] + [1] * 40
    a, b = (weights_case(rt, lens, list(range(41)), 28, 4, 128, 16, BF) for _ in range(2))
    assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("positions", [4200000, 17000000])
def test_tables_much_wider_than_the_contexts(positions):
    """All kv heads' scores at once, a few heads at a time, and none stored at all: the same weights. A weight is a sum of
    up to 2 x 2 probabilities, each off by 2^-18 (scores of some units, their exponentials and their sum) whichever way."""
    from gvirt_amd._C import Runtime, attention_weights
    runtime = Runtime(0, 1)
    H, KV, D, bs, lens, clens = 8, 4, 64, 128, [1, 0, 2, 1], [700, 5, 300, 0]
    tables, mb, NB, g = paged(5, [a + b for a, b in zip(lens, clens)], bs)
    wide = torch.zeros(4, positions // bs, dtype=torch.int32)
    wide[:, :mb] = tables
    qkv = (torch.randn(4, (H + 2 * KV) * D, generator=g) * 0.25).to(BF).to(DEV)
    k, w = torch.randn(NB, bs, KV, D, generator=g).to(BF).to(DEV), torch.rand(NB, bs, KV, generator=g).to(DEV)
    got = []
    for t in (tables, wide):
        x = w.clone()
        attention_weights(runtime, qkv, k, x, i32([0, 1, 1, 3]), i32(lens), i32(clens), t.to(DEV), H, KV, D, bs, 4, t.shape[1])
        got.append(x)
    assert not torch.equal(got[0], w)
    assert torch.allclose(got[0], got[1], rtol=2.0 ** -17, atol=0)
