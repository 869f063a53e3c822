"""Caches whose blocks lie beyond 2^32 bytes: the operators on drafted trees and on caches kept to a budget against the same call
on a small cache, bit for bit."""
import pytest
import torch

from test_gpu_evict import BF, i32

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, KV, D, BS, MB = 8, 2, 128, 64, 12
LENS, CLENS = [9, 1, 40], [300, 600, 5]


def both(near, far_blocks, run):
    """`run(tensors, tables)` on a small cache, and on one whose blocks of the tables lie spread over `far_blocks`."""
    g = torch.Generator().manual_seed(7)
    n = 3 * MB
    places = torch.randperm(n, generator=g)
    far = torch.linspace(0, far_blocks - 1, n).long()
    got = []
    for blocks, where in ((n, torch.arange(n)), (far_blocks, far)):
        tensors = {}
        for name, x in near.items():
            tensors[name] = torch.empty(blocks, *x.shape[1:], dtype=x.dtype, device=DEV)
            tensors[name][where.to(DEV)] = x.to(DEV)
        out = run(tensors, where[places].int().view(3, MB).contiguous().to(DEV))
        got.append([out] + [t[where.to(DEV)] for t in tensors.values()])
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cache", [BF, torch.int8])
def test_far_blocks(rt, cache):
    from gvirt_amd._C import attention_weights, compact_kv_cache, select_kept, tree_attention
    g = torch.Generator().manual_seed(3)
    n = 3 * MB
    bytes_ = cache == torch.int8
    raw = lambda: torch.randint(-127, 128, (n, BS, KV, D), generator=g).to(torch.int8) if bytes_ else torch.randn(n, BS, KV, D, generator=g).to(BF)  # noqa: E731
    near = dict(k=raw(), v=raw(), w=torch.rand(n, BS, KV, generator=g))
    if bytes_:
        near.update(ks=torch.rand(n, BS, KV, generator=g) * 0.02, vs=torch.rand(n, BS, KV, generator=g) * 0.02)
    T = sum(LENS)
    qkv = (torch.randn(T, (H + 2 * KV) * D, generator=g) * 0.1).to(BF).to(DEV)
    mask = torch.randint(-2 ** 31, 2 ** 31, (T, 2), generator=g).to(torch.int32).to(DEV)
    starts, lens, clens = i32([0, 9, 10]), i32(LENS), i32(CLENS)

    def run(t, tables):
        out = torch.zeros(T, H * D, dtype=BF, device=DEV)
        tree_attention(rt, qkv, t["k"], t["v"], out, mask, starts, lens, clens, tables, H, KV, D, BS, 3, MB, k_scale=t.get("ks"), v_scale=t.get("vs"))
        for window in (1, 0):     # scores stored, scores formed twice
            attention_weights(rt, qkv, t["k"], t["w"], starts, lens, clens, tables, H, KV, D, BS, 3, MB, window, k_scale=t.get("ks"))
        kept, kept_lens = torch.zeros(3, KV, 100, dtype=torch.int32, device=DEV), i32([0] * 3)
        select_kept(rt, t["w"], kept, kept_lens, clens + lens, tables, KV, BS, 3, MB, 100, 20, 4)
        compact_kv_cache(rt, t["k"], t["v"], kept, kept_lens, tables, KV, D, BS, 3, MB, weights=t["w"], k_scale=t.get("ks"), v_scale=t.get("vs"))
        return torch.cat([out.float().flatten(), kept.float().flatten(), kept_lens.float()])
    # 5 GB a cache: blocks of 32 KiB, or of 16 KiB in bytes
    both(near, 5 * 2 ** 30 // near["k"][0].nbytes, run)
