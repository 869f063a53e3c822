"""CPU checks of the operators on drafted trees and on caches kept to a budget: the host metadata, and what is refused."""
import ctypes
import random

import pytest
import torch

from gvirt_amd import _C, _lib
from gvirt_amd.mha import prepare_tree


def test_prepare_tree_masks_and_positions():
    rnd = random.Random(1)
    for _ in range(10):
        batch = rnd.randint(1, 5)
        lens = [rnd.choice([1, 2, 31, 32, 33, 70]) for _ in range(batch)]
        clens = [rnd.randint(0, 90) for _ in range(batch)]
        parents = [[rnd.randint(-1 if r == 0 or rnd.random() < 0.1 else 0, r - 1) if r else -1 for r in range(n)] for n in lens]
        bs = rnd.choice([4, 16])
        tables = [[rnd.randint(0, 99) for _ in range((l + c + bs - 1) // bs)] for l, c in zip(lens, clens)]
        meta = prepare_tree(lens, clens, tables, bs, parents, "cpu")
        assert meta.tree_mask.shape == (sum(lens), (max(lens) + 31) // 32) and meta.parents.tolist() == sum(parents, [])
        row = 0
        for i, n in enumerate(lens):
            for r in range(n):
                line, up = [], r
                while up >= 0:
                    line.append(up)
                    up = parents[i][up]
                words = [int(w) & 0xffffffff for w in meta.tree_mask[row]]
                assert [j for j in range(32 * len(words)) if words[j // 32] >> (j % 32) & 1] == sorted(line)
                assert int(meta.position[row]) == clens[i] + len(line) - 1
                assert int(meta.slot_mapping[row]) == tables[i][(clens[i] + r) // bs] * bs + (clens[i] + r) % bs
                row += 1
    # a cache that was cut down: rope positions run on from the sequence's own
    assert prepare_tree([2], [3], [[0, 1]], 4, [[-1, 0]], "cpu", positions=[10]).position.tolist() == [10, 11]


def test_prepare_tree_refusals():
    for lens, parents in (([2], [[-1, 1]]), ([2], [[-1, 2]]), ([1], [[-2]]), ([2], [[-1]]), ([1, 1], [[-1]]), ([], []), ([0], [[]])):
        with pytest.raises(RuntimeError):
            prepare_tree(lens, [0] * len(lens), [[0]] * len(lens), 16, parents, "cpu")
    u1 = ctypes.c_uint32 * 1
    par = (ctypes.c_int32 * 40)(*([-1] + list(range(39))))
    pos, mask = (ctypes.c_int64 * 40)(), (ctypes.c_int32 * 40)()
    assert _lib.load().xlite_hip_prepare_tree(u1(40), u1(0), par, 1, 1, pos, mask) < 0   # 40 nodes do not fit one word
    assert b"mask_words" in _lib.load().xlite_hip_last_error()


class FakeRt:
    device = torch.device("cuda", 0)


def test_wrappers_refuse_cpu_tensors():
    x, i, f = torch.zeros(2, 4 * 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 128, 1)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _C.tree_attention(FakeRt(), x, x, x, x, i, i, i, i, i, 2, 1, 64, 128, 2, 1)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _C.verify_tree(FakeRt(), x, i, i, i, i, i, i, i, 2)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _C.attention_weights(FakeRt(), x, x, f, i, i, i, i, 2, 1, 64, 128, 2, 1)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _C.select_kept(FakeRt(), f, i, i, i, i, 1, 128, 2, 1, 4, 2)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        _C.compact_kv_cache(FakeRt(), x, x, i, i, i, 1, 64, 128, 2, 1)
    for bad in (None, 3):
        with pytest.raises(RuntimeError, match="expected a tensor"):
            _C.select_kept(FakeRt(), bad, i, i, i, i, 1, 128, 2, 1, 4, 2)


# C entry points: everything is checked before anything is launched (the pointers are never followed)
P = ctypes.c_void_p(1 << 20)
TREE = dict(stream=None, qkv=P, k=P, v=P, out=P, mask=P, words=1, qsl=P, lens=P, clens=P, tables=P, tokens=8, heads=4, kv_heads=2, dim=64,
            block=16, batch=2, blocks=4, dtype=1, kv=0, ks=None, vs=None, ws=None, ws_bytes=0)
WEIGHTS = dict(stream=None, qkv=P, k=P, w=P, qsl=P, lens=P, clens=P, tables=P, tokens=8, heads=4, kv_heads=2, dim=64, block=16, batch=2,
               blocks=4, window=0, dtype=1, kv=0, ks=None, ws=P, ws_bytes=1 << 30)
SELECT = dict(stream=None, w=P, kept=P, kept_lens=P, lens=P, tables=P, kv_heads=2, block=16, batch=2, blocks=4, budget=8, recent=4, sink=2)
COMPACT = dict(stream=None, k=P, v=P, ks=None, vs=None, w=None, kept=P, kept_lens=P, starts=None, tables=P, kv_heads=2, dim=64, block=16,
               batch=2, blocks=4, max_kept=8, per_head=1, kv=0)
VERIFY = dict(stream=None, logits=P, tokens=P, parents=P, accepted=P, n=P, next=P, qsl=P, lens=P, total=8, vocab=100, batch=2, max_path=4,
              dtype=1, ws=P, ws_bytes=1 << 20)
BAD = [
    ("tree_attention", TREE, [dict(qkv=None), dict(mask=None), dict(tables=None), dict(words=0), dict(dim=96), dict(heads=3), dict(kv_heads=0),
                              dict(block=0), dict(blocks=0), dict(dtype=2), dict(kv=3), dict(kv=1), dict(kv=2, ks=P, vs=P, dim=256),
                              dict(blocks=1 << 28), dict(tokens=1 << 30), dict(kv=1, ks=P, vs=P, dim=64)]),
    ("attention_weights", WEIGHTS, [dict(qkv=None), dict(w=None), dict(lens=None), dict(dim=80), dict(heads=3), dict(block=0), dict(blocks=0),
                                    dict(dtype=2), dict(kv=5), dict(kv=1), dict(kv=1, ks=P, dim=256), dict(ws=None), dict(ws_bytes=0),
                                    dict(batch=70000), dict(blocks=1 << 28)]),
    ("select_kept", SELECT, [dict(w=None), dict(kept=None), dict(kept_lens=None), dict(lens=None), dict(tables=None), dict(kv_heads=0),
                             dict(block=0), dict(blocks=0), dict(budget=0), dict(budget=5), dict(recent=0xffffffff), dict(blocks=1 << 28)]),
    ("compact_kv_cache", COMPACT, [dict(k=None), dict(v=None), dict(kept=None), dict(kept_lens=None), dict(tables=None), dict(dim=4),
                                   dict(kv=1), dict(kv=7), dict(block=0), dict(k=ctypes.c_void_p((1 << 20) + 8)), dict(batch=60000),
                                   dict(blocks=1 << 28)]),
    ("verify_tree", VERIFY, [dict(logits=None), dict(tokens=None), dict(accepted=None), dict(n=None), dict(lens=None), dict(vocab=0),
                             dict(max_path=0), dict(dtype=3), dict(ws=None), dict(ws_bytes=8)]),
]


def test_c_entry_points_refuse_what_they_could_not_read():
    """Tensors off their alignment, a mask longer than any tree, lengths that the call itself would overwrite."""
    lib = _lib.load()
    off = ctypes.c_void_p((1 << 20) + 8)
    for name, good, bads, why in (("tree_attention", TREE, [dict(qkv=off), dict(k=off), dict(v=off), dict(out=off), dict(ws=off, ws_bytes=64)], b"aligned"),
                                  ("tree_attention", TREE, [dict(words=(1 << 22) + 1)], b"mask_words"),
                                  ("attention_weights", WEIGHTS, [dict(qkv=off), dict(k=off), dict(ws=off)], b"aligned"),
                                  ("select_kept", SELECT, [dict()], b"context_lens")):
        for bad in bads:
            assert getattr(lib, "xlite_hip_" + name)(*dict(good, **bad).values()) < 0, bad
            assert why in lib.xlite_hip_last_error(), (bad, lib.xlite_hip_last_error())


@pytest.mark.parametrize("name,good,bads", BAD, ids=[b[0] for b in BAD])
def test_c_entry_points_refuse(name, good, bads):
    lib = _lib.load()
    fn = getattr(lib, "xlite_hip_" + name)
    assert len(fn.argtypes) == len(good)
    for bad in bads:
        assert fn(*dict(good, **bad).values()) < 0, bad
        assert lib.xlite_hip_last_error(), bad
    if name != "verify_tree":   # (a batch of none: nothing to do, nothing followed)
        assert fn(*dict(good, batch=0).values()) == 0
