"""Caches kept to a budget on the GPU: `attention_weights`, `select_kept` and `compact_kv_cache` against plain
implementations (fp64, or exact where values are only compared or moved)."""
import random

import pytest
import torch

from gvirt_amd import workloads as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16


def paged(seed, totals, bs):
    g = torch.Generator().manual_seed(seed)
    mb = max(1, max((t + bs - 1) // bs for t in totals))
    NB = len(totals) * mb + 1
    return torch.randperm(NB, generator=g)[:len(totals) * mb].int().view(len(totals), mb), mb, NB, g


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def slots(table_row, n, bs):
    pos = torch.arange(n)
    return table_row[pos // bs].long() * bs + pos % bs


# ---- attention_weights -------------------------------------------------------------------------------------------------

def weights_case(rt, lens, clens, H, KV, D, bs, dtype, window=0, cache="same", seed=0, scale=2.0, runtime=None):
    """(result, expected, tolerance) [num_blocks, block_size, kv_heads]."""
    from gvirt_amd._C import attention_weights
    tables, mb, NB, g = paged(seed, [l + c for l, c in zip(lens, clens)], bs)
    T, G = sum(lens), H // KV
    qkv = (torch.randn(T, H + 2 * KV, D, generator=g) * D ** -0.5 * scale).to(dtype)
    k, ks = torch.randn(NB, bs, KV, D, generator=g), None
    if cache != "same":
        k, ks = W.quantize_cache(k, torch.int8 if cache == "int8" else torch.float8_e4m3fn)
    else:
        k = k.to(dtype)
    w = torch.rand(NB, bs, KV, generator=g)
    starts = [sum(lens[:i]) for i in range(len(lens))]
    got = w.to(DEV)
    attention_weights(runtime or rt, qkv.view(T, -1).to(DEV), k.to(DEV), got, i32(starts), i32(lens), i32(clens), tables.to(DEV), H, KV, D, bs, len(lens),
                      mb, window, k_scale=None if ks is None else ks.to(DEV))
    want, tol = w.double().view(-1, KV).clone(), torch.zeros(NB * bs, KV, dtype=torch.float64)
    kd = k.double() if ks is None else k.double() * ks.double().unsqueeze(-1)
    for i, (n, c, s0) in enumerate(zip(lens, clens, starts)):
        if n == 0:
            continue
        at = slots(tables[i], c + n, bs)
        key = kd.view(-1, KV, D)[at]
        want[at[c:]] = 0
        for r in range(max(0, n - window) if window else 0, n):
            for h in range(H):
                kk, q = key[:c + r + 1, h // G], qkv[s0 + r, h].double()
                s = kk @ q
                p = torch.softmax(s, 0)
                want[at[:c + r + 1], h // G] += p
                # a score is a sum of D products in fp32 (and a product with its scale), off by (D + 4) half units of
                # the sum of their sizes; that moves p by exp(2 off); the exponentials and sums add 2^-19
                off = (D + 4) * 2.0 ** -24 * float((kk.abs() @ q.abs()).max())
                tol[at[:c + r + 1], h // G] += p * (2 * off + 2.0 ** -19)
    tol += want.abs() * n_adds(lens, G) * 2.0 ** -24
    return got.cpu().double().view(-1, KV), want, tol


def n_adds(lens, G):
    return 64 + max(lens) * G / 32   # a tile's additions, then one per tile


CASES = [([1], [0]), ([1] * 5, [8, 13, 65, 11, 300]), ([0, 3, 1, 0], [7, 40, 129, 12]), ([40], [0]), ([70, 5], [63, 257]), ([33], [1000])]


@pytest.mark.parametrize("lens,clens", CASES)
@pytest.mark.parametrize("H,KV,D,bs", [(14, 2, 64, 16), (32, 8, 128, 128), (28, 4, 128, 7), (8, 2, 256, 24), (3, 3, 64, 32), (40, 1, 128, 64)])
def test_weights_shapes_and_lengths(rt, H, KV, D, bs, lens, clens):
    got, want, tol = weights_case(rt, lens, clens, H, KV, D, bs, BF if len(lens) % 2 else FP)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())


@pytest.mark.parametrize("window", [1, 2, 31, 64])
def test_weights_of_the_last_rows(rt, window):
    for lens, clens in (([40, 1, 0, 70], [3, 50, 9, 0]), ([200], [64])):
        got, want, tol = weights_case(rt, lens, clens, 8, 2, 128, 16, BF, window=window)
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("cache", ["int8", "fp8"])
def test_weights_over_caches_of_bytes(rt, cache):
    for H, KV, D, bs, dtype in ((14, 2, 64, 16, BF), (32, 8, 128, 128, FP), (28, 4, 128, 24, BF), (4, 1, 64, 5, FP)):
        for lens, clens in (([1, 1, 1], [300, 64, 0]), ([37, 2], [100, 5])):
            got, want, tol = weights_case(rt, lens, clens, H, KV, D, bs, dtype, cache=cache)
            assert ((got - want).abs() <= tol).all()


def test_weights_of_long_contexts(rt):
    got, want, tol = weights_case(rt, [2, 1], [9000, 5], 8, 2, 128, 32, BF)
    assert ((got - want).abs() <= tol).all()
    got, want, tol = weights_case(rt, [300], [1500], 4, 2, 64, 16, BF, scale=6.0)     # peaked rows
    assert ((got - want).abs() <= tol).all()


def test_weights_are_the_same_in_every_run_and_leave_others_alone(rt):
    a = weights_case(rt, [5, 0, 20], [700, 31, 40], 8, 2, 128, 16, BF)
    b = weights_case(rt, [5, 0, 20], [700, 31, 40], 8, 2, 128, 16, BF)
    assert torch.equal(a[0], b[0])
    assert (a[0] == a[1].float().double())[a[2] == 0].all()      # slots of no visible position


def test_weights_on_another_stream_and_captured(rt):
    from gvirt_amd._C import Runtime, attention_weights
    r2 = Runtime(0, 64)
    r2.blocking = False
    tables, mb, NB, g = paged(3, [700, 40], 16)
    qkv = (torch.randn(2, 12, 64, generator=g) * 0.3).to(BF).view(2, -1).to(DEV)
    k = torch.randn(NB, 16, 2, 64, generator=g).to(BF).to(DEV)
    start = torch.rand(NB, 16, 2, generator=g).to(DEV)
    args = (i32([0, 1]), i32([1, 1]), i32([699, 39]), tables.to(DEV), 8, 2, 64, 16, 2, mb)
    want = [start.clone()]
    for _ in range(3):
        want.append(want[-1].clone())
        attention_weights(rt, qkv, k, want[-1], *args)
    w = start.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_weights(r2, qkv, k, w, *args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(w, want[1])
    graph = torch.cuda.CUDAGraph()
    w.copy_(start)
    with torch.cuda.graph(graph):
        attention_weights(r2, qkv, k, w, *args)
    for turn in range(1, 4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, want[turn])
        torch.ones(1000, device=DEV).sum().item()


# ---- select_kept ---------------------------------------------------------------------------------------------------------

def plain_select(w, length, budget, recent, sink):
    if length <= budget:
        return list(range(length))
    middle = sorted(range(sink, length - recent), key=lambda j: (w[j] == w[j], -w[j] if w[j] == w[j] else 0.0, j))
    return list(range(sink)) + sorted(middle[:budget - sink - recent]) + list(range(length - recent, length))


@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("KV,bs,lens,budget,recent,sink", [
    (2, 16, [711], 512, 64, 4), (1, 7, [0, 1, 5, 6, 4], 5, 2, 1), (8, 128, [3000, 17, 64], 64, 64, 0), (4, 24, [1500, 1024, 1025], 1024, 0, 0),
    (3, 32, [40, 33], 33, 20, 13), (2, 16, [5000], 1, 0, 0), (1, 64, [20000], 3000, 100, 4), (1, 128, [41000, 9], 4096, 8, 8)])
def test_select(rt, KV, bs, lens, budget, recent, sink, kind):
    from gvirt_amd._C import select_kept
    tables, mb, NB, g = paged(budget, lens, bs)
    w = torch.rand(NB, bs, KV, generator=g)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "odd":
        w = (torch.randn(NB, bs, KV, generator=g) * 3).round()
        pick = torch.rand(NB, bs, KV, generator=g)
        w[pick < 0.05], w[(pick > 0.05) & (pick < 0.1)], w[(pick > 0.1) & (pick < 0.15)] = float("nan"), float("inf"), -float("inf")
        w[(pick > 0.15) & (pick < 0.2)] = -0.0
    kept, kept_lens = i32([[[9] * budget] * KV] * len(lens)), i32([9] * len(lens))
    select_kept(rt, w.to(DEV), kept, kept_lens, i32(lens), tables.to(DEV), KV, bs, len(lens), mb, budget, recent, sink)
    kept = kept.cpu()
    assert kept_lens.tolist() == [min(n, budget) for n in lens]
    for i, n in enumerate(lens):
        at = slots(tables[i], n, bs)
        for h in range(KV):
            want = plain_select(w.view(-1, KV)[at, h].tolist(), n, budget, recent, sink)
            assert kept[i, h].tolist() == want + [-1] * (budget - len(want)), (i, h)


@pytest.mark.parametrize("kind", ["random", "ties"])
@pytest.mark.parametrize("lens", [[32769, 4000], [33100], [65536, 2], [65601], [65700, 66], [100003]])
def test_select_long(rt, lens, kind):
    """Around the lengths at which a list's keys stop fitting a workgroup's registers."""
    from gvirt_amd._C import select_kept
    KV, bs, budget, recent, sink = 1, 48, 1000, 60, 4
    tables, mb, NB, g = paged(len(lens), lens, bs)
    w = torch.rand(NB, bs, KV, generator=g)
    if kind == "ties":
        w = (w * 4).floor()
    kept, kept_lens = i32([[[9] * budget] * KV] * len(lens)), i32([9] * len(lens))
    select_kept(rt, w.to(DEV), kept, kept_lens, i32(lens), tables.to(DEV), KV, bs, len(lens), mb, budget, recent, sink)
    kept = kept.cpu()
    assert kept_lens.tolist() == [min(n, budget) for n in lens]
    for i, n in enumerate(lens):
        want = plain_select(w.view(-1, KV)[slots(tables[i], n, bs), 0].tolist(), n, budget, recent, sink)
        assert kept[i, 0].tolist() == want + [-1] * (budget - len(want)), i


# ---- compact_kv_cache ------------------------------------------------------------------------------------------------------

def compact_case(rt, seed, totals, starts, KV, D, bs, dtype, per_head, counts, width, weights=True, lists=None):
    from gvirt_amd._C import compact_kv_cache
    tables, mb, NB, g = paged(seed, totals, bs)
    rnd = random.Random(seed)
    bytes_ = dtype not in (BF, FP)
    raw = lambda: torch.randint(0, 127, (NB, bs, KV, D), generator=g).to(torch.uint8).view(dtype) if bytes_ else torch.randn(NB, bs, KV, D, generator=g).to(dtype)  # noqa: E731
    t = dict(k=raw(), v=raw(), ks=torch.rand(NB, bs, KV, generator=g) if bytes_ else None, vs=torch.rand(NB, bs, KV, generator=g) if bytes_ else None,
             w=torch.rand(NB, bs, KV, generator=g) if weights else None)
    batch = len(totals)
    if lists is None:
        rows = [[sorted(rnd.sample(range(totals[i] - (starts[i] if starts else 0)), counts[i])) for _ in range(KV if per_head else 1)] for i in range(batch)]
    else:
        rows = lists
    kept = torch.full((batch, KV if per_head else 1, width), -1, dtype=torch.int32)
    for i in range(batch):
        for h, r in enumerate(rows[i]):
            kept[i, h, :len(r)] = torch.tensor(r, dtype=torch.int32)
    d = {n: None if x is None else x.to(DEV) for n, x in t.items()}
    compact_kv_cache(rt, d["k"], d["v"], (kept if per_head else kept[:, 0].contiguous()).to(DEV), i32(counts), tables.to(DEV), KV, D, bs, batch, mb,
                     starts=i32(starts) if starts else None, weights=d["w"], k_scale=d["ks"], v_scale=d["vs"])
    for n, x in t.items():
        if x is None:
            continue
        x = x.view(torch.uint8) if bytes_ and n in "kv" else x
        want = x.clone().view(NB * bs, KV, -1)
        old = x.view(NB * bs, KV, -1)
        for i in range(batch):
            at = slots(tables[i], mb * bs, bs)
            s0 = starts[i] if starts else 0
            for h in range(KV):
                r = rows[i][h if per_head else 0][:counts[i]]
                r = [(j, p) for j, p in enumerate(r) if j <= p < mb * bs - s0]
                want[at[[s0 + j for j, _ in r]], h] = old[at[[s0 + p for _, p in r]], h]
        got = d[n].cpu()
        got = got.view(torch.uint8) if bytes_ and n in "kv" else got
        assert torch.equal(got.view(NB * bs, KV, -1), want), n


@pytest.mark.parametrize("dtype", [BF, FP, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("KV,D,bs", [(2, 64, 16), (8, 128, 128), (4, 128, 7), (3, 256, 24), (1, 16, 5), (2, 48, 16)])
def test_compact_per_head(rt, KV, D, bs, dtype):
    compact_case(rt, 1, [300, 41, 1, 900], None, KV, D, bs, dtype, True, [128, 41, 1, 700], 700)
    compact_case(rt, 2, [64], None, KV, D, bs, dtype, True, [0], 9, weights=False)


@pytest.mark.parametrize("dtype", [BF, torch.int8])
@pytest.mark.parametrize("KV,D,bs", [(2, 64, 16), (8, 128, 128), (5, 128, 7), (4, 256, 24)])
def test_compact_accepted_paths(rt, KV, D, bs, dtype):
    compact_case(rt, 3, [120, 9, 33, 64], [100, 0, 30, 63], KV, D, bs, dtype, False, [6, 9, 1, 0], 9)


def test_compact_ignores_entries_that_break_the_rules(rt):
    lists = [[[3, 1, 2, 60, 1000000, -5, 6, 90], list(range(8))]]
    compact_case(rt, 4, [64], None, 2, 64, 16, BF, True, [8], 8, lists=lists)
    compact_case(rt, 4, [64], [60], 2, 64, 16, BF, True, [8], 8, lists=lists)
    compact_case(rt, 4, [64], None, 2, 64, 16, BF, True, [8], 8, lists=[[[7] * 8, [9, 9, 9, 9, 8, 8, 8, 7]]])   # a source twice


def test_select_and_compact_captured():
    """Both captured together, replayed on weights and rows that change, the lists written by the one and read by the other."""
    from gvirt_amd._C import Runtime, compact_kv_cache, select_kept
    r2 = Runtime(0, 8)
    r2.blocking = False
    KV, D, bs, lens, budget, recent, sink = 2, 64, 16, [100, 30, 0, 333], 48, 8, 2
    tables, mb, NB, g = paged(17, lens, bs)
    k, v, w = (torch.zeros(NB, bs, KV, x, dtype=t, device=DEV) for x, t in ((D, BF), (D, BF), (1, torch.float32)))
    w = w.view(NB, bs, KV)
    kept, kept_lens, td, ld = i32([[[0] * budget] * KV] * 4), i32([0] * 4), tables.to(DEV), i32(lens)

    def both():
        select_kept(r2, w, kept, kept_lens, ld, td, KV, bs, 4, mb, budget, recent, sink)
        compact_kv_cache(r2, k, v, kept, kept_lens, td, KV, D, bs, 4, mb, weights=w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for _ in range(3):
        w0, k0, v0 = torch.rand(NB, bs, KV, generator=g), torch.randn(NB, bs, KV, D, generator=g).to(BF), torch.randn(NB, bs, KV, D, generator=g).to(BF)
        for dst, src in ((w, w0), (k, k0), (v, v0)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        for i, n in enumerate(lens):
            at = slots(tables[i], n, bs)
            for h in range(KV):
                want = plain_select(w0.view(-1, KV)[at, h].tolist(), n, budget, recent, sink)
                assert kept[i, h].tolist() == want + [-1] * (budget - len(want))
                for new, old in ((w, w0), (k, k0), (v, v0)):
                    assert torch.equal(new.cpu().view(NB * bs, KV, -1)[at[:len(want)], h], old.view(NB * bs, KV, -1)[at[want], h])
        torch.ones(1000, device=DEV).sum().item()


def test_evicting_keeps_what_attention_sees(rt):
    """The operators as they are used: weights accumulate over decode steps, the cache is cut per kv head, and attention
    over the cut cache is attention over the kept rows."""
    from gvirt_amd._C import attention, attention_weights, compact_kv_cache, select_kept
    H, KV, D, bs, lens, budget = 8, 2, 64, 16, [200, 90, 33], 64
    tables, mb, NB, g = paged(8, [n + 8 for n in lens], bs)
    k, v = torch.randn(NB, bs, KV, D, generator=g).to(BF).to(DEV), torch.randn(NB, bs, KV, D, generator=g).to(BF).to(DEV)
    w = torch.zeros(NB, bs, KV, device=DEV)
    td = tables.to(DEV)
    for step in range(3):
        qkv = (torch.randn(3, (H + 2 * KV) * D, generator=g) * 0.3).to(BF).to(DEV)
        attention_weights(rt, qkv, k, w, i32([0, 1, 2]), i32([1] * 3), i32([n + step - 1 for n in lens]), td, H, KV, D, bs, 3, mb)
    now = [n + 2 for n in lens]
    kept, kept_lens = torch.zeros(3, KV, budget, dtype=torch.int32, device=DEV), i32([0] * 3)
    select_kept(rt, w, kept, kept_lens, i32(now), td, KV, bs, 3, mb, budget, 8, 2)
    k0, v0 = k.cpu().view(-1, KV, D).double(), v.cpu().view(-1, KV, D).double()
    compact_kv_cache(rt, k, v, kept, kept_lens, td, KV, D, bs, 3, mb, weights=w)
    out = torch.zeros(3, H * D, dtype=BF, device=DEV)
    attention(rt, qkv, k, v, out, i32([0, 1, 2]), i32([1] * 3), kept_lens - 1, td, H, KV, D, bs, 3, mb)
    for i in range(3):
        assert int(kept_lens[i]) == min(budget, now[i])
        at = slots(tables[i], now[i], bs)
        for h in range(H):
            rows = at[kept[i, h * KV // H, :int(kept_lens[i])].cpu().long()]
            q = qkv[i].cpu().double().view(-1, D)[h]
            p = torch.softmax(k0[rows, h * KV // H] @ q, 0)
            want, mass = p @ v0[rows, h * KV // H], p @ v0[rows, h * KV // H].abs()
            err = (out[i].cpu().double().view(H, D)[h] - want).abs()
            assert (err <= 2.0 ** -8 * (mass + want.abs()) + 2.0 ** -14 * mass).all()   # probabilities, result; accumulation


def test_refusals(rt):
    from gvirt_amd._C import attention_weights, compact_kv_cache, select_kept
    tables, mb, NB, g = paged(1, [60], 16)
    td, one = tables.to(DEV), i32([1])
    k = torch.zeros(NB, 16, 2, 64, dtype=BF, device=DEV)
    w = torch.zeros(NB, 16, 2, device=DEV)
    qkv = torch.zeros(1, 8 * 64, dtype=BF, device=DEV)
    kept = torch.zeros(1, 2, 8, dtype=torch.int32, device=DEV)

    def weights(**kw):
        a = dict(qkv=qkv, k=k, w=w, qsl=i32([0]), lens=one, clens=one, tables=td, H=4, KV=2, D=64, bs=16, batch=1, mb=mb, window=0)
        a.update(kw)
        scale = a.pop("k_scale", None)
        attention_weights(rt, *a.values(), k_scale=scale)

    def select(**kw):
        a = dict(w=w, kept=kept, kept_lens=i32([0]), lens=i32([60]), tables=td, KV=2, bs=16, batch=1, mb=mb, budget=8, recent=2, sink=1)
        a.update(kw)
        select_kept(rt, *a.values())

    def compact(**kw):
        a = dict(k=k, v=k.clone(), kept=kept, kept_lens=i32([4]), tables=td, KV=2, D=64, bs=16, batch=1, mb=mb)
        more = {n: kw.pop(n) for n in ("starts", "weights", "k_scale", "v_scale") if n in kw}
        a.update(kw)
        compact_kv_cache(rt, *a.values(), **more)

    bad = [(weights, [dict(w=w.half()), dict(w=w[:1]), dict(window=-1), dict(H=3), dict(D=32), dict(k=k.half()), dict(k_scale=w), dict(lens=one.long()),
                      dict(batch=2), dict(qkv=qkv.float()), dict(w=w.transpose(0, 1)), dict(tables=td.cpu())]),
           (select, [dict(budget=2), dict(recent=8), dict(sink=-1), dict(recent=-1), dict(kept=kept[:, :1]), dict(kept=kept.long()), dict(w=w.double()), dict(batch=2),
                     dict(bs=0), dict(kept_lens=one.float())]),
           (compact, [dict(kept=kept[0, 0]), dict(kept=kept[:, :1]), dict(kept=kept.long()), dict(v=k.half()), dict(weights=w.half()), dict(k_scale=w),
                      dict(k_scale=w, v_scale=w), dict(starts=one.long()), dict(k=k.float(), v=k.float()), dict(D=4, KV=32), dict(batch=3)])]
    for call, kws in bad:
        call()
        for kw in kws:
            with pytest.raises(RuntimeError):
                call(**kw)
