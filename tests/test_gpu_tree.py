"""Drafted trees on the GPU: `tree_attention` and `verify_tree` against plain implementations in fp64.

Tolerances count roundings, u = half a unit in the last place (bf16 2^-8, fp16 2^-11): the probabilities are rounded to the
products' type and the result to the output's, fp32 accumulation adds 2^-16 at most; a cache of bytes is widened to fp16
with its scale, one rounding of every K and V element, and a score that is off by e moves its probability by a factor
exp(e), the normaliser likewise."""
import random

import pytest
import torch

from gvirt_amd import workloads as W

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def tree_mask(parents, words):
    rows = []
    for r, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | (1 << r))
    return torch.tensor([[((x >> (32 * w)) & 0xffffffff) - (1 << 32 if x >> (32 * w + 31) & 1 else 0) for w in range(words)] for x in rows],
                        dtype=torch.int64).to(torch.int32)


def make(seed, lens, clens, H, KV, D, bs, dtype, cache="same", words=None, spare=3):
    g = torch.Generator().manual_seed(seed)
    rnd = random.Random(seed)
    batch, T = len(lens), sum(lens)
    mb = max(1, max((l + c + bs - 1) // bs for l, c in zip(lens, clens)))
    NB = batch * mb + 1
    qkv = torch.randn(T + spare, H + 2 * KV, D, generator=g) * D ** -0.5 * 2
    kc, vc = torch.randn(NB, bs, KV, D, generator=g), torch.randn(NB, bs, KV, D, generator=g)
    ks = vs = None
    if cache != "same":
        t = torch.int8 if cache == "int8" else torch.float8_e4m3fn
        (kc, ks), (vc, vs) = W.quantize_cache(kc, t), W.quantize_cache(vc, t)
    else:
        kc, vc = kc.to(dtype), vc.to(dtype)
    words = words or max(1, (max(lens) + 31) // 32)
    masks = [tree_mask([-1] + [rnd.randint(max(0, r - 6), r - 1) for r in range(1, n)], words) for n in lens if n]
    starts = [sum(lens[:i]) for i in range(batch)]
    return dict(qkv=qkv.reshape(T + spare, -1).to(dtype), k=kc, v=vc, ks=ks, vs=vs, mask=torch.cat(masks + [torch.full((spare, words), -1, dtype=torch.int32)]),
                qsl=torch.tensor(starts, dtype=torch.int32), lens=torch.tensor(lens, dtype=torch.int32),
                clens=torch.tensor(clens, dtype=torch.int32), tables=torch.randperm(NB, generator=g)[:batch * mb].int(),
                H=H, KV=KV, D=D, bs=bs, batch=batch, mb=mb, T=T, dtype=dtype, cache=cache)


def run(rt, w):
    from gvirt_amd._C import tree_attention
    d = W.to_device({k: v for k, v in w.items() if isinstance(v, torch.Tensor)}, DEV)
    out = torch.full((w["qkv"].shape[0], w["H"] * w["D"]), 7.0, dtype=w["dtype"], device=DEV)
    tree_attention(rt, d["qkv"], d["k"], d["v"], out, d["mask"], d["qsl"], d["lens"], d["clens"], d["tables"], w["H"], w["KV"],
                   w["D"], w["bs"], w["batch"], w["mb"], k_scale=d.get("ks"), v_scale=d.get("vs"))
    return out.cpu()


def reference(w):
    """(result, tolerance), both [tokens, heads, head_dim] in fp64; rows of no sequence are NaN."""
    H, KV, D, bs, G = w["H"], w["KV"], w["D"], w["bs"], w["H"] // w["KV"]
    out = torch.full((w["qkv"].shape[0], H, D), float("nan"), dtype=torch.float64)
    tol = out.clone()
    uo, up = U[w["dtype"]], U[w["dtype"]] if w["cache"] == "same" else 2.0 ** -11
    for i in range(w["batch"]):
        n, c, s0 = int(w["lens"][i]), int(w["clens"][i]), int(w["qsl"][i])
        pos = torch.arange(c + n)
        blk = w["tables"][i * w["mb"] + pos // bs].long()
        k, v = w["k"][blk, pos % bs].double(), w["v"][blk, pos % bs].double()
        if w["ks"] is not None:
            k, v = k * w["ks"][blk, pos % bs].double().unsqueeze(-1), v * w["vs"][blk, pos % bs].double().unsqueeze(-1)
        for r in range(n):
            words = [int(x) & 0xffffffff for x in w["mask"][s0 + r]]
            nodes = [j for j in range(n) if j < 32 * len(words) and words[j // 32] >> (j % 32) & 1]
            seen = list(range(c)) + [c + j for j in nodes]
            if not seen:
                out[s0 + r], tol[s0 + r] = 0.0, 0.0
                continue
            q = w["qkv"][s0 + r].view(-1, D)[:H].double()
            for h in range(H):
                kk, vv = k[seen, h // G], v[seen, h // G]
                s = kk @ q[h]
                p = torch.exp(s - s.max())
                p = p / p.sum()
                out[s0 + r, h] = p @ vv
                mass = p @ vv.abs()
                off = 0.0
                if w["cache"] != "same":
                    off = 2 * 2.0 ** -11 * float((kk.abs() @ q[h].abs()).max()) + 2.0 ** -11   # K, then V
                tol[s0 + r, h] = (up + off + 2.0 ** -16) * mass + uo * out[s0 + r, h].abs() + 2.0 ** -24
    return out, tol


def check(got, w):
    want, tol = reference(w)
    got = got.view(want.shape).double()
    rows = torch.isfinite(tol).all(-1).all(-1)
    assert (got[~rows] == 7.0).all(), "a row of no sequence was written"
    err = (got[rows] - want[rows]).abs()
    worst = (err / tol[rows].clamp_min(1e-30)).max() if err.numel() else torch.zeros(())
    assert (err <= tol[rows]).all(), "off by %.3g of the tolerance" % float(worst)


SHAPES = [(14, 2, 64, 16), (32, 8, 128, 128), (28, 4, 128, 32), (16, 4, 256, 48), (5, 1, 128, 7), (4, 4, 64, 24), (8, 2, 256, 16),
          (40, 2, 128, 64), (6, 3, 64, 8)]
BATCHES = [([1], [0]), ([1, 1], [17, 5]), ([8], [700]), ([3, 0, 33, 1, 0], [40, 9, 127, 128, 0]), ([70, 2], [63, 1025]), ([0, 17], [3, 64])]


@pytest.mark.parametrize("lens,clens", BATCHES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes_and_lengths(rt, shape, lens, clens):
    H, KV, D, bs = shape
    w = make(hash((shape, tuple(lens))) % 1000, lens, clens, H, KV, D, bs, torch.bfloat16 if (H + len(lens)) % 2 else torch.float16)
    check(run(rt, w), w)


@pytest.mark.parametrize("cache", ["int8", "fp8"])
@pytest.mark.parametrize("shape", [(14, 2, 64, 16), (32, 8, 128, 128), (28, 4, 128, 24), (4, 2, 128, 12), (6, 1, 64, 7)])
def test_caches_of_bytes(rt, shape, cache):
    H, KV, D, bs = shape
    for dtype in (torch.bfloat16, torch.float16):
        w = make(5, [9, 1, 40], [300, 64, 0], H, KV, D, bs, dtype, cache)
        check(run(rt, w), w)


@pytest.mark.parametrize("batch,nodes,context", [(1, 5, 9000), (3, 64, 5000), (40, 4, 600)])
def test_long_contexts_split_over_workgroups(rt, batch, nodes, context):
    w = make(3, [max(1, nodes - i) for i in range(batch)], [context - 37 * i if context > 37 * batch else context for i in range(batch)], 4, 2, 128, 32,
             torch.bfloat16)
    check(run(rt, w), w)


@pytest.mark.parametrize("cache", ["same", "int8"])
@pytest.mark.parametrize("H,KV,lens,clens", [
    (4, 2, [1, 3, 0, 5, 2] * 14, [37 * i % 200 for i in range(70)]),     # more sequences than a wave has lanes
    (8, 2, [100] + [1] * 7, [70, 0, 33, 5, 64, 1, 127, 300]),            # one tree of many times the others' rows
    (8, 2, [200, 0, 2], [40, 3, 500]), (9, 3, [90], [65]),
    (2, 2, [300], [11])])                                                # rows of mask words that do not fit next to each other
def test_many_sequences_and_many_rows(rt, H, KV, lens, clens, cache):
    w = make(6, lens, clens, H, KV, 128, 16, torch.bfloat16, cache)
    check(run(rt, w), w)


@pytest.mark.parametrize("lens,clens", BATCHES + [([100, 1, 1, 1, 1, 1, 1, 1], [70, 0, 33, 5, 64, 1, 127, 300]), ([30], [5000]),
                                                  ([2] * 70, [17 * i % 90 for i in range(70)])])
@pytest.mark.parametrize("H,KV,bs", [(16, 4, 64), (4, 1, 12), (6, 3, 7)])
def test_heads_of_256(rt, H, KV, bs, lens, clens):
    w = make(16, lens, clens, H, KV, 256, bs, torch.bfloat16 if bs % 2 else torch.float16)
    check(run(rt, w), w)


@pytest.mark.parametrize("cache", ["int8", "fp8"])
@pytest.mark.parametrize("H,KV,D,bs", [(14, 2, 64, 16), (28, 4, 128, 24), (3, 3, 64, 7), (8, 2, 128, 64)])
def test_bytes_are_widened_exactly(rt, H, KV, D, bs, cache):
    """The values of a cache of bytes are exact in fp16 and its scales stay in fp32, whatever their sizes: an fp16 model loses
    what the probabilities (times V's scale) and the result are rounded, u each. Scores are off by (D + 8) half units of the
    sum of their products' sizes in fp32, and their sum with log2 of a scale (up to 64) by 2^-18 of a factor of two."""
    w = make(14, [9, 1, 30], [300, 64, 5], H, KV, D, bs, torch.float16, cache)
    g = torch.Generator().manual_seed(1)
    w["vs"] = w["vs"] * torch.exp2(torch.randint(-20, 4, w["vs"].shape, generator=g).float())
    w["vs"][torch.rand(w["vs"].shape, generator=g) < 0.1] = 0.0
    want, tol = reference(w)
    got = run(rt, w).view(want.shape).double()
    u = 2.0 ** -11
    for i in range(3):
        n, c, s0 = int(w["lens"][i]), int(w["clens"][i]), int(w["qsl"][i])
        pos = torch.arange(c + n)
        blk = w["tables"][i * w["mb"] + pos // bs].long()
        k = w["k"][blk, pos % bs].double() * w["ks"][blk, pos % bs].double().unsqueeze(-1)
        v = w["v"][blk, pos % bs].double() * w["vs"][blk, pos % bs].double().unsqueeze(-1)
        for r in range(n):
            seen = list(range(c)) + [c + j for j in range(n) if int(w["mask"][s0 + r, j // 32]) >> (j % 32) & 1]
            q = w["qkv"][s0 + r].view(-1, D)[:H].double()
            for h in range(H):
                kk, vv = k[seen, h // (H // KV)], v[seen, h // (H // KV)]
                p = torch.softmax(kk @ q[h], 0)
                off = (D + 8) * 2.0 ** -24 * float((kk.abs() @ q[h].abs()).max()) + 2.0 ** -18
                # (a product below fp16's normal numbers, 2^-14 of the largest one's power of two, is off by 2^-25 of that)
                least = 2.0 ** -25 * 2 * float((p * vv.abs().amax(-1)).max()) * len(seen)
                bound = (u + 2 * off + 2.0 ** -16) * (p @ vv.abs()) + u * want[s0 + r, h].abs() + least + 2.0 ** -25
                assert ((got[s0 + r, h] - want[s0 + r, h]).abs() <= bound).all(), (i, r, h)


@pytest.mark.parametrize("cache", ["same", "fp8"])
@pytest.mark.parametrize("D", [64, 128])
def test_more_sequences_than_prefix_sums_fit(rt, D, cache):
    lens = [[1, 2, 0, 1, 3][i % 5] for i in range(1030)]
    w = make(15, lens, [i % 37 for i in range(1030)], 2, 1, D, 16, torch.float16, cache)
    check(run(rt, w), w)


@pytest.mark.parametrize("cache", ["same", "int8"])
def test_less_workspace_gives_the_same_attention_or_an_error(rt, cache):
    """With less scratch than a shape asks for, another kernel serves it or nothing is launched."""
    w = make(8, [9, 1, 40], [300, 64, 0], 8, 2, 128, 16, torch.bfloat16, cache)
    d = W.to_device({k: v for k, v in w.items() if isinstance(v, torch.Tensor)}, DEV)
    p = lambda n: d[n].data_ptr() if d.get(n) is not None else None  # noqa: E731
    lib, T, kv = rt._lib, w["qkv"].shape[0], 0 if cache == "same" else 1
    need = lib.xlite_hip_tree_attention_workspace_bytes(T, 8, 2, 128, 16, 3, w["mb"], kv)
    served = []
    for size in (need, need // 2, need // 4, need // 16, 64):
        ws = torch.empty(size, dtype=torch.uint8, device=DEV)
        out = torch.full((T, 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
        rc = lib.xlite_hip_tree_attention(rt.stream(), p("qkv"), p("k"), p("v"), out.data_ptr(), p("mask"), w["mask"].shape[1], p("qsl"), p("lens"),
                                          p("clens"), p("tables"), T, 8, 2, 128, 16, 3, w["mb"], 1, kv, p("ks"), p("vs"), ws.data_ptr(), size)
        torch.cuda.synchronize()
        served.append(rc)
        if rc == 0:
            check(out.cpu(), w)
        else:
            assert b"workspace" in lib.xlite_hip_last_error() and (out == 7.0).all()
    assert served[0] == 0   # (the prefill kernels run without partials: 64 bytes may be enough)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_any_mask_and_rows_that_see_nothing(rt, D):
    for clens in ([0, 0, 31], [0, 70, 0]):
        w = make(11, [37, 5, 64], clens, 4, 2, D, 16, torch.bfloat16, words=3)
        g = torch.Generator().manual_seed(4)
        w["mask"] = torch.randint(-2 ** 31, 2 ** 31, w["mask"].shape, generator=g).to(torch.int32)   # bits past the nodes too
        w["mask"][:6] = 0
        w["mask"][50] = 0
        check(run(rt, w), w)
    w = make(12, [40], [3], 4, 2, D, 16, torch.float16, words=2)
    w["mask"] = w["mask"][:, :1].contiguous()      # too few words: nodes 32 .. 39 are seen by nobody
    check(run(rt, w), w)


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (256, 16), (128, 5), (256, 6)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_not_finite_stay_where_they_are_seen(rt, D, bs, bad):
    """Node 2's K and V rows and everything behind the sequence hold `bad`; the rows that do not see node 2 are those of
    the clean batch, the ones that do get the plain formula's infinities and NaNs."""
    lens, clens = [6, 40], [21, 64]
    clean = make(9, lens, clens, 4, 2, D, bs, torch.bfloat16)
    dirty = make(9, lens, clens, 4, 2, D, bs, torch.bfloat16)
    for i in range(2):
        n, c = lens[i], clens[i]
        for p in [c + 2] + list(range(c + n, clean["mb"] * bs)):
            b = int(clean["tables"][i * clean["mb"] + p // bs])
            dirty["v"][b, p % bs, :, 3::7] = bad
            if p >= c + n or bad != bad:
                dirty["k"][b, p % bs] = bad
    a, b = run(rt, clean), run(rt, dirty)
    for i, s0 in ((0, 0), (1, 6)):
        for r in range(lens[i]):
            if int(clean["mask"][s0 + r, 0]) >> 2 & 1:
                x = b[s0 + r].view(4, D)[:, 3::7].float()
                assert (x != x).all() if bad != bad else (x == bad).all()
            else:
                assert torch.equal(a[s0 + r], b[s0 + r]), (i, r)


def test_a_chain_is_causal_attention(rt):
    """A tree without branches is the chunk that `attention` serves."""
    from gvirt_amd._C import attention
    w = make(21, [12, 30], [100, 7], 8, 2, 128, 16, torch.bfloat16, spare=0)
    w["mask"] = torch.cat([tree_mask(list(range(-1, n - 1)), 1) for n in (12, 30)])
    got = run(rt, w)
    d = W.to_device({k: v for k, v in w.items() if isinstance(v, torch.Tensor)}, DEV)
    out = torch.zeros(42, 8 * 128, dtype=torch.bfloat16, device=DEV)
    attention(rt, d["qkv"], d["k"], d["v"], out, d["qsl"], d["lens"], d["clens"], d["tables"], 8, 2, 128, 16, 2, w["mb"])
    check(got, w)
    check(out.cpu(), w)


def test_captured_calls_replay(rt):
    """Two captured calls that share the Runtime's scratch, replayed between eager work, on inputs that change."""
    from gvirt_amd._C import Runtime, tree_attention
    r2 = Runtime(0, 64)
    r2.blocking = False
    ws = [make(s, [9, 20], [600, 40], 8, 2, 128, 16, torch.bfloat16, spare=0) for s in (1, 2)]
    want = [run(rt, w) for w in ws]
    d = [W.to_device({k: v for k, v in w.items() if isinstance(v, torch.Tensor)}, DEV) for w in ws]
    outs = [torch.zeros(29, 8 * 128, dtype=torch.bfloat16, device=DEV) for _ in ws]

    def call(i):
        x = d[i]
        tree_attention(r2, x["qkv"], x["k"], x["v"], outs[i], x["mask"], x["qsl"], x["lens"], x["clens"], x["tables"], 8, 2, 128, 16, 2, ws[i]["mb"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
        call(1)
    for turn in range(3):
        for o in outs:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0].cpu(), want[turn % 2]) and torch.equal(outs[1].cpu(), want[1 - turn % 2])
        for name in ("qkv", "k", "v", "mask", "tables"):       # the two trade their inputs
            keep = d[0][name].clone()
            d[0][name].copy_(d[1][name])
            d[1][name].copy_(keep)
        torch.matmul(torch.ones(64, 64, device=DEV), torch.ones(64, 64, device=DEV)).sum().item()


# ---- verify_tree -----------------------------------------------------------------------------------------------------

def plain_verify(logits, tokens, parents, starts, lens, max_path):
    acc, counts, nxt = [], [], []
    for s0, n in zip(starts, lens):
        path, node, token = [], 0, -1
        while n and len(path) < max_path:
            path.append(node)
            row = [float("inf") if x != x else x for x in logits[s0 + node].tolist()]
            nan = [i for i, x in enumerate(logits[s0 + node].tolist()) if x != x]
            token = nan[0] if nan else row.index(max(row))
            below = [c for c in range(node + 1, n) if parents[s0 + c] == node and tokens[s0 + c] == token]
            if not below:
                break
            node = below[0]
        acc.append(path + [-1] * (max_path - len(path)))
        counts.append(len(path))
        nxt.append(token)
    return acc, counts, nxt


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab,lens,max_path", [(1, [1], 1), (7, [5, 0, 1], 3), (33, [70, 3], 8), (1001, [9, 9, 9, 64, 0], 16), (50000, [40], 16),
                                                 (131073, [3, 12], 5)])
def test_verify_paths(rt, dtype, vocab, lens, max_path):
    from gvirt_amd._C import verify_tree
    g = torch.Generator().manual_seed(vocab)
    rnd = random.Random(vocab)
    T = sum(lens)
    parents, tokens, starts = [], [], [sum(lens[:i]) for i in range(len(lens))]
    logits = torch.randn(T, vocab, generator=g).to(dtype)      # (16-bit values repeat: ties everywhere)
    for s0, n in zip(starts, lens):
        p = [-1] + [rnd.randint(max(0, r - 4), r - 1) for r in range(1, n)]
        t = [rnd.randrange(vocab) for _ in range(n)]
        node = 0
        for _ in range(rnd.randint(0, 12)):
            below = [c for c in range(node + 1, n) if p[c] == node]
            if not below:
                break
            child = rnd.choice(below)
            logits[s0 + node, t[child]] = 30.0
            for c in below:
                if rnd.random() < 0.2:
                    t[c] = t[child]          # the same token twice: the lower child goes on
            node = child
        parents += p[:n]
        tokens += t
    if T > 2 and vocab > 20:
        logits[1, 5], logits[1, 19] = float("nan"), float("nan")
        logits[2] = float("-inf")
        logits[0, 3:9] = float("inf")
    if vocab > 6 and lens[-1] == 0 and T > 4:
        logits[4] = -0.0
        logits[4, 2] = 0.0
    want = plain_verify(logits.double(), tokens, parents, starts, lens, max_path)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    acc = torch.full((len(lens), max_path), 9, dtype=torch.int32, device=DEV)
    cnt, nxt = i32([9] * len(lens)), i32([9] * len(lens))
    verify_tree(rt, logits.to(DEV), i32(tokens), i32(parents), acc, cnt, nxt, i32(starts), i32(lens), len(lens))
    assert (acc.cpu().tolist(), cnt.cpu().tolist(), nxt.cpu().tolist()) == want


def test_verify_on_another_stream_and_captured():
    """A captured call on inputs that change between its replays."""
    from gvirt_amd._C import Runtime, verify_tree
    r2 = Runtime(0, 8)
    r2.blocking = False
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    lens, starts, parents = [3, 0, 4], [0, 3, 3], [-1, 0, 0, -1, 0, 1, 1]
    cases = []
    for seed in (1, 2, 3):
        g = torch.Generator().manual_seed(seed)
        logits, tokens = torch.randn(7, 300, generator=g), torch.randint(0, 300, (7,), generator=g)
        tokens[1 + seed % 2], tokens[4] = logits[0].argmax(), logits[3].argmax()
        cases.append((logits, tokens, plain_verify(logits.double(), tokens.tolist(), parents, starts, lens, 3)))
    logits, tokens = cases[0][0].to(DEV), cases[0][1].int().to(DEV)
    acc, cnt, nxt, par, s0, n = i32([[9] * 3] * 3), i32([9] * 3), i32([9] * 3), i32(parents), i32(starts), i32(lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_tree(r2, logits, tokens, par, acc, cnt, nxt, s0, n, 3)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert (acc.tolist(), cnt.tolist(), nxt.tolist()) == cases[0][2]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        verify_tree(r2, logits, tokens, par, acc, cnt, nxt, s0, n, 3)
    for x, t, want in cases[::-1]:
        logits.copy_(x)
        tokens.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert (acc.tolist(), cnt.tolist(), nxt.tolist()) == want
        torch.ones(1000, device=DEV).sum().item()


def test_verify_ignores_parents_that_do_not_stand_before_their_child(rt):
    from gvirt_amd._C import verify_tree
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    logits = torch.zeros(4, 8, device=DEV)
    logits[:, 5] = 1.0
    acc, cnt, nxt = i32([[0] * 6]), i32([0]), i32([0])
    verify_tree(rt, logits, i32([5, 5, 5, 5]), i32([3, 0, 99, 1]), acc, cnt, nxt, i32([0]), i32([4]), 1)
    assert acc.tolist() == [[0, 1, 3, -1, -1, -1]] and cnt.tolist() == [3] and nxt.tolist() == [5]


def test_tree_attention_refuses(rt):
    from gvirt_amd._C import tree_attention, verify_tree
    w = make(1, [4], [10], 4, 2, 64, 16, torch.bfloat16, spare=0)
    d = W.to_device({k: v for k, v in w.items() if isinstance(v, torch.Tensor)}, DEV)
    out = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV)

    def call(**kw):
        a = dict(qkv=d["qkv"], k=d["k"], v=d["v"], out=out, mask=d["mask"], qsl=d["qsl"], lens=d["lens"], clens=d["clens"], tables=d["tables"], H=4, KV=2,
                 D=64, bs=16, batch=1, mb=w["mb"])
        a.update(kw)
        scales = {n: a.pop(n, None) for n in ("k_scale", "v_scale")}
        tree_attention(rt, *a.values(), **scales)
    call()
    f = torch.zeros(w["k"].shape[:3], device=DEV)
    for kw in (dict(out=out.half()), dict(k=d["k"].half()), dict(mask=d["mask"].long()), dict(mask=d["mask"][:2]), dict(lens=d["lens"].long()),
               dict(qkv=d["qkv"].t()), dict(qkv=d["qkv"].float(), out=out.float()), dict(H=3), dict(D=32), dict(bs=0), dict(batch=2), dict(mb=50),
               dict(k_scale=f), dict(k_scale=f, v_scale=f), dict(v=d["v"].cpu()), dict(out=out[:2])):
        with pytest.raises(RuntimeError):
            call(**kw)
    i = d["lens"]
    for logits, acc in ((d["k"].view(-1, 64)[:4].double(), i.view(1, 1)), (out, i), (out[0], i.view(1, 1)), (out[:2].t(), i.view(1, 1))):
        with pytest.raises(RuntimeError):
            verify_tree(rt, logits, i.repeat(4), i.repeat(4), acc, i, i, i, i, 1)
