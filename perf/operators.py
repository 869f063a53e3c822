"""The operators of drafted trees and of cache eviction, as cases to be measured.

A serving loop that drafts a tree of tokens for every sequence runs, per step: `tree_attention` in every layer (the
drafted rows read the cache and their own ancestors), `verify_tree` once (which path of the tree the model itself would
have taken), `compact_kv_cache` in every layer (the path's rows move next to the cached ones). A loop that bounds its
cache runs `attention_weights` beside the attention (what every cached position was attended to), and now and then
`select_kept` (the positions to keep, per kv head) and `compact_kv_cache`.

`run` computes an operator in its plain form, elementary torch operations in fp32, or, where `own` is true, through
gvirt_amd. Shapes: the model shapes of gvirt_amd/workloads.py (14/2 heads of 64, 32/8 and 28/4 of 128) and the 16/4 heads
of 256 that the attention tests use; block sizes from 16 to 128, odd ones among the drawn cases.
"""
import json
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_CACHES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
_HEADS = ((14, 2, 64), (32, 8, 128), (28, 4, 128), (16, 4, 256))


# ---- the cases -------------------------------------------------------------------------------------------------------

def _tree(name, heads, block, batch, nodes, context, ragged, dtype, cache="same"):
    h, kv, d = heads
    return dict(name=name, op="tree_attention", heads=h, kv_heads=kv, head_dim=d, block=block, batch=batch, nodes=nodes,
                context=context, ragged=ragged, dtype=dtype, cache=cache)


def _weights(name, heads, block, batch, rows, window, context, ragged, dtype, cache="same"):
    h, kv, d = heads
    return dict(name=name, op="attention_weights", heads=h, kv_heads=kv, head_dim=d, block=block, batch=batch, rows=rows,
                window=window, context=context, ragged=ragged, dtype=dtype, cache=cache)


def _select(name, kv, block, batch, context, budget, recent, sink, ragged):
    return dict(name=name, op="select_kept", kv_heads=kv, block=block, batch=batch, context=context, budget=budget,
                recent=recent, sink=sink, ragged=ragged)


def _compact(name, kv, d, block, batch, context, kept, per_head, ragged, dtype, cache="same"):
    return dict(name=name, op="compact_kv_cache", kv_heads=kv, head_dim=d, block=block, batch=batch, context=context,
                kept=kept, per_head=per_head, ragged=ragged, dtype=dtype, cache=cache)


def _verify(name, batch, nodes, vocab, accept, ragged, dtype):
    return dict(name=name, op="verify_tree", batch=batch, nodes=nodes, vocab=vocab, accept=accept, ragged=ragged, dtype=dtype)


def listed():
    return [
        # one user of a small model, a tree of eight: the step is bound by its launches
        _tree("tree one sequence", (14, 2, 64), 16, 1, 8, 700, False, "fp16"),
        # a serving batch in the middle of its answers: ragged contexts, ragged trees, an odd node count
        _tree("tree ragged batch", (32, 8, 128), 128, 16, 27, 4096, True, "bf16"),
        # long contexts over a cache of bytes
        _tree("tree int8 cache", (28, 4, 128), 64, 8, 16, 16384, True, "bf16", "int8"),
        # a full batch with wide trees: 2 GB of cache per pass
        _tree("tree full batch", (32, 8, 128), 128, 64, 32, 8192, False, "bf16"),
        # a decode step of a batch that bounds its caches: every step adds one row's weights
        _weights("weights decode step", (32, 8, 128), 128, 64, 1, 0, 4096, True, "bf16"),
        # a whole prefill chunk behind cached positions, every row counted
        _weights("weights prefill chunk", (28, 4, 128), 128, 2, 2048, 0, 6144, False, "bf16"),
        # one sequence just over its budget
        _select("select one sequence", 2, 16, 1, 711, 512, 64, 4, False),
        # a full batch of long prompts cut to an eighth
        _select("select full batch", 8, 128, 64, 32768, 4096, 1024, 4, True),
        # the accepted path of every sequence's tree moves next to its cached rows
        _compact("compact accepted paths", 8, 128, 128, 64, 4096, 6, False, True, "bf16"),
        # prompts cut down per kv head
        _compact("compact after eviction", 8, 128, 128, 16, 8192, 2048, True, True, "bf16"),
        # one user, a small tree: a call as long as its launches
        _verify("verify one sequence", 1, 8, 32000, 3, False, "fp16"),
        # which paths the model agrees with: a batch of trees over a large vocabulary
        _verify("verify full batch", 64, 32, 131072, 4, True, "bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("tree", "tree", "tree", "weights", "weights", "select", "compact", "verify"))
    heads = rng.choice(_HEADS)
    block = rng.choice((16, 24, 32, 48, 64, 128))
    dtype = rng.choice(("bf16", "fp16"))
    ragged = rng.random() < 0.7
    cache = rng.choice(("same", "same", "int8", "fp8")) if heads[2] <= 128 else "same"
    if op == "tree":
        batch, nodes = _log(rng, 1, 64), _log(rng, 1, 96)
        context = _log(rng, 16, max(16, min(32768, 524288 // batch, 16777216 // (batch * nodes))))
        return _drop(_tree("", heads, block, batch, nodes, context, ragged, dtype, cache))
    if op == "weights":
        batch, rows = _log(rng, 1, 64), rng.choice((1, 1, _log(rng, 2, 2048)))
        context = _log(rng, 16, max(16, min(32768, 262144 // batch, 16777216 // (batch * rows))))
        window = rng.choice((0, min(rows, _log(rng, 1, 128))))
        return _drop(_weights("", heads, block, batch, rows, window, context, ragged, dtype, cache))
    if op == "select":
        batch, kv = _log(rng, 1, 64), rng.choice((1, 2, 4, 8))
        context = _log(rng, 64, 40000)
        budget = _log(rng, 16, context + 10)
        sink = rng.choice((0, 4))
        return _drop(_select("", kv, block, batch, context, budget, rng.randrange(0, budget - sink + 1), sink, ragged))
    if op == "compact":
        batch, per_head = _log(rng, 1, 64), rng.random() < 0.5
        context = _log(rng, 64, max(64, min(16384, 262144 // batch)))
        kept = _log(rng, 1, context) if per_head else _log(rng, 1, 16)
        return _drop(_compact("", heads[1], heads[2], block, batch, context, kept, per_head, ragged, dtype, cache))
    batch, nodes = _log(rng, 1, 64), _log(rng, 1, 96)
    vocab = _log(rng, 1000, min(160000, 268435456 // (batch * nodes)))
    return _drop(_verify("", batch, nodes, vocab, rng.randrange(1, 8), ragged, rng.choice(("bf16", "fp16", "fp32"))))


def _drop(case):
    del case["name"]
    return case


def _plan(case):
    """The lengths of a case, the same for every seed: (context lengths, rows of the step) per sequence."""
    rng = random.Random(json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True))
    b, ragged = case["batch"], case["ragged"]
    rows = case.get("nodes") or case.get("rows") or 1
    ctx = case.get("context", 0)
    ctxs = [rng.randint(max(1, ctx // 4), ctx) if ragged and ctx else ctx for _ in range(b)]
    lens = [rng.randint(1, rows) if ragged else rows for _ in range(b)]
    ctxs[0], lens[0] = ctx, rows   # the longest is always there
    return ctxs, lens


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _parents(rng, n):
    """A drafted tree: node 0 is the sequence's last token, every other node hangs on one of the eight before it."""
    return [-1] + [rng.randrange(max(0, c - 8), c) for c in range(1, n)]


def _ancestors(parents, words):
    """Bit j of row r: node j is r or one of its ancestors."""
    bits = []
    for r, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | (1 << r))
    raw = b"".join(x.to_bytes(4 * words, "little") for x in bits)
    return np.frombuffer(raw, dtype=np.int32).reshape(len(parents), words)


def _pages(case, totals, gen):
    bs = case["block"]
    per = [-(-t // bs) for t in totals]
    most = max(per)
    perm = torch.randperm(sum(per) + 2, generator=gen, device="cuda").to(torch.int32)
    tables = torch.zeros(len(per), most, dtype=torch.int32, device="cuda")
    at = np.concatenate([[0], np.cumsum(per)]).tolist()
    for i, n in enumerate(per):
        tables[i, :n] = perm[at[i]:at[i] + n]
    return tables, most, int(perm.numel())


def _filled(shape, gen, dtype):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for s in range(0, flat.numel(), 1 << 27):
        piece = flat[s:s + (1 << 27)]
        piece.copy_(torch.randn(piece.numel(), generator=gen, device="cuda", dtype=torch.float32))
    return out


def _cache(case, blocks, gen):
    """One cache tensor [blocks, block, kv_heads, head_dim] and the fp32 scales of its rows (a cache of bytes) or None."""
    shape = (blocks, case["block"], case["kv_heads"], case["head_dim"])
    if case["cache"] == "same":
        return _filled(shape, gen, _TYPES[case["dtype"]]), None
    scale = torch.rand(shape[:3], generator=gen, device="cuda") * 0.02 + 0.01
    if case["cache"] == "int8":
        q = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
    else:
        q = _filled(shape, gen, torch.float32).mul_(100.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return q, scale


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    ctxs, lens = _plan(case)
    op, b = case["op"], case["batch"]
    s = dict(op=op, case=case, batch=b)
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]]).tolist()
    s.update(query_start_loc=_int(starts), lens=_int(lens), cached_lens=_int(ctxs), rows=max(lens), total_rows=sum(lens))
    if op in ("tree_attention", "attention_weights"):
        h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
        totals = [c + n for c, n in zip(ctxs, lens)]
        s["tables"], s["max_num_block"], blocks = _pages(case, totals, gen)
        s["k_cache"], s["k_scale"] = _cache(case, blocks, gen)
        # queries as rope_and_cache leaves them, scaled by head_dim^-0.5; scores of a standard deviation of two
        # (a cache of bytes has rows of about one unit and a quarter)
        s["qkv"] = _filled((sum(lens), h + 2 * kv, d), gen, torch.float32).mul_(2 * d ** -0.5).to(_TYPES[case["dtype"]]).view(sum(lens), -1)
        s["positions"] = max(totals)
        if op == "tree_attention":
            s["v_cache"], s["v_scale"] = _cache(case, blocks, gen)
            words = -(-max(lens) // 32)
            s["tree_mask"] = torch.from_numpy(np.concatenate([_ancestors(_parents(rng, n), words) for n in lens])).cuda()
            s["output"] = torch.zeros(sum(lens), h * d, dtype=_TYPES[case["dtype"]], device="cuda")
        else:
            s["weights"] = torch.rand(blocks, case["block"], kv, generator=gen, device="cuda")
    elif op == "select_kept":
        kv = case["kv_heads"]
        s["tables"], s["max_num_block"], blocks = _pages(case, ctxs, gen)
        # what a run of steps leaves: most positions little, some much
        s["weights"] = torch.rand(blocks, case["block"], kv, generator=gen, device="cuda").pow_(8.0).mul_(20.0)
        s["context_lens"], s["positions"] = _int(ctxs), max(ctxs)
        s["kept"] = torch.zeros(b, kv, case["budget"], dtype=torch.int32, device="cuda")
        s["kept_lens"] = torch.zeros(b, dtype=torch.int32, device="cuda")
    elif op == "compact_kv_cache":
        kv, d, n = case["kv_heads"], case["head_dim"], case["kept"]
        room = 2 * n + 8 if not case["per_head"] else 0   # a tree's rows behind the cached ones
        s["tables"], s["max_num_block"], blocks = _pages(case, [c + room for c in ctxs], gen)
        s["k_cache"], s["k_scale"] = _cache(case, blocks, gen)
        s["v_cache"], s["v_scale"] = _cache(case, blocks, gen)
        s["weights"] = None
        host = np.random.default_rng(seed)
        if case["per_head"]:
            lists = np.full((b, kv, n), -1, dtype=np.int32)
            counts = [min(n, c) for c in ctxs]
            for i, c in enumerate(ctxs):
                for j in range(kv):
                    lists[i, j, :counts[i]] = np.sort(host.choice(c, counts[i], replace=False))
            s["starts"], s["weights"] = None, torch.rand(blocks, case["block"], kv, generator=gen, device="cuda")
        else:
            lists = np.full((b, n), -1, dtype=np.int32)
            counts = [int(host.integers(1, n + 1)) if case["ragged"] else n for _ in ctxs]
            for i in range(b):
                lists[i, 1:counts[i]] = np.sort(1 + host.choice(room - 1, counts[i] - 1, replace=False))
                lists[i, 0] = 0
            s["starts"] = _int(ctxs)
        s["kept"], s["kept_lens"] = torch.from_numpy(lists).cuda(), _int(counts)
    else:
        t, v = sum(lens), case["vocab"]
        s["logits"] = _filled((t, v), gen, _TYPES[case["dtype"]])
        tokens = np.random.default_rng(seed).integers(0, v, t).astype(np.int32)
        parents, at, what = [], [], []
        for i, n in enumerate(lens):
            p = _parents(rng, n)
            node = 0
            for _ in range(case["accept"] - 1):     # the path that the model will agree with
                below = [c for c in range(node + 1, n) if p[c] == node]
                if not below:
                    break
                child = rng.choice(below)
                at.append(starts[i] + node)
                what.append(int(tokens[starts[i] + child]))
                node = child
            parents += p
        if at:
            s["logits"][torch.tensor(at, device="cuda"), torch.tensor(what, device="cuda")] = 16.0
        s["tokens"], s["parents"] = torch.from_numpy(tokens).cuda(), _int(parents)
        s["accepted"] = torch.zeros(b, 16, dtype=torch.int32, device="cuda")
        s["n_accepted"] = torch.zeros(b, dtype=torch.int32, device="cuda")
        s["next_token"] = torch.zeros(b, dtype=torch.int32, device="cuda")
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _slots(s):
    """The slot of every position of every sequence, [batch, positions]; padded with slots of block 0."""
    bs = s["case"]["block"]
    pos = torch.arange(s["positions"], device="cuda")
    return s["tables"].long()[:, pos // bs] * bs + pos % bs, pos


def _rows32(cache, scale, slots):
    """Cache rows of the slots in fp32, [batch, kv_heads, positions, head_dim]."""
    rows = cache.view(-1, *cache.shape[2:])[slots].float()
    if scale is not None:
        rows = rows * scale.view(-1, scale.shape[-1])[slots].unsqueeze(-1)
    return rows.permute(0, 2, 1, 3).contiguous()


def _queries(s, first, rows):
    """Rows first .. first + rows - 1 of every sequence's step in fp32, [batch, kv_heads, group * rows, head_dim]."""
    c = s["case"]
    at = s["query_start_loc"].long()[:, None] + first + torch.arange(rows, device="cuda")
    q = s["qkv"].view(s["total_rows"], -1, c["head_dim"])[at.clamp(0, s["total_rows"] - 1), :c["heads"]].float()
    g = c["heads"] // c["kv_heads"]
    return q.view(s["batch"], rows, c["kv_heads"], g, c["head_dim"]).permute(0, 2, 3, 1, 4).reshape(s["batch"], c["kv_heads"], g * rows, -1), at


def _softmax(scores, seen):
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e, total


def _plain_tree(s):
    c, rows = s["case"], s["rows"]
    g = c["heads"] // c["kv_heads"]
    slots, pos = _slots(s)
    k, v = _rows32(s["k_cache"], s["k_scale"], slots), _rows32(s["v_cache"], s["v_scale"], slots)
    q, at = _queries(s, 0, rows)
    off = pos[None, :] - s["cached_lens"].long()[:, None]                     # the node of a position
    words = s["tree_mask"][at.clamp(0, s["total_rows"] - 1)].long()           # [batch, rows, words]
    word = (off // 32).clamp(0, words.shape[-1] - 1)
    bit = (torch.gather(words, 2, word[:, None, :].expand(-1, rows, -1)) >> (off % 32)[:, None, :]) & 1
    seen = (off < 0)[:, None, :] | ((off >= 0) & (off < s["lens"].long()[:, None]))[:, None, :] & (bit == 1)
    scores = torch.matmul(q, k.transpose(2, 3)).view(s["batch"], c["kv_heads"], g, rows, -1)
    e, total = _softmax(scores, seen[:, None, None])
    out = torch.matmul(e.view(s["batch"], c["kv_heads"], g * rows, -1), v).view(s["batch"], c["kv_heads"], g, rows, -1)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).permute(0, 3, 1, 2, 4)      # [batch, rows, kv, g, d]
    token = torch.arange(s["total_rows"], device="cuda")
    seq = torch.searchsorted(s["query_start_loc"].long(), token, right=True) - 1
    s["output"].copy_(out[seq, token - s["query_start_loc"].long()[seq]].reshape(s["total_rows"], -1))
    return s["output"]


def _plain_weights(s):
    c = s["case"]
    g, kv = c["heads"] // c["kv_heads"], c["kv_heads"]
    lens, cached = s["lens"].long()[:, None], s["cached_lens"].long()[:, None]
    rows = min(s["rows"], c["window"]) if c["window"] else s["rows"]
    first = (lens - rows).clamp(min=0) if c["window"] else torch.zeros_like(lens)
    slots, pos = _slots(s)
    k = _rows32(s["k_cache"], s["k_scale"], slots)
    q, at = _queries(s, first, rows)
    r = first + torch.arange(rows, device="cuda")                             # the row of the step, [batch, rows]
    seen = pos[None, None, :] <= (cached + r)[:, :, None]
    e, total = _softmax(torch.matmul(q, k.transpose(2, 3)).view(s["batch"], kv, g, rows, -1), seen[:, None, None])
    e = e.mul_(torch.where(r < lens, 1.0, 0.0)[:, None, None, :, None] / total)
    sums = e.sum(dim=(2, 3)).transpose(1, 2)                                  # [batch, positions, kv]
    flat = s["weights"].view(-1, kv)
    sums = torch.where((pos[None] < cached)[..., None], sums, sums - flat[slots])     # the step's own positions start at zero
    sums = torch.where((pos[None] < cached + lens)[..., None], sums, torch.zeros_like(sums))
    flat.index_add_(0, slots.reshape(-1), sums.reshape(-1, kv))
    return s["weights"]


def _plain_select(s):
    c, length = s["case"], s["context_lens"].long()[:, None, None]
    slots, pos = _slots(s)
    w = s["weights"].view(-1, c["kv_heads"])[slots].transpose(1, 2)           # [batch, kv, positions]
    always = (pos < c["sink"]) | (pos >= length - c["recent"])
    w = torch.where(always, math.inf, w).masked_fill(pos >= length, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :c["budget"]]
    order = torch.where(order < length, order, s["positions"])
    kept = torch.sort(order, dim=-1).values
    s["kept"].fill_(-1)
    s["kept"][..., :kept.shape[-1]] = torch.where(kept < s["positions"], kept, -1).int()
    s["kept_lens"].copy_(s["context_lens"].clamp(max=c["budget"]))
    return [s["kept"], s["kept_lens"]]


def _plain_compact(s):
    c = s["case"]
    kv, bs, n = c["kv_heads"], c["block"], c["kept"]
    count = s["kept_lens"].long()[:, None, None]
    i = torch.arange(n, device="cuda")
    i = torch.minimum(i, (count - 1).clamp(min=0))                            # past the end: the last one again
    lists = s["kept"].long().view(s["batch"], -1, n)
    src = torch.where(count > 0, torch.gather(lists, 2, i.expand(-1, lists.shape[1], -1)), 0).expand(-1, kv, -1)
    dst = i.expand(-1, kv, -1)
    if s["starts"] is not None:
        src, dst = src + s["starts"].long()[:, None, None], dst + s["starts"].long()[:, None, None]
    head = torch.arange(kv, device="cuda")[None, :, None]
    batch = torch.arange(s["batch"], device="cuda")[:, None, None]

    def row(p):
        return (s["tables"].long()[batch, p // bs] * bs + p % bs) * kv + head

    src, dst = row(src).reshape(-1), row(dst).reshape(-1)
    out = []
    for name in ("k_cache", "v_cache", "k_scale", "v_scale", "weights"):
        if s[name] is not None:
            t = s[name].view(-1, c["head_dim"]) if name.endswith("cache") else s[name].view(-1)
            t = t.view(torch.uint8) if t.dtype in (torch.int8, torch.float8_e4m3fn) else t
            t[dst] = t[src]
            out.append(s[name])
    return out


def _plain_verify(s):
    b, rows = s["batch"], s["rows"]
    choice = s["logits"].argmax(-1).int()
    at = (s["query_start_loc"].long()[:, None] + torch.arange(rows, device="cuda"))
    here = torch.arange(rows, device="cuda") < s["lens"][:, None]
    at = at.clamp(max=s["total_rows"] - 1)
    tokens, parents, choice = s["tokens"][at], s["parents"][at], choice[at]
    node, on = torch.zeros(b, dtype=torch.long, device="cuda"), s["lens"] > 0
    nodes = torch.arange(rows, device="cuda")[None]
    s["accepted"].fill_(-1)
    s["n_accepted"].zero_()
    s["next_token"].fill_(-1)
    for i in range(s["accepted"].shape[1]):
        s["accepted"][:, i] = torch.where(on, node, -1).int()
        s["n_accepted"].add_(on.int())
        want = choice.gather(1, node[:, None])
        s["next_token"].copy_(torch.where(on, want[:, 0], s["next_token"]))
        below = here & (parents == node[:, None]) & (tokens == want) & (nodes > node[:, None])
        on = on & below.any(1)
        node = torch.where(on, torch.where(below, nodes, rows).amin(1), node)
    return [s["accepted"], s["n_accepted"], s["next_token"]]


# ---- the framework's operators -----------------------------------------------------------------------------------------

_runtime = None


def _own(s):
    global _runtime
    from gvirt_amd import _C
    if _runtime is None:
        _runtime = _C.Runtime(0, 64)
        _runtime.blocking = False
    rt, c, b = _runtime, s["case"], s["batch"]
    if s["op"] == "tree_attention":
        _C.tree_attention(rt, s["qkv"], s["k_cache"], s["v_cache"], s["output"], s["tree_mask"], s["query_start_loc"], s["lens"],
                          s["cached_lens"], s["tables"], c["heads"], c["kv_heads"], c["head_dim"], c["block"], b,
                          s["max_num_block"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return s["output"]
    if s["op"] == "attention_weights":
        _C.attention_weights(rt, s["qkv"], s["k_cache"], s["weights"], s["query_start_loc"], s["lens"], s["cached_lens"],
                             s["tables"], c["heads"], c["kv_heads"], c["head_dim"], c["block"], b, s["max_num_block"],
                             c["window"], k_scale=s["k_scale"])
        return s["weights"]
    if s["op"] == "select_kept":
        _C.select_kept(rt, s["weights"], s["kept"], s["kept_lens"], s["context_lens"], s["tables"], c["kv_heads"], c["block"],
                       b, s["max_num_block"], c["budget"], c["recent"], c["sink"])
        return [s["kept"], s["kept_lens"]]
    if s["op"] == "compact_kv_cache":
        _C.compact_kv_cache(rt, s["k_cache"], s["v_cache"], s["kept"], s["kept_lens"], s["tables"], c["kv_heads"],
                            c["head_dim"], c["block"], b, s["max_num_block"], starts=s["starts"], weights=s["weights"],
                            k_scale=s["k_scale"], v_scale=s["v_scale"])
        return [s[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale", "weights") if s[n] is not None]
    _C.verify_tree(rt, s["logits"], s["tokens"], s["parents"], s["accepted"], s["n_accepted"], s["next_token"],
                   s["query_start_loc"], s["lens"], b)
    return [s["accepted"], s["n_accepted"], s["next_token"]]


_PLAIN = {"tree_attention": _plain_tree, "attention_weights": _plain_weights, "select_kept": _plain_select,
          "compact_kv_cache": _plain_compact, "verify_tree": _plain_verify}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    ctxs, lens = _plan(case)
    op = case["op"]
    elt = {"int8": 1, "fp8": 1}.get(case.get("cache"), 2)
    row = case.get("kv_heads", 0) * (case.get("head_dim", 0) * elt + (4 if elt == 1 else 0))   # a position of K or V
    if op == "tree_attention":
        width = case["heads"] * case["head_dim"]
        pairs = sum(n * c + n * n // 2 for c, n in zip(ctxs, lens))
        return {"bytes": sum(c + n for c, n in zip(ctxs, lens)) * row * 2 + sum(lens) * width * 4, "flops": 4 * width * pairs}
    if op == "attention_weights":
        width = case["heads"] * case["head_dim"]
        counted = [min(n, case["window"]) if case["window"] else n for n in lens]
        pairs = sum(m * (c + n) - m * m // 2 for c, n, m in zip(ctxs, lens, counted))
        spots = sum(c + n for c, n in zip(ctxs, lens))
        return {"bytes": spots * (row + 8 * case["kv_heads"]) + sum(counted) * width * 2, "flops": 2 * width * pairs}
    if op == "select_kept":
        return {"bytes": 4 * case["kv_heads"] * (sum(ctxs) + sum(min(c, case["budget"]) for c in ctxs)), "flops": 0}
    if op == "compact_kv_cache":
        if case["per_head"]:   # a random list moves nearly all of its rows, unless it keeps everything
            moved = sum(min(case["kept"], c) for c in ctxs if c > case["kept"])
            return {"bytes": 4 * moved * row + 8 * moved * case["kv_heads"] + 4 * len(ctxs) * case["kept"], "flops": 0}
        moved = len(ctxs) * max(case["kept"] - 1, 1) / (2 if case["ragged"] else 1)
        return {"bytes": 4 * moved * row + 4 * len(ctxs) * case["kept"], "flops": 0}
    width = {"fp32": 4}.get(case["dtype"], 2) * case["vocab"]
    return {"bytes": sum(min(n, case["accept"]) for n in lens) * width + 8 * sum(lens), "flops": 0}


# ---- the definition, in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] not in ("tree_attention", "attention_weights"):
        return None     # copies and whole numbers
    s = prepare(case, seed)
    h, kv, d, bs = case["heads"], case["kv_heads"], case["head_dim"], case["block"]
    g = h // kv
    ctxs, lens = _plan(case)
    out = torch.zeros(sum(lens), h, d, dtype=torch.float64, device="cuda")
    new = s["weights"].double() if case["op"] == "attention_weights" else None
    t0 = 0
    for b, (c, n) in enumerate(zip(ctxs, lens)):
        pages = s["tables"][b, :-(-(c + n) // bs)].long()
        key = s["k_cache"][pages].reshape(-1, kv, d)[:c + n].double()
        if s["k_scale"] is not None:
            key = key * s["k_scale"][pages].reshape(-1, kv, 1)[:c + n].double()
        query = s["qkv"][t0:t0 + n, :h * d].view(n, h, d).double()
        if new is None:
            val = s["v_cache"][pages].reshape(-1, kv, d)[:c + n].double()
            if s["v_scale"] is not None:
                val = val * s["v_scale"][pages].reshape(-1, kv, 1)[:c + n].double()
            words = s["tree_mask"][t0:t0 + n].cpu().numpy().astype("<i4").view(np.uint8)
            tree = torch.from_numpy(np.unpackbits(words, axis=1, bitorder="little")[:, :n]).bool().cuda()
            hidden = torch.cat([torch.zeros(n, c, dtype=torch.bool, device="cuda"), ~tree], dim=1)
            for j in range(h):
                p = torch.softmax((query[:, j] @ key[:, j // g].T).masked_fill(hidden, -math.inf), dim=1)
                out[t0:t0 + n, j] = p @ val[:, j // g]
        else:
            m = min(n, case["window"]) if case["window"] else n
            later = torch.arange(c + n, device="cuda")[None] > (c + n - m + torch.arange(m, device="cuda"))[:, None]
            spots = (pages[:, None] * bs + torch.arange(bs, device="cuda")).reshape(-1)[:c + n]
            flat = new.view(-1, kv)
            flat[spots[c:]] = 0
            for j in range(h):
                p = torch.softmax((query[n - m:, j] @ key[:, j // g].T).masked_fill(later, -math.inf), dim=1)
                flat[spots, j // g] += p.sum(0)
        t0 += n
    return out.view(sum(lens), h * d) if new is None else new
