"""A small decoder stack over the attention layers, and the greedy generation loop of the reference's harness.

Mirrors the attention side of `xlite/tests/generate.py:52-103` (`generate`: a rectangular token matrix, one
prefill of the shortest prompt's length, then one position per step, prompts longer than that forced) and of
`xlite/tests/models/llama.py:640-651`, `:419-427` (`prepare_xlite_attnmeta` + `forward_xlite`: the step's
`ModelAttnMeta`, every layer over the paged caches, logits of each sequence's last token). `generate_ragged`
is the serving-shaped variant: one ragged prefill of every whole prompt, then decode steps. Two loops have no counterpart
in the reference: `generate_tree` (drafted trees verified in one step) and `generate_evicting` (caches kept to a budget).

The stack is attention only: x += Attention(RMSNorm(x)) per layer, a final RMSNorm and the vocabulary
projection; the reference's feed-forward blocks, sampling and weight loading are outside this package's
path. Norms, embedding and projections are torch operations; the attention layers run this package's operators
(`MhaLayer` or `MlaLayer`), and the metadata goes through `prepare_attn_meta` exactly as `XRuntime::PrepareAttn`
(xlite/csrc/runtime.cpp:404-550) derives it from the lists.
"""
from typing import Callable, List, Optional, Sequence, Tuple

import torch

from . import _C
from .mha import MhaLayer, StepMeta, prepare_attn, prepare_attn_meta, prepare_tree
from .mla import MlaLayer


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * weight.float()).to(x.dtype)


class DecoderModel:
    """`layers`: MhaLayer or MlaLayer objects (all of one kind); `norms`: one RMSNorm weight [hidden] per layer and
    a final one; `embed` [vocab, hidden]; `lm_head` [hidden, vocab]; `rope`: the cos|sin table of `rope_and_cache`
    (MHA) or the complex `freqs` of `mla_prepare` (MLA). Every sequence of a batch owns `ceil(max_seq_len /
    block_size)` consecutive physical blocks, as the reference's harness lays them out."""

    def __init__(self, rt: _C.Runtime, layers: Sequence, norms: Sequence[torch.Tensor], embed: torch.Tensor,
                 lm_head: torch.Tensor, rope: torch.Tensor, max_batch: int, max_seq_len: int, norm_eps: float = 1e-6):
        if len(norms) != len(layers) + 1:
            raise RuntimeError("DecoderModel: one norm per layer and a final one")
        self.rt, self.layers, self.norms, self.embed, self.lm_head, self.rope = rt, list(layers), list(norms), embed, lm_head, rope
        self.max_batch, self.max_seq_len, self.norm_eps = max_batch, max_seq_len, norm_eps
        cfg = layers[0].cfg
        self.block_size = cfg.block_size
        self.blocks_per_seq = (max_seq_len + cfg.block_size - 1) // cfg.block_size
        nb = max_batch * self.blocks_per_seq
        dev, dt = embed.device, embed.dtype
        self.is_mla = isinstance(layers[0], MlaLayer)
        if self.is_mla:
            self.caches = [(torch.zeros(nb, cfg.block_size, cfg.kv_lora_rank, dtype=dt, device=dev),
                            torch.zeros(nb, cfg.block_size, cfg.rope_head_dim, dtype=dt, device=dev)) for _ in layers]
        else:
            self.caches = [(torch.zeros(nb, cfg.block_size, cfg.n_kv_heads, cfg.head_dim, dtype=dt, device=dev),
                            torch.zeros(nb, cfg.block_size, cfg.n_kv_heads, cfg.head_dim, dtype=dt, device=dev)) for _ in layers]

    def check_batch(self, batch: int, longest: int) -> None:
        """The caches hold `max_batch` sequences of `max_seq_len` positions: anything beyond would be written and
        read outside them."""
        if batch > self.max_batch:
            raise RuntimeError("DecoderModel: batch of %d sequences exceeds max_batch=%d" % (batch, self.max_batch))
        if longest > self.max_seq_len:
            raise RuntimeError("DecoderModel: a sequence of %d positions exceeds max_seq_len=%d" % (longest, self.max_seq_len))

    def attn_meta(self, lens: Sequence[int], cached_lens: Sequence[int]) -> _C.ModelAttnMeta:
        """The step's host lists (xlite/tests/models/llama.py:640-651): sequence i uses blocks i * blocks_per_seq ..."""
        meta = _C.ModelAttnMeta()
        meta.lens = [int(x) for x in lens]
        meta.cached_lens = [int(x) for x in cached_lens]
        self.check_batch(len(meta.lens), max((l + c for l, c in zip(meta.lens, meta.cached_lens)), default=0))
        meta.block_tables = [[i * self.blocks_per_seq + b for b in range((l + c + self.block_size - 1) // self.block_size)]
                             for i, (l, c) in enumerate(zip(meta.lens, meta.cached_lens))]
        return meta

    def forward_tokens(self, tokens: torch.Tensor, lens: Sequence[int], cached_lens: Sequence[int]) -> torch.Tensor:
        """`tokens`: the step's token ids, sequence after sequence (sum(lens) of them). Returns the logits of every
        sequence's last token, [batch, vocab] in fp32. Sequences without tokens this step get a row of zeros."""
        meta = prepare_attn_meta(self.attn_meta(lens, cached_lens), self.block_size, self.embed.device)
        return self._last_logits(self._rows(tokens, meta), lens)

    def _rows(self, tokens: torch.Tensor, meta: StepMeta, weights: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
        """The step's normalised hidden rows; `weights`: what every layer's cached positions were attended to, updated."""
        x = self.embed[tokens.long()]
        for i, (layer, norm, (c0, c1)) in enumerate(zip(self.layers, self.norms, self.caches)):
            h = rms_norm(x, norm, self.norm_eps)
            more = {} if weights is None else {"weights": weights[i]}
            x = x + layer.forward(self.rt, h, c0, c1, meta, self.rope, **more)
        return rms_norm(x, self.norms[-1], self.norm_eps)

    def _last_logits(self, x: torch.Tensor, lens: Sequence[int]) -> torch.Tensor:
        ends, rows = [], []
        off = 0
        for i, l in enumerate(lens):
            off += int(l)
            if l > 0:
                ends.append(off - 1)
                rows.append(i)
        logits = torch.zeros(len(lens), self.lm_head.shape[1], dtype=torch.float32, device=x.device)
        if rows:
            last = x[torch.tensor(ends, device=x.device)]
            logits[torch.tensor(rows, device=x.device)] = torch.matmul(last, self.lm_head).float()
        return logits

    def tree_tables(self, lens: Sequence[int], cached_lens: Sequence[int]) -> List[List[int]]:
        return self.attn_meta(lens, cached_lens).block_tables

    def forward_tree(self, tokens: torch.Tensor, lens: Sequence[int], cached_lens: Sequence[int],
                     parents: Sequence[Sequence[int]]) -> Tuple[torch.Tensor, StepMeta]:
        """A step over drafted trees (multi-head layers): `parents` as in `prepare_tree`. The logits of every node, fp32
        [sum(lens), vocab], and the step's metadata."""
        if self.is_mla:
            raise RuntimeError("DecoderModel: drafted trees need multi-head attention layers")
        meta = prepare_tree(lens, cached_lens, self.tree_tables(lens, cached_lens), self.block_size, parents, self.embed.device)
        return torch.matmul(self._rows(tokens, meta), self.lm_head).float(), meta

    def forward(self, tokens: torch.Tensor, start_pos: int = 0) -> torch.Tensor:
        """The reference model's call shape (xlite/tests/models/llama.py:419-427): `tokens` [batch, seqlen], every
        sequence with `start_pos` cached tokens."""
        batch, seqlen = tokens.shape
        return self.forward_tokens(tokens.reshape(-1), [seqlen] * batch, [start_pos] * batch)


def generate(model: DecoderModel, prompt_tokens: List[List[int]], max_new_tokens: int, eos_id: int,
             temperature: float = 0.0) -> Tuple[List[List[int]], int]:
    """The rectangular loop of the reference's harness (xlite/tests/generate.py:52-103), greedy: the first call
    feeds every sequence the shortest prompt's length, every later call one position of every sequence; where a
    prompt still has a token for the position, that token stands and the model's choice is dropped. Sequences
    keep stepping after their end token so that the batch stays rectangular; the answer of each is cut at its
    first end token. Returns the new tokens per sequence and the number of model calls."""
    if temperature > 0:
        raise RuntimeError("generate: only greedy selection (temperature 0) is built")
    n = len(prompt_tokens)
    longest = max(len(t) for t in prompt_tokens)
    if longest > model.max_seq_len:
        raise RuntimeError("Prompt length exceeds model maximum sequence length (max_seq_len=%d)" % model.max_seq_len)
    model.check_batch(n, longest)
    horizon = min(model.max_seq_len, longest + max_new_tokens)
    known = [[int(x) for x in t] for t in prompt_tokens]     # per sequence: the prompt, then what was chosen
    ended = [False] * n
    fed, calls = 0, 0
    dev = model.embed.device
    for pos in range(min(len(t) for t in known), horizon):
        # every sequence holds at least `pos` tokens here: the columns fed .. pos - 1 of the token matrix
        window = torch.tensor([k[fed:pos] for k in known], dtype=torch.int32, device=dev)
        choice = model.forward(window, fed).argmax(dim=-1).tolist()
        calls += 1
        for i, k in enumerate(known):
            if len(k) == pos:          # the prompt is used up: the model's token is the sequence's next one
                k.append(int(choice[i]))
                ended[i] = ended[i] or k[-1] == eos_id
        fed = pos
        if all(ended):
            break
    answers = []
    for k, t in zip(known, prompt_tokens):
        new = k[len(t): len(t) + max_new_tokens]
        answers.append(new[: new.index(eos_id)] if eos_id in new else new)
    return answers, calls


def generate_ragged(model: DecoderModel, prompt_tokens: List[List[int]], max_new_tokens: int, eos_id: int) -> Tuple[List[List[int]], int]:
    """One ragged prefill of every whole prompt, then one decode step per new token (a sequence that has produced
    `eos_id` takes no further part: its length for the step is 0). Greedy."""
    dev = model.embed.device
    n = len(prompt_tokens)
    cached = [0] * n
    pending = [list(t) for t in prompt_tokens]     # tokens to feed next, per sequence
    out: List[List[int]] = [[] for _ in range(n)]
    done = [False] * n
    step = 0
    for _ in range(max_new_tokens):
        lens = [len(p) for p in pending]
        if sum(lens) == 0:
            break
        flat = torch.tensor([t for p in pending for t in p], dtype=torch.int32, device=dev)
        logits = model.forward_tokens(flat, lens, cached)
        nxt = logits.argmax(dim=-1).tolist()
        step += 1
        for i in range(n):
            cached[i] += lens[i]
            pending[i] = []
            if lens[i] == 0 or done[i]:
                continue
            if nxt[i] == eos_id or cached[i] + 1 > model.max_seq_len:
                done[i] = True
                continue
            out[i].append(int(nxt[i]))
            pending[i] = [int(nxt[i])]
    return out, step


def generate_tree(model: DecoderModel, prompt_tokens: List[List[int]], draft: Callable[[List[int]], Tuple[List[int], List[int]]],
                  max_new_tokens: int, eos_id: int, max_path: int = 16) -> Tuple[List[List[int]], int]:
    """Greedy generation with drafted trees: the tokens of `generate_ragged` in fewer steps. `draft(tokens so far)` returns
    (tokens, parents) of the drafted nodes: node 0 is the sequence's last token, drafted node i (from 1 on) hangs on node
    parents[i - 1] < i. A step runs all trees through the model (`tree_attention` in every layer), keeps the path that
    greedy decoding takes (`verify_tree`) and moves its cache rows next to the cached ones (`compact_kv_cache`): the path's
    tokens and one more. Multi-head layers."""
    dev, n, rt = model.embed.device, len(prompt_tokens), model.rt
    if model.is_mla:
        raise RuntimeError("generate_tree: drafted trees need multi-head attention layers")
    out: List[List[int]] = [[] for _ in range(n)]
    cached = [len(t) for t in prompt_tokens]
    live = [c > 0 for c in cached]               # (nothing follows an empty prompt, as in generate_ragged)
    if not any(live) or max_new_tokens <= 0:
        return out, 0
    flat = torch.tensor([t for p in prompt_tokens for t in p], dtype=torch.int32, device=dev)
    last = model.forward_tokens(flat, cached, [0] * n).argmax(dim=-1).tolist()     # not in the cache yet
    step = 1

    def take(i: int, token: int) -> None:
        if not live[i]:
            return
        if token == eos_id or len(out[i]) >= max_new_tokens:
            live[i] = False
            return
        out[i].append(int(token))
        live[i] = len(out[i]) < max_new_tokens

    for i in range(n):      # (a token that the cache has no room for is not taken, as in generate_ragged)
        live[i] = live[i] and cached[i] + 1 <= model.max_seq_len
        take(i, last[i])
    while any(live):
        tokens, parents = [], []
        for i in range(n):
            if not live[i]:
                tokens.append([])
                parents.append([])
                continue
            t, p = draft(list(prompt_tokens[i]) + out[i])
            if len(t) != len(p) or any(not 0 <= int(x) <= k for k, x in enumerate(p)):
                raise RuntimeError("generate_tree: a drafted node hangs on a node before it")
            room = model.max_seq_len - cached[i]                                   # nodes that still fit the cache
            tokens.append([out[i][-1]] + [int(x) for x in t][:room - 1])
            parents.append([-1] + [int(x) for x in p][:room - 1])
        lens = [len(t) for t in tokens]
        nodes = torch.tensor([x for t in tokens for x in t], dtype=torch.int32, device=dev)
        logits, meta = model.forward_tree(nodes, lens, cached, parents)
        step += 1
        accepted = torch.empty(n, max_path, dtype=torch.int32, device=dev)
        count, following = torch.empty(n, dtype=torch.int32, device=dev), torch.empty(n, dtype=torch.int32, device=dev)
        _C.verify_tree(rt, logits, nodes, meta.parents, accepted, count, following, meta.query_start_loc, meta.lens, n)
        for k_cache, v_cache in model.caches:
            cfg = model.layers[0].cfg
            _C.compact_kv_cache(rt, k_cache, v_cache, accepted, count, meta.block_tables, cfg.n_kv_heads, cfg.head_dim, cfg.block_size,
                                n, meta.max_num_blocks, starts=meta.cached_lens)
        paths, counts, nexts = accepted.tolist(), count.tolist(), following.tolist()
        for i in range(n):
            if not live[i]:
                continue
            cached[i] += counts[i]
            for node in paths[i][1:counts[i]]:
                take(i, tokens[i][node])
            live[i] = live[i] and cached[i] + 1 <= model.max_seq_len
            take(i, nexts[i])
    return out, step


def generate_evicting(model: DecoderModel, prompt_tokens: List[List[int]], max_new_tokens: int, eos_id: int, budget: int,
                      recent: int, sink: int = 0, slack: int = 0) -> Tuple[List[List[int]], List[int]]:
    """`generate_ragged` with caches kept to `budget` positions per sequence: every step accumulates what the cached
    positions were attended to (`attention_weights`), and when a sequence holds more than budget + slack positions every
    layer keeps, per kv head, its first `sink`, its last `recent` and the most attended ones of the rest (`select_kept`,
    `compact_kv_cache`). Rotary positions run on, so answers may be longer than the cache, as far as the model's rope table
    reaches. Multi-head layers. Returns the new tokens and the cached positions per sequence at the end."""
    if model.is_mla:
        raise RuntimeError("generate_evicting: accumulated weights need multi-head attention layers")
    if budget + slack + 1 > model.max_seq_len:
        raise RuntimeError("generate_evicting: budget + slack + 1 positions exceed max_seq_len=%d" % model.max_seq_len)
    dev, n, rt, cfg = model.embed.device, len(prompt_tokens), model.rt, model.layers[0].cfg
    weights = [torch.zeros(k.shape[:3], dtype=torch.float32, device=dev) for k, _ in model.caches]
    cached, position = [0] * n, [0] * n
    pending = [list(t) for t in prompt_tokens]
    out: List[List[int]] = [[] for _ in range(n)]
    for _ in range(max_new_tokens):
        lens = [len(p) for p in pending]
        if sum(lens) == 0:
            break
        if max(p + l for p, l in zip(position, lens)) > model.rope.shape[0]:
            raise RuntimeError("generate_evicting: the rope table holds %d positions" % model.rope.shape[0])
        meta = prepare_attn(lens, cached, model.attn_meta(lens, cached).block_tables, model.block_size, dev,
                            positions=torch.tensor([position[i] + k for i in range(n) for k in range(lens[i])], dtype=torch.int64))
        flat = torch.tensor([t for p in pending for t in p], dtype=torch.int32, device=dev)
        choice = model._last_logits(model._rows(flat, meta, weights), lens).argmax(dim=-1).tolist()
        for i in range(n):
            cached[i] += lens[i]
            position[i] += lens[i]
            pending[i] = []
            if lens[i] != 0 and choice[i] != eos_id:
                out[i].append(int(choice[i]))
                pending[i] = [int(choice[i])]
        if max(cached) > budget + slack:
            tables = prepare_attn([1] * n, [max(c - 1, 0) for c in cached], model.attn_meta([1] * n, [max(c - 1, 0) for c in cached]).block_tables,
                                  model.block_size, dev)
            context = torch.tensor(cached, dtype=torch.int32, device=dev)
            kept = torch.empty(n, cfg.n_kv_heads, budget, dtype=torch.int32, device=dev)
            kept_lens = torch.empty(n, dtype=torch.int32, device=dev)
            for (k_cache, v_cache), w in zip(model.caches, weights):
                _C.select_kept(rt, w, kept, kept_lens, context, tables.block_tables, cfg.n_kv_heads, cfg.block_size, n, tables.max_num_blocks,
                               budget, recent, sink)
                _C.compact_kv_cache(rt, k_cache, v_cache, kept, kept_lens, tables.block_tables, cfg.n_kv_heads, cfg.head_dim, cfg.block_size,
                                    n, tables.max_num_blocks, weights=w)
            cached = [min(c, budget) for c in cached]
    return out, cached
