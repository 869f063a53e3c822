"""The generation loops over drafted trees and over caches kept to a budget (gvirt_amd/generate.py): the operators run
together as they are used, in a small multi-layer stack."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _stack(seed, n_layers=2, hidden=256, n_heads=8, n_kv=2, d=64, vocab=97, block_size=16, max_batch=3, max_seq_len=96, rope_len=256):
    from gvirt_amd._C import Runtime
    from gvirt_amd.generate import DecoderModel
    from gvirt_amd.mha import MhaConfig, MhaLayer
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    up = lambda t: t.to(torch.bfloat16).to(DEV)  # noqa: E731
    cfg = MhaConfig(hidden=hidden, n_heads=n_heads, n_kv_heads=n_kv, head_dim=d, rot_dim=d, block_size=block_size)
    layers = [MhaLayer(cfg, up(r(hidden, (n_heads + 2 * n_kv) * d) * hidden ** -0.5), up(r(n_heads * d, hidden) * (n_heads * d) ** -0.5))
              for _ in range(n_layers)]
    fr = torch.outer(torch.arange(rope_len).float(), 1.0 / (10000.0 ** (torch.arange(0, d, 2).float() / d)))
    return DecoderModel(Runtime(0, 64), layers, [up(1 + 0.1 * r(hidden)) for _ in range(n_layers + 1)], up(r(vocab, hidden)),
                        up(r(hidden, vocab) * hidden ** -0.5), up(torch.cat([fr.cos(), fr.sin()], -1)), max_batch, max_seq_len)


def _logits_after(model_args, tokens):
    """fp32 logits of a fresh model behind every one of `tokens`, one prefill."""
    from gvirt_amd.mha import prepare_attn_meta
    m = _stack(**model_args)
    meta = prepare_attn_meta(m.attn_meta([len(tokens)], [0]), m.block_size, DEV)
    x = m._rows(torch.tensor(tokens, dtype=torch.int32, device=DEV), meta)
    return torch.matmul(x, m.lm_head).float().cpu()


@pytest.mark.parametrize("d,n_kv", [(64, 2), (128, 4)])
def test_trees_give_greedy_tokens_in_fewer_steps(d, n_kv):
    """The draft knows the continuation and hides it among other branches. Whatever a tree's step returns has to be what
    greedy decoding returns, up to logits that 16-bit roundings of two summation orders can swap: 0.06, as in the tests
    of the other generation loops."""
    from gvirt_amd.generate import generate_ragged, generate_tree
    args = dict(seed=5, d=d, n_kv=n_kv)
    prompts = [[3, 1, 4, 1, 5], [9, 2, 6], [5, 3, 5, 8, 9, 7, 9, 3, 2, 3, 8, 4, 6, 2, 6, 4, 3]]
    new = 24
    greedy, steps = generate_ragged(_stack(**args), prompts, new, -1)
    assert steps == new

    def draft(tokens):
        """Four tokens ahead, right for as long as the answer so far is the greedy one, with a wrong sibling everywhere."""
        ahead = []
        for p, g in zip(prompts, greedy):
            if tokens[:len(p)] == p and tokens[len(p):] == g[:len(tokens) - len(p)]:
                ahead = g[len(tokens) - len(p):][:4]
        t, up, at = [], [], 0
        for x in ahead:
            t += [(x + 1) % 97, x]
            up += [at, at]
            at = len(t)
        return t, up
    got, tree_steps = generate_tree(_stack(**args), prompts, draft, new, -1)
    assert all(len(x) == new for x in got)
    assert tree_steps <= 1 + new // 2          # five tokens a step where the draft is right
    for p, x in zip(prompts, got):
        logits = _logits_after(args, p + x)
        for k, token in enumerate(x):
            row = logits[len(p) + k - 1]
            assert float(row[token]) >= float(row.max()) - 0.06, k
    # wrong drafts and no drafts: one token a step
    same, n = generate_tree(_stack(**args), prompts, lambda t: ([96, 95, 94], [0, 1, 0]) if len(t) % 2 else ([], []), 5, -1)
    assert n <= 6 and all(len(x) == 5 for x in same)


def test_trees_end_with_their_token_and_with_the_cache(rt):
    from gvirt_amd.generate import generate_ragged, generate_tree
    args = dict(seed=6, max_seq_len=32)
    prompts = [[3, 1, 4, 1, 5], [9] * 28]
    greedy, _ = generate_ragged(_stack(**args), prompts, 40, -1)
    got, _ = generate_tree(_stack(**args), prompts, lambda t: ([1, 2, 3, 4, 5], [0, 1, 2, 0, 4]), 40, -1)
    assert [len(x) for x in got] == [len(x) for x in greedy]
    eos = got[0][3]
    cut, _ = generate_tree(_stack(**args), prompts, lambda t: ([], []), 40, eos)
    assert eos not in cut[0] and len(cut[0]) <= 3
    with pytest.raises(RuntimeError, match="before it"):
        generate_tree(_stack(**args), prompts, lambda t: ([1], [1]), 4, -1)


def test_evicting_with_room_for_everything_changes_nothing():
    from gvirt_amd.generate import generate_evicting, generate_ragged
    prompts = [[3, 1, 4, 1, 5], [9, 2, 6], list(range(40))]
    want, _ = generate_ragged(_stack(7), prompts, 20, -1)
    got, cached = generate_evicting(_stack(7), prompts, 20, -1, budget=80, recent=8)
    assert got == want and cached == [len(p) + 19 for p in prompts]


def test_evicting_keeps_the_cache_small_and_runs_past_it():
    from gvirt_amd.generate import generate_evicting
    prompts = [list(range(60)), [9, 2, 6], list(range(20, 50))]
    for slack in (0, 7):
        got, cached = generate_evicting(_stack(8, max_seq_len=64), prompts, 100, -1, budget=24, recent=8, sink=2, slack=slack)
        again, _ = generate_evicting(_stack(8, max_seq_len=64), prompts, 100, -1, budget=24, recent=8, sink=2, slack=slack)
        assert got == again and all(len(x) == 100 for x in got)
        assert all(24 - 1 <= c <= 24 + slack for c in cached)
    with pytest.raises(RuntimeError, match="rope table"):
        generate_evicting(_stack(8, max_seq_len=64, rope_len=70), prompts, 100, -1, budget=24, recent=8)
    with pytest.raises(RuntimeError, match="max_seq_len"):
        generate_evicting(_stack(8, max_seq_len=64), prompts, 100, -1, budget=64, recent=8)


def test_layer_weights_are_the_rows_probabilities():
    """Every row's probabilities sum to one per query head: the weights of a sequence's positions sum to rows x heads."""
    from gvirt_amd.mha import prepare_attn
    m = _stack(9)
    w = [torch.rand(k.shape[:3], device=DEV) for k, _ in m.caches]     # (positions of the step start at zero)
    lens = [7, 0, 33]
    tables = m.attn_meta(lens, [0] * 3).block_tables
    meta = prepare_attn(lens, [0] * 3, tables, m.block_size, DEV)
    m._rows(torch.arange(40, device=DEV), meta, w)
    for x in w:
        for n, t in zip(lens, tables):
            rows = x[torch.tensor(t, dtype=torch.long, device=DEV)].reshape(-1, 2)[:n]
            # sums of n * 4 probabilities, each off by a few units of 2^-22, over up to 33 positions
            assert torch.allclose(rows.sum(0), torch.full((2,), 4.0 * n, device=DEV), rtol=2.0 ** -16, atol=0)


def test_trees_and_weights_do_not_mix(rt):
    from gvirt_amd.mha import prepare_tree
    m = _stack(9)
    meta = prepare_tree([2], [0], [[0]], m.block_size, [[-1, 0]], DEV)
    w = [torch.zeros(k.shape[:3], device=DEV) for k, _ in m.caches]
    with pytest.raises(RuntimeError, match="drafted trees"):
        m._rows(torch.tensor([1, 2], device=DEV), meta, w)
