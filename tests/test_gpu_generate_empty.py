"""Prompts without tokens in the generation loops: they get no answer, whichever loop runs them."""
import pytest

from test_gpu_generate_trees import _stack

pytestmark = pytest.mark.gpu
PROMPTS = [[3, 1, 4], [], [9, 2]]


def test_trees_give_empty_prompts_no_answer(rt):
    from gvirt_amd.generate import generate_ragged, generate_tree
    want, _ = generate_ragged(_stack(5), PROMPTS, 6, -1)
    got, _ = generate_tree(_stack(5), PROMPTS, lambda t: ([], []), 6, -1)
    assert [len(x) for x in got] == [len(x) for x in want] == [6, 0, 6]


@pytest.mark.parametrize("prompts", [[[], []], []])
def test_nothing_but_empty_prompts(rt, prompts):
    from gvirt_amd.generate import generate_ragged, generate_tree
    want = generate_ragged(_stack(5), prompts, 6, -1)
    assert generate_tree(_stack(5), prompts, lambda t: ([], []), 6, -1) == want == ([[] for _ in prompts], 0)


def test_evicting_gives_empty_prompts_no_answer(rt):
    from gvirt_amd.generate import generate_evicting
    got, cached = generate_evicting(_stack(5), PROMPTS, 6, -1, budget=40, recent=4)
    assert [len(x) for x in got] == [6, 0, 6] and cached == [8, 0, 7]


def test_no_tokens_wanted(rt):
    from gvirt_amd.generate import generate_ragged, generate_tree
    assert generate_tree(_stack(5), PROMPTS, lambda t: ([], []), 0, -1) == generate_ragged(_stack(5), PROMPTS, 0, -1) == ([[], [], []], 0)
