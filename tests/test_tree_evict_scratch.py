"""How much scratch the operators on drafted trees and on caches kept to a budget ask for (host formulas)."""
import pytest

from gvirt_amd import _lib

MB = 1 << 20


def tree(tokens, heads, kv_heads, dim, block, batch, blocks, kv):
    return _lib.load().xlite_hip_tree_attention_workspace_bytes(tokens, heads, kv_heads, dim, block, batch, blocks, kv)


@pytest.mark.parametrize("kv", [1, 2])
@pytest.mark.parametrize("shape", [(1024, 32, 8, 128, 128, 64, 256), (512, 14, 2, 64, 16, 64, 2048), (64, 28, 4, 128, 24, 8, 700), (8, 6, 1, 64, 7, 1, 1000)])
def test_trees_over_bytes_need_no_copy_of_the_cache(shape, kv):
    """The kernel that serves them widens rows on their way: the same scratch as over a 16-bit cache, which a copy would
    exceed by the whole cache."""
    assert tree(*shape, kv) <= tree(*shape, 0) < 200 * MB


def test_trees_that_other_kernels_serve():
    """More sequences than the streaming kernel takes: head_dim 128 is read as it is, head_dim 64 copied."""
    copy = lambda dim, block, blocks: 2 * 2000 * blocks * block * 2 * dim * 2  # noqa: E731
    assert tree(4000, 4, 2, 128, 16, 2000, 64, 1) < copy(128, 16, 64) // 4
    assert tree(4000, 4, 2, 64, 16, 2000, 64, 1) >= copy(64, 16, 64)


def weights(tokens, heads, kv_heads, dim, block, batch, blocks, window=0):
    return _lib.load().xlite_hip_attention_weights_workspace_bytes(tokens, heads, kv_heads, dim, block, batch, blocks, window)


@pytest.mark.parametrize("shape", [(512, 32, 8, 128, 128, 512, 256), (64, 32, 8, 128, 16, 64, 8192), (512, 32, 8, 128, 128, 64, 256), (1300, 28, 4, 128, 128, 301, 64),
                                   (64, 64, 1, 64, 16, 64, 1 << 20), (4096, 28, 4, 128, 128, 64, 256, 8)])
def test_stored_scores_are_bounded(shape):
    """Decode steps, short steps and chunks of wide tables: what is stored of the scores at a time stays below 1.5 GB,
    the normalisers and statistics of scores that are not stored below 64 MB."""
    assert 0 < weights(*shape) <= 1600 * MB


def test_one_row_a_sequence_is_not_laid_out_for_more():
    """64 rows of 32 heads over tables of 4096 positions: a score of 4 bytes each, and their statistics."""
    assert weights(64, 32, 8, 128, 128, 64, 32) < 1.1 * 64 * 32 * 4096 * 4


def test_sizes_of_shapes_that_do_not_exist():
    """The size functions answer whatever they are asked (the calls themselves refuse such shapes)."""
    for heads, kv_heads, block, blocks in ((0, 2, 16, 4), (4, 0, 16, 4), (3, 2, 16, 4), (4, 2, 16, 0), (4, 2, 1 << 16, (1 << 16) - 1)):
        weights(8, heads, kv_heads, 64, block, 2, blocks)
        tree(8, heads, kv_heads, 64, block, 2, blocks, 0)
    assert weights(8, 0, 2, 64, 16, 2, 4) == 0
