"""Refusals of the operators around drafted tokens, without a GPU: every check of arguments stands in front of the launch."""
import pytest
import torch

from yalm_amd.ops import kernels


def test_tensors_that_are_not_on_the_gpu_are_refused():
    x = torch.zeros((2, 8))
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.sample_filtered(x, torch.zeros(2), torch.zeros(2, dtype=torch.int32))
    pages = torch.zeros((1, 2, 1, 64, 16)), torch.zeros((1, 2, 1, 16, 64))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.copy_pages(*pages, i, i)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.compact_lines(*pages, torch.zeros((1, 1), dtype=torch.int32), 1, i, i, torch.zeros(2, dtype=torch.int32), i, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.attn_tree(torch.zeros((1, 16)), pages[0][0], pages[1][0], torch.zeros((1, 1), dtype=torch.int32), 1, i, i, torch.zeros(2, dtype=torch.int32),
                          torch.zeros((1, 1), dtype=torch.int64), torch.zeros((1, 16)), torch.zeros(0), 1, 1, 16, 0, 1, 1)


def test_shapes_that_say_nothing_are_refused():
    with pytest.raises(ValueError, match="vocabulary"):
        kernels.sample_filtered(torch.zeros(8), None, None)
    with pytest.raises(ValueError, match="vocabulary"):
        kernels.sample_filtered(torch.zeros((2, 0)), None, None)
    with pytest.raises(ValueError, match="lines, pages"):
        kernels.compact_lines(torch.zeros((2, 64, 16)), None, None, 1, None, None, None, None, 1)
    with pytest.raises(ValueError, match="multiple"):
        kernels.attn_tree(None, None, None, None, 1, None, None, None, None, None, None, 3, 2, 64, 0, 1, 1)


def test_workspace_sizes():
    assert kernels.attn_tree_workspace_floats(7, 4, 64, 1) == 0
    assert kernels.attn_tree_workspace_floats(7, 4, 64, 3) == 7 * 4 * 3 * 66
    assert kernels.sample_filtered_workspace(3, 32000) >= 0
