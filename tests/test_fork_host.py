"""What the copies of pages and states refuse, without a device."""
import pytest
import torch

import bitnet_c_b200  # noqa: F401
from bitnet_c_b200.csrc import ops


def test_moves_are_grouped_by_source():
    groups, to = ops._page_moves([(4, 0, 9), (7, 1, 64), (4, 8, 9), (4, 2, 11)], 9)
    assert groups == [4, 9, 2, 7, 64, 1, 4, 11, 1] and to == [0, 8, 1, 2]
    assert ops._page_moves([], 3) == ([], [])


@pytest.mark.parametrize("moves,what", [
    ([(9, 0, 1)], "outside"), ([(-1, 0, 1)], "outside"), ([(0, 9, 1)], "outside"), ([(0, 1, 0)], "rows"), ([(0, 1, 65)], "rows"),
    ([(0, 1, 3), (2, 1, 3)], "written once"), ([(0, 1, 3), (1, 2, 3)], "not read"), ([(3, 3, 64)], "not read")])
def test_moves_that_are_refused(moves, what):
    with pytest.raises(ops.KernelError, match=what):
        ops._page_moves(moves, 9)


def test_tensors_that_are_refused():
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.copy_pages(torch.zeros(1, 2, 1, 64, 8), None, [(0, 1, 1)])
    with pytest.raises(ops.KernelError, match="CUDA"):
        ops.StateSlots([torch.zeros(2, 3)])
    with pytest.raises(ops.KernelError, match="slot"):
        ops.copy_slots(ops.StateSlots([]), 0, [1])
