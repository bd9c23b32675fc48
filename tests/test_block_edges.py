"""Refusals of the block operators at their edges (no GPU needed)."""
import pytest
import torch

from plastix_b200 import block
from test_readout import FakeContext


def test_inputs_that_begin_where_the_result_does_are_refused_at_another_stride():
    """A block reads rows that another one has already written: only the very rows of out may be its input."""
    c = FakeContext()
    buf = torch.zeros(8, 16)
    rows, apart = buf[:4], buf[::2]
    other = torch.zeros(4, 16)
    for call in (lambda: block.block_norm(c, rows, apart, out=rows),
                 lambda: block.block_norm(c, apart, rows, out=rows),
                 lambda: block.block_norm(c, rows, apart, out=apart),
                 lambda: block.block_norm(c, rows, other, apart, out=rows),
                 lambda: block.recurrence(c, rows, apart, out=rows),
                 lambda: block.recurrence(c, apart, rows, out=rows)):
        with pytest.raises(ValueError, match="out overlaps"):
            call()
