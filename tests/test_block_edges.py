"""Refusals of the block operators at their edges (no GPU needed)."""
import pytest
import torch

from plastix_b200 import _abi, block
from test_block import block_bwd_args, params
from test_readout import FakeContext, refused


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


def test_results_over_parameters_are_refused():
    """Every block reads parameters and offsets while others write results."""
    c, x = FakeContext(), torch.zeros(4, 16)
    buf = torch.zeros(6, 16)
    out, inside = buf[:4], buf[2]
    w = torch.zeros(16, 16)
    steps = torch.zeros(4, 16)
    offsets = steps.view(torch.int32).view(-1)[20:23]
    held = torch.zeros(2, 16)
    bad = [lambda: block.dense(c, x, w, inside, out=out),
           lambda: block.block_norm(c, x, x, inside, out=out),
           lambda: block.recurrence(c, x, x, offsets=offsets, out=steps),
           lambda: block.recurrence(c, x, x, offsets=held.view(torch.int32).view(-1)[3:6], final_out=held)]
    bad += [lambda name=name: block.block_norm(c, x, x, out=out, **{name: inside})
            for name in ("post_weight", "post_bias", "pre_weight", "pre_bias")]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError, match="overlaps"):
            call()
            pytest.fail(f"call {k} was not refused")


def overlaps(a, b):
    """Whether two views share an element, by looking at every one."""
    def touched(t):
        at = torch.arange(t.untyped_storage().nbytes() // t.element_size())
        return set(at.as_strided(t.size(), t.stride(), t.storage_offset()).flatten().tolist())
    return bool(touched(a) & touched(b))


def test_rows_side_by_side_are_told_from_rows_that_overlap():
    """All placements of two tensors of rows in a small buffer: refused where they share an element, and not
    where one lies beside the other in rows of the same stride."""
    buf = torch.zeros(80)
    a = buf.as_strided((3, 4), (11, 1), 15)
    for n in (1, 3, 5):
        for ld in (5, 11, 12):
            for at in range(0, 80 - 2 * ld - n + 1):
                b = buf.as_strided((3, n), (ld, 1), at)
                try:
                    block._check_apart(a, 11, "out", (b, ld, "x"))
                    refused = False
                except ValueError:
                    refused = True
                if overlaps(a, b):
                    assert refused, (n, ld, at)
                elif ld == 11:
                    assert not refused, (n, at)


def test_gradients_of_a_norm_that_is_not_there_are_refused():
    """They would be left as they were, where every gradient that is given is written."""
    for name in ("dw1", "db1"):
        change = {k: None for k in ("dw1", "db1") if k != name}
        refused(1, b"post", "plx_block_norm_backward", *block_bwd_args(params=params(post=0), **change))


@pytest.mark.parametrize("rows, n, most", [(600, 65536, 64), (1 << 20, 16384, 37), (1 << 20, 8192, 74), (5, 20000, 5),
                                           (1 << 20, 1024, 592), (1 << 20, 4096, 148), (1, 100, 1), (0, 100, 1)])
def test_scratch_of_block_norm_is_what_its_launches_leave(rows, n, most):
    """Five column sums of every group, and the four means of rows that are too long for registers."""
    size = _abi.lib().plx_block_norm_scratch_bytes(rows, n)
    assert size == most * 5 * n * 4 + (rows * 16 if n > 16384 else 0)
