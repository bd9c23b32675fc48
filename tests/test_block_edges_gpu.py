"""The block operators at their edges on the device, against their 64-bit formulas (U = 2^-24)."""
import numpy as np
import pytest
import torch

import block_formulas as F
from plastix_b200 import _abi, block
from plastix_b200.runtime import Context
from test_block_gpu import made, stored
from test_readout_gpu import HALF_STEP, TYPES, U, f64, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return Context(0)


@pytest.mark.parametrize("n", [515, 1024, 9001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_block_norm_in_place_of_its_gate(ctx, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(n)
    x, o, gate = (torch.randn(40, n, device="cuda", generator=g).to(TYPES[dtype]) for _ in range(3))
    r, u = block.block_norm(ctx, x, o, gate, gate_apply="sigmoid")
    r2, u2 = block.block_norm(ctx, x, o, gate, gate_apply="sigmoid", out=gate)
    ctx.sync()
    assert r2 is gate and torch.equal(r2, r) and torch.equal(u2, u)


def test_results_beside_their_inputs(ctx):
    """x and out as the two halves of wider rows."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for n in (64, 72):  # halves that start at multiples of 16 bytes, as the arrays of their own do
        x, gate = (torch.randn(300, n, device="cuda", generator=g) for _ in range(2))
        w = torch.randn(n, n, device="cuda", generator=g)
        want = (block.dense(ctx, x, w), block.block_norm(ctx, x, gate)[0], block.recurrence(ctx, x, gate)[0])
        for k, call in enumerate((lambda a, b: block.dense(ctx, a, w, out=b),
                                  lambda a, b: block.block_norm(ctx, a, gate, out=b)[0],
                                  lambda a, b: block.recurrence(ctx, a, gate, out=b)[0])):
            wide = torch.zeros(300, 2 * n, device="cuda")
            wide[:, :n] = x
            got = call(wide[:, :n], wide[:, n:])
            ctx.sync()
            assert torch.equal(wide[:, :n], x) and torch.equal(got, want[k])
