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
