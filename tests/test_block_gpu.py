"""The block operators on the device against their 64-bit formulas.

Tolerances are bounds from the operators' own arithmetic, with U = 2^-24 the unit
of a 32-bit rounding; the stored result adds half a step of its type. Backward
formulas take what the forward call returned (z, statistics, h), as the backward
call does. Inputs are rounded to their type first, so both sides read the same
values."""
import numpy as np
import pytest
import torch

import block_formulas as F
from plastix_b200 import _abi, block, readout
from plastix_b200.runtime import Context
from test_readout_gpu import HALF_STEP, TINY, TYPES, U, f64, rows_tensor, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return Context(0)


def rng(*key):
    return np.random.default_rng(list(key))


def made(a, dtype, ld=None, shift=0):
    """(tensor, its values in 64 bits, the buffer that it is a part of)"""
    t, buf = rows_tensor(a, dtype, ld, shift)
    return t, f64(t), buf


def vector(a, dtype, shift=0):
    t, _ = rows_tensor(a[None], dtype, None, shift)
    return t[0], f64(t[0])


def stored(want, tol, dtype):
    """The tolerance of a value that is rounded to its type at the end."""
    return tol + HALF_STEP[dtype] * (np.abs(want) + tol) + TINY[dtype]


# ------------------------------------------------------------------------------------ dense
def product_error(a, b, depth):
    """Bound of a sum of `depth` products in 32 bits, in any order, chopped or rounded: each of the
    terms goes through at most depth additions of 2 U; operands in two pieces leave 8 U more."""
    return (2 * depth + 40) * U * (np.abs(a) @ np.abs(b))


def act_error(z, y):
    """Of an activation: a few steps of its factors, the exponent's argument 3 U |z| off."""
    return (24 + 4 * np.minimum(np.abs(z), 100)) * U * np.maximum(np.abs(y), 2.0 ** -60) + 4 * U * np.minimum(np.abs(z), 1)


DENSE = [  # rows, n, m, dtype, apply, residual, extra row stride, shift, param
    (1, 1, 1, "f32", "identity", False, 0, 0, "f32"),
    (1, 7, 3, "bf16", "silu", True, 0, 1, "f32"),
    (5, 64, 128, "bf16", "gelu", True, 0, 0, "same"),
    (8, 512, 384, "f16", "tanh", False, 0, 0, "f32"),
    (17, 513, 257, "bf16", "sigmoid", True, 3, 1, "f32"),
    (33, 1000, 100, "f16", "relu", False, 8, 0, "same"),
    (128, 64, 256, "bf16", "identity", False, 0, 0, "f32"),
    (129, 65, 257, "f16", "silu", True, 1, 3, "f32"),
    (200, 96, 520, "f32", "tanh", True, 0, 0, "f32"),
    (131, 77, 133, "f32", "gelu", False, 5, 1, "f32"),
    (300, 1024, 768, "bf16", "silu", True, 0, 0, "same"),
    (700, 200, 72, "bf16", "gelu", False, 8, 8, "f32"),
    (64, 2048, 640, "f16", "identity", True, 0, 0, "f32"),
    (2, 4099, 1030, "bf16", "silu", False, 0, 0, "f32"),
    (16, 4096, 1024, "f32", "silu", True, 0, 0, "f32"),
    (1500, 40, 1000, "f32", "sigmoid", False, 0, 0, "f32"),
    (3000, 130, 2056, "bf16", "silu", True, 0, 0, "f32"),  # large tiles, the last ones cut on both sides
    (2700, 72, 1999, "f16", "gelu", True, 0, 0, "same"),
    (2600, 200, 1400, "f32", "gelu", True, 0, 0, "f32"),
    (2500, 70, 1401, "f32", "tanh", True, 3, 1, "f32"),
    (40, 3000, 2000, "bf16", "tanh", True, 0, 0, "f32"),  # few rows, sums shared by blocks
    (3, 1000, 300, "f32", "gelu", True, 1, 1, "f32"),
    (7, 515, 130, "f32", "relu", False, 1, 0, "f32"),
    (65, 1000, 33, "f16", "silu", True, 0, 0, "f32"),
    # wide tiles of 32-bit values, sums shared by 2, 4 and 8 blocks
    (1000, 600, 1024, "f32", "silu", True, 0, 0, "f32"),
    (513, 1001, 1020, "f32", "gelu", True, 1, 1, "f32"),
    (250, 1023, 1000, "f32", "tanh", False, 0, 0, "f32"),
    (1000, 1024, 129, "f32", "identity", True, 4, 0, "f32"),
]


def dense_inputs(rows, n, m, dtype, more, shift, param, seed=1):
    g = rng(rows, n, m, seed)
    x, xv, _ = made(g.normal(size=(rows, n)), dtype, n + more, shift)
    w, wv, _ = made(g.normal(size=(m, n)) / np.sqrt(n), dtype, n + more, shift)
    b, bv = vector(g.normal(size=m) * 0.3, dtype if param == "same" else "f32", shift)
    res, resv, _ = made(g.normal(size=(rows, m)), dtype, m + more, shift)
    dy, dyv, _ = made(g.normal(size=(rows, m)), dtype, m + more, shift)
    return (x, xv), (w, wv), (b, bv), (res, resv), (dy, dyv)


@pytest.mark.parametrize("rows, n, m, dtype, apply, residual, more, shift, param", DENSE)
def test_dense(ctx, rows, n, m, dtype, apply, residual, more, shift, param):
    (x, xv), (w, wv), (b, bv), (res, resv), _ = dense_inputs(rows, n, m, dtype, more, shift, param)
    y, z = block.dense(ctx, x, w, b, apply=apply, residual=res if residual else None, pre=True)
    only = block.dense(ctx, x, w, b, apply=apply, residual=res if residual else None)
    ctx.sync()
    want, wz = F.dense(xv, wv, bv, apply, resv if residual else None)
    ztol = product_error(xv, wv.T, n) + 4 * U * (np.abs(wz) + np.abs(bv))
    within(f64(z), wz, ztol, "z")
    a = F.act(wz, apply)[0]
    tol = 1.2 * ztol + (0 if apply == "identity" else act_error(wz, a)) + U * np.abs(want)
    within(f64(y), want, stored(want, tol, dtype), "y")
    assert torch.equal(y, only)


@pytest.mark.parametrize("rows, n, m, dtype, apply, residual, more, shift, param", DENSE)
def test_dense_backward(ctx, rows, n, m, dtype, apply, residual, more, shift, param):
    (x, xv), (w, wv), (b, bv), _, (dy, dyv) = dense_inputs(rows, n, m, dtype, more, shift, param, 2)
    _, z = block.dense(ctx, x, w, b, apply=apply, pre=True)
    dx, dw, db = block.dense_backward(ctx, dy, x, w, z, apply=apply, bias=b)
    again = block.dense_backward(ctx, dy, x, w, z, apply=apply, bias=b)
    ctx.sync()
    zv = f64(z)
    wx, ww, wb, dz = F.dense_backward(dyv, xv, wv, zv, apply)
    exact_dz = apply == "identity"
    slope = F.act(zv, apply)[1]
    off = 0 if exact_dz else np.abs(dyv) * (act_error(zv, slope) + 4 * U)
    dzerr = off if exact_dz else off + (HALF_STEP[dtype] if dtype != "f32" else 0) * (np.abs(dz) + off) + TINY[dtype]
    dzerr = dzerr + np.zeros_like(dz)
    tx = dzerr @ np.abs(wv) + product_error(dz, wv, m)
    tw = dzerr.T @ np.abs(xv) + product_error(dz.T, xv, rows)
    within(f64(dx), wx, stored(wx, tx, dtype), "dx")
    within(f64(dw), ww, stored(ww, tw, dtype), "dweight")
    tb = (off + np.zeros_like(dz)).sum(0) + (rows + 64) * U * np.abs(dz).sum(0)
    within(f64(db), wb, stored(wb, tb, dtype if param == "same" else "f32"), "dbias")
    for a, c in zip((dx, dw, db), again):
        assert torch.equal(a, c)


@pytest.mark.parametrize("rows, m, dtype", [(700, 1100, "bf16"), (2600, 1400, "f32"), (5, 1100, "bf16"), (100, 72, "f16")])
def test_dense_in_place_of_its_residual(ctx, rows, m, dtype):
    """out is the residual, a part of wider rows whose other values stay."""
    (x, _), (w, _), (b, _), (res, _), _ = dense_inputs(rows, 200, m, dtype, 8, 8, "f32", 3)
    want = block.dense(ctx, x, w, b, apply="silu", residual=res)
    wide = torch.full((rows, m + 16), 3.0, dtype=TYPES[dtype], device="cuda")
    part = wide[:, 8:8 + m]
    part.copy_(res)
    y = block.dense(ctx, x, w, b, apply="silu", residual=part, out=part)
    ctx.sync()
    assert y is part and torch.equal(part, want)
    assert (wide[:, :8] == 3.0).all() and (wide[:, 8 + m:] == 3.0).all()


def test_dense_leaves_what_lies_between_rows(ctx):
    """Results into a part of wider rows at every alignment: nothing beside them is written."""
    g = torch.Generator(device="cuda").manual_seed(6)
    for dtype in ("f32", "bf16"):
        for rows, m in ((300, 500), (1500, 640), (9, 130)):
            x = torch.randn(rows, 64, device="cuda", generator=g).to(TYPES[dtype])
            w = torch.randn(m, 64, device="cuda", generator=g).to(TYPES[dtype])
            want = block.dense(ctx, x, w)
            for shift in (0, 1, 8):
                wide = torch.full((rows + 2, m + 24), 5.0, dtype=TYPES[dtype], device="cuda")
                y = block.dense(ctx, x, w, out=wide[1:-1, shift:shift + m])
                ctx.sync()
                assert torch.equal(y, want)
                assert (wide[0] == 5.0).all() and (wide[-1] == 5.0).all()
                assert (wide[:, :shift] == 5.0).all() and (wide[:, shift + m:] == 5.0).all()


@pytest.mark.parametrize("apply", ["sigmoid", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_activations_over_their_range(ctx, dtype, apply):
    """One weight of 1: z is x, from tails to tails, zero and the smallest values among it."""
    z = np.concatenate([np.linspace(-13, 13, 4001), np.logspace(-8, 0, 300), -np.logspace(-8, 0, 300), [0.0]])
    x, xv, _ = made(z[:, None], dtype)
    y = block.dense(ctx, x, torch.ones(1, 1, device="cuda", dtype=TYPES[dtype]), apply=apply)
    ctx.sync()
    want = F.act(xv, apply)[0]
    # of 16 bits: GELU's fitted factor is off by 1e-4 at most (|z| > 10), the others by a few steps
    rel = act_error(xv, want) + (1e-4 * np.abs(want) if dtype != "f32" and apply == "gelu" else 0)
    within(f64(y), want, stored(want, rel, dtype), "y")


def test_dense_parts_and_empty(ctx):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, 40, device="cuda", generator=g)
    w = torch.randn(24, 40, device="cuda", generator=g)
    dy = torch.randn(6, 24, device="cuda", generator=g)
    full = block.dense_backward(ctx, dy, x, w, bias=w[:, 0].contiguous())
    dx, none, no_bias = block.dense_backward(ctx, dy, x, w, weight_grad=False)
    assert none is None and no_bias is None and torch.equal(dx, full[0])
    none, dw, _ = block.dense_backward(ctx, dy, x, w, input_grad=False)
    assert none is None and torch.equal(dw, full[1])
    y = block.dense(ctx, x.new_empty(0, 40), w)
    assert y.shape == (0, 24)
    dx, dw, db = block.dense_backward(ctx, dy[:0], x[:0], w, bias=w[:, 0].contiguous())
    assert dx.shape == (0, 40) and not dw.any() and not db.any()
    ctx.sync()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_dense_passes_nan_and_infinity_on(ctx, dtype):
    x = torch.ones(40, 72, device="cuda", dtype=TYPES[dtype])
    w = torch.ones(136, 72, device="cuda", dtype=TYPES[dtype])
    x[3, 5] = float("nan")
    x[7, 71] = float("inf")
    w[9, 0] = float("-inf")
    y = block.dense(ctx, x, w)
    ctx.sync()
    want = x.double() @ w.double().t()
    got = y.double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    assert torch.equal(got[fine], want[fine])


# -------------------------------------------------------------------------------- block norm
def norm_errors(v, verr, kind, eps):
    """(h, mean, rstd, error of h) of a norm of values that are off by verr."""
    h, mean, rstd = F.norm(v, kind, eps)
    n = v.shape[1]
    deep = (n / 32 + 80) * U
    # a first mean off by its roundings costs little in deviations four times as large (or is corrected)
    merr = (deep * 4 / rstd + 4 * U * np.abs(mean) + verr.mean(1, keepdims=True)) if kind == "layer" else 0.0
    rel = deep + 16 * U + rstd * (np.abs(h) * verr).mean(1, keepdims=True) + (merr * rstd) ** 2
    herr = rstd * (verr + merr + 2 * U * (np.abs(v) + np.abs(mean))) + np.abs(h) * rel
    return h, mean, rstd, herr


def gate_errors(gate, apply):
    g, slope = F.act(gate, apply)
    return g, slope, 0.0 if apply == "identity" else act_error(gate, g)


def block_forward(x, o, gate, how, eps):
    """Formulas and bounds of a forward call."""
    zero = np.zeros_like(o)
    if how["post"]:
        h1, m1, s1, e1 = norm_errors(o, zero, how["kind"], eps)
    else:
        h1, m1, s1, e1 = o, np.zeros((len(o), 1)), np.zeros((len(o), 1)), zero
    w1 = 1.0 if how["post_weight"] is None else how["post_weight"]
    b1 = 0.0 if how["post_bias"] is None else how["post_bias"]
    p = h1 * w1 + b1
    perr = np.abs(w1) * e1 + 3 * U * (np.abs(h1 * w1) + np.abs(b1))
    g, _, gerr = (1.0, 1.0, 0.0) if gate is None else gate_errors(gate, how["gate_apply"])
    r = how["scale"] * x + g * p
    rerr = np.abs(g) * perr + gerr * np.abs(p) + 3 * U * (np.abs(how["scale"] * x) + np.abs(g * p))
    h2, m2, s2, e2 = norm_errors(r, rerr, how["kind"], eps)
    w2 = 1.0 if how["pre_weight"] is None else how["pre_weight"]
    b2 = 0.0 if how["pre_bias"] is None else how["pre_bias"]
    u = h2 * w2 + b2
    uerr = np.abs(w2) * e2 + 3 * U * (np.abs(h2 * w2) + np.abs(b2))
    return r, rerr, u, uerr, np.concatenate([m1, s1, m2, s2], 1)


BLOCK = [  # rows, n, dtype, kind, gate, gate_apply, post, scale, extra row stride, shift, param, affine
    (1, 1, "f32", "rms", "none", "identity", True, 1.0, 0, 0, "f32", True),
    (3, 2, "bf16", "layer", "units", "identity", True, 0.5, 0, 0, "f32", True),
    (9, 64, "bf16", "rms", "values", "sigmoid", True, 1.0, 0, 0, "same", True),
    (20, 256, "f16", "layer", "values", "identity", True, -1.5, 0, 0, "f32", True),
    (19, 257, "f16", "rms", "units", "sigmoid", False, 1.0, 3, 1, "f32", True),
    (11, 510, "bf16", "layer", "none", "identity", False, 1.0, 2, 2, "same", False),
    (7, 1000, "f32", "layer", "values", "identity", True, 0.8, 0, 0, "f32", True),
    (7, 1001, "f32", "rms", "units", "identity", True, 0.8, 0, 0, "f32", True),
    (300, 1024, "bf16", "rms", "units", "identity", True, 1.0, 0, 0, "f32", True),
    (200, 2048, "f16", "layer", "units", "sigmoid", True, 1.0, 8, 8, "same", True),
    (170, 2050, "bf16", "rms", "values", "sigmoid", True, 1.0, 0, 0, "f32", False),
    (160, 4096, "bf16", "layer", "values", "identity", True, 1.0, 0, 0, "same", True),
    (5, 4097, "f32", "layer", "units", "identity", True, 1.0, 1, 0, "f32", True),
    (4, 8192, "bf16", "rms", "units", "sigmoid", True, 2.0, 0, 0, "f32", True),
    (4, 8200, "bf16", "layer", "values", "sigmoid", True, 1.0, 0, 0, "f32", True),
    (3, 16384, "f16", "rms", "units", "identity", True, 1.0, 0, 0, "f32", True),
    (3, 20001, "bf16", "layer", "values", "identity", True, 1.0, 0, 0, "f32", True),
    (900, 96, "f32", "layer", "units", "identity", False, 1.0, 0, 0, "f32", True),
    (2000, 33, "bf16", "rms", "values", "identity", True, 1.0, 0, 0, "same", True),
]


def block_inputs(rows, n, dtype, kind, gate, gate_apply, post, scale, more, shift, param, affine):
    g = rng(rows, n, len(kind))
    x, xv, _ = made(g.normal(size=(rows, n)) * 1.5 + g.normal(size=(rows, 1)), dtype, n + more, shift)
    o, ov, _ = made(g.normal(size=(rows, n)) * 0.7 + 0.3, dtype, n + more, shift)
    pt = dtype if param == "same" else "f32"
    gt = gv = None
    if gate == "values":
        gt, gv, _ = made(g.normal(size=(rows, n)), dtype, n + more, shift)
    elif gate == "units":
        gt, gv = vector(g.normal(size=n), pt, shift)
    how, wide = dict(kind=kind, post=post, scale=scale, gate_apply=gate_apply), {}
    for name in ("post_weight", "post_bias", "pre_weight", "pre_bias"):
        how[name] = wide[name] = None
        if affine and (post or name[:3] == "pre"):
            how[name], wide[name] = vector(g.normal(size=n) * 0.4 + ("weight" in name), pt, shift)
    dr, drv, _ = made(g.normal(size=(rows, n)), dtype, n + more, shift)
    du, duv, _ = made(g.normal(size=(rows, n)), dtype, n + more, shift)
    return (x, xv), (o, ov), (gt, gv), how, {**how, **wide, "scale": float(np.float32(scale))}, (dr, drv), (du, duv), pt


@pytest.mark.parametrize("case", BLOCK, ids=lambda c: f"{c[0]}x{c[1]}-{c[2]}-{c[3]}-{c[4]}")
def test_block_norm(ctx, case):
    (x, xv), (o, ov), (gt, gv), how, wide, _, _, _ = block_inputs(*case)
    dtype, eps = case[2], float(np.float32(1e-5))
    r, u, stats = block.block_norm(ctx, x, o, gt, stats=True, **how)
    ctx.sync()
    wr, rerr, wu, uerr, wstats = block_forward(xv, ov, gv, wide, eps)
    within(f64(r), wr, stored(wr, rerr, dtype), "r")
    within(f64(u), wu, stored(wu, uerr, dtype), "u")
    n = case[1]
    spread = np.stack([np.abs(ov).mean(1), wstats[:, 1], np.abs(wr).mean(1) + rerr.max(1) / U / 500, wstats[:, 3]], 1)
    srel = np.array([1.0, 1.0, 1.0, 1.0 + 8 * (rerr / np.maximum(np.sqrt((wr * wr).mean(1, keepdims=True)), 1e-30)).max() / U / 500])
    within(f64(stats), wstats, (n / 16 + 500) * U * spread * srel, "stats")


@pytest.mark.parametrize("n", [96, 1000, 4096, 9000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_block_norm_of_rows_far_from_zero(ctx, n, dtype):
    """Rows around a large value, whose deviations the first mean's roundings would drown."""
    g = rng(n, 7)
    x, xv, _ = made(g.normal(size=(5, n)) + 300.0, dtype)
    o, ov, _ = made(g.normal(size=(5, n)) - 900.0, dtype)
    r, u, _ = block.block_norm(ctx, x, o, kind="layer", stats=True)
    ctx.sync()
    how = dict(kind="layer", post=True, scale=1.0, gate_apply="identity", post_weight=None, post_bias=None,
               pre_weight=None, pre_bias=None)
    wr, rerr, wu, uerr, _ = block_forward(xv, ov, None, how, float(np.float32(1e-5)))
    within(f64(r), wr, stored(wr, rerr, dtype), "r")
    within(f64(u), wu, stored(wu, uerr, dtype), "u")


def test_block_norm_in_place(ctx):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(30, 515, device="cuda", generator=g)
    o = torch.randn(30, 515, device="cuda", generator=g)
    r, u = block.block_norm(ctx, x, o, kind="layer")
    for where in ("x", "o"):
        t = {"x": x.clone(), "o": o.clone()}
        r2, u2 = block.block_norm(ctx, t["x"], t["o"], kind="layer", out=t[where])
        assert r2 is t[where] and torch.equal(r2, r) and torch.equal(u2, u)
    ctx.sync()


@pytest.mark.parametrize("without", ["", "dr", "du"])
@pytest.mark.parametrize("case", BLOCK, ids=lambda c: f"{c[0]}x{c[1]}-{c[2]}-{c[3]}-{c[4]}")
def test_block_norm_backward(ctx, case, without):
    (x, xv), (o, ov), (gt, gv), how, wide, (dr, drv), (du, duv), pt = block_inputs(*case)
    rows, n, dtype, kind, gate = case[:5]
    _, _, stats = block.block_norm(ctx, x, o, gt, stats=True, **how)
    dr, drv = (None, None) if without == "dr" else (dr, drv)
    du, duv = (None, None) if without == "du" else (du, duv)
    got = block.block_norm_backward(ctx, dr, du, x, o, stats, gt, **how)
    again = block.block_norm_backward(ctx, dr, du, x, o, stats, gt, **how)
    ctx.sync()
    # values and their bounds, made of the statistics that the call is given
    m1, s1, m2, s2 = np.split(f64(stats), 4, 1)
    one = lambda v, d: d if v is None else v  # noqa: E731
    w1, b1, w2 = one(wide["post_weight"], 1.0), one(wide["post_bias"], 0.0), one(wide["pre_weight"], 1.0)
    h1 = (ov - m1) * s1 if wide["post"] else ov
    e_h1 = 3 * U * (np.abs(ov) + np.abs(m1)) * s1 if wide["post"] else 0 * ov
    p = h1 * w1 + b1
    e_p = np.abs(w1) * e_h1 + 3 * U * (np.abs(h1 * w1) + np.abs(b1))
    gv_, slope, e_g = (1.0, 1.0, 0.0) if gv is None else gate_errors(gv, wide["gate_apply"])
    e_slope = 0.0 if gv is None or wide["gate_apply"] == "identity" else act_error(gv, slope) + 4 * U
    r = wide["scale"] * xv + gv_ * p
    e_r = np.abs(gv_) * e_p + e_g * np.abs(p) + 3 * U * (np.abs(wide["scale"] * xv) + np.abs(gv_ * p))
    h2 = (r - m2) * s2
    e_h2 = s2 * (e_r + 3 * U * (np.abs(r) + np.abs(m2)))
    want = F.block_norm_backward(drv, duv, dict(h1=h1, s1=s1, p=p, g=gv_, slope=slope, h2=h2, s2=s2), kind=kind,
                                 post=wide["post"], scale=wide["scale"], gate_units=gate == "units",
                                 post_weight=wide["post_weight"], pre_weight=wide["pre_weight"])
    deep = (n / 32 + 80) * U

    def through(e, e_err, h, h_err, s):  # error of s (e - mean e - h mean(e h))
        c1 = np.abs((e * h).mean(1, keepdims=True))
        c_err = (np.abs(e) * h_err + np.abs(h) * e_err).mean(1, keepdims=True) + deep * np.abs(e * h).mean(1, keepdims=True)
        m_err = (e_err.mean(1, keepdims=True) + deep * np.abs(e).mean(1, keepdims=True)) if kind == "layer" else 0.0
        m = np.abs(e).mean(1, keepdims=True) if kind == "layer" else 0.0
        return s * (e_err + m_err + np.abs(h) * c_err + h_err * c1 + 6 * U * (np.abs(e) + np.abs(h) * c1 + m))

    d = want["dx"] / wide["scale"]
    e_d = U * np.abs(d)
    if duv is not None:
        e = duv * w2
        e_d = e_d + through(e, U * np.abs(e), h2, e_h2, s2) + U * (0 if drv is None else np.abs(drv))
    within(f64(got.dx), want["dx"], stored(want["dx"], abs(wide["scale"]) * e_d + U * np.abs(want["dx"]), dtype), "dx")
    dg = d * p * slope
    e_dg = np.abs(p * slope) * e_d + np.abs(d * slope) * e_p + np.abs(d * p) * e_slope + 3 * U * np.abs(dg)
    add = (rows + 64) * U

    def column(terms, err):
        return err.sum(0) + add * np.abs(terms).sum(0)

    if gate == "values":
        within(f64(got.dgate), want["dgate"], stored(want["dgate"], e_dg, dtype), "dgate")
    elif gate == "units":
        within(f64(got.dgate), want["dgate"], stored(want["dgate"], column(dg, e_dg), pt), "dgate")
    else:
        assert got.dgate is None
    dp = d * gv_
    e_dp = np.abs(gv_) * e_d + np.abs(d) * e_g + U * np.abs(dp)
    zero = np.zeros_like(xv)
    duz = zero if duv is None else duv
    for name, terms, err in (("dpre_weight", duz * h2, np.abs(duz) * e_h2 + U * np.abs(duz * h2)),
                             ("dpre_bias", duz, zero),
                             ("dpost_weight", dp * h1, np.abs(dp) * e_h1 + np.abs(h1) * e_dp + U * np.abs(dp * h1)),
                             ("dpost_bias", dp, e_dp)):
        value = getattr(got, name)
        if wide[name[1:]] is None:
            assert value is None
        else:
            within(f64(value), want[name], stored(want[name], column(terms, err), pt), name)
    if wide["post"]:
        f = dp * w1
        e_do = through(f, np.abs(w1) * e_dp + U * np.abs(f), h1, e_h1, s1)
    else:
        e_do = e_dp
    within(f64(got.do), want["do"], stored(want["do"], e_do + 2 * U * np.abs(want["do"]), dtype), "do")
    for a, c in zip(got, again):
        assert a is None or torch.equal(a, c)


def test_block_norm_without_rows(ctx):
    x = torch.empty(0, 24, device="cuda")
    gate = torch.ones(24, device="cuda")
    r, u, stats = block.block_norm(ctx, x, x, gate, stats=True, pre_weight=gate)
    d = block.block_norm_backward(ctx, x, x, x, x, stats, gate, pre_weight=gate)
    ctx.sync()
    assert r.shape == u.shape == (0, 24) and not d.dgate.any() and not d.dpre_weight.any()


# -------------------------------------------------------------------------------- recurrence
STREAMS = [  # streams, steps, n, dtype, kind, mix, extra row stride, shift
    (1, 1, 1, "f32", "sigmoid", False, 0, 0),
    (256, 1, 70, "bf16", "sigmoid", True, 0, 0),
    (300, 1, 33, "f16", "decay", False, 1, 1),
    (5, 3, 64, "f16", "sigmoid", False, 0, 0),
    (7, 31, 66, "bf16", "decay", True, 2, 0),
    (2, 127, 40, "f32", "sigmoid", True, 0, 0),
    (3, 128, 128, "bf16", "sigmoid", True, 0, 0),
    (3, 129, 65, "f32", "decay", False, 0, 0),
    (2, 200, 31, "bf16", "sigmoid", False, 3, 1),
    (1, 1000, 130, "f16", "sigmoid", True, 0, 2),
    (1, 6000, 34, "f32", "sigmoid", False, 0, 0),
    (4, 2500, 20, "bf16", "decay", True, 0, 0),
    (9, 65, 257, "bf16", "sigmoid", True, 0, 0),
    (1, 5000, 72, "bf16", "sigmoid", True, 0, 0),  # whole tiles at a time, in parts
    (2, 700, 192, "f32", "decay", True, 0, 0),
    (3, 1500, 64, "f16", "decay", False, 8, 8),
    (1200, 30, 264, "bf16", "sigmoid", True, 0, 0),  # several streams a walk
    (700, 100, 128, "f32", "sigmoid", False, 0, 0),
    (1, 64, 16, "bf16", "sigmoid", True, 0, 0),
    (2, 33, 64, "bf16", "sigmoid", True, 0, 0),
]


def stream_inputs(streams, rows, n, dtype, kind, more, shift):
    g = rng(streams, rows, n)
    slow = g.uniform(0, 7, size=n)
    raw = g.normal(size=(rows, n)) + slow
    if kind == "decay":
        raw = 1 / (1 + np.exp(-raw)) * np.where(g.random((rows, n)) < 0.05, -1, 1)
    x, xv, _ = made(g.normal(size=(rows, n)), dtype, n + more, shift)
    gate, gv, _ = made(raw, dtype, n + more, shift)
    dh, dhv, _ = made(g.normal(size=(rows, n)), dtype, n + more, shift)
    state, sv, _ = made(g.normal(size=(streams, n)), "f32")
    dfinal, dfv, _ = made(g.normal(size=(streams, n)), "f32")
    return (x, xv), (gate, gv), (dh, dhv), (state, sv), (dfinal, dfv)


def gate_bounds(gv, kind):
    """a, 1 - a and how far each may be off."""
    a, keep = F.gates(gv, kind)
    if kind == "decay":
        return a, keep, 0 * a, U * np.abs(keep)
    off = (8 + 4 * np.minimum(np.abs(gv), 100)) * U  # of e^-|gate|, relative
    return a, keep, a * keep * off + 3 * U * a + 1e-37, keep * (a * off + 4 * U) + 1e-37


def walk(a, b, e_a, e_b, given, cuts, back):
    """Bounds of h_t = a_t h_{t-1} + b_t folded in any order: each of its terms goes through at most two
    roundings (and a's own error) a step and a hundred in joining runs. Backwards: g_t = b_t + a_{t+1} g_{t+1}."""
    size, off = np.zeros_like(b), np.zeros_like(b)
    end, end_off = np.abs(given).copy(), np.zeros_like(given)
    for s in range(len(cuts) - 1):
        m, e = np.abs(given[s]), np.zeros(b.shape[1])
        steps = range(cuts[s], cuts[s + 1])
        for t in reversed(steps) if back else steps:
            if not back:
                e = np.abs(a[t]) * e + (e_a[t] + 2 * U * np.abs(a[t])) * m + e_b[t]
                m = np.abs(a[t]) * m + np.abs(b[t])
                size[t], off[t] = m, e
            else:
                m, e = m + np.abs(b[t]), e + e_b[t]
                size[t], off[t] = m, e
                e = np.abs(a[t]) * e + (e_a[t] + 2 * U * np.abs(a[t])) * m
                m = np.abs(a[t]) * m
        end[s], end_off[s] = m, e
    return off + 100 * U * size, end_off + 100 * U * end


def check_recurrence(ctx, streams, rows, n, dtype, kind, mix, cuts, offsets, inputs, shape):
    (x, xv), (gate, gv), (dh, dhv), (state, sv), (dfinal, dfv) = inputs
    how = dict(kind=kind, mix=mix, offsets=offsets)
    out = torch.full_like(x, 5.0) if x.is_contiguous() else None
    h, final = block.recurrence(ctx, x.view(shape), gate.view(shape), state, out=None if out is None else out.view(shape),
                                **how)
    ctx.sync()
    a, keep, e_a, e_keep = gate_bounds(gv, kind)
    b = keep * xv if mix else xv
    e_b = (np.abs(xv) * e_keep + U * np.abs(b)) if mix else 0 * xv
    want, wfinal = F.recurrence(xv, gv, sv, cuts, kind, mix)
    tol, ftol = walk(a, b, e_a, e_b, sv, cuts, False)
    owned = ~np.isnan(want)
    got = f64(h).reshape(rows, n)
    within(got[owned], want[owned], stored(want, tol, dtype)[owned], "h")
    within(f64(final), wfinal, ftol + U * np.abs(wfinal), "final")
    if out is not None:
        assert (got[~owned] == 5.0).all()
    h2, final2 = block.recurrence(ctx, x.view(shape), gate.view(shape), state, **how)
    assert torch.equal(final, final2) and np.array_equal(f64(h2).reshape(rows, n)[owned], got[owned])

    hv = np.where(owned, got, 0.0)
    dx, dgate, dstate = block.recurrence_backward(ctx, dh.view(shape), gate.view(shape), h, state, x=x.view(shape),
                                                  dfinal=dfinal, **how)
    again = block.recurrence_backward(ctx, dh.view(shape), gate.view(shape), h, state, x=x.view(shape), dfinal=dfinal, **how)
    ctx.sync()
    wx, wg, ws = F.recurrence_backward(dhv, xv, gv, hv, sv, dfv, cuts, kind, mix)
    gtol, stol = walk(a, dhv, e_a, 0 * dhv, dfv, cuts, True)
    gval = F.recurrence_backward(dhv, xv, gv, hv, sv, dfv, cuts, kind, False)[0]  # g itself
    before = np.zeros_like(xv)
    for s in range(streams):
        lo, hi = cuts[s], cuts[s + 1]
        if hi > lo:
            before[lo], before[lo + 1:hi] = sv[s], hv[lo:hi - 1]
    arm = before - xv if mix else before
    t_dx = keep * gtol + np.abs(gval) * e_keep + U * np.abs(wx) if mix else gtol
    t_da = np.abs(arm) * gtol + np.abs(gval) * 3 * U * (np.abs(before) + np.abs(xv))
    if kind == "sigmoid":
        t_da = a * keep * t_da + np.abs(gval * arm) * (keep * e_a + a * e_keep + 4 * U * a * keep)
    within(f64(dx).reshape(rows, n)[owned], wx[owned], stored(wx, t_dx, dtype)[owned], "dx")
    within(f64(dgate).reshape(rows, n)[owned], wg[owned], stored(wg, t_da, dtype)[owned], "dgate")
    within(f64(dstate), ws, stol + U * np.abs(ws), "dstate")
    assert torch.equal(dstate, again[2])
    for p, q in zip((dx, dgate), again):
        assert np.array_equal(f64(p).reshape(rows, n)[owned], f64(q).reshape(rows, n)[owned])


@pytest.mark.parametrize("streams, steps, n, dtype, kind, mix, more, shift", STREAMS)
def test_recurrence(ctx, streams, steps, n, dtype, kind, mix, more, shift):
    rows = streams * steps
    inputs = stream_inputs(streams, rows, n, dtype, kind, more, shift)
    shape = (streams, steps, n) if more == 0 and shift == 0 else (streams, steps, n) if streams == 1 else None
    if shape is None:  # rows of one stride
        inputs = tuple((t.unflatten(0, (streams, steps)), v) if t.shape[0] == rows and i < 3 else (t, v)
                       for i, (t, v) in enumerate(inputs))
        shape = inputs[0][0].shape
    cuts = [s * steps for s in range(streams + 1)]
    check_recurrence(ctx, streams, rows, n, dtype, kind, mix, cuts, None, inputs, shape)


RAGGED = [  # offsets, rows, n, dtype, kind, mix
    ([0, 1], 1, 5, "f32", "sigmoid", True),
    ([0, 0, 0, 4, 4], 4, 64, "bf16", "sigmoid", False),
    ([3, 3, 10, 11, 140, 140, 300], 333, 34, "f32", "decay", False),
    ([0, 500, 501, 502, 1400, 1400], 1500, 66, "bf16", "sigmoid", True),
    ([5, 5], 9, 8, "f16", "sigmoid", True),
    (list(range(0, 201)), 200, 40, "f32", "sigmoid", True),
    ([0, 128, 256, 257, 4000], 4000, 33, "f16", "decay", True),
    ([7, 2400], 2500, 64, "f32", "sigmoid", False),
    ([0, 3, 3, 70, 1000, 1064, 1065, 3000], 3001, 72, "bf16", "sigmoid", True),
]


@pytest.mark.parametrize("cuts, rows, n, dtype, kind, mix", RAGGED)
def test_recurrence_of_ragged_streams(ctx, cuts, rows, n, dtype, kind, mix):
    streams = len(cuts) - 1
    inputs = stream_inputs(streams, rows, n, dtype, kind, 0, 0)
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    check_recurrence(ctx, streams, rows, n, dtype, kind, mix, cuts, offsets, inputs, (rows, n))


@pytest.mark.parametrize("cuts, rows, n, dtype", [
    ([2, 130, 131, 400, 400, 900], 1000, 64, "f32"), ([3, 10], 40, 31, "bf16"), ([5, 5], 9, 8, "f16"),
    ([0, 3000], 3001, 72, "bf16"), ([9, 2400], 2400, 33, "f32"), ([0, 7, 12], 12, 40, "f32")])
def test_rows_of_no_stream_are_zero_in_new_results(ctx, cuts, rows, n, dtype):
    """In memory that held NaN; what a layer's gradients sum over padded rows stays finite."""
    g = torch.Generator(device="cuda").manual_seed(12)
    x, gate, dh = (torch.randn(rows, n, device="cuda", generator=g).to(TYPES[dtype]) for _ in range(3))
    state = torch.zeros(len(cuts) - 1, n, device="cuda")
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    none = torch.ones(rows, dtype=torch.bool, device="cuda")
    none[cuts[0]:cuts[-1]] = False
    for t in (x, gate, dh):
        t[none] = float("nan")
    for mix in (False, True):
        held = [torch.full_like(x, float("nan")) for _ in range(3)]
        del held
        h, _ = block.recurrence(ctx, x, gate, state, mix=mix, offsets=offsets)
        held = [torch.full_like(x, float("nan")) for _ in range(3)]
        del held
        dx, dgate, _ = block.recurrence_backward(ctx, dh, gate, h, state, x=x, mix=mix, offsets=offsets)
        weight = torch.ones(16, n, device="cuda").to(TYPES[dtype])
        _, dweight, _ = block.dense_backward(ctx, dx @ weight.T, h, weight)
        ctx.sync()
        for t in (h, dx, dgate):
            assert (t[none] == 0).all() and t[~none].isfinite().all()
        assert dweight.isfinite().all()


def test_streams_keep_to_themselves(ctx):
    """NaN and infinity of one stream, and in rows of none, do not reach another."""
    cuts = [2, 130, 131, 400, 400, 900]
    n, rows = 64, 1000
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, n, device="cuda", generator=g)
    gate = torch.rand(rows, n, device="cuda", generator=g)
    state = torch.randn(5, n, device="cuda", generator=g)
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    h, final = block.recurrence(ctx, x, gate, state, kind="decay", offsets=offsets)
    bad, bad_gate, bad_state = x.clone(), gate.clone(), state.clone()
    for t in (bad, bad_gate):
        t[:2] = float("nan")
        t[130:131] = float("inf")
        t[900:] = float("nan")
    bad[399], bad_state[2] = float("inf"), float("nan")
    h2, final2 = block.recurrence(ctx, bad, bad_gate, bad_state, kind="decay", offsets=offsets)
    ctx.sync()
    for lo, hi in ((2, 130), (400, 900)):
        assert torch.equal(h[lo:hi], h2[lo:hi])
    for s in (0, 3, 4):
        assert torch.equal(final[s], final2[s])
    assert not final2[1].isfinite().any()
    dh = torch.randn(rows, n, device="cuda", generator=g)
    dx, dgate, dstate = block.recurrence_backward(ctx, dh, gate, h, state, kind="decay", offsets=offsets)
    bad_dh = dh.clone()
    bad_dh[:2], bad_dh[130:400], bad_dh[900:] = float("nan"), float("inf"), float("nan")
    dx2, dgate2, dstate2 = block.recurrence_backward(ctx, bad_dh, gate, h, state, kind="decay", offsets=offsets)
    ctx.sync()
    for lo, hi in ((2, 130), (400, 900)):
        assert torch.equal(dx[lo:hi], dx2[lo:hi]) and torch.equal(dgate[lo:hi], dgate2[lo:hi])
    for s in (0, 3, 4):
        assert torch.equal(dstate[s], dstate2[s])


@pytest.mark.parametrize("streams, steps, dtype", [(6, 1, "f32"), (6, 5, "f32"), (6, 700, "f32"), (6, 700, "bf16"),
                                                   (5000, 40, "bf16"), (6, 60, "bf16"), (6, 1, "f16")])
def test_recurrence_in_place(ctx, streams, steps, dtype):
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(streams, steps, 48, device="cuda", generator=g).to(TYPES[dtype])
    gate = torch.randn(streams, steps, 48, device="cuda", generator=g).to(TYPES[dtype])
    state = torch.randn(streams, 48, device="cuda", generator=g)
    h, final = block.recurrence(ctx, x, gate, state)
    for where in ("x", "gate"):
        t = {"x": x.clone(), "gate": gate.clone()}
        st = state.clone()
        h2, f2 = block.recurrence(ctx, t["x"], t["gate"], st, out=t[where], final_out=st)
        assert h2 is t[where] and f2 is st and torch.equal(h2, h) and torch.equal(st, final)
    empty, same = block.recurrence(ctx, x[:, :0], gate[:, :0], state)
    assert empty.shape == (streams, 0, 48) and torch.equal(same, state)
    ctx.sync()


def test_a_stream_in_two_calls_has_the_values_of_one(ctx):
    """The state that a call leaves is what the next one goes on from: to the last bit where the cut is
    between tiles that are walked in the same order."""
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(1, 128, 64, device="cuda", generator=g)
    gate = torch.randn(1, 128, 64, device="cuda", generator=g) + 2
    h, final = block.recurrence(ctx, x, gate)
    one, state = block.recurrence(ctx, x[:, :64], gate[:, :64])
    two, last = block.recurrence(ctx, x[:, 64:], gate[:, 64:], state)
    ctx.sync()
    both = torch.cat([one, two], 1)
    # values of order one through a hundred roundings of half a step at most
    assert (both - h).abs().max() < 100 * U * 4 and (last - final).abs().max() < 100 * U * 4


@pytest.mark.parametrize("rows, cuts", [(None, None), (3000, [0, 10, 10, 1500, 3000])])
def test_recurrence_backward_in_place_in_c(ctx, rows, cuts):
    """dx over dh, dgate over gate and dstate over dfinal, as the C interface allows."""
    g = torch.Generator(device="cuda").manual_seed(9)
    for streams, steps, n in ((40, 6, 24), (3, 900, 64), (2, 333, 31)):
        if cuts:
            streams, total, offsets = len(cuts) - 1, rows, torch.tensor(cuts, dtype=torch.int32, device="cuda")
        else:
            total, offsets = streams * steps, None
        shape = (total, n) if cuts else (streams, steps, n)
        x, gate, dh = (torch.randn(shape, device="cuda", generator=g) for _ in range(3))
        state, dfinal = (torch.randn(streams, n, device="cuda", generator=g) for _ in range(2))
        h, _ = block.recurrence(ctx, x, gate, state, mix=True, offsets=offsets)
        want = block.recurrence_backward(ctx, dh, gate, h, state, x=x, dfinal=dfinal, mix=True, offsets=offsets)
        size = _abi.lib().plx_recurrence_scratch_bytes(streams, total, n, 0, int(offsets is not None), 1, 1)
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        at = None if offsets is None else offsets.data_ptr()
        _abi.call("plx_recurrence_backward", ctx.handle, streams, total, n, 0, at, dh.data_ptr(), n, x.data_ptr(), n,
                  gate.data_ptr(), n, 1, 1, h.data_ptr(), n, state.data_ptr(), dfinal.data_ptr(), dh.data_ptr(), n,
                  gate.data_ptr(), n, dfinal.data_ptr(), scratch.data_ptr(), size)
        ctx.sync()
        for a, b in zip((dh, gate, dfinal), want):
            assert torch.equal(a, b)


def test_bad_offsets_are_reported(ctx):
    x = torch.zeros(40, 32, device="cuda")
    for cuts in ([0, 20, 10, 40], [0, 20, 41], [-1, 40]):
        block.recurrence(ctx, x, x, offsets=torch.tensor(cuts, dtype=torch.int32, device="cuda"))
        with pytest.raises(_abi.PlxError, match="offsets"):
            ctx.sync()
    ctx.sync()


# --------------------------------------------------------------------------------- together
class Layers:
    """One recurrent block between two norms, and the read-out behind it."""

    def __init__(self, n, wide, outputs, dtype, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale=1.0, mean=0.0):
            return torch.empty(shape, device="cuda").normal_(mean, scale, generator=g).to(dtype)

        self.p = {"w_in": normal(wide, n, scale=n ** -0.5), "b_in": normal(wide, scale=0.1),
                  "w_gate": normal(wide, n, scale=n ** -0.5), "b_gate": normal(wide, scale=1.0, mean=2.0),
                  "w_out": normal(n, wide, scale=wide ** -0.5), "scale": normal(n, scale=0.2, mean=0.8),
                  "post": normal(n, scale=0.1, mean=1.0), "pre": normal(n, scale=0.1, mean=1.0),
                  "w_read": normal(outputs, n, scale=n ** -0.5)}

    def step(self, ctx, x, u, state, target, minus):
        """Loss and gradients by the framework's calls."""
        p = self.p
        flat = u.view(-1, u.shape[-1])
        z, z_pre = block.dense(ctx, u, p["w_in"], p["b_in"], apply="silu", pre=True)
        gate = block.dense(ctx, u, p["w_gate"], p["b_gate"])
        h, final = block.recurrence(ctx, z, gate, state, mix=True)
        o = block.dense(ctx, h, p["w_out"])
        how = dict(post_weight=p["post"], pre_weight=p["pre"])
        r, v, stats = block.block_norm(ctx, x, o, p["scale"], stats=True, **how)
        logits = block.dense(ctx, v, p["w_read"])
        s = readout.log_probs(ctx, logits, target)
        d = readout.log_probs_backward(ctx, logits, s.lse, target, minus)
        dv, g_read, _ = block.dense_backward(ctx, d, v, p["w_read"])
        n = block.block_norm_backward(ctx, None, dv, x, o, stats, p["scale"], **how)
        dh, g_out, _ = block.dense_backward(ctx, n.do, h, p["w_out"])
        dz, dgate, dstate = block.recurrence_backward(ctx, dh, gate, h, state, x=z, mix=True)
        du1, g_in, gb_in = block.dense_backward(ctx, dz, u, p["w_in"], z_pre, apply="silu", bias=p["b_in"])
        du2, g_gate, gb_gate = block.dense_backward(ctx, dgate, u, p["w_gate"], bias=p["b_gate"])
        assert flat.shape[0] == target.numel()
        return {"logp": s.logp, "final": final, "r": r, "dx": n.dx, "du": du1 + du2, "dstate": dstate, "w_read": g_read,
                "w_out": g_out, "w_in": g_in, "b_in": gb_in, "w_gate": g_gate, "b_gate": gb_gate, "scale": n.dgate,
                "post": n.dpost_weight, "pre": n.dpre_weight}

    def exact(self, x, u, state, target):
        """The same by automatic differentiation in 64 bits."""
        leaf = {k: v.double().requires_grad_() for k, v in {**self.p, "dx": x, "du": u, "dstate": state}.items()}
        f = torch.nn.functional
        z = f.silu(f.linear(leaf["du"], leaf["w_in"], leaf["b_in"]))
        a = torch.sigmoid(f.linear(leaf["du"], leaf["w_gate"], leaf["b_gate"]))
        now, steps = leaf["dstate"], []
        for t in range(x.shape[1]):
            now = a[:, t] * now + (1 - a[:, t]) * z[:, t]
            steps.append(now)
        o = f.linear(torch.stack(steps, 1), leaf["w_out"])

        def norm(v, w):
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w

        r = leaf["dx"] + leaf["scale"] * norm(o, leaf["post"])
        logits = f.linear(norm(r, leaf["pre"]), leaf["w_read"])
        logp = torch.log_softmax(logits, -1).gather(-1, target.long()[..., None])[..., 0]
        (-logp.sum()).backward()
        return {"logp": logp.detach(), "final": now.detach(), "r": r.detach(), **{k: v.grad for k, v in leaf.items()}}


def chain_inputs(streams, steps, n, wide, outputs, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(streams, steps, n, device="cuda", generator=g).to(dtype)
    u = torch.randn(streams, steps, n, device="cuda", generator=g).to(dtype)
    state = torch.randn(streams, wide, device="cuda", generator=g)
    target = torch.randint(0, outputs, (streams, steps), device="cuda", generator=g, dtype=torch.int32)
    return x, u, state, target, torch.full((streams, steps), -1.0, device="cuda")


@pytest.mark.parametrize("dtype, tol", [("f32", 1e-4), ("bf16", 0.06), ("f16", 0.008)])
def test_block_and_readout_together(ctx, dtype, tol):
    """One training step of a recurrent block with its read-out: a handful of roundings to the rows' type
    (each half a step of every value, relative to the whole 2^-9, 2^-12 or less) between input and gradient,
    a dozen in the longest path."""
    layers = Layers(96, 160, 264, TYPES[dtype], 1)
    x, u, state, target, minus = chain_inputs(4, 150, 96, 160, 264, TYPES[dtype], 2)
    got = layers.step(ctx, x, u, state, target, minus)
    ctx.sync()
    want = layers.exact(x, u, state, target)
    assert got.keys() == want.keys()
    for k, w in want.items():
        rel = ((got[k].double() - w).norm() / w.norm()).item()
        assert rel < tol, (k, rel)


def test_chain_captured_and_replayed(ctx):
    """The step in a CUDA graph: captured in a process whose eager calls went before, replayed on new inputs."""
    layers = Layers(64, 128, 72, torch.bfloat16, 3)
    one, two = (chain_inputs(3, 300, 64, 128, 72, torch.bfloat16, s) for s in (4, 5))
    want = [layers.step(ctx, *i) for i in (one, two)]
    ctx.sync()
    held = [t.clone() for t in one]
    stream = torch.cuda.Stream()
    other = Context(0, stream)
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = layers.step(other, *held)
    for inputs, w in ((one, want[0]), (two, want[1]), (one, want[0])):
        for t, v in zip(held, inputs):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        for k in w:
            assert torch.equal(got[k], w[k]), k
    other.sync()


def test_calls_on_two_streams(ctx):
    """The same calls on two streams at once, each context with its own stream and scratch."""
    layers = Layers(64, 128, 72, torch.bfloat16, 6)
    inputs = chain_inputs(3, 500, 64, 128, 72, torch.bfloat16, 7)
    want = layers.step(ctx, *inputs)
    ctx.sync()
    streams = [torch.cuda.Stream() for _ in range(2)]
    contexts = [Context(0, s) for s in streams]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s, c in zip(streams, contexts):
            with torch.cuda.stream(s):
                got.append(layers.step(c, *inputs))
    for c in contexts:
        c.sync()
    for g in got:
        for k in want:
            assert torch.equal(g[k], want[k]), k


def test_context_stream_is_not_the_current_one(ctx):
    stream = torch.cuda.Stream()
    other = Context(0, stream)
    g = torch.Generator(device="cuda").manual_seed(8)
    x = torch.randn(40, 130, device="cuda", generator=g)
    w = torch.randn(50, 130, device="cuda", generator=g)
    want = (block.dense(ctx, x, w), *block.block_norm(ctx, x, x), *block.recurrence(ctx, x, x))
    ctx.sync()
    stream.wait_stream(torch.cuda.current_stream())
    got = (block.dense(other, x, w), *block.block_norm(other, x, x), *block.recurrence(other, x, x))
    other.sync()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_offsets_past_32_bits(ctx):
    """Rows that begin more than 2^32 values into their array."""
    n, ld = 64, 1 << 20
    rows = 4100
    buf = torch.empty((rows - 1) * ld + n, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(9)
    small = torch.randn(rows, n, device="cuda", generator=g).to(torch.bfloat16)
    far = buf.as_strided((rows, n), (ld, 1))
    far.copy_(small)
    w = torch.randn(40, n, device="cuda", generator=g).to(torch.bfloat16)
    want = (block.dense(ctx, small, w), *block.block_norm(ctx, small, small), *block.recurrence(ctx, small, small))
    got = (block.dense(ctx, far, w), *block.block_norm(ctx, far, far), *block.recurrence(ctx, far, far))
    ctx.sync()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del buf, far
    torch.cuda.empty_cache()
