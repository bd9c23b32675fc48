"""The read-out operators on the device against their 64-bit formulas.

Tolerances are bounds from the operators' own arithmetic, with U = 2^-24 the
unit of a 32-bit rounding and `depth(n)` at least the number of additions any
value of an n-term sum goes through; the stored result adds half a step of its
type. Inputs are rounded to their type first, so both sides read the same
values."""
import numpy as np
import pytest
import torch

import readout_formulas as F
from plastix_b200 import _abi, readout
from plastix_b200.runtime import Context

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 1e-37, "bf16": 1e-37, "f16": 2.0 ** -25}  # half a step of the smallest values


def depth(n):
    return n / 32 + 64


def f64(t):
    return t.detach().double().cpu().numpy()


def rows_tensor(a, dtype, ld=None, shift=0):
    """Rows on the device with the given row stride, starting `shift` elements into a buffer."""
    rows, n = a.shape
    ld = ld or n
    buf = torch.full((shift + rows * ld + 8,), 7.0, dtype=TYPES[dtype], device="cuda")
    t = buf.as_strided((rows, n), (ld, 1), shift)
    t.copy_(torch.from_numpy(np.ascontiguousarray(a)))
    return t, buf


def within(got, want, tol, what):
    got, tol = np.asarray(got, np.float64), np.broadcast_to(tol, want.shape)
    assert got.shape == want.shape, what
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    fine = np.isfinite(want)
    np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)], what)
    off = np.abs(got[fine] - want[fine])
    over = off - tol[fine]
    assert over.size == 0 or over.max() <= 0, \
        f"{what}: off by {off[over.argmax()]:.3g}, allowed {tol[fine][over.argmax()]:.3g}"


# ------------------------------------------------------------------------------- layer norm
def norm_tolerance(x, w, b, eps, rstd, half):
    n = x.shape[1]
    mean_err = depth(n) * U * np.abs(x).mean(1)
    rel = (depth(n) + 12) * U + (mean_err * rstd) ** 2
    h = (x - x.mean(1, keepdims=True)) * rstd[:, None]
    h_err = (mean_err * rstd)[:, None] + np.abs(h) * rel[:, None]
    y = h * w + b
    return mean_err + U * np.abs(x.mean(1)), rel * rstd, \
        (np.abs(w) * h_err + 3 * U * (np.abs(h * w) + np.abs(b))) * (1 + half) + half * np.abs(y)


def gradient_tolerance(dy, x, mean, rstd, w, dx, dw, db, half, ph):
    """Of dx, dw and db with the statistics that the call was given."""
    rows, n = x.shape
    h, g = (x - mean[:, None]) * rstd[:, None], dy * w
    e1 = (depth(n) + 2) * U * np.abs(g).mean(1, keepdims=True)
    e2 = (depth(n) + 6) * U * np.abs(g * h).mean(1, keepdims=True)
    c1, c2 = g.mean(1, keepdims=True), (g * h).mean(1, keepdims=True)
    err = rstd[:, None] * (e1 + np.abs(h) * e2 + 6 * U * (np.abs(g) + np.abs(c1) + np.abs(h * c2)))
    down = (min(rows, rows / 16 + 700) + 8) * U
    return err * (1 + half) + half * np.abs(dx), \
        down * np.abs(dy * h).sum(0) * (1 + ph) + ph * np.abs(dw), \
        down * np.abs(dy).sum(0) * (1 + ph) + ph * np.abs(db)


NORM_CASES = [  # rows, n, type, type of the weights, row stride beyond n, elements before the first row
    (1, 1, "f32", "f32", 0, 0), (5, 1, "bf16", "bf16", 0, 1), (3, 2, "f16", "f16", 1, 1),
    (7, 33, "f32", "f32", 0, 0), (1, 1024, "bf16", "bf16", 0, 0), (33, 1024, "f16", "f32", 0, 0),
    (129, 1000, "bf16", "f32", 0, 0), (65, 1001, "f32", "f32", 0, 0), (64, 1001, "bf16", "bf16", 7, 3),
    (300, 256, "bf16", "bf16", 0, 0), (1000, 96, "f32", "f32", 0, 0), (40, 2048, "f32", "f32", 8, 0),
    (600, 4096, "bf16", "bf16", 0, 0), (50, 4097, "f16", "f16", 0, 0), (37, 8192, "bf16", "f32", 0, 0),
    (20, 8200, "f32", "f32", 0, 4), (9, 20001, "bf16", "bf16", 0, 0), (3, 65536, "f32", "f32", 0, 0),
    (2500, 40, "f16", "f16", 0, 0), (700, 520, "f32", "f32", 3, 1),
    (21, 512, "bf16", "bf16", 0, 0), (19, 200, "f32", "f32", 0, 0), (13, 1536, "bf16", "f32", 0, 0),
    (7, 16384, "bf16", "bf16", 0, 0), (5, 4096, "f32", "f32", 0, 0), (5, 8192, "f32", "f32", 0, 0),
    (11, 254, "bf16", "bf16", 0, 0), (11, 1002, "f16", "f32", 0, 2), (9, 2050, "bf16", "bf16", 0, 0),
    (6, 5002, "f16", "f16", 0, 0), (4, 9002, "bf16", "bf16", 0, 0), (9, 129, "f16", "f16", 0, 0),
    (9, 777, "bf16", "bf16", 0, 0), (9, 1501, "bf16", "f32", 0, 0), (9, 2301, "f16", "f16", 0, 3),
    (9, 3333, "f16", "f16", 0, 0), (9, 5001, "bf16", "bf16", 0, 0), (9, 7777, "f32", "f32", 0, 0),
    (6000, 255, "bf16", "bf16", 0, 0), (5000, 128, "f32", "f32", 0, 0), (700, 4097, "f16", "f16", 0, 0),
    (1, 8191, "bf16", "bf16", 0, 1), (2, 3, "bf16", "bf16", 0, 0), (1200, 1024, "f32", "f32", 0, 0),
    (150, 17000, "bf16", "bf16", 0, 0), (70, 16385, "f32", "f32", 0, 0), (130, 16384, "f16", "f16", 0, 1),
]


@pytest.mark.parametrize("rows, n, dtype, pdtype, pad, shift", NORM_CASES)
def test_layer_norm_and_its_gradient(ctx, rows, n, dtype, pdtype, pad, shift):
    r = np.random.default_rng(rows * 1000 + n)
    x, bufx = rows_tensor(r.normal(size=(rows, n)) * 1.7 + r.normal(size=(rows, 1)), dtype, n + pad, shift)
    dy, _ = rows_tensor(r.normal(size=(rows, n)), dtype, n + pad, shift)
    w = torch.from_numpy(1 + 0.3 * r.normal(size=n)).to("cuda", TYPES[pdtype])
    b = torch.from_numpy(0.3 * r.normal(size=n)).to("cuda", TYPES[pdtype])
    before = bufx.clone()
    half, eps = HALF_STEP[dtype], 1e-5
    y, mean, rstd = readout.layer_norm(ctx, x, w, b, eps=eps, stats=True)
    dx, dw, db = readout.layer_norm_backward(ctx, dy, x, mean, rstd, w)
    again = readout.layer_norm_backward(ctx, dy, x, mean, rstd, w)
    ctx.sync()
    assert torch.equal(bufx, before)
    for one, two in zip((dx, dw, db), again):
        assert torch.equal(one, two)
    X, W, B, DY = f64(x), f64(w), f64(b), f64(dy)
    Y, M, R = F.layer_norm(X, W, B, eps)
    tm, tr, ty = norm_tolerance(X, W, B, eps, R, half)
    within(f64(mean), M, tm, "mean")
    within(f64(rstd), R, tr, "rstd")
    within(f64(y), Y, ty + TINY[dtype], "y")
    # the gradient's formula with the statistics that the call was given
    M, R = f64(mean), f64(rstd)
    DX, DW, DB = F.layer_norm_backward(DY, X, M, R, W)
    tx, tw, tb = gradient_tolerance(DY, X, M, R, W, DX, DW, DB, half, HALF_STEP[pdtype])
    within(f64(dx), DX, tx + TINY[dtype], "dx")
    within(f64(dw), DW, tw + TINY[pdtype], "dw")
    within(f64(db), DB, tb + TINY[pdtype], "db")


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("rows, n, pdtype", [
    (5, 1, "f32"), (5, 2, "bf16"), (5, 7, "f32"), (5, 8, "bf16"), (5, 9, "f32"), (5, 23, "bf16"),
    (5, 250, "bf16"), (5, 249, "f32"), (5, 256, "bf16"), (5, 257, "f32"), (5, 505, "bf16"),
    (5, 513, "f32"), (5, 1000, "bf16"), (5, 1027, "f32"), (5, 2046, "bf16"), (5, 2055, "f32"),
    (5, 4098, "bf16"), (5, 8190, "f32"), (5, 16377, "bf16"), (310, 1001, "bf16"), (400, 5001, "bf16"),
    (2500, 77, "f32"), (1, 1001, "bf16"), (170, 9003, "bf16")])
def test_layer_norm_at_every_offset_writes_its_own_columns_only(ctx, rows, n, pdtype, apart):
    """Rows that start anywhere (`apart`: x, dy, y and dx each elsewhere), weights anywhere, y
    and dx in the middle of something else."""
    r = np.random.default_rng(n)
    ax, ad = r.normal(size=(rows, n)) + 0.5, r.normal(size=(rows, n))
    weight = torch.from_numpy(1 + 0.3 * r.normal(size=n)).to("cuda", TYPES[pdtype])
    half, ph = HALF_STEP["bf16"], HALF_STEP[pdtype]
    for shift in range(8) if rows < 100 else (0, 3):
        def place(a, k):
            return rows_tensor(a, "bf16", n + (9 + 2 * k if apart else 9), (shift + 3 * k * apart) % 8)
        (x, _), (dy, _), (out, guard), (dx, dguard) = (place(a, k) for k, a in
                                                       enumerate((ax, ad, ad * 0, ad * 0)))
        w = torch.empty(n + 8, device="cuda", dtype=weight.dtype)[shift:shift + n].copy_(weight)
        y, mean, rstd = readout.layer_norm(ctx, x, w, w, stats=True, out=out)
        _, dw, db = readout.layer_norm_backward(ctx, dy, x, mean, rstd, w, out=dx)
        ctx.sync()
        for t, g in ((out, guard), (dx, dguard)):
            rest = g.clone()
            rest.as_strided(t.shape, t.stride(), t.storage_offset()).fill_(7.0)
            assert torch.equal(rest, torch.full_like(rest, 7.0))
        W, X, DY = f64(w), f64(x), f64(dy)
        Y, M, R = F.layer_norm(X, W, W, 1e-5)
        tm, tr, ty = norm_tolerance(X, W, W, 1e-5, R, half)
        within(f64(mean), M, tm, "mean")
        within(f64(rstd), R, tr, "rstd")
        within(f64(out), Y, ty + TINY["bf16"], "y")
        M, R = f64(mean), f64(rstd)
        DX, DW, DB = F.layer_norm_backward(DY, X, M, R, W)
        tx, tw, tb = gradient_tolerance(DY, X, M, R, W, DX, DW, DB, half, ph)
        within(f64(dx), DX, tx + TINY["bf16"], "dx")
        within(f64(dw), DW, tw + TINY[pdtype], "dw")
        within(f64(db), DB, tb + TINY[pdtype], "db")
        if not apart:  # in place, the same kernels
            readout.layer_norm_backward(ctx, dy, x, mean, rstd, w, out=dy)
            readout.layer_norm(ctx, x, w, w, out=x)
            assert torch.equal(dy, dx) and torch.equal(x, out)


def test_layer_norm_without_weights_in_place_and_without_rows(ctx):
    r = np.random.default_rng(0)
    a = r.normal(size=(11, 300))
    x, _ = rows_tensor(a, "f32")
    want = readout.layer_norm(ctx, x)
    assert readout.layer_norm(ctx, x, out=x) is x
    ctx.sync()
    assert torch.equal(x, want)
    X = a.astype(np.float32).astype(np.float64)
    one, zero = np.ones(300), np.zeros(300)
    Y, _, R = F.layer_norm(X, one, zero, 1e-5)
    within(f64(want), Y, norm_tolerance(X, one, zero, 1e-5, R, U)[2], "y")
    y, mean, rstd = readout.layer_norm(ctx, want, stats=True)
    dy = torch.ones_like(y)
    dx, dw, db = readout.layer_norm_backward(ctx, dy, want, mean, rstd, out=dy)
    assert dx is dy and dw is None and db is None
    e = torch.empty(0, 300, device="cuda")
    w = torch.ones(300, device="cuda")
    y, mean, rstd = readout.layer_norm(ctx, e, w, stats=True)
    dx, dw, db = readout.layer_norm_backward(ctx, e, e, mean, rstd, w)
    ctx.sync()
    assert y.shape == (0, 300) and not dw.any() and not db.any()


def test_layer_norm_rows_that_are_constant_or_not_finite(ctx):
    x = torch.randn(6, 513, device="cuda")
    x[1] = 3.0
    x[2, 5] = float("nan")
    x[4, 7] = float("inf")
    y, mean, rstd = readout.layer_norm(ctx, x, stats=True)
    ctx.sync()
    assert torch.equal(y[1], torch.zeros(513, device="cuda"))
    # variance 0 exactly: 1/sqrt(eps), with eps and three roundings of 32 bits
    assert abs(float(rstd[1]) * 1e-5 ** 0.5 - 1) < 4 * U
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all()
    for r in (0, 3, 5):
        assert torch.isfinite(y[r]).all()


def test_layer_norm_large_offset_keeps_the_variance(ctx):
    # mean 1000, deviation 1: squares are taken after the mean is subtracted
    r = np.random.default_rng(5)
    x, _ = rows_tensor(1000 + r.normal(size=(4, 4096)), "f32")
    X = f64(x)
    y = readout.layer_norm(ctx, x)
    ctx.sync()
    one, zero = np.ones(4096), np.zeros(4096)
    Y, _, R = F.layer_norm(X, one, zero, 1e-5)
    within(f64(y), Y, norm_tolerance(X, one, zero, 1e-5, R, U)[2], "y")


# -------------------------------------------------------------------------- log probabilities
def score_errors(x, scale, logs, lse, entropy):
    """Bounds on the error of lse and of an entropy, rows whose lse is finite."""
    with np.errstate(invalid="ignore"):
        most = np.where(np.isfinite(x.max(1)), x.max(1), 0.0)
        log_s = np.where(np.isfinite(lse), lse - scale * most, 0.0)
        spread = np.where(np.isfinite(entropy), np.abs(log_s - entropy), 0.0)  # sum e |d| / s
        e = U * (4 + 3 * spread + depth(x.shape[1]))
        le = e + 4 * U * (np.abs(np.where(np.isfinite(lse), lse, 0)) + np.abs(log_s))
        he = e + 4 * U * np.abs(log_s) + spread * (2 * e + 6 * U) + U * np.abs(np.where(np.isfinite(entropy), entropy, 0))
    return e, le, he, most, log_s


def logp_tolerance(x_at, scale, e, most, log_s):
    d = np.abs(scale * (np.where(np.isfinite(x_at), x_at, 0.0) - most))
    return e + 4 * U * (d + np.abs(log_s)) + 1e-37


SCORE_CASES = [  # rows, n, type, top, scale, row stride beyond n, elements before the first row
    (1, 1, "f32", 1, 1.0, 0, 0), (3, 2, "bf16", 2, 1.0, 0, 1), (4, 7, "f16", 7, 0.5, 2, 1),
    (6, 64, "f32", 64, 1.3, 0, 0), (5, 65, "bf16", 64, 1.0, 0, 0), (130, 255, "f32", 3, 1.0, 0, 0),
    (17, 1000, "bf16", 5, 0.7, 0, 0), (64, 1001, "f16", 20, 1.0, 0, 0), (9, 4096, "f32", 40, 2.0, 8, 0),
    (1, 32000, "bf16", 64, 1.0, 0, 0), (8, 32003, "bf16", 5, 1.0, 0, 0), (3, 50001, "f32", 1, 1.0, 5, 2),
    (700, 2048, "bf16", 2, 1.0, 0, 0), (2, 131072, "f32", 20, 1.0, 0, 0), (1, 300007, "f16", 10, 1.0, 0, 0),
    (300, 20000, "f32", 8, 1.0, 0, 0), (170, 40010, "f16", 33, 0.25, 6, 0), (5, 1 << 20, "bf16", 16, 1.0, 0, 0),
    (200, 12000, "bf16", 4, 1.0, 0, 0), (150, 9001, "f32", 64, 1.0, 0, 1), (151, 70003, "f16", 17, 1.0, 0, 0),
]


@pytest.mark.parametrize("rows, n, dtype, top, scale, pad, shift", SCORE_CASES)
def test_log_probs_and_their_gradient(ctx, rows, n, dtype, top, scale, pad, shift):
    r = np.random.default_rng(rows * 7919 + n)
    a = r.normal(size=(rows, n)) * 2.5
    a[::3] = np.where(r.random(a[::3].shape) < 0.4, -np.inf, a[::3])
    a[::3, r.integers(n)] = 0.25  # at least one output that counts
    if rows > 4:
        a[4] = 1000.0 + a[4]  # a large common offset
    scale = float(np.float32(scale))
    x, bufx = rows_tensor(a, dtype, n + pad, shift)
    target = torch.from_numpy(r.integers(0, n, rows)).int().cuda()
    target[1::5] = -1
    before = bufx.clone()
    got = readout.log_probs(ctx, x, target, top=top, scale=scale, entropy=True)
    plain = readout.log_probs(ctx, x, scale=scale)
    gl = torch.from_numpy(r.normal(size=rows)).float().cuda()
    ge = torch.from_numpy(r.normal(size=rows)).float().cuda()
    dx = readout.log_probs_backward(ctx, x, got.lse, target, gl, got.entropy, ge, scale=scale)
    dl = readout.log_probs_backward(ctx, x, got.lse, target, gl, scale=scale)
    dh = readout.log_probs_backward(ctx, x, got.lse, entropy=got.entropy, grad_entropy=ge, scale=scale)
    ctx.sync()
    assert torch.equal(bufx, before)
    assert plain.logp is None and plain.entropy is None and plain.top_ids is None
    X, at = f64(x), target.cpu().numpy()
    want = F.log_probs(X, at, scale, top)
    logs, lse = F.log_softmax(X * scale)
    e, le, he, most, log_s = score_errors(X, scale, logs, lse, want["entropy"])
    within(f64(got.lse), want["lse"], le, "lse")
    within(f64(plain.lse), want["lse"], le, "lse alone")
    within(f64(got.entropy), want["entropy"], he, "entropy")
    x_at = X[np.arange(rows), np.maximum(at, 0)]
    within(f64(got.logp), want["logp"], logp_tolerance(x_at, scale, e, most, log_s), "logp")
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), want["top_ids"])
    x_top = np.take_along_axis(X, want["top_ids"], 1)
    within(f64(got.top_logp), want["top_logp"],
           logp_tolerance(x_top, scale, e[:, None], most[:, None], log_s[:, None]), "top_logp")
    # gradients: p is off by what lse is off and by its own exponent
    p = np.exp(logs)
    safe = np.where(np.isfinite(logs), logs, 0.0)
    pe = le[:, None] + U * (8 + 4 * np.abs(safe))
    half = HALF_STEP[dtype]
    for d, GL, GE in ((dx, f64(gl), f64(ge)), (dl, f64(gl), None), (dh, None, f64(ge))):
        DX = F.log_probs_backward(X, at, scale, GL, GE)
        G = 0.0 if GL is None else np.abs(np.where(at < 0, 0.0, GL))[:, None]
        H = 0.0 if GE is None else np.abs(GE)[:, None]
        inner = G + H * (np.abs(safe) + want["entropy"][:, None])
        err = scale * (p * (pe * inner + H * (le + he)[:, None] + 6 * U * inner) + 2 * U * G)
        within(f64(d), DX, err * (1 + half) + half * np.abs(DX) + 2 * TINY[dtype], "gradient")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [3, 100, 4099, 70000])
def test_alternatives_among_equals_take_the_lowest_index(ctx, dtype, n):
    r = np.random.default_rng(n)
    top = min(n, 37)
    a = np.stack([np.zeros(n), np.where(r.random(n) < 0.5, 0.0, -0.0),
                  r.integers(0, 3, n).astype(float),  # long runs of equals
                  np.full(n, -np.inf), np.arange(n) % 2.0,
                  np.minimum(np.arange(n), 2000.0),  # the best at the end, equal there
                  -np.arange(n, dtype=float).clip(0, 2000),
                  np.full(n, np.nan), np.where(np.arange(n) % 3 == 2, np.nan, np.inf),
                  np.where(np.arange(n) % 5 == 4, -0.0, -1.0),  # the best are zeros below zero
                  np.where(np.arange(n) >= n - 3, 1.0, 0.0)])
    a[3, n // 2:] = np.where(np.arange(n - n // 2) % 7 == 1, -5.0, -np.inf)  # fewer finite than asked for
    x, _ = rows_tensor(a, dtype)
    got = readout.log_probs(ctx, x, top=top)
    ctx.sync()
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), F.order(f64(x))[:, :top])


@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_alternatives_of_few_distinct_values(ctx, rows, dtype):
    # many threads tie at the threshold, with few or many elements above it, at any place
    n, top = 33333, 64
    r = np.random.default_rng(rows)
    a = r.integers(0, 40, (rows, n)) / 4.0
    a[:, :n // 2] = np.minimum(a[:, :n // 2], 9.0)
    a[::2] = np.minimum(a[::2], r.integers(1, 40, (len(a[::2]), 1)) / 4.0)
    for row in range(0, rows, 3):
        a[row, r.integers(0, n, 50)] = 30.0
    x, _ = rows_tensor(a, dtype)
    got = readout.log_probs(ctx, x, top=top)
    ctx.sync()
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), F.order(f64(x))[:, :top])


@pytest.mark.parametrize("stride", [1, 8, 256, 1024, 2048, 4096, 8192])
def test_alternatives_that_all_sit_in_one_place(ctx, stride):
    # the best values at a fixed distance: whatever part of the row one thread has, it may hold them all
    n, top = 131072, 64
    a = np.random.default_rng(stride).normal(size=(2, n))
    at = (np.arange(top) * stride + 5) % n
    a[0, at] = 10.0 + np.arange(top) / 8
    a[1, at] = 10.0
    x, _ = rows_tensor(a, "f32")
    got = readout.log_probs(ctx, x, top=top)
    ctx.sync()
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), F.order(f64(x))[:, :top])


@pytest.mark.parametrize("n", [5, 1000, 40001])
def test_log_probs_of_masked_and_non_finite_rows(ctx, n):
    x = torch.randn(6, n, device="cuda")
    x[1] = -float("inf")
    x[2, n // 2] = float("nan")
    x[3, n // 3] = float("inf")
    x[4] = -float("inf")
    x[4, n - 1] = 3.0
    x[5] = torch.finfo(torch.float32).min  # every output at the type's lowest value: uniform
    target = torch.tensor([0, 1, 2, 3, n - 1, 4], dtype=torch.int32, device="cuda")
    top = min(5, n)
    r = readout.log_probs(ctx, x, target, top=top, entropy=True)
    one = torch.ones(6, device="cuda")
    dx = readout.log_probs_backward(ctx, x, r.lse, target, one, r.entropy, one)
    ctx.sync()
    inf = float("inf")
    assert float(r.lse[1]) == -inf and float(r.logp[1]) == -inf and float(r.entropy[1]) == 0
    assert r.top_ids[1].tolist() == list(range(top)) and (r.top_logp[1] == -inf).all()
    want = torch.zeros(n, device="cuda")
    want[1] = 1.0  # p is 0 everywhere: only the target's own term is left
    assert torch.equal(dx[1], want)
    for row in (2, 3):
        assert torch.isnan(r.entropy[row]) and torch.isnan(r.top_logp[row, 0])
    assert torch.isnan(r.lse[2]) and int(r.top_ids[2, 0]) == n // 2
    assert int(r.top_ids[3, 0]) == n // 3
    assert float(r.logp[4]) == 0 and float(r.entropy[4]) == 0 and float(r.lse[4]) == 3.0
    assert int(r.top_ids[4, 0]) == n - 1 and not dx[4].any()
    # n equal probabilities: log n, with the logarithm's and one sum's roundings
    assert abs(float(r.entropy[5]) - np.log(n)) <= U * (depth(n) + 8 * np.log(n))
    assert abs(float(r.logp[5]) + np.log(n)) <= U * (depth(n) + 8 * np.log(n))


def test_entropy_of_rows_as_wide_as_the_type(ctx):
    # the running maximum moves from the type's lowest value upwards, masked values in between
    low, inf = torch.finfo(torch.float32).min, float("inf")
    x = torch.full((3, 50000), low, device="cuda")
    x[0, ::3] = -inf
    x[0, 40000] = 5.0
    x[1, :25000] = -inf
    x[2, 100:] = 1.0
    r = readout.log_probs(ctx, x, top=1, entropy=True)
    ctx.sync()
    for row, ways in ((0, 1), (1, 25000), (2, 49900)):
        assert abs(float(r.entropy[row]) - np.log(ways)) <= U * (depth(50000) + 8 * np.log(50000))


def test_a_target_outside_its_row_is_reported(ctx):
    x = torch.randn(3, 50, device="cuda")
    for bad in (50, -2, 2 ** 31 - 1):
        target = torch.tensor([1, bad, 2], dtype=torch.int32, device="cuda")
        r = readout.log_probs(ctx, x, target)
        with pytest.raises(_abi.PlxError, match="outside its row"):
            ctx.sync()
        assert float(r.logp[1]) == 0 and float(r.logp[0]) < 0
        dx = readout.log_probs_backward(ctx, x, r.lse, target, torch.ones(3, device="cuda"))
        ctx.sync()
        assert not dx[1].any() and dx[0].any()


# -------------------------------------------------------------------------------- distillation
DISTILL_CASES = [  # rows, n, type, k, temperature, kind, row stride beyond n, elements before the first row
    (1, 1, "f32", 1, 1.0, "logits", 0, 0), (3, 5, "f32", 3, 2.0, "log_probs", 0, 1),
    (4, 7, "bf16", 64, 1.0, "logits", 1, 0), (33, 250, "f16", 9, 0.5, "logits", 0, 0),
    (17, 1000, "bf16", 8, 1.0, "log_probs", 0, 0), (64, 1001, "f32", 50, 3.0, "logits", 6, 3),
    (16, 4096, "f32", 8, 1.0, "logits", 0, 0), (700, 2048, "bf16", 16, 2.0, "logits", 0, 0),
    (40, 20011, "f16", 50, 2.0, "logits", 0, 0), (9, 65536, "bf16", 32, 2.0, "log_probs", 0, 0),
    (2, 131072, "f32", 64, 1.0, "logits", 0, 0), (1, 300007, "bf16", 20, 1.0, "log_probs", 0, 1),
    (160, 40000, "f32", 4, 1.0, "logits", 0, 0), (3, 1 << 20, "f16", 12, 1.5, "logits", 8, 0),
    (2, 1000003, "f32", 7, 1.0, "logits", 0, 0), (300, 20001, "f16", 12, 1.0, "logits", 0, 0), (300, 12345, "bf16", 33, 1.0, "logits", 0, 0),
]


@pytest.mark.parametrize("rows, n, dtype, k, tau, kind, pad, shift", DISTILL_CASES)
def test_distill(ctx, rows, n, dtype, k, tau, kind, pad, shift):
    r = np.random.default_rng(rows * 104729 + n + k)
    a = r.normal(size=(rows, n)) * 2.0
    ids = r.integers(0, n, (rows, k))  # the same output twice here and there
    ids[r.random((rows, k)) < 0.2] = -1
    values = r.normal(size=(rows, k)) * 1.5
    if kind == "log_probs":
        values -= np.log(np.exp(values).sum(1, keepdims=True)) + 0.3
    values[r.random((rows, k)) < 0.1] = -np.inf
    weight = r.normal(size=rows) + 1.5
    if rows > 2:
        ids[1] = -1  # no teacher
        weight[2] = 0.0
        a[2, 0] = np.nan  # does not count
        a[::4] = np.where(r.random(a[::4].shape) < 0.3, -np.inf, a[::4])
        for row in range(0, rows, 4):
            a[row, np.maximum(ids[row], 0)] = 0.5  # what the teacher lists is not masked
    x, bufx = rows_tensor(a, dtype, n + pad, shift)
    I, V = torch.from_numpy(ids).int().cuda(), torch.from_numpy(values).float().cuda()
    W = torch.from_numpy(weight).float().cuda()
    before = bufx.clone()
    loss, dx = readout.distill(ctx, x, I, V, temperature=tau, kind=kind, weight=W)
    alone, none = readout.distill(ctx, x, I, V, temperature=tau, kind=kind, weight=W, grad=False)
    ctx.sync()
    assert torch.equal(bufx.nan_to_num(), before.nan_to_num()) and none is None
    X, VV, WW = f64(x), f64(V), f64(W)
    L, DX = F.distill(X, ids, VV, tau, kind, WW)
    counts = (ids >= 0).any(1) & (WW != 0)
    Z = np.where(np.isnan(X), 0.0, X)
    logs, lse = F.log_softmax(Z / tau)
    s = F.log_probs(Z, None, 1 / tau)
    e, le, _, most, log_s = score_errors(Z, 1 / tau, logs, lse, s["entropy"])
    big = np.where(np.isfinite(VV) & (ids >= 0), np.abs(VV), 0.0).max(1) / (tau if kind == "logits" else 1.0)
    qe = U * (24 + 8 * big + 16)
    t = np.where((ids >= 0) & np.isfinite(VV), VV, -np.inf)
    t = F.log_softmax(t / tau)[0] if kind == "logits" else t
    q = np.exp(t)
    lp = np.where(q > 0, np.take_along_axis(logs, np.maximum(ids, 0), 1), 0.0)
    lt = np.where(q > 0, t, 0.0)
    le_at = e[:, None] + 8 * U * (np.abs(lp) + np.abs(log_s)[:, None] + np.abs(most)[:, None] / tau)
    tol = np.abs(WW) * tau ** 2 * (q * (qe[:, None] * (1 + np.abs(lt) + np.abs(lp)) + le_at + 8 * U * (np.abs(lt) + np.abs(lp)))).sum(1)
    within(f64(loss), L, np.where(counts, tol, 0.0) + 1e-37, "loss")
    within(f64(alone), L, np.where(counts, tol, 0.0) + 1e-37, "loss alone")
    p, Q = np.exp(logs), q.sum(1)
    err = Q[:, None] * p * (qe[:, None] + le[:, None] + U * (16 + 6 * np.abs(np.where(np.isfinite(logs), logs, 0))))
    np.add.at(err, (np.arange(rows)[:, None], np.maximum(ids, 0)), q * qe[:, None] * 2)
    err *= np.abs(WW)[:, None] * tau
    half = HALF_STEP[dtype]
    within(f64(dx), DX, np.where(counts[:, None], err * (1 + half) + half * np.abs(DX), 0.0) + 2 * TINY[dtype], "dx")
    if rows > 2:
        assert not dx[1:3].any() and not loss[1:3].any()
    into, _ = rows_tensor(a, dtype, n + pad, shift)  # the gradient in place of the logits
    loss2, dx2 = readout.distill(ctx, into, I, V, temperature=tau, kind=kind, weight=W, out=into)
    ctx.sync()
    assert dx2 is into and torch.equal(dx2, dx) and torch.equal(loss2, loss)


def test_distill_edge_rows(ctx):
    n, inf = 300, float("inf")
    x = torch.randn(6, n, device="cuda")
    x[0, 7] = -inf       # the teacher lists a masked output
    x[1] = -inf          # the student masks everything
    x[2, 9] = float("nan")
    x[3] = inf           # does not count
    ids = torch.tensor([[7, 8], [3, 3], [1, 2], [1, 2], [5, 5], [6, -1]], dtype=torch.int32, device="cuda")
    vals = torch.zeros(6, 2, device="cuda")
    vals[5, 1] = float("nan")  # an empty entry's value is not read into anything
    w = torch.tensor([1.0, 2.0, 1.0, 0.0, 1.0, 1.0], device="cuda")
    loss, dx = readout.distill(ctx, x, ids, vals, temperature=2.0, weight=w)
    ctx.sync()
    assert float(loss[0]) == inf and float(dx[0, 7]) == -1.0  # -w tau q, q = 1/2
    assert float(loss[1]) == inf and float(dx[1, 3]) == -4.0 and int((dx[1] != 0).sum()) == 1
    assert torch.isnan(loss[2]) and torch.isnan(dx[2]).all()
    assert float(loss[3]) == 0 and not dx[3].any()
    L, DX = F.distill(f64(x[4:]), ids[4:].cpu().numpy(), f64(vals[4:]), 2.0, "logits", np.ones(2))
    # values of order ten; sums of 300: a bound on all roundings
    np.testing.assert_allclose(f64(loss[4:]), L, atol=10 * U * (depth(n) + 60))
    np.testing.assert_allclose(f64(dx[4:]), DX, atol=2 * U * (depth(n) + 60))
    bad = ids.clone()
    bad[5, 1] = n
    readout.distill(ctx, x, bad, vals)
    with pytest.raises(_abi.PlxError, match="outside its row"):
        ctx.sync()
    ctx.sync()


@pytest.mark.parametrize("kind", ["logits", "log_probs"])
def test_distill_where_the_teacher_masks_all_it_lists(ctx, kind):
    x = torch.randn(2, 90, device="cuda")
    ids = torch.tensor([[4, 5], [4, -1]], dtype=torch.int32, device="cuda")
    loss, dx = readout.distill(ctx, x, ids, torch.full((2, 2), -float("inf"), device="cuda"), kind=kind)
    ctx.sync()
    assert not loss.any() and not dx.any()


def test_distill_gradient_against_differences_of_the_loss(ctx):
    r = np.random.default_rng(11)
    n, k, tau, h = 64, 6, 1.5, 2.0 ** -5
    a = r.normal(size=(1, n))
    v = r.normal(size=(1, n))
    v /= np.abs(v).sum()  # along v the second and third derivative of the loss are at most 1
    I = torch.from_numpy(r.integers(0, n, (1, k))).int().cuda()
    V = torch.from_numpy(r.normal(size=(1, k))).float().cuda()
    at = lambda b: rows_tensor(b, "f32")[0]  # noqa: E731
    dx = readout.distill(ctx, at(a), I, V, temperature=tau)[1]
    up = readout.distill(ctx, at(a + h * v), I, V, temperature=tau, grad=False)[0]
    down = readout.distill(ctx, at(a - h * v), I, V, temperature=tau, grad=False)[0]
    ctx.sync()
    slope = (float(up) - float(down)) / (2 * h)
    # h^2/6 from the third derivative; the losses (below 16) are off by at most 80 roundings each
    assert abs(slope - float((f64(dx) * v).sum())) <= h * h / 6 + 2 * 16 * 80 * U / (2 * h)


# ------------------------------------------------------------------------ how the calls are made
def everything(ctx, s):
    """All five calls on one set of inputs."""
    y, mean, rstd = readout.layer_norm(ctx, s["x"], s["w"], s["b"], stats=True)
    r = readout.log_probs(ctx, s["z"], s["target"], top=4, entropy=True)
    dz = readout.log_probs_backward(ctx, s["z"], r.lse, s["target"], s["g"], r.entropy, s["g"])
    loss, dl = readout.distill(ctx, s["z"], r.top_ids, r.top_logp, kind="log_probs", weight=s["g"])
    dx, dw, db = readout.layer_norm_backward(ctx, s["x"], y, mean, rstd, s["w"])
    return [y, mean, rstd, *r, dz, loss, dl, dx, dw, db]


def inputs(seed, rows=70, n=1500, units=9000, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return {"x": rand(rows, n).to(dtype), "w": rand(n).to(dtype), "b": rand(n).to(dtype),
            "z": (2 * rand(rows, units)).to(dtype), "g": rand(rows),
            "target": torch.randint(-1, units, (rows,), device="cuda", generator=g, dtype=torch.int32)}


def test_calls_are_captured_and_replayed():
    stream = torch.cuda.Stream()
    c = Context(0, stream)
    sets = [inputs(k) for k in range(3)]
    want = []
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        want = [[t.clone() for t in everything(c, s)] for s in sets]
        static = {k: v.clone() for k, v in sets[0].items()}
        everything(c, static)
    c.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = everything(c, static)
    for s, w in list(zip(sets, want))[::-1]:
        with torch.cuda.stream(stream):
            for k in static:
                static[k].copy_(s[k])
            graph.replay()
        c.sync()
        for a, b in zip(out, w):
            assert torch.equal(a, b)
    del graph
    c.close()


def test_first_calls_of_a_process_can_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from plastix_b200 import readout
from plastix_b200.runtime import Context
s = torch.cuda.Stream()
c = Context(0, s)
x = torch.randn(40, 40960, device="cuda"); w = torch.ones(40960, device="cuda")
t = torch.zeros(40, dtype=torch.int32, device="cuda"); one = torch.ones(40, device="cuda")
torch.cuda.synchronize()
def calls():
    y, m, r = readout.layer_norm(c, x[:, :2048], w[:2048], stats=True)
    d = readout.layer_norm_backward(c, y, x[:, :2048], m, r, w[:2048])
    p = readout.log_probs(c, x, t, top=3, entropy=True)
    return [y, *d, *p, readout.log_probs_backward(c, x, p.lse, t, one, p.entropy, one),
            *readout.distill(c, x, p.top_ids, p.top_logp, kind="log_probs")]
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    got = calls()
with torch.cuda.stream(s):
    g.replay()
    want = calls()
c.sync()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("captured")
"""
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


def test_results_beside_their_input_in_one_buffer(ctx):
    buf = torch.randn(9, 2 * 1001, device="cuda").bfloat16()
    x, out = buf[:, :1001], buf[:, 1001:]
    keep = x.clone()
    assert torch.equal(readout.layer_norm(ctx, x, out=out), readout.layer_norm(ctx, keep))
    y, mean, rstd = readout.layer_norm(ctx, keep, stats=True)
    want = readout.layer_norm_backward(ctx, y, keep, mean, rstd)[0]
    got = readout.layer_norm_backward(ctx, y, x, mean, rstd, out=x)[0]  # dx takes x's place
    ctx.sync()
    assert got is x and torch.equal(got, want)
    with pytest.raises(ValueError, match="overlaps"):
        readout.layer_norm_backward(ctx, y, x, mean, rstd, out=buf[:, 500:1501])


def test_two_contexts_on_two_streams_at_once(ctx):
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    both = [Context(0, s) for s in streams]
    sets = [inputs(20, rows=300), inputs(21, rows=260)]
    want = [everything(ctx, s) for s in sets]
    ctx.sync()
    torch.cuda.synchronize()
    for _ in range(3):  # the streams are not torch's current one: results belong to the context's
        got = [everything(c, s) for c, s in zip(both, sets)]
        for c in both:
            c.sync()
        for g, w in zip(got, want):
            for a, b in zip(g, w):
                assert torch.equal(a, b)
    for c in both:
        c.close()


def test_offsets_past_32_bits(ctx):
    n, ld = 1000, (1 << 30) + 8
    big = torch.zeros(2 * ld + n, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((3, n), (ld, 1))
    x.copy_(torch.randn(3, n, device="cuda"))
    small = x.clone()
    out = torch.zeros_like(big).as_strided((3, n), (ld, 1))
    w = torch.ones(n, device="cuda")
    y, mean, rstd = readout.layer_norm(ctx, x, w, w, stats=True)
    sy, smean, srstd = readout.layer_norm(ctx, small, w, w, stats=True)
    assert torch.equal(readout.layer_norm(ctx, x, w, w, out=out), sy)
    a = readout.layer_norm_backward(ctx, x, x, mean, rstd, w, out=out)
    b = readout.layer_norm_backward(ctx, small, small, smean, srstd, w)
    for p, q in zip((y, *a), (sy, *b)):
        assert torch.equal(p, q)
    target = torch.tensor([3, 4, 5], dtype=torch.int32, device="cuda")
    g = torch.ones(3, device="cuda")
    r, s = (readout.log_probs(ctx, t, target, top=3, entropy=True) for t in (x, small))
    for p, q in zip(r, s):
        assert torch.equal(p, q)
    assert torch.equal(readout.log_probs_backward(ctx, x, r.lse, target, g, out=out),
                       readout.log_probs_backward(ctx, small, r.lse, target, g))
    for p, q in zip(readout.distill(ctx, x, r.top_ids, r.top_logp, out=out),
                    readout.distill(ctx, small, r.top_ids, r.top_logp)):
        assert torch.equal(p, q)
    ctx.sync()


def test_rows_of_several_dimensions(ctx):
    x = torch.randn(2, 3, 5, 40, device="cuda")
    flat = x.reshape(30, 40)
    assert torch.equal(readout.layer_norm(ctx, x).view(30, 40), readout.layer_norm(ctx, flat))
    r, s = readout.log_probs(ctx, x, top=2), readout.log_probs(ctx, flat, top=2)
    assert r.top_ids.shape == (2, 3, 5, 2) and torch.equal(r.top_ids.view(30, 2), s.top_ids)
    one = readout.log_probs(ctx, flat[0], top=2)
    assert one.lse.shape == () and torch.equal(one.top_ids, s.top_ids[0])
    with pytest.raises(ValueError):
        readout.layer_norm(ctx, x.transpose(0, 1))
    with pytest.raises(_abi.PlxError):
        readout.log_probs(ctx, flat, top=41)
    ctx.sync()


# ------------------------------------------------------------------------------- used together
def test_a_student_learns_from_a_teacher_through_the_whole_read_out(ctx):
    """Teacher: norm, projection, best alternatives. Student: norm, projection, distillation and
    back to the hidden layer. Against 64-bit automatic differentiation of the same chain."""
    rows, hidden, units, k = 48, 96, 700, 12
    g = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ht, hs, proj = rand(rows, hidden), rand(rows, hidden), rand(units, hidden) / hidden ** 0.5
    w, b = 1 + 0.1 * rand(hidden), 0.1 * rand(hidden)
    up = torch.full((rows,), 1.0 / rows)
    c = [t.cuda() for t in (ht, hs, proj, w, b, up)]
    old = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        teacher = readout.log_probs(ctx, readout.layer_norm(ctx, c[0], c[3], c[4]) @ c[2].t(), top=k)
        y, mean, rstd = readout.layer_norm(ctx, c[1], c[3], c[4], stats=True)
        logits = y @ c[2].t()
        loss, dl = readout.distill(ctx, logits, teacher.top_ids, teacher.top_logp, kind="log_probs",
                                   weight=c[5])
        dproj = dl.t() @ y
        dx, dw, db = readout.layer_norm_backward(ctx, dl @ c[2], c[1], mean, rstd, c[3])
        ctx.sync()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = old
    HT, HS, PR, W, B = (t.double().requires_grad_() for t in (ht, hs, proj, w, b))
    norm = torch.nn.functional.layer_norm
    t = torch.log_softmax(norm(HT, (hidden,), W, B) @ PR.t(), 1)
    best, ids = t.topk(k, 1)
    assert torch.equal(ids.int().sort(1).values, teacher.top_ids.cpu().sort(1).values)
    best = best.detach()
    s = torch.log_softmax(norm(HS, (hidden,), W, B) @ PR.t(), 1)
    total = ((best.exp() * (best - s.gather(1, ids))).sum(1) / rows).sum()
    DX, DP, DW, DB = torch.autograd.grad(total, (HS, PR, W, B))
    # every value goes through sums of 96, 700 and 96 terms and a dozen other roundings, each
    # of them relative to terms no larger than the largest gradient times ten
    for got, want in ((dx, DX), (dproj, DP), (dw, DW), (db, DB)):
        tol = 10 * U * (hidden + units + hidden + 100) * float(want.abs().max())
        assert float((got.cpu().double() - want).abs().max()) <= tol
    assert abs(float(loss.double().sum()) - float(total.detach())) \
        <= 10 * U * (hidden + units + 100) * max(1.0, float(total.detach()))
