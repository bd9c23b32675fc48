"""The read-out operators on the device where 32 bits are tight or an array ends: rows far from
zero, rows of one value, single values of long rows, results and scratch between guards.

Bounds count the kernels' own roundings (U = 2^-24 each) on the inputs as rounded to their type."""
import numpy as np
import pytest
import torch

import readout_formulas as F
from plastix_b200 import _abi, readout
from test_readout_gpu import HALF_STEP, TINY, TYPES, U, f64, rows_tensor, within

pytestmark = pytest.mark.gpu


def batches(n):
    """Steps of sixteen values or more in which a thread goes over its share of a row: 64 threads
    have fewer than 8,192 values between them, 128 or more take the longer rows."""
    return 8 + n / 2048


def sum_error(n, spread):
    """Relative error of sum exp(d): a value is added within its step (16), over the steps, a
    warp (5), a block (5) and a cluster (8); the sum is moved to a new maximum once a step and
    twelve times while it is joined at most, at 6 U each (2^x to 4 U and a product); 2^x has 4 U, and its
    argument four roundings of its size (`spread`: the mean of |d| under the softmax)."""
    return U * (40 + batches(n) + 6 * (batches(n) + 12) + 4 * spread)


# ------------------------------------------------------------------- gradients far from zero
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [100, 4099, 70000, 300007])
@pytest.mark.parametrize("scale", [1.0, 2.0])
def test_gradient_of_log_probs_far_from_zero(ctx, dtype, n, scale):
    """Rows around large values, and rows of the type's lowest value, have the gradient of the
    same row around zero: no bound below depends on the offset."""
    r = np.random.default_rng(n)
    low = float(torch.finfo(TYPES[dtype]).min)
    a = r.normal(size=(10, n)) * 2.5
    a += np.array([0.0, 25.0, 40.0, 1000.0, -1000.0, 30000.0, -30000.0, 0.0, 0.0, 0.0])[:, None]
    a[7] = low
    a[8] = np.where(np.arange(n) % 3 == 1, low, -np.inf)
    a[9] = -np.inf
    x, _ = rows_tensor(a, dtype)
    target = torch.from_numpy(r.integers(0, n, 10)).int().cuda()
    target[8] = 1
    gl = torch.from_numpy(r.normal(size=10)).float().cuda()
    ge = torch.from_numpy(r.normal(size=10)).float().cuda()
    s = readout.log_probs(ctx, x, target, scale=scale, entropy=True)
    both = readout.log_probs_backward(ctx, x, s.lse, target, gl, s.entropy, ge, scale=scale)
    alone = readout.log_probs_backward(ctx, x, s.lse, target, gl, scale=scale)
    into = x.clone()
    assert readout.log_probs_backward(ctx, into, s.lse, target, gl, scale=scale, out=into) is into
    ctx.sync()
    assert torch.equal(into, alone)
    X, at, GL, GE = f64(x), target.cpu().numpy(), f64(gl), f64(ge)
    # an offset changes nothing, and the lowest value would take log n with it in 64 bits too
    X -= np.where(np.isfinite(X.max(1, keepdims=True)), X.max(1, keepdims=True), 0.0)
    logs, lse = F.log_softmax(X * scale)
    p = np.exp(logs)
    l = np.where(p > 0, np.abs(logs), 0.0)  # noqa: E741
    with np.errstate(invalid="ignore"):
        d = np.where(p > 0, np.abs(scale * X), 0.0)
    ls = np.where(np.isfinite(lse), lse, 0.0)  # log of the sum
    entropy, spread = (p * l).sum(1), (p * d).sum(1)
    e = sum_error(n, spread)
    # log p: the argument and its difference (3 |l| + 2 |d|), the logarithm (2 |ls|), lse rounded below
    # 32 (16), 2^x and the products (12)
    pe = e[:, None] + U * (28 + 3 * l + 2 * d + 2 * ls[:, None])
    # entropy: log s, and sum e d / s whose terms are off by twice what the sum is
    he = (e + 4 * U * ls + spread * (2 * e + 6 * U) + U * entropy)[:, None]
    half = HALF_STEP[dtype]
    for got, ge_ in ((alone, None), (both, GE)):
        want = F.log_probs_backward(X, at, scale, GL, ge_)
        g, h = np.abs(GL)[:, None], 0.0 if ge_ is None else np.abs(GE)[:, None]
        inner = g + h * (l + entropy[:, None])
        err = scale * (p * (pe * (inner + h) + h * he + 6 * U * inner) + 2 * U * g)
        within(f64(got), want, err * (1 + half) + half * np.abs(want) + 2 * TINY[dtype], "gradient")


# --------------------------------------------------------------------- layer norm far from zero
def norm_depth(n):
    """Additions a value goes through: pairs of up to 16 values a thread and two sums' exchange
    over a block, or, in rows too long for registers, n / 1,024 a thread and two steps of 32."""
    return 80 + n / 1024


@pytest.mark.parametrize("n", [3, 100, 513, 1000, 1001, 2049, 4096, 5001, 8190, 16384, 20001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_of_rows_of_one_value(ctx, dtype, n):
    """The mean may be a rounding off, delta <= (depth + 2) U |x|; the deviations, all delta, have a
    mean of their own, which is off by (depth + 2) U of it and is taken away."""
    r = np.random.default_rng(n)
    a = np.repeat(r.uniform(-1000, 1000, (40, 1)), n, 1)
    x, _ = rows_tensor(a, dtype)
    y, mean, rstd = readout.layer_norm(ctx, x, eps=1e-5, stats=True)
    ctx.sync()
    X = f64(x)
    k = (norm_depth(n) + 4) * U
    delta = k * np.abs(X[:, :1])
    root = 1e5 ** 0.5
    within(f64(y), X * 0, np.broadcast_to(1.01 * root * k * delta, X.shape), "y")
    within(f64(mean), X[:, 0], U * np.abs(X[:, 0]) + 2 * k * delta[:, 0], "mean")
    # the variance left is 3 k delta^2 at most; eps in 32 bits, its root and two more roundings
    within(f64(rstd), np.full(40, root), root * (2 * k * delta[:, 0] ** 2 / 1e-5 + 6 * U), "rstd")


@pytest.mark.parametrize("rows, n, dtype", [(50, 1000, "f32"), (50, 1001, "f32"), (30, 4096, "f32"),
                                            (20, 16384, "f32"), (20, 20000, "f32"), (50, 4096, "f16"),
                                            (50, 1001, "f16")])
def test_layer_norm_around_a_large_value(ctx, rows, n, dtype):
    """Deviations of about one around 1e6 (f32) or 1,000 (f16): x - mean is exact there, so only
    the deviations' own mean, variance and products round."""
    r = np.random.default_rng(n)
    x, _ = rows_tensor((1e6 if dtype == "f32" else 1000.0) + 2 * r.normal(size=(rows, n)), dtype)
    y, mean, rstd = readout.layer_norm(ctx, x, eps=1e-5, stats=True)
    ctx.sync()
    X = f64(x)
    Y, M, R = F.layer_norm(X, np.ones(n), np.zeros(n), 1e-5)
    k = norm_depth(n) * U
    delta = (k + 2 * U) * np.abs(M)  # of the first mean
    shift = (k + 3 * U) * (delta + np.abs(X - M[:, None]).mean(1))  # what is left of it
    # variance: sums of squares (deviation^2 + delta^2) to k, less the square of the shift
    rel = (k + 6 * U) * (1 + 2 * (delta * R) ** 2) + 2 * shift * delta * R * R + (shift * R) ** 2
    h = np.abs(Y) + (delta * R)[:, None]
    half = HALF_STEP[dtype]
    tol = (shift * R)[:, None] + h * rel[:, None] + 4 * U * h
    within(f64(y), Y, tol * (1 + half) + half * np.abs(Y) + TINY[dtype], "y")
    within(f64(mean), M, U * np.abs(M) + 2 * shift, "mean")
    within(f64(rstd), R, R * (rel + 4 * U), "rstd")


# ----------------------------------------------------------------------------- the bias' gradient
@pytest.mark.parametrize("rows, n, dtype, btype", [(37, 513, "f32", "f32"), (300, 1024, "bf16", "bf16"),
                                                   (9, 20001, "f16", "f32"), (0, 40, "f32", "f32")])
def test_gradient_of_a_bias_without_a_weight(ctx, rows, n, dtype, btype):
    r = np.random.default_rng(n)
    x, dy = (rows_tensor(r.normal(size=(rows, n)), dtype)[0] for _ in range(2))
    b = torch.from_numpy(r.normal(size=n)).to("cuda", TYPES[btype])
    y, mean, rstd = readout.layer_norm(ctx, x, None, b, stats=True)
    dx, dw, db = readout.layer_norm_backward(ctx, dy, x, mean, rstd, bias=b)
    want = readout.layer_norm_backward(ctx, dy, x, mean, rstd)
    one = torch.ones_like(b)
    full = readout.layer_norm_backward(ctx, dy, x, mean, rstd, one, bias=b)
    ctx.sync()
    assert dw is None and want[1] is None and want[2] is None and torch.equal(dx, want[0])
    assert db.dtype == b.dtype and torch.equal(db, full[2]) and torch.equal(dx, full[0])
    DY = f64(dy)
    half = HALF_STEP[btype]
    tol = (rows + 8) * U * np.abs(DY).sum(0)  # every sum, whatever its order
    within(f64(db), DY.sum(0), tol * (1 + half) + half * np.abs(DY.sum(0)) + TINY[btype], "db")


# -------------------------------------------------------------------------- scratch between guards
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 120, 128, 250, 256, 510, 512, 1000, 1001, 1024, 1030, 2048, 2049, 2050,
                               4096, 4098, 5001, 5120, 8190, 8192, 8193, 9000, 16384, 16392])
def test_layer_norm_backward_keeps_to_its_scratch(ctx, dtype, n):
    for rows in (1, 100, 1300, 20000):
        if rows * n > 1 << 25:
            continue
        x = torch.randn(rows, n, device="cuda").to(TYPES[dtype])
        w = torch.randn(n, device="cuda")
        _, mean, rstd = readout.layer_norm(ctx, x, w, stats=True)
        size = _abi.lib().plx_layer_norm_scratch_bytes(rows, n)
        room = torch.full((size + 8192,), 0x5A, dtype=torch.uint8, device="cuda")
        scratch = room[4096:4096 + size]
        assert scratch.data_ptr() % 16 == 0
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        _abi.call("plx_layer_norm_backward", ctx.handle, rows, n, readout._TYPES[x.dtype], x.data_ptr(), n,
                  x.data_ptr(), n, mean.data_ptr(), rstd.data_ptr(), _abi.F32, w.data_ptr(), dx.data_ptr(), n,
                  dw.data_ptr(), db.data_ptr(), scratch.data_ptr(), size)
        ctx.sync()
        assert (room[:4096] == 0x5A).all() and (room[4096 + size:] == 0x5A).all()
        # every sum of `rows` terms, in whatever order
        want = x.double().sum(0)
        off = (db.double() - want).abs()
        assert bool((off <= (rows + 2) * U * x.double().abs().sum(0)).all())


# ------------------------------------------------------------- every value of a row, every branch
COUNTED = [1, 7, 64, 1000, 4099, 8191, 20011, 32003, 65536, 131072, 131077, 1 << 20]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 8, 400])
def test_no_value_of_a_row_is_left_out(ctx, dtype, rows):
    """n equal values: the sum is n exactly in whatever order (a whole number below 2^24), so lse is
    off by the logarithm's and two more roundings only, far less than one value of a million."""
    for n in COUNTED:
        if rows * n > 1 << 26:
            continue
        for shift in (0, 1, 5):
            room = torch.full((shift + rows * (n + 3) + 8,), 7.0, dtype=TYPES[dtype], device="cuda")
            x = room.as_strided((rows, n), (n + 3, 1), shift).zero_()
            want = np.log(n)
            target = torch.full((rows,), n - 1, dtype=torch.int32, device="cuda")
            got = [readout.log_probs(ctx, x), readout.log_probs(ctx, x, target, entropy=True),
                   readout.log_probs(ctx, x, top=min(3, n)),
                   readout.log_probs(ctx, x, target, entropy=True, top=min(3, n))]
            ids = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
            loss = readout.distill(ctx, x, ids, torch.zeros(rows, 1, device="cuda"))[0]
            ctx.sync()
            # logf: one unit in the last place, two half units at most of its size; two more roundings
            tol = 4 * U * want
            for r in got:
                within(f64(r.lse), np.full(rows, want), tol, "lse")
                if r.entropy is not None:
                    within(f64(r.entropy), np.full(rows, want), tol, "entropy")
                    within(f64(r.logp), np.full(rows, -want), tol, "logp")
            within(f64(loss), np.full(rows, want), tol, "loss")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, n", [(3, 1), (600, 1), (5, 900), (600, 5000), (400, 9000), (600, 20011),
                                     (300, 40000), (7, 50001), (2, 300007)])
def test_entropy_without_alternatives(ctx, rows, n, dtype):
    r = np.random.default_rng(rows + n)
    a = r.normal(size=(rows, n)) * 2.5
    if n > 1:
        a[::3] = np.where(r.random(a[::3].shape) < 0.3, -np.inf, a[::3])
        a[::3, n // 2] = 0.5
        a[-1] = -np.inf
        a[1, 0] = np.nan
    x, _ = rows_tensor(a, dtype)
    target = torch.from_numpy(r.integers(-1, n, rows)).int().cuda()
    got = readout.log_probs(ctx, x, target, scale=0.75, entropy=True)
    ctx.sync()
    assert got.top_ids is None and got.top_logp is None
    X, at = f64(x), target.cpu().numpy()
    want = F.log_probs(X, at, 0.75)
    logs, lse = F.log_softmax(0.75 * X)
    fine = np.isfinite(lse)
    top = np.where(fine, np.where(np.isnan(X), -np.inf, X).max(1), 0.0)
    with np.errstate(invalid="ignore"):
        ls = np.where(fine, lse - 0.75 * top, 0.0)
        p = np.where(fine[:, None], np.exp(logs), 0.0)
        d = np.where(p > 0, np.abs(0.75 * (X - top[:, None])), 0.0)
    spread = (p * d).sum(1)
    e = sum_error(n, spread)
    near = e + 4 * U * np.abs(ls)
    within(f64(got.lse), want["lse"], near + 4 * U * np.abs(np.where(fine, lse, 0)), "lse")
    within(f64(got.entropy), want["entropy"],
           near + spread * (2 * e + 6 * U) + U * np.where(fine, np.abs(want["entropy"]), 0), "entropy")
    x_at = X[np.arange(rows), np.maximum(at, 0)]
    with np.errstate(invalid="ignore"):
        away = np.where(np.isfinite(x_at), np.abs(0.75 * (x_at - top)), 0.0)
    within(f64(got.logp), want["logp"], near + 4 * U * away, "logp")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 40, 150])
def test_alternatives_of_rows_whose_best_values_few_threads_hold(ctx, rows, dtype):
    """In every 16,384 values, 20 threads of 256 hold 1,280 of the best: too many to be ordered at
    once, and fewer threads than alternatives. Odd rows have equals among them."""
    n, top = 131072, 64
    r = np.random.default_rng(rows)
    a = r.normal(size=(rows, n)).clip(-6, 6)
    v = 16 // torch.empty(0, dtype=TYPES[dtype]).element_size()
    at = np.arange(n) // v % 256 < 20
    best = r.uniform(10, 20, (rows, int(at.sum())))
    best[1::2] = np.floor(best[1::2] * 4) / 4
    a[:, at] = best
    x, _ = rows_tensor(a, dtype)
    got = readout.log_probs(ctx, x, top=top)
    ctx.sync()
    np.testing.assert_array_equal(got.top_ids.cpu().numpy(), F.order(f64(x))[:, :top])


# --------------------------------------------------------------------- behind a network's layers
def test_the_read_out_of_a_network_trained_on_log_probability(ctx):
    """One sample through a network's layers, the last without a sigmoid: its output units are the
    logits, the gradient of -log p goes where the layers' backward pass reads, and the weights
    follow. Against automatic differentiation in 64 bits."""
    from plastix_b200.runtime import MlpTopoNet, sweep_forward, sweep_update

    sizes, rate = [5, 24, 37], 0.5
    r = np.random.default_rng(17)
    w = (r.normal(size=5 * 24 + 24 * 37) * 0.4).astype(np.float32)
    x = torch.from_numpy(r.normal(size=5)).float().cuda()
    net = MlpTopoNet(ctx, sizes, w)
    (i0, i1), (h0, h1), (o0, o1) = ((net.begin[k], net.begin[k + 1]) for k in range(3))
    net.act[i0:i1] = x
    sweep_forward(ctx, net.csr[0], net.from_id[0], net.w[0], net.act, net.act[h0:h1], apply=_abi.APPLY_SIGMOID)
    sweep_forward(ctx, net.csr[1], net.from_id[1], net.w[1], net.act, net.act[o0:o1], apply=_abi.APPLY_IDENTITY)
    logits, target = net.act[o0:o1], torch.tensor(11, dtype=torch.int32, device="cuda")
    s = readout.log_probs(ctx, logits, target, top=3)
    down = torch.tensor(-1.0, device="cuda")
    readout.log_probs_backward(ctx, logits, s.lse, target, down, out=net.grad[o0:o1])
    net.bwd[1].refresh_weight(net.w[1])
    net.bwd[1].backward(net.grad, net.grad[h0:h1], net.act[h0:h1], _abi.APPLY_SIGMOID_GRAD)
    for k, (b0, b1) in enumerate(((h0, h1), (o0, o1))):
        sweep_update(ctx, net.csr[k], net.from_id[k], net.act, net.grad[b0:b1], net.w[k], net.w[k],
                     kind=_abi.UPDATE_GRADIENT, rate=rate)
    ctx.sync()
    w1 = torch.from_numpy(w[:120].reshape(24, 5)).double().requires_grad_()
    w2 = torch.from_numpy(w[120:].reshape(37, 24)).double().requires_grad_()
    z = w2 @ torch.sigmoid(w1 @ x.cpu().double())
    z.retain_grad()
    logp = torch.log_softmax(z, 0)
    (-logp[11]).backward()
    # values below 8 go through sums of 5, 24 and 37 terms and some 30 other roundings, forth and back
    tol = 8 * U * 2 * (5 + 24 + 37 + 30)
    assert abs(float(s.logp) - float(logp[11].detach())) <= tol
    assert s.top_ids.tolist() == logp.topk(3).indices.tolist()
    within(f64(net.grad[o0:o1]), z.grad.numpy(), tol, "gradient of the outputs")
    within(f64(net.w[0]), (w1 - rate * w1.grad).detach().numpy().reshape(-1), tol, "weights into the hidden layer")
    within(f64(net.w[1]), (w2 - rate * w2.grad).detach().numpy().reshape(-1), tol, "weights into the outputs")
