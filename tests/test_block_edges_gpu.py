"""The block operators at their edges on the device, against their 64-bit formulas (U = 2^-24)."""
import numpy as np
import pytest
import torch
from scipy.special import erfc

import block_formulas as F
from plastix_b200 import _abi, block
from plastix_b200.runtime import Context
from test_block_gpu import act_error, dense_inputs, gate_bounds, made, product_error, stored, walk
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


# ------------------------------------------------------------------- decays of any size
def placed(a):
    t, v, _ = made(a, "f32")
    return t, v


def decay_inputs(streams, steps, n, kind, at):
    """Streams whose decays' product leaves 32 bits though no h or g does, from step `at` on.
    "grown": decays of 1e5 (or 1.5, over many steps) while h is 0; x begins behind them, dh ends before them.
    "cut": decays of 1e20, 1e20 and 0 on values of 1e-30."""
    g = np.random.default_rng([streams, steps, n, at])
    rows = (streams, steps, n)
    gate = g.uniform(0.3, 0.95, size=rows) * np.where(g.random(rows) < 0.1, -1, 1)
    x, dh = g.normal(size=rows), g.normal(size=rows)
    state, dfinal = g.normal(size=(streams, n)), g.normal(size=(streams, n))
    if kind == "cut":
        gate[:, at - 1], x[:, at - 1], dh[:, at] = 0.0, 1e-30, 1e-30
        gate[:, at], gate[:, at + 1], gate[:, at + 2] = 1e20, 1e20, 0.0
        x[:, at:at + 2], dh[:, at + 1] = 0.0, 0.0
    else:
        value, count = (1e5, 16) if kind == "grown" else (1.5, min(steps - at - 2, 700))
        gate[:, at:at + count] = value
        x[:, :at + count], dh[:, at:] = 0.0, 0.0
        state[:], dfinal[:] = 0.0, 0.0
    flat = (lambda a: placed(a.reshape(-1, n)))
    return flat(x), flat(gate), flat(dh), placed(state), placed(dfinal)


def check_decays(ctx, streams, n, mix, cuts, offsets, inputs, shape):
    """Forwards and backwards against the formulas, as test_block_gpu's check, for 1 - a of either sign."""
    (x, xv), (gate, gv), (dh, dhv), (state, sv), (dfinal, dfv) = inputs
    how = dict(kind="decay", mix=mix, offsets=offsets)
    xs, gates, dhs = (t.view(shape) for t in (x, gate, dh))
    h, final = block.recurrence(ctx, xs, gates, state, **how)
    again = block.recurrence(ctx, xs, gates, state, **how)
    ctx.sync()
    assert torch.equal(h, again[0]) and torch.equal(final, again[1])
    a, keep, e_a, e_keep = gate_bounds(gv, "decay")
    b, e_b = (keep * xv, np.abs(xv) * e_keep + U * np.abs(keep * xv)) if mix else (xv, 0 * xv)
    want, wfinal = F.recurrence(xv, gv, sv, cuts, "decay", mix)
    tol, ftol = walk(a, b, e_a, e_b, sv, cuts, False)
    owned = ~np.isnan(want)
    got = f64(h).reshape(-1, n)
    within(got[owned], want[owned], stored(want, tol, "f32")[owned], "h")
    within(f64(final), wfinal, ftol + U * np.abs(wfinal), "final")
    assert (got[~owned] == 0).all()

    back = dict(x=xs, dfinal=dfinal, **how)
    dx, dgate, dstate = block.recurrence_backward(ctx, dhs, gates, h, state, **back)
    again = block.recurrence_backward(ctx, dhs, gates, h, state, **back)
    ctx.sync()
    for p, q in zip((dx, dgate, dstate), again):
        assert torch.equal(p, q)
    wx, wg, ws = F.recurrence_backward(dhv, xv, gv, got, sv, dfv, cuts, "decay", mix)
    gtol, stol = walk(a, dhv, e_a, 0 * dhv, dfv, cuts, True)
    g = F.recurrence_backward(dhv, xv, gv, got, sv, dfv, cuts, "decay", False)[0]
    before = np.zeros_like(xv)
    for s in range(streams):
        lo, hi = cuts[s], cuts[s + 1]
        if hi > lo:
            before[lo], before[lo + 1:hi] = sv[s], got[lo:hi - 1]
    arm = before - xv if mix else before
    t_dx = np.abs(keep) * gtol + np.abs(g) * e_keep + U * np.abs(wx) if mix else gtol
    t_da = np.abs(arm) * gtol + np.abs(g) * 3 * U * (np.abs(before) + np.abs(xv))
    for name, t, w, off in (("dx", dx, wx, t_dx), ("dgate", dgate, wg, t_da)):
        t = f64(t).reshape(-1, n)
        within(t[owned], w[owned], stored(w, off, "f32")[owned], name)
        assert (t[~owned] == 0).all()
    within(f64(dstate), ws, stol + U * np.abs(ws), "dstate")


DECAYS = [  # streams, steps, n, kind, at
    (5, 24, 40, "grown", 3),     # whole streams in a tile
    (300, 30, 33, "grown", 9),
    (4, 20, 64, "cut", 2),
    (4, 20, 64, "cut", 6),       # over the border of two runs
    (3, 90, 48, "slow", 0),
    (600, 200, 64, "grown", 50),  # walks of several streams
    (3, 500, 4096, "grown", 100),  # a walk a stream
    (2, 700, 31, "grown", 120),  # over the border of two tiles, or in parts
    (1, 5000, 64, "slow", 100),  # in parts
    (1, 5000, 64, "slow", 4200),
    (1, 4000, 37, "slow", 1900),
    (1, 4000, 64, "cut", 126),   # over the border of two parts
    (1, 4000, 64, "cut", 127),
    (1, 4000, 33, "cut", 63),
    (2, 3000, 64, "grown", 120),
    (2, 4000, 1024, "slow", 300),  # in long parts
]


@pytest.mark.parametrize("mix", [False, True])
@pytest.mark.parametrize("streams, steps, n, kind, at", DECAYS)
def test_decays_of_any_size(ctx, streams, steps, n, kind, at, mix):
    cuts = [s * steps for s in range(streams + 1)]
    inputs = decay_inputs(streams, steps, n, kind, at)
    with np.errstate(all="ignore"):
        check_decays(ctx, streams, n, mix, cuts, None, inputs, (streams, steps, n))


@pytest.mark.parametrize("cuts, rows", [([0, 5, 1300, 1300, 3000], 3100), ([4, 900, 2600], 2600),
                                        ([0, 40, 90, 99], 120)])
@pytest.mark.parametrize("n", [64, 33])
def test_decays_of_any_size_in_ragged_streams(ctx, cuts, rows, n):
    """Products that leave 32 bits in every stream that is long enough, and in rows of no stream."""
    g = np.random.default_rng([rows, n])
    gate = g.uniform(0.3, 0.95, size=(rows, n))
    x, dh = g.normal(size=(rows, n)), g.normal(size=(rows, n))
    streams = len(cuts) - 1
    state, dfinal = g.normal(size=(streams, n)), g.normal(size=(streams, n))
    for s in range(streams):
        lo, hi = cuts[s], cuts[s + 1]
        if hi - lo > 30:
            end = lo + 20 + (hi - lo - 30) // 2
            gate[lo + 10:end] = 1e5
            x[lo:end], dh[lo + 10:hi] = 0.0, 0.0
            state[s], dfinal[s] = 0.0, 0.0
    gate[:cuts[0]], gate[cuts[-1]:] = 1e30, 1e30
    inputs = placed(x), placed(gate), placed(dh), placed(state), placed(dfinal)
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    with np.errstate(all="ignore"):
        check_decays(ctx, streams, n, True, cuts, offsets, inputs, (rows, n))


@pytest.mark.parametrize("steps, n, dtype", [(20, 64, "f32"), (300, 64, "f32"), (5000, 64, "bf16"), (5000, 33, "f32"),
                                             (4000, 1024, "bf16")])
@pytest.mark.parametrize("kind", ["decay", "sigmoid"])
def test_infinity_stays_what_it_is_step_by_step(ctx, steps, n, dtype, kind):
    """h behind an infinite x is infinite of its sign until a decay of 0 (which makes NaN of it), not NaN because a
    product of decays is 0 (behind sigmoids it is not finite); other units keep their bits."""
    g = torch.Generator(device="cuda").manual_seed(steps + n)
    x = torch.randn(2, steps, n, device="cuda", generator=g).to(TYPES[dtype])
    gate = (torch.rand(2, steps, n, device="cuda", generator=g) * 0.5 + 0.25).to(TYPES[dtype])
    want, _ = block.recurrence(ctx, x, gate, kind=kind)
    bad = x.clone()
    bad[0, 5, 3], bad[1, 2, 7] = float("inf"), float("-inf")
    bad_gate = gate.clone()
    if kind == "decay":
        bad_gate[1, steps - 4, 7] = 0.0
    h, final = block.recurrence(ctx, bad, bad_gate, kind=kind)
    ctx.sync()
    if kind == "decay":
        assert (h[0, 5:, 3] == float("inf")).all() and final[0, 3] == float("inf")
        assert (h[1, 2:steps - 4, 7] == float("-inf")).all() and h[1, steps - 4:, 7].isnan().all()
    assert not h[0, 5:, 3].isfinite().any() and not h[1, 2:, 7].isfinite().any()
    assert torch.equal(h[0, :5, 3], want[0, :5, 3]) and torch.equal(h[1, :2, 7], want[1, :2, 7])
    others = [u for u in range(n) if u not in (3, 7)]
    assert torch.equal(h[:, :, others], want[:, :, others])
    assert torch.equal(h[1, :, 3], want[1, :, 3]) and torch.equal(h[0, :, 7], want[0, :, 7])


@pytest.mark.parametrize("streams, steps, n, kind, at", [(4, 24, 64, "grown", 3), (2, 3000, 64, "grown", 120),
                                                         (1, 4000, 33, "cut", 63), (2, 4000, 1024, "slow", 300)])
def test_decays_of_any_size_in_place(ctx, streams, steps, n, kind, at):
    """The part that a block goes on into is not written by another one; backwards dx over dh, dgate over gate and
    dstate over dfinal, as the C interface allows."""
    (x, _), (gate, _), (dh, _), (state, _), (dfinal, _) = decay_inputs(streams, steps, n, kind, at)
    shape = (streams, steps, n)
    x, gate, dh = (t.view(shape) for t in (x, gate, dh))
    h, final = block.recurrence(ctx, x, gate, state, kind="decay", mix=True)
    for where in (0, 1):
        t, s = [x.clone(), gate.clone()], state.clone()
        h2, _ = block.recurrence(ctx, *t, s, kind="decay", mix=True, out=t[where], final_out=s)
        ctx.sync()
        assert h.isfinite().all() and torch.equal(h2, h) and torch.equal(s, final)
    want = block.recurrence_backward(ctx, dh, gate, h, state, x=x, dfinal=dfinal, kind="decay", mix=True)
    size = _abi.lib().plx_recurrence_scratch_bytes(streams, streams * steps, n, 0, 0, 1, 1)
    scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
    _abi.call("plx_recurrence_backward", ctx.handle, streams, streams * steps, n, 0, None, dh.data_ptr(), n,
              x.data_ptr(), n, gate.data_ptr(), n, 0, 1, h.data_ptr(), n, state.data_ptr(), dfinal.data_ptr(),
              dh.data_ptr(), n, gate.data_ptr(), n, dfinal.data_ptr(), scratch.data_ptr(), size)
    ctx.sync()
    for a, b in zip((dh, gate, dfinal), want):
        assert torch.equal(a, b)


def test_calls_with_a_flooded_stream_can_be_captured(ctx):
    """What is done where pairs are not finite is decided on the device: a graph that was captured on ordinary values
    gives the eager call's on others."""
    stream = torch.cuda.Stream()
    other = Context(0, stream)
    (x, _), (gate, _), _, (state, _), _ = decay_inputs(2, 3000, 64, "grown", 120)
    x, gate = x.view(2, 3000, 64), gate.view(2, 3000, 64)
    want, wfinal = block.recurrence(ctx, x, gate, state, kind="decay")
    ctx.sync()
    held, held_gate = torch.randn_like(x), torch.full_like(gate, 0.5)
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        h, final = block.recurrence(other, held, held_gate, state, kind="decay")
    graph.replay()
    held.copy_(x)
    held_gate.copy_(gate)
    graph.replay()
    torch.cuda.synchronize()
    other.sync()
    assert torch.equal(h, want) and torch.equal(final, wfinal)


# ------------------------------------------------------------------- float16 gradients
@pytest.mark.parametrize("rows, n, m, more", [(2000, 72, 136, 0), (2000, 33, 70, 1), (7, 300, 130, 8), (1, 40, 9, 0)])
@pytest.mark.parametrize("size", [1e-6, 1e-4, 1.0, 3e4])
@pytest.mark.parametrize("apply", ["tanh", "gelu"])
def test_dense_gradients_of_small_and_large_float16(ctx, rows, n, m, more, size, apply):
    """dz of dy that float16 holds, but whose products with a slope it would not: each is off by half a step of its
    own size and 2^-38 of the largest dy, whatever the gradients' magnitude."""
    g = np.random.default_rng([rows, n, m])
    even = min(1.0, 10 / size)  # keeps sums of large gradients in float16
    x, xv, _ = made((np.abs(g.normal(size=(rows, n))) + 0.5) * even, "f16", n + more)
    w, wv, _ = made(g.normal(size=(m, n)) * even, "f16", n + more)
    dy, dyv, _ = made(np.minimum(np.abs(g.normal(size=(rows, m))) + 0.2, 2.1) * size, "f16", m + more)
    z, zv, _ = made(g.normal(size=(rows, m)) + 1.0, "f32")
    b, _, _ = made(g.normal(size=(1, m)), "f32")
    dx, dw, db = block.dense_backward(ctx, dy, x, w, z, apply=apply, bias=b[0])
    again = block.dense_backward(ctx, dy, x, w, z, apply=apply, bias=b[0])
    ctx.sync()
    for p, q in zip((dx, dw, db), again):
        assert torch.equal(p, q)
    wx, ww, wb, dz = F.dense_backward(dyv, xv, wv, zv, apply)
    slope = F.act(zv, apply)[1]
    off = np.abs(dyv) * (act_error(zv, slope) + 4 * U)
    dzerr = off + HALF_STEP["f16"] * (np.abs(dz) + off) + 2.0 ** -38 * np.abs(dyv).max()
    tx = dzerr @ np.abs(wv) + product_error(dz, wv, m)
    tw = dzerr.T @ np.abs(xv) + product_error(dz.T, xv, rows)
    assert np.abs(wx).max() < 65000 and np.abs(ww).max() < 65000
    within(f64(dx), wx, stored(wx, tx, "f16"), "dx")
    within(f64(dw), ww, stored(ww, tw, "f16"), "dweight")
    within(f64(db), wb, stored(wb, off.sum(0) + (rows + 64) * U * np.abs(dz).sum(0), "f32"), "dbias")


def test_float16_gradients_beside_infinities_and_zeros(ctx):
    """An infinite dy has no part in the others' scale; gradients of 0 are 0."""
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(300, 64, device="cuda", generator=g).half()
    w = torch.randn(80, 64, device="cuda", generator=g).half()
    z = torch.randn(300, 80, device="cuda", generator=g)
    dy = (torch.randn(300, 80, device="cuda", generator=g) * 1e-5).half()
    dy[0, 0] = 0.0
    dx, dw, _ = block.dense_backward(ctx, dy, x, w, z, apply="tanh")
    bad = dy.clone()
    bad[0, 0] = float("inf")
    dx2, dw2, _ = block.dense_backward(ctx, bad, x, w, z, apply="tanh")
    none = block.dense_backward(ctx, torch.zeros_like(dy), x, w, z, apply="tanh")
    ctx.sync()
    assert torch.equal(dx[1:], dx2[1:]) and torch.equal(dw[1:], dw2[1:])
    assert not dx2[0].isfinite().any() and not dw2[0].isfinite().any()
    assert not none[0].any() and not none[1].any()


# ------------------------------------------------------------------- offsets without rows
@pytest.mark.parametrize("cuts", [[0, 5], [0, 0, 3, 3], [-1, 0], [2, 2]])
def test_bad_offsets_are_reported_without_rows(ctx, cuts):
    x = torch.zeros(0, 32, device="cuda")
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    block.recurrence(ctx, x, x, offsets=offsets)
    with pytest.raises(_abi.PlxError, match="offsets"):
        ctx.sync()
    block.recurrence_backward(ctx, x, x, x, offsets=offsets)
    with pytest.raises(_abi.PlxError, match="offsets"):
        ctx.sync()
    state = torch.randn(700, 32, device="cuda")
    none = torch.zeros(701, dtype=torch.int32, device="cuda")
    h, final = block.recurrence(ctx, x, x, state, offsets=none)
    _, _, dstate = block.recurrence_backward(ctx, x, x, h, state, dfinal=final, offsets=none)
    ctx.sync()
    assert torch.equal(final, state) and torch.equal(dstate, state)


# ------------------------------------------------------------------- how exact products are
def pre_of(ctx, a, b):
    """z of rows and weights as they are, in 64 bits."""
    _, z = block.dense(ctx, a, b, pre=True)
    ctx.sync()
    return z.double()


@pytest.mark.parametrize("n", range(1, 9))
@pytest.mark.parametrize("rows", [9, 64, 300])
def test_products_of_32_bit_values_with_all_bits_set(ctx, n, rows):
    """Parts of a value are up to 2^-7 and 2^-15 of it, so that the products that are not made are 8 U of a
    product. The first parts' products are added last: in that step each of n + 1 terms may be cut by 2 U of the
    sum, in the five before by 2^-6 of that; one rounding in registers and one of the result."""
    g = torch.Generator(device="cuda").manual_seed(n)
    a, b = (1 + torch.rand(k, n, device="cuda", generator=g) for k in (rows, 130))
    a, b = ((t.view(torch.int32) | 0x7fff).view(torch.float32) for t in (a, b))
    want = a.double() @ b.double().t()
    tol = (8 + 2 * (n + 1) * (1 + 5 / 64) + 2) * U
    assert ((pre_of(ctx, a, b) - want).abs() <= tol * want).all()


@pytest.mark.parametrize("rows, n, m", [(64, 1001, 130), (300, 1001, 520), (16, 4096, 64), (1000, 2000, 1024)])
def test_sums_of_32_bit_values_leave_the_tensor_cores(ctx, rows, n, m):
    """Terms of one sign. In the tensor cores a step is cut by 2 U of its sum; those of 64 terms alone are made
    there: the four of the first parts with a quarter, two, three and four quarters of it cost 5 U of the 64 terms'
    sum, the others 2^-6 of as much. Those sums are added with roundings of U of the sum so far, half of the whole
    on average. (All steps in the tensor cores: 24 for 64 terms, off by 1e-5, 160 U, at 1,001.)"""
    g = torch.Generator(device="cuda").manual_seed(n)
    a, b = (torch.rand(k, n, device="cuda", generator=g) + 0.1 for k in (rows, m))
    want = a.double() @ b.double().t()
    tol = (8 + 6 + (n // 64 + 1) / 2 + 2) * U
    assert ((pre_of(ctx, a, b) - want).abs() <= tol * want).all()


# ------------------------------------------------------------------- 16-bit activations
@pytest.mark.parametrize("apply", ["sigmoid", "tanh", "silu", "gelu"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_16_bit_activations_within_their_bounds(ctx, dtype, apply):
    """Off by half a step of the value that is stored, besides what the kernel's header states: sigmoids
    (9 + 1.3 |z|) U, tanh 8e-6, GELU's factor 1e-5 where |z| < 10 (a 50th of a float16's half step)."""
    z = np.concatenate([np.linspace(-9.99, 9.99, 60001), np.linspace(-0.1, 0.1, 4001), np.linspace(-85, 10, 4001)])
    z = z[np.abs(z) < 10] if apply == "gelu" else z
    x, xv, _ = made(z[:, None], dtype)
    y = block.dense(ctx, x, torch.ones(1, 1, device="cuda", dtype=TYPES[dtype]), apply=apply)
    ctx.sync()
    # (1 + erf, as the formulas have it, is off by 1e-16: all of GELU's factor below z = -8)
    want = xv * 0.5 * erfc(xv / -np.sqrt(2)) if apply == "gelu" else F.act(xv, apply)[0]
    rel = {"tanh": 8e-6, "gelu": 1e-5}.get(apply, (9 + 1.3 * np.abs(xv)) * U)
    size = np.maximum(np.abs(want) * (1 + rel), 2.0 ** -126)
    half = 2.0 ** (np.floor(np.log2(size)) - (8 if dtype == "bf16" else 11))
    if dtype == "f16":
        half = np.maximum(half, 2.0 ** -25)
    within(f64(y), want, rel * np.abs(want) + half, "y")


# ------------------------------------------------------------------- long sums of 16-bit values
LONG = [  # terms, rows, units, dtype
    (16384, 130, 70, "f16"), (40001, 1100, 1032, "f16"), (200000, 5, 100, "f16"), (140000, 2000, 1400, "f16"),
    (1 << 22, 64, 40, "f16"),  # (kept in one sum by each of eight blocks: 55,000 U)
    (200000, 300, 520, "bf16"), (700001, 20, 300, "bf16"), (270000, 1000, 1032, "bf16")]


@pytest.mark.parametrize("terms, rows, m, dtype", LONG)
def test_long_sums_leave_the_tensor_cores(ctx, terms, rows, m, dtype):
    """Terms of one sign. 16 of them are a step there, in which each and the sum so far, half of the whole on average,
    may be cut by 2 U of that sum; sums of 16,384 (131,072) are added by roundings of U at most."""
    g = torch.Generator(device="cuda").manual_seed(terms)
    a, b = ((torch.rand(k, terms, device="cuda", generator=g) + 0.1).to(TYPES[dtype]) for k in (rows, m))
    got = pre_of(ctx, a, b)
    want = torch.zeros_like(got)
    for k in range(0, terms, 65536):
        want += a[:, k:k + 65536].double() @ b[:, k:k + 65536].double().t()
    most = 16384 if dtype == "f16" else 131072
    tol = (17 * min(terms, most) / 16 + terms // most + 2) * U
    assert ((got - want).abs() <= tol * want).all()
    dy = (a * 2.0 ** -8).t().contiguous()  # [terms, rows]: dweight = sums over the terms
    x = b.t().contiguous()
    weight = torch.zeros(rows, m, device="cuda", dtype=TYPES[dtype])
    _, dw, _ = block.dense_backward(ctx, dy, x, weight, input_grad=False)
    ctx.sync()
    want = want * 2.0 ** -8
    assert want.max() < 65000
    assert ((dw.double() - want).abs() <= (tol + HALF_STEP[dtype] * (1 + tol)) * want).all()


@pytest.mark.parametrize("rows, m", [(1100, 1032), (700, 100), (40, 300), (300, 70)])
def test_long_sums_with_all_that_follows_them(ctx, rows, m):
    """Bias, activation, residual and z of float16 rows of 17,000 inputs."""
    (x, xv), (w, wv), (b, bv), (res, resv), _ = dense_inputs(rows, 17000, m, "f16", 0, 0, "f32")
    y, z = block.dense(ctx, x, w, b, apply="gelu", residual=res, pre=True)
    only = block.dense(ctx, x, w, b, apply="gelu", residual=res)
    ctx.sync()
    want, wz = F.dense(xv, wv, bv, "gelu", resv)
    ztol = product_error(xv, wv.T, 17000) + 4 * U * (np.abs(wz) + np.abs(bv))
    within(f64(z), wz, ztol, "z")
    a = F.act(wz, "gelu")[0]
    within(f64(y), want, stored(want, 1.2 * ztol + act_error(wz, a) + U * np.abs(want), "f16"), "y")
    assert torch.equal(y, only)
