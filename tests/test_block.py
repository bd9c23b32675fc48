"""Refusals of the block operators (no GPU needed), and their 64-bit formulas against differences."""
import ctypes

import numpy as np
import pytest
import torch

import block_formulas as F
from plastix_b200 import _abi, block
from test_readout import CTX, DIFF, ODD, FakeContext, P, differences, refused

BIG = 1 << 24
DENSE = dict(ctx=CTX, rows=4, n=8, m=6, dtype=0, x=P, ldx=8, w=P, ldw=8, pdtype=0, bias=P, act=1, res=P, ldr=6, y=P,
             ldy=6, pre=P, scratch=P, size=BIG)
DENSE_BWD = dict(ctx=CTX, rows=4, n=8, m=6, dtype=0, dy=P, lddy=6, x=P, ldx=8, w=P, ldw=8, act=1, pre=P, dx=P, lddx=8,
                 dw=P, lddw=8, pdtype=0, db=P, scratch=P, size=BIG)
RECUR = dict(ctx=CTX, streams=2, rows=400, n=8, dtype=0, offsets=P, x=P, ldx=8, gate=P, ldg=8, kind=1, mix=1, state=P,
             h=P, ldh=8, final=P, scratch=P, size=BIG)
RECUR_BWD = dict(ctx=CTX, streams=2, rows=400, n=8, dtype=0, offsets=P, dh=P, lddh=8, x=P, ldx=8, gate=P, ldg=8, kind=1,
                 mix=1, h=P, ldh=8, state=P, dfinal=P, dx=P, lddx=8, dgate=P, lddg=8, dstate=P, scratch=P, size=BIG)
Q = ctypes.c_void_p(0x4000)


def params(**change):
    v = dict(kind=0, post=1, gate=2, gate_sigmoid=0, param_dtype=0, scale=1.0, eps=1e-5, gate_values=0x2000, ldg=8,
             post_weight=0x2000, post_bias=0x2000, pre_weight=0x2000, pre_bias=0x2000)
    return ctypes.byref(_abi.BlockNormParams(**{**v, **change}))


def block_args(**change):
    v = dict(ctx=CTX, rows=4, n=8, dtype=0, x=P, ldx=8, o=P, ldo=8, params=params(), r=P, ldr=8, u=Q, ldu=8, stats=P)
    return {**v, **change}.values()


def block_bwd_args(**change):
    v = dict(ctx=CTX, rows=4, n=8, dtype=0, dr=P, lddr=8, du=P, lddu=8, x=P, ldx=8, o=P, ldo=8, stats=P, params=params(),
             dx=P, lddx=8, do=Q, lddo=8, dgate=ctypes.c_void_p(0x6000), lddg=8, dw1=P, db1=P, dw2=P, db2=P, scratch=P,
             size=BIG)
    return {**v, **change}.values()


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=3), 1, b"dtype"), (dict(n=0), 1, b"n = 0"), (dict(m=0), 1, b"m = 0"),
    (dict(n=1 << 31), 1, b"out of range"), (dict(m=1 << 31), 1, b"out of range"),
    (dict(rows=1 << 31), 3, b"fewer than 2^31"), (dict(pdtype=1), 1, b"param_dtype"), (dict(act=6), 1, b"act 6"),
    (dict(act=-1), 1, b"act -1"), (dict(x=None), 1, b"required"), (dict(w=None), 1, b"required"),
    (dict(y=None), 1, b"required"), (dict(ldx=7), 1, b"stride"), (dict(ldw=7), 1, b"ldw"), (dict(ldr=5), 1, b"stride"),
    (dict(ldy=5), 1, b"stride"), (dict(scratch=ctypes.c_void_p(0x2008)), 1, b"16-byte")])
def test_dense_refuses(change, code, text):
    refused(code, text, "plx_dense", *{**DENSE, **change}.values())


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=3), 1, b"dtype"), (dict(act=9), 1, b"act"), (dict(dy=None), 1, b"dy"),
    (dict(x=None), 1, b"needs x"), (dict(w=None), 1, b"needs weight"), (dict(pre=None), 1, b"pre is required"),
    (dict(lddy=5), 1, b"stride"), (dict(ldx=7), 1, b"stride"), (dict(lddx=7), 1, b"stride"), (dict(ldw=7), 1, b"stride"),
    (dict(lddw=7), 1, b"stride"), (dict(scratch=None), 1, b"scratch"), (dict(size=8), 1, b"scratch"),
    (dict(scratch=ctypes.c_void_p(0x2008)), 1, b"16-byte"), (dict(rows=1 << 31), 3, b"fewer than 2^31")])
def test_dense_backward_refuses(change, code, text):
    refused(code, text, "plx_dense_backward", *{**DENSE_BWD, **change}.values())


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(params=None), 1, b"params"), (dict(dtype=3), 1, b"dtype"),
    (dict(n=0), 1, b"n = 0"), (dict(rows=1 << 31), 3, b"fewer than 2^31"), (dict(params=params(kind=2)), 1, b"kind"),
    (dict(params=params(gate=3)), 1, b"gate"), (dict(params=params(param_dtype=1)), 1, b"param_dtype"),
    (dict(params=params(scale=float("nan"))), 1, b"scale"), (dict(params=params(scale=float("inf"))), 1, b"scale"),
    (dict(params=params(eps=-1.0)), 1, b"eps"), (dict(params=params(eps=float("nan"))), 1, b"eps"),
    (dict(params=params(gate_values=None)), 1, b"gate_values"), (dict(params=params(ldg=7)), 1, b"stride"),
    (dict(params=params(pre_bias=0x2002)), 1, b"not aligned"), (dict(params=params(gate_values=0x2002)), 1, b"not aligned"),
    (dict(x=None), 1, b"required"), (dict(o=None), 1, b"required"), (dict(r=None), 1, b"required"),
    (dict(u=None), 1, b"required"), (dict(u=P), 1, b"same array"), (dict(ldx=7), 1, b"stride"), (dict(ldu=7), 1, b"stride"),
    (dict(stats=ctypes.c_void_p(0x2008)), 1, b"16-byte")])
def test_block_norm_refuses(change, code, text):
    refused(code, text, "plx_block_norm", *block_args(**change))


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(params=None), 1, b"params"), (dict(dr=None, du=None), 1, b"dr or du"),
    (dict(x=None), 1, b"required"), (dict(stats=None), 1, b"required"), (dict(dx=None), 1, b"required"),
    (dict(do=P), 1, b"same array"), (dict(dgate=P), 1, b"same array"), (dict(lddr=7), 1, b"stride"),
    (dict(lddu=7), 1, b"stride"), (dict(lddo=7), 1, b"stride"), (dict(lddg=7), 1, b"stride"),
    (dict(scratch=None), 1, b"scratch"), (dict(size=8), 1, b"scratch"),
    (dict(stats=ctypes.c_void_p(0x2008)), 1, b"16-byte")])
def test_block_norm_backward_refuses(change, code, text):
    refused(code, text, "plx_block_norm_backward", *block_bwd_args(**change))


@pytest.mark.parametrize("name, args", [("plx_recurrence", RECUR), ("plx_recurrence_backward", RECUR_BWD)])
@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=3), 1, b"dtype"), (dict(kind=2), 1, b"gate_kind"), (dict(n=0), 1, b"n = 0"),
    (dict(streams=1 << 31), 1, b"fewer than 2^31"), (dict(rows=1 << 31), 3, b"fewer than 2^31"),
    (dict(streams=0), 1, b"of no stream"), (dict(offsets=None, streams=3), 1, b"same number of steps"),
    (dict(gate=None), 1, b"required"), (dict(x=None), 1, b"required"), (dict(h=None), 1, b"required"),
    (dict(ldx=7), 1, b"stride"), (dict(ldg=7), 1, b"stride"), (dict(ldh=7), 1, b"stride"),
    (dict(scratch=None), 1, b"scratch"), (dict(size=64), 1, b"scratch"),
    (dict(scratch=ctypes.c_void_p(0x2008)), 1, b"16-byte")])
def test_recurrence_refuses(name, args, change, code, text):
    refused(code, text, name, *{**args, **change}.values())


@pytest.mark.parametrize("name, args, arrays", [
    ("plx_dense", DENSE, "x w bias res y pre"), ("plx_dense_backward", DENSE_BWD, "dy x w pre dx dw db"),
    ("plx_recurrence", RECUR, "offsets x gate state h final"),
    ("plx_recurrence_backward", RECUR_BWD, "offsets dh x gate h state dfinal dx dgate dstate")])
def test_arrays_off_their_elements_are_refused(name, args, arrays):
    for a in arrays.split():
        refused(1, b"not aligned", name, *{**args, a: ODD}.values())


def test_no_rows_are_no_work():
    lib = _abi.lib()
    assert lib.plx_dense(*{**DENSE, "rows": 0, "x": None}.values()) == 0
    assert lib.plx_block_norm(*block_args(rows=0, x=None)) == 0
    assert lib.plx_recurrence(*{**RECUR, "streams": 0, "rows": 0, "x": None}.values()) == 0
    assert lib.plx_recurrence_backward(*{**RECUR_BWD, "streams": 0, "rows": 0, "x": None}.values()) == 0


def test_python_layer_refuses():
    c, x, w = FakeContext(), torch.zeros(4, 8), torch.zeros(6, 8)
    dy, i32 = torch.zeros(4, 6), torch.zeros(3, dtype=torch.int32)
    st = torch.zeros(4, 4)
    bad = [
        lambda: block.dense(c, x.double(), w.double()),
        lambda: block.dense(c, x, w.bfloat16()),
        lambda: block.dense(c, x, torch.zeros(6, 7)),
        lambda: block.dense(c, x, torch.zeros(0, 8)),
        lambda: block.dense(c, x, torch.zeros(8)),
        lambda: block.dense(c, x, torch.zeros(8, 6).t()),
        lambda: block.dense(c, x, w, apply="softmax"),
        lambda: block.dense(c, x, w, torch.zeros(8)),
        lambda: block.dense(c, x, w, torch.zeros(6).bfloat16()),
        lambda: block.dense(c, x, w, residual=x),
        lambda: block.dense(c, x, w, residual=dy.bfloat16()),
        lambda: block.dense(c, x, w, out=x),
        lambda: block.dense(c, x, torch.zeros(8, 8), out=x),
        lambda: block.dense(c, x, torch.zeros(8, 8), residual=torch.zeros(4, 8), out=x),
        lambda: block.dense_backward(c, x, x, w),
        lambda: block.dense_backward(c, dy, x, w, apply="silu"),
        lambda: block.dense_backward(c, dy, x, w, dy.bfloat16(), apply="silu"),
        lambda: block.dense_backward(c, dy, x, w, torch.zeros(6, 4).t(), apply="silu"),
        lambda: block.dense_backward(c, dy, x, w, bias=torch.zeros(8)),
        lambda: block.block_norm(c, x, dy),
        lambda: block.block_norm(c, x, x.bfloat16()),
        lambda: block.block_norm(c, x, x, torch.zeros(7)),
        lambda: block.block_norm(c, x, x, dy),
        lambda: block.block_norm(c, x, x, x[:1].expand(4, 8)),
        lambda: block.block_norm(c, x, x, kind="group"),
        lambda: block.block_norm(c, x, x, gate_apply="tanh"),
        lambda: block.block_norm(c, x, x, post=False, post_weight=torch.zeros(8)),
        lambda: block.block_norm(c, x.bfloat16(), x.bfloat16(), torch.zeros(8).bfloat16(), pre_weight=torch.zeros(8)),
        lambda: block.block_norm(c, x, x, pre_bias=torch.zeros(4)),
        lambda: block.block_norm(c, x, torch.zeros(4, 8), torch.zeros(4, 8)[1:], out=x),
        lambda: block.block_norm_backward(c, None, None, x, x, st),
        lambda: block.block_norm_backward(c, x, dy, x, x, st),
        lambda: block.block_norm_backward(c, x, x, x, x, torch.zeros(4, 2)),
        lambda: block.recurrence(c, x, dy),
        lambda: block.recurrence(c, x, x, kind="tanh"),
        lambda: block.recurrence(c, x, x, torch.zeros(2, 8)),
        lambda: block.recurrence(c, x, x, torch.zeros(1, 8).bfloat16()),
        lambda: block.recurrence(c, x[0], x[0]),
        lambda: block.recurrence(c, torch.zeros(2, 2, 2, 8), torch.zeros(2, 2, 2, 8)),
        lambda: block.recurrence(c, x, x, offsets=i32.long()),
        lambda: block.recurrence(c, x, x, offsets=i32[:0]),
        lambda: block.recurrence(c, x[None], x[None], offsets=i32),
        lambda: block.recurrence(c, x, x, torch.zeros(1, 8), offsets=i32),
        lambda: block.recurrence(c, torch.zeros(5, 8)[:4], torch.zeros(4, 8), out=torch.zeros(4, 9)[:, :8].bfloat16()),
        lambda: block.recurrence_backward(c, x, x, dy),
        lambda: block.recurrence_backward(c, x, x, x, mix=True),
        lambda: block.recurrence_backward(c, x, x, x, x=dy),
        lambda: block.recurrence_backward(c, x, x, x, dfinal=torch.zeros(3, 8)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")
    other = FakeContext()
    other.device = torch.device("cuda", 0)
    for call in (lambda: block.dense(other, x, w), lambda: block.block_norm(other, x, x),
                 lambda: block.recurrence(other, x, x)):
        with pytest.raises(ValueError, match="on cpu"):
            call()


def test_states_that_overlap_rows_are_refused():
    c = FakeContext()
    flat = torch.zeros(64)
    rows, x = flat[:32].view(4, 8), torch.zeros(4, 8)
    for state in (flat[:8].view(1, 8), flat[24:32].view(1, 8)):
        for call in (lambda: block.recurrence(c, x, x, state, out=rows),
                     lambda: block.recurrence(c, x, x, out=rows, final_out=state),
                     lambda: block.recurrence(c, rows, x, final_out=state),
                     lambda: block.recurrence(c, x, rows, state, final_out=state)):
            with pytest.raises(ValueError, match="overlaps"):
                call()


def test_results_that_overlap_other_inputs_are_refused():
    c = FakeContext()
    both = torch.zeros(9, 8)
    with pytest.raises(ValueError, match="overlaps"):
        block.recurrence(c, both[:4], both[2:6], out=both[2:6])
    with pytest.raises(ValueError, match="overlaps"):
        block.recurrence(c, both[:4], both[4:8], out=both[1:5])
    state = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="overlaps"):
        block.recurrence(c, torch.zeros(2, 4, 8), torch.zeros(2, 4, 8), state[:2], final_out=state[1:])
    with pytest.raises(ValueError, match="overlaps"):
        block.block_norm(c, both[:4], both[2:6], out=both[2:6])
    with pytest.raises(ValueError, match="overlaps"):
        block.dense(c, torch.zeros(4, 8), both[:8], out=both[5:9])


# ---- the formulas against differences, in 64 bits --------------------------------------------
@pytest.mark.parametrize("apply", ["identity", "sigmoid", "tanh", "silu", "gelu", "relu"])
def test_dense_formula(apply):
    r = np.random.default_rng(1)
    x, w, b, dy = r.normal(size=(3, 4)), r.normal(size=(5, 4)), r.normal(size=5), r.normal(size=(3, 5))
    z = F.dense(x, w, b, apply)[1]
    assert np.abs(z).min() > 1e-3  # no kink of relu within the differences
    dx, dw, db, _ = F.dense_backward(dy, x, w, z, apply)
    of = lambda x, w, b: float((F.dense(x, w, b, apply)[0] * dy).sum())  # noqa: E731
    np.testing.assert_allclose(dx, differences(lambda v: of(v, w, b), x), atol=DIFF)
    np.testing.assert_allclose(dw, differences(lambda v: of(x, v, b), w), atol=DIFF)
    np.testing.assert_allclose(db, differences(lambda v: of(x, w, v), b), atol=DIFF)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("gate_apply", ["identity", "sigmoid"])
@pytest.mark.parametrize("units", [True, False])
def test_block_norm_formula(kind, post, gate_apply, units):
    r = np.random.default_rng(2)
    x, o, dr, du = (r.normal(size=(3, 5)) for _ in range(4))
    v = {"gate": r.normal(size=5 if units else (3, 5)), "post_weight": r.normal(size=5), "post_bias": r.normal(size=5),
         "pre_weight": r.normal(size=5), "pre_bias": r.normal(size=5)}
    if not post:
        v["post_weight"] = v["post_bias"] = None

    def of(x, o, v):
        rr, u, _ = F.block_norm(x, o, kind=kind, post=post, scale=0.7, gate_apply=gate_apply, **v)
        return float((rr * dr + u * du).sum())

    k = F.block_norm(x, o, kind=kind, post=post, scale=0.7, gate_apply=gate_apply, **v)[2]
    got = F.block_norm_backward(dr, du, k, kind=kind, post=post, scale=0.7, gate_units=units,
                                post_weight=v["post_weight"], pre_weight=v["pre_weight"])
    np.testing.assert_allclose(got["dx"], differences(lambda t: of(t, o, v), x), atol=DIFF)
    np.testing.assert_allclose(got["do"], differences(lambda t: of(x, t, v), o), atol=DIFF)
    for name, value in v.items():
        if value is not None:
            np.testing.assert_allclose(got["d" + name], differences(lambda t: of(x, o, {**v, name: t}), value), atol=DIFF)


@pytest.mark.parametrize("kind", ["sigmoid", "decay"])
@pytest.mark.parametrize("mix", [True, False])
def test_recurrence_formula(kind, mix):
    r = np.random.default_rng(3)
    cuts, rows = [1, 4, 4, 9], 10
    x, gate, dh = r.normal(size=(rows, 3)), r.uniform(0.2, 0.9, size=(rows, 3)), r.normal(size=(rows, 3))
    state, dfinal = r.normal(size=(3, 3)), r.normal(size=(3, 3))

    def of(x, gate, state):
        h, final = F.recurrence(x, gate, state, cuts, kind, mix)
        return float(np.nansum(h * dh) + (final * dfinal).sum())

    h = F.recurrence(x, gate, state, cuts, kind, mix)[0]
    dx, dgate, dstate = F.recurrence_backward(dh, x, gate, h, state, dfinal, cuts, kind, mix)
    np.testing.assert_allclose(np.nan_to_num(dx), differences(lambda t: of(t, gate, state), x), atol=DIFF)
    np.testing.assert_allclose(np.nan_to_num(dgate), differences(lambda t: of(x, t, state), gate), atol=DIFF)
    np.testing.assert_allclose(dstate, differences(lambda t: of(x, gate, t), state), atol=DIFF)
