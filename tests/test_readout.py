"""Refusals of the read-out operators: bad arguments end in a status or a
ValueError before any device work (no GPU needed), and the 64-bit formulas that
the GPU tests compare with agree with differences."""
import ctypes

import numpy as np
import pytest
import torch

import readout_formulas as F
from plastix_b200 import _abi, readout

CTX = ctypes.c_void_p(0x1000)  # never dereferenced: every call here is refused first
P = ctypes.c_void_p(0x2000)


def refused(code, text, name, *args):
    lib = _abi.lib()
    assert getattr(lib, name)(*args) == code
    assert text in lib.plx_last_error(), lib.plx_last_error()


NORM = dict(ctx=CTX, rows=4, n=8, dtype=0, x=P, ldx=8, pdtype=0, w=P, b=P, eps=1e-5, y=P, ldy=8,
            mean=P, rstd=P)
NORM_BWD = dict(ctx=CTX, rows=4, n=8, dtype=0, dy=P, lddy=8, x=P, ldx=8, mean=P, rstd=P, pdtype=0,
                w=P, dx=P, lddx=8, dw=P, db=P, scratch=P, size=1 << 20)
SCORE = dict(ctx=CTX, rows=4, n=8, dtype=0, x=P, ld=8, target=P, scale=1.0, top=2, logp=P, lse=P,
             entropy=P, ids=P, best=P)
SCORE_BWD = dict(ctx=CTX, rows=4, n=8, dtype=0, x=P, ld=8, target=P, scale=1.0, lse=P, entropy=P,
                 gl=P, ge=P, dx=P, ldd=8)
DISTILL = dict(ctx=CTX, rows=4, n=8, dtype=0, x=P, ld=8, k=3, ids=P, values=P, kind=0, tau=1.0,
               w=P, loss=P, dx=P, ldd=8)


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=3), 1, b"dtype"), (dict(dtype=-1), 1, b"dtype"),
    (dict(n=0), 1, b"n = 0"), (dict(n=1 << 31), 1, b"out of range"),
    (dict(rows=1 << 31), 3, b"fewer than 2^31"), (dict(pdtype=1), 1, b"param_dtype"),
    (dict(eps=-1.0), 1, b"eps"), (dict(eps=float("nan")), 1, b"eps"), (dict(x=None), 1, b"x and y"),
    (dict(y=None), 1, b"x and y"), (dict(ldx=7), 1, b"ldx"), (dict(ldy=7), 1, b"ldy")])
def test_layer_norm_refuses(change, code, text):
    refused(code, text, "plx_layer_norm", *{**NORM, **change}.values())


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=7), 1, b"dtype"), (dict(n=0), 1, b"n = 0"),
    (dict(rows=1 << 31), 3, b"fewer than 2^31"), (dict(pdtype=2), 1, b"param_dtype"),
    (dict(dy=None), 1, b"required"), (dict(mean=None), 1, b"required"),
    (dict(scratch=None), 1, b"scratch"), (dict(size=8), 1, b"scratch"),
    (dict(scratch=ctypes.c_void_p(0x2008)), 1, b"16-byte"), (dict(lddx=7), 1, b"stride"),
    (dict(lddy=7), 1, b"stride"), (dict(ldx=7), 1, b"stride")])
def test_layer_norm_backward_refuses(change, code, text):
    refused(code, text, "plx_layer_norm_backward", *{**NORM_BWD, **change}.values())


@pytest.mark.parametrize("rows", [600, 100_000])
@pytest.mark.parametrize("n", [16_385, 65_536, 1_000_003])
def test_layer_norm_scratch_of_long_rows_is_less_than_600_rows(rows, n):
    """Column sums of many long rows take a fraction of what 600 of them take."""
    size = _abi.lib().plx_layer_norm_scratch_bytes(rows, n)
    assert 2 * 4 * n <= size < 600 * n * 2


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=3), 1, b"dtype"), (dict(n=0), 1, b"n = 0"),
    (dict(rows=1 << 31), 3, b"fewer than 2^31"), (dict(x=None), 1, b"logits"),
    (dict(ld=7), 1, b"stride"), (dict(scale=0.0), 1, b"scale"), (dict(scale=-1.0), 1, b"scale"),
    (dict(scale=float("inf")), 1, b"scale"), (dict(scale=float("nan")), 1, b"scale"),
    (dict(top=9), 1, b"exceeds"), (dict(n=100, ld=100, top=65), 3, b"at most 64"),
    (dict(lse=None), 1, b"lse"), (dict(target=None), 1, b"go together"),
    (dict(logp=None), 1, b"go together"), (dict(ids=None), 1, b"top_ids"),
    (dict(best=None), 1, b"top_ids")])
def test_log_probs_refuses(change, code, text):
    refused(code, text, "plx_log_probs", *{**SCORE, **change}.values())


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=3), 1, b"dtype"), (dict(scale=0.0), 1, b"scale"),
    (dict(gl=None, ge=None), 1, b"grad_logp or"), (dict(target=None), 1, b"needs target"),
    (dict(entropy=None), 1, b"needs entropy"), (dict(lse=None), 1, b"lse"),
    (dict(dx=None), 1, b"dlogits"), (dict(ldd=7), 1, b"stride"), (dict(ld=7), 1, b"stride")])
def test_log_probs_backward_refuses(change, code, text):
    refused(code, text, "plx_log_probs_backward", *{**SCORE_BWD, **change}.values())


@pytest.mark.parametrize("change, code, text", [
    (dict(ctx=None), 1, b"ctx"), (dict(dtype=3), 1, b"dtype"), (dict(tau=0.0), 1, b"temperature"),
    (dict(tau=float("nan")), 1, b"temperature"), (dict(tau=1e-39), 1, b"too small"),
    (dict(kind=2), 1, b"teacher_kind"), (dict(k=0), 1, b"positive"), (dict(k=65), 3, b"at most 64"),
    (dict(ids=None), 1, b"required"), (dict(values=None), 1, b"required"),
    (dict(loss=None), 1, b"required"), (dict(ldd=7), 1, b"stride"), (dict(ld=7), 1, b"stride"),
    (dict(rows=1 << 31), 3, b"fewer than 2^31")])
def test_distill_refuses(change, code, text):
    refused(code, text, "plx_distill", *{**DISTILL, **change}.values())


ODD = ctypes.c_void_p(0x2002)  # aligned to 16-bit values, not to 32-bit ones


@pytest.mark.parametrize("name, args, arrays", [
    ("plx_layer_norm", NORM, "x y w b mean rstd"),
    ("plx_layer_norm_backward", NORM_BWD, "dy x mean rstd w dx dw db"),
    ("plx_log_probs", SCORE, "x target logp lse entropy ids best"),
    ("plx_log_probs_backward", SCORE_BWD, "x target lse entropy gl ge dx"),
    ("plx_distill", DISTILL, "x ids values w loss dx")])
def test_arrays_off_their_elements_are_refused(name, args, arrays):
    for a in arrays.split():
        refused(1, b"not aligned", name, *{**args, a: ODD}.values())
    refused(1, b"not aligned", name, *{**args, "dtype": 1, "x": ctypes.c_void_p(0x2001)}.values())


def test_no_rows_are_no_work():
    lib = _abi.lib()
    assert lib.plx_layer_norm(*{**NORM, "rows": 0, "x": None, "y": None}.values()) == 0
    assert lib.plx_log_probs(*{**SCORE, "rows": 0, "x": None}.values()) == 0
    assert lib.plx_log_probs_backward(*{**SCORE_BWD, "rows": 0, "x": None}.values()) == 0
    assert lib.plx_distill(*{**DISTILL, "rows": 0, "x": None}.values()) == 0


class FakeContext:
    """A context on the CPU: every call here is refused before its handle counts."""
    device = torch.device("cpu")
    handle = None


def test_python_layer_refuses():
    c, x = FakeContext(), torch.zeros(4, 8)
    bad = [
        lambda: readout.layer_norm(c, x.to(torch.float64)),
        lambda: readout.layer_norm(c, torch.zeros(4, 0)),
        lambda: readout.layer_norm(c, torch.tensor(1.0)),
        lambda: readout.layer_norm(c, x.t()),
        lambda: readout.layer_norm(c, x[:1].expand(4, 8)),
        lambda: readout.layer_norm(c, torch.zeros(3, 4, 2, 8)[:, :, 0].transpose(0, 1)),
        lambda: readout.layer_norm(c, x, torch.zeros(7)),
        lambda: readout.layer_norm(c, x, torch.zeros(8, dtype=torch.bfloat16)),
        lambda: readout.layer_norm(c, x.bfloat16(), torch.zeros(8), torch.zeros(8).bfloat16()),
        lambda: readout.layer_norm_backward(c, x[:3], x, torch.zeros(4), torch.zeros(4)),
        lambda: readout.layer_norm_backward(c, x, x, torch.zeros(3), torch.zeros(4)),
        lambda: readout.layer_norm_backward(c, x, x, torch.zeros(4), torch.zeros(4).double()),
        lambda: readout.log_probs(c, x, torch.zeros(4, dtype=torch.int64)),
        lambda: readout.log_probs(c, x, torch.zeros(3, dtype=torch.int32)),
        lambda: readout.log_probs_backward(c, x, torch.zeros(4)),
        lambda: readout.log_probs_backward(c, x, torch.zeros(4), None, torch.zeros(4)),
        lambda: readout.log_probs_backward(c, x, torch.zeros(4), grad_entropy=torch.zeros(4)),
        lambda: readout.distill(c, x, torch.zeros(4, 2).int(), torch.zeros(4, 3)),
        lambda: readout.distill(c, x, torch.zeros(4, 2).int(), torch.zeros(4, 2), kind="soft"),
        lambda: readout.distill(c, x, torch.zeros(4, 2).int(), torch.zeros(4, 2).half()),
        lambda: readout.distill(c, x, torch.zeros(4, 2).int(), torch.zeros(4, 2),
                                weight=torch.zeros(4, 1)),
        lambda: readout.distill(c, x, torch.zeros(4, 2).int(), torch.zeros(4, 2), grad=False,
                                out=x),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    other = FakeContext()
    other.device = torch.device("cuda", 0)
    with pytest.raises(ValueError, match="on cpu"):
        readout.layer_norm(other, x)


def test_result_of_a_call_is_new_or_the_input_itself():
    c, x = FakeContext(), torch.zeros(8, 8)
    assert readout._result(c, x, x, 8, "out") == (x, 8)
    for other in (x[1:5], x[0:8:2]):
        with pytest.raises(ValueError, match="overlaps"):
            readout._result(c, other, x[0:4], 8, "out")
    readout._result(c, x[4:], x[:4], 8, "out")
    readout._result(c, x[:, 4:], x[:, :4], 8, "out")  # side by side
    readout._result(c, x[:, :4], x[:, 4:], 8, "out")
    with pytest.raises(ValueError, match="overlaps"):
        readout._result(c, x[:, 3:7], x[:, :4], 8, "out")
    with pytest.raises(ValueError):
        readout._result(c, x[:4].bfloat16(), x[:4], 8, "out")


# ---- the formulas against differences, in 64 bits --------------------------------------------
def differences(f, x, h=1e-5):
    out = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[i] += h
        b[i] -= h
        out[i] = (f(a) - f(b)) / (2 * h)
    return out


# Central differences are off by h^2/6 times the third derivative (below 1e-8 for these functions,
# whose derivatives are of order one) and by rounding of f (|f| < 100) over h: 100 * 2^-53 / 1e-5 < 2e-9.
DIFF = 1e-7


def test_formulas_agree_with_differences():
    r = np.random.default_rng(3)
    x, dy, w, b = r.normal(size=(3, 7)), r.normal(size=(3, 7)), r.normal(size=7), r.normal(size=7)
    y, mean, rstd = F.layer_norm(x, w, b, 1e-5)
    dx, dw, db = F.layer_norm_backward(dy, x, mean, rstd, w)
    of = lambda x, w, b: float((F.layer_norm(x, w, b, 1e-5)[0] * dy).sum())  # noqa: E731
    np.testing.assert_allclose(dx, differences(lambda v: of(v, w, b), x), atol=DIFF)
    np.testing.assert_allclose(dw, differences(lambda v: of(x, v, b), w), atol=DIFF)
    np.testing.assert_allclose(db, differences(lambda v: of(x, w, v), b), atol=DIFF)

    target, gl, ge = np.array([2, -1, 6]), r.normal(size=3), r.normal(size=3)

    def scored(v):
        s = F.log_probs(v, target, 0.7)
        return float((gl * s["logp"] + ge * s["entropy"]).sum())
    np.testing.assert_allclose(F.log_probs_backward(x, target, 0.7, gl, ge),
                               differences(scored, x), atol=DIFF)

    ids = np.array([[0, 3, -1], [5, 5, 1], [6, 2, 4]])
    values, weight = r.normal(size=(3, 3)), np.array([1.0, 0.5, 0.0])
    for kind in ("logits", "log_probs"):
        f = lambda v: float(F.distill(v, ids, values, 1.7, kind, weight)[0].sum())  # noqa: E731,B023
        np.testing.assert_allclose(F.distill(x, ids, values, 1.7, kind, weight)[1],
                                   differences(f, x), atol=DIFF)
