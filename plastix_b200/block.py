"""A block of hidden units on rows of torch tensors: what lies between a
network's input and its read-out (``plastix_b200.readout``), many rows
(samples, or steps of streams) at once.

``dense`` / ``dense_backward``              a fully connected layer
``recurrence`` / ``recurrence_backward``    gated linear recurrence of the units
                                            over the steps of streams
``block_norm`` / ``block_norm_backward``    the norm after a block and the one
                                            before the next, gate and residual

The reference steps one sample at a time through sparse connections
(include/plastix/plastix.hpp:101-256); a dense layer's weights are in the order
of its FullyConnected builder (include/plastix/layers.hpp:49-77): row i holds
what reaches unit i. Rows, streams and captures as in ``readout``: float32,
bfloat16 or float16 with a stride of 1 in the last dimension, dimensions before
it that collapse into rows of one stride, kernels on the context's stream,
nothing kept between calls.
"""
from __future__ import annotations

from ctypes import byref
from typing import NamedTuple, Optional

import torch

from . import _abi
from .readout import (_TYPES, _address, _check_count, _check_result, _like, _param, _rows,
                      _scope)
from .runtime import Context

_ACTS = {"identity": _abi.ACT_IDENTITY, "sigmoid": _abi.ACT_SIGMOID, "tanh": _abi.ACT_TANH,
         "relu": _abi.ACT_RELU, "silu": _abi.ACT_SILU, "gelu": _abi.ACT_GELU}
_NORMS = {"rms": _abi.NORM_RMS, "layer": _abi.NORM_LAYER}
_GATES = {"decay": _abi.GATE_DECAY, "sigmoid": _abi.GATE_SIGMOID}
_GATE_APPLY = {"identity": 0, "sigmoid": 1}


class BlockNormGrads(NamedTuple):
    dx: torch.Tensor
    do: torch.Tensor
    dgate: Optional[torch.Tensor]          # like the gate
    dpost_weight: Optional[torch.Tensor]   # None where there is no such parameter
    dpost_bias: Optional[torch.Tensor]
    dpre_weight: Optional[torch.Tensor]
    dpre_bias: Optional[torch.Tensor]


def _one_of(table: dict, key: str, name: str) -> int:
    value = table.get(key)
    if value is None:
        raise ValueError(f"{name} {key!r} is none of {', '.join(map(repr, table))}")
    return value


def _plain_rows(ctx: Context, t: torch.Tensor, name: str):
    """(rows, n, row stride, type number), as ``_rows``; quickly for contiguous tensors."""
    kind, shape = _TYPES.get(t.dtype), t.shape
    if kind is not None and shape and 0 < shape[-1] < 1 << 31 and t.is_contiguous() \
            and t.device == ctx.device:
        n = shape[-1]
        return t.numel() // n, n, n, kind
    return _rows(ctx, t, name)


def _same_rows(ctx: Context, t: torch.Tensor, like: torch.Tensor, name: str, of: str) -> int:
    """The row stride of a tensor that has to have another one's shape and type."""
    if t.shape == like.shape and t.dtype is like.dtype and t.is_contiguous() \
            and t.device == ctx.device:
        return t.shape[-1]
    if t.shape != like.shape or t.dtype != like.dtype:
        raise ValueError(f"{name} has to be {like.dtype} {tuple(like.shape)} like {of}, got "
                         f"{t.dtype} {tuple(t.shape)}")
    return _rows(ctx, t, name)[2]


def _vector(ctx: Context, t: torch.Tensor, n: int, dtype, name: str) -> int:
    """The type number of a parameter of every unit, as ``_param``."""
    if t.dtype is dtype and t.dim() == 1 and t.shape[0] == n and t.is_contiguous() \
            and t.device == ctx.device:
        return _TYPES[dtype]
    return _param(ctx, t, n, dtype, name)


def _span(t: torch.Tensor, ld: int):
    """First and last address + 1 of a tensor of rows."""
    n = t.shape[-1]
    rows = t.numel() // n
    return t.data_ptr(), t.data_ptr() + ((rows - 1) * ld + n) * t.element_size()


def _check_apart(out: torch.Tensor, ldo: int, name: str, *others) -> None:
    """Refuses an output that touches any of the inputs (tensor, row stride, name)."""
    if out.numel() == 0:
        return
    a, b = _span(out, ldo)
    size = out.element_size()
    for t, ld, other in others:
        if t is not None and t.numel():
            c, d = _span(t, ld)
            if a < d and c < b:
                # side by side in rows of the same stride
                if ld == ldo and t.element_size() == size and (c - a) % size == 0:
                    between = (c - a) // size % ld
                    if out.shape[-1] <= between <= ld - t.shape[-1]:
                        continue
                raise ValueError(f"{name} overlaps {other}")


def _new(like: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor of another one's shape and type."""
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)


def _in_place_of(ctx: Context, out: torch.Tensor, *inputs) -> int:
    """The row stride of ``out``, which may be one of the inputs (tensor, row
    stride, name) and touches no other. Inputs that are the same rows count as
    one; rows that only begin where out does are others."""
    ldo = _same_rows(ctx, out, inputs[0][0], "out", inputs[0][2])
    _check_apart(out, ldo, "out", *(i for i in inputs
                                    if i[0].data_ptr() != out.data_ptr() or i[1] != ldo))
    return ldo


# ------------------------------------------------------------------------------- dense layer
def _weight(ctx: Context, weight: torch.Tensor, n: int, dtype):
    """(units, row stride) of a layer's weights for rows of n values."""
    if weight.dim() != 2 or weight.shape[1] != n or weight.dtype != dtype:
        raise ValueError(f"weight has to be {dtype} [units, {n}], got {weight.dtype} "
                         f"{tuple(weight.shape)}")
    m, _, ld, _ = _plain_rows(ctx, weight, "weight")
    if not 0 < m < 1 << 31:
        raise ValueError(f"weight has {m} units: 1 to fewer than 2^31 are supported")
    return m, ld


def _aligned(*rows) -> bool:
    """Whether tensors of rows (tensor, row stride, rows) start at, and have
    strides of, multiples of 16 bytes."""
    for t, ld, count in rows:
        if t.data_ptr() % 16 or (count > 1 and ld * t.element_size() % 16):
            return False
    return True


def dense(ctx: Context, x: torch.Tensor, weight: torch.Tensor,
          bias: Optional[torch.Tensor] = None, *, apply: str = "identity",
          residual: Optional[torch.Tensor] = None, pre: bool = False,
          out: Optional[torch.Tensor] = None):
    """act(x weight^T + bias) + residual for rows of ``x`` [..., n], ``weight``
    [m, n] of x's type, ``bias`` [m] (float32 or x's type) and ``residual``
    [..., m]. ``apply``: "identity", "sigmoid", "tanh", "relu", "silu" (z
    sigmoid(z)) or "gelu" (z Phi(z)). With ``pre`` returns (y, z): z = x
    weight^T + bias in float32, which ``dense_backward`` takes. ``out`` may be
    residual."""
    rows, n, ldx, dtype = _plain_rows(ctx, x, "x")
    m, ldw = _weight(ctx, weight, n, x.dtype)
    act = _one_of(_ACTS, apply, "apply")
    kind = _abi.F32 if bias is None else _vector(ctx, bias, m, x.dtype, "bias")
    shape = x.shape[:-1] + (m,)
    ldr = 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != x.dtype:
            raise ValueError(f"residual has to be {x.dtype} {tuple(shape)}, got "
                             f"{residual.dtype} {tuple(residual.shape)}")
        ldr = _rows(ctx, residual, "residual")[2]
    y, ldy = out, m
    if out is not None:
        if out.shape != shape or out.dtype != x.dtype:
            raise ValueError(f"out has to be {x.dtype} {tuple(shape)}, got {out.dtype} "
                             f"{tuple(out.shape)}")
        ldy = _rows(ctx, out, "out")[2]
        if residual is not None:
            _check_result(out, ldy, residual, ldr, "out")
        _check_apart(out, ldy, "out", (x, ldx, "x"), (weight, ldw, "weight"), (bias, m, "bias"))
    # aligned rows of 16-bit values need no scratch
    size = 0 if dtype != _abi.F32 and _aligned((x, ldx, rows), (weight, ldw, m)) else \
        _abi.lib().plx_dense_scratch_bytes(rows, n, m, dtype, 0, 0)
    with _scope(ctx, x, weight, bias, residual, out):
        if out is None:
            y = x.new_empty(shape)
        z = x.new_empty(shape, dtype=torch.float32) if pre else None
        scratch = x.new_empty(size, dtype=torch.uint8) if size else None
        _abi.call("plx_dense", ctx.handle, rows, n, m, dtype, x.data_ptr(), ldx,
                  weight.data_ptr(), ldw, kind, _address(bias), act, _address(residual), ldr,
                  y.data_ptr(), ldy, _address(z), _address(scratch), size)
    return (y, z) if pre else y


def dense_backward(ctx: Context, dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                   pre: Optional[torch.Tensor] = None, *, apply: str = "identity",
                   bias: Optional[torch.Tensor] = None, input_grad: bool = True,
                   weight_grad: bool = True):
    """(dx, dweight, dbias) of ``dense``; the residual's gradient is dy itself.
    ``pre`` is z as ``dense`` returned it (not needed for "identity"). dx is
    None without ``input_grad``, dweight without ``weight_grad``; dbias, in
    bias's type, comes with ``bias``."""
    rows, n, ldx, dtype = _plain_rows(ctx, x, "x")
    m, ldw = _weight(ctx, weight, n, x.dtype)
    act = _one_of(_ACTS, apply, "apply")
    shape = x.shape[:-1] + (m,)
    if dy.shape != shape or dy.dtype != x.dtype:
        raise ValueError(f"dy has to be {x.dtype} {tuple(shape)}, got {dy.dtype} "
                         f"{tuple(dy.shape)}")
    lddy = _rows(ctx, dy, "dy")[2]
    if pre is not None:
        _like(ctx, pre, shape, torch.float32, "pre")
    elif act != _abi.ACT_IDENTITY:
        raise ValueError(f"pre is required for {apply!r}")
    kind = _abi.F32 if bias is None else _vector(ctx, bias, m, x.dtype, "bias")
    with _scope(ctx, dy, x, weight, pre, bias):
        dx = x.new_empty(x.shape) if input_grad else None
        dw = weight.new_empty(weight.shape) if weight_grad else None
        db = torch.empty_like(bias) if bias is not None else None
        size = _abi.lib().plx_dense_scratch_bytes(
            rows, n, m, dtype, 1, _aligned((x, ldx, rows), (weight, ldw, m), (dy, lddy, rows)))
        scratch = x.new_empty(size, dtype=torch.uint8)
        _abi.call("plx_dense_backward", ctx.handle, rows, n, m, dtype, dy.data_ptr(), lddy,
                  x.data_ptr(), ldx, weight.data_ptr(), ldw, act, _address(pre), _address(dx), n,
                  _address(dw), n, kind, _address(db), scratch.data_ptr(), size)
    return dx, dw, db


# ------------------------------------------------------------------------------- block norm
def _block_params(ctx: Context, x, gate, gate_apply, kind, post, scale, eps, post_weight,
                  post_bias, pre_weight, pre_bias):
    """The call's parameters, and what they were made of."""
    n, dtype = x.shape[-1], x.dtype
    if not post and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias need post=True")
    how, address, ldg, units = _abi.BLOCK_GATE_NONE, None, 0, None
    if gate is not None:
        address = gate.data_ptr()
        if gate.dim() == 1 and x.dim() != 1:
            how, units = _abi.BLOCK_GATE_UNITS, gate
        else:
            how, ldg = _abi.BLOCK_GATE_VALUES, _same_rows(ctx, gate, x, "gate", "x")
    param = None
    for name, v in (("gate", units), ("post_weight", post_weight), ("post_bias", post_bias),
                    ("pre_weight", pre_weight), ("pre_bias", pre_bias)):
        if v is not None:
            of = _vector(ctx, v, n, dtype, name)
            if param is not None and of != param:
                raise ValueError("the parameters have different types")
            param = of
    return _abi.BlockNormParams(
        _one_of(_NORMS, kind, "kind"), 1 if post else 0, how,
        _one_of(_GATE_APPLY, gate_apply, "gate_apply"), _abi.F32 if param is None else param, scale,
        eps, address, ldg, _address(post_weight), _address(post_bias), _address(pre_weight),
        _address(pre_bias))


def block_norm(ctx: Context, x: torch.Tensor, o: torch.Tensor,
               gate: Optional[torch.Tensor] = None, *, kind: str = "rms", post: bool = True,
               scale: float = 1.0, gate_apply: str = "identity", eps: float = 1e-5,
               post_weight: Optional[torch.Tensor] = None,
               post_bias: Optional[torch.Tensor] = None,
               pre_weight: Optional[torch.Tensor] = None,
               pre_bias: Optional[torch.Tensor] = None, stats: bool = False,
               out: Optional[torch.Tensor] = None):
    """(r, u): r = scale * x + gate * p, the residual stream after a block, and
    u = N(r) pre_weight + pre_bias, the next block's input, where p = N(o)
    post_weight + post_bias is the block's output ``o`` normalised (o itself
    with ``post=False``). N divides by the root of the mean square ("rms"), or
    takes the mean away first ("layer"). ``gate``: a value of every unit ([n],
    as the parameters float32 or x's type), of every unit of every row (like x;
    so is a gate for an x of one dimension), or None for 1; ``gate_apply``
    "sigmoid" takes its sigmoid. With ``stats`` returns (r, u, stats), which
    ``block_norm_backward`` takes. ``out`` (for r) may be x, o or a gate of
    every value."""
    rows, n, ldx, dtype = _plain_rows(ctx, x, "x")
    ldo = _same_rows(ctx, o, x, "o", "x")
    p = _block_params(ctx, x, gate, gate_apply, kind, post, scale, eps, post_weight, post_bias,
                      pre_weight, pre_bias)
    r, ldr = out, n
    if out is not None:
        inputs = [(x, ldx, "x"), (o, ldo, "o")]
        if p.gate == _abi.BLOCK_GATE_VALUES:
            inputs.append((gate, p.ldg, "gate"))
        ldr = _in_place_of(ctx, out, *inputs)
        units = gate if p.gate == _abi.BLOCK_GATE_UNITS else None
        _check_apart(out, ldr, "out", (units, n, "gate"),
                     (post_weight, n, "post_weight"), (post_bias, n, "post_bias"),
                     (pre_weight, n, "pre_weight"), (pre_bias, n, "pre_bias"))
    with _scope(ctx, x, o, gate, post_weight, post_bias, pre_weight, pre_bias, out):
        if out is None:
            r = _new(x)
        u = _new(x)
        st = x.new_empty(x.shape[:-1] + (4,), dtype=torch.float32) if stats else None
        _abi.call("plx_block_norm", ctx.handle, rows, n, dtype, x.data_ptr(), ldx, o.data_ptr(),
                  ldo, byref(p), r.data_ptr(), ldr, u.data_ptr(), n, _address(st))
    return (r, u, st) if stats else (r, u)


def block_norm_backward(ctx: Context, dr: Optional[torch.Tensor], du: Optional[torch.Tensor],
                        x: torch.Tensor, o: torch.Tensor, stats: torch.Tensor,
                        gate: Optional[torch.Tensor] = None, *, kind: str = "rms",
                        post: bool = True, scale: float = 1.0, gate_apply: str = "identity",
                        post_weight: Optional[torch.Tensor] = None,
                        post_bias: Optional[torch.Tensor] = None,
                        pre_weight: Optional[torch.Tensor] = None,
                        pre_bias: Optional[torch.Tensor] = None) -> BlockNormGrads:
    """Gradients of sum(dr * r) + sum(du * u) for the arguments and statistics
    of ``block_norm``; dr or du may be None. Gradients of the parameters and of
    a gate of every unit are summed over the rows, the same bits on every
    call."""
    rows, n, ldx, dtype = _plain_rows(ctx, x, "x")
    ldo = _same_rows(ctx, o, x, "o", "x")
    if dr is None and du is None:
        raise ValueError("dr or du is required")
    lddr = 0 if dr is None else _same_rows(ctx, dr, x, "dr", "x")
    lddu = 0 if du is None else _same_rows(ctx, du, x, "du", "x")
    stats_p = _like(ctx, stats, x.shape[:-1] + (4,), torch.float32, "stats")
    p = _block_params(ctx, x, gate, gate_apply, kind, post, scale, 0.0, post_weight, post_bias,
                      pre_weight, pre_bias)
    with _scope(ctx, dr, du, x, o, stats, gate, post_weight, post_bias, pre_weight, pre_bias):
        dx, do = _new(x), _new(x)
        dgate = None if gate is None else gate.new_empty(gate.shape)
        dw1, db1, dw2, db2 = (None if v is None else torch.empty_like(v)
                              for v in (post_weight, post_bias, pre_weight, pre_bias))
        size = _abi.lib().plx_block_norm_scratch_bytes(rows, n)
        scratch = x.new_empty(size, dtype=torch.uint8)
        _abi.call("plx_block_norm_backward", ctx.handle, rows, n, dtype, _address(dr), lddr,
                  _address(du), lddu, x.data_ptr(), ldx, o.data_ptr(), ldo, stats_p, byref(p),
                  dx.data_ptr(), n, do.data_ptr(), n, _address(dgate), n, _address(dw1),
                  _address(db1), _address(dw2), _address(db2), scratch.data_ptr(), size)
    return BlockNormGrads(dx, do, dgate, dw1, db1, dw2, db2)


# ------------------------------------------------------------------------------- recurrence
def _streams(ctx: Context, x: torch.Tensor, offsets: Optional[torch.Tensor]):
    """(streams, address of the offsets) of rows that are steps of streams."""
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] == 0:
            raise ValueError("offsets needs one dimension of streams + 1 values, got shape "
                             f"{tuple(offsets.shape)}")
        streams = offsets.shape[0] - 1
        _check_count(streams, "the number of streams")
        if x.dim() != 2:
            raise ValueError(f"with offsets x needs two dimensions, [rows, n], got {x.dim()}")
        return streams, _like(ctx, offsets, offsets.shape, torch.int32, "offsets")
    if x.dim() not in (2, 3):
        raise ValueError("x needs two dimensions, [steps, n] of one stream, or three, "
                         f"[streams, steps, n], got {x.dim()}")
    streams = 1 if x.dim() == 2 else x.shape[0]
    _check_count(streams, "the number of streams")
    return streams, None


def _state(ctx: Context, t: Optional[torch.Tensor], x: torch.Tensor, streams: int, name: str):
    """Shape and address of a state of every stream ([n] for the one of a 2-D x)."""
    shape = (streams, x.shape[-1])
    if t is not None:
        _like(ctx, t, shape, torch.float32, name)
    return _address(t)


def recurrence(ctx: Context, x: torch.Tensor, gate: torch.Tensor,
               state: Optional[torch.Tensor] = None, *, kind: str = "sigmoid",
               mix: bool = False, offsets: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None, final_out: Optional[torch.Tensor] = None):
    """(h, final): h_t = a_t h_{t-1} + x_t over the steps of streams, or with
    ``mix`` a_t h_{t-1} + (1 - a_t) x_t, every unit by itself. ``x`` and
    ``gate`` are [streams, steps, n], [steps, n] for one stream, or with
    ``offsets`` (int32 [streams + 1]) [rows, n] with stream s in the rows from
    offsets[s] to before offsets[s + 1]; rows of no stream are left as they
    are in ``out``, and zero in a new h. a is the gate ("decay") or its sigmoid
    ("sigmoid"). ``state`` [streams, n] in float32 is h before the first steps
    (None: 0), ``final`` h after the last ones, what ``state`` was for streams
    without steps. ``out`` may be x or gate, ``final_out`` state: a step in
    place."""
    rows, n, ldx, dtype = _plain_rows(ctx, x, "x")
    ldg = _same_rows(ctx, gate, x, "gate", "x")
    gate_kind = _one_of(_GATES, kind, "kind")
    streams, offsets_p = _streams(ctx, x, offsets)
    state_p = _state(ctx, state, x, streams, "state")
    h, ldh = out, n
    if out is not None:
        ldh = _in_place_of(ctx, out, (x, ldx, "x"), (gate, ldg, "gate"))
        _check_apart(out, ldh, "out", (state, n, "state"), (offsets, 0, "offsets"))
    final = final_out
    if final is not None:
        _state(ctx, final, x, streams, "final_out")
        if final.data_ptr() != state_p:
            _check_apart(final, n, "final_out", (state, n, "state"))
        _check_apart(final, n, "final_out", (x, ldx, "x"), (gate, ldg, "gate"), (out, ldh, "out"),
                     (offsets, 0, "offsets"))
    with _scope(ctx, x, gate, state, offsets, out, final_out):
        if out is None:
            h = _new(x)
        if final is None:
            final = x.new_empty((streams, n), dtype=torch.float32)
        size = _abi.lib().plx_recurrence_scratch_bytes(streams, rows, n, dtype,
                                                       offsets is not None, int(mix), 0)
        scratch = x.new_empty(size, dtype=torch.uint8) if size else None
        _abi.call("plx_recurrence_new" if out is None else "plx_recurrence", ctx.handle, streams,
                  rows, n, dtype, offsets_p, x.data_ptr(), ldx, gate.data_ptr(), ldg, gate_kind,
                  int(mix), state_p, h.data_ptr(), ldh, final.data_ptr(), _address(scratch), size)
    return h, final


def recurrence_backward(ctx: Context, dh: torch.Tensor, gate: torch.Tensor, h: torch.Tensor,
                        state: Optional[torch.Tensor] = None, *,
                        x: Optional[torch.Tensor] = None, dfinal: Optional[torch.Tensor] = None,
                        kind: str = "sigmoid", mix: bool = False,
                        offsets: Optional[torch.Tensor] = None):
    """(dx, dgate, dstate): gradients of sum(dh * h) + sum(dfinal * final) for
    the arguments of ``recurrence`` and the h that it returned. ``x`` is needed
    with ``mix`` alone; ``dfinal`` may be None. dstate is None without a state.
    dx and dgate are zero in rows of no stream."""
    rows, n, ldg, dtype = _plain_rows(ctx, gate, "gate")
    lddh = _same_rows(ctx, dh, gate, "dh", "gate")
    ldh = _same_rows(ctx, h, gate, "h", "gate")
    if mix and x is None:
        raise ValueError("x is required with mix")
    ldx = 0 if x is None else _same_rows(ctx, x, gate, "x", "gate")
    gate_kind = _one_of(_GATES, kind, "kind")
    streams, offsets_p = _streams(ctx, gate, offsets)
    state_p = _state(ctx, state, gate, streams, "state")
    dfinal_p = _state(ctx, dfinal, gate, streams, "dfinal")
    with _scope(ctx, dh, gate, h, x, state, dfinal, offsets):
        dx, dgate = _new(gate), _new(gate)
        dstate = None if state is None else torch.empty_like(state)
        size = _abi.lib().plx_recurrence_scratch_bytes(streams, rows, n, dtype,
                                                       offsets is not None, int(mix), 1)
        scratch = gate.new_empty(size, dtype=torch.uint8) if size else None
        _abi.call("plx_recurrence_backward", ctx.handle, streams, rows, n, dtype, offsets_p,
                  dh.data_ptr(), lddh, _address(x), ldx, gate.data_ptr(), ldg, gate_kind,
                  int(mix), h.data_ptr(), ldh, state_p, dfinal_p, dx.data_ptr(), n,
                  dgate.data_ptr(), n, _address(dstate), _address(scratch), size)
    return dx, dgate, dstate
