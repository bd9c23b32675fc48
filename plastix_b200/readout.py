"""The read-out of a network on torch tensors: rows (samples, or steps of a
stream) of unit activations, normalised, scored and trained against a teacher.

``layer_norm`` / ``layer_norm_backward``    the last hidden layer, per row
``log_probs`` / ``log_probs_backward``      log probability of given outputs,
                                            entropy, best alternatives
``distill``                                 loss and gradient against a
                                            teacher's top outputs

The alternatives that ``log_probs`` returns for a teacher are ``distill``'s
entries for its student (``kind="log_probs"``, same scale); the losses of the
reference for comparison are in include/plastix/traits.hpp:185-240. Rows are
float32, bfloat16 or float16 tensors whose last dimension is the units, with a
stride of 1; the dimensions before it have to collapse into rows of one
stride. Kernels run on the context's stream: tensors from another stream have
to be ready there, and results belong to it. Nothing is kept from one call to
the next, so calls can be captured into CUDA graphs and repeated.
"""
from __future__ import annotations

from contextlib import nullcontext
from typing import NamedTuple, Optional

import torch

from . import _abi
from .runtime import Context

_TYPES = {torch.float32: _abi.F32, torch.bfloat16: _abi.BF16, torch.float16: _abi.F16}
_HERE = nullcontext()
_KINDS = {"logits": _abi.TEACHER_LOGITS, "log_probs": _abi.TEACHER_LOG_PROBS}


class LogProbs(NamedTuple):
    logp: Optional[torch.Tensor]      # of the targets (None without targets)
    lse: torch.Tensor                 # log of the sum of exp(scale * logits)
    entropy: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]   # int32, largest logit first
    top_logp: Optional[torch.Tensor]


def _check_count(count: int, name: str) -> None:
    """Counts are 32-bit arguments of the library, which would take 2^32 + 8 as 8."""
    if not 0 <= count < 1 << 31:
        raise ValueError(f"{name} is {count}: 0 to fewer than 2^31 are supported")


def _rows(ctx: Context, t: torch.Tensor, name: str):
    """(rows, n, row stride, type number) of a tensor of rows on the context's
    device."""
    if t.device != ctx.device:
        raise ValueError(f"{name} is on {t.device}, the context on {ctx.device}")
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{name} is {t.dtype}: float32, bfloat16 and float16 are supported")
    shape = t.shape
    if len(shape) == 0 or shape[-1] == 0:
        raise ValueError(f"{name} needs a last dimension of units, got shape {tuple(shape)}")
    n = shape[-1]
    _check_count(n, f"the last dimension of {name}")
    if len(shape) != 2:
        try:
            t = t.view(-1, n) if t.numel() else t.reshape(-1, n)
        except RuntimeError:
            raise ValueError(f"the dimensions of {name} before the last do not collapse into "
                             f"rows of one stride (strides {t.stride()})") from None
        shape = t.shape
    rows = shape[0]
    ld, one = t.stride()
    if one != 1 and n > 1:
        raise ValueError(f"{name} needs a stride of 1 in its last dimension, got {one}")
    if rows <= 1:
        ld = n
    elif ld < n:
        raise ValueError(f"the rows of {name} overlap (row stride {ld}, {n} units)")
    return rows, n, ld, kind


def _like(ctx: Context, t: torch.Tensor, shape, dtype, name: str) -> int:
    """Address of a contiguous tensor of the given shape and type."""
    if t.dtype != dtype or t.shape != shape or t.device != ctx.device or not t.is_contiguous():
        if t.device != ctx.device:
            raise ValueError(f"{name} is on {t.device}, the context on {ctx.device}")
        raise ValueError(f"{name} has to be a contiguous {dtype} tensor of shape {tuple(shape)}, "
                         f"got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def _apart(a: torch.Tensor, lda: int, b: torch.Tensor, ldb: int) -> bool:
    """Whether two tensors of rows of the same shape and type share no element."""
    if a.numel() == 0:
        return True
    n, size = a.shape[-1], a.element_size()
    rows = a.numel() // n
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + ((rows - 1) * lda + n) * size <= pb or pb + ((rows - 1) * ldb + n) * size <= pa:
        return True
    # side by side in rows of the same stride
    return lda == ldb and n <= (pb - pa) // size % lda <= lda - n


def _result(ctx: Context, out: Optional[torch.Tensor], source: torch.Tensor, ld: int, name: str):
    """The tensor of rows that a call writes, and its row stride: ``out``, or
    a new one like ``source``. ``out`` may be the source itself."""
    if out is None:
        return (torch.empty_like(source) if source.is_contiguous() else
                source.new_empty(source.shape)), source.shape[-1]
    if out.shape != source.shape or out.dtype != source.dtype:
        raise ValueError(f"{name} has to be {source.dtype} {tuple(source.shape)}, got {out.dtype} "
                         f"{tuple(out.shape)}")
    ldo = _rows(ctx, out, name)[2]
    _check_result(out, ldo, source, ld, name)
    return out, ldo


def _check_result(out, ldo, source, ld, name) -> None:
    if out is not source and not (out.data_ptr() == source.data_ptr() and ldo == ld) \
            and not _apart(out, ldo, source, ld):
        raise ValueError(f"{name} overlaps an input and is not the input itself")


def _scope(ctx: Context, *used):
    """The context's stream as the current one, where it is not already, so
    that what a call allocates belongs to it; what the call uses is kept from
    being given out again until that stream is done with it."""
    # the handle alone: making a Stream object of it costs more than a small kernel
    if torch._C._cuda_getCurrentRawStream(ctx.device.index) == ctx.stream.cuda_stream:
        return _HERE
    for t in used:
        if t is not None:
            t.record_stream(ctx.stream)
    return torch.cuda.stream(ctx.stream)


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _param(ctx: Context, t: torch.Tensor, n: int, dtype, name: str) -> int:
    """The type number of an affine parameter of rows of the given type."""
    if t.dtype != torch.float32 and t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}: float32 or the rows' {dtype} is supported")
    _like(ctx, t, (n,), t.dtype, name)
    return _TYPES[t.dtype]


def _params(ctx: Context, weight, bias, n: int, dtype) -> int:
    """The type number of a weight and a bias, either of which may be None."""
    kind = _abi.F32
    if bias is not None:
        kind = _param(ctx, bias, n, dtype, "bias")
    if weight is not None:
        other, kind = kind, _param(ctx, weight, n, dtype, "weight")
        if bias is not None and other != kind:
            raise ValueError("weight and bias have different types")
    return kind


def layer_norm(ctx: Context, x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5, stats: bool = False,
               out: Optional[torch.Tensor] = None):
    """Rows of ``x`` with mean 0 and variance 1 (plus ``eps``), times
    ``weight`` plus ``bias`` ([n], float32 or x's type). With ``stats`` returns
    (y, mean, rstd), which ``layer_norm_backward`` takes. ``out`` may be x."""
    rows, n, ld, dtype = _rows(ctx, x, "x")
    kind = _params(ctx, weight, bias, n, x.dtype)
    with _scope(ctx, x, weight, bias, out):
        y, ldy = _result(ctx, out, x, ld, "out")
        mean = rstd = None
        if stats:
            mean = x.new_empty(x.shape[:-1], dtype=torch.float32)
            rstd = torch.empty_like(mean)
        _abi.call("plx_layer_norm", ctx.handle, rows, n, dtype, x.data_ptr(), ld, kind,
                  _address(weight), _address(bias), eps, y.data_ptr(), ldy, _address(mean),
                  _address(rstd))
    return (y, mean, rstd) if stats else y


def layer_norm_backward(ctx: Context, dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                        bias: Optional[torch.Tensor] = None,
                        out: Optional[torch.Tensor] = None):
    """(dx, dweight, dbias) for the rows and statistics of ``layer_norm``.
    dweight is None without a weight; dbias comes with a weight or with
    ``bias``, which only a call without a weight needs to give. Both have the
    parameters' type and the same bits on every call. ``out`` (for dx) may be
    dy or x."""
    rows, n, ld, dtype = _rows(ctx, x, "x")
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy has to be {x.dtype} {tuple(x.shape)}, got {dy.dtype} "
                         f"{tuple(dy.shape)}")
    lddy = _rows(ctx, dy, "dy")[2]
    lead = x.shape[:-1]
    mean_p = _like(ctx, mean, lead, torch.float32, "mean")
    rstd_p = _like(ctx, rstd, lead, torch.float32, "rstd")
    kind = _params(ctx, weight, bias, n, x.dtype)
    with _scope(ctx, dy, x, mean, rstd, weight, bias, out):
        dx, lddx = _result(ctx, out, dy, lddy, "out")
        if out is not None:
            _check_result(dx, lddx, x, ld, "out")
        dw = db = scratch = None
        size = 0
        if weight is not None:
            dw = torch.empty_like(weight)
        if weight is not None or bias is not None:
            db = torch.empty_like(weight if bias is None else bias)
            size = _abi.lib().plx_layer_norm_scratch_bytes(rows, n)
            scratch = x.new_empty(size, dtype=torch.uint8)
        _abi.call("plx_layer_norm_backward", ctx.handle, rows, n, dtype, dy.data_ptr(), lddy,
                  x.data_ptr(), ld, mean_p, rstd_p, kind, _address(weight), dx.data_ptr(), lddx,
                  _address(dw), _address(db), _address(scratch), size)
    return dx, dw, db


def log_probs(ctx: Context, logits: torch.Tensor, target: Optional[torch.Tensor] = None, *,
              top: int = 0, scale: float = 1.0, entropy: bool = False) -> LogProbs:
    """Softmax of ``scale * logits`` in each row: log probability of
    ``target`` (int32, -1 = none), entropy, and the ``top`` best alternatives
    with theirs. See plx_log_probs for masked and non-finite rows."""
    rows, n, ld, dtype = _rows(ctx, logits, "logits")
    lead = logits.shape[:-1]
    target_p = None if target is None else _like(ctx, target, lead, torch.int32, "target")
    _check_count(top, "top")
    with _scope(ctx, logits, target):
        lse = logits.new_empty(lead, dtype=torch.float32)
        logp = None if target is None else torch.empty_like(lse)
        ent = torch.empty_like(lse) if entropy else None
        ids = best = None
        if top:
            ids = logits.new_empty(lead + (top,), dtype=torch.int32)
            best = torch.empty_like(ids, dtype=torch.float32)
        _abi.call("plx_log_probs", ctx.handle, rows, n, dtype, logits.data_ptr(), ld,
                  target_p, scale, top, _address(logp), lse.data_ptr(), _address(ent),
                  _address(ids), _address(best))
    return LogProbs(logp, lse, ent, ids, best)


def log_probs_backward(ctx: Context, logits: torch.Tensor, lse: torch.Tensor,
                       target: Optional[torch.Tensor] = None,
                       grad_logp: Optional[torch.Tensor] = None,
                       entropy: Optional[torch.Tensor] = None,
                       grad_entropy: Optional[torch.Tensor] = None, *, scale: float = 1.0,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of sum(grad_logp * logp) + sum(grad_entropy * entropy) with
    respect to the logits; lse and entropy as ``log_probs`` returned them for
    the same logits and scale. ``out`` may be logits."""
    rows, n, ld, dtype = _rows(ctx, logits, "logits")
    lead = logits.shape[:-1]
    lse_p = _like(ctx, lse, lead, torch.float32, "lse")
    if target is not None:
        _like(ctx, target, lead, torch.int32, "target")
    if grad_logp is not None:
        _like(ctx, grad_logp, lead, torch.float32, "grad_logp")
    if entropy is not None:
        _like(ctx, entropy, lead, torch.float32, "entropy")
    if grad_entropy is not None:
        _like(ctx, grad_entropy, lead, torch.float32, "grad_entropy")
    if grad_logp is None and grad_entropy is None:
        raise ValueError("grad_logp or grad_entropy is required")
    if grad_logp is not None and target is None:
        raise ValueError("grad_logp needs target")
    if grad_entropy is not None and entropy is None:
        raise ValueError("grad_entropy needs entropy")
    with _scope(ctx, logits, lse, target, grad_logp, entropy, grad_entropy, out):
        dx, ldd = _result(ctx, out, logits, ld, "out")
        _abi.call("plx_log_probs_backward", ctx.handle, rows, n, dtype, logits.data_ptr(), ld,
                  _address(target), scale, lse_p, _address(entropy),
                  _address(grad_logp), _address(grad_entropy), dx.data_ptr(), ldd)
    return dx


def distill(ctx: Context, logits: torch.Tensor, teacher_ids: torch.Tensor,
            teacher_values: torch.Tensor, *, temperature: float = 1.0, kind: str = "logits",
            weight: Optional[torch.Tensor] = None, grad: bool = True,
            out: Optional[torch.Tensor] = None):
    """(loss, dlogits): per row weight * temperature^2 * KL from the teacher's
    listed outputs (``teacher_ids`` int32, -1 = empty entry, and
    ``teacher_values`` float32, both [..., k]) to softmax(logits /
    temperature), and the gradient of its sum over the rows (None without
    ``grad``). ``kind``: what the values are, the teacher's "logits" or its
    "log_probs" at this temperature. ``out`` (for dlogits) may be logits."""
    rows, n, ld, dtype = _rows(ctx, logits, "logits")
    lead = logits.shape[:-1]
    if kind not in _KINDS:
        raise ValueError(f"kind {kind!r} is neither 'logits' nor 'log_probs'")
    if teacher_ids.dim() == 0:
        raise ValueError("teacher_ids needs a last dimension of entries")
    k = teacher_ids.shape[-1]
    _check_count(k, "the last dimension of teacher_ids")
    ids_p = _like(ctx, teacher_ids, lead + (k,), torch.int32, "teacher_ids")
    values_p = _like(ctx, teacher_values, lead + (k,), torch.float32, "teacher_values")
    if weight is not None:
        _like(ctx, weight, lead, torch.float32, "weight")
    if out is not None and not grad:
        raise ValueError("out is for the gradient: it needs grad=True")
    with _scope(ctx, logits, teacher_ids, teacher_values, weight, out):
        loss = teacher_values.new_empty(lead)
        dx, ldd = _result(ctx, out, logits, ld, "out") if grad else (None, 0)
        _abi.call("plx_distill", ctx.handle, rows, n, dtype, logits.data_ptr(), ld,
                  k, ids_p, values_p, _KINDS[kind], temperature, _address(weight),
                  loss.data_ptr(), _address(dx), ldd)
    return loss, dx
