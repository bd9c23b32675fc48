"""The read-out operators in 64 bits on numpy arrays, row by row from their
definitions: what the device kernels are compared with."""
import numpy as np


def layer_norm(x, w, b, eps):
    mean = x.mean(1)
    rstd = 1 / np.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    return (x - mean[:, None]) * rstd[:, None] * w + b, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, w):
    h = (x - mean[:, None]) * rstd[:, None]
    g = dy * w
    dx = rstd[:, None] * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def log_softmax(z):
    """Rows of -inf have no distribution: -inf everywhere. NaN and +inf give NaN."""
    with np.errstate(invalid="ignore", divide="ignore"):
        m = z.max(1, keepdims=True)
        m = np.where(m == -np.inf, 0.0, m)
        s = np.exp(z - m).sum(1, keepdims=True)
        lse = m + np.log(s)
        return np.where(lse == -np.inf, -np.inf, z - lse), lse[:, 0]


def order(x):
    """Indexes by value, largest first, NaN before all, lower index first among equals."""
    key = np.where(np.isnan(x), np.inf, x)
    n = np.arange(x.shape[1])
    return np.stack([np.lexsort((n, -k, ~np.isnan(r))) for k, r in zip(key, x)])


def log_probs(x, target, scale, top=0):
    logs, lse = log_softmax(x * scale)
    p = np.exp(logs)
    with np.errstate(invalid="ignore"):
        entropy = -np.where(p == 0, 0.0, p * logs).sum(1)
    out = {"lse": lse, "entropy": entropy}
    if target is not None:
        rows = np.arange(len(x))
        out["logp"] = np.where(target < 0, 0.0, logs[rows, np.maximum(target, 0)])
    if top:
        out["top_ids"] = order(x)[:, :top]
        out["top_logp"] = np.take_along_axis(logs, out["top_ids"], 1)
    return out


def log_probs_backward(x, target, scale, grad_logp, grad_entropy):
    logs, _ = log_softmax(x * scale)
    p = np.exp(logs)
    g = np.zeros(len(x)) if grad_logp is None else np.where(target < 0, 0.0, grad_logp)
    dx = -g[:, None] * p
    if grad_logp is not None:
        dx[np.arange(len(x)), np.maximum(target, 0)] += g
    if grad_entropy is not None:
        with np.errstate(invalid="ignore"):
            pl = np.where(p == 0, 0.0, p * logs)
        dx -= grad_entropy[:, None] * (pl - p * pl.sum(1, keepdims=True))
    return dx * scale


def distill(x, ids, values, tau, kind, weight):
    logs, _ = log_softmax(x / tau)
    loss, dx = np.zeros(len(x)), np.zeros_like(x)
    for r in range(len(x)):
        given = ids[r] >= 0
        t = np.where(given, values[r], -np.inf)
        if kind == "logits":
            t = log_softmax(t[None] / tau)[0][0]
        q = np.exp(t)
        if weight[r] == 0 or not q.sum() > 0:
            continue
        with np.errstate(invalid="ignore"):
            terms = np.where(q > 0, q * (t - logs[r, np.maximum(ids[r], 0)]), 0.0)
        loss[r] = weight[r] * tau * tau * terms.sum()
        dx[r] = q.sum() * np.exp(logs[r])
        np.add.at(dx[r], ids[r][given], -q[given])
        dx[r] *= weight[r] * tau
    return loss, dx
