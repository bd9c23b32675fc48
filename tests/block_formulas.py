"""The block operators' formulas in 64 bits (numpy), one step or one value after the other."""
import numpy as np
from scipy.special import erf


def act(z, apply):
    """(act(z), act'(z))"""
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.where(z >= 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))
        keep = np.where(z < 0, 1 / (1 + np.exp(-np.abs(z))), np.exp(-np.abs(z)) / (1 + np.exp(-np.abs(z))))
        if apply == "identity":
            return z, np.ones_like(z)
        if apply == "sigmoid":
            return s, s * keep
        if apply == "tanh":
            return np.tanh(z), 1 - np.tanh(z) ** 2
        if apply == "relu":
            return np.where(z > 0, z, np.where(np.isnan(z), z, 0.0)), np.where(z > 0, 1.0, 0.0)
        if apply == "silu":
            return z * s, s * (1 + z * keep)
        cdf = 0.5 * (1 + erf(z / np.sqrt(2)))
        return z * cdf, cdf + z * np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)


def dense(x, w, b=None, apply="identity", residual=None):
    z = x @ w.T + (0 if b is None else b)
    y = act(z, apply)[0]
    return (y if residual is None else y + residual), z


def dense_backward(dy, x, w, z, apply="identity"):
    dz = dy * act(z, apply)[1]
    return dz @ w, dz.T @ x, dz.sum(0), dz


def norm(v, kind, eps):
    mean = v.mean(1, keepdims=True) if kind == "layer" else np.zeros((len(v), 1))
    d = v - mean
    rstd = 1 / np.sqrt((d * d).mean(1, keepdims=True) + eps)
    return d * rstd, mean, rstd


def _affine(h, w, b):
    h = h if w is None else h * w
    return h if b is None else h + b


def block_norm(x, o, gate=None, *, kind="rms", post=True, scale=1.0, gate_apply="identity", eps=1e-5,
               post_weight=None, post_bias=None, pre_weight=None, pre_bias=None):
    """r, u and what the backward pass needs."""
    h1, m1, s1 = norm(o, kind, eps) if post else (o, np.zeros((len(o), 1)), np.zeros((len(o), 1)))
    p = _affine(h1, post_weight, post_bias)
    g, slope = (1.0, 1.0) if gate is None else act(gate, gate_apply)
    r = scale * x + g * p
    h2, m2, s2 = norm(r, kind, eps)
    u = _affine(h2, pre_weight, pre_bias)
    return r, u, dict(h1=h1, s1=s1, p=p, g=g, slope=slope, h2=h2, s2=s2, stats=np.concatenate([m1, s1, m2, s2], 1))


def _norm_backward(e, h, s, kind):
    back = e - h * (e * h).mean(1, keepdims=True)
    return s * (back - (e.mean(1, keepdims=True) if kind == "layer" else 0.0))


def block_norm_backward(dr, du, k, *, kind="rms", post=True, scale=1.0, gate_units=False, post_weight=None,
                        pre_weight=None):
    d = np.zeros_like(k["h2"]) if dr is None else dr.copy()
    out = {}
    if du is not None:
        d = d + _norm_backward(du if pre_weight is None else du * pre_weight, k["h2"], k["s2"], kind)
        out["dpre_weight"], out["dpre_bias"] = (du * k["h2"]).sum(0), du.sum(0)
    else:
        out["dpre_weight"] = out["dpre_bias"] = np.zeros(d.shape[1])
    out["dx"] = scale * d
    dgate = d * k["p"] * k["slope"]
    out["dgate"] = dgate.sum(0) if gate_units else dgate
    dp = d * k["g"]
    out["dpost_weight"], out["dpost_bias"] = (dp * k["h1"]).sum(0), dp.sum(0)
    if post:
        dp = _norm_backward(dp if post_weight is None else dp * post_weight, k["h1"], k["s1"], kind)
    out["do"] = dp
    return out


def gates(gate, kind):
    if kind == "decay":
        return gate, 1 - gate
    a = act(gate, "sigmoid")[0]
    return a, act(-gate, "sigmoid")[0]


def recurrence(x, gate, state, offsets, kind="sigmoid", mix=False):
    """h (NaN in rows of no stream) and the final states of rows cut by offsets."""
    a, keep = gates(gate, kind)
    b = keep * x if mix else x
    h, final = np.full_like(x, np.nan), state.copy()
    for s in range(len(offsets) - 1):
        for t in range(offsets[s], offsets[s + 1]):
            h[t] = final[s] = a[t] * final[s] + b[t]
    return h, final


def recurrence_backward(dh, x, gate, h, state, dfinal, offsets, kind="sigmoid", mix=False):
    a, keep = gates(gate, kind)
    dx, dgate, dstate = np.full_like(gate, np.nan), np.full_like(gate, np.nan), dfinal.copy()
    for s in range(len(offsets) - 1):
        for t in range(offsets[s + 1] - 1, offsets[s] - 1, -1):
            g = dh[t] + dstate[s]
            before = h[t - 1] if t > offsets[s] else state[s]
            da = g * (before - x[t] if mix else before)
            dx[t] = g * keep[t] if mix else g
            dgate[t] = da * a[t] * keep[t] if kind == "sigmoid" else da
            dstate[s] = a[t] * g
    return dx, dgate, dstate
