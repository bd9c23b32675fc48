"""A block of hidden units on rows (dense layer, norms around a block, gated linear recurrence) as
cases to be measured.

Three operators in the order a network uses them between its input and its read-out: a fully
connected layer (``dense``), the gated linear recurrence of the units over the steps of a stream
(``recurrence``), and the norms after a block and before the next one with gate and residual scale
(``block_norm``). ``run`` computes a case in plain torch operations, or through
``plastix_b200.block`` where ``own`` is true.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5
_SQRT_HALF = math.sqrt(0.5)
_context = None


# ------------------------------------------------------------------------------------------ cases
def _dense(name, rows, n, m, dtype, apply, residual=False, train=False):
    return {"name": name, "op": "dense", "rows": rows, "n": n, "m": m, "dtype": dtype,
            "apply": apply, "residual": residual, "train": train}


def _block_norm(name, rows, n, dtype, kind, gate, gate_apply="identity", scale=1.0, post=True, train=False):
    return {"name": name, "op": "block_norm", "rows": rows, "n": n, "dtype": dtype, "kind": kind,
            "gate": gate, "gate_apply": gate_apply, "scale": scale, "post": post, "train": train}


def _recurrence(name, streams, steps, n, dtype, kind, mix, ragged=False, train=False):
    return {"name": name, "op": "recurrence", "streams": streams, "steps": steps, "n": n,
            "dtype": dtype, "kind": kind, "mix": mix, "ragged": ragged, "train": train}


def listed():
    return [
        # one step of eight streams through a layer: the weights are what is read
        _dense("dense_step_8x4096x4096_bf16", 8, 4096, 4096, "bf16", "silu"),
        # evaluation of a large batch through the first layer of a block
        _dense("dense_eval_16384x4096x4096_bf16", 16384, 4096, 4096, "bf16", "gelu", residual=True),
        # training of a narrowing layer on a batch, all gradients
        _dense("dense_train_8192x4096x2048_f16", 8192, 4096, 2048, "f16", "silu", train=True),
        # training in the framework's own type, sizes that no tile divides
        _dense("dense_train_1501x1001x777_f32", 1501, 1001, 777, "f32", "tanh", train=True),
        # one step of sixteen streams around a block: launch and latency count
        _block_norm("block_norm_step_16x1024_bf16", 16, 1024, "bf16", "rms", "units"),
        # evaluation of a large batch, a gate of every value
        _block_norm("block_norm_eval_16384x4096_bf16", 16384, 4096, "bf16", "rms", "values", "sigmoid"),
        # training at full size, a learned scale of every unit
        _block_norm("block_norm_train_16384x4096_bf16", 16384, 4096, "bf16", "rms", "units", train=True),
        # training in the framework's own type, mean and deviation, odd sizes, a scaled residual
        _block_norm("block_norm_train_3001x1001_f32", 3001, 1001, "f32", "layer", "values", scale=0.8, train=True),
        # one step of 256 streams from their states
        _recurrence("recurrence_step_256x1x2048_bf16", 256, 1, 2048, "bf16", "sigmoid", True),
        # training on a batch of streams
        _recurrence("recurrence_train_8x2048x4096_bf16", 8, 2048, 4096, "bf16", "sigmoid", True, train=True),
        # one long stream of few units: work has to be split over its steps
        _recurrence("recurrence_1x65536x512_bf16", 1, 65536, 512, "bf16", "sigmoid", False),
        # episodes of unequal length behind each other, decays given, the framework's own type
        _recurrence("recurrence_train_ragged_37x541x501_f32", 37, 541, 501, "f32", "decay", False, ragged=True, train=True),
    ]


def _size(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 128:  # half of the sizes are multiples of 64, as most layers' are
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["dense", "block_norm", "recurrence"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.5
    if op == "dense":
        n, m = _size(rng, 32, 8192), _size(rng, 32, 8192)
        most = (1 << (33 if dtype == "f32" else 36 if train else 37)) // (n * m)
        rows = _size(rng, 1, max(1, min(16384, most)))
        c = _dense("", rows, n, m, dtype, rng.choice(["identity", "sigmoid", "tanh", "relu", "silu", "gelu"]),
                   rng.random() < 0.5, train)
    elif op == "block_norm":
        n = _size(rng, 32, 8192)
        rows = _size(rng, 1, min(32768, (1 << (24 if dtype == "f32" else 25)) // n))
        c = _block_norm("", rows, n, dtype, rng.choice(["rms", "layer"]), rng.choice(["none", "units", "values"]),
                        rng.choice(["identity", "sigmoid"]), rng.choice([1.0, 0.8, 2.0]), rng.random() < 0.8, train)
    else:
        n = _size(rng, 32, 8192)
        most = (1 << (24 if dtype == "f32" else 25)) // n
        streams = _size(rng, 1, min(256, most))
        steps = _size(rng, 1, max(1, min(65536, most // streams)))
        c = _recurrence("", streams, steps, n, dtype, rng.choice(["sigmoid", "decay"]), rng.random() < 0.5,
                        rng.random() < 0.3, train)
    del c["name"]
    return c


def work(case):
    e = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    n = case["n"]
    if case["op"] == "dense":
        rows, m = case["rows"], case["m"]
        nbytes = e * (rows * n + n * m + m + rows * m * (1 + case["residual"]))
        flops = 2 * rows * n * m
        if case["train"]:  # dy and, once more, x and the weights read; dx, dweight and dbias written
            nbytes, flops = nbytes + e * (rows * m + 2 * rows * n + 2 * n * m + m), 3 * flops
    elif case["op"] == "block_norm":
        cells = case["rows"] * n
        gated = case["gate"] == "values"
        vectors = (case["gate"] == "units") + (1 + (case["kind"] == "layer")) * (1 + case["post"])
        nbytes, flops = e * ((4 + gated) * cells + vectors * n), 16 * cells
        if case["train"]:  # dr, du, x, o read, dx and do written; the gate and its gradient
            nbytes, flops = nbytes + e * ((6 + 2 * gated) * cells + 2 * vectors * n), flops + 40 * cells
    else:
        cells = case["streams"] * case["steps"] * n
        nbytes, flops = 3 * e * cells + 8 * case["streams"] * n, 8 * cells
        if case["train"]:  # dh, gate, h and, mixed, x read; dx and dgate written; gradients of the states
            nbytes = nbytes + (5 + case["mix"]) * e * cells + 12 * case["streams"] * n
            flops = flops + 16 * cells
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, n = _TYPES[case["dtype"]], case["n"]

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, scale, generator=g)

    s = dict(case)
    if case["op"] == "dense":
        rows, m = case["rows"], case["m"]
        s["x"] = normal(rows, n).to(dt)
        s["weight"] = normal(m, n, scale=n ** -0.5).to(dt)
        s["bias"] = normal(m, scale=0.2).to(dt)
        s["residual_rows"] = normal(rows, m).to(dt) if case["residual"] else None
        if case["train"]:
            s["dy"] = normal(rows, m).to(dt)
    elif case["op"] == "block_norm":
        rows = case["rows"]
        s["x"] = normal(rows, n, scale=1.7).add_(normal(rows, 1, scale=0.3)).to(dt)
        s["o"] = normal(rows, n, scale=0.6).add_(normal(rows, 1, scale=0.2)).to(dt)
        s["gate_values"] = None
        if case["gate"] == "units":  # a learned scale of the block's part
            s["gate_values"] = normal(n, scale=0.3, mean=0.7).to(dt)
        elif case["gate"] == "values":
            s["gate_values"] = normal(rows, n).to(dt)
        for part in ("post", "pre"):
            used = part == "pre" or case["post"]
            s[part + "_weight"] = normal(n, scale=0.2, mean=1.0).to(dt) if used else None
            s[part + "_bias"] = normal(n, scale=0.2).to(dt) if used and case["kind"] == "layer" else None
        if case["train"]:
            s["dr"], s["du"] = normal(rows, n).to(dt), normal(rows, n).to(dt)
    else:
        streams, steps = case["streams"], case["steps"]
        rows = streams * steps
        s["x"] = normal(rows, n).to(dt)
        # units keep what they hold for one step to about a thousand
        slow = torch.empty(n, device="cuda").uniform_(0.0, 7.0, generator=g)
        gate = normal(rows, n).add_(slow)
        s["gate"] = (gate if case["kind"] == "sigmoid" else torch.sigmoid(gate)).to(dt)
        s["state"] = normal(streams, n)
        s["offsets"] = None
        if case["ragged"]:  # episodes of any length, empty ones among them, behind each other
            cuts = torch.randint(0, rows + 1, (streams - 1,), device="cuda", generator=g).sort().values
            ends = [cuts.new_zeros(1), cuts, cuts.new_full((1,), rows)]
            s["offsets"] = torch.cat(ends).int()
        else:
            s["x"], s["gate"] = s["x"].view(streams, steps, n), s["gate"].view(streams, steps, n)
        if case["train"]:
            s["dh"] = normal(rows, n).to(dt).view(s["x"].shape)
            s["dfinal"] = normal(streams, n)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _activate(z, apply):
    """(act(z), act'(z))"""
    if apply == "identity":
        return z, torch.ones_like(z)
    if apply == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).to(z.dtype)
    if apply == "tanh":
        t = torch.tanh(z)
        return t, 1 - t * t
    if apply == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * _SQRT_HALF))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    p = 1 / (1 + torch.exp(-z))
    if apply == "sigmoid":
        return p, p * (1 - p)
    return z * p, p * (1 + z * (1 - p))


def _plain_dense(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    y, slope = _activate(x @ w.t() + s["bias"].float(), s["apply"])
    if s["residual"]:
        y = y + s["residual_rows"].float()
    out = {"y": y.to(dt)}
    if s["train"]:
        dz = s["dy"].float() * slope
        out |= {"dx": (dz @ w).to(dt), "dweight": (dz.t() @ x).to(dt), "dbias": dz.sum(0).to(dt)}
    return out


def _normalised(v, kind):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS)
    return v * rstd, rstd


def _normalised_backward(d, h, rstd, kind):
    back = d - h * (d * h).mean(1, keepdim=True)
    if kind == "layer":
        back = back - d.mean(1, keepdim=True)
    return back * rstd


def _plain_block_norm(s):
    dt, kind = s["x"].dtype, s["kind"]
    wide = {k: None if s[k] is None else s[k].float()
            for k in ("gate_values", "post_weight", "post_bias", "pre_weight", "pre_bias")}
    p = s["o"].float()
    if s["post"]:
        h1, rstd1 = _normalised(p, kind)
        p = h1 * wide["post_weight"] + (wide["post_bias"] if kind == "layer" else 0.0)
    gate = slope = 1.0
    if s["gate"] != "none":
        gate = wide["gate_values"]
        if s["gate_apply"] == "sigmoid":
            gate, slope = _activate(gate, "sigmoid")
    r = s["scale"] * s["x"].float() + gate * p
    h2, rstd2 = _normalised(r, kind)
    u = h2 * wide["pre_weight"] + (wide["pre_bias"] if kind == "layer" else 0.0)
    out = {"r": r.to(dt), "u": u.to(dt)}
    if not s["train"]:
        return out
    du = s["du"].float()
    d = s["dr"].float() + _normalised_backward(du * wide["pre_weight"], h2, rstd2, kind)
    out |= {"dx": (s["scale"] * d).to(dt), "dpre_weight": (du * h2).sum(0).to(dt)}
    if kind == "layer":
        out["dpre_bias"] = du.sum(0).to(dt)
    if s["gate"] != "none":
        dgate = d * p * slope
        out["dgate"] = (dgate.sum(0) if s["gate"] == "units" else dgate).to(dt)
    dp = d * gate
    if s["post"]:
        out["dpost_weight"] = (dp * h1).sum(0).to(dt)
        if kind == "layer":
            out["dpost_bias"] = dp.sum(0).to(dt)
        dp = _normalised_backward(dp * wide["post_weight"], h1, rstd1, kind)
    out["do"] = dp.to(dt)
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 0, from 0: pairs of steps first, then what lies between."""
    steps = a.shape[0]
    if steps == 1:
        return b
    even = steps // 2 * 2
    a0, a1, b0, b1 = a[0:even:2], a[1:even:2], b[0:even:2], b[1:even:2]
    odd_h = _scan(a1 * a0, a1 * b0 + b1)
    h = torch.empty_like(b)
    h[1::2] = odd_h
    h[0] = b[0]
    h[2::2] = a[2::2] * odd_h[: (steps - 1) // 2] + b[2::2]
    return h


def _plain_recurrence(s):
    dt, n, shape = s["x"].dtype, s["n"], s["x"].shape
    x, gate = s["x"].float().view(-1, n), s["gate"].float().view(-1, n)
    rows, streams = x.shape[0], s["streams"]
    if s["offsets"] is not None:
        begin, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    else:
        begin = torch.arange(streams, device=x.device) * s["steps"]
        end = begin + s["steps"]
    # empty episodes take a row behind the last, which nothing reads
    first, last = torch.where(end > begin, begin, rows), torch.where(end > begin, end - 1, rows)
    a = 1 / (1 + torch.exp(-gate)) if s["kind"] == "sigmoid" else gate
    keep = 1 / (1 + torch.exp(gate)) if s["kind"] == "sigmoid" else 1 - a  # 1 - a
    b = keep * x if s["mix"] else x
    b = torch.cat([b, b.new_zeros(1, n)])
    cut = torch.cat([a, a.new_zeros(1, n)])
    held = cut[first] * s["state"]
    b[first] += held
    cut[first] = 0.0
    h = _scan(cut[:rows], b[:rows])
    final = torch.where((end > begin)[:, None], h[last.clamp(max=rows - 1)], s["state"])
    out = {"h": h.to(dt).view(shape), "final": final}
    if not s["train"]:
        return out
    # backwards: g_t = dh_t + a_{t+1} g_{t+1} within an episode
    dh = torch.cat([s["dh"].float().view(-1, n), b.new_zeros(1, n)])
    dh[last] += s["dfinal"]
    g = _scan(torch.cat([cut[:1], cut[1:rows].flip(0)]), dh[:rows].flip(0)).flip(0)
    before = torch.cat([h[:1], h])  # h_{t-1}
    before[first] = s["state"]
    before = before[:rows]
    da = g * (before - x if s["mix"] else before)
    out["dx"] = (keep * g if s["mix"] else g).to(dt).view(shape)
    out["dgate"] = (da * a * keep if s["kind"] == "sigmoid" else da).to(dt).view(shape)
    ag = torch.cat([a * g, g[:1]])
    out["dstate"] = torch.where((end > begin)[:, None], ag[first], s["dfinal"])
    return out


# ------------------------------------------------------------------------------ the framework's own
def _own(s):
    global _context
    from plastix_b200 import block
    from plastix_b200.runtime import Context

    device = s["x"].device
    if _context is None or _context.device != device:
        _context = Context(device.index)
    ctx = _context
    # a context works on one stream: here torch's current one (asked for by its handle, which is cheap)
    if torch._C._cuda_getCurrentRawStream(device.index) != ctx.stream.cuda_stream:
        ctx.use_stream(torch.cuda.current_stream(device))
    if s["op"] == "dense":
        if not s["train"]:
            return {"y": block.dense(ctx, s["x"], s["weight"], s["bias"], apply=s["apply"],
                                     residual=s["residual_rows"])}
        y, z = block.dense(ctx, s["x"], s["weight"], s["bias"], apply=s["apply"],
                           residual=s["residual_rows"], pre=True)
        dx, dw, db = block.dense_backward(ctx, s["dy"], s["x"], s["weight"], z, apply=s["apply"], bias=s["bias"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if s["op"] == "block_norm":
        how = {"kind": s["kind"], "gate_apply": s["gate_apply"], "scale": s["scale"], "post": s["post"],
               "post_weight": s["post_weight"], "post_bias": s["post_bias"],
               "pre_weight": s["pre_weight"], "pre_bias": s["pre_bias"]}
        if not s["train"]:
            r, u = block.block_norm(ctx, s["x"], s["o"], s["gate_values"], eps=_EPS, **how)
            return {"r": r, "u": u}
        r, u, stats = block.block_norm(ctx, s["x"], s["o"], s["gate_values"], eps=_EPS, stats=True, **how)
        d = block.block_norm_backward(ctx, s["dr"], s["du"], s["x"], s["o"], stats, s["gate_values"], **how)
        out = {"r": r, "u": u, "dx": d.dx, "do": d.do, "dgate": d.dgate,
               "dpost_weight": d.dpost_weight, "dpost_bias": d.dpost_bias,
               "dpre_weight": d.dpre_weight, "dpre_bias": d.dpre_bias}
        return {k: v for k, v in out.items() if v is not None}
    h, final = block.recurrence(ctx, s["x"], s["gate"], s["state"], kind=s["kind"], mix=s["mix"], offsets=s["offsets"])
    out = {"h": h, "final": final}
    if s["train"]:
        out["dx"], out["dgate"], out["dstate"] = block.recurrence_backward(
            ctx, s["dh"], s["gate"], h, s["state"], x=s["x"] if s["mix"] else None, dfinal=s["dfinal"],
            kind=s["kind"], mix=s["mix"], offsets=s["offsets"])
    return out


def run(state):
    if own:
        return _own(state)
    return {"dense": _plain_dense, "block_norm": _plain_block_norm,
            "recurrence": _plain_recurrence}[state["op"]](state)


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions in 64 bits: library activations and automatic differentiation, one step after the other."""
    s = prepare(case, seed)

    def wide(name):
        v = s.get(name)
        return None if v is None else v.double().requires_grad_(case["train"])

    def gradients(loss_of, of):
        """The gradients of sums of products with given tensors; the rows are freed as they go."""
        total = sum((v * d.double()).sum() for v, d in loss_of)
        used = {k: v for k, v in of.items() if v is not None}
        return dict(zip(used, torch.autograd.grad(total, list(used.values()))))

    if case["op"] == "dense":
        x, w, b = wide("x"), wide("weight"), wide("bias")
        library = {"identity": lambda z: z, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "relu": torch.relu,
                   "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[case["apply"]]
        y = library(torch.nn.functional.linear(x, w, b))
        if case["residual"]:
            y = y + s["residual_rows"].double()
        out = {"y": y.detach()}
        if case["train"]:
            out |= gradients([(y, s["dy"])], {"dx": x, "dweight": w, "dbias": b})
        return out
    if case["op"] == "block_norm":
        x, o, gate = wide("x"), wide("o"), wide("gate_values")
        w1, b1, w2, b2 = wide("post_weight"), wide("post_bias"), wide("pre_weight"), wide("pre_bias")

        def norm(v, w, b):
            if case["kind"] == "layer":
                return torch.nn.functional.layer_norm(v, (case["n"],), w, b, _EPS)
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + _EPS) * w

        p = norm(o, w1, b1) if case["post"] else o
        if gate is not None:
            p = p * (torch.sigmoid(gate) if case["gate_apply"] == "sigmoid" else gate)
        r = x * case["scale"] + p
        u = norm(r, w2, b2)
        out = {"r": r.detach(), "u": u.detach()}
        if case["train"]:
            out |= gradients([(r, s["dr"]), (u, s["du"])],
                             {"dx": x, "do": o, "dgate": gate, "dpost_weight": w1, "dpost_bias": b1,
                              "dpre_weight": w2, "dpre_bias": b2})
        return out
    n, shape = case["n"], s["x"].shape
    streams = case["streams"]
    # steps of all streams at once, or those of the episodes behind each other
    if case["ragged"]:
        at = s["offsets"].tolist()
        groups = [(slice(i, i + 1), at[i], at[i + 1], 1) for i in range(streams)]
    else:
        groups = [(slice(0, streams), 0, case["steps"], streams)]
    if sum(end - begin for _, begin, end, _ in groups) > 70000:
        return None

    def by_step(v):
        v = v.double()
        return v.view(-1, 1, n) if case["ragged"] else v.transpose(0, 1)

    x, gate = by_step(s["x"]), by_step(s["gate"])
    a = torch.sigmoid(gate) if case["kind"] == "sigmoid" else gate
    keep = 1 - a if case["kind"] == "decay" else torch.sigmoid(-gate)
    h, final = torch.empty_like(x), s["state"].double()
    was = torch.empty_like(x) if case["train"] else None
    for who, begin, end, _ in groups:
        now = final[who]
        for t in range(begin, end):
            if was is not None:
                was[t] = now
            now = a[t] * now + (keep[t] * x[t] if case["mix"] else x[t])
            h[t] = now
        final[who] = now
    back = (lambda v: v.reshape(shape)) if case["ragged"] else (lambda v: v.transpose(0, 1).reshape(shape))
    out = {"h": back(h), "final": final}
    if not case["train"]:
        return out
    dh, dstate = by_step(s["dh"]), s["dfinal"].double()
    g = torch.empty_like(h)
    for who, begin, end, _ in groups:
        now = dstate[who]
        for t in range(end - 1, begin - 1, -1):
            g[t] = dh[t] + now
            now = a[t] * g[t]
        dstate[who] = now
    da = g * (was - x) if case["mix"] else g * was
    out["dx"] = back(g * keep if case["mix"] else g)
    out["dgate"] = back(da * a * keep if case["kind"] == "sigmoid" else da)
    out["dstate"] = dstate
    return out
