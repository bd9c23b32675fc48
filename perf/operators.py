"""The read-out operators (layer norm, log probabilities, distillation) as cases to be measured.

Three operators in the order a network's read-out uses them: the last hidden layer is normalised
(``norm``), its output units are scored (``score``: log probability of a given output, entropy, best
alternatives) or trained against a teacher's best outputs (``distill``). ``run`` computes a case in
plain torch operations, or through ``plastix_b200.readout`` where ``own`` is true.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-5
_context = None


# ------------------------------------------------------------------------------------------ cases
def _norm(name, rows, n, dtype, train):
    return {"name": name, "op": "norm", "rows": rows, "n": n, "dtype": dtype, "train": train}


def _score(name, rows, n, dtype, top, entropy=True, train=False, scale=1.0, masked=0.0):
    return {"name": name, "op": "score", "rows": rows, "n": n, "dtype": dtype, "top": top,
            "entropy": entropy, "train": train, "scale": scale, "masked": masked}


def _distill(name, rows, n, dtype, k, train=True, tau=1.0, kind="logits", ragged=False):
    return {"name": name, "op": "distill", "rows": rows, "n": n, "dtype": dtype, "k": k,
            "train": train, "tau": tau, "kind": kind, "ragged": ragged}


def listed():
    return [
        # one step of sixteen streams through the normalisation: launch and latency count
        _norm("norm_step_16x1024_bf16", 16, 1024, "bf16", False),
        # evaluation of a large batch
        _norm("norm_eval_32768x4096_bf16", 32768, 4096, "bf16", False),
        # training in the framework's own type, sizes that no vector divides
        _norm("norm_train_3001x1001_f32", 3001, 1001, "f32", True),
        # training at full size, forward and backward
        _norm("norm_train_16384x4096_bf16", 16384, 4096, "bf16", True),
        # one step of eight answers: score what was chosen, five alternatives
        _score("score_step_8x32000_bf16", 8, 32000, "bf16", 5),
        # one long row: the whole device on a single answer
        _score("score_1x131072_f32", 1, 131072, "f32", 20),
        # scoring of a batch of sequences, as a teacher is run over a data set
        _score("score_4096x65536_bf16", 4096, 65536, "bf16", 8),
        # training on log probability and entropy: an odd number of outputs, a tenth of the rows with masked ones
        _score("score_train_1500x32003_f16", 1500, 32003, "f16", 0, train=True, scale=0.7, masked=0.3),
        # a small network's online distillation step
        _distill("distill_16x4096_f32", 16, 4096, "f32", 8),
        # lists of unequal length, rows that do not count, odd sizes
        _distill("distill_2047x20011_f16", 2047, 20011, "f16", 50, tau=2.0, ragged=True),
        # a training batch at full size
        _distill("distill_4096x65536_bf16", 4096, 65536, "bf16", 32, tau=2.0, kind="log_probs"),
        # the loss alone, on held-out rows
        _distill("distill_eval_1024x131072_bf16", 1024, 131072, "bf16", 64, train=False),
    ]


def _size(rng, low, high):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 128:  # half of the sizes are multiples of 64, as most layers' are
        v = v // 64 * 64
    return max(low, min(high, v))


def draw(rng):
    op = rng.choice(["norm", "score", "distill"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        n = _size(rng, 32, 8192)
        rows = _size(rng, 1, min(32768, (1 << (25 if dtype == "f32" else 26)) // n))
        c = _norm("", rows, n, dtype, rng.random() < 0.6)
    else:
        n = _size(rng, 256, 131072)
        rows = _size(rng, 1, min(4096, (1 << (26 if dtype == "f32" else 27)) // n))
        if op == "score":
            c = _score("", rows, n, dtype, rng.choice([0, 1, rng.randint(2, 64)]), rng.random() < 0.7,
                       rng.random() < 0.4, rng.choice([1.0, 0.5, 1.3]), rng.choice([0.0, 0.0, 0.5]))
        else:
            c = _distill("", rows, n, dtype, rng.randint(1, 64), rng.random() < 0.7, rng.choice([1.0, 2.0, 3.5]),
                         rng.choice(["logits", "log_probs"]), rng.random() < 0.5)
    del c["name"]
    return c


def work(case):
    rows, n = case["rows"], case["n"]
    cells, e = rows * n, {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] == "norm":
        nbytes, flops = 2 * cells * e + 2 * n * e, 8 * cells
        if case["train"]:  # backward: x and dy read, dx written; mean and rstd written and read; weight gradients
            nbytes, flops = nbytes + 3 * cells * e + 16 * rows + 3 * n * e, flops + 15 * cells
    elif case["op"] == "score":
        nbytes, flops = cells * e + rows * (12 + 4 * case["entropy"] + 8 * case["top"]), 6 * cells
        if case["train"]:
            nbytes, flops = nbytes + 2 * cells * e + 20 * rows, flops + 8 * cells
    else:
        nbytes, flops = cells * e + rows * (8 * case["k"] + 8), 5 * cells
        if case["train"]:
            nbytes, flops = nbytes + cells * e, flops + 5 * cells
    return {"bytes": nbytes, "flops": flops}


# ----------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, n, dt = case["rows"], case["n"], _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.empty(shape, device="cuda").normal_(0.0, scale, generator=g)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, device="cuda", generator=g, dtype=torch.int32)

    s = dict(case)
    if case["op"] == "norm":
        s["x"] = normal(rows, n, scale=1.7).add_(normal(rows, 1)).to(dt)
        s["w"] = normal(n, scale=0.2).add_(1.0).to(dt)
        s["b"] = normal(n, scale=0.2).to(dt)
        if case["train"]:
            s["dy"] = normal(rows, n).to(dt)
        return s
    x = normal(rows, n, scale=2.5)
    if case["op"] == "score":
        s["target"] = whole(0, n, rows)
        if case["masked"]:  # every tenth row: outputs that are not allowed there, and rows without a target
            part = x[::10]
            part.masked_fill_(torch.empty_like(part).uniform_(generator=g) < case["masked"], -math.inf)
            part.scatter_(1, s["target"][::10, None].long(), 1.0)
            s["target"][5::10] = -1
        if case["train"]:
            s["grad_logp"] = normal(rows)
            s["grad_entropy"] = normal(rows, scale=0.1) if case["entropy"] else None
    else:
        k = min(case["k"], n)
        first, apart = whole(0, n, rows, 1), n // k
        s["ids"] = ((first.long() + torch.arange(k, device="cuda") * apart) % n).int()
        t = normal(rows, k, scale=2.0).sort(dim=1, descending=True).values
        x.scatter_add_(1, s["ids"].long(), t + 4.0)  # the student has learnt something already
        if case["kind"] == "log_probs":  # what the teacher lists holds between half and all of its mass
            t = t - t.logsumexp(1, keepdim=True) + torch.empty_like(t[:, :1]).uniform_(0.5, 1.0, generator=g).log()
        # a mean over the rows; in f16 with the loss scaled up, as training in that type does it
        s["weight"] = torch.full((rows,), 2048.0 if case["dtype"] == "f16" else 1.0 / rows, device="cuda")
        if case["ragged"]:
            left = whole(1, k + 1, rows, 1)
            s["ids"].masked_fill_(torch.arange(k, device="cuda") >= left, -1)
            s["weight"][::7] = 0.0
        s["values"] = t.contiguous()
    s["x"] = x.to(dt)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(1, keepdim=True) + _EPS)
    h = xc * rstd
    y = (h * w + b).to(s["x"].dtype)
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].float()
    dh = dy * w
    dx = rstd * (dh - dh.mean(1, keepdim=True) - h * (dh * h).mean(1, keepdim=True))
    return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0], "dx": dx.to(s["x"].dtype),
            "dw": (dy * h).sum(0).to(s["w"].dtype), "db": dy.sum(0).to(s["w"].dtype)}


def _best(x, k):
    """The k largest of every row, the lower index first among equals: one sortable key for each value and its index."""
    bits = (x + 0.0).view(torch.int32)
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    at = torch.arange(x.shape[1], device=x.device)
    key = (order.long() << 32) + (0xFFFFFFFF - at)
    return (0xFFFFFFFF - (key.topk(k, dim=1).values & 0xFFFFFFFF)).int()


def _plain_score(s):
    x, scale = s["x"].float(), s["scale"]
    top = min(s["top"], s["n"])
    most = x.max(1, keepdim=True).values
    d = (x - most) * scale
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    has = s["target"] >= 0
    at = s["target"].clamp(min=0).long()[:, None]
    logp = torch.where(has, (d.gather(1, at) - log_total)[:, 0], 0.0)
    out = {"logp": logp, "lse": (scale * most + log_total)[:, 0]}
    if s["entropy"]:
        ed = torch.where(e > 0, e * d, 0.0)
        out["entropy"] = (log_total - ed.sum(1, keepdim=True) / total)[:, 0]
    if top:
        ids = _best(x, top)
        out["top_ids"] = ids
        out["top_logp"] = d.gather(1, ids.long()) - log_total
    if s["train"]:
        gl = torch.where(has, s["grad_logp"], 0.0)[:, None]
        p = e / total
        dx = -gl * p
        dx.scatter_add_(1, at, gl)
        if s["entropy"]:
            pl = torch.where(p > 0, p * (d - log_total + out["entropy"][:, None]), 0.0)
            dx = dx - s["grad_entropy"][:, None] * pl
        out["dx"] = (dx * scale).to(s["x"].dtype)
    return out


def _plain_distill(s):
    x, tau = s["x"].float(), s["tau"]
    given = s["ids"] >= 0
    at = s["ids"].clamp(min=0).long()
    t = s["values"] / tau if s["kind"] == "logits" else s["values"]
    t = torch.where(given, t, -math.inf)
    if s["kind"] == "logits":
        t = t - t.max(1, keepdim=True).values
        t = t - torch.log(torch.exp(t).sum(1, keepdim=True))
    q = torch.exp(t)
    d = (x - x.max(1, keepdim=True).values) / tau
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    logp = d.gather(1, at) - torch.log(total)
    w = s["weight"]
    out = {"loss": w * tau * tau * torch.where(given, q * (t - logp), 0.0).sum(1)}
    if s["train"]:
        grad = e / total * q.sum(1, keepdim=True)
        grad.scatter_add_(1, at, -q)
        out["dx"] = (grad * (w * tau)[:, None]).to(s["x"].dtype)
    return out


# ------------------------------------------------------------------------------ the framework's own
def _own(s):
    global _context
    from plastix_b200 import readout
    from plastix_b200.runtime import Context

    device = s["x"].device
    if _context is None or _context.device != device:
        _context = Context(device.index)
    ctx = _context
    # a context works on one stream: here torch's current one (asked for by its handle, which is cheap)
    if torch._C._cuda_getCurrentRawStream(device.index) != ctx.stream.cuda_stream:
        ctx.use_stream(torch.cuda.current_stream(device))
    if s["op"] == "norm":
        if not s["train"]:
            return {"y": readout.layer_norm(ctx, s["x"], s["w"], s["b"], eps=_EPS)}
        y, mean, rstd = readout.layer_norm(ctx, s["x"], s["w"], s["b"], eps=_EPS, stats=True)
        dx, dw, db = readout.layer_norm_backward(ctx, s["dy"], s["x"], mean, rstd, s["w"])
        return {"y": y, "mean": mean, "rstd": rstd, "dx": dx, "dw": dw, "db": db}
    if s["op"] == "score":
        top = min(s["top"], s["n"])
        r = readout.log_probs(ctx, s["x"], s["target"], top=top, scale=s["scale"], entropy=s["entropy"])
        out = {"logp": r.logp, "lse": r.lse}
        if s["entropy"]:
            out["entropy"] = r.entropy
        if top:
            out["top_ids"], out["top_logp"] = r.top_ids, r.top_logp
        if s["train"]:
            out["dx"] = readout.log_probs_backward(ctx, s["x"], r.lse, s["target"], s["grad_logp"], r.entropy,
                                                   s["grad_entropy"], scale=s["scale"])
        return out
    loss, dx = readout.distill(ctx, s["x"], s["ids"], s["values"], temperature=s["tau"], kind=s["kind"],
                               weight=s["weight"], grad=s["train"])
    return {"loss": loss, "dx": dx} if s["train"] else {"loss": loss}


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "score": _plain_score, "distill": _plain_distill}[state["op"]](state)


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions in 64 bits: library softmax and sort, derivatives of the losses by hand."""
    s = prepare(case, seed)
    x = s["x"].double()
    if case["op"] == "norm":
        w, b = s["w"].double(), s["b"].double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        sd = torch.sqrt(var + _EPS)
        y = w * (x - mean) / sd + b
        if not case["train"]:
            return {"y": y}
        dy = s["dy"].double()
        # dL/dx through x - mean and through the deviation, each by the chain rule
        up = dy * w / sd
        through_sd = -(dy * w * (x - mean)).sum(1, keepdim=True) / sd ** 2
        dx = up - up.mean(1, keepdim=True) + through_sd * (x - mean) / (case["n"] * sd)
        return {"y": y, "mean": mean[:, 0], "rstd": 1 / sd[:, 0], "dx": dx,
                "dw": (dy * (x - mean) / sd).sum(0), "db": dy.sum(0)}
    if case["op"] == "score":
        z = x * case["scale"]
        logs = torch.log_softmax(z, 1)
        p = logs.exp()
        has = s["target"] >= 0
        at = s["target"].clamp(min=0).long()
        out = {"logp": torch.where(has, logs[torch.arange(len(x), device=x.device), at], 0.0),
               "lse": torch.logsumexp(z, 1)}
        surprise = torch.where(p > 0, -p * logs, 0.0).sum(1)
        if case["entropy"]:
            out["entropy"] = surprise
        top = min(case["top"], case["n"])
        if top:
            best, ids = torch.sort(logs, dim=1, descending=True, stable=True)
            out["top_ids"], out["top_logp"] = None, best[:, :top].contiguous()
            del best, ids
        if case["train"]:
            gl = torch.where(has, s["grad_logp"].double(), 0.0)
            hot = torch.zeros_like(p)
            hot[torch.arange(len(x), device=x.device), at] = gl
            dx = hot - gl[:, None] * p
            if case["entropy"]:
                inner = torch.where(p > 0, p * logs, 0.0) + p * surprise[:, None]
                dx -= s["grad_entropy"].double()[:, None] * inner
            out["dx"] = dx * case["scale"]
        return out
    tau = case["tau"]
    logs = torch.log_softmax(x / tau, 1)
    given = s["ids"] >= 0
    at = s["ids"].clamp(min=0).long()
    t = torch.where(given, s["values"].double(), -math.inf)
    logq = torch.log_softmax(t / tau, 1) if case["kind"] == "logits" else t
    q = logq.exp()
    w = s["weight"].double() * tau
    out = {"loss": w * tau * torch.where(q > 0, q * (logq - logs.gather(1, at)), 0.0).sum(1)}
    if case["train"]:
        out["dx"] = w[:, None] * (logs.exp() * q.sum(1, keepdim=True)).scatter_add(1, at, -q)
    return out
