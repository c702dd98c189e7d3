"""The operators a trained stack of recurrent layers needs around its mixers, as cases that can be
timed and checked: the gated linear recurrence (forward, forward with backward, one decode step),
layer norm (forward, forward with backward) and the clipping of gradients by their global norm.

`run` computes a case in its plain form (elementary torch operations in float32, rounded once at
the end) or, with `own` set, by this package's operators; `exact` computes it in float64 from the
definitions.

Gated linear recurrence, per batch row and channel, with sigma the logistic function:
    log a_t = -exp(nu_log) sigma(retention_t)
    h_t     = a_t h_{t-1} + sqrt(1 - a_t^2) sigma(write_t) x_t          (a_t -> 0 where t starts a segment)
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
ELEMENTS = 8 * 16384 * 2048  # the most activations of one tensor: the largest layer configuration
GRADIENTS = 4 * 4 * 4096 * 2048 + 1000000  # the most gradient values


def listed():
    return [
        # one user's token through a narrow layer: nothing but latency
        dict(name="step_b1_w512_f32", op="step", batch=1, width=512, dtype="float32", packed=False),
        # the decode configuration's batch and width, some rows starting a new sequence
        dict(name="step_b256_w2048_bf16", op="step", batch=256, width=2048, dtype="bfloat16", packed=True),
        # a prompt of one user, the gates and the input as columns of one projection: few rows, a long axis
        dict(name="prefill_b1_t16384_w2048_bf16", op="scan", batch=1, length=16384, width=2048, dtype="bfloat16",
             packed=False, state=False, split=True, train=False),
        # a training step of the default layer configuration
        dict(name="train_b8_t2048_w512_f32", op="scan", batch=8, length=2048, width=512, dtype="float32",
             packed=False, state=False, split=False, train=True),
        # a training step of the largest layer configuration
        dict(name="train_b8_t16384_w2048_bf16", op="scan", batch=8, length=16384, width=2048, dtype="bfloat16",
             packed=False, state=False, split=False, train=True),
        # packed documents of odd lengths, continued from a carried state (truncated backpropagation)
        dict(name="train_packed_b3_t1021_w777_bf16", op="scan", batch=3, length=1021, width=777, dtype="bfloat16",
             packed=True, state=True, split=False, train=True),
        # layer norm of a decode batch
        dict(name="norm_64x2048_bf16", op="norm", rows=64, width=2048, dtype="bfloat16", bias=True, train=False),
        # layer norm in a training step: the default layer's tokens, the largest layer's, odd sizes
        dict(name="norm_train_16384x512_f32", op="norm", rows=16384, width=512, dtype="float32", bias=True, train=True),
        dict(name="norm_train_131072x2048_bf16", op="norm", rows=131072, width=2048, dtype="bfloat16", bias=True,
             train=True),
        dict(name="norm_train_1021x777_bf16", op="norm", rows=1021, width=777, dtype="bfloat16", bias=False, train=True),
        # the gradients of four mixer layers: many short vectors
        dict(name="clip_mixers_4x2048_f32", op="clip", layers=4, width=2048, matrices=0, dtype="float32", max_norm=1.0),
        # the gradients of four projection layers: matrices and vectors, more than the caches hold
        dict(name="clip_projections_4x4096_f32", op="clip", layers=4, width=4096, matrices=4, dtype="float32",
             max_norm=1.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("step", "scan", "scan", "scan", "norm", "norm", "clip"))
    dtype = rng.choice(tuple(DTYPES))
    if op == "step":
        return dict(op=op, batch=_log_int(rng, 1, 1024), width=_log_int(rng, 1, 8192), dtype=dtype,
                    packed=rng.random() < 0.5)
    if op == "scan":
        while True:
            b, t, w = _log_int(rng, 1, 64), _log_int(rng, 1, 32768), _log_int(rng, 1, 8192)
            if 256 <= b * t * w <= ELEMENTS // (2 if dtype == "float32" else 1):
                break
        return dict(op=op, batch=b, length=t, width=w, dtype=dtype, packed=rng.random() < 0.5,
                    state=rng.random() < 0.5, split=rng.random() < 0.3, train=rng.random() < 0.7)
    if op == "norm":
        while True:
            r, w = _log_int(rng, 1, 262144), _log_int(rng, 8, 16384)
            if r * w <= ELEMENTS // (2 if dtype == "float32" else 1):
                break
        return dict(op=op, rows=r, width=w, dtype=dtype, bias=rng.random() < 0.7, train=rng.random() < 0.7)
    while True:
        layers, w, m = _log_int(rng, 1, 6), 2 * _log_int(rng, 8, 4096), rng.choice((0, 1, 2, 4))
        if layers * (10 + m) < 64 and layers * (m * w * (w // 2) + 7 * w) <= GRADIENTS:
            break
    return dict(op=op, layers=layers, width=w, matrices=m, dtype=dtype, max_norm=rng.choice((0.5, 1.0, 1.0e6)))


def _gradient_shapes(case):
    """The parameters of the framework's layers: seven vectors of half the width, two of the
    width + 1, the norm's weight, and in projection layers the content and readout matrices."""
    w = case["width"]
    layer = [(w // 2,)] * 7 + [(w + 1,)] * 2 + [(w,)] + [(w, w // 2)] * case["matrices"]
    return layer * case["layers"]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        out = torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, 1.0, generator=g)
        return out if scale == 1.0 and shift == 0.0 else out.mul_(scale).add_(shift)

    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "clip":
        shapes = _gradient_shapes(case)
        # each parameter has its own scale, as gradients of gains, directions and matrices do
        scales = torch.empty(len(shapes), device="cuda").uniform_(-9.0, -2.0, generator=g).exp_().tolist()
        state["grads"] = [normal(*s, dtype=dtype, scale=k) for s, k in zip(shapes, scales)]
        state["out"] = [torch.empty_like(t) for t in state["grads"]]
        return state
    w = case["width"]
    if case["op"] == "norm":
        # features with their own means and spreads, as in a residual stream
        centre, spread = normal(w, scale=0.3), normal(w, scale=0.3).exp_()
        x = normal(case["rows"], w, dtype=dtype)
        state["x"] = x.mul_(spread.to(dtype)).add_(centre.to(dtype))
        state["weight"] = normal(w, scale=0.2, shift=1.0)
        state["bias"] = normal(w, scale=0.2) if case["bias"] else None
        if case["train"]:
            state["dy"] = normal(case["rows"], w, dtype=dtype)
            for name in ("x", "weight", "bias"):
                if state[name] is not None:
                    state[name].requires_grad_(True)
        return state
    b = case["batch"]
    tokens = (b,) if case["op"] == "step" else (b, case["length"])
    if case.get("split"):  # one projection's columns: x, the retention gate, the write gate
        p = normal(*tokens, 3 * w, dtype=dtype)
        state["x"], state["retention"], state["write"] = p.split(w, dim=-1)
    else:
        for name in ("x", "retention", "write"):
            state[name] = normal(*tokens, w, dtype=dtype)
    # exp(-exp(nu_log)), the least a_t, between 0.9 and 0.999
    state["nu_log"] = torch.empty(w, device="cuda").uniform_(0.9, 0.999, generator=g).log_().neg_().log_()
    state["state"] = normal(b, w) if case["op"] == "step" or case["state"] else None
    state["segment_pos"] = None
    if case["packed"]:
        # positions within a segment; a new one starts at about every 200th token, and in a step in every tenth row
        starts = torch.rand(tokens, generator=g, device="cuda") < (0.1 if case["op"] == "step" else 0.005)
        if case["op"] == "step":
            state["segment_pos"] = torch.where(starts, 0, 100)
        else:
            at = torch.arange(case["length"], device="cuda").expand(tokens)
            last = torch.where(starts, at, -1).cummax(dim=1).values
            state["segment_pos"] = torch.where(last < 0, at + 100, at - last)
    if case.get("train"):
        state["dy"] = normal(*tokens, w, dtype=dtype)
        state["dlast"] = normal(b, w)
        for name in ("x", "retention", "write", "nu_log", "state"):
            if state[name] is not None:
                state[name] = state[name].detach().requires_grad_(True)
    return state


# ------------------------------------------------------------------ the plain forms (float32)

def _gates(s):
    """x, sigma(retention), sigma(write), log a, a, sqrt(1 - a^2) in float32."""
    x = s["x"].detach().float()
    keep = 1.0 / (1.0 + torch.exp(-s["retention"].detach().float()))
    write = 1.0 / (1.0 + torch.exp(-s["write"].detach().float()))
    log_a = -torch.exp(s["nu_log"].detach()) * keep
    a = torch.exp(log_a)
    return x, keep, write, log_a, a, torch.sqrt(-torch.expm1(2.0 * log_a))


def _prefix(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from zero, in place of b, by doubling spans (a is lost)."""
    d = 1
    while d < a.shape[1]:
        b[:, d:] += a[:, d:] * b[:, :-d]
        a[:, d:] = a[:, d:] * a[:, :-d]
        d *= 2
    return b


def _plain_scan(s):
    x, keep, write, log_a, a, beta = _gates(s)
    carried = a if s["segment_pos"] is None else a * (s["segment_pos"] != 0).unsqueeze(-1)
    b = beta * write * x
    if s["state"] is not None:
        b[:, 0] += carried[:, 0] * s["state"].detach()
    h = _prefix(carried.clone(), b)
    if not s["train"]:
        return h.to(s["x"].dtype), h[:, -1].clone()
    # the adjoint lambda_t = dy_t + a_{t+1} lambda_{t+1}: the same recurrence on the reversed axis
    dy = s["dy"].float()
    dy[:, -1] += s["dlast"]
    behind = torch.zeros_like(a)
    behind[:, 1:] = carried.flip(1)[:, :-1]
    adj = _prefix(behind, dy.flip(1)).flip(1)
    before = torch.zeros_like(h)
    before[:, 1:] = h[:, :-1]
    if s["state"] is not None:
        before[:, 0] = s["state"].detach()
    dx = adj * beta * write
    dwrite = dx * x * (1.0 - write)
    # d log a: through the carried state, and through sqrt(1 - a^2), whose slope is -a^2 / sqrt(1 - a^2)
    part = adj * (carried * before * log_a - write * x * a * a * (log_a / beta))
    t = s["x"].dtype
    out = [h.to(t), h[:, -1].clone(), dx.to(t), (part * (1.0 - keep)).to(t), dwrite.to(t),
           part.sum(dim=(0, 1), dtype=torch.float64).float()]
    if s["state"] is not None:
        out.append(carried[:, 0] * adj[:, 0])
    return out


def _plain_step(s):
    x, keep, write, log_a, a, beta = _gates(s)
    if s["segment_pos"] is not None:
        a = a * (s["segment_pos"] != 0).unsqueeze(-1)
    h = a * s["state"] + beta * write * x
    return h.to(s["x"].dtype), h


def _plain_norm(s):
    x, weight = s["x"].detach().float(), s["weight"].detach()
    centred = x - x.mean(dim=1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + 1e-5)
    n = centred * rstd
    y = n * weight
    if s["bias"] is not None:
        y = y + s["bias"].detach()
    if not s["train"]:
        return y.to(s["x"].dtype)
    dy = s["dy"].float()
    dn = dy * weight
    dx = rstd * (dn - dn.mean(dim=1, keepdim=True) - n * (dn * n).mean(dim=1, keepdim=True))
    out = [y.to(s["x"].dtype), dx.to(s["x"].dtype), (dy * n).sum(dim=0, dtype=torch.float64).float()]
    if s["bias"] is not None:
        out.append(dy.sum(dim=0, dtype=torch.float64).float())
    return out


def _plain_clip(s):
    squares = torch.stack([g.float().square().sum(dtype=torch.float64) for g in s["grads"]])
    norm = torch.sqrt(squares.sum()).float()
    scale = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    return [norm] + [(g.float() * scale).to(g.dtype) for g in s["grads"]]


def _own(s):
    import sparc_b200

    if s["op"] == "clip":
        norm = sparc_b200.clip_grads(s["grads"], s["max_norm"], out=s["out"])
        return [norm] + s["out"]
    if s["op"] == "norm":
        y = sparc_b200.layer_norm(s["x"], s["weight"], s["bias"], eps=1e-5)
        if not s["train"]:
            return y
        leaves = [s["x"], s["weight"]] + ([] if s["bias"] is None else [s["bias"]])
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
    if s["op"] == "step":
        return sparc_b200.gated_scan_step(s["x"], s["retention"], s["write"], s["nu_log"], s["state"],
                                          segment_pos=s["segment_pos"])
    y, last = sparc_b200.gated_scan(s["x"], s["retention"], s["write"], s["nu_log"], state=s["state"],
                                    segment_pos=s["segment_pos"], return_last=True)
    if not s["train"]:
        return y, last
    leaves = [s[k] for k in ("x", "retention", "write", "nu_log", "state") if s[k] is not None]
    out = [y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (s["dy"], s["dlast"]))]
    if s["dy"].dtype == torch.float32:
        # the plain form adds the last state's gradient to a float32 dy where it lies; so does this, behind
        # the calls, so that both sides are given the same dy on every pass over a state
        s["dy"][:, -1] += s["dlast"]
    return out


def run(state):
    if own:
        return _own(state)
    return {"clip": _plain_clip, "norm": _plain_norm, "step": _plain_step, "scan": _plain_scan}[state["op"]](state)


# ------------------------------------------------------------------ the definitions in float64

def _exact_scan(s):
    f = torch.float64
    x, r, w = (s[k].detach().to(f) for k in ("x", "retention", "write"))
    if s["op"] == "step":
        x, r, w = x[:, None], r[:, None], w[:, None]
    B, T, D = x.shape
    nu = s["nu_log"].detach().to(f).exp()
    sr, sw = torch.sigmoid(r), torch.sigmoid(w)
    closed_r = torch.sigmoid(-r)
    del r
    u = -nu * sr
    a, gain = torch.exp(u), (-torch.expm1(2 * u)).sqrt()
    go = a
    if s["segment_pos"] is not None:
        go = a.masked_fill((s["segment_pos"] == 0).view(B, T, 1), 0.0)
    b = gain * sw * x
    h0 = torch.zeros(B, D, dtype=f, device=x.device) if s["state"] is None else s["state"].detach().to(f)
    hs = torch.empty(B, T + 1, D, dtype=f, device=x.device)
    hs[:, 0] = h0
    for t in range(T):
        torch.addcmul(b[:, t], go[:, t], hs[:, t], out=hs[:, t + 1])
    del b
    if s["op"] == "step":
        return hs[:, 1], hs[:, 1]
    if not s["train"]:
        return hs[:, 1:], hs[:, -1]
    adj = s["dy"].to(f)
    adj[:, -1] += s["dlast"].to(f)
    for t in range(T - 2, -1, -1):
        adj[:, t].addcmul_(go[:, t + 1], adj[:, t + 1])
    dx = adj * gain * sw
    dw = adj * gain * x * sw * torch.sigmoid(-s["write"].detach().to(f))
    du = adj * (go * hs[:, :-1] - sw * x * a * a / gain) * u
    out = [hs[:, 1:], hs[:, -1], dx, du * closed_r, dw, du.sum(dim=(0, 1))]
    if s["state"] is not None:
        out.append(go[:, 0] * adj[:, 0])
    return out


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.to(f)) for g in s["grads"]]))
        factor = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
        return [norm] + [g.to(f) * factor for g in s["grads"]]
    if case["op"] in ("scan", "step"):
        return _exact_scan(s)
    x = s["x"].detach().to(f).requires_grad_(case["train"])
    weight = s["weight"].detach().to(f).requires_grad_(case["train"])
    bias = None if s["bias"] is None else s["bias"].detach().to(f).requires_grad_(case["train"])
    y = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * weight
    y = y if bias is None else y + bias
    if not case["train"]:
        return y
    leaves = [x, weight] + ([] if bias is None else [bias])
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"].to(f))]


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "clip":
        n = sum(math.prod(s) for s in _gradient_shapes(case))
        return {"bytes": 2 * n * size + 4, "flops": 3 * n}
    w = case["width"]
    if case["op"] == "norm":
        n, rows, params = case["rows"] * w, case["rows"], 2 if case["bias"] else 1
        if case["train"]:
            return {"bytes": 4 * n * size + 2 * params * w * 4, "flops": 21 * n}
        return {"bytes": 2 * n * size + params * w * 4, "flops": 8 * n}
    rows = case["batch"] * w
    if case["op"] == "step":
        return {"bytes": 4 * rows * size + 2 * rows * 4 + w * 4 + (8 * case["batch"] if case["packed"] else 0),
                "flops": 20 * rows}
    n = rows * case["length"]
    small = w * 4 + rows * 4 * (2 if case["state"] else 1) + (8 * case["batch"] * case["length"] if case["packed"] else 0)
    if case["train"]:  # in: x, two gates, dy; out: y and the gradients of x and the gates
        return {"bytes": 8 * n * size + small + w * 4 + rows * 4 * (2 if case["state"] else 1), "flops": 50 * n}
    return {"bytes": 4 * n * size + small, "flops": 20 * n}
