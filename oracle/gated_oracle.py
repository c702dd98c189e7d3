"""Float64 restatement of the gated linear recurrence, its gradients, and a running bound of the
float32 kernels' rounding errors (test infrastructure).

    log a_t = -exp(nu_log) s(r_t),  h_t = c_t h_{t-1} + sqrt(1 - a_t^2) s(w_t) x_t,  c_t = a_t or 0 at a segment start
"""
import numpy as np

U = 2.0 ** -24  # half a float32 step


def _sigmoid(v):
    return np.where(v >= 0, 1.0 / (1.0 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1.0 + np.exp(-np.abs(v))))


def _parts(r, w, nu_log, starts):
    with np.errstate(over="ignore"):
        u = -np.exp(nu_log) * _sigmoid(r)
    a = np.exp(u)
    beta = np.sqrt(-np.expm1(2.0 * u))
    c = a if starts is None else np.where(starts[..., None], 0.0, a)
    return u, a, beta, c, _sigmoid(w)


def _drop(c, v, t, starts):
    """c_t v, exactly zero where token t starts a segment (whatever v is)."""
    o = c[:, t] * v
    return o if starts is None else np.where(starts[:, t, None], 0.0, o)


def forward(x, r, w, nu_log, h0=None, starts=None):
    """(h [B, T, D], last [B, D])."""
    u, a, beta, c, sw = _parts(r, w, nu_log, starts)
    h = np.zeros_like(x)
    s = np.zeros(x[:, 0].shape) if h0 is None else h0
    for t in range(x.shape[1]):
        s = _drop(c, s, t, starts) + (beta * sw * x)[:, t]
        h[:, t] = s
    return h, s


def backward(x, r, w, nu_log, dy, h0=None, starts=None, dlast=None):
    """Gradients: dict x, r, w, nu_log, h0."""
    u, a, beta, c, sw = _parts(r, w, nu_log, starts)
    h, _ = forward(x, r, w, nu_log, h0, starts)
    T = x.shape[1]
    lam = np.zeros_like(x)
    v = np.zeros(x[:, 0].shape) if dlast is None else dlast
    for t in range(T - 1, -1, -1):
        lam[:, t] = dy[:, t] + v
        v = _drop(c, lam[:, t], t, starts)
    before = np.concatenate([(np.zeros_like(x[:, 0]) if h0 is None else h0)[:, None], h[:, :-1]], axis=1)
    if starts is not None:
        before = np.where(starts[..., None], 0.0, before)
    dx = lam * beta * sw
    # u a^2 / sqrt(1 - a^2) -> 0 with u
    ub = np.where(u == 0.0, 0.0, u / np.where(beta == 0.0, 1.0, beta))
    du = lam * (c * before * u - x * sw * a * a * ub)
    return dict(x=dx, r=du * _sigmoid(-r), w=dx * x * _sigmoid(-w), nu_log=du.sum(axis=(0, 1)), h0=v)


def bounds(x, r, w, nu_log, dy=None, h0=None, starts=None, dlast=None):
    """Bounds of the float32 kernels' absolute errors before the final rounding to the outputs' type.

    Relative errors, in units of 2^-24, of what the kernels form per token: a hardware exp2 is off
    by 4, a reciprocal, square root or inverse square root by 2 to 3, an operation by 1, and the
    argument of e^{-v} by |v| in the bfloat16 kernels (gates up to 8 in magnitude: 8). So a
    logistic value is off by 8 + 4 + 2 + 1 = 15 and u by 16. a = e^u: 16 |u| from u, |u| + 4 from
    its own exp2, 1 to round. a - 1: 16 + 3 by the series, and at most 16 + 6 a / (1 - a) <= 26
    where u < -1/2 by exp2; its square root half of that, so sqrt(1 - a^2) s(w) x is off by 13 + 3
    + 15 + 3 = 34. The states then carry their errors along: E_t = c_t E_{t-1} + (error of c_t)
    |h|_{t-1} + (error of b_t) + 4 roundings of |h|_t (the recurrence's own and those of the composed
    maps), with |h| the recurrence of absolute values; the adjoints likewise."""
    u, a, beta, c, sw = _parts(r, w, nu_log, starts)
    da, db = (17.0 * np.abs(u) + 6.0) * U, 34.0 * U
    B, T, D = x.shape
    b = beta * sw * np.abs(x)
    mag, err = np.zeros_like(x), np.zeros_like(x)
    m, e = (np.zeros((B, D)) if h0 is None else np.abs(h0)), np.zeros((B, D))
    m0 = m
    for t in range(T):
        ca = c[:, t] * (1.0 + da[:, t])
        e = ca * e + c[:, t] * m * da[:, t] + b[:, t] * db
        m = c[:, t] * m + b[:, t]
        e = e + 4.0 * U * m
        mag[:, t], err[:, t] = m, e
    out = dict(h=err, last=e)
    if dy is None:
        return out
    lmag, lerr = np.zeros_like(x), np.zeros_like(x)
    m, e = (np.zeros((B, D)) if dlast is None else np.abs(dlast)), np.zeros((B, D))
    for t in range(T - 1, -1, -1):
        m = np.abs(dy[:, t]) + m
        e = e + 4.0 * U * m
        lmag[:, t], lerr[:, t] = m, e
        e = c[:, t] * (1.0 + da[:, t]) * e + c[:, t] * m * da[:, t]
        m = c[:, t] * m
    g = beta * sw
    out["x"] = lerr * g + lmag * g * db
    # 1 - s(w) = e s: off by 12 + 15 + 1
    out["w"] = (lerr * b + lmag * b * (db + 30.0 * U)) * _sigmoid(-w)
    before = np.concatenate([m0[:, None], mag[:, :-1]], axis=1)
    berr = np.concatenate([np.zeros((B, 1, D)), err[:, :-1]], axis=1)
    ub = np.abs(u) / np.where(beta == 0.0, 1.0, beta)
    q1, q2 = c * np.abs(u), sw * np.abs(x) * a * a * ub
    # q1: u 16, a; q2: s(w) 15, a^2 twice a's, u 16, its square root 13 + 3, products
    eq = q1 * berr + q1 * before * (da + 18.0 * U) + q2 * (2.0 * da + 52.0 * U)
    du = lerr * (q1 * before + q2) + lmag * (eq + 2.0 * U * (q1 * before + q2))
    out["r"] = (du + lmag * (q1 * before + q2) * 30.0 * U) * _sigmoid(-r)
    out["nu_log"] = du.sum(axis=(0, 1)) + 4.0 * U * (lmag * (q1 * before + q2)).sum(axis=(0, 1))
    out["h0"] = e
    return out
