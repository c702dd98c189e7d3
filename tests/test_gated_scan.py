"""The gated linear recurrence without a GPU: the oracle's gradients against differences, and the
refusals of the Python functions and of the C entry points (no pointer passed is dereferenced)."""
import ctypes

import numpy as np
import pytest
import torch

import sparc_b200
from oracle import gated_oracle as G
from sparc_b200 import _lib

ARG, SHAPE, DTYPE, WORKSPACE = -1, -2, -3, -4
FAKE = 0x100000


@pytest.fixture(scope="module")
def L():
    return _lib.load_library()


@pytest.fixture(scope="module", autouse=True)
def built():
    from sparc_b200 import _build

    _build.build()
    _build.build_torch_ops()


def _message(L):
    return L.sparc_last_error().decode()


# ------------------------------------------------------------------ the oracle

@pytest.mark.parametrize("with_state,with_starts", [(False, False), (True, False), (True, True)])
def test_oracle_gradients_match_differences(with_state, with_starts):
    """Central differences in float64: the truncation is h^2 / 6 times the third derivative, the
    rounding 2^-53 / h; with h = 1e-5 both are below 1e-9 of values near 1."""
    rng = np.random.default_rng(0)
    B, T, D = 2, 7, 3
    p = dict(x=rng.standard_normal((B, T, D)), r=rng.standard_normal((B, T, D)), w=rng.standard_normal((B, T, D)),
             nu_log=rng.uniform(-3, 0, D), h0=rng.standard_normal((B, D)))
    starts = rng.random((B, T)) < 0.3 if with_starts else None
    dy, dlast = rng.standard_normal((B, T, D)), rng.standard_normal((B, D))

    def loss(q):
        h, last = G.forward(q["x"], q["r"], q["w"], q["nu_log"], q["h0"] if with_state else None, starts)
        return (h * dy).sum() + (last * dlast).sum()

    grads = G.backward(p["x"], p["r"], p["w"], p["nu_log"], dy, p["h0"] if with_state else None, starts, dlast)
    for name in p if with_state else ("x", "r", "w", "nu_log"):
        for i in np.ndindex(p[name].shape):
            hi, lo = ({k: v.copy() for k, v in p.items()} for _ in range(2))
            hi[name][i] += 1e-5
            lo[name][i] -= 1e-5
            d = (loss(hi) - loss(lo)) / 2e-5
            assert abs(d - grads[name][i]) < 1e-7, (name, i)


def test_oracle_drops_what_came_before_a_segment():
    x = np.ones((1, 4, 1))
    x[0, 1] = np.nan
    z = np.zeros((1, 4, 1))
    starts = np.array([[False, False, True, False]])
    h, _ = G.forward(x, z, z, np.zeros(1), None, starts)
    assert np.isnan(h[0, 1, 0]) and np.isfinite(h[0, 2:]).all()


# ------------------------------------------------------------------ Python refusals

def _args(B=2, T=3, D=4, dtype=torch.float32):
    return [torch.zeros(B, T, D, dtype=dtype) for _ in range(3)] + [torch.zeros(D)]


def test_scan_refusals():
    f = sparc_b200.gated_scan
    x, r, w, nu = _args()
    with pytest.raises(ValueError, match="one shape"):
        f(x, r[:, :2], w, nu)
    with pytest.raises(ValueError, match="one shape"):
        f(x[0], r[0], w[0], nu)
    with pytest.raises(ValueError, match=r"nu_log must have shape \[channels\]"):
        f(x, r, w, nu[:3])
    with pytest.raises(ValueError, match=r"state must have shape \[batch, channels\]"):
        f(x, r, w, nu, state=torch.zeros(2, 3))
    with pytest.raises(ValueError, match="segment_pos must have shape"):
        f(x, r, w, nu, segment_pos=torch.zeros(2, 4, dtype=torch.long))
    for shape in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        with pytest.raises(ValueError, match="at least one"):
            f(*_args(*shape))
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        f(*_args(dtype=torch.float16))
    with pytest.raises(TypeError, match="one dtype"):
        f(x, r.bfloat16(), w, nu)
    with pytest.raises(TypeError, match="integer tensor"):
        f(x, r, w, nu, segment_pos=torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x, r, w, nu)


def test_step_refusals():
    f = sparc_b200.gated_scan_step
    x, r, w, nu = (t[:, 0] if t.dim() == 3 else t for t in _args())
    s = torch.zeros(2, 4)
    with pytest.raises(ValueError, match="one shape"):
        f(x, r[:1], w, nu, s)
    with pytest.raises(ValueError, match="one shape"):
        f(x[:, None], r[:, None], w[:, None], nu, s)
    with pytest.raises(ValueError, match="state must have shape"):
        f(x, r, w, nu, s[:1])
    with pytest.raises(ValueError, match="segment_pos must have shape"):
        f(x, r, w, nu, s, segment_pos=torch.zeros(3, dtype=torch.long))
    with pytest.raises(TypeError):
        f(x.double(), r.double(), w.double(), nu, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x, r, w, nu, s)


# ------------------------------------------------------------------ C refusals

def _fwd(**kw):
    a = _lib.GatedFwdArgs()
    for n in ("x", "retention_gate", "write_gate", "nu_log", "y"):
        setattr(a, n, FAKE)
    a.batch, a.length, a.channels, a.dtype = 2, 3, 4, 0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _bwd(L, **kw):
    a = _lib.GatedBwdArgs()
    for n in ("x", "retention_gate", "write_gate", "nu_log", "dy", "carry", "grad_x", "grad_retention_gate",
              "grad_write_gate", "grad_nu_log", "workspace"):
        setattr(a, n, FAKE)
    a.batch, a.length, a.channels, a.dtype = 2, 3, 4, 0
    a.workspace_bytes = L.sparc_gated_workspace_bytes(2, 3, 4)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _step(**kw):
    a = _lib.GatedStepArgs()
    for n in ("x", "retention_gate", "write_gate", "nu_log", "state", "y", "new_state"):
        setattr(a, n, FAKE)
    a.batch, a.channels, a.dtype = 2, 4, 0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_c_entry_points_refuse(L):
    f = lambda a: L.sparc_gated_scan_forward(ctypes.byref(a), None)  # noqa: E731
    assert L.sparc_gated_scan_forward(None, None) == ARG and _message(L) == "null args"
    for n in ("x", "retention_gate", "write_gate", "nu_log", "y"):
        assert f(_fwd(**{n: None})) == ARG and "null tensor" in _message(L)
    for n in ("batch", "length", "channels"):
        assert f(_fwd(**{n: 0})) == SHAPE and "positive" in _message(L)
    assert f(_fwd(channels=(1 << 22) + 1)) == SHAPE
    assert f(_fwd(batch=1 << 30, length=1 << 30, channels=1 << 20)) == SHAPE
    assert f(_fwd(dtype=2)) == DTYPE
    assert f(_fwd(segment_pos=FAKE, segment_pos_bytes=3)) == ARG and "segment_pos_bytes" in _message(L)
    assert f(_fwd(x=FAKE + 2)) == ARG and "misaligned" in _message(L)
    assert f(_fwd(y=FAKE + 1, dtype=1)) == ARG and "misaligned" in _message(L)
    g = lambda a: L.sparc_gated_scan_backward(ctypes.byref(a), None)  # noqa: E731
    assert L.sparc_gated_scan_backward(None, None) == ARG
    for n in ("x", "dy", "carry", "grad_x", "grad_retention_gate", "grad_write_gate", "grad_nu_log"):
        assert g(_bwd(L, **{n: None})) == ARG and "null tensor" in _message(L)
    assert g(_bwd(L, length=-1)) == SHAPE
    assert g(_bwd(L, dtype=7)) == DTYPE
    assert g(_bwd(L, workspace=None)) == WORKSPACE
    assert g(_bwd(L, workspace=FAKE + 4)) == WORKSPACE
    assert g(_bwd(L, workspace_bytes=8)) == WORKSPACE and "too small" in _message(L)
    assert g(_bwd(L, grad_write_gate=FAKE + 2)) == ARG and "misaligned" in _message(L)
    h = lambda a: L.sparc_gated_step(ctypes.byref(a), None)  # noqa: E731
    assert L.sparc_gated_step(None, None) == ARG
    for n in ("x", "state", "new_state", "y"):
        assert h(_step(**{n: None})) == ARG
    assert h(_step(batch=0)) == SHAPE
    assert h(_step(dtype=-1)) == DTYPE
    assert h(_step(segment_pos=FAKE, segment_pos_bytes=0)) == ARG


def test_sizes(L):
    assert L.sparc_gated_chunk_tokens() == 32
    assert [L.sparc_gated_carry_chunks(n) for n in (0, 1, 32, 33, 1 << 40)] == [0, 1, 1, 2, 1 << 35]
    assert L.sparc_gated_workspace_bytes(0, 1, 1) == 0
    # the partial sums stay bounded however many rows there are
    assert L.sparc_gated_workspace_bytes(1 << 20, 1, 64) <= 148 * 16 * 64 * 8


def test_struct_layouts_match_the_header():
    import os
    import re

    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "sparc_b200.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    for cname, py in (("SparcGatedFwdArgs", _lib.GatedFwdArgs), ("SparcGatedBwdArgs", _lib.GatedBwdArgs),
                      ("SparcGatedStepArgs", _lib.GatedStepArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % cname, src, flags=re.S).group(1)
        fields = [re.sub(r"\[.*", "", d.split()[-1].lstrip("*")) for d in body.split(";") if d.strip()]
        assert fields == [f[0] for f in py._fields_], cname
