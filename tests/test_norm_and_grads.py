"""Refusals of the layer norm and of the gradient norm and clipping, without a GPU: the Python
functions and the C entry points (no pointer passed is dereferenced on the device)."""
import ctypes
import os
import re

import pytest
import torch

import sparc_b200
from sparc_b200 import _lib

ARG, SHAPE, DTYPE, WORKSPACE = -1, -2, -3, -4
FAKE = 0x100000
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


def test_layer_norm_refusals():
    x, w = torch.zeros(2, 3, 8), torch.ones(8)
    f = sparc_b200.layer_norm
    for bad in (lambda: f(x, w[:4]), lambda: f(x, w.view(1, 8)), lambda: f(torch.zeros(()), w), lambda: f(x, w, w[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="at least one column"):
        f(torch.zeros(2, 0), torch.zeros(0))
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            f(x, w, eps=eps)
    with pytest.raises(TypeError):
        f(x.half(), w)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x, w, w)
    with pytest.raises(RuntimeError, match="CUDA"):
        sparc_b200.LayerNorm(8)(x)


def test_stack_norm_choice():
    with pytest.raises(ValueError, match="'rms' or 'layer'"):
        sparc_b200.SPARCStack(8, layers=1, norm="none")
    s = sparc_b200.SPARCStack(8, layers=2, norm="layer")
    assert {"norms.0.weight", "norms.0.bias", "norms.1.bias"} <= set(s.state_dict()) and not s.fused
    assert "norms.0.bias" not in sparc_b200.SPARCStack(8, layers=1).state_dict()


def test_grad_refusals():
    t = [torch.zeros(3), torch.zeros(2, 2)]
    for f in (sparc_b200.grad_norm, lambda g: sparc_b200.clip_grads(g, 1.0)):
        with pytest.raises(ValueError, match="at least one"):
            f([])
        with pytest.raises(TypeError):
            f([torch.zeros(3, dtype=torch.float16)])
        with pytest.raises(TypeError, match="dense"):
            f([torch.zeros(3, 3).to_sparse()])
        with pytest.raises(RuntimeError, match="CUDA"):
            f(t)
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, eps=-1.0)):
        with pytest.raises(ValueError, match="negative"):
            sparc_b200.clip_grads(t, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        sparc_b200.clip_grads(t, 1.0, out=t)
    p = torch.nn.Parameter(torch.zeros(2))
    assert float(sparc_b200.clip_grad_norm_([p], 1.0)) == 0.0  # no gradients
    assert float(sparc_b200.clip_grad_norm_([], 1.0)) == 0.0


def test_layer_norm_c_refusals(L):
    def fwd(**kw):
        a = _lib.LayerNormFwdArgs(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 8, 2, 8, 1e-5, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.sparc_layer_norm_forward(ctypes.byref(a), None)

    def bwd(**kw):
        a = _lib.LayerNormBwdArgs(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                                  L.sparc_layer_norm_workspace_bytes(2, 8), 8, 8, 2, 8, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.sparc_layer_norm_backward(ctypes.byref(a), None)

    assert L.sparc_layer_norm_forward(None, None) == ARG and L.sparc_layer_norm_backward(None, None) == ARG
    for n in ("x", "weight", "y"):
        assert fwd(**{n: None}) == ARG
    assert fwd(mean=None) == ARG and "together" in _message(L)
    assert fwd(rows=0) == SHAPE and fwd(width=0) == SHAPE and fwd(width=(1 << 24) + 1) == SHAPE
    assert fwd(dtype=5) == DTYPE
    assert fwd(x=FAKE + 2) == ARG and "misaligned" in _message(L)
    for n in ("x", "dy", "dx", "weight", "mean", "rstd"):
        assert bwd(**{n: None}) == ARG
    assert bwd(rows=-1) == SHAPE and bwd(dtype=-1) == DTYPE
    assert bwd(workspace=None) == WORKSPACE and bwd(workspace_bytes=4) == WORKSPACE
    assert bwd(dy=FAKE + 1, dtype=1) == ARG
    assert L.sparc_layer_norm_workspace_bytes(0, 8) == 0
    assert L.sparc_layer_norm_workspace_bytes(1 << 30, 8) <= 148 * 8 * 2 * 8 * 4


def _clip(L, grads, counts, dtypes=None, out=None, **kw):
    n = len(grads)
    a = _lib.GradClipArgs((ctypes.c_void_p * n)(*grads), None if out is None else (ctypes.c_void_p * n)(*out),
                          (ctypes.c_longlong * n)(*counts), (ctypes.c_int * n)(*(dtypes or [0] * n)), n, 1.0, 1e-6, FAKE,
                          FAKE, L.sparc_grad_clip_workspace_bytes(n))
    for k, v in kw.items():
        setattr(a, k, v)
    return L.sparc_grad_clip(ctypes.byref(a), None)


def test_grad_clip_c_refusals(L):
    assert L.sparc_grad_clip(None, None) == ARG
    A, B = FAKE, FAKE + 4096
    assert _clip(L, [], []) == SHAPE
    assert _clip(L, [A], [4], tensors=-1) == SHAPE
    assert _clip(L, [A], [4], norm=None) == ARG
    assert _clip(L, [A], [4], workspace=None) == WORKSPACE and _clip(L, [A], [4], workspace_bytes=8) == WORKSPACE
    assert _clip(L, [A, 0], [4, 4]) == ARG and _clip(L, [A, B], [4, 4], out=[A, 0]) == ARG
    assert _clip(L, [A + 2], [4]) == ARG and "misaligned" in _message(L)
    assert _clip(L, [A], [4], dtypes=[9]) == DTYPE
    assert _clip(L, [A], [-1]) == SHAPE and _clip(L, [A, B], [1 << 43, 1]) == SHAPE
    for m in (-1.0, float("nan")):
        assert _clip(L, [A], [4], out=[A], max_norm=m) == ARG
    assert _clip(L, [A], [4], out=[A], eps=-1.0) == ARG
    for grads, counts, out in (([A, A], [4, 4], [A, A]), ([A, A + 8], [4, 4], [A, A + 8]), ([A, B], [4, 4], [B, A]),
                               ([A], [4], [A + 4]), ([A, B], [2000, 4], [A, B]), ([A, B], [4, 4], [A + 64, A + 72])):
        assert _clip(L, grads, counts, out=out) == ARG and "overlaps" in _message(L)
    assert L.sparc_grad_clip_workspace_bytes(-1) == 0
    assert L.sparc_grad_clip_workspace_bytes(257) == 2 * L.sparc_grad_clip_workspace_bytes(256)


def test_struct_layouts_match_the_header():
    src = open(os.path.join(ROOT, "include", "sparc_b200.h")).read()
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    for cname, py in (("SparcLayerNormFwdArgs", _lib.LayerNormFwdArgs), ("SparcLayerNormBwdArgs", _lib.LayerNormBwdArgs),
                      ("SparcGradClipArgs", _lib.GradClipArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % cname, src, flags=re.S).group(1)
        fields = [re.sub(r"\[.*", "", d.split()[-1].lstrip("*")) for d in body.split(";") if d.strip()]
        assert fields == [f[0] for f in py._fields_], cname


def test_timing_names_cover_every_kernel(L):
    names = [L.sparc_timing_kernel_name(i).decode() for i in range(L.sparc_timing_read(None, None, 0))]
    assert all(names) and len(set(names)) == len(names)
    assert {"gated_fwd_kernel", "layer_norm_bwd_kernel", "grad_clip_kernel"} <= set(names)
