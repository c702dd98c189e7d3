"""The gated linear recurrence on the GPU where its inputs, its callers or its waits go wrong: NaN gates
behind a segment start, and waits between the CTAs of a cluster that run out."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _inputs(B, T, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = [torch.randn(B, T, D, generator=g).to(dtype).cuda() for _ in range(3)]
    nu = torch.log(-torch.log(torch.empty(D).uniform_(0.7, 0.999, generator=g))).cuda()
    dy = torch.randn(B, T, D, generator=g).to(dtype).cuda()
    return t, nu, torch.randn(B, D, generator=g).cuda(), dy, torch.randn(B, D, generator=g).cuda()


def _run(t, nu, h0, pos, dy, dlast):
    """y, last and the gradients of x, the gates, nu_log and the state."""
    import sparc_b200

    leaves = [v.detach().requires_grad_(True) for v in (*t, nu, h0)]
    y, last = sparc_b200.gated_scan(*leaves[:4], state=leaves[4], segment_pos=pos, return_last=True)
    return [y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (dy, dlast))]


# ------------------------------------------------------------------ NaN gates behind a segment start

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,T,D", [(300, 100, 64), (1, 1100, 66)])  # clusters of one CTA; of several, odd lanes
@pytest.mark.parametrize("nu_max", [0.3, 1.5])  # (above 1/2 a warp takes other arithmetic for its gates)
@pytest.mark.parametrize("after,sign", [(1, 1), (3, 1), (6, 1), (0, -1), (3, -1)])
def test_nan_gate_behind_a_start(B, T, D, after, sign, nu_max, dtype):
    """A NaN retention gate `after` tokens behind a segment start, in the same span of eight tokens: the
    start lets nothing of it back to the segments before, whose outputs and gradients keep their bits. A
    NaN of either sign stays a NaN to its segment's end, whatever the sign of the NaN itself."""
    t, nu, h0, dy, dlast = _inputs(B, T, D, dtype, seed=after)
    nu.clamp_(max=math.log(0.3))
    nu[:3] = math.log(nu_max)
    nan = torch.full((), float("nan"), dtype=dtype)
    nan = (nan.view(torch.int16) if dtype == BF16 else nan.view(torch.int32)).abs()  # (its sign bit is clear)
    nan = (nan if sign > 0 else nan | torch.iinfo(nan.dtype).min).view(dtype).cuda()
    assert torch.isnan(nan) and bool(torch.signbit(nan)) == (sign < 0)
    starts = [16, 64, T - T % 8 - 8]
    pos = torch.full((B, T), 5, device="cuda")
    pos[:, starts] = 0
    want = _run(t, nu, h0, pos, dy, dlast)
    assert all(torch.isfinite(v).all() for v in want)
    for s in starts:
        bad = [v.clone() for v in t]
        bad[1][:, s + after] = nan
        got = _run(bad, nu, h0, pos, dy, dlast)
        end = min([e for e in starts if e > s], default=T)
        for k, name in ((0, "y"), (2, "dx"), (3, "dretention"), (4, "dwrite")):
            assert torch.equal(got[k][:, :s], want[k][:, :s]), f"{name} before token {s}"
            assert torch.equal(got[k][:, end:], want[k][:, end:]), f"{name} from token {end} on"
        assert torch.equal(got[6], want[6]), f"dstate with NaN behind token {s}"
        first = s + max(after, 1)  # (of a start's own gate only the write's factor counts)
        assert torch.isnan(got[0][:, first:end]).all()
        assert torch.isnan(got[3][:, s + after]).all()


# ------------------------------------------------------------------ waits that run out

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,tokens,reverse_tokens", [(6000, 1024, 512), (200, 256, 128), (130, 128, 128)])
def test_withheld_map(T, tokens, reverse_tokens, dtype):
    """A CTA that withholds its map at the first, a middle or the last step (of clusters of sixteen, four and
    two CTAs, which take `tokens` a step): the others' waits run out, the kernel says so and ends, what
    the steps before wrote is right, and the next call is none the worse for it."""
    from sparc_b200 import _lib

    L = _lib.lib()
    B, D = 1, 66
    t, nu, h0, dy, _ = _inputs(B, T, D, dtype)
    st, nb = (T * D, D), L.sparc_gated_workspace_bytes(B, T, D)
    stream = torch.cuda.current_stream().cuda_stream
    p, code = [v.data_ptr() for v in t], _lib.dtype_code(dtype)
    carry = torch.zeros(B, L.sparc_gated_carry_chunks(T), D, device="cuda")

    def forward(step):
        y, status = torch.zeros(B, T, D, device="cuda", dtype=dtype), torch.zeros(1, device="cuda", dtype=torch.int32)
        kept = carry if step == 0 else torch.zeros_like(carry)
        a = _lib.GatedFwdArgs(*p, nu.data_ptr(), h0.data_ptr(), None, 0, y.data_ptr(), None, kept.data_ptr(), *st, *st, *st,
                              B, T, D, code, 4 if step else 0, status.data_ptr(), step)
        assert L.sparc_gated_scan_forward(ctypes.byref(a), stream) == 0
        return y, int(status)

    def backward(step):
        out = [torch.zeros(B, T, D, device="cuda", dtype=dtype) for _ in range(3)]
        gnu, status = torch.zeros(D, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.int32)
        ws = torch.zeros(nb, device="cuda", dtype=torch.uint8)
        a = _lib.GatedBwdArgs(*p, nu.data_ptr(), dy.data_ptr(), carry.data_ptr(), None, None, 0, *(v.data_ptr() for v in out),
                              gnu.data_ptr(), None, ws.data_ptr(), nb, *st, *st, *st, *st, B, T, D, code, 4 if step else 0,
                              status.data_ptr(), step)
        assert L.sparc_gated_scan_backward(ctypes.byref(a), stream) == 0
        return out, int(status)

    y, status = forward(0)
    assert status == 0
    steps = -(-T // tokens)
    for step in {1, (steps + 1) // 2, steps}:
        got, status = forward(step)
        assert status == _lib.STATUS_TIMEOUT, f"forward, step {step} of {steps}"
        assert torch.equal(got[:, :(step - 1) * tokens], y[:, :(step - 1) * tokens])
        again, status = forward(0)
        assert status == 0 and torch.equal(again, y)
    out, status = backward(0)
    assert status == 0
    steps = -(-T // reverse_tokens)
    for step in {1, (steps + 1) // 2, steps}:
        got, status = backward(step)
        assert status == _lib.STATUS_TIMEOUT, f"backward, step {step} of {steps}"
        done = (steps - step + 1) * reverse_tokens
        assert all(torch.equal(a[:, done:], b[:, done:]) for a, b in zip(got, out))
        again, status = backward(0)
        assert status == 0 and all(torch.equal(a, b) for a, b in zip(again, out))


FIRST_CALL_CAPTURED = """
import torch, sparc_b200
from sparc_b200 import torch_ops
x, nu = torch.randn(2, 300, 32, device="cuda"), torch.full((32,), -3.0, device="cuda")
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = sparc_b200.gated_scan(x, x, x, nu)
words = torch_ops.wait_status()
assert len(words) == 1 and words[0].device == x.device and int(words[0]) == 0, words
g.replay()
sparc_b200.check_status()
assert torch.equal(y, sparc_b200.gated_scan(x, x, x, nu))
again = torch_ops.wait_status()
assert len(again) == 1 and again[0].data_ptr() == words[0].data_ptr()
words[0].fill_(1)  # what a wait that ran out in a replay leaves
try:
    sparc_b200.check_status()
except RuntimeError as e:
    assert "timed out" in str(e)
else:
    raise AssertionError("no error")
sparc_b200.check_status()
print("captured first")
"""


def test_first_call_of_a_process_captured():
    """The status word is there for a graph whose capture is a process's first call (a process of its own)."""
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_status_word_of_the_device():
    """The library's word is one per device, and what the operators' calls are given."""
    import sparc_b200
    from sparc_b200 import _lib, torch_ops

    L, p = _lib.lib(), ctypes.c_void_p()
    assert L.sparc_gated_status_word(ctypes.byref(p)) == 0 and p.value
    t, nu, h0, _, _ = _inputs(1, 4, 8, F32)
    sparc_b200.gated_scan(*t, nu, state=h0)
    assert p.value in [w.data_ptr() for w in torch_ops.wait_status()]
    assert L.sparc_gated_status_word(None) == -1
