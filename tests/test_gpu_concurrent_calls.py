"""Host threads that call one kernel at once, in forms that take different amounts of shared memory: no
call may change what another's launch is allowed."""
import ctypes
import threading

import pytest
import torch

from sparc_b200 import _lib

pytestmark = pytest.mark.gpu

CALLS = 3000


def _at_once(calls):
    """Each (function, arguments) CALLS times from a thread of its own, on a stream of its own; the codes that
    were not zero."""
    streams, codes = [torch.cuda.Stream() for _ in calls], [[] for _ in calls]
    device, gate = torch.cuda.current_device(), threading.Barrier(len(calls))
    torch.cuda.synchronize()

    def work(k):
        torch.cuda.set_device(device)
        f, args = calls[k]
        gate.wait()
        codes[k] = [rc for rc in (f(ctypes.byref(args), streams[k].cuda_stream) for _ in range(CALLS)) if rc != 0]

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(calls))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    return codes


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_scan(dtype):
    """One sequence that a cluster of sixteen CTAs walks, and many rows of one CTA each."""
    L = _lib.lib()
    keep, forward, backward = [], [], []
    for B, T, D in ((1, 1024, 64), (640, 2, 64)):
        t = [torch.randn(B, T, D, device="cuda").to(dtype) for _ in range(4)]
        out = [torch.empty(B, T, D, device="cuda", dtype=dtype) for _ in range(4)]
        nu, gnu = torch.full((D,), -3.0, device="cuda"), torch.empty(D, device="cuda")
        carry = torch.zeros(B, L.sparc_gated_carry_chunks(T), D, device="cuda")
        nb = L.sparc_gated_workspace_bytes(B, T, D)
        ws = torch.empty(nb, device="cuda", dtype=torch.uint8)
        st, code = (T * D, D), _lib.dtype_code(dtype)
        p = [v.data_ptr() for v in t]
        forward.append((L.sparc_gated_scan_forward,
                        _lib.GatedFwdArgs(*p[:3], nu.data_ptr(), None, None, 0, out[3].data_ptr(), None, None, *st, *st, *st,
                                          B, T, D, code)))
        backward.append((L.sparc_gated_scan_backward,
                         _lib.GatedBwdArgs(*p[:3], nu.data_ptr(), p[3], carry.data_ptr(), None, None, 0,
                                           *(v.data_ptr() for v in out[:3]), gnu.data_ptr(), None, ws.data_ptr(), nb,
                                           *st, *st, *st, *st, B, T, D, code)))
        keep += [t, out, nu, gnu, carry, ws]
    assert _at_once(forward) == [[], []]
    assert _at_once(backward) == [[], []]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_backward(dtype):
    """Rows of 16384 columns with and without the parameters' gradients."""
    L = _lib.lib()
    R, W, code = 2, 16384, _lib.dtype_code(dtype)
    keep, calls = [], []
    for sums in (True, False):
        x, dy = (torch.randn(R, W, device="cuda").to(dtype) for _ in range(2))
        dx = torch.empty_like(x)
        w, gw, gb = (torch.ones(W, device="cuda") for _ in range(3))
        stats = torch.ones(2, R, device="cuda")
        nb = L.sparc_layer_norm_workspace_bytes(R, W)
        ws = torch.empty(nb, device="cuda", dtype=torch.uint8)
        calls.append((L.sparc_layer_norm_backward,
                      _lib.LayerNormBwdArgs(x.data_ptr(), dy.data_ptr(), w.data_ptr(), stats[0].data_ptr(),
                                            stats[1].data_ptr(), dx.data_ptr(), gw.data_ptr() if sums else None,
                                            gb.data_ptr() if sums else None, ws.data_ptr() if sums else None,
                                            nb if sums else 0, W, W, R, W, code)))
        keep += [x, dy, dx, w, gw, gb, stats, ws]
    assert _at_once(calls) == [[], []]
