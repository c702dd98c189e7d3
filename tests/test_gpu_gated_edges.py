"""The gated linear recurrence on the GPU where its inputs, its callers or its waits go wrong: NaN gates
behind a segment start."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


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
