"""Layer norm on the GPU where a warp or a CTA walks many rows one after the other: forward rows of 513 to 2048
columns in one warp (from 2368 rows on), and the backward of 513 to 8192 columns, whose rows are
on the way into a ring of slots in shared memory; against the definition in float64.

Tolerances, in units of U = 2^-24. A thread adds up to E = 64 values of a row one after the other (16 in
the backward and in rows that several warps share), a warp adds its threads in 5 steps, up to 16 warps are joined
in order, and two products follow: D = E + 5 + 16 + 2 roundings at most. The mean is off by D U |x|max and
d = x - mean by as much; the sum of squares is off by D U relatively (that its mean is off too is of the
second order), so that rstd is by D / 2 U, and by 4 U more for its root and quotient; n = d rstd adds 2 U. y = n w + b
adds 2 U of its terms. Half a step of the output's type comes on top."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
D_FORWARD, D_BACKWARD = 64 + 23, 16 + 23


def _close(got, ref, bound, what):
    half = torch.finfo(got.dtype).eps / 2
    tol = bound + half * (ref.abs() + bound) + 1e-30
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max()):.3g} tolerances"


def _rows(R, W, dtype, shift, spread, seed):
    """[R, W] with its first value `shift` values past an aligned one and rows `spread` values apart beyond W."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    flat = torch.randn(shift + R * (W + spread), generator=g, device="cuda").to(dtype)
    return flat[shift:].view(R, W + spread)[:, :W]


def _check(R, W, dtype, shift=0, spread=0):
    import sparc_b200

    x, dy = _rows(R, W, dtype, shift, spread, R + W), _rows(R, W, dtype, shift, spread, R + W + 1)
    g = torch.Generator(device="cuda").manual_seed(W)
    w = torch.randn(W, generator=g, device="cuda") * 0.3 + 1.0
    b = torch.randn(W, generator=g, device="cuda")
    leaves = [x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    y = sparc_b200.layer_norm(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    x, w, b, y = x.detach(), w.detach(), b.detach(), y.detach()
    with torch.no_grad():
        assert torch.equal(sparc_b200.layer_norm(x, w, b), y)
    sums = [torch.zeros(W, dtype=torch.float64, device="cuda") for _ in range(4)]
    for k in range(0, R, 4096):  # (float64 in pieces)
        at = slice(k, k + 4096)
        xd, dd, wd, bd = x[at].double(), dy[at].double(), w.double(), b.double()
        mean = xd.mean(1, keepdim=True)
        rstd = ((xd - mean).square().mean(1, keepdim=True) + 1e-5).rsqrt()
        n = (xd - mean) * rstd
        en = D_FORWARD * U * xd.abs().amax(1, keepdim=True) * rstd + (D_FORWARD / 2 + 6) * U * n.abs()
        ref = n * wd + bd
        _close(y[at], ref, en * wd.abs() + 2 * U * ((n * wd).abs() + ref.abs()), f"y from row {k}")
        dn = dd * wd
        c1, c2 = dn.mean(1, keepdim=True), (dn * n).mean(1, keepdim=True)
        e1 = (D_BACKWARD + 1) * U * dn.abs().mean(1, keepdim=True)
        e2 = (D_BACKWARD + 2) * U * (dn * n).abs().mean(1, keepdim=True) + (dn.abs() * en).mean(1, keepdim=True)
        # the terms' own roundings, of rstd (D_FORWARD / 2 + 4) and of the products and sums (8)
        parts = (D_FORWARD / 2 + 12) * U * (dn.abs() + c1.abs() + (n * c2).abs())
        _close(grads[0][at], rstd * (dn - c1 - n * c2), rstd * (e1 + n.abs() * e2 + en * c2.abs() + parts), f"dx from row {k}")
        for s, v in zip(sums, ((dd * n).sum(0), dd.sum(0), (dd.abs() * en).sum(0), (dd * n).abs().sum(0))):
            s += v
    # a column's sum: float32 over the rows of a CTA (148 of them at least, or a row each), then over 8 warps; float64
    depth = (R / 148 + 2 + 8) * U
    _close(grads[1], sums[0], sums[2] + depth * (sums[3] + sums[2]), "dweight")
    _close(grads[2], sums[1], depth * dy.double().abs().sum(0), "dbias")


# columns of vectors, of pairs and of single elements, each instance's border; rows enough that every warp
# takes more of them than its ring has slots
FORWARD = [(30000, 520), (30000, 777), (30000, 1024), (14000, 1025), (14000, 1374), (14000, 2047), (14000, 2048),
           (2368, 2048), (2367, 2048)]
BACKWARD = [(6000, 2056), (6000, 4095), (3000, 4097), (3000, 8191), (3000, 8192)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,W", FORWARD + BACKWARD)
def test_many_rows(R, W, dtype):
    _check(R, W, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift,spread", [(1, 0), (2, 2), (3, 5)])
@pytest.mark.parametrize("R,W", [(30000, 520), (14000, 1374), (14000, 2048), (6000, 4096), (3000, 8191)])
def test_many_rows_beginning_anywhere(R, W, shift, spread, dtype):
    _check(R, W, dtype, shift, spread)
