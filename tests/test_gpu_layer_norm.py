"""Layer norm on the GPU (sparc_b200.layer_norm, LayerNorm) against its definition in float64.

Tolerances, in units of U = 2^-24, from the float32 arithmetic: the mean of W values is off by
(depth of the sum) U times the mean magnitude, at most 24 additions deep here (16 in a thread, 5
across a warp, then the warps); n = (x - mean) rstd is therefore off by D = 32 U (|x|max row) rstd
absolutely and 40 U relatively (rstd: the sum of squares and its root), y = n w + b adds 2 U of its
terms. Half a step of the output's type comes on top."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
U = 2.0 ** -24


def _close(got, ref, bound, what):
    half = torch.finfo(got.dtype).eps / 2
    tol = bound + half * (ref.abs() + bound) + 1e-30
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max()):.3g} tolerances"


def _check(x, w, b, dy, eps=1e-5):
    import sparc_b200

    lx, lw = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    lb = None if b is None else b.detach().requires_grad_(True)
    y = sparc_b200.layer_norm(lx, lw, lb, eps)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    grads = torch.autograd.grad(y, [lx, lw] + ([lb] if lb is not None else []), dy)
    W = x.shape[-1]
    xd, wd, dd = x.detach().double().reshape(-1, W), w.detach().double(), dy.double().reshape(-1, W)
    mean = xd.mean(1, keepdim=True)
    rstd = ((xd - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    n = (xd - mean) * rstd
    # the error of n, and what it does to the outputs; a rounding of the mean is common to the row
    en = 32 * U * xd.abs().amax(1, keepdim=True) * rstd + 40 * U * n.abs()
    ref = n * wd + (0 if b is None else b.detach().double())
    _close(y.reshape(-1, W), ref, en * wd.abs() + 2 * U * ((n * wd).abs() + ref.abs()), "y")
    dn = dd * wd
    c2 = (dn * n).mean(1, keepdim=True)
    dx = rstd * (dn - dn.mean(1, keepdim=True) - n * c2)
    # the two means: 26 U of the mean magnitudes, and n's error through the second
    e1 = 26 * U * dn.abs().mean(1, keepdim=True)
    e2 = 26 * U * (dn * n).abs().mean(1, keepdim=True) + (dn.abs() * en).mean(1, keepdim=True)
    parts = dn.abs() + dn.mean(1, keepdim=True).abs() + (n * c2).abs()
    _close(grads[0].reshape(-1, W), dx, rstd * (e1 + n.abs() * e2 + en * c2.abs() + 40 * U * parts), "dx")
    # each column's sum over the rows: float32 over one CTA's rows (at most 1 + R / 1184 of them, 8
    # times that where 8 warps' sums are added), then float64
    R = xd.shape[0]
    depth = (2 + R / 1184 + 8) * U
    _close(grads[1], (dd * n).sum(0), (dd.abs() * (en + (depth + U) * n.abs())).sum(0), "dweight")
    if b is not None:
        _close(grads[2], dd.sum(0), depth * dd.abs().sum(0), "dbias")
    with torch.no_grad():
        assert torch.equal(sparc_b200.layer_norm(x, w, b, eps), y)
    return y, grads


def _inputs(shape, dtype, seed=0, shift=0.0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    W = shape[-1]
    x = (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(dtype)
    w = torch.randn(W, generator=g, device="cuda") * 0.3 + 1.0
    b = torch.randn(W, generator=g, device="cuda")
    return x, w, b, torch.randn(shape, generator=g, device="cuda").to(dtype)


# one column to the widest rows: every instance (rows of one warp, of four to sixteen, the wide
# kernels), in vectors and in single elements, each width's border and one past it
WIDTHS = [1, 2, 7, 31, 32, 33, 128, 129, 255, 256, 512, 513, 520, 777, 1024, 2048, 2056, 4096, 4097, 8192, 8193, 8200,
          16384, 20011, 40000]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W", WIDTHS)
def test_widths(W, dtype):
    x, w, b, dy = _inputs((13, W), dtype, seed=W)
    _check(x, w, b, dy)
    _check(x[:1], w, None, dy[:1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(5000, 64), (20000, 33), (3001, 1024), (1500, 8192), (1300, 8448), (3, 5, 7, 48), (96,)])
def test_rows(shape, dtype):
    """More rows than CTAs, several leading dimensions, none."""
    _check(*_inputs(shape, dtype, seed=1))


@pytest.mark.parametrize("W", [48, 777, 2048, 16384])
def test_mean_far_from_zero(W):
    """A common offset a thousand times the spread: the variance is of the deviations."""
    _check(*_inputs((9, W), F32, shift=1000.0))
    _check(*_inputs((9, W), BF16, shift=64.0))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales(dtype):
    for scale in (1e-6, 1e6, 1e15):
        _check(*_inputs((6, 200), dtype, scale=scale), eps=1e-12)


def test_constant_rows():
    """No variance: n = 0, rstd = eps^(-1/2); a row of one column likewise."""
    import sparc_b200

    for shape in ((4, 100), (4, 1), (2, 9000)):
        x = torch.full(shape, 3.0, device="cuda")
        w, b = torch.full(shape[-1:], 2.0, device="cuda"), torch.full(shape[-1:], 0.5, device="cuda")
        assert torch.equal(sparc_b200.layer_norm(x, w, b), torch.full(shape, 0.5, device="cuda"))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W", [64, 65, 2048, 8200])
def test_strides(W, dtype):
    """Columns of a wider tensor, a transposed batch, columns that are not adjacent, a misaligned
    base, a broadcast row, a strided dy: the same bits as dense copies."""
    x, w, b, dy = _inputs((4, 6, W), dtype)
    want_y, want = _check(x, w, b, dy)

    def same(xs, ds):
        y, g = _check(xs, w, b, ds)
        assert torch.allclose(y.float(), want_y.float(), rtol=2 ** -7, atol=1e-4)
        return y, g

    wide = torch.empty(4, 6, W + 24, dtype=dtype, device="cuda")
    wide[..., 8:8 + W] = x
    same(wide[..., 8:8 + W], dy)
    wide[..., 3:3 + W] = x
    same(wide[..., 3:3 + W], dy)
    t = x.transpose(0, 1).contiguous().transpose(0, 1)
    same(t, dy.transpose(0, 1).contiguous().transpose(0, 1))
    far = x.transpose(1, 2).contiguous().transpose(1, 2)
    same(far, dy.transpose(1, 2).contiguous().transpose(1, 2))
    off = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape)
    off.copy_(x)
    same(off, dy)
    _check(x[:1, :1].expand(4, 6, W), w, b, dy)
    _check(x, w, b, dy[:1, :1].expand(4, 6, W))
    _check(x, w[:1].expand(W), b, dy)


def test_parameters_in_other_types_and_partial_gradients():
    import sparc_b200

    x, w, b, dy = _inputs((7, 96), BF16)
    wb, bb = w.bfloat16().requires_grad_(True), b.bfloat16().requires_grad_(True)
    y = sparc_b200.layer_norm(x, wb, bb)
    gw, gb = torch.autograd.grad(y, (wb, bb), dy, retain_graph=True)
    assert gw.dtype == BF16 and gb.dtype == BF16
    assert torch.equal(y, sparc_b200.layer_norm(x, wb.detach().float(), bb.detach().float()))
    lw = w.clone().requires_grad_(True)
    lb = b.clone().requires_grad_(True)
    lx = x.clone().requires_grad_(True)
    full = torch.autograd.grad(sparc_b200.layer_norm(lx, lw, lb), (lx, lw, lb), dy)
    assert torch.equal(torch.autograd.grad(sparc_b200.layer_norm(lx, w, b), lx, dy)[0], full[0])
    assert torch.equal(torch.autograd.grad(sparc_b200.layer_norm(x, lw, b), lw, dy)[0], full[1])
    assert torch.equal(torch.autograd.grad(sparc_b200.layer_norm(x, w, lb), lb, dy)[0], full[2])


def test_no_rows():
    import sparc_b200

    x = torch.empty(0, 5, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    b = torch.ones(16, device="cuda", requires_grad=True)
    y = sparc_b200.layer_norm(x, w, b)
    assert y.shape == x.shape
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert gx.shape == x.shape and not gw.any() and not gb.any()


def test_nan_stays_in_its_row():
    import sparc_b200

    for W in (40, 2048, 9001):
        x, w, b, _ = _inputs((6, W), F32)
        want = sparc_b200.layer_norm(x, w, b)
        x[2, W - 1] = float("nan")
        x[4, 0] = float("inf")
        y = sparc_b200.layer_norm(x, w, b)
        assert torch.isnan(y[2]).all() and torch.isnan(y[4]).any()
        for r in (0, 1, 3, 5):
            assert torch.equal(y[r], want[r])


def test_offsets_beyond_32_bits():
    far = (1 << 31) + 64
    buf = torch.empty(far + 256, dtype=BF16, device="cuda")
    v = buf.as_strided((2, 256), (far, 1))
    x, w, b, dy = _inputs((2, 256), BF16)
    v.copy_(x)
    y, _ = _check(v, w, b, dy)
    assert torch.equal(y, _check(x, w, b, dy)[0])


def test_reproducible_streams_and_graphs():
    """The same bits in every run, on a side stream, and in two captured graphs replayed at once."""
    import sparc_b200

    def run(x, w, b, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = sparc_b200.layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    sets = [_inputs((4000, 520), BF16, seed=k) for k in range(2)]
    want = [run(*s) for s in sets]
    assert all(torch.equal(a, b) for a, b in zip(want[0], run(*sets[0])))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(*sets[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want[0], got))
    graphs = []
    for s in sets:
        static = [torch.zeros_like(t) for t in s]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(*static)
        for a, b in zip(static, s):
            a.copy_(b)
        graphs.append((g, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), ref in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_gradient_against_differences():
    """Central differences of the float64 definition at two of the layer's own inputs."""
    import sparc_b200

    x, w, b, dy = _inputs((3, 40), F32)

    def loss(xx, ww, bb):
        m = xx.mean(-1, keepdim=True)
        return (((xx - m) / ((xx - m).square().mean(-1, keepdim=True) + 1e-5).sqrt() * ww + bb) * dy.double()).sum()

    lx, lw, lb = (t.clone().requires_grad_(True) for t in (x, w, b))
    grads = torch.autograd.grad(sparc_b200.layer_norm(lx, lw, lb), (lx, lw, lb), dy)
    p = [t.double() for t in (x, w, b)]
    for which, idx in ((0, (1, 5)), (0, (2, 39)), (1, (0,)), (2, (17,))):
        hi, lo = [t.clone() for t in p], [t.clone() for t in p]
        hi[which][idx] += 1e-5
        lo[which][idx] -= 1e-5
        d = float((loss(*hi) - loss(*lo)) / 2e-5)
        # differences: h^2 / 6 times a third derivative of order 1, 2^-53 |loss| / h; the kernel: float32
        assert abs(d - float(grads[which][idx])) < 1e-4 * (1 + abs(d))


def test_module_and_stack():
    """LayerNorm's state dict is torch.nn.LayerNorm's; SPARCStack(norm="layer") is x + mixer(norm(x))
    layer by layer, with gradients for every parameter, and the default stack is what it was."""
    import sparc_b200

    torch.manual_seed(0)
    m = sparc_b200.LayerNorm(64).cuda()
    ref = torch.nn.LayerNorm(64, eps=1e-5).cuda()
    m.load_state_dict(ref.state_dict())
    assert sparc_b200.LayerNorm(8, bias=False).bias is None
    stack = sparc_b200.SPARCStack(64, layers=2, norm="layer").cuda()
    x = torch.randn(2, 40, 64, device="cuda", requires_grad=True)
    y = stack(x)
    z = x
    for norm, mixer in zip(stack.norms, stack.mixers):
        z = z + mixer(sparc_b200.layer_norm(z, norm.weight, norm.bias, norm.eps))[0]
    assert torch.equal(y, z)
    y.square().sum().backward()
    assert x.grad is not None
    for name, p in stack.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all(), name
    block = sparc_b200.SPARCBlock(64, norm="layer").cuda()
    assert torch.equal(block(x.detach()), x.detach() + block.mixer(block.norm(x.detach()))[0])
    with pytest.raises(ValueError):
        sparc_b200.SPARCStack(64, norm="batch")
    assert sparc_b200.SPARCStack(64).fused and set(sparc_b200.SPARCBlock(64).state_dict()) >= {"norm.weight"}
    assert "norm.bias" not in sparc_b200.SPARCBlock(64).state_dict()


def test_canaries():
    """Nothing is written outside the outputs (C ABI, outputs inside a larger buffer)."""
    import ctypes

    from sparc_b200 import _lib

    L = _lib.lib()
    for R, W, dtype in ((3, 33, F32), (5, 256, BF16), (2, 2056, BF16), (2, 9001, F32)):
        x, w, b, dy = _inputs((R, W), dtype)

        def guarded(n, t):
            buf = torch.full((n + 512,), -7.0, dtype=t, device="cuda")
            return buf, buf[256:256 + n]

        bufs = [guarded(R * W, dtype), guarded(R, F32), guarded(R, F32), guarded(R * W, dtype), guarded(W, F32), guarded(W, F32)]
        y, mean, rstd, dx, dw, db = (v for _, v in bufs)
        nb = L.sparc_layer_norm_workspace_bytes(R, W)
        wsb = torch.full((nb + 512,), 77, dtype=torch.uint8, device="cuda")
        ws = wsb[256:256 + nb]
        s = torch.cuda.current_stream().cuda_stream
        f = _lib.LayerNormFwdArgs(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr(), mean.data_ptr(),
                                  rstd.data_ptr(), W, R, W, 1e-5, _lib.dtype_code(dtype))
        assert L.sparc_layer_norm_forward(ctypes.byref(f), s) == 0
        a = _lib.LayerNormBwdArgs(x.data_ptr(), dy.data_ptr(), w.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                  dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), nb, W, W, R, W,
                                  _lib.dtype_code(dtype))
        assert L.sparc_layer_norm_backward(ctypes.byref(a), s) == 0
        torch.cuda.synchronize()
        for buf, view in bufs:
            assert (buf[:256] == -7).all() and (buf[256 + view.numel():] == -7).all()
            assert not (view == -7).all()
        assert (wsb[:256] == 77).all() and (wsb[256 + nb:] == 77).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("W", [8200, 9001, 12290, 16383])
def test_tall_rows(W, dtype):
    """Rows that CTAs walk two and three of, of every vector width, in place in wider rows; and dx alone."""
    import sparc_b200

    x, w, b, dy = _inputs((333, W + 8), dtype, seed=W)
    x, dy, w, b = x[:, 8:], dy[:, :W], w[8:], b[8:]
    _, grads = _check(x, w, b, dy)
    lx = x.detach().requires_grad_(True)
    y = sparc_b200.layer_norm(lx, w, b)
    assert torch.equal(torch.autograd.grad(y, lx, dy)[0], grads[0])


def test_the_widest_row():
    """The width limit, with the parameters' gradients: as many columns as the launches have to cover."""
    import sparc_b200

    W = 1 << 24
    x = torch.zeros(1, W, device="cuda", dtype=BF16)
    x[0, ::2] = 1.0
    w = torch.ones(W, device="cuda", requires_grad=True)
    b = torch.zeros(W, device="cuda", requires_grad=True)
    y = sparc_b200.layer_norm(x, w, b, 0.0)  # mean 1/2, deviation 1/2, both exact: y is +-1
    assert torch.equal(y, x * 2 - 1)
    dw, db = torch.autograd.grad(y, (w, b), torch.ones_like(y))
    assert torch.equal(dw, (x[0] * 2 - 1).float()) and torch.equal(db, torch.ones_like(db))


@pytest.mark.parametrize("value", [1e20, -7e18, 12345.678])
def test_wide_rows_without_variance(value):
    """What rounding leaves of the variance may not turn it negative."""
    import sparc_b200

    x = torch.full((2, 20001), value, device="cuda")
    w = torch.ones(20001, device="cuda")
    assert bool(torch.isfinite(sparc_b200.layer_norm(x, w)).all())


def test_negated_views():
    """A view that PyTorch holds with the sign of its memory reversed."""
    import sparc_b200

    x = torch.randn(7, 1, device="cuda")
    n = torch.complex(torch.zeros_like(x), -x).conj().imag
    w = torch.full((1,), 2.0, device="cuda")
    b = torch.complex(torch.zeros(1, device="cuda"), torch.full((1,), -3.0, device="cuda")).conj().imag
    assert n.is_neg() and b.is_neg()
    assert bool((sparc_b200.layer_norm(n, w, b) == 3.0).all())
