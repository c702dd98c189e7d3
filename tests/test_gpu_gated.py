"""The gated linear recurrence on the GPU (sparc_b200.gated_scan, gated_scan_step) against the
float64 oracle. Every element's tolerance is the oracle's running bound of the float32 rounding
errors plus half a step of the output's type (torch.finfo(t).eps / 2 of the value)."""
import numpy as np
import pytest
import torch

from oracle import gated_oracle as G

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, bound, what):
    half = torch.finfo(got.dtype).eps / 2
    g = _np(got)
    tol = bound + half * (np.abs(ref) + bound) + 1e-30
    bad = ~(np.abs(g - ref) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(g - ref) / tol):.3g} tolerances"


def _inputs(B, T, D, dtype, seed=0, state=True, segments=True, low=0.5, high=0.9999):
    g = torch.Generator().manual_seed(seed)
    t = [torch.randn(B, T, D, generator=g).to(dtype).cuda() for _ in range(3)]
    t[1].clamp_(-8, 8)
    t[2].clamp_(-8, 8)
    nu = torch.log(-torch.log(torch.empty(D).uniform_(low, high, generator=g))).cuda()
    h0 = torch.randn(B, D, generator=g).cuda() if state else None
    pos = None
    if segments:
        pos = torch.where(torch.rand(B, T, generator=g) < 0.05, 0, 7).cuda()
    return t, nu, h0, pos


def _check(t, nu, h0, pos, seed=1, dy=None):
    import sparc_b200

    x, r, w = t
    B, T, D = x.shape
    g = torch.Generator().manual_seed(seed)
    dy = torch.randn(B, T, D, generator=g).to(x.dtype).cuda() if dy is None else dy
    dl = torch.randn(B, D, generator=g).cuda()
    leaves = [v.detach().requires_grad_(True) for v in (x, r, w, nu)]
    s = None if h0 is None else h0.detach().requires_grad_(True)
    y, last = sparc_b200.gated_scan(*leaves, state=s, segment_pos=pos, return_last=True)
    assert y.dtype == x.dtype and y.shape == x.shape and last.dtype == F32 and last.shape == (B, D)
    grads = torch.autograd.grad((y, last), leaves + ([s] if s is not None else []), (dy, dl))
    n = [_np(v) for v in (x, r, w, nu)]
    starts = None if pos is None else pos.cpu().numpy() == 0
    hn = None if h0 is None else _np(h0)
    h, hl = G.forward(*n, hn, starts)
    ref = G.backward(*n, _np(dy), hn, starts, _np(dl))
    bd = G.bounds(*n, _np(dy), hn, starts, _np(dl))
    _close(y, h, bd["h"], "y")
    _close(last, hl, bd["last"], "last")
    for name, got in zip(("x", "r", "w", "nu_log", "h0"), grads):
        _close(got, ref[name], bd[name], "d" + name)
    with torch.no_grad():  # the form without carries
        y2, last2 = sparc_b200.gated_scan(x, r, w, nu, state=h0, segment_pos=pos, return_last=True)
    assert torch.equal(y2, y) and torch.equal(last2, last)
    return y, last, grads


SHAPES = [(1, 1, 1), (2, 1, 66), (2, 3, 5), (3, 8, 64), (1, 9, 2), (2, 33, 64), (3, 64, 66), (2, 65, 130), (1, 129, 31),
          (1, 1000, 34), (2, 513, 7), (1, 2049, 2), (4, 300, 65), (1, 1100, 64), (5, 515, 128)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [0.5, 0.7])  # the least decay: nu above 1/2 in some channels, in none
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_matches_oracle(B, T, D, low, dtype):
    """One token to many tiles, odd channels, clusters of one to sixteen CTAs, ragged last tiles."""
    _check(*_inputs(B, T, D, dtype, seed=B * T + D, low=low))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 66, 33])
def test_long_rows_without_segments(D, dtype):
    """Clusters of sixteen over many steps, each kind of read."""
    _check(*_inputs(1, 2500, D, dtype, segments=False, low=0.7))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("state,segments", [(False, False), (True, False), (False, True)])
def test_optional_arguments(state, segments, dtype):
    _check(*_inputs(2, 150, 40, dtype, state=state, segments=segments))


@pytest.mark.parametrize("B,T,D", [(3000, 2, 3), (700, 40, 256), (40, 70, 1030)])
def test_many_rows(B, T, D):
    """More rows than clusters: each cluster walks several rows and sums their dnu_log."""
    _check(*_inputs(B, T, D, F32, segments=False))


def test_strong_and_weak_decay():
    """a down to zero, and so near 1 that 1 - a is a few float32 steps."""
    t, nu, h0, pos = _inputs(2, 200, 64, F32, segments=False)
    nu[:16] = 6.0     # e^6 = 403: a underflows for most gates
    nu[16:32] = -16.0  # 1 - a about 1e-7
    nu[32:40] = -40.0
    _check(t, nu, h0, pos)


@pytest.mark.parametrize("nu_value", [1.0, 0.25])
def test_gates_at_infinity(nu_value):
    """s(-inf) is exactly 0 and s(inf) exactly 1: a closed retention gate keeps the state (and
    writes nothing, as 1 - a^2 = 0), a closed write gate writes nothing; gradients are finite, and
    those of a closed write gate's x are exactly zero."""
    import sparc_b200

    inf = float("inf")
    x = torch.randn(1, 4, 8, device="cuda")
    for dtype in (F32, BF16):
        h0 = torch.randn(1, 8, device="cuda")
        closed = torch.full((1, 4, 8), -inf, device="cuda", dtype=dtype)
        opened = torch.full((1, 4, 8), inf, device="cuda", dtype=dtype)
        nu = torch.full((8,), float(np.log(nu_value)), device="cuda")
        xx = x.to(dtype)
        args = [v.clone().requires_grad_(True) for v in (xx, closed, opened, nu, h0)]
        y, last = sparc_b200.gated_scan(*args[:4], state=args[4], return_last=True)
        assert torch.equal(last, h0)
        for g in torch.autograd.grad((y, last), args, (torch.ones_like(y), torch.ones_like(last))):
            assert torch.isfinite(g).all()
        y = sparc_b200.gated_scan(xx, opened, closed, nu, state=h0)
        xc = xx.clone().requires_grad_(True)
        yc = sparc_b200.gated_scan(xc, opened, closed, nu, state=h0)
        assert not torch.autograd.grad(yc, xc, torch.ones_like(yc))[0].any()
        a = torch.exp(torch.tensor(-nu_value, dtype=torch.float64))
        want = torch.stack([h0.double() * a ** (k + 1) for k in range(4)], 1)
        # four exp2 values, each off by 6 units, and their products
        assert ((y.double() - want).abs() <= want.abs() * (40 * G.U + torch.finfo(dtype).eps / 2)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_nothing_crosses_a_segment_start(dtype):
    """Infinities and NaN of one segment leave the next one (and, backwards, the one before) as
    they would be without them; two adjacent starts and a start at the first and last token too."""
    import sparc_b200

    for T in (7, 100, 700):
        t, nu, h0, _ = _inputs(2, T, 34, dtype, segments=False)
        pos = torch.full((2, T), 5, device="cuda")
        cut = T // 2
        pos[:, cut] = 0
        pos[:, cut + 1] = 0
        pos[0, 0] = 0
        pos[1, T - 1] = 0
        clean = [v.clone().requires_grad_(True) for v in t]
        dirty = [v.clone() for v in t]
        dirty[0][:, cut - 1] = float("nan")
        dirty[1][:, cut - 2] = float("inf")
        dirty[0][:, cut - 3] = float("inf")
        dirty = [v.requires_grad_(True) for v in dirty]
        hn = h0.clone()
        hn[0] = float("nan")  # row 0 starts a segment at its first token
        y1 = sparc_b200.gated_scan(*clean, nu, state=h0, segment_pos=pos)
        y2 = sparc_b200.gated_scan(*dirty, nu, state=hn, segment_pos=pos)
        assert torch.equal(y1[:, cut:], y2[:, cut:]) and torch.isfinite(y2[:, cut:]).all()
        assert torch.equal(y1[:, :cut - 3], y2[:, :cut - 3])
        dy = torch.randn(2, T, 34, device="cuda").to(dtype)
        g1 = torch.autograd.grad(y1, clean, dy)
        g2 = torch.autograd.grad(y2, dirty, dy)
        for a, b in zip(g1, g2):
            assert torch.equal(a[:, cut:], b[:, cut:])
        dn = dy.clone()
        dn[:, cut:] = float("nan")  # a later segment's gradient does not reach an earlier one
        y1 = sparc_b200.gated_scan(*clean, nu, state=h0, segment_pos=pos)
        g3 = torch.autograd.grad(y1, clean, dn)
        for a, b in zip(g1, g3):
            assert torch.equal(a[:, :cut], b[:, :cut]) and torch.isfinite(b[:, :cut]).all()


@pytest.mark.parametrize("low", [0.5, 0.7])
def test_nan_inputs_are_not_lost(low):
    import sparc_b200

    for which in range(3):
        for dtype in (F32, BF16):
            t, nu, _, _ = _inputs(1, 70, 33, dtype, state=False, segments=False, low=low)
            t[which][0, 20, 3] = float("nan")
            y = sparc_b200.gated_scan(*t, nu)
            assert torch.isnan(y[0, 20:, 3]).all()
            y[0, 20:, 3] = 0
            assert torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pos_dtype", [torch.int64, torch.int32, torch.int16, torch.uint8, torch.bool])
def test_position_types(pos_dtype, dtype):
    import sparc_b200

    t, nu, h0, pos = _inputs(2, 90, 10, dtype)
    want = sparc_b200.gated_scan(*t, nu, state=h0, segment_pos=pos)
    p = (pos * 256 if pos_dtype in (torch.int64, torch.int32, torch.int16) else pos).to(pos_dtype)
    assert torch.equal(sparc_b200.gated_scan(*t, nu, state=h0, segment_pos=p), want)
    pt = p.t().contiguous().t()  # strided positions
    assert torch.equal(sparc_b200.gated_scan(*t, nu, state=h0, segment_pos=pt), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 33])
def test_strides(D, dtype):
    """Columns of one projection, a transposed batch, a broadcast x, channels that are not
    adjacent, a misaligned base and a strided dy."""
    t, nu, h0, pos = _inputs(2, 100, D, dtype)
    p = torch.cat(t, dim=-1)
    y, last, grads = _check(list(p.split(D, dim=-1)), nu, h0, pos)
    tr = [v.transpose(0, 1).contiguous().transpose(0, 1) for v in t]
    y2, _, g2 = _check(tr, nu, h0, pos)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, g2))
    far = [v.transpose(1, 2).contiguous().transpose(1, 2) for v in t]
    y3, _, g3 = _check(far, nu, h0, pos)
    assert torch.equal(y, y3) and all(torch.equal(a, b) for a, b in zip(grads, g3))
    off = []
    for v in t:
        buf = torch.empty(v.numel() + 1, dtype=dtype, device="cuda")[1:].view(v.shape)
        buf.copy_(v)
        off.append(buf)
    _check(off, nu, h0, pos)
    _check([t[0][:, :1].expand(2, 100, D), t[1], t[2][:1].expand(2, 100, D)], nu, h0, pos)
    dy = torch.randn(100, 2, D, device="cuda").to(dtype).transpose(0, 1)
    _check(t, nu, h0, pos, dy=dy)
    dy = torch.randn(2, D, 100, device="cuda").to(dtype).transpose(1, 2)
    _check(t, nu, h0, pos, dy=dy)


def test_offsets_beyond_32_bits():
    """Rows more than 2^32 bytes (and 2^31 elements) apart."""
    far = (1 << 31) + 64
    need = far + 40 * 192
    buf = torch.empty(need, dtype=BF16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    v = buf.as_strided((2, 40, 192), (far, 192, 1))
    v.copy_(torch.randn(2, 40, 192, generator=g, device="cuda"))
    _, nu, h0, pos = _inputs(2, 40, 64, BF16)
    _check(list(v.split(64, dim=-1)), nu, h0, pos)


def test_gradients_of_one_output():
    import sparc_b200

    t, nu, h0, pos = _inputs(2, 70, 12, F32)
    n = [_np(v) for v in (*t, nu)]
    starts = pos.cpu().numpy() == 0
    for which in (0, 1):
        leaves = [v.detach().clone().requires_grad_(True) for v in (*t, nu, h0)]
        out = sparc_b200.gated_scan(*leaves[:4], state=leaves[4], segment_pos=pos, return_last=True)
        g = torch.randn(out[which].shape, device="cuda")
        grads = torch.autograd.grad(out[which], leaves, g)
        dy = _np(g) if which == 0 else np.zeros((2, 70, 12))
        dl = None if which == 0 else _np(g)
        ref = G.backward(*n, dy, _np(h0), starts, dl)
        bd = G.bounds(*n, dy, _np(h0), starts, dl)
        for name, got in zip(("x", "r", "w", "nu_log", "h0"), grads):
            _close(got, ref[name], bd[name], name)


def test_parameter_dtypes():
    """nu_log and the state in other float types: used in float32, gradients in their own."""
    import sparc_b200

    t, nu, h0, _ = _inputs(2, 40, 16, BF16, segments=False)
    nb, hb = nu.bfloat16().requires_grad_(True), h0.double().requires_grad_(True)
    y = sparc_b200.gated_scan(*t, nb, state=hb)
    gn, gh = torch.autograd.grad(y, (nb, hb), torch.ones_like(y))
    assert gn.dtype == BF16 and gh.dtype == torch.float64
    assert torch.equal(y, sparc_b200.gated_scan(*t, nu.bfloat16().float(), state=h0))


def test_reproducible_bitwise():
    t, nu, h0, pos = _inputs(2, 3000, 130, BF16)
    first = _check_only(t, nu, h0, pos)
    for _ in range(3):
        for a, b in zip(first, _check_only(t, nu, h0, pos)):
            assert torch.equal(a, b)


def _check_only(t, nu, h0, pos):
    import sparc_b200

    leaves = [v.detach().requires_grad_(True) for v in (*t, nu, h0)]
    y, last = sparc_b200.gated_scan(*leaves[:4], state=leaves[4], segment_pos=pos, return_last=True)
    return [y.detach(), last.detach(),
            *torch.autograd.grad((y, last), leaves, (torch.ones_like(y), torch.ones_like(last)))]


def test_second_derivative_is_refused():
    import sparc_b200

    t, nu, _, _ = _inputs(1, 5, 4, F32, state=False, segments=False)
    x = t[0].requires_grad_(True)
    y = sparc_b200.gated_scan(x, t[1], t[2], nu)
    (g,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_streams_and_graphs():
    """On a side stream, and captured (forward and backward, two graphs) and replayed in turn and
    at once on new inputs: the same bits as eager calls."""
    import sparc_b200

    t, nu, h0, pos = _inputs(2, 300, 64, BF16)
    want = _check_only(t, nu, h0, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _check_only(t, nu, h0, pos)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for k in range(2):
        static = [v.clone() for v in (*t, nu, h0)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            _check_only(static[:3], static[3], static[4], pos)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _check_only(static[:3], static[3], static[4], pos)
        graphs.append((graph, static, out))
    fresh = [_inputs(2, 300, 64, BF16, seed=11 + k, segments=False) for k in range(2)]
    for (graph, static, out), (tt, nn, hh, _) in zip(graphs, fresh):
        for a, b in zip(static, (*tt, nn, hh)):
            a.copy_(b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for (graph, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (graph, static, out), (tt, nn, hh, _) in zip(graphs, fresh):
        assert all(torch.equal(a, b) for a, b in zip(out, _check_only(tt, nn, hh, pos)))


def test_stays_in_bounds():
    """Nothing outside the outputs is written: through the C ABI, outputs inside canaried buffers at
    every alignment an element allows, odd and even widths, ragged lengths, one and many CTAs."""
    import ctypes

    from sparc_b200 import _lib

    L = _lib.lib()
    stream = torch.cuda.current_stream().cuda_stream
    for B, T, D, dtype, shift in ((2, 37, 33, BF16, 1), (1, 700, 64, BF16, 0), (3, 65, 10, F32, 1), (2, 100, 66, BF16, 2),
                                  (1, 1, 7, F32, 3), (1, 1030, 31, F32, 0)):
        t, nu, h0, pos = _inputs(B, T, D, dtype)
        dy = torch.randn(B, T, D, device="cuda").to(dtype)

        def guarded(n, kind):
            buf = torch.full((n + 1024,), -9.0, dtype=kind, device="cuda")
            return buf, buf[512 + shift:512 + shift + n]

        chunks = L.sparc_gated_carry_chunks(T)
        bufs = [guarded(B * T * D, dtype) for _ in range(4)] + [guarded(B * D, F32), guarded(B * chunks * D, F32),
                                                               guarded(D, F32), guarded(B * D, F32)]
        y, dx, dr, dw, last, carry, dnu, dh0 = (v for _, v in bufs)
        nb = L.sparc_gated_workspace_bytes(B, T, D)
        wsb = torch.full((nb + 512,), 77, dtype=torch.uint8, device="cuda")
        ws = wsb[256:256 + nb]
        st = (T * D, D)
        f = _lib.GatedFwdArgs(*[v.data_ptr() for v in t], nu.data_ptr(), h0.data_ptr(), pos.data_ptr(), 8, y.data_ptr(),
                              last.data_ptr(), carry.data_ptr(), *st, *st, *st, B, T, D, _lib.dtype_code(dtype))
        assert L.sparc_gated_scan_forward(ctypes.byref(f), stream) == 0
        b = _lib.GatedBwdArgs(*[v.data_ptr() for v in t], nu.data_ptr(), dy.data_ptr(), carry.data_ptr(), None,
                              pos.data_ptr(), 8, dx.data_ptr(), dr.data_ptr(), dw.data_ptr(), dnu.data_ptr(), dh0.data_ptr(),
                              ws.data_ptr(), nb, *st, *st, *st, *st, B, T, D, _lib.dtype_code(dtype))
        assert L.sparc_gated_scan_backward(ctypes.byref(b), stream) == 0
        torch.cuda.synchronize()
        for buf, v in bufs:
            assert (buf[:512 + shift] == -9).all() and (buf[512 + shift + v.numel():] == -9).all()
            assert not (v == -9).any()
        assert (wsb[:256] == 77).all() and (wsb[256 + nb:] == 77).all()
        h, _ = G.forward(*[_np(v) for v in (*t, nu)], _np(h0), pos.cpu().numpy() == 0)
        bd = G.bounds(*[_np(v) for v in (*t, nu)], None, _np(h0), pos.cpu().numpy() == 0)
        _close(y.view(B, T, D), h, bd["h"], "y")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_short_waits_end(dtype):
    """One poll for each wait between the CTAs of a cluster: where none ran out the results are those of
    the ordinary bound, else the status says so; either way both directions end."""
    from sparc_b200 import _lib

    L = _lib.lib()
    B, T, D = 1, 6000, 66
    t, nu, h0, pos = _inputs(B, T, D, dtype, segments=False)
    dy = torch.randn(B, T, D, device="cuda").to(dtype)
    st, nb = (T * D, D), L.sparc_gated_workspace_bytes(B, T, D)
    s = torch.cuda.current_stream().cuda_stream
    got = {}
    for spin in (0, 1):
        y, gx, gr, gw = (torch.zeros(B, T, D, device="cuda", dtype=dtype) for _ in range(4))
        carry = torch.zeros(B, L.sparc_gated_carry_chunks(T), D, device="cuda")
        gn, ws = torch.zeros(D, device="cuda"), torch.zeros(nb, device="cuda", dtype=torch.uint8)
        fw, bw = torch.zeros(1, device="cuda", dtype=torch.int32), torch.zeros(1, device="cuda", dtype=torch.int32)
        f = _lib.GatedFwdArgs(*[v.data_ptr() for v in t], nu.data_ptr(), h0.data_ptr(), None, 0, y.data_ptr(), None,
                              carry.data_ptr(), *st, *st, *st, B, T, D, _lib.dtype_code(dtype), spin, fw.data_ptr())
        assert L.sparc_gated_scan_forward(f, s) == 0
        c = got[0][0][1] if spin else carry  # the backward's own waits, on good carries
        b = _lib.GatedBwdArgs(*[v.data_ptr() for v in t], nu.data_ptr(), dy.data_ptr(), c.data_ptr(), None, None, 0,
                              gx.data_ptr(), gr.data_ptr(), gw.data_ptr(), gn.data_ptr(), None, ws.data_ptr(), nb, *st, *st,
                              *st, *st, B, T, D, _lib.dtype_code(dtype), spin, bw.data_ptr())
        assert L.sparc_gated_scan_backward(b, s) == 0
        torch.cuda.synchronize()
        got[spin] = (y, carry), (gx, gr, gw, gn), (int(fw), int(bw))
    assert got[0][2] == (0, 0) and all(v in (0, 4) for v in got[1][2])
    for k in (0, 1):
        if got[1][2][k] == 0:
            assert all(torch.equal(a, b) for a, b in zip(got[0][k], got[1][k]))


def test_negated_views():
    """Views that PyTorch holds with the sign of their memory reversed."""
    import sparc_b200

    t, nu, h0, _ = _inputs(2, 9, 1, F32, segments=False)
    z = [torch.complex(torch.zeros_like(v), -v).conj().imag for v in (*t, h0)]
    assert all(v.is_neg() for v in z)
    x, r, w, s = z
    assert torch.equal(sparc_b200.gated_scan(x, r, w, nu, state=s), sparc_b200.gated_scan(*t, nu, state=h0))
    a = sparc_b200.gated_scan_step(x[:, 0], r[:, 0], w[:, 0], nu, s)
    b = sparc_b200.gated_scan_step(*(v[:, 0] for v in t), nu, h0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_modes_of_the_caller():
    """Under inference mode, and compiled (the graph breaks around the operators): the eager bits."""
    import sparc_b200

    t, nu, h0, pos = _inputs(2, 70, 40, BF16)
    want = sparc_b200.gated_scan(*t, nu, state=h0, segment_pos=pos)
    w = torch.ones(40, device="cuda")
    with torch.inference_mode():
        assert torch.equal(sparc_b200.gated_scan(*t, nu, state=h0, segment_pos=pos), want)
        g = [torch.ones(10, device="cuda")]
        sparc_b200.clip_grads(g, 0.5)
        ln = sparc_b200.layer_norm(want, w)
    sparc_b200.check_status()

    def f(x, r, w_, n):
        y = sparc_b200.layer_norm(x * 1.0, w)
        return sparc_b200.gated_scan(y, r, w_, n, state=h0, segment_pos=pos) * 2.0

    leaves = [v.clone().requires_grad_(True) for v in (*t, nu)]
    y = f(*leaves)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    c = torch.compile(f, backend="eager")
    yc = c(*leaves)
    assert torch.equal(y, yc) and ln.shape == want.shape
    for a, b in zip(grads, torch.autograd.grad(yc, leaves, torch.ones_like(yc))):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ one token

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low", [0.5, 0.7])
@pytest.mark.parametrize("B,D", [(1, 1), (1, 512), (3, 65), (257, 130), (40000, 2), (64, 2048)])
def test_step(B, D, low, dtype):
    """Against the oracle, and bit for bit the length-1 scan."""
    import sparc_b200

    t, nu, h0, pos = _inputs(B, 1, D, dtype, low=low)
    pos = torch.where(torch.arange(B, device="cuda") % 3 == 1, 0, 4)
    q = [v[:, 0] for v in t]
    y, new = sparc_b200.gated_scan_step(*q, nu, h0, segment_pos=pos)
    assert y.dtype == dtype and new.dtype == F32
    n = [_np(v) for v in (*t, nu)]
    starts = pos.cpu().numpy()[:, None] == 0
    h, last = G.forward(*n, _np(h0), starts)
    bd = G.bounds(*n, None, _np(h0), starts)
    _close(y, h[:, 0], bd["h"][:, 0], "y")
    _close(new, last, bd["last"], "state")
    ys, ls = sparc_b200.gated_scan(*t, nu, state=h0, segment_pos=pos[:, None], return_last=True)
    assert torch.equal(ys[:, 0], y) and torch.equal(ls, new)
    p = torch.cat(q, dim=-1)  # columns of one projection
    y2, new2 = sparc_b200.gated_scan_step(*p.split(D, dim=-1), nu, h0, segment_pos=pos)
    assert torch.equal(y2, y) and torch.equal(new2, new)


def test_steps_follow_the_scan():
    """Decoding token by token after a prefill gives the full scan's states within both bounds."""
    import sparc_b200

    t, nu, h0, pos = _inputs(3, 96, 48, F32)
    y, last = sparc_b200.gated_scan(*t, nu, state=h0, segment_pos=pos, return_last=True)
    _, s = sparc_b200.gated_scan(*(v[:, :60] for v in t), nu, state=h0, segment_pos=pos[:, :60], return_last=True)
    n = [_np(v) for v in (*t, nu)]
    starts = pos.cpu().numpy() == 0
    h, _ = G.forward(*n, _np(h0), starts)
    bd = G.bounds(*n, None, _np(h0), starts)["h"]
    for k in range(60, 96):
        yk, s = sparc_b200.gated_scan_step(*(v[:, k] for v in t), nu, s, segment_pos=pos[:, k])
        _close(yk, h[:, k], bd[:, k], f"token {k}")
    _close(s, h[:, -1], bd[:, -1], "state")


def test_step_starts_drop_the_state():
    import sparc_b200

    t, nu, h0, _ = _inputs(2, 1, 8, F32, segments=False)
    h0[0] = float("nan")
    y, new = sparc_b200.gated_scan_step(*(v[:, 0] for v in t), nu, h0, segment_pos=torch.tensor([0, 3], device="cuda"))
    assert torch.isfinite(y).all() and torch.isfinite(new).all()
