"""The global gradient norm and clipping by it on the GPU (sparc_b200.grad_norm, clip_grads,
clip_grad_norm_) against float64.

Tolerances, U = 2^-24: a thread's group of squares is summed in float32 (at most 9 U, all terms
positive), everything else in float64, so the norm is off by 5 U and its own rounding by U; the
factor by as much and its rounding, the product by half a step of the gradient's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def _grads(sizes, seed=0, scale=1.0, dtypes=(F32,)):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def _norm(grads):
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()


def _check(grads, max_norm, eps=1e-6, out=False):
    import sparc_b200

    ref = _norm(grads)
    k = min(1.0, max_norm / (float(ref) + eps))
    before = [g.clone() for g in grads]
    n0 = sparc_b200.grad_norm(grads)
    assert n0.shape == () and n0.dtype == F32 and all(torch.equal(a, b) for a, b in zip(grads, before))
    target = [torch.full_like(g, 5.0) for g in grads] if out else None
    norm = sparc_b200.clip_grads(grads, max_norm, out=target, eps=eps)
    assert torch.equal(norm, n0)
    assert abs(float(norm) - float(ref)) <= 6 * U * float(ref)
    for b, g, t in zip(before, grads, target or grads):
        want = b.double() * k
        half = torch.finfo(b.dtype).eps / 2
        # the factor 7 U, a bfloat16 product twice rounded (float32, then its type)
        tol = want.abs() * (8 * U + half * (1 + 8 * U)) + 1e-44
        assert bool(((t.double() - want).abs() <= tol).all())
        if out:
            assert torch.equal(b, g)
        if k == 1.0:
            assert torch.equal(t, b)
    return norm


@pytest.mark.parametrize("out", [False, True])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e6, float("inf")])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F32, BF16)])
def test_sizes_and_types(dtypes, max_norm, out):
    """Empty tensors, one element, a chunk's border and one past it, several dimensions."""
    sizes = [(1,), (0,), (7,), (8,), (9,), (256,), (8191,), (8192,), (8193,), (3, 5, 7), (130, 257), (), (100000,)]
    _check(_grads(sizes, dtypes=dtypes), max_norm, out=out)


def test_many_tensors():
    """More tensors than one launch takes, and more chunks than CTAs."""
    _check(_grads([(k % 97 + 1,) for k in range(700)], dtypes=(F32, BF16)), 1.0)
    _check(_grads([(3000, 3001), (5,), (4096, 512)]), 0.1)
    _check(_grads([(1,)] * 256 + [(2,)]), 0.1)


def test_one_element_each():
    for dtype in (F32, BF16):
        _check(_grads([(1,)], dtypes=(dtype,)), 1e-3)


def test_only_empty_tensors():
    import sparc_b200

    g = [torch.empty(0, device="cuda"), torch.empty(0, 4, device="cuda")]
    assert float(sparc_b200.grad_norm(g)) == 0.0
    assert float(sparc_b200.clip_grads(g, 1.0)) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_extreme_magnitudes(dtype):
    """Squares that overflow or underflow float32, alone and among ordinary ones."""
    for scale in (1e-30, 1e-22, 1e22, 1e30):
        _check(_grads([(1000,), (77,)], scale=scale, dtypes=(dtype,)), scale, eps=0.0)
    g = _grads([(1000,), (1000,)], dtypes=(dtype,))
    g[0][:500] *= 1e30
    g[1][3] = 1e-30
    _check(g, 1.0)
    z = [torch.zeros(5000, dtype=dtype, device="cuda")]
    assert float(_check(z, 1.0)) == 0.0


def test_not_finite():
    """A NaN makes the norm and every gradient NaN; an infinity makes the norm infinite, the factor
    0, so the other gradients become 0 and itself NaN. With max_norm infinite nothing is touched."""
    import sparc_b200

    g = _grads([(100,), (9000,)])
    g[1][8999] = float("nan")
    assert torch.isnan(sparc_b200.clip_grads(g, 1.0)) and all(torch.isnan(t).all() for t in g)
    g = _grads([(100,), (9000,)])
    g[1][10] = float("inf")
    keep = [t.clone() for t in g]
    assert torch.isinf(sparc_b200.clip_grads(g, float("inf"))) and all(torch.equal(a, b) for a, b in zip(g, keep))
    assert torch.isinf(sparc_b200.clip_grads(g, 1.0))
    assert torch.isnan(g[1][10]) and not g[0].any() and not g[1][:10].any()


def test_strides_and_alignment():
    """Transposed, sliced and misaligned gradients, in place and into strided outputs."""
    import sparc_b200

    base = _grads([(64, 96), (50, 40), (1001,)])
    make = lambda: [base[0].clone().t(), base[1].clone()[:, ::2], base[2].clone()[1:]]  # noqa: E731
    _check(make(), 0.5)
    g = make()
    ref = _norm(g)
    out = [torch.empty(64, 96, device="cuda").t(), torch.empty(50, 40, device="cuda")[:, ::2],
           torch.empty(1003, device="cuda")[3:]]
    norm = sparc_b200.clip_grads(g, 0.5, out=out)
    for a, o in zip(g, out):
        want = a.double() * (0.5 / (float(ref) + 1e-6))
        assert bool(((o.double() - want).abs() <= want.abs() * 9 * U).all())
    assert abs(float(norm) - float(ref)) <= 6 * U * float(ref)
    buf = torch.full((400,), 9.0, dtype=BF16, device="cuda")  # neighbours of a slice stay
    buf[101:300] = 1.0
    sparc_b200.clip_grads([buf[101:300]], 0.1)
    assert (buf[:101] == 9).all() and (buf[300:] == 9).all() and (buf[101:300] < 1).all()


def test_overlaps_are_refused():
    import sparc_b200

    t = torch.ones(100, device="cuda")
    for bad in ([t, t], [t[:60], t[50:]], [t, t[99:]]):
        with pytest.raises(RuntimeError, match="overlaps"):
            sparc_b200.clip_grads(bad, 0.5)
    with pytest.raises(RuntimeError, match="overlaps"):
        sparc_b200.clip_grads([t[:50], t[50:]], 0.5, out=[t[50:], t[:50]])
    with pytest.raises(RuntimeError, match="overlaps"):
        sparc_b200.clip_grads([t[:50]], 0.5, out=[t[1:51]])
    assert (t == 1).all()
    assert abs(float(sparc_b200.grad_norm([t, t])) - 200 ** 0.5) < 1e-5  # read only: counted twice


def test_parameters():
    import sparc_b200

    torch.manual_seed(0)
    m = sparc_b200.SPARCMixer(64).cuda()
    m(torch.randn(2, 30, 64, device="cuda"))[0].square().sum().backward()
    grads = [p.grad.clone() for p in m.parameters() if p.grad is not None]
    ps = list(m.parameters())
    unused = torch.nn.Parameter(torch.ones(3, device="cuda"))
    norm = sparc_b200.clip_grad_norm_(ps + [ps[0], unused], 0.5)
    ref = _norm(grads)
    assert abs(float(norm) - float(ref)) <= 6 * U * float(ref)
    k = min(1.0, 0.5 / (float(ref) + 1e-6))
    for p, g in zip((p for p in ps if p.grad is not None), grads):
        assert bool(((p.grad.double() - g.double() * k).abs() <= g.double().abs() * k * 9 * U).all())
    assert float(sparc_b200.clip_grad_norm_(unused, 1.0)) == 0.0
    p = torch.nn.Parameter(torch.ones(3, device="cuda"))
    p.grad = torch.full((3,), 2.0, device="cuda")
    sparc_b200.clip_grad_norm_(p, 1.0)
    assert abs(float(p.grad.norm()) - 1.0) < 1e-5
    sparc_b200.clip_grad_norm_((q for q in [p]), 0.5)  # a generator
    assert abs(float(p.grad.norm()) - 0.5) < 1e-5


def test_reproducible_streams_and_graphs():
    import sparc_b200

    g = _grads([(100000,), (33, 3), (2048, 300)], dtypes=(F32, BF16))
    norms = [sparc_b200.grad_norm(g) for _ in range(5)]
    assert all(torch.equal(n, norms[0]) for n in norms)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(sparc_b200.grad_norm(g), norms[0])
    torch.cuda.synchronize()
    want = [torch.empty_like(t) for t in g]
    sparc_b200.clip_grads(g, 0.5, out=want)
    runs = []
    for _ in range(2):
        static = [torch.zeros_like(t) for t in g]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n = sparc_b200.clip_grads(static, 0.5)
        for a, b in zip(static, g):
            a.copy_(b)
        runs.append((graph, static, n))
    torch.cuda.synchronize()
    for graph, _, _ in runs:
        with torch.cuda.stream(torch.cuda.Stream()):
            graph.replay()
    torch.cuda.synchronize()
    for _, static, n in runs:
        assert torch.equal(n, norms[0]) and all(torch.equal(a, b) for a, b in zip(static, want))


@pytest.mark.parametrize("shape", [(1,), (5, 3)])
def test_negated_views(shape):
    """Gradients that PyTorch holds with the sign of their memory reversed, in place and into such outputs."""
    import sparc_b200

    g = torch.full(shape, 2.0, device="cuda")
    n = float(g.square().sum().sqrt())

    def negated(v):
        return torch.complex(torch.zeros_like(v), -v).conj().imag

    a = negated(g)
    assert a.is_neg()
    assert abs(float(sparc_b200.clip_grads([a], n / 2, eps=0.0)) - n) <= 6 * U * n
    assert bool(((a - 1.0).abs() <= 16 * U).all())
    o = negated(torch.zeros_like(g))
    sparc_b200.clip_grads([g], n / 2, out=[o], eps=0.0)
    assert bool(((o - 1.0).abs() <= 16 * U).all()) and bool((g == 2.0).all())
