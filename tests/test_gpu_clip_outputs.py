"""Gradient clipping on the GPU into outputs that are not dense."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_refused_calls_leave_the_gradients():
    """An expanded gradient among others, a strided one given twice: nothing has been scaled when the call ends."""
    import sparc_b200

    a, m = torch.full((5,), 3.0, device="cuda"), torch.ones(4, 4, device="cuda")
    for bad in (torch.full((1,), 4.0, device="cuda").expand(4), m.t()[:, ::2]):
        keep = bad.clone()
        with pytest.raises(RuntimeError, match="overlaps"):
            sparc_b200.clip_grads([a, bad, bad], 1.0)
        assert torch.equal(bad, keep) and (a == 3.0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_halves_of_one_matrix(dtype):
    """Two views that interleave, in place, as outputs that are their own gradients, and the one into the other:
    the product by max / (norm + eps), rounded to float32 (its norm by 2^-23 at most) and to the type."""
    import sparc_b200

    x = torch.randn(6, 8, device="cuda").to(dtype)
    whole, half = x.double().norm(), x[:, ::2].double().norm()

    def close(got, scaled):
        assert bool(((got.double() - scaled).abs() <= scaled.abs() * (torch.finfo(dtype).eps / 2 + 3 * 2.0 ** -23)).all())

    m = x.clone()
    sparc_b200.clip_grads([m[:, ::2], m[:, 1::2]], 0.5)
    close(m, x.double() * 0.5 / (whole + 1e-6))
    m = x.clone()
    v = m[:, ::2]
    sparc_b200.clip_grads([v], 0.5, out=[m[:, ::2]])
    close(v, x[:, ::2].double() * 0.5 / (half + 1e-6))
    assert torch.equal(m[:, 1::2], x[:, 1::2])
    m = x.clone()
    sparc_b200.clip_grads([m[:, ::2]], 0.5, out=[m[:, 1::2]])
    close(m[:, 1::2], x[:, ::2].double() * 0.5 / (half + 1e-6))
    assert torch.equal(m[:, ::2], x[:, ::2])
