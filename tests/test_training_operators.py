"""What the operators of recurrent training refuse or declare, without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import sparc_b200
from sparc_b200 import torch_ops


@pytest.fixture(scope="module", autouse=True)
def built():
    from sparc_b200 import _build

    _build.build()
    _build.build_torch_ops()


def test_forward_mode_is_refused():
    """A tangent that an operator cannot carry on is refused, in whichever input it comes, also where no
    gradient is recorded; without forward mode the same call goes on to the check of its device."""
    x3, x2, w, s = torch.ones(2, 3, 8), torch.ones(2, 8), torch.ones(8), torch.ones(2, 8)
    calls = {
        "gated_scan": (lambda *a: sparc_b200.gated_scan(*a[:4], state=a[4]), [x3, x3, x3, w, s]),
        "gated_scan_step": (sparc_b200.gated_scan_step, [x2, x2, x2, w, s]),
        "layer_norm": (sparc_b200.layer_norm, [x3, w, w]),
        "grad_norm": (lambda *a: sparc_b200.grad_norm(a), [x2, w]),
        "clip_grads": (lambda *a: sparc_b200.clip_grads(a[:2], 1.0, out=a[2:]), [x2, w, x2.clone(), w.clone()]),
    }
    for name, (f, args) in calls.items():
        for k in range(len(args)):
            with fwAD.dual_level():
                dual = [fwAD.make_dual(a, torch.ones_like(a)) if i == k else a for i, a in enumerate(args)]
                with pytest.raises(NotImplementedError, match="forward"):
                    f(*dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
                    f(*dual)
                with fwAD._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="CUDA"):
                    f(*dual)
        with pytest.raises(RuntimeError, match="CUDA"):
            f(*args)


def test_clip_refuses_outputs_that_overlap():
    """Outputs that are not dense are refused like dense ones, before anything is scaled: an expanded one, one
    view twice, a transposed view of a gradient; halves of one matrix go on to the check of their device."""
    m = torch.ones(4, 4)
    half, square = m[:, ::2], torch.ones(4, 4)
    bad = {
        "expanded": ([torch.ones(3), torch.ones(1).expand(4)], None),
        "expanded rows": ([torch.ones(3, 1).expand(3, 2)], None),
        "one strided view twice": ([half, m[:, ::2]], None),
        "one strided tensor twice": ([half, half], None),
        "one strided output twice": ([torch.ones(4, 2), torch.ones(4, 2)], [half, m[:, ::2]]),
        "an expanded output": ([torch.ones(4)], [torch.ones(1).expand(4)]),
        "transposed onto its own gradient": ([square], [square.t()]),
        "transposed onto another gradient": ([torch.ones(4, 4), square], [square.t(), torch.ones(4, 4)]),
    }
    for name, (grads, out) in bad.items():
        with pytest.raises(RuntimeError, match="overlaps"):
            sparc_b200.clip_grads(grads, 1.0, out=out)
            raise AssertionError(name)
    fine = [([half, m[:, 1::2]], None), ([half], [half]), ([half], [m[:, ::2]]), ([half.contiguous(), half], [m[:, 1::2], half]),
            ([square], [torch.ones(4, 4).t()]), ([torch.ones(0, 1).expand(0, 3)] * 2, None)]
    for grads, out in fine:
        with pytest.raises(RuntimeError, match="CUDA"):
            sparc_b200.clip_grads(grads, 1.0, out=out)
    with pytest.raises(RuntimeError, match="CUDA"):
        sparc_b200.grad_norm([half, half, torch.ones(1).expand(4)])  # (nothing is written)


def test_schemas_say_what_is_written():
    ops = torch_ops.load()
    written = {name: [a.name for a in getattr(ops, name).default._schema.arguments if a.alias_info and a.alias_info.is_write]
               for name in ("gated_scan", "gated_scan_step", "layer_norm", "grad_clip")}
    assert written == {"gated_scan": [], "gated_scan_step": [], "layer_norm": [], "grad_clip": ["grads", "out"]}
    assert ops.grad_clip.default._schema.is_mutable
