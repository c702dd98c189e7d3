"""The training operators as a recurrent stack uses them: layer norm, a projection to x and the two
gates, the gated recurrence, the residual, over two blocks and a SPARC mixer block, with the
gradients clipped by their global norm; then decoding with the state a prefill left. Against the
same computation in float64 (torch autograd through the definitions)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F64 = torch.float64


class Block(torch.nn.Module):
    def __init__(self, width):
        super().__init__()
        import sparc_b200

        self.norm = sparc_b200.LayerNorm(width)
        self.proj = torch.nn.Linear(width, 3 * width)
        self.nu_log = torch.nn.Parameter(torch.empty(width).uniform_(0.9, 0.999).log().neg().log())

    def forward(self, x, state=None, segment_pos=None):
        import sparc_b200

        v, r, w = self.proj(self.norm(x)).chunk(3, dim=-1)
        y, last = sparc_b200.gated_scan(v, r, w, self.nu_log, state=state, segment_pos=segment_pos, return_last=True)
        return x + y, last

    def step(self, x, state):
        import sparc_b200

        v, r, w = self.proj(self.norm(x)).chunk(3, dim=-1)
        y, new = sparc_b200.gated_scan_step(v, r, w, self.nu_log, state)
        return x + y, new


def _exact(x, params, pos):
    """Two blocks in float64; params: (weight, bias, proj weight, proj bias, nu_log) each."""
    for g, b, pw, pb, nu in params:
        n = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * g + b
        v, r, w = (n @ pw.t() + pb).chunk(3, dim=-1)
        u = -nu.exp() * torch.sigmoid(r)
        c = u.exp() * (pos != 0).unsqueeze(-1)
        b_t = (-torch.expm1(2 * u)).sqrt() * torch.sigmoid(w) * v
        h, out = torch.zeros_like(x[:, 0]), []
        for t in range(x.shape[1]):
            h = c[:, t] * h + b_t[:, t]
            out.append(h)
        x = x + torch.stack(out, 1)
    return x


def test_training_step_and_decode():
    """float32: every value within 1e-4 of the largest of its tensor. (The projections are float32
    matrix products, exact to about 1e-6 of their terms; through two blocks, each a norm and 60 steps
    of the recurrence, and the gradient's sums over 180 tokens, less than a hundred such roundings add.)"""
    import sparc_b200

    torch.backends.cuda.matmul.allow_tf32 = False
    torch.manual_seed(0)
    blocks = torch.nn.ModuleList(Block(48) for _ in range(2)).cuda()
    x = torch.randn(3, 60, 48, device="cuda")
    target = torch.randn(3, 60, 48, device="cuda")
    pos = torch.arange(60, device="cuda").expand(3, 60).clone()
    pos[1, 20:] -= 20
    pos[2, 33:] -= 33

    y = x
    for b in blocks:
        y, _ = b(y, segment_pos=pos)
    loss = (y - target).square().sum()
    loss.backward()
    got = {n: p.grad.clone() for n, p in blocks.named_parameters()}
    norm = sparc_b200.clip_grad_norm_(blocks.parameters(), 1.0)

    ps = {n: p.detach().to(F64).requires_grad_(True) for n, p in blocks.named_parameters()}
    params = [(ps[f"{i}.norm.weight"], ps[f"{i}.norm.bias"], ps[f"{i}.proj.weight"], ps[f"{i}.proj.bias"], ps[f"{i}.nu_log"])
              for i in range(2)]
    ye = _exact(x.to(F64), params, pos)
    le = (ye - target.to(F64)).square().sum()
    ge = dict(zip(ps, torch.autograd.grad(le, list(ps.values()))))
    assert float((y.detach().to(F64) - ye).abs().max() / ye.abs().max()) < 1e-4
    for n in ps:
        assert float((got[n].to(F64) - ge[n]).abs().max() / ge[n].abs().max()) < 1e-4, n
    ne = torch.stack([g.square().sum() for g in ge.values()]).sum().sqrt()
    assert abs(float(norm) / float(ne) - 1) < 1e-4
    for n, p in blocks.named_parameters():
        want = ge[n] / (ne + 1e-6)
        assert float((p.grad.to(F64) - want).abs().max() / want.abs().max()) < 2e-4, n

    # the same tokens: a prefill of 40, then one at a time
    with torch.no_grad():
        full = x
        for b in blocks:
            full, _ = b(full)
        h, states = x[:, :40], []
        for b in blocks:
            h, s = b(h)
            states.append(s)
        for t in range(40, 60):
            v = x[:, t]
            for i, b in enumerate(blocks):
                v, states[i] = b.step(v, states[i])
            assert float((v - full[:, t]).abs().max() / full.abs().max()) < 1e-4
    sparc_b200.check_status()


def test_truncated_sequences_carry_the_state():
    """A sequence in two pieces with the state between them: the second piece's outputs, the state's
    gradient through the first, and the parameter gradients of both pieces together are those of the
    whole sequence (float32, to 1e-5 of each tensor's largest value: the two differ in how the
    recurrence's maps are composed, a few roundings per chunk)."""
    import sparc_b200

    torch.manual_seed(1)
    t = [torch.randn(2, 300, 70, device="cuda", requires_grad=True) for _ in range(3)]
    nu = torch.empty(70, device="cuda").uniform_(0.9, 0.999).log_().neg_().log_().requires_grad_(True)
    g = torch.randn(2, 300, 70, device="cuda")
    whole = sparc_b200.gated_scan(*t, nu)
    ref = torch.autograd.grad(whole, t + [nu], g)
    y1, s = sparc_b200.gated_scan(*(v[:, :130] for v in t), nu, return_last=True)
    y2 = sparc_b200.gated_scan(*(v[:, 130:] for v in t), nu, state=s)
    y = torch.cat([y1, y2], 1)
    assert float((y - whole).abs().max() / whole.abs().max()) < 1e-5
    for a, b in zip(torch.autograd.grad(y, t + [nu], g), ref):
        assert float((a - b).abs().max() / b.abs().max()) < 1e-5


def test_captured_training_step():
    """The whole step (norm, recurrence, gradients, clipping) in one CUDA graph, replayed on new
    inputs: bit for bit the eager step."""
    import sparc_b200

    torch.manual_seed(2)
    norm = sparc_b200.LayerNorm(64).cuda()
    nu = torch.nn.Parameter(torch.empty(64, device="cuda").uniform_(0.9, 0.999).log_().neg_().log_())
    params = [norm.weight, norm.bias, nu]

    def step(x, r, w, dy):
        y = sparc_b200.gated_scan(norm(x), r, w, nu)
        grads = list(torch.autograd.grad(y, params, dy))
        n = sparc_b200.clip_grads(grads, 0.5)
        return [y.detach(), n, *grads]

    sets = [[torch.randn(2, 100, 64, device="cuda").bfloat16() for _ in range(4)] for _ in range(2)]
    want = [[t.clone() for t in step(*s)] for s in sets]
    static = [t.clone() for t in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for s, ref in zip(sets, want):
        for a, b in zip(static, s):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref))
