"""The new operators as a user runs them together: a small gated recurrent network (norm - projection - scan - projection -
norm / gate / residual, twice) trained by FusedMuon (matrices) and FusedAdam (vectors), against the same network in float64 torch;
continued token by token; captured."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
D, H, B, T = 40, 48, 3, 37


class Net(torch.nn.Module):
    def __init__(self):
        from cpcsv import modules as M
        super().__init__()
        self.first = M.RMSNorm(D)
        self.rec = torch.nn.ModuleList([M.GatedRecurrence(D, H), M.GatedRecurrence(D, H, out_gate=False)])
        self.out = torch.nn.ModuleList([M.Linear(H, D), M.Linear(H, D)])
        self.norm = torch.nn.ModuleList([M.NormResidual(D, scale=0.5), M.NormResidual(D, last=True)])

    def dense(self, lin, u):
        from cpcsv import _lib, modules as M
        lay = M._layer_for(lin, None, _lib.ACT_NONE, 0, out_mode="f32")
        return lay(u.reshape(-1, H).float()).view(u.shape[:-1] + (D,))

    def forward(self, x, cond, lengths=None, states=None):
        z = self.first(x)
        last = []
        for i in range(2):
            y, h = self.rec[i](z, states[i] if states is not None else None, lengths)
            last.append(h)
            u = self.dense(self.out[i], y)
            if i == 0:
                x, z = self.norm[0](x, u, gate=cond[:, None, :])
            else:
                x = self.norm[1](x, u)
        return x, last

    def token(self, x, cond, states):
        z = self.first(x)
        for i in range(2):
            u = self.dense(self.out[i], self.rec[i].step(z, states[i]))
            if i == 0:
                x, z = self.norm[0](x, u, gate=cond)
            else:
                x = self.norm[1](x, u)
        return x


def reference(sd, x, cond, lengths):
    """The network in float64 from its state dict, padded tokens' outputs left out by the caller."""
    rms = lambda a, w: a / torch.sqrt(a.square().mean(-1, keepdim=True) + 1e-6) * w
    z = rms(x, sd["first.weight"])
    for i in range(2):
        p = z @ sd["rec.%d.proj.weight" % i].T + sd["rec.%d.proj.bias" % i]
        f, v = torch.sigmoid(p[..., :H]), p[..., H:2 * H]
        h, ys = torch.zeros(B, H, dtype=torch.float64), []
        for t in range(x.shape[1]):
            on = (t < lengths)[:, None]
            h = torch.where(on, f[:, t] * h + (1 - f[:, t]) * v[:, t], h)
            ys.append(torch.where(on, h, 0.0))
        y = torch.stack(ys, 1)
        if i == 0:
            y = y * torch.nn.functional.silu(p[..., 2 * H:])
        u = y @ sd["out.%d.weight" % i].T + sd["out.%d.bias" % i]
        r = rms(u, sd["norm.%d.weight_post" % i])
        if i == 0:
            x = x + sd["norm.0.scale"] * cond[:, None] * r
            z = rms(x, sd["norm.0.weight_next"])
        else:
            x = x + r
    return x


@pytest.fixture(autouse=True)
def _fp32():
    from cpcsv import runtime
    keep = runtime.compute_dtype_name()
    runtime.set_compute_dtype("fp32")
    yield
    runtime.set_compute_dtype(keep)


def data():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g)
    return r(B, T, D), r(B, D), torch.tensor([T, 20, 5], dtype=torch.int32), r(B, T, D)


def build():
    torch.manual_seed(5)
    return Net().cuda()


def test_gradients_match_float64():
    """Every value passes some twenty fp32 operators of a few hundred roundings, each amplified by norms of order 1: 1e-4 of each
    gradient's largest entry leaves two orders of magnitude to what single operators are held to elsewhere."""
    x, cond, n, w = data()
    net = build()
    live = (torch.arange(T)[None, :, None] < n[:, None, None])
    xg, cg = x.cuda().requires_grad_(), cond.cuda().requires_grad_()
    out, _ = net(xg, cg, n.cuda())
    names = [k for k, _ in net.named_parameters()]
    grads = torch.autograd.grad((out * (w * live).cuda()).sum(), [xg, cg] + list(net.parameters()))
    sd = {k: v.detach().cpu().double().requires_grad_() for k, v in net.named_parameters()}
    xr, cr = x.double().requires_grad_(), cond.double().requires_grad_()
    ref = reference(sd, xr, cr, n)
    want = torch.autograd.grad((ref * w * live).sum(), [xr, cr] + [sd[k] for k in names])
    assert ((out.detach().cpu().double() - ref.detach()).abs() * live).max() < 1e-4
    for k, a, b in zip(["x", "cond"] + names, grads, want):
        assert (a.cpu().double() - b).abs().max() < 1e-4 * max(1.0, b.abs().max().item()), k


def test_tokens_continue_the_sequence():
    """States kept from a prefix, the rest token by token: the sequence's own outputs (the same operators in another order of sums
    where a chunk's border falls: 1e-5)."""
    x, cond, _, _ = data()
    net = build()
    xg, cg = x.cuda(), cond.cuda()
    with torch.no_grad():
        whole, _ = net(xg, cg)
        _, states = net(xg[:, :20], cg)
        got = torch.stack([net.token(xg[:, t], cg, states) for t in range(20, T)], 1)
    assert (got - whole[:, 20:]).abs().max() < 1e-5 * whole.abs().max()


def train(net, steps):
    from cpcsv.optim import FusedAdam, FusedMuon
    x, cond, n, w = (t.cuda() for t in data())
    mats = [p for p in net.parameters() if p.dim() >= 2]
    vecs = [p for p in net.parameters() if p.dim() < 2]
    muon, adam = FusedMuon(mats, lr=0.01, weight_decay=0.01), FusedAdam(vecs, lr=1e-3)
    params = mats + vecs
    for p in params:
        p.grad = torch.zeros_like(p)

    def step():
        out, _ = net(x, cond, n)
        for p, g in zip(params, torch.autograd.grad((out * w).sum(), params)):
            p.grad.copy_(g)
        muon.step()
        adam.step()
    for _ in range(steps):
        step()
    return step


def test_training_runs_repeat_and_replay():
    """Three eager steps twice: the same bits (operand caches follow FusedMuon's writes, no sum depends on the run); two steps and a
    replay of a captured third: the same again."""
    nets = [build() for _ in range(3)]
    before = copy.deepcopy(nets[0].state_dict())
    train(nets[0], 3)
    train(nets[1], 3)
    step = train(nets[2], 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    graph.replay()
    torch.cuda.synchronize()
    for (k, a), b, c in zip(nets[0].named_parameters(), nets[1].parameters(), nets[2].parameters()):
        assert torch.equal(a, b), k
        assert torch.equal(a, c), k
        assert torch.isfinite(a).all() and not torch.equal(a, before[k]), k


def test_bf16_projections_reach_the_scan():
    """Large projections multiply in the compute dtype: p and y are bfloat16 then, padded columns are cut off, gradients flow back."""
    from cpcsv import modules as M, runtime
    runtime.set_compute_dtype("bf16")
    torch.manual_seed(1)
    rec = M.GatedRecurrence(1500, 500).cuda()
    x = torch.randn(2, 70, 1500).cuda().requires_grad_()
    y, h = rec(x)
    assert y.dtype == torch.bfloat16 and y.shape == (2, 70, 500) and h.dtype == torch.float32
    gx, gw = torch.autograd.grad([y, h], [x, rec.proj.weight], [torch.ones_like(y), torch.ones_like(h)])
    assert gx.shape == x.shape and torch.isfinite(gx).all() and gw.abs().sum() > 0
    state = torch.zeros(2, 500).cuda()
    step = torch.stack([rec.step(x[:, t], state) for t in range(3)], 1)
    # a product's sums may run in another order for 2 rows than for 140: a bf16 step of p at most, 2^-8 of values below 8
    assert (step.float() - y[:, :3].float()).abs().max() < 2.0 ** -4


def test_modules_refuse():
    from cpcsv import modules as M
    rec = M.GatedRecurrence(8, 4).cuda()
    for x in (torch.zeros(2, 8).cuda(), torch.zeros(2, 3, 9).cuda()):
        with pytest.raises(ValueError, match="GatedRecurrence"):
            rec(x)
    with pytest.raises(ValueError, match="GatedRecurrence"):
        rec.step(torch.zeros(2, 3, 8).cuda(), torch.zeros(2, 4).cuda())


def test_gradients_of_gradients_are_refused():
    """create_graph=True gives first derivatives; a second one through the operators raises."""
    from cpcsv import functional as F
    p = torch.randn(2, 40, 12, device="cuda", requires_grad=True)
    x = torch.randn(2, 40, 4, device="cuda", requires_grad=True)
    w = torch.ones(4, device="cuda")
    for f, leaf in ((lambda: F.gated_scan(p)[0], p), (lambda: F.norm_residual(x, x, w), x), (lambda: F.rms_norm(x, w), x)):
        want, = torch.autograd.grad(f().square().sum(), leaf)
        got, = torch.autograd.grad(f().square().sum(), leaf, create_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            got.sum().backward()
