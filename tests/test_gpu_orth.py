"""Orthogonalised updates (cpcsv.optim.orthogonalize / FusedMuon, csrc/orth.hip) against the iteration in float64.

Tolerance: one step maps singular values by f(x) = a x + b x^3 + c x^5; on [0, 1.21] (where they stay) |f'| <= 3.9, and so are the
divided differences that carry a perturbation of X to the next step. Rounding in one step - the planes' 2^-24, sums of 3 K / 16
partial products whose roundings have random signs, the scaled sum - adds at most (8 + sqrt(3 K / 16)) 2^-23 of |X|_F, K the longer
side. Five steps behind the normalisation: |error|_F <= (1 + 3.9 + ... + 3.9^4) (8 + sqrt(3 K / 16)) 2^-23 |X|_F. That bound knows no
condition number; what is claimed beyond it is fp32's own accuracy: at most four times the error of the same iteration in fp32."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
NS = (3.4445, -4.7750, 2.0315)
GROW = sum(3.9 ** k for k in range(5))


def iterate(g, steps, eps, dtype=torch.float64):
    x = g.to(dtype)
    x = x / (x.norm() + eps)
    x = x.T if g.shape[0] > g.shape[1] else x
    for _ in range(steps):
        a = x @ x.T
        x = NS[0] * x + (NS[1] * a + NS[2] * (a @ a)) @ x
    return x.T if g.shape[0] > g.shape[1] else x


def bound(shape):
    return GROW * (8 + math.sqrt(3 * max(shape) / 16)) * 2.0 ** -23


def check(got, g, steps=5, eps=1e-7):
    got, want = got.cpu(), iterate(g, steps, eps)
    assert got.dtype == g.dtype and got.shape == g.shape
    err, scale = (got.double() - want).norm().item(), want.norm().item()
    half = torch.finfo(g.dtype).eps / 2
    assert err <= (bound(g.shape) + half) * scale, (g.shape, err / max(scale, 1e-300))
    if g.dtype == torch.float32:
        own = (iterate(g, steps, eps, torch.float32).double() - want).norm().item()
        assert err <= 4 * own + 2.0 ** -22 * scale, (g.shape, err, own)
    else:                                                    # each stored value is the fp32 result's nearest
        assert bool(((got.double() - want).abs() <= bound(g.shape) * scale + want.abs() * half * (1 + 2.0 ** -8)).all())


def spectrum(rows, cols, kind, seed):
    g = torch.Generator().manual_seed(seed)
    n = torch.randn(rows, cols, generator=g)
    k = min(rows, cols)
    if kind == "gauss":
        return n
    if kind == "strong":                                      # a few strong directions over noise
        return 0.05 * n + torch.randn(rows, 4, generator=g) @ torch.randn(4, cols, generator=g)
    if kind == "rank":
        return torch.randn(rows, 4, generator=g) @ torch.randn(4, cols, generator=g)
    u = torch.linalg.qr(torch.randn(rows, k, generator=g))[0]
    v = torch.linalg.qr(torch.randn(cols, k, generator=g))[0]
    return (u * torch.logspace(0, -4, k)) @ v.T


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (9, 1), (3, 5), (64, 64), (100, 130), (128, 128), (129, 127), (40, 1000), (700, 33),
                                       (365, 465), (1095, 465), (512, 768), (520, 520)])
def test_orthogonalize_matches_float64(rows, cols, dtype):
    from cpcsv.optim import orthogonalize
    g = spectrum(rows, cols, "gauss", rows + cols).to(dtype)
    check(orthogonalize(g.cuda()), g)


@pytest.mark.parametrize("kind", ["strong", "rank", "logspace"])
@pytest.mark.parametrize("rows,cols", [(192, 768), (256, 256), (500, 130), (130, 2000)])
def test_ill_conditioned_gradients(rows, cols, kind):
    from cpcsv.optim import orthogonalize
    g = spectrum(rows, cols, kind, 3)
    check(orthogonalize(g.cuda()), g)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e30])
def test_scale_does_not_matter(scale):
    """Squares of such gradients leave fp32's range; eps = 0, so that only the direction counts."""
    from cpcsv.optim import orthogonalize
    g = spectrum(70, 90, "gauss", 4)
    a, b = orthogonalize(g.cuda(), eps=0.0), orthogonalize((g * scale).cuda(), eps=0.0)
    assert (a - b).norm() <= bound(g.shape) * a.norm()


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7])
def test_other_step_counts(steps):
    """(the bound's growth factor is that of five steps: more steps than that are held to fp32's own error only)"""
    from cpcsv.optim import orthogonalize
    for rows, cols in ((150, 170), (100, 900)):
        g = spectrum(rows, cols, "gauss", steps)
        got = orthogonalize(g.cuda(), steps=steps).cpu().double()
        want = iterate(g, steps, 1e-7)
        own = (iterate(g, steps, 1e-7, torch.float32).double() - want).norm()
        assert (got - want).norm() <= 4 * own + 2.0 ** -22 * want.norm()


def test_stacks_share_launches_and_keep_bits():
    """19 matrices (more than one job list): each as by itself, bit for bit; twice the same."""
    from cpcsv.optim import orthogonalize
    g = torch.stack([spectrum(90, 140, "gauss", i) for i in range(19)]).cuda()
    out = orthogonalize(g)
    assert torch.equal(out, orthogonalize(g))
    for i in range(19):
        assert torch.equal(out[i], orthogonalize(g[i])), i
    assert orthogonalize(g[:0]).shape == (0, 90, 140)


def test_zero_non_finite_and_strided():
    from cpcsv.optim import orthogonalize
    g = spectrum(60, 80, "gauss", 5).cuda()
    assert not orthogonalize(torch.zeros_like(g)).any()
    stack = torch.stack([g, g, g])
    stack[1, 3, 4] = float("nan")
    out = orthogonalize(stack)
    assert torch.equal(out[0], out[2]) and torch.equal(out[0], orthogonalize(g)) and torch.isnan(out[1]).all()
    assert torch.equal(orthogonalize(g.T.contiguous().T), out[0])
    wide = torch.zeros(60, 99).cuda()
    wide[:, 7:87] = g
    assert torch.equal(orthogonalize(wide[:, 7:87]), out[0])


SHAPES = [(124, 124), (248, 1780), (63, 124), (1095, 465), (16, 8, 3, 3), (40, 3, 4, 4), (7, 2), (1, 64, 3, 3)]


def step64(w, g, m, lr, mu, nesterov, decay, steps=5):
    w, g, m = (t.double().reshape(t.shape[0], -1) for t in (w, g, m))
    m = mu * m + g
    x = iterate(g + mu * m if nesterov else m, steps, 1e-7)
    s = lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
    return w * (1 - lr * decay) - s * x, m, s * x.norm().item()


@pytest.mark.parametrize("nesterov,decay", [(True, 0.0), (False, 0.1)])
def test_muon_steps_match_float64(nesterov, decay):
    """Two steps over matrices of the framework's kinds, the learning rate changed in between; errors of the update are lr-sized."""
    from cpcsv.optim import FusedMuon
    gen = torch.Generator().manual_seed(1)
    ps = [torch.nn.Parameter((0.05 * torch.randn(s, generator=gen)).cuda()) for s in SHAPES] + [torch.nn.Parameter(torch.ones(4, 4).cuda())]
    opt = FusedMuon(ps, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=decay)
    ref = [(p.detach().cpu().double(), torch.zeros(p.shape).double()) for p in ps]
    tol = [0.0] * len(ps)
    for it in range(2):
        lr = (0.02, 0.005)[it]
        opt.param_groups[0]["lr"] = lr
        epochs = [getattr(p, "_cpcsv_epoch", 0) for p in ps]
        for p in ps[:-1]:
            p.grad = torch.randn(p.shape, generator=gen).cuda()
        opt.step()
        for i, p in enumerate(ps[:-1]):
            w, m, size = step64(ref[i][0], p.grad.cpu(), ref[i][1], lr, 0.9, nesterov, decay)
            ref[i] = (w, m)
            tol[i] += bound(w.shape) * size + 3 * 2.0 ** -24 * w.norm().item()
            got = p.detach().cpu().double().reshape(w.shape)
            assert (got - w).norm().item() <= tol[i], (SHAPES[i], it)
            mom = opt.state[p]["momentum_buffer"].cpu().double().reshape(m.shape)
            assert (mom - m).abs().max() <= 4 * 2.0 ** -24 * (it + 1) * m.abs().max()
            assert p._cpcsv_epoch == epochs[i] + 1
    assert torch.equal(ps[-1], torch.ones(4, 4).cuda()) and not opt.state[ps[-1]]       # (no gradient: untouched)


def test_muon_many_groups_and_state_dict():
    """20 matrices in two groups (two job lists); a run resumed from a state dict continues with the same bits."""
    from cpcsv.optim import FusedMuon
    gen = torch.Generator().manual_seed(2)
    w0 = [torch.randn(20 + i, 50, generator=gen) for i in range(20)]
    grads = [[torch.randn(w.shape, generator=gen).cuda() for w in w0] for _ in range(2)]

    def start():
        ps = [torch.nn.Parameter(w.cuda()) for w in w0]
        return ps, FusedMuon([{"params": ps[:18]}, {"params": ps[18:], "lr": 0.1, "nesterov": False}], lr=0.01)

    def one(ps, opt, gs):
        for p, g in zip(ps, gs):
            p.grad = g
        opt.step()
    pa, oa = start()
    one(pa, oa, grads[0])
    pb, ob = start()
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))        # (load_state_dict keeps the tensors it is given)
    with torch.no_grad():
        for p, q in zip(pb, pa):
            p.copy_(q)
    one(pa, oa, grads[1])
    one(pb, ob, grads[1])
    for p, q in zip(pa, pb):
        assert torch.equal(p, q)
    w, _, size = step64(w0[19], grads[0][19].cpu(), torch.zeros(39, 50), 0.1, 0.95, False, 0.0)
    pc, oc = start()
    one(pc, oc, grads[0])
    assert (pc[19].detach().cpu().double() - w).norm() <= bound(w.shape) * size + 3 * 2.0 ** -24 * w.norm()


def test_muon_captured_steps_follow_the_learning_rate():
    """A captured step replayed with eager work in between, the learning rate pushed by sync_lr(): the eager run's bits."""
    from cpcsv.optim import FusedMuon
    gen = torch.Generator().manual_seed(3)
    w0 = [torch.randn(s, generator=gen) for s in ((150, 200), (64, 3, 4, 4))]
    gs = [[torch.randn(w.shape, generator=gen).cuda() for w in w0] for _ in range(4)]

    def start():
        ps = [torch.nn.Parameter(w.cuda()) for w in w0]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, FusedMuon(ps, lr=0.02, weight_decay=0.1)
    pe, oe = start()
    for i, g in enumerate(gs):
        oe.param_groups[0]["lr"] = 0.02 / (i + 1)
        for p, q in zip(pe, g):
            p.grad.copy_(q)
        oe.step()
    pg, og = start()
    for p, q in zip(pg, gs[0]):
        p.grad.copy_(q)
    og.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        og.step()
    for i, g in enumerate(gs[1:]):
        og.param_groups[0]["lr"] = 0.02 / (i + 2)
        og.sync_lr()
        for p, q in zip(pg, g):
            p.grad.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
    for p, q in zip(pe, pg):
        assert torch.equal(p, q)


def test_side_stream():
    from cpcsv.optim import orthogonalize
    g = spectrum(300, 200, "gauss", 6).cuda()
    want = orthogonalize(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = orthogonalize(g)
    s.synchronize()
    assert torch.equal(got, want)


def test_muon_refuses_on_the_gpu():
    from cpcsv.optim import FusedMuon
    for w, g in ((torch.zeros(4, 6).cuda().T, None), (torch.zeros(4, 6).cuda().double(), None), (torch.zeros(4, 6).cuda(), torch.zeros(6, 4).cuda().T)):
        p = torch.nn.Parameter(w)
        p.grad = torch.zeros_like(p) if g is None else g
        with pytest.raises(RuntimeError, match="contiguous fp32"):
            FusedMuon([p]).step()
    p = torch.nn.Parameter(torch.zeros(4, 6).cuda())
    p.grad = torch.zeros_like(p)
    opt = FusedMuon([p])
    opt.state[p]["momentum_buffer"] = torch.zeros(6, 4).cuda()
    with pytest.raises(RuntimeError, match="momentum"):
        opt.step()
    q = torch.nn.Parameter(torch.zeros(4, 6).cuda())
    late = FusedMuon([torch.nn.Parameter(torch.zeros(4, 6).cuda()), q])
    late.param_groups[0]["params"][0].grad = torch.zeros(4, 6).cuda()
    late.step()
    q.grad = torch.ones_like(q)
    with pytest.MonkeyPatch.context() as m:                  # (its first gradient arrives while a step is captured)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="without momentum during capture"):
            late.step()
        with pytest.raises(RuntimeError, match="run one step before"):
            other = FusedMuon([q])
            other.state[q]["momentum_buffer"] = torch.zeros_like(q)
            other.step()
    late.step()
    assert not torch.equal(q, torch.zeros_like(q))


# padded sides by what they reach: whole and sliced tiles of the three shapes, both orientations
LARGE = [(2049, 2050), (1600, 5200), (6400, 2816), (900, 16300), (2304, 5376), (4990, 5000), (5700, 5760)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", LARGE)
def test_large_matrices(rows, cols, dtype):
    from cpcsv.optim import orthogonalize
    g = torch.randn(rows, cols, generator=torch.Generator("cuda").manual_seed(rows), device="cuda").to(dtype)
    got, want = orthogonalize(g), iterate(g, 5, 1e-7)
    err, scale = (got.double() - want).norm().item(), want.norm().item()
    assert err <= (bound(g.shape) + torch.finfo(dtype).eps / 2) * scale, err / scale
    if dtype == torch.float32:
        own = (iterate(g, 5, 1e-7, torch.float32).double() - want).norm().item()
        assert err <= 4 * own + 2.0 ** -22 * scale, (err, own)
    assert torch.equal(got, orthogonalize(g))


@pytest.mark.parametrize("rows,cols", [(5200, 1600), (6400, 2816), (900, 16300), (2049, 2050)])
def test_muon_large_matrices(rows, cols):
    """The weight is updated in the tail of the last products: tall, wide, joined from slices; a small matrix beside it."""
    from cpcsv.optim import FusedMuon
    gen = torch.Generator("cuda").manual_seed(cols)
    ps = [torch.nn.Parameter(0.05 * torch.randn(s, generator=gen, device="cuda")) for s in ((rows, cols), (70, 90))]
    opt = FusedMuon(ps, lr=0.02, momentum=0.9, weight_decay=0.1)
    want = []
    for p in ps:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda")
        w, _, size = step64(p.detach(), p.grad, torch.zeros_like(p), 0.02, 0.9, True, 0.1)
        want.append((w, bound(p.shape) * size + 3 * 2.0 ** -24 * w.norm().item()))
    opt.step()
    for p, (w, tol) in zip(ps, want):
        assert (p.detach().double() - w).norm().item() <= tol, tuple(p.shape)


def test_copies_of_the_optimiser_continue():
    import pickle
    from cpcsv.optim import FusedMuon
    p = torch.nn.Parameter(torch.eye(8, 12).cuda())
    p.grad = torch.ones_like(p)
    opt = FusedMuon([p], lr=0.1)
    opt.step()
    twins = [copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))]
    opt.step()
    for t in twins:
        q = t.param_groups[0]["params"][0]
        q.grad = torch.ones_like(q)
        t.step()
        assert torch.equal(q, p)


def test_two_calls_at_once():
    from cpcsv.optim import orthogonalize
    gs = [spectrum(600, 900, "gauss", i).cuda() for i in (7, 8)]
    want = [orthogonalize(g) for g in gs]
    streams = [torch.cuda.Stream() for _ in gs]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for g, s in zip(gs, streams):
            with torch.cuda.stream(s):
                got.append(orthogonalize(g))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 2]), i
