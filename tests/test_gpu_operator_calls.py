"""Calls that the documentation of the gated recurrence, the block norms and the orthogonalised updates allows beside the ordinary ones
(csrc/scan.hip, csrc/blocknorm.hip, csrc/orth.hip): each gives the definition's values or is refused, none goes wrong without a word."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_forward_mode_is_refused():
    """No operator here has a forward-mode derivative: a tangent on any input raises (a result without one would count as a zero
    derivative). Inputs without tangents give the same bits inside a dual level as outside."""
    import torch.autograd.forward_ad as fw
    from cpcsv import functional as F
    from cpcsv.optim import orthogonalize
    r = lambda *s: torch.randn(*s, device="cuda")
    p, h0, x, u, g, w, s, n = r(2, 40, 12), r(2, 4), r(2, 5, 8), r(2, 5, 8), r(2, 1, 8), r(8), r(8), r(8)
    scan = lambda a, b: F.gated_scan(a, b)[0]
    norm = lambda *a: F.norm_residual(*a[:3], gate=a[3], scale=a[4], w_next=a[5])[1]
    step = lambda a, b: F.gated_scan_step(a, b)
    calls = [(scan, (p, h0)), (norm, (x, u, w, g, s, n)), (F.rms_norm, (x, w)), (step, (p[:, 0], h0.clone())), (orthogonalize, (r(6, 9),))]
    for f, args in calls:
        state = args[1].clone() if f is step else None
        want = f(*args)
        if f is step:
            args[1].copy_(state)
        with fw.dual_level():
            got = f(*args)
            assert torch.equal(got, want)
            for i, t in enumerate(args):
                dual = fw.make_dual(t.detach(), torch.ones_like(t))
                for grads in (True, False):
                    with torch.set_grad_enabled(grads), pytest.raises(NotImplementedError):
                        f(*args[:i], dual, *args[i + 1:])


def test_updated_weights_count_as_modified():
    """A backward pass through a graph that saved a weight (or the momentum) from before FusedMuon's step is refused, as after torch's own
    optimisers; a parameter without a gradient is not touched."""
    from cpcsv.optim import FusedMuon
    w, still = (torch.nn.Parameter(torch.randn(6, 9, device="cuda")) for _ in range(2))
    opt = FusedMuon([w, still], lr=0.1)
    w.grad = torch.randn_like(w)
    opt.step()
    m = opt.state[w]["momentum_buffer"]
    x = torch.randn(9, 3, device="cuda", requires_grad=True)
    y, z, q = w @ x, (x[:, 0] * m).sum(), still @ x
    opt.step()
    for out in (y, z):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
    q.sum().backward()
    assert still._version == 0


def test_inference_weights_are_updated():
    """Tensors made in inference mode have no versions; they are stepped all the same."""
    from cpcsv.optim import FusedMuon
    with torch.inference_mode():
        w = torch.nn.Parameter(torch.ones(6, 9, device="cuda"), requires_grad=False)
        w.grad = torch.randn(6, 9, device="cuda")
        opt = FusedMuon([w], lr=0.1)
        for _ in range(2):
            before = w.clone()
            opt.step()
            assert not torch.equal(w, before)


def dense_error(y, x, w, b, cast):
    """|y - (x w^T + b)| over its bound: operands rounded once to `cast` (half a step each), sums of K products in fp32, y stored in fp32."""
    x, w, b = x.detach().double().cpu(), w.detach().double().cpu(), b.detach().double().cpu()
    u = 0.0 if cast == torch.float32 else torch.finfo(cast).eps
    lim = (x.abs() @ w.abs().T) * (u * (1 + u) + (x.shape[1] + 2) * 2.0 ** -24) + b.abs() * 2.0 ** -23
    return ((y.detach().double().cpu() - (x @ w.T + b)).abs() / lim).max().item()


def muon_layer(cin, cout, opt_cls="FusedMuon"):
    """-> layer, its weight, a step with a constant gradient that moves every entry visibly"""
    from cpcsv import modules as M, optim
    torch.manual_seed(3)
    layer = M.FusedSequential(M.Linear(cin, cout), out_mode="f32").cuda()
    w = layer[0].weight
    w.grad = torch.randn_like(w)
    opt = getattr(optim, opt_cls)([w], lr=0.5)
    return layer, w, layer[0].bias, opt


@pytest.fixture
def bf16():
    from cpcsv import runtime
    keep = runtime.compute_dtype_name()
    runtime.set_compute_dtype("bf16")
    yield
    runtime.set_compute_dtype(keep)


@pytest.mark.parametrize("cin,cout,cast", [(40, 24, torch.float32), (2048, 1032, torch.bfloat16)])
def test_eager_layers_follow_replayed_steps(cin, cout, cast, bf16):
    """Only the optimiser's step is captured: every eager forward and backward behind a replay multiplies with the weights of that replay
    (small layers in fp32, larger ones through copies in the compute type)."""
    layer, w, b, opt = muon_layer(cin, cout)
    opt.step()
    x = torch.randn(70, cin, device="cuda", requires_grad=True)
    dy = torch.randn(70, cout, device="cuda")

    def check():
        y = layer(x)
        assert dense_error(y, x, w, b, cast) <= 1
        gx, = torch.autograd.grad(y, x, dy)
        dyc = dy.to(cast).float()
        assert dense_error(gx, dyc, w.T, torch.zeros(cin, device="cuda"), cast) <= 1 if cast == torch.float32 else \
            (gx - dyc @ w.to(cast).float()).abs().max() <= 2.0 ** -7 * (dyc.abs() @ w.abs()).max()
    check()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    check()
    for _ in range(3):
        before = w.detach().clone()
        graph.replay()
        check()
        assert (w - before).norm() > 0.01 * before.norm()
    opt.step()
    check()


@pytest.mark.parametrize("first", [True, False])
def test_captured_layers_follow_later_steps(first, bf16):
    """A captured forward (here without a step in it) reads the weights of its replay, whether the copies it multiplies with were there
    before the capture or not."""
    layer, w, b, opt = muon_layer(40, 24)
    x = torch.randn(70, 40, device="cuda")
    with torch.no_grad():
        layer(x)
        if first:
            opt.step()
        layer(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer(x)
        for _ in range(3):
            opt.step()
            graph.replay()
            torch.cuda.synchronize()
            assert dense_error(y, x, w, b, torch.float32) <= 1
            assert dense_error(layer(x), x, w, b, torch.float32) <= 1


def test_a_captured_training_step_and_eager_evaluations(bf16):
    """Forward, backward and step in one graph, captured behind an eager evaluation, an evaluation behind each replay: the weights and
    outputs of the same steps run eagerly."""
    runs = []
    for captured in (False, True):
        layer, w, b, opt = muon_layer(40, 24)
        gen = torch.Generator("cuda").manual_seed(9)
        x, dy = torch.randn(70, 40, generator=gen, device="cuda"), torch.randn(70, 24, generator=gen, device="cuda")
        w.grad.zero_()

        def step():
            g, = torch.autograd.grad(layer(x), w, dy)
            w.grad.copy_(g)
            opt.step()

        def evaluate():
            with torch.no_grad():
                return layer(x).clone()
        for _ in range(2):
            step()
        outs = [evaluate()]
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        for _ in range(3):
            graph.replay() if captured else step()
            torch.cuda.synchronize()
            outs.append(evaluate())
            assert dense_error(outs[-1], x, w, b, torch.float32) <= 1
        runs.append(outs + [w.detach().clone()])
    for a, c in zip(*runs):
        assert torch.equal(a, c)


def test_eager_layers_follow_replayed_adam_steps(bf16):
    """The same of FusedAdam's captured step."""
    layer, w, b, opt = muon_layer(40, 24, "FusedAdam")
    x = torch.randn(70, 40, device="cuda")
    opt.step()
    layer(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        before = w.detach().clone()
        graph.replay()
        assert dense_error(layer(x), x, w, b, torch.float32) <= 1
        assert not torch.equal(w, before)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [20, 100, 700, 1500])
def test_infinities_stay_infinite(t, dtype):
    """An infinite state (given, or from an infinite v) or gradient stays infinite however many gates it passes: a product of gates that
    underflows is still no zero. Where the definition, run token by token, is finite, infinite or NaN, so is the result."""
    from cpcsv import functional as F
    g = torch.Generator().manual_seed(t)
    h = 6
    p = torch.randn(2, t, 2 * h, generator=g).to(dtype)
    p[..., :h] -= 3.0                                   # gates about 0.05: sixteen tokens leave 1e-21
    h0 = torch.randn(2, h, generator=g)
    h0[0, 0], h0[0, 1], h0[1, 2] = float("inf"), float("-inf"), float("nan")
    p[0, 3, h + 2], p[1, t // 2, h + 3] = float("inf"), float("-inf")
    p[1, 1, h + 4], p[1, t - 2, h + 4] = float("inf"), float("-inf")            # meets its opposite: NaN
    dy, dl = torch.randn(2, t, h, generator=g).to(dtype), torch.randn(2, h, generator=g)
    dl[0, 5], dl[1, 5], dy[1, t - 4, 0] = float("inf"), float("-inf"), float("inf")
    z, zc, v = torch.sigmoid(p[..., :h].double()), torch.sigmoid(-p[..., :h].double()), p[..., h:].double()
    hs, x = [], h0.double()
    for i in range(t):
        x = z[:, i] * x + zc[:, i] * v[:, i]
        hs.append(x)
    D, dvs = dl.double(), [None] * t
    for i in range(t - 1, -1, -1):
        D = D + dy[:, i].double()
        dvs[i] = D * zc[:, i]
        D = D * z[:, i]
    pg, hg = p.cuda().requires_grad_(), h0.cuda().requires_grad_()
    y, last = F.gated_scan(pg, hg, out_gate=False)
    dp, dh0 = torch.autograd.grad([y, last], [pg, hg], [dy.cuda(), dl.cuda()])
    for got, want in ((y, torch.stack(hs, 1)), (last, x), (dp[..., h:], torch.stack(dvs, 1)), (dh0, D)):
        got = got.detach().cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        assert torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])


@pytest.mark.parametrize("dtype,h", [(torch.bfloat16, 512), (torch.float32, 250)])
def test_more_blocks_than_the_chip_holds(dtype, h):
    """One call of over a thousand blocks forward and two thousand backward (512 of either fit), 17 and 33 tiles a row: blocks start when
    others retire, states pass several runs of tiles. Against the recurrence in 64 bits, with the bounds of the recurrence's own tests."""
    from tests.test_gpu_scan import check, make
    b, t = 16, 2100
    groups = -(-h // (128 if dtype == torch.bfloat16 else 64))
    assert -(-t // 128) * b * groups > 1024 and -(-t // 64) * b * groups > 2048
    check(*make(b, t, h, True, dtype, seed=11, lengths=[t, 1, 0, 2049, 2048, 1025, 130] + [t - 64 * i for i in range(9)]), True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zero_and_tiny_matrices_without_eps(dtype):
    """eps = 0: a matrix of zeros stays zero, and one whose norm lies below 2^-112 (16384 over it leaves fp32's range), subnormal
    numbers included, has the direction it has. The scaled matrix holds the same digits, so the results are the same bits."""
    from cpcsv.optim import FusedMuon, orthogonalize
    g = torch.randn(70, 90, generator=torch.Generator().manual_seed(4))
    zero = torch.zeros(70, 90).to(dtype).cuda()
    assert torch.equal(orthogonalize(zero, eps=0.0), zero)
    both = orthogonalize(torch.stack([zero, g.to(dtype).cuda()]), eps=0.0)
    assert torch.equal(both[0], zero) and torch.equal(both[1], orthogonalize(g.to(dtype).cuda(), eps=0.0))
    g = (g * 64).round().clamp(-127, 127)                # whole numbers of 7 bits: exact in either type at 2^-149 too
    for e in (-149, -130, -120, -100, 100):
        small = (g.double() * 2.0 ** e).to(dtype).cuda()
        if dtype == torch.bfloat16 and e < -133:
            continue                                     # (below bfloat16's smallest)
        assert torch.equal(orthogonalize(small, eps=0.0), orthogonalize(g.to(dtype).cuda(), eps=0.0)), e
    w = torch.nn.Parameter(torch.ones(70, 90, device="cuda"))
    w.grad = torch.zeros_like(w)
    FusedMuon([w], lr=0.1, eps=0.0).step()
    assert torch.equal(w, torch.ones_like(w))


@pytest.mark.parametrize("rows,cols", [(63, 124), (500, 130), (992, 7936)])
def test_16_bit_results_are_the_fp32_results_rounded(rows, cols):
    """A bf16 gradient gives the fp32 call's result of the same numbers, rounded once: where it differs from another form's result, that
    form's fp32 value lay on the other side of a rounding border. Repeated with other matrices in between, the same bits."""
    from cpcsv.optim import orthogonalize
    gen = torch.Generator("cuda").manual_seed(rows)
    g, other = ((torch.randn(rows, cols, generator=gen, device="cuda") + torch.randn(rows, 4, generator=gen, device="cuda") @ torch.randn(
        4, cols, generator=gen, device="cuda")).bfloat16() for _ in range(2))
    got = orthogonalize(g)
    assert torch.equal(got, orthogonalize(g.float()).bfloat16())
    for _ in range(5):
        orthogonalize(other)
        assert torch.equal(orthogonalize(g), got)


@pytest.mark.parametrize("kind", ["gauss", "strong"])
@pytest.mark.parametrize("rows,cols", [(17, 23), (32, 32), (64, 64), (63, 124), (128, 128), (90, 500), (12, 700), (2048, 16)])
def test_small_matrices_keep_the_accuracy_of_fp32(rows, cols, kind):
    """Over twenty matrices, the mean distance from the 64-bit result is at most one and a half times that of the same iteration in fp32."""
    from cpcsv.optim import orthogonalize
    from tests.test_gpu_orth import iterate, spectrum
    own = kernel = 0.0
    for seed in range(20):
        g = spectrum(rows, cols, kind, seed).cuda()
        want = iterate(g, 5, 1e-7)
        own += ((iterate(g, 5, 1e-7, torch.float32).double() - want).norm() / want.norm()).item()
        kernel += ((orthogonalize(g).double() - want).norm() / want.norm()).item()
    assert kernel <= 1.5 * own, (kernel / 20, own / 20)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 7])
def test_matrices_of_all_aspects_share_a_step(steps):
    """Near-square and wide matrices, whose iterations form X at different times, in one call: each with the bits that it has alone, and
    the smaller ones within their distance from the 64-bit result."""
    from cpcsv.optim import FusedMuon
    from tests.test_gpu_orth import bound, iterate
    shapes = [(60, 60), (70, 900), (300, 310), (1000, 40), (129, 700), (1600, 1700), (520, 8), (1030, 5000)]
    gen = torch.Generator("cuda").manual_seed(steps)
    w0, gs = ([torch.randn(s, generator=gen, device="cuda") for s in shapes] for _ in range(2))

    def step(which):
        ps = [torch.nn.Parameter(w0[i].clone()) for i in which]
        for p, i in zip(ps, which):
            p.grad = gs[i].clone()
        FusedMuon(ps, lr=0.1, momentum=0.0, steps=steps).step()
        return [p.detach() for p in ps]
    together = step(range(len(shapes)))
    assert all(torch.equal(a, b) for a, b in zip(together[::-1], step(range(len(shapes))[::-1])))
    for i, (r, c) in enumerate(shapes):
        assert torch.equal(together[i], step([i])[0]), shapes[i]
        x = 0.1 * max(1.0, r / c) ** 0.5 * iterate(gs[i], steps, 1e-7)
        assert (together[i].double() - (w0[i].double() - x)).norm() <= bound(shapes[i]) * 3.9 ** max(0, steps - 5) * x.norm() + 3 * 2.0 ** -24 * w0[i].norm(), shapes[i]


def test_a_learning_rate_tensor_changed_in_place_is_followed():
    """lr may be a tensor, which schedulers change in place: each step and sync_lr() read its value."""
    from cpcsv.optim import FusedMuon
    gen = torch.Generator("cuda").manual_seed(1)
    w0, g = torch.randn(30, 40, generator=gen, device="cuda"), torch.randn(30, 40, generator=gen, device="cuda")
    ends = []
    for lr in (0.1, torch.tensor(0.1)):
        w = torch.nn.Parameter(w0.clone())
        w.grad = g.clone()
        opt = FusedMuon([w], lr=lr)
        opt.step()
        for v in (0.025, 0.5):
            if torch.is_tensor(lr):
                lr.fill_(v)
            else:
                opt.param_groups[0]["lr"] = v
            opt.sync_lr()
            opt.step()
            if torch.is_tensor(lr):
                lr.fill_(2 * v)
            else:
                opt.param_groups[0]["lr"] = 2 * v
            opt.step()
        ends.append(w.detach())
    assert torch.equal(*ends)


@pytest.mark.parametrize("shape", [(0, 4, 8), (2, 0, 8)])
def test_a_recurrence_over_no_tokens(shape):
    """GatedRecurrence over an empty batch or empty sequences: as gated_scan, the state passes through; the weights' gradients are zero."""
    from cpcsv import modules as M
    for out_gate in (True, False):
        rec = M.GatedRecurrence(8, 4, out_gate=out_gate).cuda()
        x, h0 = torch.zeros(shape, device="cuda", requires_grad=True), torch.randn(shape[0], 4, device="cuda", requires_grad=True)
        y, last = rec(x, h0)
        assert y.shape == shape[:2] + (4,) and y.dtype == rec(torch.zeros(2, 3, 8, device="cuda"))[0].dtype and torch.equal(last, h0)
        grads = torch.autograd.grad([y.float().sum() + last.sum()], [x, h0, rec.proj.weight, rec.proj.bias])
        assert grads[0].shape == shape and torch.equal(grads[1], torch.ones_like(h0)) and not grads[2].any() and not grads[3].any()
        assert rec.step(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 4, device="cuda")).shape == (0, 4)


@pytest.mark.parametrize("d,h", [(40, 48), (365, 100)])
def test_the_documented_block_runs(d, h, bf16):
    """The documents' example as it is printed, then a step of its optimisers."""
    import glob
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    blocks = [b for f in glob.glob(os.path.join(root, "*.md")) for b in re.findall(r"```python\n(.*?)```", open(f).read(), re.S) if "GatedRecurrence(" in b]
    assert blocks
    for text in blocks:
        from cpcsv import functional, modules, runtime
        x, x_t = torch.randn(3, 7, d, device="cuda"), torch.randn(3, d, device="cuda")
        names = dict(torch=torch, M=modules, F=functional, runtime=runtime, d=d, h=h, x=x, x_t=x_t,
                     lengths=torch.tensor([7, 0, 3], dtype=torch.int32, device="cuda"))
        exec(text, names)
        assert names["y_t"].shape == (3, h) and names["z"].shape == x.shape
        (names["x1"].sum() + names["z"].square().sum()).backward()
        held = [p for m in ("norm", "rec", "out", "post") for p in names[m].parameters()]
        before = [p.detach().clone() for p in held]
        assert sorted(id(p) for o in names["opt"] for g in o.param_groups for p in g["params"]) == sorted(id(p) for p in held)
        for o in names["opt"]:
            o.step()
        assert all(torch.isfinite(p).all() and not torch.equal(p, q) for p, q in zip(held, before))
