"""The gated linear recurrence (cpcsv.functional.gated_scan / gated_scan_step, csrc/scan.hip) against the recurrence run token by
token in 64 bits, forward and backward.

Tolerances follow from the arithmetic: every h_t is a sum of terms that went through at most T gate products, each off by at most
eps_g = (4 + |f|_max) 2^-24 relative (the exponential's argument is rounded at |f| and scaled; a handful of further roundings), so
|error of h_t| <= habs_t F with F = 2 (T + 4) eps_g and habs the same recurrence run on absolute values; the same holds for D_t.
Storing a value adds half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(b, t, h, gate, dtype, seed=0, lengths=None):
    g = torch.Generator().manual_seed(seed)
    p = torch.randn(b, t, (3 if gate else 2) * h, generator=g)
    p[..., :h] = 1.5 * p[..., :h] + 2.0
    p = p.to(dtype)
    h0, dl = torch.randn(b, h, generator=g), torch.randn(b, h, generator=g)
    dy = torch.randn(b, t, h, generator=g).to(dtype)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return p, h0, dy, dl, n


def reference(p, h0, dy, dl, lengths, gate):
    """Outputs, gradients and the error bounds without storage rounding, all in float64."""
    b, t, k = p.shape
    h = k // (3 if gate else 2)
    p, dy = p.double(), dy.double()
    f, v = p[..., :h], p[..., h:2 * h]
    o = p[..., 2 * h:] if gate else None
    live = torch.ones(b, t, 1, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(t).view(1, t, 1) < lengths.view(b, 1, 1)
    f, v = torch.where(live, f, 0.0), torch.where(live, v, 0.0)
    dy = torch.where(live, dy, 0.0)
    z, zc = torch.sigmoid(f), torch.sigmoid(-f)
    if gate:
        o = torch.where(live, o, 0.0)
        sg = torch.sigmoid(o)
        act, dact, dabs = o * sg, sg * (1 + o * (1 - sg)), sg * (1 + o.abs() * (1 - sg))
    else:
        act = torch.ones_like(v)
    hs, ha, prev, pa = (torch.zeros(b, t, h, dtype=torch.float64) for _ in range(4))
    x = h0.double() if h0 is not None else torch.zeros(b, h, dtype=torch.float64)
    xa = x.abs()
    for i in range(t):
        prev[:, i], pa[:, i] = x, xa
        x = torch.where(live[:, i], z[:, i] * x + zc[:, i] * v[:, i], x)
        xa = torch.where(live[:, i], z[:, i] * xa + zc[:, i] * v[:, i].abs(), xa)
        hs[:, i], ha[:, i] = x, xa
    fmax = max(1.0, p[live.expand_as(p)].abs().max().item() if live.any() else 1.0)
    F = 2 * (t + 4) * (4 + fmax) * 2.0 ** -24
    y = torch.where(live, hs * act, 0.0)
    out = {"y": (y, ha * act.abs() * 2 * F), "last": (x, xa * F)}
    D = dl.double() if dl is not None else torch.zeros(b, h, dtype=torch.float64)
    Da = D.abs()
    dp, tol = torch.zeros_like(p), torch.zeros_like(p)
    for i in range(t - 1, -1, -1):
        on = live[:, i]
        D, Da = D + dy[:, i] * act[:, i], Da + (dy[:, i] * act[:, i]).abs()
        zz = z[:, i] * zc[:, i]
        dp[:, i, :h] = torch.where(on, D * (prev[:, i] - v[:, i]) * zz, 0.0)
        tol[:, i, :h] = torch.where(on, Da * (pa[:, i] + v[:, i].abs()) * zz * 3 * F, 0.0)
        dp[:, i, h:2 * h] = torch.where(on, D * zc[:, i], 0.0)
        tol[:, i, h:2 * h] = torch.where(on, Da * zc[:, i] * 2 * F, 0.0)
        D, Da = torch.where(on, D * z[:, i], D), torch.where(on, Da * z[:, i], Da)
    if gate:
        dp[..., 2 * h:] = torch.where(live, dy * hs * dact, 0.0)
        tol[..., 2 * h:] = torch.where(live, dy.abs() * ha * dabs * 2 * F, 0.0)
    out["dp"], out["dh0"] = (dp, tol), (D, Da * F)
    return out


def within(got, want, bound, what):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    lim = bound + want.abs() * half * (1 + 2.0 ** -8) + 1e-37       # (1e-37: results below fp32's normal range)
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), (what, (err / lim).max().item(), err.max().item())


def run(p, h0, dy, dl, n, gate, place=lambda t: t):
    from cpcsv import functional as F
    dev = "cuda"
    pg = place(p.to(dev)).requires_grad_()
    hg = h0.to(dev).requires_grad_() if h0 is not None else None
    y, last = F.gated_scan(pg, hg, lengths=n.to(dev) if n is not None else None, out_gate=gate)
    leaves = [pg] + ([hg] if hg is not None else [])
    grads = torch.autograd.grad([y, last], leaves, [dy.to(dev), dl.to(dev)])
    return {"y": y, "last": last, "dp": grads[0], "dh0": grads[1] if hg is not None else None}


def check(p, h0, dy, dl, n, gate, place=lambda t: t):
    got, want = run(p, h0, dy, dl, n, gate, place), reference(p, h0, dy, dl, n, gate)
    for k, (w, tol) in want.items():
        if got[k] is not None:
            within(got[k], w, tol, k)
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,h,gate", [(1, 1, 1, True), (3, 1, 64, False), (2, 2, 5, True), (1, 31, 7, True), (2, 32, 130, True), (2, 33, 66, False),
                                        (1, 64, 365, True), (3, 100, 124, True), (1, 257, 18, False), (2, 1023, 33, True), (5, 700, 256, True)])
def test_scan_matches_float64(b, t, h, gate, dtype):
    check(*make(b, t, h, gate, dtype, seed=t), gate)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t,lengths", [(40, [40, 0, 1, 31, 32, 33]), (7, [0, 0, 7]), (130, [0, 129, 64, 65]), (300, [300, 5, 0]), (64, [-3, 1000, 2])])
def test_sequences_end_at_their_lengths(t, lengths, dtype):
    """Values behind a sequence's end are not read (NaN and infinities there change nothing); y and dp are zero there, length 0 hands
    h0 through; lengths are clamped to 0..T."""
    p, h0, dy, dl, n = make(len(lengths), t, 36, True, dtype, seed=t, lengths=lengths)
    dead = torch.arange(t).view(1, t, 1) >= n.view(-1, 1, 1)
    p = torch.where(dead, torch.tensor(float("nan"), dtype=dtype), p)
    dy = torch.where(dead, torch.tensor(float("inf"), dtype=dtype), dy)
    got = check(p, h0, dy, dl, n.clamp(0, t), True)
    again = run(p, h0, dy, dl, n, True)
    for k in got:
        assert torch.equal(got[k], again[k]), k
    dead = dead.cuda()
    assert not got["y"][dead.expand_as(got["y"])].any() and not got["dp"][dead.expand_as(got["dp"])].any()
    assert torch.equal(got["last"][n.cuda() <= 0], h0.cuda()[n.cuda() <= 0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [5, 100])
def test_strides_and_alignment(t, dtype):
    """Time-major storage, rows cut out of wider ones, odd element offsets, a column-major projection: the same bits as contiguous."""
    p, h0, dy, dl, n = make(3, t, 24, True, dtype, seed=3)
    want = run(p, h0, dy, dl, n, True)

    def odd(x):
        wide = torch.zeros(x.shape[0], x.shape[1], x.shape[2] + 5, dtype=x.dtype, device=x.device)
        wide[..., 3:3 + x.shape[2]] = x
        return wide[..., 3:3 + x.shape[2]].detach()
    for place in (lambda x: x.transpose(0, 1).contiguous().transpose(0, 1), odd, lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
                  lambda x: x[:, ::1].flip(1).contiguous().flip(1)):
        got = run(p, h0, dy, dl, n, True, place)
        for k in want:
            assert torch.equal(got[k], want[k]), k


def test_broadcast_batch():
    """One projection seen by several rows (stride 0): its gradient is the sum over them."""
    from cpcsv import functional as F
    p, h0, dy, dl, _ = make(1, 50, 20, True, torch.float32, seed=9)
    h0, dy = torch.cat([h0, -h0, 2 * h0]), torch.cat([dy, 0.5 * dy, -dy])
    dl = dl.expand(3, -1).contiguous()
    pg = p.cuda().requires_grad_()
    hg = h0.cuda().requires_grad_()
    y, last = F.gated_scan(pg.expand(3, -1, -1), hg)
    gp, gh = torch.autograd.grad([y, last], [pg, hg], [dy.cuda(), dl.cuda()])
    want = reference(p.expand(3, -1, -1), h0, dy, dl, None, True)
    within(y, *want["y"], "y")
    within(gh, *want["dh0"], "dh0")
    within(gp, want["dp"][0].sum(0, keepdim=True), want["dp"][1].sum(0, keepdim=True) + 3 * 2.0 ** -24 * want["dp"][0].abs().sum(0, keepdim=True), "dp")


@pytest.mark.parametrize("t", [9, 200])
def test_without_a_state_and_partial_gradients(t):
    from cpcsv import functional as F
    p, _, dy, dl, _ = make(2, t, 12, True, torch.float32, seed=5)
    check(p, None, dy, dl, None, True)
    pg = p.cuda().requires_grad_()
    y, last = F.gated_scan(pg)
    only_y, = torch.autograd.grad([y], [pg], [dy.cuda()], retain_graph=True)
    only_last, = torch.autograd.grad([last], [pg], [dl.cuda()], retain_graph=True)
    want_y = reference(p, None, dy, torch.zeros_like(dl), None, True)["dp"]
    want_l = reference(p, None, torch.zeros_like(dy), dl, None, True)["dp"]
    within(only_y, *want_y, "dp of y")
    within(only_last, *want_l, "dp of last")
    strided = torch.autograd.grad([y], [pg], [dy.cuda().transpose(0, 2).contiguous().transpose(0, 2)])[0]
    assert torch.equal(strided, only_y)


def test_gradient_matches_differences():
    """Central differences of a weighted sum of the outputs, in the direction of a random vector, with fp32 outputs summed in 64 bits.
    The step is 2^-6: third-order terms stay below 2^-12 of the slope's scale and the outputs' rounding (2^-24 each) below 2^-17 of it."""
    from cpcsv import functional as F
    p, h0, dy, dl, _ = make(2, 70, 16, True, torch.float32, seed=8)
    g = torch.Generator().manual_seed(1)
    vp, vh = torch.randn(p.shape, generator=g), torch.randn(h0.shape, generator=g)
    got = run(p, h0, dy, dl, None, True)
    slope = (got["dp"].cpu().double() * vp).sum() + (got["dh0"].cpu().double() * vh).sum()
    scale = (got["dp"].cpu().double() * vp).abs().sum() + (got["dh0"].cpu().double() * vh).abs().sum()

    def loss(e):
        y, last = F.gated_scan((p + e * vp).cuda(), (h0 + e * vh).cuda())
        return (y.cpu().double() * dy).sum() + (last.cpu().double() * dl).sum()
    e = 2.0 ** -6
    assert abs((loss(e) - loss(-e)) / (2 * e) - slope) < 2.0 ** -9 * scale


def test_extreme_gates():
    """Closed and open gates (|f| up to the type's range): z or 1 - z underflows to 0 or stays exact, never NaN."""
    from cpcsv import functional as F
    f = torch.tensor([-3e38, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 200.0, 3e38])
    v = torch.linspace(-2, 2, 9)
    p = torch.cat([f, v]).view(1, 1, 18).expand(1, 40, 18).contiguous()
    h0 = torch.full((1, 9), 5.0)
    dy, dl = torch.ones(1, 40, 9), torch.ones(1, 9)
    got = run(p, h0, dy, dl, None, False)
    want = reference(p, h0, dy, dl, None, False)
    assert all(torch.isfinite(got[k]).all() for k in got)
    # |f| = 3e38 gives exact gates and would only blow up the stated bound: 200 is the largest argument that is rounded
    F_ = 2 * 44 * 204 * 2.0 ** -24
    assert (got["y"].cpu().double() - want["y"][0]).abs().max() <= 5 * F_
    assert (got["last"].cpu().double() - want["last"][0]).abs().max() <= 5 * F_
    assert (got["dh0"].cpu().double() - want["dh0"][0]).abs().max() <= 41 * F_


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,h,gate", [(1, 1, True), (64, 512, True), (5, 365, False)])
def test_steps_equal_the_scan(b, h, gate, dtype):
    """Token by token with the state updated in place: the sequence's own outputs (the same roundings inside a chunk: bit-equal)."""
    from cpcsv import functional as F
    p, h0, _, _, _ = make(b, 20, h, gate, dtype, seed=2)
    pd, state = p.cuda(), h0.cuda()
    y, last = F.gated_scan(pd, state.clone(), out_gate=gate)
    for i in range(20):
        assert torch.equal(F.gated_scan_step(pd[:, i], state, out_gate=gate), y[:, i]), i
    assert torch.equal(state, last)


def test_runs_are_identical_and_graphs_replay():
    """Captured forward + backward: replays (with eager work between them) give the eager result, also after the inputs changed; two
    graphs of the same call do not disturb each other."""
    from cpcsv import functional as F
    p, h0, dy, dl, n = make(3, 300, 40, True, torch.bfloat16, seed=4, lengths=[300, 170, 0])
    want = run(p, h0, dy, dl, n, True)
    want2 = run(-p, 2 * h0, dy, dl, n, True)
    ps, hs, dys, dls, ns = (x.cuda() for x in (p, h0, dy, dl, n))
    ps.requires_grad_()
    hs.requires_grad_()

    def step():
        y, last = F.gated_scan(ps, hs, lengths=ns)
        gp, gh = torch.autograd.grad([y, last], [ps, hs], [dys, dls])
        return {"y": y.detach(), "last": last.detach(), "dp": gp, "dh0": gh}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for rep in range(3):
        with torch.no_grad():
            ps.copy_((p if rep != 1 else -p).cuda())
            hs.copy_((h0 if rep != 1 else 2 * h0).cuda())
        for gr, _ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        eager = run(p, h0, dy, dl, n, True)
        for _, out in graphs:
            for k in out:
                assert torch.equal(out[k], (want if rep != 1 else want2)[k]), (rep, k)
        for k in eager:
            assert torch.equal(eager[k], want[k])


def test_side_stream():
    p, h0, dy, dl, _ = make(2, 90, 48, True, torch.float32, seed=6)
    want = run(p, h0, dy, dl, None, True)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(p, h0, dy, dl, None, True)
    s.synchronize()
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_step_refuses_states_it_cannot_update():
    from cpcsv import functional as F
    p = torch.zeros(2, 12).cuda()
    for h in (None, torch.zeros(4, 2).cuda().T, torch.zeros(2, 4).cuda().requires_grad_()):
        with pytest.raises(ValueError, match="in place"):
            F.gated_scan_step(p, h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,h,lengths", [(1, 5000, 70, None), (2, 2305, 130, [2305, 1100]), (300, 40, 6, None), (1, 129, 2000, None)])
def test_many_tiles(b, t, h, lengths, dtype):
    """Several published states on the way, more blocks than the chip holds, a last tile of one token."""
    check(*make(b, t, h, True, dtype, seed=t, lengths=lengths), True)


def test_empty():
    from cpcsv import functional as F
    h0 = torch.randn(2, 3).cuda().requires_grad_()
    p = torch.zeros(2, 0, 9).cuda().requires_grad_()
    y, last = F.gated_scan(p, h0)
    assert y.shape == (2, 0, 3) and torch.equal(last, h0)
    gp, gh = torch.autograd.grad([last.sum()], [p, h0])
    assert gp.shape == p.shape and torch.equal(gh, torch.ones_like(gh))
    y, last = F.gated_scan(torch.zeros(0, 4, 9).cuda())
    assert y.shape == (0, 4, 3) and last.shape == (0, 3)
    assert F.gated_scan_step(torch.zeros(0, 9).cuda(), torch.zeros(0, 3).cuda()).shape == (0, 3)


@pytest.mark.parametrize("t", [1, 40])
def test_long_offsets(t):
    """A batch stride beyond 2^31 elements: rows far apart in one allocation."""
    from cpcsv import functional as F
    h = 8
    far = (1 << 31) + 64
    base = torch.zeros(far + t * 3 * h, dtype=torch.bfloat16, device="cuda")
    p, h0, _, _, _ = make(2, t, h, True, torch.bfloat16, seed=7)
    view = base.as_strided((2, t, 3 * h), (far, 3 * h, 1))
    view.copy_(p.cuda())
    y, last = F.gated_scan(view, h0.cuda())
    y2, last2 = F.gated_scan(p.cuda(), h0.cuda())
    assert torch.equal(y, y2) and torch.equal(last, last2)


@pytest.mark.parametrize("t", [20, 100])
def test_a_state_updated_in_place_is_not_used_backward(t):
    """gated_scan keeps its initial state for the backward pass: stepping that very tensor on is noticed."""
    from cpcsv import functional as F
    p, h0, dy, _, _ = make(2, t, 8, True, torch.float32, seed=8)
    p, h = p.cuda().requires_grad_(), h0.cuda()
    y, _ = F.gated_scan(p, h)
    F.gated_scan_step(p.detach()[:, 0].contiguous(), h)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy.cuda())
    with torch.inference_mode():
        q, g = p.detach()[:, 0].clone(), h.clone()
        F.gated_scan_step(q, g)
    assert not torch.equal(g, h)


def test_two_calls_at_once():
    """Two streams, more blocks than the chip holds: each call waits for its own blocks only."""
    cases = [[q.cuda() if q is not None else None for q in make(3, 3000, 512, True, torch.bfloat16, seed=s)] for s in (9, 10)]
    want = [run(*[q.detach() if q is not None else None for q in c], True) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(run(*[q.detach() if q is not None else None for q in c], True))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for k in g:
            assert torch.equal(g[k], want[i % 2][k]), (i, k)
