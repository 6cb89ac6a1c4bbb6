"""The norms around a block with its gate and residual scale (cpcsv.functional.norm_residual / rms_norm, csrc/blocknorm.hip) against
the formulas in float64, forward and backward.

Tolerances: every value is a sum of products of at most 64 serially added terms a thread (plus 14 joins) and a few further roundings,
so it is off by at most K = 128 (1 + kappa) 2^-24 of the same expression on absolute values, where kappa = mean (|x| + |branch|)^2 /
mean x'^2 of the row counts what cancels in the residual sum; a column sum adds one rounding a row. Storing adds half a step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def make(shape, xdt, udt, gate, scale, nxt, seed=0):
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]
    r = lambda *s: torch.randn(*s, generator=g)
    q = {"x": (2 * r(*shape)).to(xdt), "u": r(*shape).to(udt), "w_post": 1 + 0.2 * r(d)}
    q["gate"] = None if gate is None else ((0.5 + r(*shape)) if gate == "token" else (0.5 + r(shape[0], *([1] * (len(shape) - 2)), d))).to(udt)
    q["scale"] = 0.3 + 0.1 * r(d) if scale else None
    q["w_next"] = 1 + 0.2 * r(d) if nxt else None
    return q, r(*shape).to(xdt), r(*shape).to(udt)


def reference(q, dxo, dz, eps):
    """{name: (value, bound)} in float64, from the formulas and from the same formulas on absolute values."""
    v = {k: (t.double() if t is not None else None) for k, t in q.items()}
    x, u = v["x"], v["u"]
    one = torch.ones((), dtype=torch.float64)
    g, s, wp, wn = (v[k] if v[k] is not None else one for k in ("gate", "scale", "w_post", "w_next"))
    if u is not None:
        ru = (u.square().mean(-1, keepdim=True) + eps).rsqrt()
        uh = u * ru
        branch = s * g * wp * uh
    else:
        uh = branch = torch.zeros_like(x)
    x1, xa = x + branch, x.abs() + branch.abs()
    rx = (x1.square().mean(-1, keepdim=True) + eps).rsqrt()
    kap = 1 + xa.square().mean(-1, keepdim=True) * rx.square()
    K = 128 * kap * U
    xh, xha = x1 * rx, xa * rx
    out = {}
    if u is not None:
        out["xo"] = (x1, xa * 64 * U)
    if v["w_next"] is not None:
        out["z"] = (xh * wn, (xha * wn).abs() * K)
    if dxo is None and dz is None:
        return out
    dxo = dxo.double() if dxo is not None else torch.zeros_like(x)
    gz = dz.double() * wn if (dz is not None and v["w_next"] is not None) else torch.zeros_like(x)
    dx = dxo + rx * (gz - xh * (gz * xh).mean(-1, keepdim=True))
    dxa = dxo.abs() + rx * (gz.abs() + xha * (gz.abs() * xha).mean(-1, keepdim=True))
    out["dx"] = (dx, dxa * K)
    rows = x[..., 0].numel()
    cols = lambda t: t.reshape(-1, t.shape[-1]).sum(0)
    colb = lambda t: cols(t * (K + rows * U))
    if v["w_next"] is not None and dz is not None:
        out["dw_next"] = (cols(dz.double() * xh), colb(dz.double().abs() * xha))
    if u is not None:
        f, fa = s * g * wp, (s * g * wp).abs()
        qv, qa = dx * f, dxa * fa
        out["du"] = (ru * (qv - uh * (qv * uh).mean(-1, keepdim=True)), ru * (qa + uh.abs() * (qa * uh.abs()).mean(-1, keepdim=True)) * 2 * K)
        out["dw_post"] = (cols(dx * s * g * uh), colb(dxa * (s * g * uh).abs()))
        if v["scale"] is not None:
            out["dscale"] = (cols(dx * g * wp * uh), colb(dxa * (g * wp * uh).abs()))
        if v["gate"] is not None:
            t, ta = dx * s * wp * uh, dxa * (s * wp * uh).abs() * (K + rows * U)
            if v["gate"].shape != x.shape:
                dims = tuple(range(1, x.dim() - 1))
                t, ta = t.sum(dims, keepdim=True).reshape(v["gate"].shape), ta.sum(dims, keepdim=True).reshape(v["gate"].shape)
            out["dgate"] = (t, ta)
    return out


def within(got, want, bound, what):
    got = got.detach().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    half = torch.finfo(got.dtype).eps / 2
    lim = bound + want.abs() * half * (1 + 2.0 ** -8) + 1e-37
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), (what, (err / lim).max().item(), err.max().item())


def run(q, dxo, dz, eps=1e-6, place=lambda t: t):
    from cpcsv import functional as F
    c = {k: (place(t.cuda()).requires_grad_() if t is not None else None) for k, t in q.items()}
    if c["u"] is None:
        out = {"z": F.rms_norm(c["x"], c["w_next"], eps, out_dtype=dz.dtype)}
    else:
        r = F.norm_residual(c["x"], c["u"], c["w_post"], gate=c["gate"], scale=c["scale"], w_next=c["w_next"], eps=eps)
        out = dict(zip(("xo", "z"), r)) if c["w_next"] is not None else {"xo": r}
    ups = {"xo": dxo, "z": dz}
    outs = [k for k in out if ups[k] is not None]
    names = [k for k, t in c.items() if t is not None]
    grads = torch.autograd.grad([out[k] for k in outs], [c[k] for k in names], [ups[k].cuda() for k in outs], allow_unused=True)
    out.update({"d" + k: gr for k, gr in zip(names, grads) if gr is not None})
    return out


def check(q, dxo, dz, eps=1e-6, place=lambda t: t):
    got, want = run(q, dxo, dz, eps, place), reference(q, dxo, dz, eps)
    for k, (w, b) in want.items():
        within(got[k], w, b, k)
    return got


TYPES = [(F32, F32), (BF16, BF16), (F32, BF16)]


@pytest.mark.parametrize("xdt,udt", TYPES)
@pytest.mark.parametrize("shape,gate,scale,nxt", [
    ((1, 1), None, False, True), ((3, 2), "token", True, True), ((5, 7), None, True, False), ((2, 3, 8), "sample", False, True),
    ((130, 64), "token", False, True), ((4, 33, 100), "sample", True, True), ((3, 41, 365), None, True, True), ((2, 9, 512), "token", True, True),
    ((7, 520), None, False, True), ((3, 5, 1000), "sample", True, False), ((4, 30, 2048), "token", True, True), ((2, 6, 4096), "sample", True, True),
    ((3, 4100), "token", True, True), ((2, 4, 8192), "sample", True, True), ((3, 8203), "token", False, True), ((2, 2, 16384), "token", True, True),
    ((2, 2, 16383), "sample", True, True)])
def test_norm_residual_matches_float64(shape, gate, scale, nxt, xdt, udt):
    q, dxo, dz = make(shape, xdt, udt, gate, scale, nxt, seed=shape[-1])
    check(q, dxo, dz if nxt else None)


@pytest.mark.parametrize("shape,gate", [((5000, 8), "token"), ((9001, 16), None), ((1100, 2, 24), "sample"), ((1, 700, 72), "sample"),
                                        ((2050, 5, 9), "sample"), ((6, 1, 40), "sample"), ((3, 4, 5, 48), "sample"), ((2600, 264), "token")])
def test_many_rows(shape, gate):
    """More rows than one sweep of the grid, samples shared out over several blocks, more samples than blocks, one token a sample."""
    check(*make(shape, F32, BF16, gate, True, True, seed=1))


@pytest.mark.parametrize("xdt,zdt", TYPES)
@pytest.mark.parametrize("shape", [(1,), (3, 1), (300, 40), (2, 3, 365), (5, 2048), (2, 8200)])
def test_rms_norm_matches_float64(shape, xdt, zdt):
    q, _, dz = make(shape, xdt, zdt, None, False, True, seed=2)
    q["u"] = q["w_post"] = None
    check(q, None, dz)


@pytest.mark.parametrize("ups", ["xo", "z"])
def test_one_of_the_outputs(ups):
    """Only one output is used: the other's gradient counts as zero."""
    q, dxo, dz = make((3, 20, 136), F32, F32, "token", True, True, seed=3)
    got = run(q, dxo if ups == "xo" else None, dz if ups == "z" else None)
    want = reference(q, dxo if ups == "xo" else None, dz if ups == "z" else None, 1e-6)
    for k in want:
        if k in got:
            within(got[k], *want[k], k)
    if ups == "xo":
        assert not got["dw_next"].any()


@pytest.mark.parametrize("frozen", [("w_post", "scale", "w_next"), ("gate",), ("u", "x"), ("x", "u", "w_post", "scale", "w_next")])
def test_partly_frozen(frozen):
    """Gradients that nobody asks for are not formed; the others keep their bits."""
    from cpcsv import functional as F
    q, dxo, dz = make((4, 11, 200), F32, BF16, "sample", True, True, seed=4)
    full = run(q, dxo, dz)
    c = {k: t.cuda() for k, t in q.items()}
    live = [k for k in c if k not in frozen]
    for k in live:
        c[k].requires_grad_()
    out = F.norm_residual(c["x"], c["u"], c["w_post"], gate=c["gate"], scale=c["scale"], w_next=c["w_next"])
    for k, g in zip(live, torch.autograd.grad(out, [c[k] for k in live], [dxo.cuda(), dz.cuda()])):
        assert torch.equal(g, full["d" + k]), k


@pytest.mark.parametrize("xdt,udt", TYPES)
def test_layouts(xdt, udt):
    """Transposed storage, odd offsets (no 16-byte rows), an expanded residual row: the values of contiguous tensors. The single-element
    path adds in another order: float64's bounds hold for it too."""
    q, dxo, dz = make((4, 6, 72), xdt, udt, "token", True, True, seed=5)
    want = run(q, dxo, dz)

    def odd(t):
        flat = torch.zeros(t.numel() + 3, dtype=t.dtype, device=t.device)
        flat[3:] = t.reshape(-1)
        return flat[3:].view(t.shape).detach()
    got = run(q, dxo, dz, place=lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    check(q, dxo, dz, place=odd)


def test_broadcast_residual():
    from cpcsv import functional as F
    q, dxo, dz = make((5, 3, 48), F32, F32, None, True, True, seed=6)
    row = q["x"][:1, :1].clone()
    q["x"] = row.expand(5, 3, 48)
    want = reference(q, dxo, dz, 1e-6)
    x = row.cuda().requires_grad_()
    out = F.norm_residual(x.expand(5, 3, 48), q["u"].cuda(), q["w_post"].cuda(), scale=q["scale"].cuda(), w_next=q["w_next"].cuda())
    dx, = torch.autograd.grad(out, [x], [dxo.cuda(), dz.cuda()])
    within(dx, want["dx"][0].sum((0, 1), keepdim=True), want["dx"][1].sum((0, 1), keepdim=True) + 15 * U * want["dx"][0].abs().sum((0, 1), keepdim=True), "dx")


def test_zero_and_extreme_rows():
    """All-zero rows (eps alone under the root), rows of 1e18 and of 1e-15: the formula's values."""
    q, dxo, dz = make((4, 64), F32, F32, "token", True, True, seed=7)
    for k in ("x", "u"):
        q[k][0] = 0
        q[k][1] *= 1e18
        q[k][2] *= 1e-15
    check(q, dxo, dz)


def test_non_finite_rows_stay_in_their_row():
    """A NaN or infinity makes its own row NaN in z, as the formula does, and leaves the others' bits alone."""
    from cpcsv import functional as F
    q, _, _ = make((6, 128), F32, F32, None, True, True, seed=8)
    c = {k: t.cuda() for k, t in q.items() if t is not None}
    good = F.norm_residual(c["x"], c["u"], c["w_post"], scale=c["scale"], w_next=c["w_next"])
    c["u"][2, 5], c["x"][4, 7] = float("nan"), float("nan")
    bad = F.norm_residual(c["x"], c["u"], c["w_post"], scale=c["scale"], w_next=c["w_next"])
    rows = torch.tensor([0, 1, 3, 5]).cuda()
    assert torch.equal(bad[0][rows], good[0][rows]) and torch.equal(bad[1][rows], good[1][rows])
    assert torch.isnan(bad[1][2]).all() and torch.isnan(bad[1][4]).all() and torch.isnan(bad[0][4, 7])


def test_gradient_matches_differences():
    """Central differences in a random direction; step 2^-6, see the scan's test: third-order terms and roundings stay below 2^-9 of
    the slope's scale."""
    from cpcsv import functional as F
    q, dxo, dz = make((3, 10, 96), F32, F32, "sample", True, True, seed=9)
    g = torch.Generator().manual_seed(3)
    names = list(q)
    way = {k: torch.randn(q[k].shape, generator=g) for k in names}
    got = run(q, dxo, dz)
    parts = [(got["d" + k].cpu().double() * way[k]).sum() for k in names]
    scale = sum((got["d" + k].cpu().double() * way[k]).abs().sum() for k in names)

    def loss(e):
        c = {k: (q[k].double() + e * way[k]).float().cuda() for k in names}
        xo, z = F.norm_residual(c["x"], c["u"], c["w_post"], gate=c["gate"], scale=c["scale"], w_next=c["w_next"])
        return (xo.cpu().double() * dxo).sum() + (z.cpu().double() * dz).sum()
    e = 2.0 ** -6
    assert abs((loss(e) - loss(-e)) / (2 * e) - sum(parts)) < 2.0 ** -9 * scale


@pytest.mark.parametrize("gate", ["token", "sample"])
def test_graphs_replay(gate):
    from cpcsv import functional as F
    q, dxo, dz = make((6, 50, 144), F32, BF16, gate, True, True, seed=10)
    want = run(q, dxo, dz)
    c = {k: t.cuda().requires_grad_() for k, t in q.items()}
    ups = [dxo.cuda(), dz.cuda()]

    def step():
        out = F.norm_residual(c["x"], c["u"], c["w_post"], gate=c["gate"], scale=c["scale"], w_next=c["w_next"])
        gr = torch.autograd.grad(out, list(c.values()), ups)
        return dict(zip(["xo", "z"] + ["d" + k for k in c], [o.detach() for o in out] + list(gr)))
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
        for gr, out in graphs:
            for t in out.values():
                t.zero_()
            gr.replay()
        torch.cuda.synchronize()
        eager = run(q, dxo, dz)
        for k in want:
            assert torch.equal(eager[k], want[k]), k
            for _, out in graphs:
                assert torch.equal(out[k], want[k]), (rep, k)


def test_side_stream():
    q, dxo, dz = make((3, 17, 365), F32, F32, "sample", True, True, seed=11)
    want = run(q, dxo, dz)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(q, dxo, dz)
    s.synchronize()
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_empty():
    from cpcsv import functional as F
    w = torch.ones(8).cuda().requires_grad_()
    x = torch.zeros(0, 5, 8).cuda().requires_grad_()
    xo, z = F.norm_residual(x, x, w, gate=torch.zeros(0, 1, 8).cuda(), w_next=w)
    dx, dw = torch.autograd.grad([xo, z], [x, w], [torch.zeros_like(xo), torch.zeros_like(z)])
    assert xo.shape == z.shape == dx.shape == x.shape and not dw.any()
    assert F.rms_norm(torch.zeros(3, 0, 8).cuda(), w).shape == (3, 0, 8)
