"""Newton-Schulz orthogonalisation and the Muon update on the GPU against plain float64 ones.

Tolerances, in Frobenius norms |.|, with u = 2^-24.  A matrix held as two fp16 halves is off by 2^-22 of each value, a
product of halves leaves out 2^-22 of each term and sums its 3 K terms in fp32, so with d(K) = 2^-21 + 3 K u and s the
largest singular value of X (m x n), a step adds
    d1 = d(n) |X|^2                                       to A = X X^T,
    d2 = d(m) |c| |A|^2 + 2^-21 |b| |A|                   to B,
    s (|b| + 2 |c| s^2) d1 + s d2 + d(m) |B| |X| + 2^-21 a |X|    to X,
and multiplies the error that X came with by at most max |p'| over [0, s], p(s) = a s + b s^3 + c s^5 (the divided
differences of an odd polynomial; twice that covers s, |A|, |B| being the exact iteration's).  X starts off by 2^-21 |X|
and fp16's least step, at most 2^-24 over the matrix.  From 256 columns on fp32's own summation, sqrt(K) u and more, is
above 2^-22, and there the result has to be as near as twice what fp32 products give.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32 = torch.bfloat16, torch.float32
COEF = (3.4445, -4.7750, 2.0315)


def _muon():
    from llattn_amd import muon
    return muon


def _ns(x, steps=5, eps=1e-7, coef=COEF):
    """The iteration on [.., m, n] in x's type."""
    a, b, c = coef
    flip = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if flip else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT.contiguous() if flip else x


def _matrices(batch, m, n, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = min(m, n)
    x = torch.randn(batch, m, n, generator=g)
    if kind == "decay":
        u, _ = torch.linalg.qr(torch.randn(batch, m, k, generator=g))
        v, _ = torch.linalg.qr(torch.randn(batch, n, k, generator=g))
        x = (u * torch.logspace(0, -4, k)) @ v.mT
    elif kind == "lowrank":
        r = max(1, k // 16)
        x = torch.randn(batch, m, r, generator=g) @ torch.randn(batch, r, n, generator=g)
    return x.to(DEV)


def _bound(x, steps=5, eps=1e-7, coef=COEF):
    """The bound above for each matrix of x (float64)."""
    a, b, c = (abs(v) for v in coef)
    x = x.double()
    x = x.mT.contiguous() if x.shape[-2] > x.shape[-1] else x
    m, n = x.shape[-2:]
    x = x / (torch.linalg.matrix_norm(x)[..., None, None] + eps)
    d = lambda k: 2.0 ** -21 + 3 * k * 2.0 ** -24  # noqa: E731
    f = torch.linalg.matrix_norm
    err = 2.0 ** -21 * f(x) + 2.0 ** -24
    for _ in range(steps):
        g = x @ x.mT.contiguous()
        q = coef[1] * g + coef[2] * (g @ g)
        s = torch.linalg.eigvalsh(g).amax(-1).clamp(min=0).sqrt()
        at = s[..., None] * torch.linspace(0, 1, 2001, dtype=torch.float64, device=x.device)
        slope = (coef[0] + 3 * coef[1] * at ** 2 + 5 * coef[2] * at ** 4).abs().amax(-1)
        d1 = d(n) * f(x) ** 2
        d2 = d(m) * c * f(g) ** 2 + 2.0 ** -21 * b * f(g)
        err = slope * err + s * (b + 2 * c * s * s) * d1 + s * d2 + d(m) * f(q) * f(x) + 2.0 ** -21 * a * f(x)
        x = coef[0] * x + q @ x
    return 2 * err


def _near(got, x, what, **kw):
    want = _ns(x.double(), **kw)
    norm = torch.linalg.matrix_norm(want)
    off = torch.linalg.matrix_norm(got.double() - want)
    step = torch.finfo(got.dtype).eps / 2 * norm
    bound = _bound(x, **kw) + step
    ref = torch.linalg.matrix_norm(_ns(x.float(), **kw).double() - want)
    if min(x.shape[-2:]) >= 256:
        bound = torch.minimum(bound, 2 * ref + step)
    print(f"{what}: off {float((off / norm).max()):.2e}, fp32 {float((ref / norm).max()):.2e}, bound {float((bound / norm).min()):.2e}", flush=True)
    assert bool((off <= bound).all()), f"{what}: off {off.tolist()} bound {bound.tolist()}"


SHAPES = [(1, 1, 1), (2, 1, 7), (2, 9, 1), (3, 5, 5), (1, 32, 33), (4, 64, 128), (2, 65, 63), (3, 128, 64), (1, 100, 300),
          (1, 129, 1000), (2, 640, 257), (1, 512, 1408), (5, 1030, 520), (24, 256, 512), (130, 16, 24)]


@pytest.mark.parametrize("batch,m,n", SHAPES)
@pytest.mark.parametrize("kind", ["flat", "decay", "lowrank"])
def test_orthogonalize(batch, m, n, kind):
    x = _matrices(batch, m, n, kind, seed=m + n)
    _near(_muon().orthogonalize(x), x, f"{batch}x{m}x{n} {kind}")


@pytest.mark.parametrize("tiles", [1, 2, 3, 4])
@pytest.mark.parametrize("batch,m,n", [(2, 33, 70), (1, 64, 64), (3, 130, 200), (2, 257, 130), (1, 333, 1001), (2, 390, 514),
                                       (9, 450, 449), (1, 1408, 700)])
def test_every_workgroup_of_the_products(tiles, batch, m, n, monkeypatch):
    """Tiles inside the matrices, ragged, half outside and larger than them; an update of the same in place."""
    mu = _muon()
    monkeypatch.setattr(mu, "TILES", tiles)
    x = _matrices(batch, m, n, "decay", seed=m + tiles)
    _near(mu.orthogonalize(x), x, f"tiles {tiles}: {batch}x{m}x{n}")
    ws, ms = [torch.zeros(m, n, device=DEV) for _ in x], [torch.zeros(m, n, device=DEV) for _ in x]
    mu.muon_update(ws, list(x), ms, lr=1.0, momentum=0.0)  # W = -s ns(G)
    _near(torch.stack(ws) / -math.sqrt(max(1.0, m / n)), x, f"tiles {tiles}: update")


@pytest.mark.parametrize("batch,m,n", [(1, 1408, 4096), (6, 1000, 1500), (16, 640, 1300), (2, 2048, 640), (12, 1408, 1408)])
def test_large_matrices(batch, m, n):
    x = _matrices(batch, m, n, "flat")
    _near(_muon().orthogonalize(x), x, f"{batch}x{m}x{n}")


@pytest.mark.parametrize("m,n", [(70, 90), (90, 70), (256, 256)])
def test_orthogonalize_bf16(m, n):
    x = _matrices(3, m, n, "decay").to(BF16)
    got = _muon().orthogonalize(x)
    assert got.dtype is BF16
    _near(got, x, f"bf16 {m}x{n}")


@pytest.mark.parametrize("steps,coef", [(1, COEF), (2, COEF), (10, COEF), (12, (1.5, -0.5, 0.0)), (6, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coef):
    x = _matrices(2, 48, 80, "flat")
    _near(_muon().orthogonalize(x, steps=steps, coefficients=coef), x, f"{steps} steps of {coef}", steps=steps, coef=coef)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1.0, 1e30])
def test_sizes_of_values(size):
    """Squares that fp32 does not hold; far below eps the matrix stays small in proportion (to fp16's least step)."""
    x = (_matrices(2, 40, 60, "flat").double() * size).float()
    got = _muon().orthogonalize(x)
    want = _ns(x.double())
    assert bool((torch.linalg.matrix_norm(got.double() - want) <= _bound(x) + 2.0 ** -24 * torch.linalg.matrix_norm(want)).all())


def test_zero_infinite_and_nan():
    x = _matrices(4, 30, 50, "flat")
    x[0] = 0.0
    x[2, 3, 4] = float("inf")
    x[3, 1, 1] = float("nan")
    got = _muon().orthogonalize(x)
    assert not got[0].any() and torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
    _near(got[1:2], x[1:2], "beside them")


def test_views_and_out():
    mu = _muon()
    x = _matrices(6, 33, 47, "flat")
    want = mu.orthogonalize(x)
    wide = torch.zeros(6, 33, 100, device=DEV)
    wide[:, :, 3:50] = x
    assert torch.equal(mu.orthogonalize(wide[:, :, 3:50]), want)
    assert torch.equal(mu.orthogonalize(x.mT.contiguous().mT), want)
    assert torch.equal(mu.orthogonalize(x.view(2, 3, 33, 47)), want.view(2, 3, 33, 47))
    out = torch.full_like(x, 7.0)
    assert mu.orthogonalize(x, out=out) is out and torch.equal(out, want)
    y = x.clone()
    assert torch.equal(mu.orthogonalize(y, out=y), want)
    shifted = torch.zeros(x.numel() + 1, device=DEV)[1:].view_as(x).copy_(x)  # rows that are not 16-byte aligned
    assert torch.equal(mu.orthogonalize(shifted), want)
    assert mu.orthogonalize(torch.zeros(0, 4, 5, device=DEV)).shape == (0, 4, 5)
    assert mu.orthogonalize(x[0]).shape == (33, 47) and torch.equal(mu.orthogonalize(x[0]), want[0])


def _plain_update(w, g, m, lr, mu, nesterov, wd, scale, dtype):
    w, g, m = w.to(dtype), g.to(dtype), m.to(dtype)
    m = mu * m + (1 - mu) * g
    u = (1 - mu) * g + mu * m if nesterov else m
    rows, cols = w.shape
    s = math.sqrt(max(1.0, rows / cols)) if scale == "aspect" else 0.2 * math.sqrt(max(rows, cols))
    return (1 - lr * wd) * w - lr * s * _ns(u), m


def _update_bound(w, g, m64, w64, lr, mu, nesterov, wd, scale):
    """The orthogonalisation's error in the weight (U itself is off by 2^-21 of its terms, which its first error covers
    where they do not cancel), the sum's and its rounding."""
    u = (1 - mu) * g.double() + mu * m64 if nesterov else m64
    rows, cols = w.shape
    s = math.sqrt(max(1.0, rows / cols)) if scale == "aspect" else 0.2 * math.sqrt(max(rows, cols))
    parts = ((1 - mu) * g.double()).norm() + 2 * m64.norm()
    own = float(_bound(u)) * float(parts / u.norm())
    return lr * s * own + 2.0 ** -22 * float(w.double().norm() + lr * s * _ns(u).norm()) + torch.finfo(w.dtype).eps / 2 * float(w64.norm())


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", ["aspect", "rms"])
@pytest.mark.parametrize("wt,gt", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)])
def test_muon_update(nesterov, scale, wt, gt):
    """Shapes mixed in one call, tall and wide; new weights and momenta in place and in buffers of their own."""
    lr, mu, wd = 0.03, 0.9, 0.1
    shapes = [(40, 70), (130, 64), (40, 70), (1, 9), (64, 64), (130, 64), (40, 70)]
    ws = [_matrices(1, *s, "flat", i)[0].mul(0.05).to(wt) for i, s in enumerate(shapes)]
    gs = [_matrices(1, *s, "lowrank", i + 50)[0].to(gt) for i, s in enumerate(shapes)]
    ms = [_matrices(1, *s, "decay", i + 90)[0] for i, s in enumerate(shapes)]
    out = ([torch.empty_like(w) for w in ws], [torch.empty_like(m) for m in ms])
    keep = [t.clone() for t in ws + gs + ms]
    kw = dict(lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=scale)
    _muon().muon_update(ws, gs, ms, out=out, **kw)
    assert all(torch.equal(a, b) for a, b in zip(keep, ws + gs + ms))
    for i in range(len(shapes)):
        w64, m64 = _plain_update(ws[i], gs[i], ms[i], lr, mu, nesterov, wd, scale, torch.float64)
        # momentum: two products and a sum, each rounded
        assert bool(((out[1][i].double() - m64).abs() <= 2.0 ** -22 * (ms[i].abs() + gs[i].abs()).double()).all())
        assert float((out[0][i].double() - w64).norm()) <= _update_bound(ws[i], gs[i], m64, w64, lr, mu, nesterov, wd, scale), (i, shapes[i])
    _muon().muon_update(ws, gs, ms, **kw)
    assert all(torch.equal(a, b) for a, b in zip(ws + ms, out[0] + out[1]))


def test_repeats_bit_for_bit_and_under_a_graph():
    mu = _muon()
    shapes = [(96, 200), (200, 96), (96, 200)]
    sets = [[[_matrices(1, *s, "decay", 7 * k + j + 3 * i)[0] for i, s in enumerate(shapes)] for j in range(3)] for k in range(2)]
    def step(ws, gs, ms):
        out = ([torch.empty_like(w) for w in ws], [torch.empty_like(m) for m in ms])
        mu.muon_update(ws, gs, ms, lr=0.1, out=out)
        return out[0] + out[1] + [mu.orthogonalize(gs[0])]
    want = [step(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*sets[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want[0]))
    held = [[t.clone() for t in v] for v in sets[0]]
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for k in (0, 1, 0):
        for a, b in zip(held, sets[k]):
            for x, y in zip(a, b):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        step(*sets[1])
        assert all(torch.equal(a, b) for a, b in zip(got, want[k]))


def test_in_place_updates_are_seen_by_autograd():
    w = torch.randn(32, 32, device=DEV, requires_grad=True)
    y = (w * w).sum()
    _muon().muon_update([w], [torch.randn(32, 32, device=DEV)], [torch.zeros(32, 32, device=DEV)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_optimisers():
    """Muon over parameters, some without a gradient; state that is saved and loaded goes on alike; with AdamW beside."""
    mu = _muon()
    def model():
        torch.manual_seed(0)
        return torch.nn.Sequential(torch.nn.Linear(24, 48), torch.nn.GELU(), torch.nn.Linear(48, 8)).to(DEV)
    def build(net):
        mats = [p for p in net.parameters() if p.dim() == 2]
        return mu.MuonAdamW(mats, [p for p in net.parameters() if p.dim() == 1], dict(lr=0.05, weight_decay=0.1), lr=1e-2, weight_decay=0.0)
    x = torch.randn(16, 24, generator=torch.Generator().manual_seed(1)).to(DEV)
    def go(net, opt, n):
        for _ in range(n):
            net(x).square().mean().backward()
            opt.step()
            opt.zero_grad(set_to_none=True)
    a = model()
    oa = build(a)
    go(a, oa, 4)
    b = model()
    ob = build(b)
    go(b, ob, 2)
    c = model()
    c.load_state_dict(b.state_dict())
    oc = build(c)
    oc.load_state_dict(ob.state_dict())
    go(c, oc, 2)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), c.parameters()))
    # the first step by hand
    d = model()
    od = build(d)
    sched = torch.optim.lr_scheduler.LambdaLR(od, lambda i: 1.0)
    w0 = d[0].weight.detach().clone()
    d(x).square().mean().backward()
    grad = d[0].weight.grad.clone()
    d[2].weight.grad = None
    before = d[2].weight.detach().clone()
    od.step()
    sched.step()
    want, _ = _plain_update(w0, grad, torch.zeros_like(w0), 0.05, 0.95, True, 0.1, "aspect", torch.float64)
    assert float((d[0].weight.detach().double() - want).norm()) <= _update_bound(w0, grad, 0.05 * grad.double(), want, 0.05, 0.95, True, 0.1, "aspect")
    assert torch.equal(d[2].weight, before)
    only = mu.Muon([p for p in d.parameters() if p.dim() == 2])
    d(x).sum().backward()
    assert float(only.step(lambda: torch.tensor(3.0))) == 3.0


@pytest.mark.parametrize("m,n", [(20, 30), (100, 140)])
@pytest.mark.parametrize("shift", [1, -1])
def test_an_output_across_its_input(m, n, shift):
    """One matrix of a batch along, for matrices of one workgroup each and of many."""
    x = _matrices(6, m, n, "flat")
    want = _muon().orthogonalize(x[:5] if shift > 0 else x[1:])
    src, out = (x[:5], x[1:]) if shift > 0 else (x[1:], x[:5])
    assert _muon().orthogonalize(src, out=out) is out and torch.equal(out, want)


def test_first_step_is_not_captured():
    """Momenta made during a capture would begin at zero in every replay; made before it, replays go on like eager steps."""
    mu = _muon()
    p, q = (torch.nn.Parameter(_matrices(1, 40, 70, "flat")[0]) for _ in range(2))
    p.grad = q.grad = _matrices(1, 40, 70, "lowrank")[0]
    a, b = mu.Muon([p], lr=0.01), mu.Muon([q], lr=0.01)
    with pytest.raises(RuntimeError, match="before a step is captured"), torch.cuda.graph(torch.cuda.CUDAGraph()):
        a.step()
    assert "momentum_buffer" not in a.state[p]
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        assert torch.equal(p, q) and torch.equal(a.state[p]["momentum_buffer"], b.state[q]["momentum_buffer"])


# ---- to fp32's own error ----------------------------------------------------------------------------------------------
# The bound above adds worst cases and lets pass what loses half of the bits at small sizes.  Here the result is held to
# twice the sum of the errors that fp32 products have and that the scheme of two halves has (emulated below with exact
# sums), with a floor: a step rounds X, A and B to fp32 (2^-24 each) whatever its sums, and the steps behind multiply a
# relative error of a singular value s by |s p'(s) / p(s)| each; over all s in [0, 1] and five steps the products of those
# factors add up to 27.2 at most, so 3 * 27.2 * 2^-24 of the result.
FLOOR = 82 * 2.0 ** -24


def _emulated(x, lo=True, steps=5, eps=1e-7, coef=COEF):
    """The iteration on two fp16 halves of X, A and B (lo False: on the upper ones alone), sums in 64 bits."""
    a, b, c = coef
    flip = x.shape[-2] > x.shape[-1]
    x = (x.mT if flip else x).double()
    m, n = x.shape[-2:]
    s = 2.0 ** min(14, int(0.5 * math.log2(m * n)))

    def halves(v):
        h = v.float().half().double()
        return h, (v.float().double() - h).half().double() if lo else torch.zeros_like(h)

    def times(p, q):
        return p[0] @ q[0] + p[0] @ q[1] + p[1] @ q[0]

    def flipped(p):
        return [v.mT.contiguous() for v in p]

    x = halves(s * x / (torch.linalg.matrix_norm(x)[..., None, None] + eps))
    for _ in range(steps):
        g = halves(4096.0 / s ** 2 * times(x, flipped(x)))
        q = halves(b * (g[0] + g[1]) + c / 4096.0 * times(g, flipped(g)))
        new = a * (x[0] + x[1]) + times(q, x) / 4096.0
        x = halves(new)
    out = (new / s).float()
    return out.mT.contiguous() if flip else out


def _errors(u32, want):
    """|error| against ``want`` (float64) allowed to the iteration on ``u32``."""
    norm = torch.linalg.matrix_norm
    return 2 * (norm(_emulated(u32).double() - want) + norm(_ns(u32).double() - want)) + FLOOR * norm(want)


@pytest.mark.parametrize("batch,m,n", [(4, 64, 128), (3, 65, 63), (3, 128, 64), (2, 100, 300), (2, 129, 1000), (2, 40, 70), (1, 64, 448),
                                       (2, 448, 64), (2, 64, 449), (2, 449, 64), (1, 65, 448), (3, 20, 448), (1, 33, 4100), (2, 250, 255)])
@pytest.mark.parametrize("kind", ["flat", "decay", "lowrank"])
def test_as_exact_as_fp32(batch, m, n, kind):
    """At small sizes too, and at both sides of where one workgroup takes a matrix (64 rows, 448 columns)."""
    x = _matrices(batch, m, n, kind, seed=m * n)
    want = _ns(x.double())
    got, most = torch.linalg.matrix_norm(_muon().orthogonalize(x).double() - want), _errors(x, want)
    print(f"{batch}x{m}x{n} {kind}: {float((got / most).max()):.3f} of the bound", flush=True)
    assert bool((got <= most).all())
    if kind == "flat":  # what the upper halves alone give is outside
        assert bool((torch.linalg.matrix_norm(_emulated(x, lo=False).double() - want) > 10 * most).all())


TILED = [(130, 200), (200, 130), (333, 70), (257, 514), (96, 450), (130, 200), (65, 64), (451, 33)]


@pytest.mark.parametrize("tiles", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("wt,gt", [(F32, F32), (BF16, BF16), (F32, BF16), (BF16, F32)])
def test_updates_of_matrices_over_many_workgroups(tiles, nesterov, wt, gt, monkeypatch):
    """Shapes mixed in one call, none of which one workgroup takes alone: weights, momenta and decay by value, into buffers
    of their own and in place."""
    mu = _muon()
    monkeypatch.setattr(mu, "TILES", tiles)
    lr, beta, wd = 0.03, 0.9, 2.0
    ws = [_matrices(1, *s, "flat", i)[0].mul(0.05).to(wt) for i, s in enumerate(TILED)]
    gs = [_matrices(1, *s, "lowrank", i + 50)[0].to(gt) for i, s in enumerate(TILED)]
    ms = [_matrices(1, *s, "decay", i + 90)[0] for i, s in enumerate(TILED)]
    out = ([torch.full_like(w, 9.0) for w in ws], [torch.full_like(m, 9.0) for m in ms])
    kw = dict(lr=lr, momentum=beta, nesterov=nesterov, weight_decay=wd)
    mu.muon_update(ws, gs, ms, out=out, **kw)
    for w, g, m, nw, nm in zip(ws, gs, ms, *out):
        m32 = beta * m + (1 - beta) * g.float()
        m64 = beta * m.double() + (1 - beta) * g.double()
        u32 = (1 - beta) * g.float() + beta * m32 if nesterov else m32
        u64 = (1 - beta) * g.double() + beta * m64 if nesterov else m64
        assert bool(((nm.double() - m64).abs() <= 2.0 ** -22 * (m.abs() + g.abs()).double()).all())
        o, s = _ns(u64), math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        want = (1 - lr * wd) * w.double() - lr * s * o
        # the products' and the sum's roundings in fp32, and the one to the weight's type
        most = lr * s * float(_errors(u32, o)) + 2.0 ** -22 * float(w.double().norm() + lr * s * o.norm()) \
            + torch.finfo(wt).eps / 2 * float(want.norm())
        off = float((nw.double() - want).norm())
        assert off <= most, (tuple(w.shape), off, most)
        assert lr * wd * float(w.double().norm()) > 5 * most  # a decay or a weight that is not this one's would show
    mu.muon_update(ws, gs, ms, **kw)
    assert all(torch.equal(a, b) for a, b in zip(ws + ms, out[0] + out[1]))


# The library takes the coefficients in fp32.  Off by up to 2^-25 of themselves, they move a singular value by up to 27.2
# times that over the steps (see FLOOR), more than the one rounding that the results below are held to.
COEF32 = tuple(float(torch.tensor(c)) for c in COEF)

THIN = [(5, 1, 1), (3, 1, 29), (1, 82, 1), (2, 2, 3), (9, 3079, 1), (4, 5, 448), (2, 5, 4096), (70, 6, 262), (1, 9, 17), (2, 15, 16),
        (3, 16, 16), (2, 16, 1000), (1, 16, 32768), (1, 32768, 13), (2, 255, 16), (2, 257, 7)]


@pytest.mark.parametrize("batch,m,n", THIN)
@pytest.mark.parametrize("kind", ["flat", "decay", "lowrank"])
def test_thin_matrices_are_rounded_once(batch, m, n, kind):
    """A smaller side of up to 16 is taken in 64 bits: half a step of the result's type, and next to nothing besides."""
    x = _matrices(batch, m, n, kind, seed=m + 3 * n)
    for v in (x, x.to(BF16)):
        want = _ns(v.double(), coef=COEF32)
        norm = torch.linalg.matrix_norm(want)
        off = torch.linalg.matrix_norm(_muon().orthogonalize(v).double() - want)
        assert bool((off <= 1.01 * torch.finfo(v.dtype).eps / 2 * norm).all()), (off / norm).max()


def test_thin_matrices_beside_others():
    """Small, thin and large ones in one call, weights by value and in place; each has the bits that it has by itself."""
    mu = _muon()
    shapes = [(130, 200), (7, 300), (40, 70), (300, 7), (1, 9), (130, 200), (7, 300), (16, 17), (20, 17)]
    for types in ((F32, F32), (BF16, F32), (F32, BF16)):
        ws = [_matrices(1, *s, "flat", i)[0].mul(0.05).to(types[0]) for i, s in enumerate(shapes)]
        gs = [_matrices(1, *s, "flat", i + 50)[0].to(types[1]) for i, s in enumerate(shapes)]
        ms = [_matrices(1, *s, "flat", i + 90)[0] for i, s in enumerate(shapes)]
        out = ([torch.full_like(w, 9.0) for w in ws], [torch.full_like(m, 9.0) for m in ms])
        kw = dict(lr=0.03, momentum=0.9, weight_decay=2.0)
        mu.muon_update(ws, gs, ms, out=out, **kw)
        for w, g, m, nw, nm in zip(ws, gs, ms, *out):
            w64, m64 = _plain_update(w, g, m, 0.03, 0.9, True, 2.0, "aspect", torch.float64)
            assert bool(((nm.double() - m64).abs() <= 2.0 ** -22 * (m.abs() + g.abs()).double()).all())
            u = 0.1 * g.float() + 0.9 * (0.9 * m + 0.1 * g.float())
            o = _ns(0.1 * g.double() + 0.9 * m64)
            s = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
            most = 0.03 * s * float(_errors(u, o)) + 2.0 ** -22 * float(w.double().norm() + 0.03 * s * o.norm())
            assert float((nw.double() - w64).norm()) <= most + torch.finfo(types[0]).eps / 2 * float(w64.norm()), tuple(w.shape)
            if min(w.shape) <= 16:
                one = [w.clone()], [m.clone()]
                mu.muon_update(one[0], [g], one[1], **kw)
                assert torch.equal(one[0][0], nw) and torch.equal(one[1][0], nm)
        mu.muon_update(ws, gs, ms, **kw)
        assert all(torch.equal(a, b) for a, b in zip(ws + ms, out[0] + out[1]))


def test_thin_matrices_of_any_values_and_places():
    mu = _muon()
    x = _matrices(5, 6, 50, "flat")
    x[0] = 0.0
    x[2, 3, 4] = float("inf")
    x[3, 1, 1] = float("nan")
    want = _ns(x[[1, 4]].double(), coef=COEF32)
    got = mu.orthogonalize(x)
    assert not got[0].any() and torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
    assert bool((torch.linalg.matrix_norm(got[[1, 4]].double() - want) <= 1.01 * 2.0 ** -24 * torch.linalg.matrix_norm(want)).all())
    y = x[[1, 4]]
    got = got[[1, 4]]
    shifted = torch.zeros(y.numel() + 1, device=DEV)[1:].view_as(y).copy_(y)
    assert torch.equal(mu.orthogonalize(shifted), got) and torch.equal(mu.orthogonalize(y.mT).mT, got)
    assert mu.orthogonalize(shifted, out=shifted) is shifted and torch.equal(shifted, got)
    big, small = (y.double() * 1e30).float(), (y.double() * 1e-30).float()
    assert float((mu.orthogonalize(big).double() - _ns(big.double(), coef=COEF32)).norm()) <= 1.01 * 2.0 ** -24 * float(want.norm())
    far = _ns(small.double(), coef=COEF32)
    assert float((mu.orthogonalize(small).double() - far).norm()) <= 1.01 * 2.0 ** -24 * float(far.norm())


@pytest.mark.parametrize("batch,m,n", [(4, 64, 256), (4, 64, 257), (64, 33, 256), (65, 33, 128), (65, 33, 129), (128, 128, 64), (129, 64, 65)])
def test_where_matrices_go_to_one_workgroup_each(batch, m, n):
    """Both sides of the limits: 64 rows, 256 columns, 64 matrices a launch."""
    x = _matrices(batch, m, n, "decay", seed=batch)
    want = _ns(x.double())
    off = torch.linalg.matrix_norm(_muon().orthogonalize(x).double() - want)
    assert bool((off <= _errors(x, want)).all())


@pytest.mark.parametrize("steps", [5, 9, 10, 16, 20, 40])
@pytest.mark.parametrize("m,n", [(10, 40), (40, 10), (16, 3000), (3, 5)])
def test_thin_matrices_of_low_rank_over_many_steps(m, n, steps):
    """Rows of which some are others' copies: directions without a singular value stay as small as they are, whatever the
    number of steps, and the others stay in their band (the iteration maps [0, 1.21] into itself)."""
    k = min(m, n)
    x = _matrices(2, max(1, k // 3), max(m, n), "flat", seed=steps)
    x = x.repeat(1, 4, 1)[:, :k]
    x = x.mT.contiguous() if m > n else x
    got = _muon().orthogonalize(x, steps=steps)
    assert torch.isfinite(got).all()
    s = torch.linalg.svdvals(got.double())
    assert bool((s <= 1.21).all()) and bool((s[:, :max(1, k // 3)] >= 0.6).all())
    if steps <= 9:
        want = _ns(x.double(), steps=steps, coef=COEF32)
        assert bool((torch.linalg.matrix_norm(got.double() - want) <= 1.01 * 2.0 ** -24 * torch.linalg.matrix_norm(want)).all())
