"""The gated feed-forward (``llattn_amd.gated_feed_forward``) on the GPU against a plain float64 one.

Tolerances are counted, elementwise, with b = 2^-8 (half a step of bf16) and u = 2^-24 (of fp32).  A sum of K products of
exact bf16 values is off by at most (K + 2) u of the sum of their sizes.  The activations have slopes of at most 1.13 and
curvatures of at most 0.8 and are evaluated to 2e-5 of themselves (their slopes to 2e-5).  h, da and du are rounded to bf16 once
each (up to 64 rows to two bf16 values), p = act(a) and s = act'(a) u cut off after 24 bits (2^-15 of themselves), results rounded
once more.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U, B16 = 2.0 ** -24, 2.0 ** -8
BF16, F32 = torch.bfloat16, torch.float32
NAMES = ("y", "dx", "dw1", "db1", "dw3", "db3", "dw2", "db2")


def _ffn(*a, **k):
    from llattn_amd import gated_feed_forward
    return gated_feed_forward(*a, **k)


def _layers(D, F, Do, dtype=BF16, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n_in, n_out in ((D, F), (D, F), (F, Do)):
        m = torch.nn.Linear(n_in, n_out, bias=bias)
        m.weight = torch.nn.Parameter((torch.randn(n_out, n_in, generator=g) / n_in ** 0.5).to(dtype))
        if bias:
            m.bias = torch.nn.Parameter((0.5 * torch.randn(n_out, generator=g)).to(dtype))
        out.append(m.to(DEV))
    return out


def _grads(x, layers, act, dy, **k):
    """(y, dx, dw1, db1, dw3, db3, dw2, db2), None for biases that are not there."""
    y = _ffn(x, *layers, act=act, **k)
    ps = [x] + [p for m in layers for p in (m.weight, m.bias)]
    got = iter(torch.autograd.grad(y, [p for p in ps if p is not None and p.requires_grad], dy))
    return [y.detach()] + [next(got) if p is not None and p.requires_grad else None for p in ps]


def _act(name, a):
    """act(a) and its slope in 64 bits."""
    if name == "silu":
        g = torch.sigmoid(a)
        return a * g, g * (1 + a * (1 - g))
    cdf = 0.5 * torch.erfc(-a * 0.5 ** 0.5)
    return a * cdf, cdf + a * torch.exp(-0.5 * a * a) * 0.3989422804014327


def _exact(x, layers, act, dy):
    """Pairs (value, bound of the error before the last rounding) in 64 bits, in the order of NAMES.  Up to 64 rows h, da and du are
    the sums of two bf16 values: the lower one rounds what the upper one has left (2^-8 of the value at most) by 2^-8 of that."""
    half = B16 if x.shape[0] > 64 else 2.0 ** -16
    x, dy = x.detach().to(BF16).double(), dy.to(BF16).double()
    w1, w3, w2 = (m.weight.detach().to(BF16).double() for m in layers)
    b1, b3, b2 = (torch.zeros((), dtype=torch.float64, device=DEV) if m.bias is None else m.bias.detach().double() for m in layers)
    (N, D), Fd, Do = x.shape, w1.shape[0], w2.shape[0]
    c = lambda k: (k + 2) * U  # noqa: E731
    a, u = x @ w1.t() + b1, x @ w3.t() + b3
    ea = c(D) * (x.abs() @ w1.abs().t() + b1.abs())
    eu = c(D) * (x.abs() @ w3.abs().t() + b3.abs())
    f, df = _act(act, a)
    ef, edf = 1.13 * ea + 2e-5 * f.abs(), 0.8 * ea + 2e-5
    h = f * u
    eh = f.abs() * eu + u.abs() * ef + ef * eu
    eh = eh + half * (h.abs() + eh)
    y = h @ w2.t() + b2
    ey = eh @ w2.abs().t() + c(Fd) * ((h.abs() + eh) @ w2.abs().t() + b2.abs())
    p, ep = f, ef + 2.0 ** -15 * (f.abs() + ef)
    s = df * u
    es = df.abs() * eu + u.abs() * edf + edf * eu
    es = es + 2.0 ** -15 * (s.abs() + es)
    dh = dy @ w2
    edh = c(Do) * (dy.abs() @ w2.abs())
    prod = lambda m, em: (dh * m, (t := dh.abs() * em + m.abs() * edh + em * edh) + half * ((dh * m).abs() + t))  # noqa: E731
    (da, eda), (du, edu) = prod(s, es), prod(p, ep)
    dx = da @ w1 + du @ w3
    size = (da.abs() + eda) @ w1.abs() + (du.abs() + edu) @ w3.abs()
    out = [(y, ey), (dx, eda @ w1.abs() + edu @ w3.abs() + c(2 * Fd) * size)]
    for g, eg, z, ez in ((da, eda, x, None), (du, edu, x, None), (dy, torch.zeros_like(dy), h, eh)):
        e = eg.t() @ z.abs() + c(N) * ((g.abs() + eg).t() @ z.abs())
        if ez is not None:
            e = e + (1 + c(N)) * (g.abs().t() @ ez)
        out.append((g.t() @ z, e))
        out.append((g.sum(0), eg.sum(0) + c(N) * (g.abs() + eg).sum(0)))
    return out


def _near(got, want, err, what):
    assert got.shape == want.shape, what
    # dx is rounded to bf16 before it is widened to an fp32 x: its last rounding is b of itself whatever its type
    half = B16 if what == "dx" else torch.finfo(got.dtype).eps / 2
    bad = ~((got.double() - want).abs() <= err + half * (want.abs() + err) + 2.0 ** -120)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float(((got.double() - want).abs() / (err + half * want.abs() + 1e-30)).max())}"


# (N, D, F, D_out, act, bias, type of x, type of the weights)
CASES = [
    (1, 8, 8, 8, "silu", False, BF16, BF16),
    (1, 1408, 4096, 1408, "silu", False, BF16, BF16),
    (2, 64, 200, 64, "gelu", True, BF16, F32),
    (2, 1536, 210, 250, "silu", True, BF16, F32),
    (7, 136, 72, 24, "silu", True, F32, F32),
    (16, 1408, 4096, 1408, "gelu", True, BF16, BF16),
    (17, 250, 333, 250, "silu", True, BF16, BF16),
    (17, 64, 229, 64, "silu", False, BF16, F32),
    (33, 777, 1001, 777, "gelu", False, BF16, BF16),
    (64, 128, 256, 128, "gelu", True, BF16, F32),
    (64, 1408, 1096, 520, "silu", True, BF16, F32),
    (65, 72, 64, 200, "silu", False, BF16, BF16),
    (129, 1, 3, 5, "silu", True, F32, BF16),
    (333, 264, 520, 264, "silu", True, BF16, F32),
    (700, 512, 1096, 384, "gelu", True, BF16, BF16),
    (1500, 1024, 1408, 1024, "silu", False, BF16, BF16),
    (4100, 256, 640, 256, "silu", True, BF16, BF16),
    (4100, 64, 4096, 64, "silu", False, BF16, BF16),  # more tiles of both gated products than run at a time
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_values_and_gradients(case):
    N, D, F, Do, act, bias, xt, wt = case
    layers = _layers(D, F, Do, wt, bias)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(N, D, generator=g).to(xt).to(DEV).requires_grad_()
    dy = torch.randn(N, Do, generator=g).to(BF16).to(DEV)
    got = _grads(x, layers, act, dy)
    assert got[0].dtype is BF16 and got[1].dtype is xt and all(t is None or t.dtype is wt for t in got[2:])
    for name, t, (want, err) in zip(NAMES, got, _exact(x, layers, act, dy)):
        if t is not None:
            _near(t, want, err, name)
    with torch.no_grad():  # nothing kept: the same values, from other kernels up to 32 rows
        y = _ffn(x, *layers, act=act)
    if N > 32:
        assert torch.equal(y, got[0])
    _near(y, *_exact(x, layers, act, dy)[0], "y alone")
    again = _grads(x, layers, act, dy)
    assert all(a is None or torch.equal(a, b) for a, b in zip(got, again))


def _whole(N, D, F, Do, seed=0):
    """Whole numbers for which every step is exact: a >= 32, where SiLU is a and its slope 1 in fp32."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(1, 3, (N, D), generator=g).double()
    w1, w3, w2 = torch.zeros(F, D).double(), torch.zeros(F, D).double(), torch.zeros(Do, F).double()
    f, o = torch.arange(F), torch.arange(Do)
    w1[f, f % D] = 32
    w3[f, (3 * f + 1) % D] = torch.randint(0, 2, (F,), generator=g).double() * 2 - 1
    w2[o, (5 * o + 2) % F] = torch.randint(0, 2, (Do,), generator=g).double() * 2 - 1
    dy = torch.randint(-1, 3, (N, Do), generator=g).double()
    return [t.to(DEV) for t in (x, w1, w3, w2, dy)]


@pytest.mark.parametrize("shape", [(1, 8, 8, 8), (3, 16, 64, 8), (40, 64, 72, 64), (64, 200, 136, 136), (65, 8, 1000, 24), (130, 264, 264, 520),
                                   (257, 128, 320, 128), (513, 520, 776, 264), (2100, 64, 128, 64)], ids=str)
def test_whole_numbers_are_exact(shape):
    N, D, F, Do = shape
    x, w1, w3, w2, dy = _whole(N, D, F, Do)
    layers = []
    for w in (w1, w3, w2):
        m = torch.nn.Linear(*reversed(w.shape), bias=False, device="meta")
        m.weight = torch.nn.Parameter(w.to(BF16))
        layers.append(m)
    got = _grads(x.to(BF16).requires_grad_(), layers, "silu", dy.to(BF16))
    a, u, dh = x @ w1.t(), x @ w3.t(), dy @ w2
    da, du = dh * u, dh * a
    want = [(a * u) @ w2.t(), da @ w1 + du @ w3, da.t() @ x, None, du.t() @ x, None, dy.t() @ (a * u), None]
    for name, t, v in zip(NAMES, got, want):
        if v is not None:
            assert torch.equal(t, v.to(BF16)), name
    # differences: y is quadratic here, so a central difference of a whole step is its derivative
    for n, d in ((0, 0), (N - 1, D // 2)):
        step = torch.zeros_like(x)
        step[n, d] = 1
        w = [m.weight.detach() for m in layers]
        up, down = ((a_ := (x + k * step) @ w1.t()) * ((x + k * step) @ w3.t()) for k in (1, -1))
        diff = float((((up - down) @ w2.t()) * dy).sum() / 2)
        assert float(got[1][n, d]) == float(torch.tensor(diff).to(BF16)) and len(w) == 3


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_over_their_range(act):
    """One input, one unit: act(a) u for a from -12 to 12, relative to itself (bf16 of h and of y: 2 b), and both gradients."""
    a = torch.linspace(-12, 12, 4096).to(BF16)
    x = torch.zeros(4096, 8)
    x[:, 0], x[:, 1] = a.float(), 1.0
    x = x.to(BF16).to(DEV).requires_grad_()
    layers = _layers(8, 8, 8, bias=False)
    with torch.no_grad():
        for m in layers:
            m.weight.zero_()
        layers[0].weight[0, 0] = layers[1].weight[0, 1] = layers[2].weight[0, 0] = 1.0
    dy = torch.zeros(4096, 8, dtype=BF16, device=DEV)
    dy[:, 0] = 1.0
    y, dx, *_ = _grads(x, layers, act, dy)
    f, df = _act(act, a.double().to(DEV))
    tiny = 2.0 ** -100
    assert bool(((y[:, 0].double() - f).abs() <= (2 * B16 + 3e-5) * f.abs() + tiny).all())
    assert bool(((dx[:, 1].double() - f).abs() <= (2 * B16 + 1e-4) * f.abs() + tiny).all())
    assert bool(((dx[:, 0].double() - df).abs() <= (2 * B16 + 1e-4) * df.abs() + 2e-5).all())


@pytest.mark.parametrize("lead", [(0,), (2, 0), (2, 3, 5), ()])
def test_leading_axes(lead):
    layers = _layers(24, 40, 16)
    x = torch.randn(*lead, 24, generator=torch.Generator().manual_seed(2)).to(BF16).to(DEV).requires_grad_()
    dy = torch.ones(*lead, 16, dtype=BF16, device=DEV)
    got = _grads(x, layers, "silu", dy)
    assert got[0].shape == (*lead, 16) and got[1].shape == x.shape
    flat = _grads(x.detach().reshape(-1, 24).requires_grad_(), layers, "silu", dy.reshape(-1, 16))
    assert all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, flat))
    if x.numel() == 0:
        assert all(bool((t == 0).all()) for t in got[1:])


def test_strides_and_alignment():
    layers = _layers(64, 96, 64, bias=False)
    big = torch.randn(50, 3, 67, generator=torch.Generator().manual_seed(3)).to(BF16).to(DEV)
    x = big[:, 1, 2:66]
    with torch.no_grad():
        want = _ffn(x.contiguous(), *layers)
        assert torch.equal(_ffn(x, *layers), want)
        assert torch.equal(_ffn(x.t().contiguous().t(), *layers), want)
    other = []
    for m in layers:
        n = torch.nn.Linear(1, 1, bias=False)
        flat = torch.empty(m.weight.numel() + 1, dtype=BF16, device=DEV)
        flat[1:] = m.weight.detach().t().reshape(-1)
        n.weight = torch.nn.Parameter(flat[1:].view(m.weight.shape[1], m.weight.shape[0]).t())
        other.append(n)
    with torch.no_grad():
        assert torch.equal(_ffn(x, *other), want)
    dy = torch.randn(64, generator=torch.Generator().manual_seed(4)).to(BF16).to(DEV)
    x0 = x.detach().requires_grad_()
    a = _grads(x0, layers, "silu", dy.expand(50, 64))
    b = _grads(x.contiguous().requires_grad_(), other, "silu", dy.expand(50, 64).contiguous())
    assert all(s is None or torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("which", range(7))
def test_single_gradients(which):
    """Whatever asks for a gradient alone gets the same bits as with the others."""
    layers = _layers(72, 136, 40)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(90, 72, generator=g).to(BF16).to(DEV).requires_grad_()
    dy = torch.randn(90, 40, generator=g).to(BF16).to(DEV)
    full = _grads(x, layers, "gelu", dy)
    ps = [x] + [p for m in layers for p in (m.weight, m.bias)]
    for i, p in enumerate(ps):
        p.requires_grad_(i == which)
    got = _grads(x, layers, "gelu", dy)
    assert torch.equal(got[0], full[0]) and torch.equal(got[1 + which], full[1 + which])
    assert sum(t is not None for t in got) == 2


def test_rows_stay_apart():
    """NaN and infinities in one row reach that row of y and dx alone (and every weight gradient, as in any product)."""
    layers = _layers(64, 128, 64, bias=False)
    g = torch.Generator().manual_seed(6)
    x = torch.randn(200, 64, generator=g).to(BF16).to(DEV)
    dy = torch.randn(200, 64, generator=g).to(BF16).to(DEV)
    clean = _grads(x.clone().requires_grad_(), layers, "silu", dy)
    x[77, 3], x[150, 9] = float("nan"), float("inf")
    got = _grads(x.requires_grad_(), layers, "silu", dy)
    keep = torch.ones(200, dtype=torch.bool, device=DEV)
    keep[77] = keep[150] = False
    for i in (0, 1):
        assert torch.equal(got[i][keep], clean[i][keep]) and bool(got[i][77].isnan().all())
    with torch.no_grad():  # the kernels for few rows
        a, b = _ffn(x[60:84].detach(), *layers), _ffn(x[140:160].detach(), *layers)
        c = _ffn(torch.where(x.isfinite(), x, 0.0)[60:84].detach(), *layers)
    keep = torch.arange(24, device=DEV) != 17
    assert torch.equal(a[keep], c[keep]) and bool(a[17].isnan().all())
    assert bool(b[10].isnan().any()) and bool(b[:10].isfinite().all()) and bool(b[11:].isfinite().all())


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 23, 24, 31, 32])
def test_few_rows_forward_alone(N):
    """The kernels for up to 32 rows: exact on whole numbers, each row's bits whatever the others are."""
    for D, F, Do in ((8, 8, 8), (24, 40, 8), (264, 520, 72), (1408, 4096, 1408)):
        x, w1, w3, w2, _ = _whole(N, D, F, Do)
        layers = []
        for w in (w1, w3, w2):
            m = torch.nn.Linear(*reversed(w.shape), bias=False, device="meta")
            m.weight = torch.nn.Parameter(w.to(BF16))
            layers.append(m)
        with torch.no_grad():
            y = _ffn(x.to(BF16), *layers)
        assert torch.equal(y, (((x @ w1.t()) * (x @ w3.t())) @ w2.t()).to(BF16)), (D, F, Do)
    layers = _layers(136, 264, 136)
    x = torch.randn(N, 136, generator=torch.Generator().manual_seed(N)).to(BF16).to(DEV)
    with torch.no_grad():
        y = _ffn(x, *layers, act="gelu")
        for i in {0, N // 2, N - 1}:
            assert torch.equal(_ffn(x[i:i + 1], *layers, act="gelu")[0], y[i])


def test_a_large_h_of_few_rows():
    """h past bf16's range, which its two halves cannot hold: infinite, as where it is rounded."""
    layers = _layers(8, 8, 8, bias=False)
    with torch.no_grad():
        for m in layers:
            m.weight.zero_()
        layers[0].weight[0, 0] = layers[1].weight[0, 1] = layers[2].weight[0, 0] = 1.0
        x = torch.zeros(2, 8, dtype=BF16, device=DEV)
        x[0, 0], x[0, 1] = 2.0 ** 64, 2.0 ** 63
        x[1, 0], x[1, 1] = 2.0 ** 100, 2.0 ** 100
        y = _ffn(x, *layers)
    assert float(y[0, 0]) == 2.0 ** 127 and float(y[1, 0]) == float("inf")


def test_streams_and_replays():
    layers = _layers(128, 320, 128)
    ps = [p for m in layers for p in (m.weight, m.bias)]
    g = torch.Generator().manual_seed(7)
    xs = [torch.randn(300, 128, generator=g).to(BF16).to(DEV) for _ in range(3)]
    dy = torch.randn(300, 128, generator=g).to(BF16).to(DEV)
    want = [_grads(x.clone().requires_grad_(), layers, "silu", dy) for x in xs]
    torch.cuda.synchronize()
    got = []
    for x in xs[:2]:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(_grads(x.clone().requires_grad_(), layers, "silu", dy))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(s, t) for s, t in zip(a, b))
    held = xs[0].clone().requires_grad_()
    copies = _layers(128, 320, 128)
    for m, n in zip(copies, layers):
        m.load_state_dict(n.state_dict())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _grads(held, copies, "silu", dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _grads(held, copies, "silu", dy)
    for i in (1, 0, 2):
        with torch.no_grad():
            held.copy_(xs[i])
        eager = _grads(xs[i].clone().requires_grad_(), layers, "silu", dy)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s, t) and torch.equal(s, e) for s, t, e in zip(out, want[i], eager))
    assert len(ps) == 6


@pytest.mark.parametrize("N", [3, 70])
def test_an_infinite_gradient_stays_infinite(N):
    # positive weights and values: every gradient of row 0 is infinite, none is 0 times infinity (but the lower half of h in few
    # rows).  F is no whole step of the products over F, and W2 has zeros in the rows that dy's row 0 does not read
    layers = _layers(8, 8, 16, bias=False)
    with torch.no_grad():
        for m in layers:
            m.weight.fill_(0.5)
        layers[2].weight[1:] = 0.0
    x = torch.ones(N, 8, dtype=BF16, device=DEV, requires_grad=True)
    dy = torch.zeros(N, 16, dtype=BF16, device=DEV)
    dy[0, 0], dy[1:] = float("inf"), 1.0
    y = _ffn(x, *layers)
    dx, dw1, dw3, dw2 = torch.autograd.grad(y, [x] + [m.weight for m in layers], dy)
    assert bool((dx[0] == float("inf")).all()) and bool(dx[1:].isfinite().all())
    assert bool((dw1 == float("inf")).all()) and bool((dw3 == float("inf")).all())
    assert bool((dw2[0] == float("inf")).all() if N > 64 else (~dw2[0].isfinite()).all()) and bool(dw2[1:].isfinite().all())


def test_no_second_derivatives():
    layers = _layers(16, 24, 16)
    x = torch.randn(5, 16, device=DEV, dtype=BF16, requires_grad=True)
    dx, = torch.autograd.grad(_ffn(x, *layers).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.float().sum().backward()


def test_two_graphs_at_once():
    # each has its own memory: replayed side by side on two streams they give what each gives alone
    g = torch.Generator().manual_seed(11)
    runs = []

    def call(x, layers, dy):
        out = _grads(x, layers, "gelu", dy)
        with torch.no_grad():  # forward alone
            return out + [_ffn(x, *layers, act="gelu")]
    for n, seed in ((300, 0), (5, 1)):
        layers = _layers(128, 320, 128, seed=seed)
        x = torch.randn(n, 128, generator=g).to(BF16).to(DEV).requires_grad_()
        dy = torch.randn(n, 128, generator=g).to(BF16).to(DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = [t.clone() for t in call(x, layers, dy)]
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(x, layers, dy)
        runs.append((graph, out, want, side, layers, x, dy))
    for _ in range(3):
        torch.cuda.synchronize()
        for graph, *_, side, _, _, _ in runs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, *_ in runs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_vectorised_calls_are_refused():
    layers = _layers(16, 24, 16)
    x = torch.randn(2, 5, 16, device=DEV, dtype=BF16)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda v: _ffn(v, *layers))(x)


@pytest.mark.parametrize("N", [1, 5, 40, 64, 70, 200])
@pytest.mark.parametrize("sizes", [(8, 8, 8), (40, 136, 24), (136, 24, 40), (56, 200, 56)], ids=str)
def test_nothing_behind_the_operands_is_read(N, sizes):
    """x, the weights and dy end where NaN begin: of rows shorter than 64 elements too, no result depends on what lies behind them."""
    D, F, Do = sizes

    def held(rows, cols, behind, size=1.0):
        t = torch.full((rows * cols + 4096,), behind, dtype=BF16, device=DEV)
        t[:rows * cols] = (torch.randn(rows * cols, generator=torch.Generator().manual_seed(rows * 1000 + cols)) * size).to(BF16).to(DEV)
        return t[:rows * cols].view(rows, cols)

    def results(behind):
        layers = _layers(D, F, Do)
        for m in layers:
            m.weight = torch.nn.Parameter(held(*m.weight.shape, behind, m.weight.shape[1] ** -0.5))
        x, dy = held(N, D, behind).requires_grad_(), held(N, Do, behind)
        out = _grads(x, layers, "gelu", dy)
        with torch.no_grad():
            return out + [_ffn(x, *layers, act="gelu")]
    for name, a, b in zip((*NAMES, "y alone"), results(float("nan")), results(0.0)):
        assert bool(a.isfinite().all()) and torch.equal(a, b), name


# Sizes whose products take the larger tiles, and which of them do (tests/test_lm_operators.py holds the choice to this list): rows and
# columns end inside tiles, with biases and without, both activations, weight gradients of both types.  "split": the contraction is.
LARGE = [
    ((333, 1408, 4096, 1408, "silu", False, BF16, F32), {"dw": "WIDE"}),
    ((4100, 1536, 1024, 1536, "gelu", True, BF16, BF16), {"gate": "BIG"}),
    ((8190, 1408, 1200, 1408, "silu", True, BF16, BF16), {"out": "WIDE", "dx": "WIDE"}),
    ((5000, 777, 3001, 777, "gelu", True, F32, F32), {"gate": "BIG", "dx": "BIG split"}),  # more tiles of the gate than run at a time
    ((9432, 1160, 200, 1160, "silu", True, BF16, F32), {"out": "BIG", "dx": "BIG"}),
    ((4542, 89, 6841, 521, "silu", True, BF16, F32), {"gate": "BIG", "out": "WIDE split", "dgate": "BIG", "dw2": "BIG split"}),
    ((73, 1792, 2536, 3896, "gelu", False, BF16, BF16), {"dw": "WIDE", "dw2": "WIDE"}),
    ((70, 2001, 3877, 3488, "silu", True, BF16, F32), {"dw": "BIG", "dw2": "BIG"}),
    ((9469, 136, 3832, 8, "gelu", False, BF16, BF16), {"gate": "BIG", "dx": "WIDE split", "dw": "WIDE split"}),
    ((5105, 824, 2555, 8, "silu", False, BF16, F32), {"gate": "BIG", "dx": "BIG split", "dw": "BIG split"}),
    ((1219, 24, 4176, 3267, "gelu", True, BF16, BF16), {"gate": "BIG", "out": "BIG split", "dw2": "BIG"}),
    ((10806, 8, 792, 2408, "silu", True, BF16, F32), {"out": "BIG", "dgate": "BIG", "dw2": "WIDE split"}),
]


@pytest.fixture
def unwritten_memory_is_nan():
    """New buffers hold NaN: what is read of them without having been written shows."""
    held = torch.utils.deterministic.fill_uninitialized_memory, torch.are_deterministic_algorithms_enabled()
    torch.utils.deterministic.fill_uninitialized_memory = True
    torch.use_deterministic_algorithms(True, warn_only=True)
    yield
    torch.utils.deterministic.fill_uninitialized_memory = held[0]
    torch.use_deterministic_algorithms(held[1])


@pytest.mark.parametrize("case", [c for c, _ in LARGE], ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_values_and_gradients_on_the_larger_tiles(case, unwritten_memory_is_nan):
    test_values_and_gradients(case)


@pytest.mark.parametrize("shape", [c[:4] for c, _ in LARGE], ids=str)
def test_whole_numbers_on_the_larger_tiles(shape):
    test_whole_numbers_are_exact(shape)


@pytest.mark.parametrize("N", [1, 5, 33, 64, 65, 200])
@pytest.mark.parametrize("sizes", [(72, 136, 40), (264, 520, 264), (777, 1001, 250)], ids=str)
def test_nothing_is_read_that_was_not_written(N, sizes, unwritten_memory_is_nan):
    D, F, Do = sizes
    layers = _layers(D, F, Do)
    g = torch.Generator().manual_seed(N)
    x = torch.randn(N, D, generator=g).to(BF16).to(DEV).requires_grad_()
    dy = torch.randn(N, Do, generator=g).to(BF16).to(DEV)
    assert bool(torch.empty(1000, dtype=torch.uint8, device=DEV).eq(255).all())
    got = _grads(x, layers, "silu", dy)
    with torch.no_grad():
        got.append(_ffn(x, *layers))
    torch.utils.deterministic.fill_uninitialized_memory = False
    want = _grads(x, layers, "silu", dy)
    for name, a, b in zip((*NAMES, "y alone"), got, want + [got[-1]]):
        assert bool(a.isfinite().all()), name
        assert torch.equal(a, b), (name, int((a != b).sum()), float((a.double() - b.double()).abs().max()), (a != b).nonzero()[:4].tolist())


def test_the_work_that_calls_log():
    """Operations of the products: 2 N F for each column of x read twice and of y written once, and twice that backward."""
    from llattn_amd import ops
    N, D, F, Do = 70, 16, 24, 40
    layers = _layers(D, F, Do)
    x = torch.ones(N, D, dtype=BF16, device=DEV, requires_grad=True)
    ops.EVENT_LOG = []
    try:
        _grads(x, layers, "silu", torch.ones(N, Do, dtype=BF16, device=DEV))
        work = {name: w for name, _, _, w in ops.EVENT_LOG}
    finally:
        ops.EVENT_LOG = None
    n = 2 * N * F * (2 * D + Do)
    assert work["llattn_gated_fwd"] == n and work["llattn_gated_bwd"] == 2 * n
