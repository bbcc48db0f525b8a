"""The piecewise head loss (``llattn_amd.xent.piecewise_head_loss``) on the GPU against a plain float64 one.

Tolerances are counted, not fitted.  With u = 2^-24 (half a step of fp32) and b = 2^-8 (of bf16): a logit of D exact
bf16 products summed in fp32 is off by at most D u (|h| |W|^T); the loss adds the base-2 exponentials and the sums
(a few u each, at most V / 64 + 300 in a row).  dl is rounded to bf16 once (b of itself) and follows the logits' error
e (2 e of itself); the gradients sum those, in fp32, and are rounded once more to their own type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U, B16 = 2.0 ** -24, 2.0 ** -8
BF16, F32 = torch.bfloat16, torch.float32


def _loss(*a, **k):
    from llattn_amd.xent import piecewise_head_loss
    return piecewise_head_loss(*a, **k)


def _inputs(N, D, V, seed=0, dtype=BF16, scale=1.0, ignore=0.2):
    g = torch.Generator().manual_seed(seed)
    h = (torch.randn(N, D, generator=g) * scale).to(dtype)
    w = (torch.randn(V, D, generator=g) * 2.0 / D ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), generator=g)
    t[torch.rand(N, generator=g) < ignore] = -100
    return h.to(DEV), w.to(DEV), t.to(DEV)


def _exact(h, w, t, grad=None, reduction="mean"):
    """float64 (loss, dh, dw) and the bounds of their errors; h and w as bf16 holds them."""
    h, w = h.to(BF16).double(), w.to(BF16).double()
    V, D = w.shape
    logits = h @ w.t()
    mag = (h.abs() @ w.abs().t()).amax(1)
    lse = torch.logsumexp(logits, 1)
    keep = t != -100
    at = t.clamp(0, V - 1)
    rows = torch.arange(len(t), device=t.device)
    loss = torch.where(keep, lse - logits[rows, at], 0.0)
    e = U * (2 * (D + 8) * mag + (V / 64 + 300) * (1 + loss.abs() + lse.abs()))
    n = keep.sum()
    s = torch.ones_like(loss) if reduction != "mean" else torch.ones_like(loss) / n
    if grad is not None:
        s = s * grad.double()
    s = torch.where(keep, s, 0.0)
    p = torch.exp(logits - lse[:, None])
    p[rows, at] -= 1.0
    dl = p * s[:, None]
    el = (B16 * dl.abs() + (2 * e + 8 * U)[:, None] * torch.exp(logits - lse[:, None]) * s[:, None].abs())
    dh, dw = dl @ w, dl.t() @ h
    K = max(V, len(t))
    eh = el @ w.abs() + K * U * (dl.abs() @ w.abs())
    ew = el.t() @ h.abs() + K * U * (dl.abs().t() @ h.abs())
    return (loss, e), (dh, eh), (dw, ew)


def _near(got, want, err, dtype, what):
    assert got.dtype is dtype, what
    step = B16 if dtype is BF16 else U
    off = (got.double() - want).abs()
    bound = 1.01 * (err + step * (want.abs() + err)) + 1e-30
    worst = float((off / bound).max()) if off.numel() else 0.0
    print(f"{what}: {worst:.3f} of the bound", flush=True)
    assert torch.isfinite(got).all() and worst <= 1.0, f"{what}: {worst} of the bound"


SIZES = [(1, 8, 1), (1, 64, 100), (5, 24, 7), (63, 128, 509), (64, 136, 1000), (65, 128, 1001), (129, 250, 4099),
         (333, 77, 513), (257, 64, 2048), (1000, 264, 3001), (700, 1408, 1000), (300, 128, 40000)]


@pytest.mark.parametrize("N,D,V", SIZES)
@pytest.mark.parametrize("piece", [0, 256])
def test_loss_and_gradients(N, D, V, piece):
    if piece and V > 5000:
        piece = 8192
    h, w, t = _inputs(N, D, V, seed=N + V)
    if N > 1:
        t[0] = 0
    h.requires_grad_(True)
    w.requires_grad_(True)
    (l, el), (dh, eh), (dw, ew) = _exact(h.detach(), w.detach(), t)
    rows = _loss(h.detach(), w.detach(), t, reduction="none")
    _near(rows, l, el, F32, "loss")
    if bool((t == -100).all()):
        return
    loss = _loss(h, w, t, piece=piece)
    n = int((t != -100).sum())
    _near(loss.detach(), l.sum() / n, el.sum() / n, F32, "mean")
    gh, gw = torch.autograd.grad(loss, (h, w))
    _near(gh, dh, eh, BF16, "dh")
    _near(gw, dw, ew, BF16, "dw")


@pytest.mark.parametrize("N,D,V", [(40, 200, 200003), (300, 72, 70001), (777, 64, 33000), (2100, 192, 40001)])
def test_many_tiles_a_workgroup(N, D, V):
    """More tiles than workgroups: odd numbers of steps, rows and columns that end inside a tile, gradients row by row,
    targets that count for nothing or lie outside."""
    h, w, t = _inputs(N, D, V, seed=V)
    g = torch.randn(N, generator=torch.Generator().manual_seed(2)).to(DEV)
    t[N // 2], t[N - 1] = V - 1, -100
    (l, el), (dh, eh), (dw, ew) = _exact(h, w, t, g, "none")
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    rows, pred = _loss(hg, wg, t, reduction="none", return_pred=True)
    _near(rows.detach(), l, el, F32, "loss")
    assert torch.equal(rows.detach(), _loss(h, w, t, reduction="none"))
    gh, gw = torch.autograd.grad(rows, (hg, wg), g)
    _near(gh, dh, eh, BF16, "dh")
    _near(gw, dw, ew, BF16, "dw")
    logits = h.double() @ w.double().t()
    top = logits.gather(1, pred.long()[:, None]).squeeze(1)
    assert bool((logits.amax(1) - top <= 2 * D * U * (h.double().abs() @ w.double().abs().t()).amax(1)).all())
    t[1] = V
    rows = _loss(h, w, t, reduction="none")
    assert torch.isnan(rows).nonzero().flatten().tolist() == [1]


@pytest.mark.parametrize("reduction", ["sum", "none", "mean"])
@pytest.mark.parametrize("which", ["h", "w", "both"])
def test_reductions_and_upstream_gradients(reduction, which):
    """A gradient that is not 1, per row for "none"; one input frozen."""
    N, D, V = 200, 96, 777
    h, w, t = _inputs(N, D, V, seed=3)
    h, w = h.view(4, 50, D).requires_grad_(which != "w"), w.requires_grad_(which != "h")
    t3 = t.view(4, 50)
    out = _loss(h, w, t3, reduction=reduction)
    g = torch.randn(N, generator=torch.Generator().manual_seed(1)).to(DEV) if reduction == "none" else torch.full((N,), -2.5, device=DEV)
    assert out.shape == (t3.shape if reduction == "none" else ())
    out.backward(g.view(4, 50) if reduction == "none" else g[0])
    (l, el), (dh, eh), (dw, ew) = _exact(h.detach().view(N, D), w.detach(), t, g, reduction)
    if reduction == "sum":
        _near(out.detach(), l.sum(), el.sum(), F32, "sum")
    if which != "w":
        _near(h.grad.view(N, D), dh, eh, BF16, "dh")
    else:
        assert h.grad is None
    if which != "h":
        _near(w.grad, dw, ew, BF16, "dw")
    else:
        assert w.grad is None


def test_fp32_inputs_are_rounded_as_under_autocast():
    h, w, t = _inputs(150, 64, 999, seed=4, dtype=F32)
    h.requires_grad_(True)
    w.requires_grad_(True)
    gh, gw = torch.autograd.grad(_loss(h, w, t), (h, w))
    _, (dh, eh), (dw, ew) = _exact(h.detach(), w.detach(), t)
    _near(gh, dh, eh + B16 * (dh.abs() + eh), F32, "dh")  # formed in bf16, handed over in fp32
    _near(gw, dw, ew, F32, "dw")


def test_strided_and_shifted_inputs():
    """Rows inside wider ones, a column step, an unaligned base, transposed weights, int32 targets."""
    N, D, V = 97, 64, 300
    h, w, t = _inputs(N, D, V, seed=5)
    want = _loss(h, w, t, reduction="none")
    wide = torch.zeros(N, 3 * D, dtype=BF16, device=DEV)
    wide[:, D:2 * D] = h
    step = torch.zeros(N, 2 * D, dtype=BF16, device=DEV)
    step[:, ::2] = h
    flat = torch.zeros(N * D + 1, dtype=BF16, device=DEV)
    flat[1:] = h.reshape(-1)
    for x in (wide[:, D:2 * D], step[:, ::2], flat[1:].view(N, D), h.t().contiguous().t()):
        assert torch.equal(_loss(x, w, t.to(torch.int32), reduction="none"), want)
    assert torch.equal(_loss(h, w.t().contiguous().t(), t, reduction="none"), want)
    row = h[:1].expand(N, D)  # one row, broadcast: its gradient is the sum
    leaf = h[:1].clone().requires_grad_(True)
    _loss(leaf.expand(N, D), w, t, reduction="sum").backward()
    _, (dh, eh), _ = _exact(row, w, t, None, "sum")
    _near(leaf.grad, dh.sum(0, keepdim=True), eh.sum(0, keepdim=True) + N * B16 * dh.abs().sum(0, keepdim=True), BF16, "dh")


def test_rows_that_do_not_count():
    h, w, t = _inputs(70, 64, 300, seed=6)
    t[:] = -100
    h.requires_grad_(True)
    w.requires_grad_(True)
    loss = _loss(h, w, t)
    assert torch.isnan(loss)
    gh, gw = torch.autograd.grad(loss, (h, w))
    assert not gh.any() and not gw.any()
    assert float(_loss(h, w, t, reduction="sum")) == 0.0
    # values that are not finite in an ignored row reach neither the loss nor dh of the others
    t[:35] = 1
    bad = h.detach().clone()
    bad[40] = float("inf")
    assert torch.equal(_loss(bad, w.detach(), t, reduction="none"), _loss(h.detach(), w.detach(), t, reduction="none"))
    bad.requires_grad_(True)
    gh, = torch.autograd.grad(_loss(bad, w.detach(), t), bad)
    assert torch.isfinite(gh).all() and not gh[35:].any()


def test_targets_out_of_range_give_nan():
    h, w, t = _inputs(70, 64, 300, seed=7, ignore=0.0)
    t[3], t[5] = 300, -1
    h.requires_grad_(True)
    rows = _loss(h, w, t, reduction="none")
    assert torch.isnan(rows).nonzero().flatten().tolist() == [3, 5]
    gh, = torch.autograd.grad(rows, h, torch.ones_like(rows))
    assert torch.isnan(gh).any(1).nonzero().flatten().tolist() == [3, 5]
    other = _loss(h.detach(), w, t, ignore_index=-1, reduction="none")  # another index to ignore
    assert torch.isnan(other).nonzero().flatten().tolist() == [3] and float(other[5]) == 0.0


def test_no_rows():
    w = torch.randn(50, 16, device=DEV).to(BF16).requires_grad_(True)
    h = torch.zeros(2, 0, 16, device=DEV, dtype=BF16, requires_grad=True)
    t = torch.zeros(2, 0, device=DEV, dtype=torch.int64)
    assert _loss(h, w, t, reduction="none").shape == (2, 0)
    assert float(_loss(h, w, t, reduction="sum")) == 0.0
    loss = _loss(h, w, t)
    assert torch.isnan(loss)
    gh, gw = torch.autograd.grad(loss, (h, w))
    assert gh.shape == h.shape and not gw.any()


def test_large_logits_and_infinities():
    """Logits of thousands do not overflow; an infinite one gives NaN in its row alone, as logsumexp - x does."""
    N, D, V = 40, 32, 700
    h, w, t = _inputs(N, D, V, seed=8, scale=3000.0, ignore=0.0)
    (l, el), _, _ = _exact(h, w, t)
    _near(_loss(h, w, t, reduction="none"), l, el, F32, "loss")
    x = h.clone()
    x[7, 3] = float("inf")
    rows = _loss(x, w, t, reduction="none")
    assert torch.isnan(rows).nonzero().flatten().tolist() == [7]
    # a vocabulary row at -inf everywhere has probability 0 and leaves the others' losses finite
    w2, h2 = w.clone(), h.abs() + 1
    w2[11] = float("-inf")
    t[t == 11] = 12
    rows = _loss(h2, w2, t, reduction="none")
    keep = torch.arange(V, device=DEV) != 11
    (l, el), _, _ = _exact(h2, w2[keep], torch.where(t > 11, t - 1, t))
    _near(rows, l, el, F32, "loss beside -inf")


def test_first_argmax():
    N, D, V = 130, 64, 5001
    h, w, t = _inputs(N, D, V, seed=9)
    w[700] = w[4000] = 0.0
    h[5] = 0.0          # every logit ties at 0
    h[6] = 0.0
    h[6, 0], w[:, 0] = 1.0, 0.0
    w[4000, 0] = w[700, 0] = 2.0  # two maxima, tiles apart
    loss, pred = _loss(h, w, t, reduction="none", return_pred=True)
    assert torch.equal(loss, _loss(h, w, t, reduction="none")) and pred.dtype is torch.int32
    assert int(pred[5]) == 0 and int(pred[6]) == 700
    logits = h.double() @ w.double().t()
    top = logits.gather(1, pred.long()[:, None]).squeeze(1)
    err = D * U * (h.double().abs() @ w.double().abs().t()).amax(1)
    assert bool((logits.amax(1) - top <= 2 * err).all())


def test_repeats_bit_for_bit_and_under_a_graph():
    """The same bits on every call, on another stream and in the replays of a captured step, eager work between them."""
    N, D, V = 300, 128, 3001
    h, w, t = _inputs(N, D, V, seed=10)
    h2, w2, t2 = _inputs(N, D, V, seed=11)
    def step(h, w, t):
        h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
        loss = _loss(h, w, t, piece=1024)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))
    first, second = step(h, w, t), step(h2, w2, t2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(h, w, t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(first, other))
    bh, bw, bt = h.clone(), w.clone(), t.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(bh, bw, bt)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(bh, bw, bt)
    for src, want in (((h, w, t), first), ((h2, w2, t2), second), ((h, w, t), first)):
        for b, s in zip((bh, bw, bt), src):
            b.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        step(h2, w2, t2)
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_in_place_use_of_the_loss():
    """The loss may be scaled in place (gradient accumulation) and the hidden states are watched for changes."""
    h, w, t = _inputs(60, 64, 300, seed=12)
    h.requires_grad_(True)
    want, = torch.autograd.grad(_loss(h, w, t) / 4, h)
    loss = _loss(h, w, t)
    loss /= 4
    got, = torch.autograd.grad(loss, h)
    assert torch.equal(got, want)
    x = (h * 1.0)
    loss = _loss(x, w, t)
    x.data_ptr()
    with torch.no_grad():
        x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_against_the_row_chunked_loss():
    """The same head through lm_head_loss, which rounds its logits to bf16: equal up to that (half a step of 2^-8 of
    each logit, at both ends of the loss)."""
    from llattn_amd.xent import lm_head_loss
    h, w, t = _inputs(500, 128, 2048, seed=13)
    a, pa = lm_head_loss(h, w, t)
    b, pb = _loss(h, w, t, return_pred=True)
    most = float((h.double() @ w.double().t()).abs().max())
    assert abs(float(a) - float(b)) <= 2 * B16 * most
    assert float((pa == pb).float().mean()) > 0.9


def test_forward_in_several_ranges():
    """So many rows that the row sums of a few columns are joined at a time (256 MB of them): 300000 rows, 40 columns of
    tiles; checked on rows spread over the whole."""
    N, D, V = 300000, 8, 5200
    h, w, t = _inputs(N, D, V, seed=20)
    rows, pred = _loss(h, w, t, reduction="none", return_pred=True)
    at = torch.arange(0, N, 997, device=DEV)
    (l, el), _, _ = _exact(h[at], w, t[at])
    _near(rows[at], l, el, F32, "loss")
    logits = h[at].double() @ w.double().t()
    top = logits.gather(1, pred[at].long()[:, None]).squeeze(1)
    assert bool((logits.amax(1) - top <= 2 * D * U * (h[at].double().abs() @ w.double().abs().t()).amax(1)).all())


def test_evaluation_of_parameters():
    """Under no_grad leaves that require gradients take the same path as plain tensors: the same bits, no graph."""
    h, w, t = _inputs(90, 64, 700, seed=21)
    want, pred = _loss(h, w, t, return_pred=True)
    with torch.no_grad():
        got, p = _loss(h.clone().requires_grad_(True), torch.nn.Parameter(w), t, return_pred=True)
    assert not got.requires_grad and torch.equal(got, want) and torch.equal(p, pred)
    live = _loss(h, torch.nn.Parameter(w), t)
    assert live.requires_grad and torch.equal(live.detach(), want)


@pytest.mark.parametrize("B", [1, 3])
def test_last_position_of_long_sequences(B):
    """hidden[:, -1] of sequences so long that its rows lie 2^23 elements and more apart, and a weight of one far row."""
    T, D, V = 8192, 1024, 300
    g = torch.Generator().manual_seed(22)
    hidden = torch.zeros(B, T, D, dtype=BF16, device=DEV)
    hidden[:, -1] = torch.randn(B, D, generator=g).to(BF16).to(DEV)
    w = (torch.randn(V, D, generator=g) * 0.06).to(BF16).to(DEV)
    t = torch.randint(0, V, (B,), generator=g).to(DEV)
    leaf = hidden.clone().requires_grad_(True)
    weight = w.clone().requires_grad_(True)
    want = hidden[:, -1].clone().requires_grad_(True)
    rows = _loss(leaf[:, -1], weight, t, reduction="none")
    ref = _loss(want, weight, t, reduction="none")
    assert torch.equal(rows, ref)
    rows.sum().backward()
    gh, = torch.autograd.grad(ref.sum(), want)
    assert torch.equal(leaf.grad[:, -1], gh) and not leaf.grad[:, :-1].any()
    one = torch.zeros_like(t)  # a vocabulary of one, a row far along
    (l, el), _, _ = _exact(want.detach(), hidden[0, -1:], one)
    _near(_loss(want.detach(), hidden[:1, -1], one, reduction="none"), l, el, F32, "one column")


def _backward(h, w, t, lse2, grad, stride, inv):
    """llattn_head_bwd itself: (dh, dW)."""
    import ctypes
    from llattn_amd import _lib as L
    (N, D), V = h.shape, w.shape[0]
    cfg = L.LlattnHeadCfg(N, V, D, 256, L.BF16)
    n = L.load().llattn_head_bytes(ctypes.byref(cfg), 1)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    dh, dw = torch.empty_like(h), torch.empty(V + -V % 8, D, dtype=BF16, device=DEV)
    p = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    L.check(L.load().llattn_head_bwd(ctypes.byref(cfg), p(h), D, p(w), D, p(t), -100, p(lse2), p(grad), stride, p(inv), p(dh), p(dw),
                                     p(ws), n, L.stream_ptr(DEV)), "llattn_head_bwd")
    return dh, dw[:V]


@pytest.mark.parametrize("N,D,V", [(70, 64, 500), (300, 264, 1001)])
def test_the_rows_share_of_a_gradient_per_row(N, D, V):
    """s_n = grad[n * grad_stride] * inv: with gradients row by row as with one, and the power of two changes no bit."""
    h, w, t = _inputs(N, D, V, seed=23)
    lse2 = torch.logsumexp(h.float() @ w.float().t(), 1) / torch.log(torch.tensor(2.0))
    g = torch.randn(N, generator=torch.Generator().manual_seed(24)).to(DEV)
    inv = torch.tensor(0.125, device=DEV)
    for grad, stride in ((g, 1), (g[:1].clone(), 0)):
        want = _backward(h, w, t, lse2, grad / 8, stride, None)
        got = _backward(h, w, t, lse2, grad, stride, inv)
        assert any(x.any() for x in want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_gradient_for_all_rows_is_the_means(dtype):
    """reduction="none" with the same gradient in every row that counts, whatever stands in the others: the bits of the
    mean, whose scale is never rounded into the logits' gradient (1 / n would be, alike in every row's entry near -1)."""
    h, w, t = _inputs(333, 72, 1003, seed=25, dtype=dtype)
    h.requires_grad_(True)
    w.requires_grad_(True)
    want = torch.autograd.grad(_loss(h, w, t, piece=256), (h, w))
    keep = t != -100
    n = int(keep.sum())
    for other in (0.0, 1.0 / n, 5.0, float("nan")):
        g = torch.where(keep, torch.tensor(1.0 / n, device=DEV), torch.tensor(other, device=DEV))
        got = torch.autograd.grad(_loss(h, w, t, reduction="none", piece=256), (h, w), g)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), other
    g = torch.where(keep, torch.tensor(-1.0 / n, device=DEV), 0.0)
    got = torch.autograd.grad(_loss(h, w, t, reduction="none", piece=256), (h, w), g)
    assert all(torch.equal(a, -b) for a, b in zip(got, want))


@pytest.mark.parametrize("size", [1e-36, 1e-3, 1e30])
def test_gradients_of_any_size_row_by_row(size):
    """Some of them zero; none but zeros gives zeros."""
    h, w, t = _inputs(150, 64, 700, seed=26, ignore=0.1)
    g = torch.randn(150, generator=torch.Generator().manual_seed(27)).to(DEV) * size
    g[::3] = 0.0
    h.requires_grad_(True)
    w.requires_grad_(True)
    rows = _loss(h, w, t, reduction="none")
    gh, gw = torch.autograd.grad(rows, (h, w), g, retain_graph=True)
    _, (dh, eh), (dw, ew) = _exact(h.detach(), w.detach(), t, g, "none")
    for got, want, err, name in ((gh, dh, eh, "dh"), (gw, dw, ew, "dw")):
        # rounded once more here; below 2^-126 half a step of bf16 is 2^-134
        _near((got.double() / size).to(BF16), want / size, err / size + B16 * want.abs() / size + 2.0 ** -134 / size, BF16, name)
    gh, gw = torch.autograd.grad(rows, (h, w), torch.zeros_like(g))
    assert not gh.any() and not gw.any()
    g[1] = float("inf")  # its own row alone
    t1 = t.clone()
    t1[1] = 5
    gh, = torch.autograd.grad(_loss(h, w, t1, reduction="none"), h, g)
    assert not torch.isfinite(gh[1]).any() and torch.isfinite(gh[2:]).all() and torch.isfinite(gh[0]).all()


@pytest.mark.parametrize("N,D,V", [(1, 8, 1), (5, 24, 70), (70, 40, 509), (200, 56, 1000)])
@pytest.mark.parametrize("piece", [0, 256])
def test_nothing_behind_the_operands_is_read(N, D, V, piece):
    """h and the weight end where NaN begin: of rows shorter than 64 elements too, no result depends on what lies behind them."""
    h0, w0, t = _inputs(N, D, V)

    def results(behind):
        leaves = []
        for v in (h0, w0):
            flat = torch.full((v.numel() + 4096,), behind, dtype=BF16, device=DEV)
            flat[:v.numel()] = v.flatten()
            leaves.append(flat[:v.numel()].view(v.shape).requires_grad_())
        loss = _loss(*leaves, t, reduction="sum", piece=piece)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    for a, b in zip(results(float("nan")), results(0.0)):
        assert bool(a.isfinite().all()) and torch.equal(a, b)
