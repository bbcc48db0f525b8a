"""Token and position rows (``llattn_amd.embed``) on the GPU against plain float64 ones.

Tolerances are counted.  Half a step is ``eps / 2`` of a type (fp32 2^-24, bf16 2^-8).  A row is one fused multiply-add in
fp32 and a rounding to its type.  A gradient is a sum of L values in fp32, in whatever order off by at most L 2^-24 of
the sum of their sizes, a product with the scale and a rounding to its type.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def _embed(*a, **k):
    from llattn_amd import embed
    return embed(*a, **k)


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tables(V, P, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g).to(dtype).to(DEV)
    p = torch.randn(P, D, generator=g).to(dtype).to(DEV) if P else None
    return w, p


def _ids(shape, V, seed=1, kind="frequent"):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full(shape, V - 1, device=DEV)
    if kind == "frequent":
        return (torch.exp(torch.rand(shape, generator=g) * torch.log(torch.tensor(V + 1.0))).long() - 1).clamp(0, V - 1).to(DEV)
    return torch.randint(0, V, shape, generator=g).to(DEV)


def _check_rows(out, ids, w, p, pos, scale):
    """Forward of valid indices."""
    want = scale * w.double()[ids]
    if p is not None:
        want = want + p.double()[pos]
    bound = (_half(w.dtype) + U) * (1 + U) * want.abs() + 2.0 ** -126
    assert out.dtype is w.dtype and out.shape == want.shape
    assert bool(((out.double() - want).abs() <= bound).all())


def _check_sums(got, keys, dy, rows, scale, skip=None):
    """A table's gradient: keys [N] (those outside [0, rows) and `skip` have none), dy [N, D]."""
    ok = (keys >= 0) & (keys < rows)
    if skip is not None:
        ok &= keys != skip
    k, d = keys[ok], dy.double()[ok]
    want = torch.zeros((rows, dy.shape[1]), dtype=torch.float64, device=DEV).index_add_(0, k, d)
    size = torch.zeros_like(want).index_add_(0, k, d.abs())
    L = torch.bincount(k, minlength=rows).double().unsqueeze(1)
    err = (L + 2) * U * size * abs(scale)
    assert got.shape == want.shape
    bad = (got.double() - scale * want).abs() > err + _half(got.dtype) * ((scale * want).abs() + err) + 2.0 ** -126
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()}"


# (B, T, V, P, D, dtype, scale, kind of ids, positions given)
CASES = [
    (1, 1, 1, 1, 8, F32, 1.0, "one", False),
    (1, 1, 32000, 64, 1408, BF16, 1.0, "frequent", True),
    (3, 7, 50, 9, 1, F32, 2.5, "even", False),
    (3, 7, 50, 9, 1, BF16, 2.5, "even", True),
    (2, 333, 509, 1024, 128, F32, 1.0, "frequent", False),
    (4, 129, 300, 129, 250, BF16, 250 ** 0.5, "frequent", True),
    (5, 211, 1000, 300, 777, F32, -0.5, "frequent", True),
    (5, 211, 1000, 300, 777, BF16, 1.0, "frequent", False),
    (1, 5000, 7, 5000, 24, F32, 1.0, "one", False),          # a bucket that does not fit its list, a run of 4 x 1024 rows and more
    (40, 130, 5, 130, 72, BF16, 3.0, "even", True),          # runs of about 1040 rows
    (1100, 2, 3, 4, 36, F32, 1.0, "even", False),            # positions of 1100 rows each
    (2, 64, 200001, 70, 40, F32, 1.0, "even", False),        # more than 256 buckets
    (8, 512, 32000, 512, 136, BF16, 1.0, "frequent", True),
    (16, 1024, 3000, 1024, 24, F32, 1.0, "frequent", True),  # as many rows as 16 steps of keys hold, and one more
    (5, 3277, 3000, 3277, 24, BF16, 1.0, "frequent", True),
    (1, 32769, 700, 32769, 8, F32, 1.0, "frequent", True),   # more than 32 steps hold
    (4, 10001, 150000, 10001, 16, F32, 1.0, "even", False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(str(v) for v in c[:5]) + f"-{str(c[5])[6:]}-{c[7]}-{c[8]}")
def test_rows_and_gradients(case):
    B, T, V, P, D, dtype, scale, kind, given = case
    w, p = _tables(V, P, D, dtype)
    ids = _ids((B, T), V, kind=kind)
    pos = torch.randint(0, P, (B, T), generator=torch.Generator().manual_seed(2)).to(DEV) if given else None
    w.requires_grad_()
    p.requires_grad_()
    out = _embed(ids, w, p, positions=pos, scale=scale)
    at = torch.arange(T, device=DEV).expand(B, T) if pos is None else pos
    _check_rows(out.detach(), ids, w.detach(), p.detach(), at, scale)
    dy = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).to(dtype).to(DEV)
    dw, dp = torch.autograd.grad(out, (w, p), dy)
    assert dw.dtype is dtype and dp.dtype is dtype
    d = dy.reshape(-1, D)
    _check_sums(dw, ids.reshape(-1), d, V, scale)
    _check_sums(dp, at.reshape(-1), d, P, 1.0)
    # the forward without a gradient gives the same bits
    with torch.no_grad():
        assert torch.equal(_embed(ids, w, p, positions=pos, scale=scale), out)


@pytest.mark.parametrize("L", [0, 1, 2, 31, 32, 33, 63, 64, 65, 1023, 1024, 1025, 1055, 1056, 2048, 3105])
def test_runs_of_every_kind_of_length(L):
    """One token of L rows among others: its sum's value, and its bits whatever the others are."""
    N, V, D = 3200, 40, 20
    g = torch.Generator().manual_seed(L)
    mine = torch.randperm(N, generator=g)[:L].sort().values
    dy = torch.randn(N, D, generator=g).to(DEV)
    got = []
    for seed, lo in ((0, 0), (1, 18), (2, 30)):
        others = torch.randint(lo, V - 1, (N,), generator=torch.Generator().manual_seed(seed))
        ids = torch.where(others >= 17, others + 1, others)
        ids[mine] = 17
        w = torch.zeros(V, D, device=DEV, requires_grad=True)
        dw, = torch.autograd.grad(_embed(ids.to(DEV), w), w, dy)
        _check_sums(dw, ids.to(DEV), dy, V, 1.0)
        got.append(dw[17])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    # the rows of that token alone
    w = torch.zeros(V, D, device=DEV, requires_grad=True)
    dw, = torch.autograd.grad(_embed(torch.full((L,), 17, device=DEV), w), w, dy[mine.to(DEV)])
    assert torch.equal(dw[17], got[0])


def test_fp32_without_scale_equals_the_sum_of_two_lookups():
    w, p = _tables(300, 50, 88, F32)
    ids = _ids((3, 50), 300)
    assert torch.equal(_embed(ids, w, p), w[ids] + p[:50])
    assert torch.equal(_embed(ids, w), w[ids])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_position_rows_and_single_gradients(dtype):
    w, p = _tables(64, 30, 40, dtype)
    ids = _ids((2, 30), 64)
    dy = torch.randn(2, 30, 40, generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    w.requires_grad_()
    dw, = torch.autograd.grad(_embed(ids, w, scale=2.0), w, dy)
    _check_sums(dw, ids.reshape(-1), dy.reshape(-1, 40), 64, 2.0)
    both, = torch.autograd.grad(_embed(ids, w, p, scale=2.0), w, dy)
    assert torch.equal(both, dw)
    p.requires_grad_()
    dp, = torch.autograd.grad(_embed(ids, w.detach(), p), p, dy)
    _check_sums(dp, torch.arange(30, device=DEV).repeat(2), dy.reshape(-1, 40), 30, 1.0)


def test_padding_and_indices_out_of_range():
    V, P, D = 20, 6, 12
    w, p = _tables(V, P, D, F32)
    ids = torch.tensor([[3, -1, 20, 5, 3, 7], [5, 3, 2 ** 40, -2 ** 40, 19, 3]], device=DEV)
    pos = torch.tensor([[0, 1, 2, -1, 6, 2 ** 33], [5, 5, 5, 5, 0, 0]], device=DEV)
    w.requires_grad_()
    p.requires_grad_()
    out = _embed(ids, w, p, positions=pos, padding_idx=5)
    bad = (ids < 0) | (ids >= V) | (pos < 0) | (pos >= P)
    assert bool(out[bad].isnan().all()) and bool(out[~bad].isfinite().all())
    assert torch.equal(out[~bad], (w.detach()[ids[~bad]] + p.detach()[pos[~bad]]))
    dy = torch.randn(2, 6, D, generator=torch.Generator().manual_seed(6)).to(DEV)
    dw, dp = torch.autograd.grad(out, (w, p), dy)
    _check_sums(dw, ids.reshape(-1), dy.reshape(-1, D), V, 1.0, skip=5)
    _check_sums(dp, pos.reshape(-1), dy.reshape(-1, D), P, 1.0)
    assert bool((dw[5] == 0).all())
    # counted from the end, as torch counts it
    out = _embed(ids, w, p, positions=pos, padding_idx=5 - V)
    assert torch.equal(torch.autograd.grad(out, w, dy)[0], dw)


@pytest.mark.parametrize("shape", [(0,), (3, 0), (0, 5)])
def test_no_tokens(shape):
    w, p = _tables(9, 6, 16, F32)
    w.requires_grad_()
    p.requires_grad_()
    out = _embed(torch.zeros(shape, dtype=torch.int64, device=DEV), w, p)
    assert out.shape == (*shape, 16)
    dw, dp = torch.autograd.grad(out.sum(), (w, p))
    assert bool((dw == 0).all()) and bool((dp == 0).all()) and dw.shape == w.shape and dp.shape == p.shape


def test_one_token_without_an_axis_and_many_axes():
    w, p = _tables(9, 6, 16, F32)
    assert torch.equal(_embed(torch.tensor(4, device=DEV), w, p), w[4] + p[0])
    ids = _ids((2, 3, 2, 5), 9)
    assert torch.equal(_embed(ids, w, p), w[ids] + p[:5])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(dtype):
    """Tables that are columns of wider ones, start off 16 bytes or lie transposed; indices of 32 bits and of a slice; an upstream
    gradient that is broadcast."""
    V, P, D = 60, 33, 50
    wide = torch.randn(V, 131, generator=torch.Generator().manual_seed(7)).to(dtype).to(DEV)
    w = wide[:, 3:3 + D]
    p = torch.randn(D, P, generator=torch.Generator().manual_seed(8)).to(dtype).to(DEV).t()
    ids = _ids((4, 66), V)[:, ::2]
    want = _embed(ids.contiguous(), w.contiguous(), p.contiguous())
    for i in (ids, ids.to(torch.int32), ids.to(torch.int16), ids.to(torch.uint8)):
        assert torch.equal(_embed(i, w, p), want)
    pos = torch.arange(33, device=DEV, dtype=torch.int32).expand(4, 33)
    assert torch.equal(_embed(ids, w, p, positions=pos), want)
    w0, p0 = w.detach().requires_grad_(), p.detach().requires_grad_()
    dy = torch.randn(D, generator=torch.Generator().manual_seed(9)).to(dtype).to(DEV)
    dw, dp = torch.autograd.grad(_embed(ids, w0, p0), (w0, p0), dy.expand(4, 33, D))
    full = dy.expand(4, 33, D).reshape(-1, D)
    _check_sums(dw, ids.reshape(-1), full, V, 1.0)
    _check_sums(dp, torch.arange(33, device=DEV).repeat(4), full, P, 1.0)


def test_special_values_stay_in_their_rows():
    w, p = _tables(6, 3, 9, F32)
    w[1, 2], w[2, 3], p[0, 1] = float("inf"), float("nan"), float("-inf")
    ids = torch.tensor([[0, 1, 2], [3, 1, 0]], device=DEV)
    assert torch.equal(_embed(ids, w, p).nan_to_num(nan=123.0), (w[ids] + p).nan_to_num(nan=123.0))
    w0 = torch.zeros(6, 9, device=DEV, requires_grad=True)
    dy = torch.ones(2, 3, 9, device=DEV)
    dy[0, 1] = float("nan")
    dy[1, 2, 4] = float("inf")
    dw, = torch.autograd.grad(_embed(ids, w0), w0, dy)
    want = torch.zeros(6, 9)
    want[0], want[1], want[2], want[3] = 2, float("nan"), 1, 1
    want[0, 4] = float("inf")
    assert torch.equal(dw.cpu().nan_to_num(nan=123.0, posinf=456.0), want.nan_to_num(nan=123.0, posinf=456.0))


def test_differences():
    """The gradient of a weighted sum of the output against differences of it (exact: the output is linear)."""
    w, p = _tables(11, 8, 6, F32)
    ids = _ids((3, 8), 11, kind="even")
    dy = torch.randint(-4, 5, (3, 8, 6), generator=torch.Generator().manual_seed(4)).float().to(DEV)
    w, p = w.mul(8).round(), p.mul(8).round()
    w.requires_grad_()
    p.requires_grad_()
    dw, dp = torch.autograd.grad(_embed(ids, w, p, scale=2.0), (w, p), dy)
    with torch.no_grad():
        f = lambda a, b: (_embed(ids, a, b, scale=2.0) * dy).double().sum()  # noqa: E731
        base = f(w, p)
        for table, grad in ((0, dw), (1, dp)):
            for r, c in ((0, 0), (3, 5), (7, 2)):
                t = [w.detach().clone(), p.detach().clone()]
                t[table][r, c] += 1.0
                assert float(f(*t) - base) == float(grad[r, c])


def test_another_stream_and_two_at_once():
    w, p = _tables(500, 100, 264, F32)
    w.requires_grad_()
    p.requires_grad_()
    work = [(_ids((6, 100), 500, seed=s), torch.randn(6, 100, 264, generator=torch.Generator().manual_seed(s)).to(DEV)) for s in (1, 2)]
    want = [torch.autograd.grad(_embed(i, w, p), (w, p), d) for i, d in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    got = []
    for s, (i, d) in zip(streams, work):
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(_embed(i, w, p), (w, p), d))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_and_replayed():
    """Forward and backward in a graph, replayed with other tokens, eager work between the replays."""
    V, P, D, B, T = 700, 90, 128, 20, 90
    w, p = _tables(V, P, D, F32)
    w.requires_grad_()
    p.requires_grad_()
    ids = _ids((B, T), V)
    dy = torch.randn(B, T, D, generator=torch.Generator().manual_seed(1)).to(DEV)
    leaves = [t.detach().clone().requires_grad_() for t in (w, p)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(_embed(ids, *leaves, scale=3.0), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _embed(ids, *leaves, scale=3.0)
        dw, dp = torch.autograd.grad(out, leaves, dy)
    for seed in range(4):
        new = _ids((B, T), V, seed=10 + seed, kind="one" if seed == 2 else "frequent")
        ids.copy_(new)
        want = _embed(new, w, p, scale=3.0)
        grads = torch.autograd.grad(want, (w, p), dy)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(dw, grads[0]) and torch.equal(dp, grads[1])


def test_offsets_past_32_bits():
    """An output and tables of more than 2^32 bytes: the last rows are as right as the first."""
    V, D, N = 70000, 16384, 140000
    w = torch.zeros((V, D), dtype=BF16, device=DEV)
    rows = torch.tensor([0, 1, V - 2, V - 1], device=DEV)
    w[rows] = torch.arange(4 * D, device=DEV).reshape(4, D).remainder(251).to(BF16)
    ids = torch.full((N,), V - 1, device=DEV, dtype=torch.int32)
    ids[:4] = rows.int()
    ids[5::7] = 2
    w.requires_grad_()
    out = _embed(ids, w)
    for i in (0, 1, 2, 3, 4, N - 1):
        assert torch.equal(out[i], w.detach()[int(ids[i])])
    dy = torch.zeros_like(out)
    dy[-1], dy[-2], dy[3] = 1.0, 2.0, 4.0
    dw, = torch.autograd.grad(out, w, dy)
    last = [v for v, at in ((1.0, N - 1), (2.0, N - 2), (4.0, 3)) if int(ids[at]) == V - 1]
    assert bool((dw[V - 1] == sum(last)).all()) and bool((dw[3:V - 1] == 0).all())


def test_no_second_derivatives():
    w, p = (t.requires_grad_() for t in _tables(11, 6, 8, F32))
    y = _embed(_ids((2, 6), 11), w, p)
    dw, = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dw.sum().backward()


def test_vectorised_calls_are_refused():
    w, _ = _tables(11, 0, 8, F32)
    with pytest.raises(RuntimeError):
        torch.vmap(lambda i: _embed(i, w))(_ids((2, 6), 11))


def test_two_graphs_at_once():
    # each has its own memory: replayed side by side on two streams they give what each gives alone
    runs = []
    for shape, V, P in (((4, 700), 5000, 700), ((3, 900), 300, 1000)):
        w, p = (t.requires_grad_() for t in _tables(V, P, 136, F32))
        ids, dy = _ids(shape, V), torch.randn(*shape, 136, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())

        def call(ids=ids, w=w, p=p, dy=dy):
            y = _embed(ids, w, p)
            return [y.detach(), *torch.autograd.grad(y, (w, p), dy)]
        with torch.cuda.stream(side):
            want = [t.clone() for t in call()]
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        runs.append((graph, out, want, side, call))  # a graph reads its inputs where they are
    for _ in range(3):
        torch.cuda.synchronize()
        for graph, _, _, side, _ in runs:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _, _ in runs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("value", [-1, 4999, 5000, 1 << 20, (1 << 31) - 1, 1 << 40])
def test_indices_written_over_before_the_backward(value):
    # past the version counter, which refuses the backward otherwise: the tokens' sums are anything, the positions' right
    w, p = (t.requires_grad_() for t in _tables(5000, 700, 136, F32))
    ids = _ids((4, 700), 5000)
    y = _embed(ids, w, p, positions=torch.arange(700, device=DEV).expand(4, 700).contiguous())
    ids.data.fill_(value)
    dw, dp = torch.autograd.grad(y, (w, p), torch.ones_like(y))
    assert dw.shape == w.shape and torch.equal(dp, torch.full_like(dp, 4.0))
    ids = _ids((4, 700), 5000)
    y = _embed(ids, w, p)
    ids.fill_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, (w, p), torch.ones_like(y))


@pytest.mark.parametrize("n", [1100, 5000, 16384, 40001])  # 16 and 32 steps of keys, and more
def test_many_rows_without_a_run(n):
    """Most rows padded or out of range, more of them than are looked through: the order counts the others alone, and the sums over
    blocks read nothing behind those."""
    from llattn_amd import embedding
    V, P, D = 50, 9, 24
    w, p = (t.requires_grad_() for t in _tables(V, P, D, F32))
    g = torch.Generator().manual_seed(n)
    ids = torch.where(torch.rand(n, generator=g) < 0.3, torch.randint(0, V, (n,), generator=g), 5)
    ids[::7], ids[3::11] = -1, V
    pos = torch.where(torch.rand(n, generator=g) < 0.6, torch.randint(0, P, (n,), generator=g), P + 3)
    ids, pos = ids.to(DEV), pos.to(DEV)
    _, i, q, cfg = embedding._forward(ids, w, p, pos, 1.0, 5)
    order = embedding._order(i, q, cfg, True, True)
    want = [int(((ids >= 0) & (ids < V) & (ids != 5)).sum()), int((pos < P).sum())]
    assert order[:8].view(torch.int32).tolist() == want
    dy = torch.randn(n, D, generator=g).to(DEV)
    for scale in (1.0, -2.5):
        dw, dp = torch.autograd.grad(_embed(ids, w, p, positions=pos, padding_idx=5, scale=scale), (w, p), dy)
        _check_sums(dw, ids, dy, V, scale, skip=5)
        _check_sums(dp, pos, dy, P, 1.0)


def test_rows_of_padding_alone():
    w, p = (t.requires_grad_() for t in _tables(3000, 700, 136, BF16))
    ids = torch.full((8, 700), 17, device=DEV)
    y = _embed(ids, w, p, positions=torch.full_like(ids, -1), padding_idx=17)
    dw, dp = torch.autograd.grad(y, (w, p), torch.ones_like(y))
    assert bool(y.isnan().all()) and bool((dw == 0).all()) and bool((dp == 0).all())


def test_the_most_rows():
    """2^31 - 1 rows, nearly all of one token, so that the rows, a wave's share of them and a key's run lie next to 2^31.  Whole numbers:
    column 0 counts the rows, and a sum of them takes two additions that are rounded (the blocks of 1024, below 2^21 of them, are
    exact); column 1 has single rows next to where the shares of 2^27 end, powers of two that add up exactly."""
    N = (1 << 31) - 1
    ids = torch.full((N,), 2, dtype=torch.int32, device=DEV)
    few = {0: 0, 77: 1, 1 << 30: 1, N - 1: 0}
    for at, token in few.items():
        ids[at] = token
    w = torch.tensor([[1.0, 2.0], [3.0, 4.0], [5.0, 6.0]], device=DEV, requires_grad=True)
    out = _embed(ids, w)
    assert out.shape == (N, 2) and all(torch.equal(out[at], w.detach()[t]) for at, t in few.items())
    assert torch.equal(out[N - 2], w.detach()[2]) and torch.equal(out[N // 3], w.detach()[2])
    dy = torch.zeros(N, 2, device=DEV)
    dy[:, 0] = 1.0
    edges = [k * (1 << 27) + d for k in (1, 5, 9, 13, 15) for d in (-1, 0)] + [1, N - 2]
    for k, at in enumerate(edges):
        dy[at, 1] = 2.0 ** k
    for at in few:
        dy[at, 1] = 7.0
    dw, = torch.autograd.grad(out, w, dy)
    assert dw[:2].tolist() == [[2.0, 14.0], [2.0, 14.0]]
    assert float(dw[2, 1]) == 2.0 ** len(edges) - 1 and abs(float(dw[2, 0]) - (N - 4)) <= 2 * U * N


@pytest.mark.parametrize("want", ["both", "tokens", "positions"])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("N,T", [(600, 300), (2800, 700), (40000, 2000)])
def test_nothing_is_read_that_was_not_written(N, T, given, want):
    """New buffers filled with ones in every bit (NaN, and -1 as an index; the indices and gradients lie within wider memory, so that
    even such an index reads what is there): the same bits."""
    V, P, D = 300, T + 5, 40
    g = torch.Generator().manual_seed(N)
    w, p = _tables(V, P, D, F32)
    w.requires_grad_(want != "positions")
    p.requires_grad_(want != "tokens")
    held = [torch.randint(-3, n, (N + 64,), generator=g).to(DEV) for n in (V + 3, P + 3)]
    ids, pos = (h[32:N + 32].view(-1, T) for h in held)
    dy = torch.randn(N + 64, D, generator=g).to(DEV)[32:N + 32].view(-1, T, D)

    def call():
        y = _embed(ids, w, p, positions=pos if given else None, padding_idx=7)
        return [y.detach(), *torch.autograd.grad(y, [t for t in (w, p) if t.requires_grad], dy)]
    clean = call()
    was = torch.utils.deterministic.fill_uninitialized_memory
    torch.use_deterministic_algorithms(True, warn_only=True)
    torch.utils.deterministic.fill_uninitialized_memory = True
    try:
        assert bool(torch.empty(1000, dtype=torch.uint8, device=DEV).eq(255).all())
        got = call()
    finally:
        torch.use_deterministic_algorithms(False)
        torch.utils.deterministic.fill_uninitialized_memory = was
    assert bool(torch.equal(got[0].nan_to_num(nan=7.0), clean[0].nan_to_num(nan=7.0)))
    assert all(torch.equal(a, b) and bool(a.isfinite().all()) for a, b in zip(got[1:], clean[1:]))
