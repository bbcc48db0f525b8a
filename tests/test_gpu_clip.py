"""The norm over a list of gradients and their clipping (``llattn_amd.grad_norm`` and its kin) on the GPU against plain
float64 ones.

Tolerances are counted: squares, their sum (n terms, each addition off by 2^-53 of it) and the coefficient are 64-bit, so a norm
is off by its rounding to fp32 (2^-24) and n 2^-53, and a clipped value by the rounding to its type (bf16: by way of fp32).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32 = torch.bfloat16, torch.float32
TINY = 2.0 ** -149


def _make(shapes, dtype=F32, seed=0, size=1.0):
    g = torch.Generator().manual_seed(seed)
    types = [dtype] * len(shapes) if isinstance(dtype, torch.dtype) else [dtype[i % len(dtype)] for i in range(len(shapes))]
    return [(torch.randn(s, generator=g) * size).to(t).to(DEV) for s, t in zip(shapes, types)]


def _norm(grads):
    return float(torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()) if grads else 0.0


def _check(got, grads, before, most):
    """`grads` (clipped) and the norm `got` from `before`."""
    want = _norm(before)
    n = sum(b.numel() for b in before)
    assert got.dtype is F32 and got.shape == () and abs(float(got) - want) <= (2.0 ** -24 + (n + 9) * 2.0 ** -53) * want + TINY
    c = min(1.0, most / (want + 1e-6))
    for a, b in zip(grads, before):
        assert a.dtype is b.dtype and a.shape == b.shape
        w = b.double() * c
        half = torch.finfo(a.dtype).eps / 2 + (2.0 ** -24 if a.dtype is BF16 else 0.0) + (n + 9) * 2.0 ** -53
        floor = 2.0 ** -134 if a.dtype is BF16 else TINY
        assert bool(((a.double() - w).abs() <= half * w.abs() + floor).all())


LISTS = {
    "one": [(1,)],
    "odd": [(3,), (7, 5), (1, 1), (129,), (333, 7), (2, 3, 5)],
    "empty among others": [(0,), (4, 0), (17,), (0, 3)],
    "chunks": [(16384,), (16385,), (16383,), (5, 16384), (3 * 16384 + 4,)],
    "many": [(1 + i % 37, 1 + i % 11) for i in range(300)],
    "a layer": [(384, 128), (384,), (64, 128), (64,), (128, 256), (128,)],
    "large": [(1500, 4000), (8,), (4001, 1003)],
    "over 2048 workgroups": [(2100, 16384), (999,)],
}


@pytest.mark.parametrize("dtype", [F32, BF16, (F32, BF16)], ids=["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("name", LISTS)
def test_norm_and_clipping(name, dtype):
    from llattn_amd import clip_grad_norm, grad_norm
    before = _make(LISTS[name], dtype)
    for share in (0.37, 2.0):
        most = share * _norm(before)
        grads = [g.clone() for g in before]
        _check(grad_norm(grads), grads, before, float("inf"))
        out = [torch.full_like(g, float("nan")) for g in grads]
        _check(clip_grad_norm(grads, most, out=out), out, before, most)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))  # the inputs stay
        _check(clip_grad_norm(grads, most), grads, before, most)
        assert all(torch.equal(a, b) for a, b in zip(grads, out))  # in place: the same bits
        if share > 1:
            assert all(torch.equal(a, b) for a, b in zip(grads, before))


@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e18, 1e30])
def test_squares_that_fp32_does_not_hold(size):
    from llattn_amd import clip_grad_norm
    before = _make([(100, 30), (7,)], size=size)
    grads = [g.clone() for g in before]
    _check(clip_grad_norm(grads, 1.0), grads, before, 1.0)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_norms_that_are_not_finite(bad, dtype):
    """As 0 times the values (infinity) or NaN times them."""
    from llattn_amd import clip_grad_norm, clip_grad_norm_
    before = _make([(50, 3), (20000,)], dtype)
    before[1][777] = bad
    grads = [g.clone() for g in before]
    norm = clip_grad_norm(grads, 1.0)
    for a, b in zip(grads, before):
        want = b * (float("nan") if bad != bad else 0.0)
        assert torch.equal(a.isnan(), want.isnan()) and bool((a.nan_to_num() == want.nan_to_num()).all())
    assert bool(norm.isnan()) if bad != bad else float(norm) == float("inf")
    params = [torch.nn.Parameter(torch.zeros_like(b)) for b in before]
    for p, b in zip(params, before):
        p.grad = b.clone()
    with pytest.raises(RuntimeError, match="norm is"):
        clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    assert all(torch.equal(p.grad.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0)) for p, b in zip(params, before))


def test_zero_gradients_and_a_zero_limit():
    from llattn_amd import clip_grad_norm
    z = [torch.zeros(10, device=DEV)]
    assert float(clip_grad_norm(z, 1.0)) == 0.0 and bool((z[0] == 0).all())
    g = _make([(10,)])
    clip_grad_norm(g, 0.0)
    assert bool((g[0] == 0).all())
    g = _make([(10,)])
    keep = g[0].clone()
    clip_grad_norm(g, float("inf"))
    assert torch.equal(g[0], keep)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("a,b", [(1, 1), (1, 0), (0, 3), (5, 2)])
def test_views_at_any_element(dtype, a, b):
    """Gradients and outputs that begin at any element of a flat buffer; what lies around them stays."""
    from llattn_amd import clip_grad_norm
    n, m = 16384 * 2 + 77, 1001
    flat = _make([(a + n + 3 + m + 9,)], dtype)[0]
    out = torch.full((b + n + m + 20,), 9.0, dtype=dtype, device=DEV)
    g = [flat[a:a + n], flat[a + n + 3:a + n + 3 + m]]
    o = [out[b:b + n], out[b + n + 1:b + n + 1 + m]]
    _check(clip_grad_norm(g, 1.0, out=o), o, g, 1.0)
    assert bool((out[:b] == 9).all()) and bool((out[b + n] == 9).all()) and bool((out[b + n + 1 + m:] == 9).all())
    before = flat.clone()
    clip_grad_norm(g, 1.0)
    assert torch.equal(g[0], o[0]) and torch.equal(g[1], o[1])
    assert torch.equal(flat[:a], before[:a]) and torch.equal(flat[a + n:a + n + 3], before[a + n:a + n + 3])


def test_other_orders_and_strides():
    from llattn_amd import clip_grad_norm, grad_norm
    base = _make([(40, 30), (6, 50), (4, 5, 6)])
    before = [base[0].t(), base[1][:, ::3], base[2].permute(2, 0, 1)]
    copies = [base[0].clone().t(), base[1].clone()[:, ::3], base[2].clone().permute(2, 0, 1)]
    _check(clip_grad_norm(copies, 0.5), copies, before, 0.5)
    out = [torch.empty(30, 40, device=DEV), torch.empty(50, 6, device=DEV).t()[:, :17], torch.empty(6, 4, 5, device=DEV)]
    _check(clip_grad_norm(before, 0.5, out=out), out, before, 0.5)
    wide = torch.full((6, 50), 3.0, device=DEV)
    held = wide.clone()
    clip_grad_norm([wide[:, ::3]], 1.0)
    assert torch.equal(wide[:, 1::3], held[:, 1::3]) and torch.equal(wide[:, 2::3], held[:, 2::3])
    e = torch.ones(3, device=DEV).expand(5, 3)
    assert abs(float(grad_norm([e])) - 15 ** 0.5) < 1e-6
    with pytest.raises(ValueError, match="several places"):
        clip_grad_norm([e], 1.0)


def test_tensors_that_overlap_are_refused():
    from llattn_amd import clip_grad_norm, grad_norm
    g = _make([(100,)])[0]
    keep = g.clone()
    for lists, out in [(([g, g]), None), ([g[:60], g[50:]], None), ([g[:50], g[50:]], [g[50:], g[:50]]),
                       ([g[:50]], [g[10:60]]), ([g, keep], [keep, g])]:
        with pytest.raises(ValueError, match="overlap"):
            clip_grad_norm(lists, 0.1, out=out)
    assert torch.equal(g, keep)
    # read twice, written apart: each counts
    out = [torch.empty_like(g), torch.empty_like(g)]
    assert abs(float(clip_grad_norm([g, g], 1.0, out=out)) - 2 ** 0.5 * _norm([g])) < 1e-5 and torch.equal(*out)
    assert float(grad_norm([g, g])) > float(grad_norm([g]))
    clip_grad_norm([g[:50], g[50:]], 0.1)  # side by side


def test_parameters():
    from llattn_amd import clip_grad_norm_, clip_grads_with_norm_
    m = torch.nn.Sequential(torch.nn.Linear(30, 50), torch.nn.Linear(50, 7)).to(DEV)
    m[0].bias.requires_grad_(False)
    x = torch.randn(9, 30, generator=torch.Generator().manual_seed(0)).to(DEV)
    m(x).square().sum().backward()
    before = [p.grad.clone() for p in m.parameters() if p.grad is not None]
    versions = [p.grad._version for p in m.parameters() if p.grad is not None]
    norm = clip_grad_norm_(m.parameters(), 0.7)
    after = [p.grad for p in m.parameters() if p.grad is not None]
    _check(norm, after, before, 0.7)
    assert all(g._version > v for g, v in zip(after, versions))
    for p, b in zip([p for p in m.parameters() if p.grad is not None], before):
        p.grad = b.clone()
    want = torch.nn.utils.clip_grad_norm_(m.parameters(), 0.7)
    assert torch.allclose(want, norm, rtol=1e-6)
    assert all(torch.allclose(p, q, rtol=1e-6, atol=0) for p, q in zip([p.grad for p in m.parameters() if p.grad is not None], after))
    for p, b in zip([p for p in m.parameters() if p.grad is not None], before):
        p.grad = b.clone()
    clip_grads_with_norm_(m.parameters(), 0.7, norm)
    # by the norm in fp32: 2^-24 further off
    for p, a in zip([p.grad for p in m.parameters() if p.grad is not None], after):
        assert bool(((p - a).abs() <= 3 * 2.0 ** -24 * a.abs()).all())
    one = torch.nn.Parameter(torch.zeros(3, device=DEV))
    assert float(clip_grad_norm_([one], 1.0)) == 0.0  # no gradient at all
    one.grad = torch.tensor([3.0, 4.0, 0.0], device=DEV)
    assert float(clip_grad_norm_(one, 1.0, error_if_nonfinite=True)) == 5.0


def test_captured_and_replayed():
    from llattn_amd import clip_grad_norm
    shapes = LISTS["many"] + [(2100, 16384)]
    grads = _make(shapes)
    with torch.cuda.stream(torch.cuda.Stream()):
        clip_grad_norm([g.clone() for g in grads], 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm(grads, 1.0)
    for seed in range(3):
        new = _make(shapes, seed=seed, size=1e-6 if seed == 1 else 1.0)
        for g, n in zip(grads, new):
            g.copy_(n)
        want = clip_grad_norm(new, 1.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(grads, new))


def test_two_streams_at_once():
    from llattn_amd import clip_grad_norm
    lists = [_make([(500, 900), (31,)], seed=s) for s in (1, 2)]
    want = [[g.clone() for g in one] for one in lists]
    norms = [clip_grad_norm(w, 1.0) for w in want]
    torch.cuda.synchronize()
    got = []
    for one in lists:
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(clip_grad_norm(one, 1.0))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, norms))
    assert all(torch.equal(a, b) for x, y in zip(lists, want) for a, b in zip(x, y))


def test_a_tensor_past_32_bit_offsets():
    from llattn_amd import clip_grad_norm
    n = (1 << 31) + 12345
    g = torch.zeros(n, dtype=BF16, device=DEV)
    g[0], g[-1], g[n // 2] = 3.0, 4.0, 12.0
    assert float(clip_grad_norm([g], 6.5)) == 13.0
    assert [float(g[i]) for i in (0, n // 2, n - 1)] == [1.5, 6.0, 2.0] and int((g != 0).sum()) == 3


def test_a_given_norm_within_a_gradient_is_refused():
    from llattn_amd import clip_grads_with_norm_
    p = torch.nn.Parameter(torch.ones(8, device=DEV))
    p.grad = torch.ones(8, device=DEV)
    with pytest.raises(ValueError, match="holds the norm"):
        clip_grads_with_norm_([p], 1.0, p.grad[3])
    assert bool((p.grad == 1).all())


@pytest.mark.parametrize("where", ["grad_norm", "gradients", "out"])
def test_sparse_tensors_are_refused(where):
    from llattn_amd import clip_grad_norm, grad_norm
    g = torch.eye(4, device=DEV)
    for t in (g.to_sparse(), g.to_sparse_csr()):
        with pytest.raises(ValueError, match="dense"):
            if where == "grad_norm":
                grad_norm([g, t])
            elif where == "gradients":
                clip_grad_norm([t], 1.0)
            else:
                clip_grad_norm([g], 1.0, out=[t])


def test_strided_tensors_that_overlap_are_refused():
    """As contiguous ones are; interleaved slices of one buffer are not refused, and each is scaled once."""
    from llattn_amd import clip_grad_norm
    a = _make([(60, 80)])[0]
    keep = a.clone()
    even, odd = a[:, ::2], a[:, 1::2]
    for g, out in (([even, even], None), ([even, a], None), ([a[:, :50], a[:, 40:]], None), ([even, odd], [odd, even]),
                   ([a[:, :60]], [a[:, :60].t()]), ([even], [a[:, 1:41]])):
        with pytest.raises(ValueError, match="overlap|shapes"):
            clip_grad_norm(g, 0.1, out=out)
    assert torch.equal(a, keep)
    _check(clip_grad_norm([even, odd], 0.5), [even, odd], [keep[:, ::2], keep[:, 1::2]], 0.5)
    a.copy_(keep)
    _check(clip_grad_norm([even, odd], 0.5, out=[even, odd]), [even, odd], [keep[:, ::2], keep[:, 1::2]], 0.5)
