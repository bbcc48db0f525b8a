"""CPU tests of the language model's operators: the C interface (include/llattn_lm.h), and what is refused before anything
is launched."""
import ctypes
import re
import subprocess
from array import array

import pytest
import torch

from conftest import REPO
from llattn_amd import _lib as L
from llattn_amd import clip, clip_grad_norm, clip_grad_norm_, clip_grads_with_norm_, embed, gated_feed_forward, grad_norm
from llattn_amd.lm import FeedForward, GatedFeedForward, build_model, train_step

BF16 = torch.bfloat16
AT = 1 << 20  # a pointer that nothing reads


def test_header_matches_the_binding(tmp_path):
    text = (REPO / "include" / "llattn_lm.h").read_text()
    names = set(re.findall(r"^\s*(?:int32_t|size_t)\s+(llattn_\w+)\s*\(", text, re.M))
    assert names == set(L.LM_SIGNATURES) and all(hasattr(L.load(), n) for n in names)
    structs = {"llattn_embed_cfg": L.LlattnEmbedCfg, "llattn_gated_cfg": L.LlattnGatedCfg,
               "llattn_gated_weights": L.LlattnGatedWeights, "llattn_gated_grads": L.LlattnGatedGrads}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "llattn_lm.h"', "int main(void) {"]
    for c, t in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in t._fields_]
    src = tmp_path / "l.c"
    src.write_text("\n".join([*lines, "return 0; }"]))
    subprocess.run(["gcc", f"-I{REPO / 'include'}", str(src), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for t in structs.values():
        want.append(ctypes.sizeof(t))
        want += [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want


# ---------------------------------------------------------------------------
# token and position rows
# ---------------------------------------------------------------------------

def _cfg(rows=6, T=3, V=10, P=4, D=8, dtype=0, index_bytes=8, padding=-1, scale=1.0):
    return L.LlattnEmbedCfg(rows, T, V, P, D, dtype, index_bytes, padding, scale)


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(rows=1 << 31), dict(V=0), dict(V=(1 << 22) + 1), dict(P=-1), dict(P=(1 << 22) + 1),
                                dict(D=0), dict(D=(1 << 20) + 1), dict(T=0), dict(T=5), dict(rows=7), dict(dtype=2),
                                dict(index_bytes=2), dict(padding=10), dict(padding=-2)], ids=str)
def test_embed_sizes_refused(kw):
    for which in (L.EMBED_ORDER, L.EMBED_BACKWARD):
        assert L.load().llattn_embed_bytes(ctypes.byref(_cfg(**kw)), 0, which) == 0 and L.load().llattn_last_error()


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan")])
def test_scales_that_are_not_finite_are_refused(scale):
    """They would reach the rows of the gradient that no token names, which are zero."""
    assert L.load().llattn_embed_bytes(ctypes.byref(_cfg(scale=scale)), 0, 0) == 0 and b"finite" in L.load().llattn_last_error()
    assert L.load().llattn_embed_fwd(ctypes.byref(_cfg(scale=scale)), AT, None, AT, 8, AT, 8, AT, None) == 1
    ids, w = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(5, 4)
    for s in (scale, 3.5e38, 10 ** 400):  # infinite in fp32, or in 64 bits
        with pytest.raises(ValueError, match="finite"):
            embed(ids, w, scale=s)
    with pytest.raises(RuntimeError, match="MI355X"):
        embed(ids, w, scale=3.4e38)


def test_embed_sizes_taken():
    def n(cfg, has_pos):
        return tuple(L.load().llattn_embed_bytes(ctypes.byref(cfg), has_pos, k) for k in (L.EMBED_ORDER, L.EMBED_BACKWARD))
    assert n(_cfg(), 0) == n(_cfg(rows=0), 0) == (1, 1)  # none for few tokens
    assert n(_cfg(T=9, rows=7), 1) == n(_cfg(T=0, P=0), 0) == (1, 1)
    order, trees = n(_cfg(rows=32768, T=2048, V=32000, P=2048, D=1408), 0)
    assert 32768 * 12 + 32000 * 8 <= order < 32768 * 12 + 32000 * 8 + 4096
    assert n(_cfg(rows=32768, T=2048, V=32000, P=2048, D=1408), 1)[0] > order + 32768 * 12
    assert 2 * 32768 // 32 * 1408 * 4 <= trees < 2 * 32768 * 1408 * 4 // 31 + 4096  # sums of 32 rows and of 1024, two tables
    assert n(_cfg(rows=21, V=1 << 22), 0)[1] == 1  # too few for sums of 32
    assert L.load().llattn_embed_bytes(ctypes.byref(_cfg()), 0, 2) == 0


@pytest.mark.parametrize("kw,code", [(dict(ids=None), 3), (dict(W=None), 3), (dict(out=None), 3), (dict(Pos=None), 3), (dict(ids=AT + 4), 3),
                                     (dict(W=AT + 2), 3), (dict(out=AT + 1), 3), (dict(ldw=7), 3), (dict(ldp=7), 3)], ids=str)
def test_embed_forward_refused(kw, code):
    a = dict(ids=AT, pos=None, W=AT, ldw=8, Pos=AT, ldp=8, out=AT) | kw
    assert L.load().llattn_embed_fwd(ctypes.byref(_cfg()), *a.values(), None) == code


@pytest.mark.parametrize("kw,code", [(dict(ids=None), 3), (dict(ids=AT + 4), 3), (dict(positions=1), 3), (dict(pos=AT + 4), 3),
                                     (dict(order=None), 5), (dict(order=AT + 8), 5), (dict(n=100), 5)], ids=str)
def test_embed_order_refused(kw, code):
    a = dict(ids=AT, pos=None, tokens=1, positions=0, order=AT, n=1 << 20) | kw
    assert L.load().llattn_embed_order(ctypes.byref(_cfg(rows=1200)), *a.values(), None) == code


def test_no_order_of_few_tokens():
    assert L.load().llattn_embed_order(ctypes.byref(_cfg()), AT, None, 1, 0, None, 0, None) == 0


@pytest.mark.parametrize("kw,code", [(dict(ids=None), 3), (dict(dout=None), 3), (dict(dW=AT + 2), 3), (dict(order=None), 3),
                                     (dict(order=AT + 8), 3), (dict(dW=None, pos=AT, order=None), 3), (dict(ws=None), 5),
                                     (dict(ws=AT + 8), 5), (dict(n=100), 5), (dict(dW=None, order=None, ws=None), 5)], ids=str)
def test_embed_backward_refused(kw, code):
    lib = L.load()
    cfg = _cfg(rows=1200)  # (few tokens take no order and no workspace)
    a = dict(ids=AT, pos=None, order=AT, dout=AT, dW=AT, dPos=AT, ws=AT, n=1 << 20) | kw
    assert lib.llattn_embed_bwd(ctypes.byref(cfg), *a.values(), None) == code
    assert lib.llattn_embed_bwd(ctypes.byref(_cfg(rows=1200, P=0)), *a.values(), None) == 1


def test_embed_refusals():
    ids, w, p = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(5, 4), torch.zeros(3, 4)
    for args, kw, msg in [((ids, w[0]), {}, "matrix"), ((ids, w[:0]), {}, "matrix"), ((ids.float(), w), {}, "integers"),
                          ((ids.bool(), w), {}, "integers"), ((ids, w.double()), {}, "float32"), ((ids, w, p[:, :2]), {}, "match"),
                          ((ids, w, p[0]), {}, "match"), ((ids, w, p.to(BF16)), {}, "match"), ((ids, w, p[:2]), {}, "positions"),
                          ((ids, w), dict(positions=ids), "without"), ((ids, w, p), dict(positions=ids[:1]), "positions"),
                          ((ids, w, p), dict(positions=ids.float()), "integers"), ((ids, w), dict(scale="2"), "number"),
                          ((ids, w), dict(scale=torch.ones(())), "number"), ((ids, w), dict(padding_idx=5), "padding_idx"),
                          ((ids, w), dict(padding_idx=-6), "padding_idx"), ((ids, torch.zeros((1 << 22) + 1, 1)), {}, "at most")]:
        with pytest.raises(ValueError, match=msg):
            embed(*args, **kw)
    with pytest.raises(RuntimeError, match="MI355X"):
        embed(ids, w, p)


# ---------------------------------------------------------------------------
# the norm over gradients, and clipping
# ---------------------------------------------------------------------------

def _list(*values, code="Q"):
    a = array(code, values)
    return a, clip._at(a)


def test_grad_norm_sizes():
    lib = L.load()

    def size(*n):
        keep = array("q", n)
        return lib.llattn_grad_norm_bytes(len(n), clip._at(keep))
    assert size() == 8 and size(0, 0) == 8 and size(1) == 8 and size(16384) == 8 and size(16385) == 16 and size(1, 1) == 16
    assert size(1 << 30) == 8 * 2048 and size(*[1] * 129) == 8 * 129
    assert size(-1) == 0 and size(1 << 45) == 0 and lib.llattn_grad_norm_bytes(-1, None) == 0 and lib.llattn_grad_norm_bytes(1, None) == 0


def _clip_call(g=(AT,), out=None, numel=(10,), dtype=(0,), norm_in=None, norm=AT, ws=AT, n=1 << 20):
    keep = [_list(*g), None if out is None else _list(*out), _list(*numel, code="q"), _list(*dtype, code="i")]
    p = [k and k[1] for k in keep]
    return L.load().llattn_clip_grads(len(g), p[0], p[1], p[2], p[3], 1.0, norm_in, norm, ws, n, None)


@pytest.mark.parametrize("kw,code", [(dict(g=(0,)), 3), (dict(g=(AT + 2,)), 3), (dict(out=(0,)), 3), (dict(out=(AT + 4002,)), 3),
                                     (dict(dtype=(2,)), 2), (dict(numel=(-1,)), 1), (dict(norm=None), 3), (dict(norm_in=AT), 3),
                                     (dict(norm=None, norm_in=AT), 3), (dict(norm=None, norm_in=AT + 36), 3),
                                     (dict(norm=None, norm_in=AT + 400, out=(AT + 400,)), 3),
                                     (dict(ws=None), 5), (dict(ws=AT + 4), 5), (dict(n=7), 5),
                                     (dict(g=(AT, AT), numel=(10, 10), dtype=(0, 0)), 3),
                                     (dict(g=(AT, AT + 36), numel=(10, 10), dtype=(0, 0)), 3),
                                     (dict(out=(AT + 36,)), 3), (dict(out=(AT - 36,)), 3),
                                     (dict(g=(AT, AT + 400), out=(AT + 400, AT), numel=(10, 10), dtype=(0, 0)), 3),
                                     (dict(g=(AT, AT + 400), out=(AT, AT + 20), numel=(10, 10), dtype=(0, 0)), 3),
                                     (dict(g=(AT, AT + 400), out=(AT + 800, AT + 820), numel=(10, 10), dtype=(1, 1)), 5)], ids=str)
def test_clip_calls_refused(kw, code):
    if code == 5 and "ws" not in kw and "n" not in kw:
        kw = kw | dict(n=0)  # side by side: what is refused is the workspace
    assert _clip_call(**kw) == code and L.load().llattn_last_error()


def test_clip_refusals():
    g = torch.ones(3)
    for f, msg in [(lambda: clip_grad_norm([g], -1.0), "max_norm"), (lambda: clip_grad_norm([g], float("nan")), "max_norm"),
                   (lambda: clip_grad_norm([g], g[0]), "max_norm"), (lambda: clip_grad_norm([g], 1.0, out=[]), "outputs"),
                   (lambda: clip_grad_norm([g.half()], 1.0), "fp32 or bf16"), (lambda: grad_norm([g.long()]), "fp32 or bf16"),
                   (lambda: grad_norm([g.to_sparse()]), "dense"),
                   (lambda: clip_grad_norm([g], 1.0, out=[torch.ones(3, requires_grad=True)]), "leaves"),
                   (lambda: clip_grad_norm_([], 1.0, norm_type=1.0), "2-norm"),
                   (lambda: clip_grad_norm_([], -1.0), "max_norm")]:
        with pytest.raises(ValueError, match=msg):
            f()
    p = torch.nn.Parameter(g)
    p.grad = g
    for f in (lambda: grad_norm([g]), lambda: clip_grad_norm([g], 1.0), lambda: clip_grad_norm_(p, 1.0),
              lambda: clip_grads_with_norm_([p], 1.0, torch.ones(()))):
        with pytest.raises(RuntimeError, match="MI355X"):
            f()


def test_nothing_to_clip():
    assert float(grad_norm([])) == 0.0 and float(clip_grad_norm([], 1.0)) == 0.0
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0
    clip_grads_with_norm_([], 1.0, torch.ones(()))


def test_a_given_norm_beside_the_gradients():
    # right before and right behind what is written: what is refused is the output within the gradient
    for norm in (AT + 16, AT + 60):
        assert _clip_call(norm=None, norm_in=norm, out=(AT + 20,)) == 3 and b"output 0 overlaps" in L.load().llattn_last_error()


@pytest.mark.parametrize("which", ["embed", "gated", "norm", "clip"])
def test_forward_mode_tangents_are_refused(which):
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        t = fwd.make_dual(torch.ones(4, 3), torch.ones(4, 3))
        call = {"embed": lambda: embed(torch.zeros(2, dtype=torch.int64), t), "gated": lambda: gated_feed_forward(t, *_layers(3, 5, 2)),
                "norm": lambda: grad_norm([t]), "clip": lambda: clip_grad_norm([t], 1.0)}[which]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call()


def test_flat_views():
    """Tensors in one stretch of memory, whatever the order of their axes, are taken as they lie."""
    x = torch.arange(24.0).reshape(2, 3, 4)
    for t in (x, x.permute(2, 0, 1), x.transpose(0, 1), x[0].t()):
        f = clip._flat(t)
        assert f.is_contiguous() and f.data_ptr() == t.data_ptr() and f.numel() == t.numel()
    for t in (x[:, :, ::2], x[:, :2], torch.ones(3).expand(4, 3)):
        assert clip._flat(t) is None


def _bytes(t):
    """The bytes of a tensor's elements, one by one."""
    at = {t.data_ptr()}
    for n, s in zip(t.shape, t.stride()):
        at = {v + k * s * t.element_size() for v in at for k in range(n)}
    return {v + k for v in at for k in range(t.element_size())}


def test_tensors_that_share_memory():
    """Strided pieces of one buffer, of equal and of different types, against their bytes one by one."""
    g = torch.Generator().manual_seed(0)
    draw = lambda lo, hi: int(torch.randint(lo, hi, (), generator=g))  # noqa: E731
    flat, found = torch.zeros(400), [0, 0]

    def piece():
        base = (flat, flat.view(BF16))[draw(0, 2)]
        shape = [draw(1, 5) for _ in range(draw(1, 4))]
        return base.as_strided(shape, [draw(0, 14) for _ in shape], draw(0, 60))
    for _ in range(3000):
        a, b = piece(), piece()
        want = bool(_bytes(a) & _bytes(b))
        assert clip._meet(a, b) == want == clip._meet(b, a), (a.shape, a.stride(), b.shape, b.stride())
        found[want] += 1
    assert min(found) > 300
    big = torch.empty(1 << 13, 1 << 12, device="meta").as_strided((1 << 12, 1 << 11), (1 << 13, 2))
    assert clip._meet(big, big)


def test_strided_gradients_that_overlap_are_refused():
    a, b = torch.ones(6, 8), torch.ones(8, 6)
    even, odd = a[:, ::2], a[:, 1::2]
    for g, out in (([even, odd], None), ([a[::2], a[1::2]], None), ([a[:, :4], a[:, 4:]], None), ([a[:3, ::3], a[3:, ::2]], None), ([even], [odd]), ([even], [even]),
                   ([even, odd], [even, odd]), ([even], [b[:6, :4]]), ([even, even], [b[:6, :4], b.new_zeros(6, 4)]), ([a.t()], [b]),
                   ([a[:, ::2], a[:0]], None)):
        clip._refuse_overlap("clip", g, out)
    for g, out, what in (([even, even], None, "overlap"), ([even, a], None, "overlap"), ([a[:, ::2], a[:, ::3]], None, "overlap"),
                         ([a[:, :5], a[:, 4:]], None, "overlap"), ([even, odd], [odd, even], "overlaps gradient"),
                         ([a[:, :4]], [a[:, 1:5]], "output 0 overlaps gradient 0"), ([a[:6, :6]], [a[:6, :6].t()], "output 0 overlaps gradient 0"),
                         ([even, odd], [b[:6, :4], b[1:7, :4]], "written"), ([a, b.t()], [torch.ones(6, 8), a], "output 1 overlaps gradient 0"),
                         ([a[:, ::2], a.view(BF16)[:, 5:9]], None, "overlap")):
        with pytest.raises(ValueError, match=what):
            clip._refuse_overlap("clip", g, out)


# ---------------------------------------------------------------------------
# gated feed-forward
# ---------------------------------------------------------------------------

def _layers(D, F, Do, bias=True, dtype=torch.float32):
    return [torch.nn.Linear(i, o, bias=bias).to(dtype) for i, o in ((D, F), (D, F), (F, Do))]


def _gated_cfg(rows=10, D=16, F=24, D_out=8, act=0, dw=0, dw2=1):
    return L.LlattnGatedCfg(rows, D, F, D_out, act, dw, dw2)


@pytest.mark.parametrize("kw", [dict(rows=0), dict(rows=1 << 23), dict(D=0), dict(D=12), dict(F=4), dict(D_out=-8), dict(F=1 << 22), dict(act=2),
                                dict(dw=2), dict(dw2=-1)], ids=str)
def test_gated_sizes_refused(kw):
    for which in range(4):
        assert L.load().llattn_gated_bytes(ctypes.byref(_gated_cfg(**kw)), which) == 0 and L.load().llattn_last_error()
        assert L.load().llattn_gated_bytes(ctypes.byref(_gated_cfg()), which) > 0
    # enough tiles: no parts of y, and no workspace of a forward that keeps h
    assert L.load().llattn_gated_bytes(ctypes.byref(_gated_cfg(rows=4096, D_out=4096)), L.GATED_FORWARD) == 1
    for which in (-1, 4):
        assert L.load().llattn_gated_bytes(ctypes.byref(_gated_cfg()), which) == 0


@pytest.mark.parametrize("kept", [AT, None])
@pytest.mark.parametrize("kw,code", [(dict(x=None), 3), (dict(x=AT + 8), 3), (dict(ldx=8), 3), (dict(ldx=20), 3), (dict(ldx=1 << 23), 3), (dict(W1=None), 3),
                                     (dict(W3=AT + 2), 3), (dict(b1=AT + 4), 3), (dict(y=None), 3), (dict(y=AT + 8), 3), (dict(kept=AT + 8), 3),
                                     (dict(ws=None), 5), (dict(ws=AT + 8), 5), (dict(n=100), 5)], ids=str)
def test_gated_forward_refused(kw, code, kept):
    lib, cfg = L.load(), _gated_cfg()
    a = dict(x=AT, ldx=16, W1=AT, W3=AT, W2=AT, b1=None, kept=kept, y=AT, ws=AT, n=1 << 20) | kw
    w = L.LlattnGatedWeights(a["W1"], a["W3"], a["W2"], a["b1"], None, None)
    assert lib.llattn_gated_fwd(ctypes.byref(cfg), a["x"], a["ldx"], ctypes.byref(w), a["kept"], a["y"], a["ws"], a["n"], None) == code


@pytest.mark.parametrize("kw,code", [(dict(x=None), 3), (dict(kept=None), 3), (dict(dy=None), 3), (dict(kept=AT + 8), 3), (dict(dx=AT + 8), 3),
                                     (dict(dW1=None), 3), (dict(dW3=None), 3), (dict(ws=None), 5), (dict(n=100), 5)], ids=str)
def test_gated_backward_refused(kw, code):
    lib, cfg = L.load(), _gated_cfg()
    a = dict(x=AT, kept=AT, dy=AT, dx=AT, dW1=AT, dW3=AT, dW2=AT, ws=AT, n=lib.llattn_gated_bytes(ctypes.byref(cfg), L.GATED_BACKWARD)) | kw
    w = L.LlattnGatedWeights(AT, AT, AT, None, None, None)
    g = L.LlattnGatedGrads(a["dx"], a["dW1"], a["dW3"], a["dW2"], None, None, None)
    assert lib.llattn_gated_bwd(ctypes.byref(cfg), a["x"], 16, ctypes.byref(w), a["kept"], a["dy"], ctypes.byref(g), a["ws"],
                                a["n"], None) == code


def test_gated_refusals():
    x, ls = torch.zeros(2, 3), _layers(3, 5, 2)
    for args, kw, msg in [((x, *ls), dict(act="relu"), "act"), ((x[:, :2], *ls), {}, "match"), ((x, ls[0], ls[2], ls[2]), {}, "match"),
                          ((x, ls[0], ls[1], ls[0]), {}, "match"), ((torch.zeros(()), *ls), {}, "match"), ((x.double(), *ls), {}, "float32"),
                          ((x, ls[0], ls[1].half(), ls[2]), {}, "float32")]:
        with pytest.raises(ValueError, match=msg):
            gated_feed_forward(*args, **kw)
    bad = _layers(3, 5, 2)
    bad[0].bias = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="bias"):
        gated_feed_forward(x, *bad)
    with pytest.raises(RuntimeError, match="MI355X"):
        gated_feed_forward(x, *_layers(3, 5, 2))


@pytest.mark.parametrize("transposed", [False, True])
def test_weights_are_cast_on_their_own_device(transposed, monkeypatch):
    """The launch that rounds fp32 weights stands under their device, whichever one is current: a stream of another device's would
    be refused, and the default streams, which have no handle, are not told apart."""
    import contextlib
    from llattn_amd import linear, ops
    inside, calls = [], []

    @contextlib.contextmanager
    def on_device(device):
        inside.append(device)
        yield
        inside.pop()
    monkeypatch.setattr(L, "on_device", on_device)
    monkeypatch.setattr(L, "require_gpu", lambda *t: None)
    monkeypatch.setattr(L, "stream_ptr", lambda device: None)
    monkeypatch.setattr(ops, "_call", lambda name, *a, **k: calls.append((name, list(inside))))
    ws = [torch.zeros(8, 16) for _ in range(2 * linear.MAX_SEGS + 1)]
    linear.pack_params([([w], BF16, transposed) for w in ws])
    name = "llattn_cast_transposed" if transposed else "llattn_cast"
    assert calls == [(name, [torch.device("cpu")])] * 3 and not inside


def test_which_tiles_the_larger_cases_take(tmp_path):
    """The sizes that tests/test_gpu_gated.py keeps for the kernels of larger tiles do take those, by the library's own choice."""
    from llattn_amd import _build
    from test_gpu_gated import CASES, LARGE
    up = lambda n: -(-n // 8) * 8  # noqa: E731
    lines = ['#include "llattn_gated.hip"', "namespace llattn { namespace {"]
    taken = set()
    for k, (case, kinds) in enumerate([*LARGE, *((c, {}) for c in CASES)]):
        N, D, F, Do = case[0], *map(up, case[1:4])
        lines.append(f"constexpr llattn_gated_cfg c{k}{{{N}, {D}, {F}, {Do}, 0, 0, 0}};")
        for product in ("gate", "out", "dgate", "dx", "dw", "dw2"):
            kind, *split = kinds.get(product, "SQUARE").split()
            way = "OF_FORWARD" if product in ("gate", "out") else "OF_BACKWARD"
            at = f"tilings_of(&c{k}, {way}).{product}"
            lines.append(f"static_assert({at}.kind == {kind}, \"{case} {product}\");")
            if kind != "SQUARE":
                lines.append(f"static_assert(({at}.splits > 1) == {str(bool(split)).lower()}, \"{case} {product}\");")
                taken.add((product, kind, bool(split)))
    assert taken == {("gate", "BIG", False), ("dgate", "BIG", False),
                     *((p, k, s) for p in ("out", "dx", "dw", "dw2") for k in ("BIG", "WIDE") for s in (False, True))}
    src = tmp_path / "tilings.hip"
    src.write_text("\n".join([*lines, "} }"]))
    run = subprocess.run([_build.hipcc(), f"--offload-arch={_build.ARCH}", "--offload-host-only", "-fsyntax-only", "-std=c++17",
                          f"-I{_build.INCLUDE_DIR}", f"-I{_build.SRC_DIR}", str(src)], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]


# ---------------------------------------------------------------------------
# the model
# ---------------------------------------------------------------------------

def _model(**kw):
    return build_model(vocab_size=40, max_seq_len=16, d_model=16, n_heads=2, n_layers=2, d_ff=24, latent_d_model=8, latent_heads=1, **kw)


def test_models_with_a_gate():
    m = _model()
    assert type(m.blocks[0].ff) is FeedForward and m.config.ffn == "gelu"
    for name, act in (("swiglu", "silu"), ("geglu", "gelu")):
        m = _model(ffn=name)
        ff = m.blocks[1].ff
        assert type(ff) is GatedFeedForward and ff.act == act and ff.w3.weight.shape == (24, 16)
        assert float(ff.w2.weight.std()) < 0.8 * float(ff.w3.weight.std())  # scaled as an output projection
        x = torch.randn(3, 16)
        f = torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu
        assert torch.equal(ff(x), ff.w2(f(ff.w1(x)) * ff.w3(x)))  # on the CPU: torch's own
    with pytest.raises(ValueError, match="ffn"):
        _model(ffn="relu")


class _Adapter(torch.nn.Linear):
    """A linear layer that adds something of its own."""

    def forward(self, x):
        return super().forward(x) + 1


def _stood_around(ff, name):
    """The ways in which a layer of a feed-forward comes to be more than its weight and bias: (what it is, undo)."""
    m = getattr(ff, name)

    def own(_):
        a = _Adapter(m.in_features, m.out_features).to(m.weight)
        a.load_state_dict(m.state_dict())
        setattr(ff, name, a)
        return lambda: setattr(ff, name, m)

    def wrapped(_):
        setattr(ff, name, torch.nn.Sequential(m))
        return lambda: setattr(ff, name, m)

    def replaced(_):
        m.forward = lambda x: torch.nn.functional.linear(x, m.weight, m.bias) + 1
        return lambda: delattr(m, "forward")

    def weight_made_before(_):
        torch.nn.utils.weight_norm(m)
        return lambda: torch.nn.utils.remove_weight_norm(m)
    hooks = [lambda _: m.register_forward_hook(lambda *a: a[2] + 1).remove, lambda _: m.register_forward_pre_hook(lambda *a: None).remove,
             lambda _: m.register_full_backward_hook(lambda *a: None).remove, lambda _: m.register_full_backward_pre_hook(lambda *a: None).remove,
             lambda _: torch.nn.modules.module.register_module_forward_hook(lambda *a: None).remove]
    return [own, wrapped, replaced, weight_made_before, *hooks]


@pytest.mark.parametrize("name", ["w1", "w3", "w2"])
def test_projections_that_the_gated_feed_forward_leaves_alone(name):
    """Layers with a forward of their own, replaced ones and hooked ones are called, not read."""
    ff, x = _model(ffn="swiglu").blocks[0].ff.bfloat16(), torch.zeros(1, dtype=BF16)
    assert ff._fusable(x)
    for way in _stood_around(ff, name):
        undo = way(ff)
        assert not ff._fusable(x)
        undo()
        assert ff._fusable(x)
    torch.nn.utils.parametrize.register_parametrization(getattr(ff, name), "weight", torch.nn.Identity())
    assert ff._fusable(x)  # its weight is what a call reads


def test_dropout_of_a_gated_feed_forward():
    ff, x = _model(ffn="geglu").blocks[0].ff.bfloat16(), torch.zeros(1, dtype=BF16)
    ff.dropout.p = 0.5
    assert not ff._fusable(x) and ff.eval()._fusable(x)
    ff.dropout.train()  # alone: as dropout is switched on to sample from a model
    assert not ff._fusable(x)
    ff.dropout = torch.nn.Identity()
    assert not ff._fusable(x)


def test_lookups_on_the_cpu_are_torchs():
    m = _model()
    ids = torch.zeros(2, 5, dtype=torch.int64)
    assert not m._fused_embeddings(ids) and not m.config.fused_embeddings
    m = _model(fused_embeddings=True)
    assert m.fuse_embeddings and not m._fused_embeddings(ids)


@pytest.mark.parametrize("fused", [False, True])
def test_the_training_step_clips_as_asked(fused, monkeypatch):
    from llattn_amd import lm
    calls = []
    monkeypatch.setattr(lm, "clip_grad_norm_", lambda p, most: calls.append(("own", most)))
    monkeypatch.setattr(torch.nn.utils, "clip_grad_norm_", lambda p, most: calls.append(("torch", most)))

    class Linear(torch.nn.Linear):
        def loss(self, x, t):
            return (self(x) - t).square().mean(), {}
    m = Linear(3, 2)
    train_step(m, torch.optim.SGD(m.parameters(), 0.1), torch.ones(4, 3), torch.ones(4, 2), grad_clip=0.5, fused_clip=fused)
    assert calls == [("own" if fused else "torch", 0.5)]
