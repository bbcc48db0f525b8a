"""CPU tests of the head loss and the weight update: the C interface (include/llattn_train.h), and what is refused before
anything is launched."""
import copy
import ctypes
import pickle
import re
import subprocess

import pytest
import torch

from conftest import REPO
from llattn_amd import _lib as L
from llattn_amd import muon
from llattn_amd.lm import build_model, make_optimizer, train_step
from llattn_amd.xent import _bf16_rows, piecewise_head_loss

BF16 = torch.bfloat16


def test_header_matches_the_binding(tmp_path):
    text = (REPO / "include" / "llattn_train.h").read_text()
    names = set(re.findall(r"^\s*(?:int32_t|size_t)\s+(llattn_\w+)\s*\(", text, re.M))
    assert names == set(L.TRAIN_SIGNATURES) and all(hasattr(L.load(), n) for n in names)
    structs = {"llattn_head_cfg": L.LlattnHeadCfg, "llattn_muon_cfg": L.LlattnMuonCfg,
               "llattn_muon_group": L.LlattnMuonGroup}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "llattn_train.h"', "int main(void) {"]
    for c, t in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in t._fields_]
    lines += ['printf("%d\\n%d\\n", LLATTN_MUON_BATCH, LLATTN_MUON_GROUPS);', "return 0; }"]
    src = tmp_path / "l.c"
    src.write_text("\n".join(lines))
    subprocess.run(["gcc", f"-I{REPO / 'include'}", str(src), "-o", str(tmp_path / "l")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for t in structs.values():
        want.append(ctypes.sizeof(t))
        want += [getattr(t, f[0]).offset for f in t._fields_]
    assert got == want + [L.MUON_BATCH, L.MUON_GROUPS]


@pytest.mark.parametrize("cfg,which", [((0, 10, 8, 0, 0), 0), ((4, 0, 8, 0, 0), 0), ((4, 10, 0, 0, 0), 0), ((4, 10, 12, 0, 0), 1),
                                       ((4, 10, 8, 100, 0), 1), ((4, 10, 8, -256, 0), 1), ((4, 10, 8, 0, 7), 1),
                                       ((4, 10, 8, 0, 0), 2)])
def test_head_sizes_refused(cfg, which):
    assert L.load().llattn_head_bytes(ctypes.byref(L.LlattnHeadCfg(*cfg)), which) == 0
    assert L.load().llattn_last_error()


def test_head_workspace_stays_bounded():
    """Row sums of a forward over any vocabulary within 512 MB or a few columns a row; a piece of the backward within
    512 MB (or 256 columns), whatever the vocabulary."""
    n = L.load().llattn_head_bytes
    assert 0 < n(ctypes.byref(L.LlattnHeadCfg(8192, 2 ** 31 - 257, 64, 0, 0)), 0) < 512 << 20
    # beside the piece (rows a cache line apart): the sums of dh in fp32, in four k splits (192 tiles of 256 x 256)
    assert n(ctypes.byref(L.LlattnHeadCfg(8192, 131072, 1536, 0, 1)), 1) <= (512 << 20) + 8192 * 128 + 4 * 8192 * 1536 * 4 + 1024


def _head_fwd(rows=4, V=10, D=8, h=1 << 20, ldh=8, w=1 << 20, ldw=8, t=1 << 20, loss=1 << 20, lse=1 << 20, total=None, inv=None,
              ws=1 << 20, n=1 << 30):
    p = lambda v: None if not v else ctypes.c_void_p(v)  # noqa: E731
    cfg = L.LlattnHeadCfg(rows, V, D, 0, 0)
    return L.load().llattn_head_fwd(ctypes.byref(cfg), p(h), ldh, p(w), ldw, p(t), -100, p(loss), p(lse), None, p(total), p(inv),
                                    p(ws), n, None)


@pytest.mark.parametrize("kw,code", [
    (dict(h=0), L.ERR_LAYOUT), (dict(w=0), L.ERR_LAYOUT), (dict(t=0), L.ERR_LAYOUT), (dict(loss=0), L.ERR_LAYOUT),
    (dict(lse=0), L.ERR_LAYOUT), (dict(inv=1 << 20), L.ERR_LAYOUT), (dict(ldh=4), L.ERR_LAYOUT), (dict(ldw=12), L.ERR_LAYOUT),
    (dict(h=(1 << 20) + 2), L.ERR_LAYOUT), (dict(ldw=1 << 23), L.ERR_LAYOUT), (dict(ws=0), L.ERR_WORKSPACE), (dict(n=1), L.ERR_WORKSPACE),
    (dict(D=9), L.ERR_SHAPE), (dict(rows=1 << 23), L.ERR_SHAPE)])
def test_head_forward_refused(kw, code):
    assert _head_fwd(**kw) == code


def test_head_backward_refused():
    lib, cfg = L.load(), L.LlattnHeadCfg(4, 10, 8, 0, 0)
    p = ctypes.c_void_p
    def call(lse=1 << 20, grad=1 << 20, stride=0, dh=1 << 20, ws=1 << 20):
        return lib.llattn_head_bwd(ctypes.byref(cfg), p(1 << 20), 8, p(1 << 20), 8, p(1 << 20), -100, p(lse), p(grad), stride, None,
                                   p(dh), None, p(ws), 1 << 30, None)
    assert call(lse=0) == call(grad=0) == call(stride=2) == call(stride=-1) == call(dh=(1 << 20) + 4) == L.ERR_LAYOUT
    assert call(ws=0) == L.ERR_WORKSPACE


def test_piecewise_head_loss_refusals():
    h, w, t = torch.zeros(4, 8, dtype=BF16), torch.zeros(10, 8, dtype=BF16), torch.zeros(4, dtype=torch.int64)
    bad = [dict(h=torch.zeros(4, 16, dtype=BF16)), dict(weight=w[0]), dict(weight=torch.zeros(0, 8, dtype=BF16)), dict(targets=t[:3]),
           dict(targets=t.float()), dict(targets=t.bool()), dict(reduction="avg"), dict(h=h.half()), dict(weight=w.double()),
           dict(piece=100), dict(piece=-256)]
    for kw in bad:
        with pytest.raises(ValueError):
            piecewise_head_loss(**{**dict(h=h, weight=w, targets=t), **kw})
    with pytest.raises(RuntimeError, match="no CPU path"):
        piecewise_head_loss(h, w, t)


CFG = dict(n_groups=1, steps=5, nesterov=1, tiles=0, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, mu=0.95)
GROUP = dict(batch=1, rows=4, cols=8, g_dtype=0, w_dtype=0, keep=1.0, step=0.1)


def _muon_cfg(**kw):
    group = L.LlattnMuonGroup(*{**GROUP, **{k: v for k, v in kw.items() if k in GROUP}}.values())
    return L.LlattnMuonCfg(*{**CFG, **{k: v for k, v in kw.items() if k in CFG}}.values()), (L.LlattnMuonGroup * 20)(*[group] * 20)


@pytest.mark.parametrize("kw", [dict(batch=0), dict(batch=129), dict(rows=0), dict(cols=-1), dict(rows=32769), dict(g_dtype=2),
                                dict(w_dtype=-1), dict(steps=0), dict(steps=101), dict(eps=-1.0), dict(eps=float("nan")),
                                dict(a=5.0), dict(a=2.0, b=0.0, c=0.0), dict(b=-20.0), dict(c=float("nan")), dict(n_groups=0),
                                dict(n_groups=17), dict(n_groups=2, batch=65), dict(tiles=-1), dict(tiles=5)])
def test_muon_configurations_refused(kw):
    lib = L.load()
    cfg, groups = _muon_cfg()
    assert lib.llattn_muon_bytes(ctypes.byref(cfg), groups) > 0
    cfg, groups = _muon_cfg(**kw)
    assert lib.llattn_muon_bytes(ctypes.byref(cfg), groups) == 0
    assert b"llattn_muon" in lib.llattn_last_error()


def test_muon_calls_refused():
    lib, p = L.load(), ctypes.c_void_p
    cfg, groups = _muon_cfg()
    one, odd, none = (muon._pointers([v]) for v in (1 << 20, (1 << 20) + 2, None))
    ref = ctypes.byref(cfg), groups
    assert lib.llattn_orthogonalize(*ref, one, one, None, 1 << 30, None) == L.ERR_WORKSPACE
    assert lib.llattn_orthogonalize(*ref, one, one, p(1 << 20), 16, None) == L.ERR_WORKSPACE
    for g, o in ((none, one), (one, none), (odd, one), (one, odd), (None, one), (one, None)):
        assert lib.llattn_orthogonalize(*ref, g, o, p(1 << 20), 1 << 40, None) == L.ERR_LAYOUT
    for k in range(5):
        for v in (none, odd, None):
            args = [one] * 5
            args[k] = v
            assert lib.llattn_muon_update(*ref, *args, p(1 << 20), 1 << 40, None) == L.ERR_LAYOUT
    bad, groups = _muon_cfg(mu=1.0)
    assert lib.llattn_muon_update(ctypes.byref(bad), groups, *[one] * 5, p(1 << 20), 1 << 40, None) == L.ERR_SHAPE


def test_muon_calls_are_cut():
    """Every matrix once, in order, within 16 kinds, 128 matrices and the workspace that the library asks for."""
    for kinds in ([((64, 128), 300)], [((8 + i, 9), 1 + i) for i in range(40)], [((4096, 4096), 60), ((16, 16), 3)],
                  [((32768, 32768), 2), ((8, 8), 1)], []):
        seen = [[] for _ in kinds]
        for call in muon._calls(kinds):
            assert 0 < len(call) <= L.MUON_GROUPS and sum(n for _, _, n in call) <= L.MUON_BATCH
            groups = [L.LlattnMuonGroup(n, *kinds[k][0], 0, 0, 1.0, 0.1) for k, _, n in call]
            cfg, _ = _muon_cfg(n_groups=len(groups))
            n = L.load().llattn_muon_bytes(ctypes.byref(cfg), (L.LlattnMuonGroup * len(groups))(*groups))
            assert n > 0 and (n <= muon.WORKSPACE_BYTES + (1 << 20) or len(groups) == groups[0].batch == 1)
            for k, first, n in call:
                seen[k] += range(first, first + n)
        assert seen == [list(range(c)) for _, c in kinds]


def test_orthogonalize_refusals():
    x = torch.zeros(3, 4)
    for args, kw in (((x[0],), {}), ((x.half(),), {}), ((x,), dict(steps=0)), ((x,), dict(steps=2.5)), ((x,), dict(eps=-1.0)),
                     ((x,), dict(coefficients=(1.0, 2.0))), ((x.clone().requires_grad_(True),), {})):
        with pytest.raises(ValueError):
            muon.orthogonalize(*args, **kw)
    with pytest.raises(RuntimeError, match="no CPU path"):
        muon.orthogonalize(x)


def test_muon_update_refusals():
    w, g, m = torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6)
    other = torch.zeros(4, 6)
    bad = [(([w], [g], []), {}), (([w[0]], [g[0]], [m[0]]), {}), (([w.half()], [g], [m]), {}), (([w], [g.t()], [m]), {}),
           (([w], [g], [m.to(BF16)]), {}), (([w.t()], [g.t()], [m.t()]), {}), (([w, w], [g, g], [m, other]), {}),
           (([w], [g], [w]), {}), (([w], [w], [m]), {}), (([w, other], [g, g], [m, other.clone()]), dict(out=([other, w], [m, g.clone()]))),
           (([w], [g], [m]), dict(out=([other],))), (([w], [g], [m]), dict(out=([other.to(BF16)], [m]))),
           (([w], [g], [m]), dict(lr=torch.tensor(0.1))), (([w], [g], [m]), dict(momentum=1.0)), (([w], [g], [m]), dict(scale="none")),
           (([w], [g], [m]), dict(steps=-1)), ((torch.zeros(1, 0, 4), torch.zeros(1, 0, 4), torch.zeros(1, 0, 4)), {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            muon.muon_update(*args, **{"lr": 0.1, **kw})
    with pytest.raises(RuntimeError, match="no CPU path"):
        muon.muon_update([w], [g], [m], lr=0.1)
    muon.muon_update([], [], [], lr=0.1)


def test_optimisers_refuse_vectors_and_unknown_choices():
    with pytest.raises(ValueError):
        muon.Muon([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        muon.Muon([torch.nn.Parameter(torch.zeros(3, 4))], scale="max")
    model = build_model(vocab_size=32, max_seq_len=16, d_model=16, n_heads=2, n_layers=2, d_ff=32, latent_d_model=8, latent_heads=2)
    with pytest.raises(ValueError):
        make_optimizer(model, matrices="sgd")
    opt = make_optimizer(model, matrices="muon")
    mats = {id(p) for p in opt.param_groups[0]["params"]}
    names = {n for n, p in model.named_parameters() if id(p) in mats}
    assert len(names) == 2 * 7 and not any("embedding" in n or "position" in n or "gate" in n for n in names)
    assert sum(len(g["params"]) for g in opt.param_groups) == len(list(model.parameters()))
    assert isinstance(make_optimizer(model), torch.optim.AdamW)


def test_groups_added_to_the_joint_optimiser_are_adamws():
    w, b, e = (torch.nn.Parameter(torch.zeros(s)) for s in ((4, 8), (4,), (3, 4)))
    opt = muon.MuonAdamW([w], [b], dict(lr=0.1), lr=1e-3, betas=(0.9, 0.95))
    opt.add_param_group({"params": [e], "weight_decay": 0.0})
    b.grad, e.grad = torch.ones(4), torch.ones(3, 4)
    opt.step()
    assert not w.detach().any()
    assert torch.allclose(e.detach(), torch.full((3, 4), -1e-3)) and torch.allclose(b.detach(), torch.full((4,), -1e-3))
    again = muon.MuonAdamW([w], [{"params": [b]}, {"params": [e], "weight_decay": 0.0}], dict(lr=0.1), lr=1e-3)
    again.load_state_dict(opt.state_dict())
    assert again.param_groups[2]["betas"] == (0.9, 0.95) and again.param_groups[0]["momentum"] == 0.95


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_tangents_are_refused(which):
    """A dual tensor whose primal needs no gradient: an answer without a tangent would read as a derivative of zero."""
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        def dual(*shape, dtype=torch.float32):
            return fw.make_dual(torch.zeros(*shape, dtype=dtype), torch.ones(*shape, dtype=dtype))
        h, w, t = torch.zeros(4, 8, dtype=BF16), torch.zeros(10, 8, dtype=BF16), torch.zeros(4, dtype=torch.int64)
        x = [torch.zeros(4, 6) for _ in range(3)]
        calls = [lambda: piecewise_head_loss(dual(4, 8, dtype=BF16), w, t),
                 lambda: piecewise_head_loss(h, dual(10, 8, dtype=BF16), t, reduction="none"),
                 lambda: muon.orthogonalize(dual(3, 4)),
                 *[lambda k=k: muon.muon_update(*[[dual(4, 6) if i == k else v] for i, v in enumerate(x)], lr=0.1) for k in range(3)]]
        with pytest.raises(NotImplementedError, match="forward-mode"):
            calls[which]()
        with pytest.raises(RuntimeError, match="no CPU path"):  # plain tensors beside an open level
            piecewise_head_loss(h, w, t)


def _optimiser(kind, mats, vecs):
    return muon.Muon(mats, lr=0.1) if kind == "muon" else muon.MuonAdamW(mats, vecs, dict(lr=0.1), lr=1e-3)


@pytest.mark.parametrize("kind", ["muon", "joint"])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_momenta_are_loaded_in_fp32(kind, dtype):
    """A state saved and loaded has the same bits, bf16 parameters' momenta too, and shares no memory with the dict."""
    def build():
        return _optimiser(kind, [torch.nn.Parameter(torch.zeros(3, 5, dtype=dtype)) for _ in range(3)], [torch.nn.Parameter(torch.zeros(4))])
    a, b = build(), build()
    want = {i: torch.randn(3, 5, generator=torch.Generator().manual_seed(i)) for i in (0, 2)}  # the second has not been updated yet
    for i, m in want.items():
        a.state[a.param_groups[0]["params"][i]]["momentum_buffer"] = m.clone()
    saved = a.state_dict()
    b.load_state_dict(saved)
    for i, p in enumerate(b.param_groups[0]["params"]):
        assert (i in want) == ("momentum_buffer" in b.state.get(p, {}))
        if i in want:
            got = b.state[p]["momentum_buffer"]
            assert got.dtype is torch.float32 and torch.equal(got, want[i])
            assert got.data_ptr() != saved["state"][i]["momentum_buffer"].data_ptr()


@pytest.mark.parametrize("how", ["deepcopy", "pickle"])
def test_copies_of_the_optimisers_go_on(how):
    """A copy has its own parameters and state and steps like the original (vectors; matrices need a GPU)."""
    w, b = torch.nn.Parameter(torch.zeros(4, 8)), torch.nn.Parameter(torch.zeros(4))
    opt = muon.MuonAdamW([w], [b], dict(lr=0.1), lr=1e-3, betas=(0.9, 0.95))
    b.grad = torch.ones(4)
    opt.step()
    opt.state[w]["momentum_buffer"] = torch.ones(4, 8)
    twin = copy.deepcopy(opt) if how == "deepcopy" else pickle.loads(pickle.dumps(opt))
    (w2,), (b2,) = (g["params"] for g in twin.param_groups)
    assert b2 is not b and torch.equal(b2, b) and torch.equal(twin.state[w2]["momentum_buffer"], torch.ones(4, 8))
    assert twin.param_groups[0]["momentum"] == 0.95 and twin.param_groups[1]["betas"] == (0.9, 0.95)
    b.grad, b2.grad = torch.full((4,), -2.0), torch.full((4,), -2.0)
    opt.step()
    before = b.detach().clone()
    assert not torch.equal(b2, b)
    twin.step()
    assert torch.equal(b2, b) and torch.equal(b, before)
    twin.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))]})
    assert twin.param_groups[2]["betas"] == (0.9, 0.95) and len(opt.param_groups) == 2
    twin.zero_grad()
    twin.step()
    only = muon.Muon([w], lr=0.1)
    again = copy.deepcopy(only) if how == "deepcopy" else pickle.loads(pickle.dumps(only))
    again.step()  # no gradients
    assert again.param_groups[0]["lr"] == 0.1


def test_groups_of_matrices_are_all_muons(monkeypatch):
    """Matrices in several groups, each with options of its own: none is left to AdamW."""
    seen = []
    monkeypatch.setattr(muon, "muon_update", lambda w, g, m, **kw: seen.append((list(w), kw["lr"], kw["momentum"])))
    u, v, w = (torch.nn.Parameter(torch.zeros(4, 8)) for _ in range(3))
    b = torch.nn.Parameter(torch.zeros(4))
    opt = muon.MuonAdamW([{"params": [u]}, {"params": [v, w], "lr": 0.5}], [b], dict(lr=0.1, momentum=0.9), lr=1e-3)
    for p in (u, v, b):
        p.grad = torch.ones_like(p)
    opt.step()
    assert [([id(p) for p in ps], lr, mu) for ps, lr, mu in seen] == [([id(u)], 0.1, 0.9), ([id(v)], 0.5, 0.9)]
    assert not any(p.detach().any() for p in (u, v, w)) and torch.allclose(b.detach(), torch.full((4,), -1e-3))


def _row_views():
    """[R, 64] bf16 views whose rows the kernels do not read as they are."""
    x = torch.randn(2 * (1 << 23) + 64, generator=torch.Generator().manual_seed(0)).to(BF16)
    return [("far apart", x.as_strided((2, 64), (1 << 23, 1))), ("farther", x.as_strided((2, 64), ((1 << 23) + 8, 1))),
            ("one row, far stride", x.as_strided((1, 64), (1 << 25, 1))), ("one row, stride 1", x.as_strided((1, 64), (1, 1))),
            ("one row, stride 0", x[:64].expand(1, 64).as_strided((1, 64), (0, 1))), ("overlapping", x.as_strided((3, 64), (8, 1))),
            ("odd stride", x.as_strided((3, 64), (65, 1))), ("shifted", x[1:129].view(2, 64)), ("columns", x[:128].view(64, 2).t())]


@pytest.mark.parametrize("k", range(9))
def test_rows_come_in_a_layout_that_the_kernels_take(k):
    name, t = _row_views()[k]
    got = _bf16_rows(t, 0)
    assert got.stride(1) == 1 and 64 <= got.stride(0) < 1 << 23 and got.stride(0) % 8 == 0 and got.data_ptr() % 16 == 0, name
    assert torch.equal(got, t)
    L.check(L.OK if _head_fwd(rows=len(got), D=64, ldh=got.stride(0), ldw=64, n=1) == L.ERR_WORKSPACE else L.ERR_LAYOUT, name)


def test_rows_that_the_kernels_take_are_not_copied():
    x = torch.zeros(6, 128, dtype=BF16)
    for t in (x, x[:, :64], x[1:, 64:], x[::2]):
        assert _bf16_rows(t, 0).data_ptr() == t.data_ptr() and _bf16_rows(t, 0).stride() == t.stride()


class _OwnLoss(torch.nn.Module):
    """A model whose loss takes inputs and targets alone."""

    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.ones(3))

    def loss(self, inputs, targets):
        return (self.w * inputs).sum() - targets.sum(), {}


def test_train_step_asks_for_pieces_only_where_told():
    model = _OwnLoss()
    opt = torch.optim.SGD(model.parameters(), lr=0.5)
    loss = train_step(model, opt, torch.tensor([1.0, 0.0, 2.0]), torch.zeros(1), grad_clip=0.0)
    assert float(loss) == 3.0 and model.w.tolist() == [0.5, 1.0, 0.0]
    with pytest.raises(TypeError):
        train_step(model, opt, torch.ones(3), torch.zeros(1), vocab_piece=256)


def test_train_step_refuses_pieces_of_full_logits():
    model = _OwnLoss()
    with pytest.raises(ValueError, match="vocab_piece"):
        train_step(model, torch.optim.SGD(model.parameters(), lr=0.5), torch.ones(3), torch.zeros(1), fused_loss=False, vocab_piece=0)


def test_a_list_is_refused_before_any_of_it_is_updated():
    """A matrix that the library refuses, in a place that a later call of several would reach."""
    small, wide = [torch.zeros(4, 6) for _ in range(3)], [torch.zeros(1, 32769) for _ in range(3)]
    for order in ((small, wide), (wide, small)):
        with pytest.raises(ValueError, match="32768"):
            muon.muon_update(*([v[i] for v in order] for i in range(3)), lr=0.1)
    fits = [torch.zeros(32768, 1) for _ in range(3)]
    with pytest.raises(RuntimeError, match="no CPU path"):
        muon.muon_update(*([v] for v in fits), lr=0.1)


@pytest.mark.parametrize("src,out,copied", [((0, 4), (0, 4), False), ((1, 5), (0, 4), True), ((0, 4), (1, 5), True), ((0, 4), (4, 8), False),
                                            ((4, 8), (0, 4), False), ((0, 4), (3, 7), True)])
def test_an_output_across_its_input_gets_a_copy(src, out, copied):
    x = torch.arange(8 * 6, dtype=torch.float32).view(8, 2, 3)
    a, b = x[src[0]:src[1]], x[out[0]:out[1]]
    got = muon._apart(a, b)
    assert torch.equal(got, a) and (got.data_ptr() != a.data_ptr()) == copied


@pytest.mark.parametrize("eps", [1e-46, 1e-300, 2.0 ** -149, 1e-7, 0.0])
def test_an_eps_above_zero_stays_above_zero(eps):
    """Rounded to fp32, in which the library takes it, it would be 0, and a zero matrix NaN instead of zero."""
    got = muon._config(5, muon.COEFFICIENTS, eps).eps
    assert (got > 0) == (eps > 0) and got == pytest.approx(max(eps, 2.0 ** -149) if eps else 0.0)


def test_whole_numbers_of_steps():
    """A whole number of any type counts; what is none is refused as such."""
    x = torch.zeros(3, 4)
    assert muon._config(5.0, muon.COEFFICIENTS, 1e-7).steps == 5
    for steps in (5, 5.0):
        with pytest.raises(RuntimeError, match="no CPU path"):
            muon.orthogonalize(x, steps=steps)
    for steps in (float("inf"), float("nan"), 2 ** 32 + 5, None, "5"):
        with pytest.raises(ValueError, match="steps"):
            muon.orthogonalize(x, steps=steps)


def test_head_workspace_of_the_present_plan():
    """q of a piece, the sums of dh over splits (4 for 192 tiles of 256 x 256 on 256 CUs), the shared scale: nothing besides."""
    n = L.load().llattn_head_bytes
    assert n(ctypes.byref(L.LlattnHeadCfg(8192, 131072, 1536, 0, 1)), 1) == (512 << 20) + 4 * 8192 * 1536 * 4 + 256
