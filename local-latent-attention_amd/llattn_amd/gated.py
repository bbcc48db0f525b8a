"""Gated feed-forward ``w2(act(w1 x) * w3 x)`` on the gfx950 kernels (``llattn_gated_fwd/bwd`` of ``include/llattn_lm.h``),
the counterpart with a gate of :func:`llattn_amd.ffn.feed_forward`.

Both projections, the activation and the product are one kernel; the backward's first product leaves the gradients of both
projections, and both weight gradients come out of one more.  Numerics: bf16 operands, fp32 sums, ``w1 x`` and ``w3 x`` not
rounded, their gated product and its counterparts backward rounded to bf16 (two bf16 values up to 64 rows); the backward keeps
``act(w1 x)`` and ``act'(w1 x) w3 x`` in 24 bits.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import ops
from .ffn import _param
from .linear import pack_params
from .xent import _bf16_rows

BF16, F32 = torch.bfloat16, torch.float32
TYPES = (F32, BF16)  # by LLATTN_F32, LLATTN_BF16
ACTS = {"silu": 0, "gelu": 1}  # LLATTN_GATE_*
MOST_ROWS, MOST_WIDTH = 1 << 23, 1 << 22


def _ptr(t):
    return None if t is None else t.data_ptr()


def _weights(ws, pads):
    """The weights in bf16, whole and aligned, with ``pads`` zero rows and columns behind; fp32 ones in one launch."""
    if ws[0].dtype is ws[1].dtype is ws[2].dtype is BF16 and not any(map(any, pads)):
        ws = [w if w.is_contiguous() else w.detach().contiguous() for w in ws]
        return [w.detach().clone() if w.data_ptr() & 15 else w for w in ws]
    cast = [w for w in ws if w.dtype is F32]
    done = dict(zip(map(id, cast), pack_params([([w], BF16) for w in cast]))) if cast else {}
    out = []
    for w, (rows, cols) in zip(ws, pads):
        w = done.get(id(w), w).detach()
        if rows or cols:
            w = F.pad(w, (0, cols, 0, rows))
        w = w.contiguous()
        out.append(w.clone() if w.data_ptr() & 15 else w)
    return out


def _bias(b, pad):
    if b is None:
        return None
    b = b.detach().to(F32).contiguous()
    if pad:
        return F.pad(b, (0, pad))
    return b.clone() if b.data_ptr() & 15 else b


def _buffer(cfg, which, device):
    n = L.load().llattn_gated_bytes(ctypes.byref(cfg), which)
    if n == 0:
        L.check(L.ERR_SHAPE, "llattn_gated_bytes")
    return torch.empty((n,), dtype=torch.uint8, device=device) if n > 1 else None, n


def _forward(x, act, ps, saved):
    """(y, configuration, what a backward reads)."""
    (w1, b1, w3, b3, w2, b2), dev = ps, x.device
    (Fd, D), Do = w1.shape, w2.shape[0]
    pd, pf, po = -D % 8, -Fd % 8, -Do % 8
    xb = _bf16_rows(x if x.dim() == 2 else x.reshape(-1, D), pd)
    N = xb.shape[0]
    ws = _weights((w1, w3, w2), ((pf, pd), (pf, pd), (po, pf)))
    cfg = L.LlattnGatedCfg(N, D + pd, Fd + pf, Do + po, act, L.F32 if w1.dtype is F32 or w3.dtype is F32 else L.BF16,
                           L.F32 if w2.dtype is F32 else L.BF16)
    y = torch.empty((N, Do + po), dtype=BF16, device=dev)
    kept = None
    if N:
        bs = (_bias(b1, pf), _bias(b3, pf), _bias(b2, po))
        if saved:
            kept, _ = _buffer(cfg, L.GATED_KEPT, dev)
        work, n = _buffer(cfg, L.GATED_FORWARD if saved else L.GATED_ALONE, dev)
        with L.on_device(dev):
            ops._call("llattn_gated_fwd", ctypes.byref(cfg), xb.data_ptr(), xb.stride(0),
                  ctypes.byref(L.LlattnGatedWeights(*map(_ptr, ws), *map(_ptr, bs))), _ptr(kept), y.data_ptr(), _ptr(work), n,
                  L.stream_ptr(dev), work=2 * N * Fd * (2 * D + Do))
    if po:
        y = y[:, :Do]
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], Do), cfg, (xb, *ws, kept)


def _backward(ctx, dy):
    xb, w1, w3, w2, kept = ctx.saved_tensors
    cfg, x_shape, x_dtype, params = ctx.meta
    N, dev = cfg.rows, xb.device
    need = ctx.needs_input_grad
    want = (need[0], *need[2:])
    if N == 0:
        grads = [torch.zeros(m[0], dtype=m[1], device=dev) if on else None
                 for m, on in zip([(x_shape, x_dtype), *params], want)]
        return grads[0], None, *grads[1:]
    Do = params[4][0][0]
    d = dy if dy.dim() == 2 else dy.reshape(N, Do)
    if d.dtype is not BF16:
        d = d.to(BF16)
    d = F.pad(d, (0, cfg.D_out - Do)) if cfg.D_out > Do else d.contiguous()
    if d.data_ptr() & 15:
        d = d.clone()
    D, Fd, dt = cfg.D, cfg.F, TYPES[cfg.dw_dtype]
    both = want[1] or want[3]
    dx = torch.empty((N, D), dtype=BF16, device=dev) if want[0] else None
    dw1 = torch.empty((Fd, D), dtype=dt, device=dev) if both else None
    dw3 = torch.empty((Fd, D), dtype=dt, device=dev) if both else None
    dw2 = torch.empty((cfg.D_out, Fd), dtype=TYPES[cfg.dw2_dtype], device=dev) if want[5] else None
    db1, db3, db2 = (torch.empty((n,), dtype=F32, device=dev) if want[i] else None
                     for i, n in ((2, Fd), (4, Fd), (6, cfg.D_out)))
    grads = (dx, dw1, dw3, dw2, db1, db3, db2)
    work, n = _buffer(cfg, L.GATED_BACKWARD, dev)
    with L.on_device(dev):
        ops._call("llattn_gated_bwd", ctypes.byref(cfg), xb.data_ptr(), xb.stride(0),
              ctypes.byref(L.LlattnGatedWeights(w1.data_ptr(), w3.data_ptr(), w2.data_ptr(), None, None, None)), kept.data_ptr(),
              d.data_ptr(), ctypes.byref(L.LlattnGatedGrads(*map(_ptr, grads))), work.data_ptr(), n, L.stream_ptr(dev),
              work=4 * N * Fd * (2 * D + Do))
    if dx is not None:
        if D > x_shape[-1]:
            dx = dx[:, :x_shape[-1]]
        dx = dx.to(x_dtype) if len(x_shape) == 2 else dx.to(x_dtype).reshape(x_shape)
    out = [dx, None]
    for g, m, on in zip((dw1, db1, dw3, db3, dw2, db2), params, want[1:]):
        if on:
            if g.shape != m[0]:
                g = g[tuple(slice(k) for k in m[0])]
            out.append(g if g.dtype is m[1] else g.to(m[1]))
        else:
            out.append(None)
    return tuple(out)


_backward_once = once_differentiable(_backward)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, act, *ps):
        y, cfg, kept = _forward(x, act, ps, True)
        ctx.save_for_backward(*kept)
        ctx.meta = cfg, x.shape, x.dtype, [None if p is None else (p.shape, p.dtype) for p in ps]
        return y

    @staticmethod
    def backward(ctx, dy):
        # a graph of the gradients is recorded: it refuses to go on; without one the wrapper has nothing to do
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


def gated_feed_forward(x: torch.Tensor, w1: torch.nn.Linear, w3: torch.nn.Linear, w2: torch.nn.Linear,
                       act: str = "silu") -> torch.Tensor:
    """bf16 ``w2(act(w1(x)) * w3(x))`` of ``x [..., D]``; ``act``: ``"silu"`` or ``"gelu"`` (the exact one).

    ``w1`` and ``w3`` map D to F, ``w2`` F to any width, each with a bias or without.  ``x`` and the weights are bf16 or fp32,
    fp32 ones rounded to bf16 as under autocast; sums are fp32, gradients come in their input's type, those of weights and
    biases from fp32 sums, ``x``'s rounded to bf16 before it is widened.  Widths that are not multiples of 8 are padded in copies.
    Fewer than 2^23 rows; a row's bits depend on how many are beside it (other kernels up to 16, 32 and 64 rows, and its gated product is
    rounded to bf16 above 64).  The layers' weights and biases are read, their forwards and hooks are not run.  Differentiable
    once, in reverse mode.  GPU only."""
    if act not in ACTS:
        raise ValueError(f"gated_feed_forward: act must be one of {tuple(ACTS)}, got {act!r}")
    ps = [_param(m, n) for m in (w1, w3, w2) for n in ("weight", "bias")]
    a, b, c, shape = ps[0].shape, ps[2].shape, ps[4].shape, x.shape
    if not shape or len(a) != 2 or a[1] != shape[-1] or b != a or len(c) != 2 or c[1] != a[0] or 0 in a or 0 in c:
        raise ValueError(f"gated_feed_forward: weights {tuple(a)}, {tuple(b)} and {tuple(c)} do not match x {tuple(shape)}")
    tensors = [x, ps[0], ps[2], ps[4]]
    for rows, bias in ((a[0], ps[1]), (a[0], ps[3]), (c[0], ps[5])):
        if bias is not None:
            if bias.shape != (rows,):
                raise ValueError(f"gated_feed_forward: bias {tuple(bias.shape)} for {rows} outputs")
            tensors.append(bias)
    index = x.get_device()
    for t in tensors:
        L.dtype_code(t.dtype)
    if max(*a, *c) >= MOST_WIDTH - 8 or x.numel() // a[1] >= MOST_ROWS:
        raise ValueError(f"gated_feed_forward: fewer than 2^23 rows and widths below 2^22 expected, got x {tuple(shape)}, weights "
                         f"{tuple(a)} and {tuple(c)}")
    L.refuse_tangents("gated_feed_forward", tensors)
    if index < 0 or any([t.get_device() != index for t in tensors]):
        L.require_gpu(*tensors)
        raise ValueError(f"gated_feed_forward: tensors on {', '.join(sorted({str(t.device) for t in tensors}))}")
    if not (torch.is_grad_enabled() and any([t.requires_grad for t in tensors])):
        return _forward(x, ACTS[act], ps, False)[0]
    return _Gated.apply(x, ACTS[act], *ps)
