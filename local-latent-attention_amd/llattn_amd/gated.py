"""Gated feed-forward ``w2(act(w1 x) * w3 x)`` on the gfx950 kernels (``llattn_gated_fwd/bwd`` of ``include/llattn_lm.h``),
the counterpart with a gate of :func:`llattn_amd.ffn.feed_forward`.

Both projections, the activation and the product are one kernel; the backward's first product leaves the gradients of both
projections, and every weight gradient comes out of one more.  Numerics: bf16 operands, fp32 sums, ``w1 x`` and ``w3 x`` not
rounded, their gated product rounded to bf16 for the last projection; the backward keeps ``act(w1 x)`` and
``act'(w1 x) w3 x`` in 24 bits.
"""
from __future__ import annotations

import ctypes

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib as L
from .linear import pack_params
from .xent import _bf16_rows

BF16 = torch.bfloat16
ACTS = {"silu": 0, "gelu": 1}  # LLATTN_GATE_*
MOST_ROWS, MOST_WIDTH = 1 << 23, 1 << 22


def _ptr(t):
    return None if t is None else t.data_ptr()


def _weights(ws, pads):
    """The weights in bf16, whole and aligned, with ``pads`` zero rows and columns behind; fp32 ones in one launch."""
    cast = [w for w in ws if w.dtype is torch.float32]
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
    b = b.detach().to(torch.float32).contiguous()
    if pad:
        return F.pad(b, (0, pad))
    return b.clone() if b.data_ptr() & 15 else b


def _bytes(cfg, which):
    n = L.load().llattn_gated_bytes(ctypes.byref(cfg), which)
    if n == 0:
        L.check(L.ERR_SHAPE, "llattn_gated_bytes")
    return n


def _forward(x, act, ps, saved):
    """(y, what a backward reads)."""
    (w1, b1, w3, b3, w2, b2), dev = ps, x.device
    (Fd, D), Do = w1.shape, w2.shape[0]
    pd, pf, po = -D % 8, -Fd % 8, -Do % 8
    xb = _bf16_rows(x.reshape(-1, D), pd)
    N = xb.shape[0]
    ws = _weights((w1, w3, w2), ((pf, pd), (pf, pd), (po, pf)))
    bs = [_bias(b, p) for b, p in ((b1, pf), (b3, pf), (b2, po))]
    f32 = torch.float32
    cfg = L.LlattnGatedCfg(N, D + pd, Fd + pf, Do + po, act, L.F32 if w1.dtype is f32 or w3.dtype is f32 else L.BF16,
                           L.F32 if w2.dtype is f32 else L.BF16)
    y = torch.empty((N, Do + po), dtype=BF16, device=dev)
    h = p = s = None
    if saved:
        h = torch.empty((N, Fd + pf), dtype=BF16, device=dev)
        p, s = (torch.empty((3 * N * (Fd + pf),), dtype=torch.uint8, device=dev) for _ in range(2))
    if N:
        n = _bytes(cfg, 0)
        work = torch.empty((n,), dtype=torch.uint8, device=dev)
        from .ops import _call
        with L.on_device(dev):
            _call("llattn_gated_fwd", ctypes.byref(cfg), xb.data_ptr(), xb.stride(0),
                  ctypes.byref(L.LlattnGatedWeights(*map(_ptr, ws), *map(_ptr, bs))), _ptr(h), _ptr(p), _ptr(s), y.data_ptr(),
                  work.data_ptr(), n, L.stream_ptr(dev), work=6 * N * D * Fd)
    if po:
        y = y[:, :Do]
    return y.reshape(*x.shape[:-1], Do), cfg, (xb, *ws, h, p, s)


class _Gated(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, act, *ps):
        y, cfg, kept = _forward(x, act, ps, True)
        ctx.save_for_backward(*kept)
        ctx.meta = cfg, x.shape, x.dtype, [None if p is None else (p.shape, p.dtype) for p in ps]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xb, w1, w3, w2, h, p, s = ctx.saved_tensors
        cfg, x_shape, x_dtype, params = ctx.meta
        N, dev = cfg.rows, xb.device
        want = [ctx.needs_input_grad[0], *ctx.needs_input_grad[2:]]
        if N == 0:
            grads = [torch.zeros(m[0], dtype=m[1], device=dev) if on else None
                     for m, on in zip([(x_shape, x_dtype), *params], want)]
            return grads[0], None, *grads[1:]
        Do = params[4][0][0]
        d = dy.reshape(N, Do).to(BF16)
        d = F.pad(d, (0, cfg.D_out - Do)) if cfg.D_out > Do else d.contiguous()
        if d.data_ptr() & 15:
            d = d.clone()
        types = (torch.float32, BF16)
        new = lambda on, *shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=dev) if on else None  # noqa: E731
        both = want[1] or want[3]
        dx = new(want[0], N, cfg.D, dtype=BF16)
        dw1, dw3 = (new(both, cfg.F, cfg.D, dtype=types[cfg.dw_dtype]) for _ in range(2))
        dw2 = new(want[5], cfg.D_out, cfg.F, dtype=types[cfg.dw2_dtype])
        db1, db3, db2 = (new(want[i], n) for i, n in ((2, cfg.F), (4, cfg.F), (6, cfg.D_out)))
        n = _bytes(cfg, 1)
        work = torch.empty((n,), dtype=torch.uint8, device=dev)
        from .ops import _call
        with L.on_device(dev):
            _call("llattn_gated_bwd", ctypes.byref(cfg), xb.data_ptr(), xb.stride(0),
                  ctypes.byref(L.LlattnGatedWeights(_ptr(w1), _ptr(w3), _ptr(w2), None, None, None)), h.data_ptr(), p.data_ptr(),
                  s.data_ptr(), d.data_ptr(), ctypes.byref(L.LlattnGatedGrads(*map(_ptr, (dx, dw1, dw3, dw2, db1, db3, db2)))),
                  work.data_ptr(), n, L.stream_ptr(dev), work=12 * N * cfg.D * cfg.F)
        D = x_shape[-1]
        out = [dx[:, :D].to(x_dtype).reshape(x_shape) if want[0] else None, None]
        for g, m, on in zip((dw1, db1, dw3, db3, dw2, db2), params, want[1:]):
            if not on:
                out.append(None)
                continue
            for axis, k in enumerate(m[0]):
                g = g.narrow(axis, 0, k) if g.shape[axis] > k else g
            out.append(g.to(m[1]))
        return tuple(out)


def gated_feed_forward(x: torch.Tensor, w1: torch.nn.Linear, w3: torch.nn.Linear, w2: torch.nn.Linear,
                       act: str = "silu") -> torch.Tensor:
    """bf16 ``w2(act(w1(x)) * w3(x))`` of ``x [..., D]``; ``act``: ``"silu"`` or ``"gelu"`` (the exact one).

    ``w1`` and ``w3`` map D to F, ``w2`` F to any width, each with a bias or without.  ``x`` and the weights are bf16 or fp32,
    fp32 ones rounded to bf16 as under autocast; sums are fp32, gradients come in their input's type, those of weights and
    biases from fp32 sums, ``x``'s rounded to bf16 before it is widened.  Widths that are not multiples of 8 are padded in copies.  Fewer than 2^23 rows.  Differentiable
    once, in reverse mode.  GPU only."""
    from .ffn import _param
    if act not in ACTS:
        raise ValueError(f"gated_feed_forward: act must be one of {tuple(ACTS)}, got {act!r}")
    ps = [_param(m, n) for m in (w1, w3, w2) for n in ("weight", "bias")]
    a, b, c = ps[0], ps[2], ps[4]
    if x.dim() < 1 or a.dim() != 2 or a.shape[1] != x.shape[-1] or b.shape != a.shape or c.dim() != 2 or c.shape[1] != a.shape[0] \
            or 0 in a.shape or 0 in c.shape:
        raise ValueError(f"gated_feed_forward: weights {tuple(a.shape)}, {tuple(b.shape)} and {tuple(c.shape)} do not match "
                         f"x {tuple(x.shape)}")
    for w, bias in zip(ps[::2], ps[1::2]):
        if bias is not None and bias.shape != w.shape[:1]:
            raise ValueError(f"gated_feed_forward: bias {tuple(bias.shape)} for weight {tuple(w.shape)}")
    tensors = [x, *(p for p in ps if p is not None)]
    for t in tensors:
        L.dtype_code(t.dtype)
    if max(*a.shape, *c.shape) >= MOST_WIDTH - 8 or x.numel() // x.shape[-1] >= MOST_ROWS:
        raise ValueError(f"gated_feed_forward: fewer than 2^23 rows and widths below 2^22 expected, got x {tuple(x.shape)}, weights "
                         f"{tuple(a.shape)} and {tuple(c.shape)}")
    L.refuse_tangents("gated_feed_forward", tensors)
    L.require_gpu(*tensors)
    if any(t.device != x.device for t in tensors):
        raise ValueError(f"gated_feed_forward: tensors on {', '.join(sorted({str(t.device) for t in tensors}))}")
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)):
        return _forward(x, ACTS[act], ps, False)[0]
    return _Gated.apply(x, ACTS[act], *ps)
