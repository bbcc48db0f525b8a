"""Token rows plus position rows on the gfx950 kernels (``llattn_embed_fwd/bwd`` of ``include/llattn_lm.h``).

:func:`embed` is the beginning of the language model (reference models.py:505-580: the token embedding plus the learned
position embedding) as one pass over its output; its backward sums the gradients of both tables in the order of the
sorted tokens, without atomics: the same bits in every call.
"""
from __future__ import annotations

import ctypes
from numbers import Integral, Real

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import ops

MOST = 1 << 22  # rows of a table
LARGEST = torch.finfo(torch.float32).max  # size of the scale
_INDEX = (torch.int64, torch.int32)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A table whose rows are whole, any distance apart."""
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.detach().contiguous()


def _index(t: torch.Tensor) -> torch.Tensor:
    """The indices in order, of 32 or 64 bits (their shape is of no matter to a kernel)."""
    t = t if t.dtype in _INDEX else t.to(torch.int64)
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(ids, weight, position, positions, scale, padding):
    """(out, the indices and the configuration that a backward reads)."""
    V, D = weight.shape
    dev, dtype = weight.device, weight.dtype
    i, p = _index(ids), None if positions is None else _index(positions)
    if p is not None and p.dtype is not i.dtype:
        i, p = i.to(torch.int64), p.to(torch.int64)
    shape = ids.shape
    cfg = L.LlattnEmbedCfg(i.numel(), max(shape[-1] if shape else 1, 1), V, 0 if position is None else position.shape[0], D,
                           L.dtype_code(dtype), i.element_size(), padding, scale)
    out = torch.empty((*shape, D), dtype=dtype, device=dev)
    if cfg.rows:
        w, q = _rows(weight), None if position is None else _rows(position)
        with L.on_device(dev):
            ops._call("llattn_embed_fwd", ctypes.byref(cfg), i.data_ptr(), _ptr(p), w.data_ptr(), w.stride(0), _ptr(q),
                      0 if q is None else q.stride(0), out.data_ptr(), L.stream_ptr(dev),
                      work=(2 + (q is not None)) * cfg.rows * D * out.element_size())
    return out, i, p, cfg


def _buffer(ref, has_pos, which, device):
    """(a buffer of the call's, its bytes), or (None, 1) where it needs none."""
    n = L.load().llattn_embed_bytes(ref, has_pos, which)
    if n == 0:
        L.check(L.ERR_SHAPE, "llattn_embed_bytes")
    return torch.empty((n,), dtype=torch.uint8, device=device) if n > 1 else None, n


def _order(i, p, cfg, tokens, positions):
    """The order of the rows that a backward reads, None where it needs none."""
    ref, dev = ctypes.byref(cfg), i.device
    order, n = _buffer(ref, int(p is not None), L.EMBED_ORDER, dev)
    if order is not None:
        with L.on_device(dev):
            ops._call("llattn_embed_order", ref, i.data_ptr(), _ptr(p), int(tokens), int(positions), order.data_ptr(), n,
                      L.stream_ptr(dev), work=cfg.rows * cfg.index_bytes)
    return order


def _backward(ctx, dout):
    i, p, order = ctx.saved_tensors
    cfg, w_shape, p_shape = ctx.meta
    _, want_w, want_p, *_ = ctx.needs_input_grad
    dw = dout.new_empty(w_shape) if want_w else None
    dp = dout.new_empty(p_shape) if want_p else None
    d = dout if dout.is_contiguous() else dout.contiguous()
    dev, ref = d.device, ctypes.byref(cfg)
    ws, n = _buffer(ref, int(p is not None), L.EMBED_BACKWARD, dev)
    with L.on_device(dev):
        ops._call("llattn_embed_bwd", ref, i.data_ptr(), _ptr(p), _ptr(order), d.data_ptr(), _ptr(dw), _ptr(dp), _ptr(ws), n,
                  L.stream_ptr(dev), work=(cfg.rows + cfg.V + cfg.P) * cfg.D * d.element_size())
    return None, dw, dp, None, None, None


_backward_once = once_differentiable(_backward)


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, position, positions, scale, padding):
        out, i, p, cfg = _forward(ids, weight, position, positions, scale, padding)
        _, tokens, places, *_ = ctx.needs_input_grad
        places = places and p is not None
        # here and not in the backward: nothing of it waits for a gradient
        ctx.save_for_backward(i, p, _order(i, p, cfg, tokens, places) if tokens or places else None)
        ctx.meta = (cfg, weight.shape, None if position is None else position.shape)
        return out

    @staticmethod
    def backward(ctx, dout):
        # a graph of the gradients is recorded: it refuses to go on; without one the wrapper has nothing to do
        return _backward_once(ctx, dout) if torch.is_grad_enabled() else _backward(ctx, dout)


def _check_integers(name: str, t: torch.Tensor) -> None:
    if t.is_floating_point() or t.is_complex() or t.dtype is torch.bool:
        raise ValueError(f"embed: {name} must be integers, got {t.dtype}")


def embed(ids: torch.Tensor, weight: torch.Tensor, position: torch.Tensor | None = None,
          positions: torch.Tensor | None = None, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """``scale * weight[ids] + position[positions]`` for ``ids [..., T]``, ``weight [V, D]`` and ``position [P, D]``
    (fp32 or bf16, one type; any strides) and a finite ``scale``, computed in fp32 and rounded once to that type.

    Without ``positions`` (integers of ``ids``' shape, for packed documents or single tokens at their places) the tokens
    of the last axis stand at positions 0, 1, ...; without ``position`` nothing is added.  An id outside ``[0, V)`` or a
    position outside ``[0, P)`` gives a row of NaN and no gradient to the table that has no such row.  Gradients are
    whole tables in their table's type, summed in fp32 in a fixed order (no atomics); the row ``padding_idx`` of
    ``weight`` gets none.  V and P at most 2^22.  Differentiable once, in reverse mode.  GPU only."""
    w_shape, dtype = weight.shape, weight.dtype
    if len(w_shape) != 2 or 0 in w_shape:
        raise ValueError(f"embed: weight must be a non-empty matrix, got shape {tuple(w_shape)}")
    V, D = w_shape
    if ids.dtype not in _INDEX:
        _check_integers("ids", ids)
    L.dtype_code(dtype)
    tensors = [ids, weight]
    P = 0
    if position is not None:
        p_shape = position.shape
        if len(p_shape) != 2 or p_shape[1] != D or not p_shape[0] or position.dtype is not dtype:
            raise ValueError(f"embed: position {tuple(p_shape)} ({position.dtype}) does not match weight {tuple(w_shape)} ({dtype})")
        P = p_shape[0]
        tensors.append(position)
    if V > MOST or P > MOST:
        raise ValueError(f"embed: at most {MOST} rows in a table")
    if positions is not None:
        if position is None:
            raise ValueError("embed: positions without position rows")
        if positions.dtype not in _INDEX:
            _check_integers("positions", positions)
        if positions.shape != ids.shape:
            raise ValueError(f"embed: positions {tuple(positions.shape)} for ids {tuple(ids.shape)}")
        tensors.append(positions)
    elif P and ids.dim() and ids.shape[-1] > P:
        raise ValueError(f"embed: {ids.shape[-1]} tokens in a row and {P} positions")
    if type(scale) is not float and not isinstance(scale, Real):
        raise ValueError(f"embed: scale must be a number, got {type(scale).__name__}")
    if not -LARGEST <= scale <= LARGEST:  # an infinite one would make NaN of the rows that no token names
        raise ValueError(f"embed: scale must be finite in fp32, got {scale}")
    padding = -1
    if padding_idx is not None:
        if not isinstance(padding_idx, Integral) or not -V <= padding_idx < V:
            raise ValueError(f"embed: padding_idx {padding_idx} outside the {V} rows")
        padding = int(padding_idx) % V
    if ids.numel() >= 1 << 31:
        raise ValueError(f"embed: {ids.numel()} tokens, fewer than 2^31 expected")
    L.refuse_tangents("embed", tensors)
    index = weight.get_device()
    if index < 0 or any([t.get_device() != index for t in tensors]):
        L.require_gpu(*tensors)
        raise ValueError(f"embed: tensors on {', '.join(str(t.device) for t in tensors)}")
    if torch.is_grad_enabled() and (weight.requires_grad or P and position.requires_grad):
        return _Embed.apply(ids, weight, position, positions, float(scale), padding)
    return _forward(ids, weight, position, positions, float(scale), padding)[0]
