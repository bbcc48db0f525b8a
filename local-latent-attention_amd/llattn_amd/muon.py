"""Orthogonalised weight updates on the gfx950 kernels (``llattn_orthogonalize`` and ``llattn_muon_update`` of
``include/llattn_train.h``).

:func:`orthogonalize` runs the quintic Newton-Schulz iteration ``X <- a X + (b A + c A A) X``, ``A = X X^T``, on a batch
of matrices; :func:`muon_update` is one step of the Muon optimiser on a list of weights (momentum, orthogonalisation,
decay and update), and :class:`Muon` / :class:`MuonAdamW` are the optimisers made of it
(:func:`llattn_amd.lm.make_optimizer` builds the second for the language model).

The iteration runs at fp32's precision whatever the tensors' type: its matrices are held as two fp16 halves and
multiplied on the fp16 matrix cores.
"""
from __future__ import annotations

import ctypes
import math
from numbers import Real

import torch

from . import _lib as L

# coefficients that raise small singular values fastest while those near 1 stay within about 0.7 to 1.2
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
SCALES = ("aspect", "rms")
WORKSPACE_BYTES = 4 << 30  # matrices of one shape are taken together up to this


def _config(batch, shape, g_dtype, w_dtype, steps, coefficients, eps, nesterov=False, mu=0.0, keep=0.0, step=0.0):
    return L.LlattnMuonCfg(batch, *shape, L.dtype_code(g_dtype), L.dtype_code(w_dtype), steps, int(nesterov),
                           *[float(v) for v in coefficients], float(eps), mu, keep, step)


def _bytes(cfg) -> int:
    n = L.load().llattn_muon_bytes(ctypes.byref(cfg))
    if n == 0:
        L.check(L.ERR_SHAPE, "llattn_muon_bytes")
    return n


def _pointers(values):
    return (ctypes.c_void_p * len(values))(*values)


def _chunk(cfg) -> int:
    """Matrices of a call: what fits the workspace, at least one."""
    cfg.batch = 1
    return max(1, min(L.MUON_BATCH, WORKSPACE_BYTES // _bytes(cfg)))


def _check_numbers(who, steps, eps, coefficients):
    if int(steps) != steps or steps < 1:
        raise ValueError(f"{who}: steps must be a positive whole number, got {steps}")
    if not eps >= 0:
        raise ValueError(f"{who}: eps must not be negative, got {eps}")
    if len(coefficients) != 3:
        raise ValueError(f"{who}: three coefficients expected, got {coefficients}")


def orthogonalize(x: torch.Tensor, steps: int = 5, eps: float = 1e-7, coefficients=COEFFICIENTS,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Newton-Schulz iteration on every matrix of ``x [..., m, n]`` (fp32 or bf16; any strides), from ``X = x / (|x|_F +
    eps)``: towards the orthogonal factor of ``x``'s polar decomposition.  Returns ``x``'s type and shape; ``out``
    (contiguous, may be ``x``) receives the result.  A zero matrix stays zero; one that holds an infinity or NaN gives
    NaN throughout.  Not differentiable.  GPU only."""
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: expected [..., m, n], got shape {tuple(x.shape)}")
    _check_numbers("orthogonalize", steps, eps, coefficients)
    L.dtype_code(x.dtype)
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("orthogonalize has no gradient: call it under torch.no_grad() or on a detached tensor")
    L.require_gpu(x)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise ValueError("orthogonalize: out must be contiguous, of x's shape, type and device")
    m, n = x.shape[-2:]
    if x.numel() == 0:
        return out
    src = x.detach().contiguous()
    count, dev = x.numel() // (m * n), x.device
    cfg = _config(1, (m, n), x.dtype, x.dtype, steps, coefficients, eps)
    most, each = _chunk(cfg), m * n * x.element_size()
    from .ops import _call
    with L.on_device(dev):
        for i in range(0, count, most):
            cfg.batch = k = min(most, count - i)
            nws = _bytes(cfg)
            ws = torch.empty((nws,), dtype=torch.uint8, device=dev)
            _call("llattn_orthogonalize", ctypes.byref(cfg), _pointers([src.data_ptr() + (i + j) * each for j in range(k)]),
                  _pointers([out.data_ptr() + (i + j) * each for j in range(k)]), ws.data_ptr(), nws, L.stream_ptr(dev),
                  work=2 * k * each)
    _written([out])
    return out


def _written(tensors) -> None:
    """Tensors that a kernel has written in place, for autograd's checks of what it saved."""
    for t in tensors:
        torch.autograd.graph.increment_version(t)


def _update_scale(scale: str, rows: int, cols: int) -> float:
    return math.sqrt(max(1.0, rows / cols)) if scale == "aspect" else 0.2 * math.sqrt(max(rows, cols))


def _check_update(weights, grads, momenta, out):
    lists = [weights, grads, momenta, *out]
    if len({len(v) for v in lists}) != 1:
        raise ValueError(f"muon_update: lists of different lengths ({', '.join(str(len(v)) for v in lists)})")
    for w, g, m, wo, mo in zip(*lists):
        if w.dim() != 2 or 0 in w.shape:
            raise ValueError(f"muon_update: weights must be non-empty matrices, got shape {tuple(w.shape)}")
        L.dtype_code(w.dtype), L.dtype_code(g.dtype)
        if any(t.shape != w.shape or t.device != w.device for t in (g, m, wo, mo)):
            raise ValueError(f"muon_update: gradient, momentum and outputs must have their weight's shape "
                             f"{tuple(w.shape)} and device")
        if m.dtype is not torch.float32 or mo.dtype is not torch.float32 or wo.dtype is not w.dtype:
            raise ValueError("muon_update: momenta must be fp32 and new weights of their weight's type")
        if not all(t.is_contiguous() for t in (w, m, wo, mo)):
            raise ValueError("muon_update: weights, momenta and outputs must be contiguous")
    new = {}
    for k, pair in enumerate(zip(*out)):
        for t in pair:
            if new.setdefault(t.data_ptr(), k) != k or pair[0].data_ptr() == pair[1].data_ptr():
                raise ValueError("muon_update: a tensor is written twice")
    for k, (w, g, m, wo, mo) in enumerate(zip(*lists)):
        for t, own in ((w, wo), (m, mo), (g, None)):
            if t.data_ptr() in new and (own is None or new[t.data_ptr()] != k or t.data_ptr() != own.data_ptr()):
                raise ValueError("muon_update: an output is another tensor's input")


@torch.no_grad()
def muon_update(weights, grads, momenta, lr: float, momentum: float = 0.95, nesterov: bool = True,
                weight_decay: float = 0.0, steps: int = 5, eps: float = 1e-7, coefficients=COEFFICIENTS,
                scale: str = "aspect", out=None) -> None:
    """One Muon step on lists of matrices: for each weight ``W [m, n]`` (fp32 or bf16), gradient ``G`` (fp32 or bf16) and
    momentum ``M`` (fp32),

        M <- momentum M + (1 - momentum) G
        U  = (1 - momentum) G + momentum M   (nesterov; else M)
        W <- (1 - lr weight_decay) W - lr s orthogonalize(U)

    with ``s = sqrt(max(1, m / n))`` (``scale="aspect"``) or ``0.2 sqrt(max(m, n))`` (``"rms"``: the size of an AdamW
    update).  Weights and momenta change in place, or ``out = (new weights, new momenta)`` receives them.  Matrices of
    one shape share launches.  ``lr`` is a number: a captured graph keeps it.  GPU only."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    out = (weights, momenta) if out is None else tuple(list(v) for v in out)
    if len(out) != 2:
        raise ValueError("muon_update: out must be (new weights, new momenta)")
    for name, v in (("lr", lr), ("momentum", momentum), ("weight_decay", weight_decay)):
        if not isinstance(v, Real):
            raise ValueError(f"muon_update: {name} must be a number, got {type(v).__name__}")
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f"muon_update: momentum {momentum} outside [0, 1)")
    if scale not in SCALES:
        raise ValueError(f"muon_update: scale must be one of {SCALES}, got {scale!r}")
    _check_numbers("muon_update", steps, eps, coefficients)
    _check_update(weights, grads, momenta, out)
    L.require_gpu(*weights)
    groups: dict = {}
    for row in zip(weights, grads, momenta, *out):
        groups.setdefault((tuple(row[0].shape), row[0].dtype, row[1].dtype, row[0].device), []).append(row)
    from .ops import _call
    for (shape, w_dtype, g_dtype, dev), rows in groups.items():
        cfg = _config(1, shape, g_dtype, w_dtype, steps, coefficients, eps, nesterov, float(momentum),
                      1.0 - lr * weight_decay, lr * _update_scale(scale, *shape))
        most = _chunk(cfg)
        with L.on_device(dev):
            for i in range(0, len(rows), most):
                part = rows[i:i + most]
                cfg.batch = len(part)
                n = _bytes(cfg)
                ws = torch.empty((n,), dtype=torch.uint8, device=dev)
                g = [r[1].contiguous() for r in part]
                w, m, wo, mo = (_pointers([r[k].data_ptr() for r in part]) for k in (0, 2, 3, 4))
                _call("llattn_muon_update", ctypes.byref(cfg), _pointers([t.data_ptr() for t in g]), m, w, mo, wo,
                      ws.data_ptr(), n, L.stream_ptr(dev), work=12 * len(part) * shape[0] * shape[1])
    _written([t for v in out for t in v])


class Muon(torch.optim.Optimizer):
    """Muon on matrices: :func:`muon_update` of every parameter that has a gradient, momenta kept in fp32."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, eps: float = 1e-7, coefficients=COEFFICIENTS, scale: str = "aspect") -> None:
        if scale not in SCALES:
            raise ValueError(f"Muon: scale must be one of {SCALES}, got {scale!r}")
        _check_numbers("Muon", steps, eps, coefficients)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      eps=eps, coefficients=tuple(coefficients), scale=scale))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2:
                    raise ValueError(f"Muon takes matrices, got a parameter of shape {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            _muon_group(group, self.state)
        return loss


def _muon_group(group, state) -> None:
    params = [p for p in group["params"] if p.grad is not None]
    for p in params:
        buf = state[p].get("momentum_buffer")
        if buf is None:
            state[p]["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        elif buf.dtype is not torch.float32:  # load_state_dict gives a state its parameter's type
            state[p]["momentum_buffer"] = buf.float()
    muon_update(params, [p.grad for p in params], [state[p]["momentum_buffer"] for p in params],
                **{k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "eps", "coefficients", "scale")})


class MuonAdamW(torch.optim.Optimizer):
    """Muon for ``matrices``, AdamW for the other parameter groups, as one optimiser: one list of groups, one state.
    The matrices are the first group."""

    def __init__(self, matrices, others, muon: dict | None = None, **adamw) -> None:
        matrices, others = list(matrices), list(others)
        self._muon = Muon(matrices, **(muon or {}))
        self._adamw = torch.optim.AdamW(others, **adamw)
        groups = [dict(g) for g in self._muon.param_groups + self._adamw.param_groups]
        super().__init__(groups, {})

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        _muon_group(self.param_groups[0], self.state)
        # the groups and the state are this optimiser's own (schedulers and load_state_dict act on them)
        self._adamw.param_groups, self._adamw.state = self.param_groups[1:], self.state
        self._adamw.step()
        return loss
