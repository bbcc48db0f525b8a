"""Orthogonalised weight updates on the gfx950 kernels (``llattn_orthogonalize`` and ``llattn_muon_update`` of
``include/llattn_train.h``).

:func:`orthogonalize` runs the quintic Newton-Schulz iteration ``X <- a X + (b A + c A A) X``, ``A = X X^T``, on a batch
of matrices; :func:`muon_update` is one step of the Muon optimiser on a list of weights (momentum, orthogonalisation,
decay and update), and :class:`Muon` / :class:`MuonAdamW` are the optimisers made of it
(:func:`llattn_amd.lm.make_optimizer` builds the second for the language model).

The iteration runs at about fp32's precision whatever the tensors' type: its matrices are held as two fp16 halves and
multiplied on the fp16 matrix cores; those of at most 16 rows or columns are taken in 64 bits.
"""
from __future__ import annotations

import copy
import ctypes
import math
from array import array
from numbers import Real

import torch

from . import _lib as L

# coefficients that raise small singular values fastest while those near 1 stay within about 0.7 to 1.2
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
SCALES = ("aspect", "rms")
WORKSPACE_BYTES = 4 << 30  # matrices are taken together up to this
MOST = 32768  # rows and columns of a matrix


TILES = 0  # workgroups of the products: the library's choice (llattn_muon_cfg.tiles)


def _config(steps, coefficients, eps, nesterov=False, mu=0.0):
    # the library takes eps in fp32, where one below 2^-149 would be none at all
    return L.LlattnMuonCfg(0, int(steps), int(nesterov), TILES, *[float(v) for v in coefficients], eps and max(float(eps), 2.0 ** -149), mu)


def _bytes(cfg, groups) -> int:
    n = L.load().llattn_muon_bytes(ctypes.byref(cfg), groups)
    if n == 0:
        L.check(L.ERR_SHAPE, "llattn_muon_bytes")
    return n


def _pointers(values):
    """An array of pointers from data pointers (by way of an array of numbers, a tenth of ctypes' own time)."""
    return (ctypes.c_void_p * len(values)).from_buffer(array("Q", [v or 0 for v in values]))


def _padded(shape) -> int:
    """Bytes of workspace that a matrix takes."""
    m, n = (v + -v % 64 for v in sorted(shape))
    return 8 * m * (n + m)


def _calls(kinds):
    """``kinds``: a list of (shape, count) of alike matrices in a row.  Cuts it into calls: lists of (kind, first, count)
    of at most 16 kinds, 128 matrices and the workspace's bytes (one matrix at least)."""
    call, held, room = [], 0, WORKSPACE_BYTES
    for k, (shape, count) in enumerate(kinds):
        each, first = _padded(shape), 0
        while first < count:
            n = min(count - first, L.MUON_BATCH - held, max(room // each, 0 if call else 1))
            if n == 0 or len(call) == L.MUON_GROUPS:
                yield call
                call, held, room = [], 0, WORKSPACE_BYTES
                continue
            call.append((k, first, n))
            held, room, first = held + n, room - n * each, first + n
    if call:
        yield call


def _launch(name, cfg, groups, device, *pointers, work):
    """One call of ``name`` with its workspace."""
    table = (L.LlattnMuonGroup * len(groups))(*groups)
    cfg.n_groups = len(groups)
    n = _bytes(cfg, table)
    ws = torch.empty((n,), dtype=torch.uint8, device=device)
    from .ops import _call
    with L.on_device(device):
        _call(name, ctypes.byref(cfg), table, *[_pointers(p) for p in pointers], ws.data_ptr(), n, L.stream_ptr(device), work=work)


def _check_numbers(who, steps, eps, coefficients):
    if not isinstance(steps, Real) or not 1 <= steps < 2 ** 31 or int(steps) != steps:
        raise ValueError(f"{who}: steps must be a positive whole number, got {steps}")
    if not eps >= 0:
        raise ValueError(f"{who}: eps must not be negative, got {eps}")
    if len(coefficients) != 3:
        raise ValueError(f"{who}: three coefficients expected, got {coefficients}")


def _apart(src: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """``src`` (contiguous, as large as ``out``), as a copy where it lies across ``out``: a matrix is written while others are
    still read, and only its own place is safe."""
    off = src.data_ptr() - out.data_ptr()
    return src.clone() if 0 < abs(off) < out.numel() * out.element_size() else src


def orthogonalize(x: torch.Tensor, steps: int = 5, eps: float = 1e-7, coefficients=COEFFICIENTS,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Newton-Schulz iteration on every matrix of ``x [..., m, n]`` (fp32 or bf16; any strides), from ``X = x / (|x|_F +
    eps)``: towards the orthogonal factor of ``x``'s polar decomposition.  Returns ``x``'s type and shape; ``out``
    (contiguous, may be ``x`` or overlap it) receives the result.  A zero matrix stays zero (``eps`` > 0); one that holds an infinity or NaN gives
    NaN throughout.  Not differentiable.  GPU only."""
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: expected [..., m, n], got shape {tuple(x.shape)}")
    _check_numbers("orthogonalize", steps, eps, coefficients)
    L.dtype_code(x.dtype)
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("orthogonalize has no gradient: call it under torch.no_grad() or on a detached tensor")
    L.refuse_tangents("orthogonalize", (x,))
    L.require_gpu(x)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
        raise ValueError("orthogonalize: out must be contiguous, of x's shape, type and device")
    m, n = x.shape[-2:]
    if x.numel() == 0:
        return out
    src = _apart(x.detach().contiguous(), out)
    each, dt = m * n * x.element_size(), L.dtype_code(x.dtype)
    cfg = _config(steps, coefficients, eps)
    for call in _calls([((m, n), x.numel() // (m * n))]):
        (_, first, k), = call
        at = range(first * each, (first + k) * each, each)
        _launch("llattn_orthogonalize", cfg, [L.LlattnMuonGroup(k, m, n, dt, dt, 0.0, 0.0)], x.device,
                [src.data_ptr() + i for i in at], [out.data_ptr() + i for i in at], work=2 * k * each)
    _written([out])
    return out


def _written(tensors) -> None:
    """Tensors that a kernel has written in place, for autograd's checks of what it saved."""
    torch.autograd.graph.increment_version(tensors)


def _update_scale(scale: str, rows: int, cols: int) -> float:
    return math.sqrt(max(1.0, rows / cols)) if scale == "aspect" else 0.2 * math.sqrt(max(rows, cols))


def _rows(weights, grads, momenta, out):
    """The checked matrices by device and kind (shape, weight's type, gradient's type), each as data pointers (g, m, w, m_out,
    w_out); and what has to live until the launch."""
    lists = [weights, grads, momenta, *out]
    if len({len(v) for v in lists}) != 1:
        raise ValueError(f"muon_update: lists of different lengths ({', '.join(str(len(v)) for v in lists)})")
    f32, types = torch.float32, (torch.float32, torch.bfloat16)
    devices, kept, inputs, new = {}, [], [], []
    for w, g, m, wo, mo in zip(*lists):
        shape, dev, w_dtype, g_dtype = w.shape, w.get_device(), w.dtype, g.dtype
        if len(shape) != 2 or 0 in shape:
            raise ValueError(f"muon_update: weights must be non-empty matrices, got shape {tuple(shape)}")
        if w_dtype not in types or g_dtype not in types:
            raise ValueError(f"muon_update: weights and gradients must be fp32 or bf16, got {w_dtype} and {g_dtype}")
        same = g.shape == shape and m.shape == shape and g.get_device() == dev and m.get_device() == dev
        typed = m.dtype is f32
        plain = w.is_contiguous() and m.is_contiguous()
        pw, pm = w.data_ptr(), m.data_ptr()
        pwo, pmo = pw, pm
        if wo is not w:
            same = same and wo.shape == shape and wo.get_device() == dev
            typed, plain, pwo = typed and wo.dtype is w_dtype, plain and wo.is_contiguous(), wo.data_ptr()
        if mo is not m:
            same = same and mo.shape == shape and mo.get_device() == dev
            typed, plain, pmo = typed and mo.dtype is f32, plain and mo.is_contiguous(), mo.data_ptr()
        if not same:
            raise ValueError(f"muon_update: gradient, momentum and outputs must have their weight's shape {tuple(shape)} "
                             "and device")
        if not typed:
            raise ValueError("muon_update: momenta must be fp32 and new weights of their weight's type")
        if not plain:
            raise ValueError("muon_update: weights, momenta and outputs must be contiguous")
        if not g.is_contiguous():
            g = g.contiguous()
            kept.append(g)
        pg = g.data_ptr()
        inputs.append(pg)
        if pwo != pw:
            inputs.append(pw)
        if pmo != pm:
            inputs.append(pm)
        new += (pwo, pmo)
        if dev not in devices:
            devices[dev] = w.device, {}
        kinds, key = devices[dev][1], (shape, w_dtype, g_dtype)
        if key in kinds:
            kinds[key].append((pg, pm, pw, pmo, pwo))
        else:
            if max(shape) > MOST:  # before any launch: a list may take several calls, and those before would have updated
                raise ValueError(f"muon_update: at most {MOST} rows and columns, got shape {tuple(shape)}")
            kinds[key] = [(pg, pm, pw, pmo, pwo)]
    written = set(new)
    if len(written) != len(new):
        raise ValueError("muon_update: a tensor is written twice")
    if not written.isdisjoint(inputs):
        raise ValueError("muon_update: an output is another tensor's input")
    return list(devices.values()), kept


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
    update).  Weights and momenta change in place, or ``out = (new weights, new momenta)`` receives them; tensors that are
    not the same must not overlap.  ``momentum``, ``eps`` and the coefficients count as fp32 holds them (1 - momentum is
    that of the fp32 value).  The matrices of a call share launches, whatever their shapes.  ``lr`` is a number: a captured
    graph keeps it.  GPU only."""
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
    devices, kept = _rows(weights, grads, momenta, out)
    L.refuse_tangents("muon_update", weights + grads + momenta)
    L.require_gpu(*weights)
    cfg = _config(steps, coefficients, eps, nesterov, float(momentum))
    keep = 1.0 - lr * weight_decay
    for device, kinds in devices:
        keys = list(kinds)
        for call in _calls([(k[0], len(kinds[k])) for k in keys]):
            groups, part = [], []
            for k, first, n in call:
                shape, w_dtype, g_dtype = key = keys[k]
                groups.append(L.LlattnMuonGroup(n, *shape, L.dtype_code(g_dtype), L.dtype_code(w_dtype), keep,
                                                lr * _update_scale(scale, *shape)))
                part += kinds[key][first:first + n]
            _launch("llattn_muon_update", cfg, groups, device, *zip(*part),
                    work=sum(12 * q.batch * q.rows * q.cols for q in groups))
    _written([t for v in out for t in v])


class Muon(torch.optim.Optimizer):
    """Muon on matrices: :func:`muon_update` of every parameter that has a gradient, momenta kept in fp32 (and loaded in
    fp32).  A step can be captured into a graph once the momenta exist."""

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

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        _restore_momenta(self, state_dict)


def _restore_momenta(optimizer, state_dict) -> None:
    """fp32 momenta from ``state_dict``: Optimizer.load_state_dict gives a state its parameter's type, and bf16 parameters'
    momenta would lose 16 bits."""
    ids = [i for g in state_dict["param_groups"] for i in g["params"]]
    for i, p in zip(ids, [p for g in optimizer.param_groups for p in g["params"]]):
        buf = state_dict["state"].get(i, {}).get("momentum_buffer")
        if buf is not None:
            optimizer.state[p]["momentum_buffer"] = buf.detach().to(device=p.device, dtype=torch.float32, copy=True)


def _muon_group(group, state) -> None:
    params = [p for p in group["params"] if p.grad is not None]
    for p in params:
        buf = state[p].get("momentum_buffer")
        if buf is None:
            if p.is_cuda and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("Muon: momenta must exist before a step is captured (a replay would begin them at zero each "
                                   "time): take one step first, or load a state")
            state[p]["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
    muon_update(params, [p.grad for p in params], [state[p]["momentum_buffer"] for p in params],
                **{k: group[k] for k in ("lr", "momentum", "nesterov", "weight_decay", "steps", "eps", "coefficients", "scale")})


class MuonAdamW(torch.optim.Optimizer):
    """Muon for ``matrices`` (parameters or groups of them), AdamW for the other parameter groups, as one optimiser: one
    list of groups, the matrices' first, and one state.  Groups added later are AdamW's."""

    def __init__(self, matrices, others, muon: dict | None = None, **adamw) -> None:
        matrices, others = list(matrices), list(others)
        matrix_groups = Muon(matrices, **(muon or {})).param_groups
        self._adamw = torch.optim.AdamW(others, **adamw)
        groups = [dict(g) for g in matrix_groups + self._adamw.param_groups]
        super().__init__(groups, dict(self._adamw.defaults))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # the groups and the state are this optimiser's own (schedulers and load_state_dict act on them)
        for group in self.param_groups:
            if "coefficients" in group:  # Muon's, as no group of AdamW's has them
                _muon_group(group, self.state)
        self._adamw.param_groups = [g for g in self.param_groups if "coefficients" not in g]
        self._adamw.state = self.state
        self._adamw.step()
        return loss

    def __getstate__(self) -> dict:
        # Optimizer's own keeps groups, state and defaults, for copies and pickles.  The AdamW inside goes along without
        # parameters or state: step() hands it this optimiser's.
        inner = copy.copy(self._adamw)
        inner.param_groups, inner.state = [], {}
        return {**super().__getstate__(), "_adamw": inner}

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)
        _restore_momenta(self, state_dict)
