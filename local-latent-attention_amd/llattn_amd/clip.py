"""The norm over all gradients and their clipping on the gfx950 kernels (``llattn_grad_norm`` and ``llattn_clip_grads`` of
``include/llattn_lm.h``).

:func:`grad_norm` and :func:`clip_grad_norm` take lists of tensors; :func:`clip_grad_norm_` and
:func:`clip_grads_with_norm_` take parameters, as the trainer's ``clip_grad_norm_`` does (reference train.py:1021).  A list
of any length takes one launch per 128 tensors and pass; squares and sums are 64-bit whatever the tensors' type.
"""
from __future__ import annotations

import math
from array import array
from ctypes import c_void_p
from numbers import Real

import torch

from . import _lib as L

_CODE = {torch.float32: L.F32, torch.bfloat16: L.BF16}
_TYPES = set(_CODE)


def _flat(t: torch.Tensor):
    """``t`` as a contiguous tensor on the same memory where its elements fill one stretch of it (in any order of its axes), else
    None."""
    if t.is_contiguous():
        return t
    order = sorted(range(t.dim()), key=t.stride, reverse=True)
    t = t.permute(order)
    return t if t.is_contiguous() else None


def _refuse_sparse(who: str, tensors) -> None:
    layouts = {t.layout for t in tensors} - {torch.strided}
    if layouts:
        raise ValueError(f"{who}: gradients must be dense tensors, got {layouts.pop()}")


def _check(who: str, tensors) -> list:
    """The types of ``tensors`` (one at least), which are what the kernels take: dense (those that are not have no address, which
    :class:`_Arrays` meets), fp32 or bf16, on one GPU."""
    types = [t.dtype for t in tensors]
    if not _TYPES.issuperset(types):
        raise ValueError(f"{who}: gradients must be fp32 or bf16, got {(set(types) - _TYPES).pop()}")
    L.refuse_tangents(who, tensors)
    devices = {t.get_device() for t in tensors}
    if min(devices) < 0:
        _refuse_sparse(who, tensors)
        L.require_gpu(*tensors)
    if len(devices) > 1:
        raise ValueError(f"{who}: gradients on {len(devices)} devices")
    return types


def _whole_all(who: str, tensors) -> bool:
    """Whether all are contiguous; asked of every tensor before its layout, which only those that are not can have."""
    try:
        whole = all([t.is_contiguous() for t in tensors])
    except RuntimeError:
        whole = False
    if not whole:
        _refuse_sparse(who, tensors)
    return whole


def _addresses(who: str, tensors) -> array:
    try:
        return array("Q", [t.data_ptr() for t in tensors])
    except RuntimeError:
        _refuse_sparse(who, tensors)
        raise


class _Arrays:
    """The host arrays of a call on contiguous tensors."""

    def __init__(self, who, tensors, types):
        self.n = len(tensors)
        self.g = _addresses(who, tensors)
        self.numel = array("q", [t.numel() for t in tensors])
        self.dtype = array("i", [_CODE[types[0]]]) * self.n if types.count(types[0]) == self.n else array("i", [_CODE[t] for t in types])

    def workspace(self, device):
        n = L.load().llattn_grad_norm_bytes(self.n, _at(self.numel))
        if n == 0:
            L.check(L.ERR_SHAPE, "llattn_grad_norm_bytes")
        return torch.empty((n,), dtype=torch.uint8, device=device), n

    def bytes(self) -> int:
        from .ops import EVENT_LOG
        return 0 if EVENT_LOG is None else sum(n * (2 if d else 4) for n, d in zip(self.numel, self.dtype))


def _at(a):
    return c_void_p(a.buffer_info()[0])


def _most(who: str, max_norm) -> float:
    if not isinstance(max_norm, Real) or not max_norm >= 0:
        raise ValueError(f"{who}: max_norm must be a number that is not negative, got {max_norm!r}")
    return float(max_norm)


def _whole(t: torch.Tensor) -> torch.Tensor:
    f = _flat(t.detach())
    return t.detach().contiguous() if f is None else f


@torch.no_grad()
def grad_norm(tensors) -> torch.Tensor:
    """The 2-norm of all elements of ``tensors`` (fp32 or bf16, any shapes and strides, one device) as an fp32 scalar on
    their device; 0 on the CPU for an empty list.  GPU only."""
    tensors = list(tensors)
    if not tensors:
        return torch.zeros(())
    types, device = _check("grad_norm", tensors), tensors[0].device
    if not _whole_all("grad_norm", tensors):
        tensors = [_whole(t) for t in tensors]
    a = _Arrays("grad_norm", tensors, types)
    ws, n = a.workspace(device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    from .ops import _call
    with L.on_device(device):
        _call("llattn_grad_norm", a.n, _at(a.g), _at(a.numel), _at(a.dtype), norm.data_ptr(), ws.data_ptr(), n,
              L.stream_ptr(device), work=a.bytes())
    return norm


def _span(t: torch.Tensor):
    """(first byte, one past the last) of the memory that a tensor of one element at least lies in."""
    at = t.data_ptr()
    return at, at + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


_MEET_STEPS = 1 << 16


def _meet(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors whose spans intersect share memory, which interleaved slices of one buffer do not.

    Elements of a lie at sum x_k s_k, x_k < n_k along its axes, those of b likewise at y_k (where the elements' sizes differ, in bytes,
    with an element's own as one more axis).  With n_k - 1 - y_k in y_k's place both are sums with positive steps, and the
    question is whether their sum takes one value: by the largest step first, as often as those below can make up for.  Two that are
    not told apart in 2^16 steps (axes that interleave in no order) count as one."""
    size = a.element_size()
    goal = b.data_ptr() - a.data_ptr()
    bytewise = b.element_size() != size or goal % size != 0
    goal //= 1 if bytewise else size
    steps: dict[int, int] = {}
    for t in (a, b):
        unit = t.element_size() if bytewise else 1
        axes = [(n - 1, s * unit) for n, s in zip(t.shape, t.stride()) if n > 1 and s]
        for n, s in axes + [(unit - 1, 1)]:
            steps[s] = steps.get(s, 0) + n
            goal += n * s if t is b else 0
    order = sorted(((s, n) for s, n in steps.items() if n), reverse=True)
    rest, divisor = [0], [0]  # what the steps from the k-th on add up to at most, and what divides them; from the last
    for s, n in reversed(order):
        rest.append(rest[-1] + n * s)
        divisor.append(math.gcd(divisor[-1], s))
    rest.reverse()
    divisor.reverse()
    left = _MEET_STEPS

    def found(k, goal):
        nonlocal left
        left -= 1
        if not 0 <= goal <= rest[k]:
            return False
        if goal == 0 or left < 0:
            return True
        if goal % divisor[k]:
            return False
        s, n = order[k]
        first, last = max(0, -((rest[k + 1] - goal) // s)), min(n, goal // s)
        return any(found(k + 1, goal - x * s) for x in range(first, last + 1))
    return found(0, goal)


def _refuse_overlap(who: str, tensors, out) -> None:
    """As the C call does for contiguous tensors, which are all that it sees: what is written overlaps nothing else, neither another
    tensor that is written nor an input but its own in place."""
    written = tensors if out is None else out
    spans = [(*_span(t), i, t, True) for i, t in enumerate(written) if t.numel()]
    if out is not None:
        spans += [(*_span(t), i, t, False) for i, t in enumerate(tensors) if t.numel()]
    spans.sort(key=lambda s: s[0])
    held = []
    for span in spans:
        at, _, i, t, is_written = span
        held = [h for h in held if h[1] > at]
        for _, _, j, o, was_written in held:
            if not (is_written or was_written):
                continue
            if is_written and was_written:
                what = f"tensors {j} and {i}, which are written, overlap"
            elif i == j and t.data_ptr() == o.data_ptr() and t.stride() == o.stride():
                continue  # in place
            else:
                what = f"output {i if is_written else j} overlaps gradient {j if is_written else i}"
            if _meet(t, o):
                raise ValueError(f"{who}: {what}")
        held.append(span)


def _pairs(who: str, tensors, out):
    """Contiguous (sources, destinations) for gradients that are not all so; and (tensor, destination) pairs to be copied back."""
    src, dst, back = [], [], []
    copied = False  # the C call does not see all tensors where they lie
    for i, g in enumerate(tensors):
        g = g.detach()
        o = g if out is None else out[i].detach()
        same = o.stride() == g.stride()
        f = _flat(g) if same else None  # both in one order of the axes: that of memory
        d = _flat(o) if same else o if o.is_contiguous() else None
        if f is None or d is None:
            copied = True
            f = g.contiguous()
            if not o.is_contiguous():  # not in one stretch: scaled apart
                if torch._debug_has_internal_overlap(o) == 1:
                    raise ValueError(f"{who}: a tensor that is written holds one element in several places (strides {o.stride()})")
                d = torch.empty_like(f)
                back.append((o, d))
            else:
                d = o
        src.append(f)
        dst.append(d)
    if copied:
        _refuse_overlap(who, tensors, out)
    return src, dst, back


def _clip(who: str, tensors, out, max_norm: float, norm_in) -> torch.Tensor | None:
    """Scales ``tensors`` (one at least) into ``out`` (or in place); the norm where none is given."""
    types, device = _check(who, tensors), tensors[0].device
    if norm_in is not None and (norm_in.numel() != 1 or norm_in.dtype is not torch.float32 or norm_in.device != device):
        raise ValueError(f"{who}: the norm must be one fp32 value on {device}, got {tuple(norm_in.shape)} {norm_in.dtype} on {norm_in.device}")
    written = tensors if out is None else out
    if out is not None and ([t.shape for t in out] != [t.shape for t in tensors] or [t.dtype for t in out] != types
                            or {t.get_device() for t in out} != {device.index}):
        raise ValueError(f"{who}: outputs must have their gradients' shapes, types and device")
    src, dst, back = tensors, out, ()
    if not _whole_all(who, tensors) or out is not None and not _whole_all(who, out):
        src, dst, back = _pairs(who, tensors, out)
    a = _Arrays(who, src, types)
    o = None if dst is None else _addresses(who, dst)
    ws = norm = None
    n = 0
    if norm_in is None:
        ws, n = a.workspace(device)
        norm = torch.empty((), dtype=torch.float32, device=device)
    from .ops import _call
    with L.on_device(device):
        _call("llattn_clip_grads", a.n, _at(a.g), None if o is None else _at(o), _at(a.numel), _at(a.dtype), max_norm,
              None if norm_in is None else norm_in.data_ptr(), None if norm is None else norm.data_ptr(),
              None if ws is None else ws.data_ptr(), n, L.stream_ptr(device), work=(3 if norm_in is None else 2) * a.bytes())
    for to, d in back:
        to.copy_(d)
    torch.autograd.graph.increment_version(written)
    return norm


@torch.no_grad()
def clip_grad_norm(grads, max_norm: float, out=None) -> torch.Tensor:
    """Scales ``grads`` (tensors, fp32 or bf16) by ``min(1, max_norm / (norm + 1e-6))``, ``norm`` being their
    :func:`grad_norm`, which is returned.  In place, or into ``out`` (a list of as many tensors of the same shapes and types;
    each may be its gradient itself and overlaps nothing else).  Nothing waits for the GPU.  GPU only."""
    grads, most = list(grads), _most("clip_grad_norm", max_norm)
    if out is not None:
        out = list(out)
        if len(out) != len(grads):
            raise ValueError(f"clip_grad_norm: {len(out)} outputs for {len(grads)} gradients")
        if any([o.requires_grad for o in out]) and any(o.requires_grad and o.is_leaf for o in out):
            raise ValueError("clip_grad_norm: out holds leaves that require gradients")
    return torch.zeros(()) if not grads else _clip("clip_grad_norm", grads, out, most, None)


def _grads(parameters):
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return [g for p in parameters if (g := p.grad) is not None]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clips the gradients of ``parameters`` in place to a 2-norm of ``max_norm`` over all of them, as
    ``torch.nn.utils.clip_grad_norm_``, and returns the norm (fp32).  ``error_if_nonfinite`` waits for the norm and raises
    before anything is scaled.  Gradients are fp32 or bf16 (each once), on one GPU."""
    if float(norm_type) != 2.0:
        raise ValueError(f"clip_grad_norm_: the 2-norm only, got norm_type={norm_type}")
    most, grads = _most("clip_grad_norm_", max_norm), _grads(parameters)
    if not grads:
        return torch.zeros(())
    if not error_if_nonfinite:
        return _clip("clip_grad_norm_", grads, None, most, None)
    norm = grad_norm(grads)
    if not math.isfinite(norm.item()):
        raise RuntimeError(f"clip_grad_norm_: the gradients' norm is {norm.item()}; error_if_nonfinite=False scales them all the same")
    _clip("clip_grad_norm_", grads, None, most, norm)
    return norm


@torch.no_grad()
def clip_grads_with_norm_(parameters, max_norm: float, total_norm: torch.Tensor) -> None:
    """Clips the gradients of ``parameters`` in place by a norm that the caller has (one fp32 value on their device: say, one
    joined over the shards of a model)."""
    most, grads = _most("clip_grads_with_norm_", max_norm), _grads(parameters)
    if grads:
        _clip("clip_grads_with_norm_", grads, None, most, total_norm.detach())
