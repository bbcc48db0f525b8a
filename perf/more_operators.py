"""The ends and the feed-forward of a training step as cases to time and to check.

A case names an operator and its sizes:

* ``embed``  token rows, scaled, plus position rows; in training with the gradients of both tables, the tokens' summed
  in the order of the sorted tokens; ``llattn_amd.embed``;
* ``ffn``    gated feed-forward ``w2(act(w1 x) * w3 x)``; in training with the gradients of ``x`` and the three weights;
  ``llattn_amd.gated_feed_forward``;
* ``clip``   the norm over a list of gradients of any shapes, and the gradients scaled to a largest norm;
  ``llattn_amd.clip_grad_norm``.

``listed()`` gives the cases, ``draw(rng)`` one more of the same ranges; ``prepare`` makes what a program holds
before the call, ``run`` is one pass, ``exact`` the same values in float64.  With ``own`` false ``run`` computes the
operators from elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
DTYPES = {"bf16": BF16, "fp32": F32}
DEVICE = "cuda"

# gradients of one layer: matrices, their biases, norms and gate vectors (default configuration; 0.55b preset)
LAYER_DEFAULT = ("384x128,384,64x128,64,128x128,128,128x64,128,128x128,128,256x128,256,128x256,128,128,128,32,32")
LAYER_055B = ("4224x1408,4224,512x1408,512,1024x1408,1024,1408x512,1408,1408x1408,1408,4096x1408,4096,1408x4096,1408,"
              "1408,1408,88,88")
EPS = 1e-6  # beside the norm, as trainers have it


def listed():
    return [
        # one decoding step of 16 sequences, each at its own position, a half-precision model: latency
        dict(name="embed_token", kind="embed", B=16, T=1, V=32000, P=2048, D=1408, dtype="bf16", scale=1.0,
             positions=True, grad=False),
        # a training step of a small model: two sequences of a ragged length, default width
        dict(name="embed_small", kind="embed", B=2, T=333, V=509, P=1024, D=128, dtype="fp32", scale=1.0,
             positions=False, grad=True),
        # documents packed into rows (positions start anew in each), rows scaled by sqrt(D), a vocabulary of odd size
        dict(name="embed_packed", kind="embed", B=4, T=2048, V=50257, P=2048, D=1536, dtype="bf16", scale=1536 ** 0.5,
             positions=True, grad=True),
        # the training step of the 0.55b model: 16 sequences of 2048 tokens
        dict(name="embed_step", kind="embed", B=16, T=2048, V=32000, P=2048, D=1408, dtype="fp32", scale=1.0,
             positions=False, grad=True),
        # one token through a 0.55b layer's feed-forward: the weights' bytes count
        dict(name="ffn_token", kind="ffn", N=1, D=1408, F=4096, act="silu", grad=False),
        # a training step of a small model, default widths: launches and latency count
        dict(name="ffn_small", kind="ffn", N=640, D=128, F=256, act="gelu", grad=True),
        # a training step on one prompt of a ragged length
        dict(name="ffn_ragged", kind="ffn", N=333, D=1408, F=4096, act="silu", grad=True),
        # evaluation of a long document
        dict(name="ffn_eval", kind="ffn", N=8192, D=1408, F=4096, act="silu", grad=False),
        # four sequences of 2048 tokens at the other preset's width: the largest
        dict(name="ffn_step", kind="ffn", N=8192, D=1536, F=4096, act="silu", grad=True),
        # the gradients of four layers of the default configuration: launches and latency count
        dict(name="clip_default", kind="clip", shapes=",".join([LAYER_DEFAULT] * 4 + ["128x128,1024x128,128"]),
             dtype="fp32", active=True),
        # one layer's share of the 0.55b model (a pipeline stage), gradients in bf16
        dict(name="clip_layer", kind="clip", shapes=LAYER_055B, dtype="bf16", active=True),
        # all gradients of the 0.55b model: 22 layers, the embeddings and the last norm
        dict(name="clip_model", kind="clip", shapes=",".join([LAYER_055B] * 22 + ["32000x1408,2048x1408,1408"]),
             dtype="fp32", active=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "ffn", "clip"])
    if kind == "embed":
        D = rng.choice([64, 128, 136, 250, 256, 777, 1024, 1408, 1536])
        T = _log_int(rng, 1, 2048)
        B = _log_int(rng, 1, max(1, min(64, 32768 // T)))
        return dict(kind="embed", B=B, T=T, V=_log_int(rng, 100, 65536), P=T + rng.choice([0, 0, 1, 100, 1000]), D=D,
                    dtype=rng.choice(["fp32", "bf16"]), scale=rng.choice([1.0, D ** 0.5]), positions=rng.random() < 0.5,
                    grad=rng.random() < 0.7)
    if kind == "ffn":
        F = _log_int(rng, 64, 4096)
        return dict(kind="ffn", N=_log_int(rng, 1, 8192), D=rng.choice([64, 128, 136, 250, 256, 777, 1024, 1408, 1536]),
                    F=F if rng.random() < 0.2 else max(64, F // 8 * 8), act=rng.choice(["silu", "silu", "gelu"]),
                    grad=rng.random() < 0.6)
    shapes = []
    for _ in range(rng.randint(1, 40)):
        if rng.random() < 0.4:
            s = "%d" % _log_int(rng, 1, 5000)
        else:
            s = "%dx%d" % (_log_int(rng, 2, 4096), _log_int(rng, 2, 1536))
        shapes += [s] * rng.randint(1, 8)
    return dict(kind="clip", shapes=",".join(shapes), dtype=rng.choice(["fp32", "fp32", "bf16", "mixed"]),
                active=rng.random() < 0.7)


# ---------------------------------------------------------------------------
# inputs: tensors made from the seed alone
# ---------------------------------------------------------------------------

def _shapes(text):
    return [tuple(int(v) for v in s.split("x")) for s in text.split(",")]


def _numel(shape):
    return math.prod(shape)


def _types(case):
    """The type of each gradient; "mixed": matrices in bf16, vectors in fp32."""
    if case["dtype"] != "mixed":
        return [DTYPES[case["dtype"]]] * len(_shapes(case["shapes"]))
    return [BF16 if len(s) == 2 else F32 for s in _shapes(case["shapes"])]


def _normal(g, shape, std=1.0, dtype=F32):
    return (torch.randn(shape, generator=g, device=DEVICE) * std).to(dtype)


def _tokens(g, shape, V):
    """Tokens numbered by their frequency, which falls as 1 / rank: the first makes up log 2 / log V of a text."""
    u = torch.rand(shape, generator=g, device=DEVICE, dtype=F64)
    return (torch.exp(u * math.log(V + 1)).floor().to(torch.int64) - 1).clamp_(0, V - 1)


def _document_positions(g, B, T):
    """Positions that start anew where a document begins (about every 400 tokens)."""
    t = torch.arange(T, device=DEVICE).expand(B, T)
    begins = torch.rand((B, T), generator=g, device=DEVICE) < 1 / 400
    return t - torch.where(begins, t, 0).cummax(1).values


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    state = dict(case)
    if case["kind"] == "embed":
        B, T, V, P, D, dt = *(case[k] for k in "BTVPD"), DTYPES[case["dtype"]]
        pos = None
        if case["positions"]:
            pos = torch.randint(0, P, (B, 1), generator=g, device=DEVICE) if T == 1 else _document_positions(g, B, T)
        state.update(ids=_tokens(g, (B, T), V), pos=pos, w=_normal(g, (V, D), 0.02, dt).requires_grad_(case["grad"]),
                     p=_normal(g, (P, D), 0.02, dt).requires_grad_(case["grad"]),
                     dy=_normal(g, (B, T, D), 1e-3, dt) if case["grad"] else None)
    elif case["kind"] == "ffn":
        N, D, F = case["N"], case["D"], case["F"]
        layers = []
        for n_in, n_out in ((D, F), (D, F), (F, D)):  # w1, w3, w2
            m = torch.nn.Linear(n_in, n_out, bias=False, device="meta", dtype=BF16)
            m.weight = torch.nn.Parameter(_normal(g, (n_out, n_in), 1 / math.sqrt(n_in), BF16), requires_grad=case["grad"])
            layers.append(m)
        state.update(x=_normal(g, (N, D), 1.0, BF16).requires_grad_(case["grad"]), layers=layers,
                     dy=_normal(g, (N, D), 1e-3, BF16) if case["grad"] else None)
    else:
        # gradients of one layer differ in size from those of the next
        grads = [_normal(g, s, 1e-4 * math.exp(math.sin(i)), t)
                 for i, (s, t) in enumerate(zip(_shapes(case["shapes"]), _types(case)))]
        norm = math.sqrt(sum(1e-8 * math.exp(2 * math.sin(i)) * _numel(s) for i, s in enumerate(_shapes(case["shapes"]))))
        # the clipped gradients go to a flat buffer for each type, as a collective takes them (the raw ones stay for
        # statistics or a step taken back)
        flat = {t: torch.empty(sum(x.numel() for x in grads if x.dtype is t), device=DEVICE, dtype=t)
                for t in (F32, BF16) if any(x.dtype is t for x in grads)}
        out, used = [], dict.fromkeys(flat, 0)
        for x in grads:
            out.append(flat[x.dtype][used[x.dtype]:used[x.dtype] + x.numel()].view(x.shape))
            used[x.dtype] += x.numel()
        state.update(g=grads, out=out, flat=list(flat.values()), most=norm * (0.3 if case["active"] else 3.0))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "local-latent-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


def _own(s):
    _package()
    import llattn_amd
    if s["kind"] == "clip":
        return llattn_amd.clip_grad_norm(s["g"], s["most"], out=s["out"]), *s["flat"]
    if s["kind"] == "embed":
        y = llattn_amd.embed(s["ids"], s["w"], s["p"], positions=s["pos"], scale=s["scale"])
        leaves = (s["w"], s["p"])
    else:
        y = llattn_amd.gated_feed_forward(s["x"], *s["layers"], act=s["act"])
        leaves = (s["x"], *(m.weight for m in s["layers"]))
    return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"])) if s["grad"] else y


def _plain_embed(s):
    w, p, ids = s["w"].detach(), s["p"].detach(), s["ids"]
    pos = torch.arange(ids.shape[1], device=ids.device).expand_as(ids) if s["pos"] is None else s["pos"]
    y = (w[ids].float() * s["scale"] + p[pos].float()).to(w.dtype)
    if not s["grad"]:
        return y
    dy = s["dy"].flatten(0, 1).float()
    dw = torch.zeros(w.shape, device=w.device).index_add_(0, ids.flatten(), dy).mul_(s["scale"]).to(w.dtype)
    if s["pos"] is None:
        dp = torch.zeros(p.shape, device=w.device)
        dp[:ids.shape[1]] = s["dy"].float().sum(0)
    else:
        dp = torch.zeros(p.shape, device=w.device).index_add_(0, pos.flatten(), dy)
    return y, dw, dp.to(p.dtype)


def _plain_ffn(s):
    x, dt = s["x"].detach().float(), s["x"].dtype
    w1, w3, w2 = (m.weight.detach().float() for m in s["layers"])
    a, u = x @ w1.t(), x @ w3.t()
    if s["act"] == "silu":
        gate = 1 / (1 + (-a).exp())
        act = a * gate
    else:
        gate = 0.5 * (1 + torch.erf(a * math.sqrt(0.5)))
        act = a * gate
    h = act * u
    y = (h @ w2.t()).to(dt)
    if not s["grad"]:
        return y
    dy = s["dy"].float()
    slope = gate + act * (1 - gate) if s["act"] == "silu" else gate + a * (-0.5 * a * a).exp() * math.sqrt(0.5 / math.pi)
    dh = dy @ w2
    du, da = dh * act, dh * u * slope
    return (y, (da @ w1 + du @ w3).to(dt), (da.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ h).to(dt))


def _plain_clip(s):
    # a model's squares: their sum in 64 bits
    norm = torch.stack([x.float().square().sum(dtype=F64) for x in s["g"]]).sum().sqrt().float()
    c = (s["most"] / (norm + EPS)).clamp(max=1.0)
    for x, o in zip(s["g"], s["out"]):
        o.copy_(x.float() * c)
    return norm, *s["flat"]


def run(state):
    if own:
        return _own(state)
    return {"embed": _plain_embed, "ffn": _plain_ffn, "clip": _plain_clip}[state["kind"]](state)


def _distinct(N, V):
    """The number of different tokens expected among N of :func:`_tokens`."""
    v = torch.arange(V, dtype=F64)
    p = torch.log((v + 2) / (v + 1)) / math.log(V + 1)
    return float((1 - torch.exp(N * torch.log1p(-p))).sum())


def work(case):
    if case["kind"] == "embed":
        B, T, V, P, D = (case[k] for k in "BTVPD")
        N, size = B * T, 2 if case["dtype"] == "bf16" else 4
        rows = _distinct(N, V) + min(P, N if case["positions"] and T == 1 else T) + N  # tokens, positions, output
        index = (16 if case["positions"] else 8) * N
        if case["grad"]:
            rows += N + V + P  # the gradient, and those of the tables
        return {"bytes": index + size * D * rows, "flops": (4.0 if case["grad"] else 2.0) * N * D}
    if case["kind"] == "ffn":
        N, D, F = case["N"], case["D"], case["F"]
        if case["grad"]:
            return {"bytes": 8 * N * D + 12 * D * F, "flops": 18.0 * N * D * F}
        return {"bytes": 4 * N * D + 6 * D * F, "flops": 6.0 * N * D * F}
    sizes = [(_numel(s), 2 if t is BF16 else 4) for s, t in zip(_shapes(case["shapes"]), _types(case))]
    return {"bytes": sum(2 * n * size for n, size in sizes) + 4, "flops": sum(3.0 * n for n, _ in sizes)}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _exact_rows(ids, dy, rows):
    """Sums of the rows of dy with the same id, as a product with the indicator of each block of ids."""
    out = torch.zeros((rows, dy.shape[1]), dtype=F64, device=dy.device)
    order = torch.argsort(ids, stable=True)
    ids, total = ids[order], torch.cumsum(torch.bincount(ids, minlength=rows), 0)
    for lo in range(0, len(ids), 4096):  # tokens in sorted order: a block of them holds few ids
        block = ids[lo:lo + 4096]
        first, last = int(block[0]), int(block[-1])
        for v0 in range(first, last + 1, 4096):
            v = torch.arange(v0, min(v0 + 4096, last + 1), device=dy.device)
            inside = (block >= v[0]) & (block <= v[-1])
            if bool(inside.any()):
                hit = (v.unsqueeze(1) == block[inside].unsqueeze(0)).to(F64)
                out[v[0]:v[-1] + 1] += torch.matmul(hit, dy[order[lo:lo + 4096][inside]].to(F64))
    assert int(total[-1]) == len(ids)
    return out


def _exact_embed(s):
    w, p, ids = s["w"].detach().to(F64), s["p"].detach().to(F64), s["ids"]
    B, T = ids.shape
    pos = s["pos"].reshape(-1) if s["pos"] is not None else torch.arange(T, device=ids.device).repeat(B)
    y = torch.add(torch.index_select(p, 0, pos), torch.index_select(w, 0, ids.reshape(-1)), alpha=s["scale"])
    y = y.reshape(B, T, -1)
    if not s["grad"]:
        return y
    dy = s["dy"].reshape(B * T, -1)
    return y, _exact_rows(ids.reshape(-1), dy, len(w)) * s["scale"], _exact_rows(pos, dy, len(p))


def _exact_ffn(s):
    x = s["x"].detach().to(F64).requires_grad_()
    w1, w3, w2 = (m.weight.detach().to(F64).requires_grad_() for m in s["layers"])
    linear = torch.nn.functional.linear
    act = torch.nn.functional.silu if s["act"] == "silu" else torch.nn.functional.gelu
    y = linear(act(linear(x, w1)) * linear(x, w3), w2)
    if not s["grad"]:
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, (x, w1, w3, w2), s["dy"].to(F64)))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "embed":
        return _exact_embed(s)
    if case["kind"] == "ffn":
        return _exact_ffn(s)
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.to(F64)) for g in s["g"]]))
    c = torch.minimum(torch.ones((), dtype=F64, device=norm.device), s["most"] / (norm + EPS))
    clipped = {}
    for g in s["g"]:
        clipped.setdefault(g.dtype, []).append(g.to(F64).reshape(-1) * c)
    return norm, *[torch.cat(clipped[t]) for t in (F32, BF16) if t in clipped]
