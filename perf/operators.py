"""The loss and the update of a training step as cases to time and to check.

A case names an operator and its sizes:

* ``head``  softmax cross entropy of ``h W^T`` over a vocabulary: the loss of each row (evaluation), or the mean loss
  with the gradients of ``h`` and ``W`` (training); ``llattn_amd.xent.piecewise_head_loss``;
* ``orth``  Newton-Schulz orthogonalisation of a batch of matrices; ``llattn_amd.muon.orthogonalize``;
* ``muon``  momentum, orthogonalisation and weight update of a list of matrices; ``llattn_amd.muon.muon_update``.

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
IGNORE = -100

# the quintic Newton-Schulz iteration and the optimiser's constants
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
NS_STEPS, NS_EPS = 5, 1e-7
LR, MU, DECAY = 0.02, 0.95, 0.1

# the matrices of one layer (qkv, latent queries, latent keys and values, latent output, output, feed-forward):
# the default configuration, and the 0.55b preset
LAYER_DEFAULT = "384x128,64x128,128x128,128x64,128x128,256x128,128x256"
LAYER_055B = "4224x1408,512x1408,1024x1408,1408x512,1408x1408,4096x1408,1408x4096"


def listed():
    return [
        # evaluation of one short sequence by a small model: launches and latency count
        dict(name="head_eval_short", kind="head", N=64, D=128, V=509, grad=False),
        # perplexity of a long document under a large vocabulary, nothing kept for a backward
        dict(name="head_eval_wide", kind="head", N=2048, D=1408, V=131072, grad=False),
        # a training step on one prompt of a ragged length, a vocabulary of odd size
        dict(name="head_step_ragged", kind="head", N=333, D=1408, V=50257, grad=True),
        # a micro-batch of the 0.55b model: two sequences of 2048 tokens, its vocabulary of 32000
        dict(name="head_step", kind="head", N=4096, D=1408, V=32000, grad=True),
        # the other preset's width, four sequences of 2048 tokens and a vocabulary of 131072: the largest
        dict(name="head_step_wide", kind="head", N=8192, D=1536, V=131072, grad=True),
        # the latent query projections of a small model's four layers: launches and latency count
        dict(name="orth_small", kind="orth", batch=4, m=64, n=128, dtype="fp32"),
        # a few matrices of odd sizes in bf16
        dict(name="orth_ragged", kind="orth", batch=3, m=333, n=1001, dtype="bf16"),
        # one feed-forward matrix of the 0.55b model by itself
        dict(name="orth_ffn", kind="orth", batch=1, m=1408, n=4096, dtype="fp32"),
        # the update of a small model: the matrices of four layers of the default configuration
        dict(name="muon_default", kind="muon", shapes=",".join([LAYER_DEFAULT] * 4), dtype="fp32"),
        # one layer's share of the 0.55b model, as a pipeline stage or a shard of the optimiser holds it
        dict(name="muon_layer", kind="muon", shapes=LAYER_055B, dtype="fp32"),
        # the feed-forward matrices of all 22 layers of the 0.55b model, one direction
        dict(name="muon_ffn", kind="muon", shapes=",".join(["4096x1408"] * 22), dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["head", "orth", "muon"])
    if kind == "head":
        D = rng.choice([64, 128, 136, 250, 256, 777, 1024, 1408, 1536])
        V = _log_int(rng, 100, 131072)
        N = _log_int(rng, 1, 8192)
        return dict(kind="head", N=N, D=D, V=V, grad=rng.random() < 0.7)
    if kind == "orth":
        m, n = _log_int(rng, 1, 2048), _log_int(rng, 1, 4096)
        most = max(1, int(2e8 // (max(m, 64) * max(n, 64))))
        return dict(kind="orth", batch=_log_int(rng, 1, min(24, most)), m=m, n=n, dtype=rng.choice(["fp32", "fp32", "bf16"]))
    shapes = []
    for _ in range(rng.randint(1, 3)):
        m, n = _log_int(rng, 16, 2048), _log_int(rng, 16, 2048)
        shapes += ["%dx%d" % ((m, n) if rng.random() < 0.5 else (n, m))] * rng.randint(1, 6)
    return dict(kind="muon", shapes=",".join(shapes), dtype=rng.choice(["fp32", "fp32", "bf16"]))


# ---------------------------------------------------------------------------
# inputs: tensors made from the seed alone
# ---------------------------------------------------------------------------

def _shapes(text):
    return [tuple(int(v) for v in s.split("x")) for s in text.split(",")]


def _normal(g, shape, std=1.0, dtype=F32):
    return (torch.randn(shape, generator=g, device=DEVICE) * std).to(dtype)


def _gradient(g, shape, dtype):
    """A matrix like a weight gradient: a few strong directions over weaker noise."""
    m, n = shape[-2:]
    k = max(1, min(m, n) // 16)
    strong = _normal(g, (*shape[:-2], m, k)) * torch.logspace(0, -2, k, device=DEVICE)
    return ((strong @ _normal(g, (*shape[:-2], k, n)) + 0.1 * _normal(g, shape)) * (1e-3 / math.sqrt(m * n))).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    state = dict(case)
    if case["kind"] == "head":
        N, D, V = case["N"], case["D"], case["V"]
        w = _normal(g, (V, D), 0.04, BF16)
        t = torch.randint(0, V, (N,), generator=g, device=DEVICE)
        # hidden states of unit scale that lean towards their target, as a trained model's do
        h = (_normal(g, (N, D)) + 2.0 / (0.04 * math.sqrt(D)) * w[t].float() / math.sqrt(D)).to(BF16)
        t = torch.where(torch.rand((N,), generator=g, device=DEVICE) < 0.03, IGNORE, t)  # padding between documents
        state.update(h=h.requires_grad_(case["grad"]), w=w.requires_grad_(case["grad"]), t=t)
    elif case["kind"] == "orth":
        state.update(x=_gradient(g, (case["batch"], case["m"], case["n"]), DTYPES[case["dtype"]]))
    else:
        dt = DTYPES[case["dtype"]]
        shapes = _shapes(case["shapes"])
        state.update(w=[_normal(g, s, 0.02, dt) for s in shapes], g=[_gradient(g, s, dt) for s in shapes],
                     m=[_gradient(g, s, F32) for s in shapes])
        # the new weights and momenta go to buffers of their own (the old ones stay for a step that is taken back)
        state.update(out=([torch.empty_like(x) for x in state["w"]], [torch.empty_like(x) for x in state["m"]]))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "local-latent-attention_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


def _own_head(s):
    from llattn_amd.xent import piecewise_head_loss
    if not s["grad"]:
        return piecewise_head_loss(s["h"], s["w"], s["t"], reduction="none")
    loss = piecewise_head_loss(s["h"], s["w"], s["t"])
    return (loss.detach(), *torch.autograd.grad(loss, (s["h"], s["w"])))


def _plain_head(s):
    h, w, t = s["h"].detach().float(), s["w"].detach().float(), s["t"]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    e = (logits - top).exp_()
    total = e.sum(1, keepdim=True)
    rows = torch.arange(len(t), device=t.device)
    keep = t != IGNORE
    at = t.clamp(min=0)
    loss = torch.where(keep, (top + total.log()).squeeze(1) - logits[rows, at], 0.0)
    if not s["grad"]:
        return loss
    scale = 1.0 / keep.sum().float()
    e.div_(total)
    e[rows, at] -= 1.0
    e.mul_(torch.where(keep, scale, 0.0).unsqueeze(1))  # nothing from rows that do not count
    return loss.sum() * scale, (e @ w).to(BF16), (e.t().contiguous() @ h).to(BF16)


def _plain_orth(x):
    """[.., m, n] in the type of x: 32 bits from run(), 64 from exact()."""
    flip = x.shape[-2] > x.shape[-1]
    if flip:
        x = x.mT.contiguous()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    for _ in range(NS_STEPS):
        a = x @ x.mT.contiguous()
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    return x.mT.contiguous() if flip else x


def _plain_muon(w, g, m):
    m = MU * m + (1 - MU) * g.float()
    o = _plain_orth((1 - MU) * g.float() + MU * m)
    scale = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
    return ((1 - LR * DECAY) * w.float() - LR * scale * o).to(w.dtype), m


def run(state):
    if own:
        _package()
        if state["kind"] == "head":
            return _own_head(state)
        from llattn_amd.muon import muon_update, orthogonalize
        if state["kind"] == "orth":
            return orthogonalize(state["x"])
        muon_update(state["w"], state["g"], state["m"], lr=LR, momentum=MU, weight_decay=DECAY, out=state["out"])
        return state["out"]
    if state["kind"] == "head":
        return _plain_head(state)
    if state["kind"] == "orth":
        return _plain_orth(state["x"].float()).to(state["x"].dtype)
    pairs = [_plain_muon(*x) for x in zip(state["w"], state["g"], state["m"])]
    return [p[0] for p in pairs], [p[1] for p in pairs]


def _orth_flops(m, n):
    m, n = min(m, n), max(m, n)
    return NS_STEPS * (3.0 * m * m * n + m ** 3)  # x x^T and a a are symmetric: half of each


def work(case):
    if case["kind"] == "head":
        N, D, V = case["N"], case["D"], case["V"]
        if not case["grad"]:
            return {"bytes": 2 * (N + V) * D + 12 * N, "flops": 2.0 * N * D * V}
        return {"bytes": 4 * (N + V) * D + 8 * N + 4, "flops": 6.0 * N * D * V}
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "orth":
        m, n = case["m"], case["n"]
        return {"bytes": 2 * size * case["batch"] * m * n, "flops": case["batch"] * _orth_flops(m, n)}
    shapes = _shapes(case["shapes"])
    return {"bytes": sum((3 * size + 8) * m * n for m, n in shapes), "flops": sum(_orth_flops(m, n) for m, n in shapes)}


# ---------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------

def _exact_polar(x):
    """The iteration on the smaller side's Gram matrix: x <- (a + b g + c g^2) x, g = x x^T or x^T x."""
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + NS_EPS)
    wide = x.shape[-2] <= x.shape[-1]
    eye = torch.eye(min(x.shape[-2:]), dtype=F64, device=x.device)
    for _ in range(NS_STEPS):
        xt = x.mT.contiguous()
        gram = torch.matmul(x, xt) if wide else torch.matmul(xt, x)
        p = NS_A * eye + torch.matmul(NS_B * eye + NS_C * gram, gram)
        x = torch.matmul(p, x) if wide else torch.matmul(x, p)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "head":
        h, w, t = s["h"].detach().to(F64), s["w"].detach().to(F64), s["t"]
        logits = torch.matmul(h, w.t())
        logp = logits - torch.logsumexp(logits, 1, keepdim=True)
        del logits
        keep = t != IGNORE
        at = t.clamp(min=0).unsqueeze(1)
        loss = torch.where(keep, -logp.gather(1, at).squeeze(1), torch.zeros((), dtype=F64, device=t.device))
        if not case["grad"]:
            return loss
        d = logp.exp_()
        d.scatter_add_(1, at, torch.full_like(at, -1, dtype=F64))
        d = torch.where(keep.unsqueeze(1), d / keep.sum(), torch.zeros((), dtype=F64, device=t.device))
        return loss.sum() / keep.sum(), torch.matmul(d, w), torch.matmul(d.t(), h)
    if case["kind"] == "orth":
        return _exact_polar(s["x"].to(F64))
    ws, ms = [], []
    for w, g, m in zip(s["w"], s["g"], s["m"]):
        g = g.to(F64)
        m = m.to(F64) + (1 - MU) * (g - m.to(F64))
        o = _exact_polar(g + MU * (m - g))
        k = max(1.0, w.shape[0] / w.shape[1]) ** 0.5
        ws.append(w.to(F64) * (1 - LR * DECAY) - LR * k * o)
        ms.append(m)
    return ws, ms
