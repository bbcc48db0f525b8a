"""The piecewise head loss and the Muon update as the language model's training step runs them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
NS = (3.4445, -4.7750, 2.0315)


def _model(vocab):
    from llattn_amd.lm import build_model
    torch.manual_seed(0)
    return build_model(vocab_size=vocab, max_seq_len=128, d_model=64, n_heads=4, n_layers=2, d_ff=96, local_window=16,
                       local_block_size=32, latent_tokens=8, latent_d_model=32, latent_heads=2).to(DEV)


def _tokens(vocab, B=2, T=77):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, vocab, (B, T + 1), generator=g).to(DEV)
    return ids[:, :-1].contiguous(), ids[:, 1:].contiguous()


@pytest.mark.parametrize("vocab", [1000, 1003])
@pytest.mark.parametrize("piece", [0, 256])
def test_loss_of_the_model(vocab, piece):
    """LocalLatentLM.loss in pieces against the head in float64 on the same hidden states: the loss, the accuracy and the
    gradient of the tied weight's head part."""
    model = _model(vocab)
    x, t = _tokens(vocab)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss, metrics = model.loss(x, t, vocab_piece=piece)
        h = model.hidden(x).detach()
    w = model.lm_head.weight.detach().to(torch.bfloat16).double()
    logits = h.double().reshape(-1, 64) @ w.t()
    want = torch.nn.functional.cross_entropy(logits, t.reshape(-1))
    # 64 products and the sums of the row, in fp32
    assert abs(float(loss.detach()) - float(want)) <= 2.0 ** -24 * (2 * 72 * float((h.double().abs().reshape(-1, 64) @ w.abs().t()).max()) + 400 * 10)
    assert abs(float(metrics["eval_acc"]) - float((logits.argmax(-1) == t.reshape(-1)).double().mean())) < 1e-6
    assert float(metrics["eval_loss"]) == float(loss.detach())
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())


def _ns(x):
    a, b, c = NS
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / (x.norm() + 1e-7)
    for _ in range(5):
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if flip else x


def test_training_steps_with_both():
    """Two steps of train_step with the piecewise loss and Muon: every block matrix moves by the update that its (clipped)
    gradients give, the others as AdamW alone would move them, and a step repeats bit for bit."""
    from llattn_amd.lm import make_optimizer, train_step
    vocab = 1003
    x, t = _tokens(vocab)
    model, twin = _model(vocab), _model(vocab)
    opt, opt2 = make_optimizer(model, matrices="muon"), make_optimizer(twin, matrices="muon")
    mats = opt.param_groups[0]["params"]
    mom = [torch.zeros_like(p, dtype=torch.float64) for p in mats]
    for _ in range(2):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss, _ = twin.loss(x, t, vocab_piece=256)
        loss.backward()
        torch.nn.utils.clip_grad_norm_(twin.parameters(), 1.0)
        grads = [p.grad.double() for p in opt2.param_groups[0]["params"]]
        before = [p.detach().double() for p in mats]
        opt2.step()
        opt2.zero_grad(set_to_none=True)
        got = train_step(model, opt, x, t, vocab_piece=256)
        assert torch.equal(got, loss.detach())
        assert all(torch.equal(p, q) for p, q in zip(model.parameters(), twin.parameters()))
        for p, w, g, k in zip(mats, before, grads, range(len(mats))):
            mom[k] = 0.95 * mom[k] + 0.05 * g
            step = 0.02 * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * _ns(0.05 * g + 0.95 * mom[k])
            want = (1 - 0.02 * 0.1) * w - step
            # the bound of the orthogonalisation at these sizes (5 steps, at most 96 columns) is below 0.1 of the step
            assert float((p.detach().double() - want).norm()) <= 0.1 * float(step.norm()) + 2.0 ** -22 * float(w.norm())
    assert all(opt.state[p]["momentum_buffer"].dtype is torch.float32 for p in mats)


@pytest.mark.parametrize("transform", ["jvp", "vmap", "dual"])
def test_what_no_autograd_function_stands_around_refuses_transforms(transform):
    """Batched inputs and forward-mode tangents raise instead of being dropped, also where nothing needs a gradient."""
    from llattn_amd import muon_update, orthogonalize, piecewise_head_loss
    fw = torch.autograd.forward_ad
    h, w = torch.randn(5, 16, device=DEV).bfloat16(), torch.randn(50, 16, device=DEV).bfloat16()
    t, x = torch.zeros(5, dtype=torch.int64, device=DEV), torch.randn(6, 9, device=DEV)
    for fn, arg in ((lambda v: piecewise_head_loss(v, w, t, reduction="sum"), h), (lambda v: piecewise_head_loss(h, v, t), w),
                    (orthogonalize, x), (lambda v: muon_update([x.clone()], [v], [x.clone()], lr=0.1), x)):
        fn(arg)
        with pytest.raises((RuntimeError, ValueError, NotImplementedError)):
            if transform == "jvp":
                torch.func.jvp(fn, (arg,), (torch.ones_like(arg),))
            elif transform == "vmap":
                torch.func.vmap(fn)(arg[None])
            else:
                with fw.dual_level():
                    fn(fw.make_dual(arg, torch.ones_like(arg)))
