"""The language model and the trainer's step through ``embed``, ``gated_feed_forward`` and ``clip_grad_norm_`` together, on the
GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
KW = dict(vocab_size=256, max_seq_len=256, d_model=192, n_heads=2, n_layers=2, d_ff=384, local_window=32, local_block_size=64,
          latent_tokens=8, latent_d_model=64, latent_heads=2)


def _model(seed=3, **kw):
    from llattn_amd.lm import build_model
    torch.manual_seed(seed)
    return build_model(**(KW | kw)).to(DEV)


def _tokens(B, T, seed=4, V=256):
    t = torch.randint(0, V, (B, T + 1), generator=torch.Generator().manual_seed(seed)).to(DEV)
    return t[:, :-1], t[:, 1:]


def _step(model, inputs, targets, bf16=True):
    model.zero_grad(set_to_none=True)
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16, enabled=bf16):
        loss, _ = model.loss(inputs, targets)
        loss.backward()
    return loss.detach(), {n: p.grad.clone() for n, p in model.named_parameters()}


@pytest.mark.parametrize("bf16", [True, False])
def test_fused_lookups_keep_the_models_results(bf16):
    """The same loss and gradients, bit for bit, but for the tables' own: those are other orders of the same fp32 sums, over at
    most 256 tokens and the head's share, each addition off by 2^-24 of what it adds up."""
    m = _model(fused_embeddings=True)
    inputs, targets = _tokens(2, 200)
    assert m._fused_embeddings(inputs)
    loss, grads = _step(m, inputs, targets, bf16)
    m.fuse_embeddings = False
    assert not m._fused_embeddings(inputs)
    loss0, grads0 = _step(m, inputs, targets, bf16)
    with torch.no_grad():  # no gradient: in one pass whatever the configuration
        assert m._fused_embeddings(inputs)
        h = m.hidden(inputs)
        m.embedding.max_norm = 1e9
        assert not m._fused_embeddings(inputs) and torch.equal(m.hidden(inputs), h)
        m.embedding.max_norm = None
    assert torch.equal(loss, loss0)
    for n in grads:
        if n in ("embedding.weight", "position.weight"):
            assert float((grads[n] - grads0[n]).abs().max()) <= 400 * 2.0 ** -24 * float(grads0[n].abs().max()) * 4, n
        else:
            assert torch.equal(grads[n], grads0[n]), n


def test_models_that_the_fused_lookup_leaves_alone():
    """Tables that are hooked, normalised, replaced or too short for the row keep torch's own calls."""
    m = _model(fused_embeddings=True)
    ids = _tokens(1, 20)[0]
    assert m._fused_embeddings(ids) and m._fused_embeddings(ids.int())
    seen = []
    h = m.embedding.register_forward_hook(lambda *a: seen.append(1))
    m.hidden(ids)
    assert seen == [1] and not m._fused_embeddings(ids)
    h.remove()
    assert m._fused_embeddings(ids)
    m.position.max_norm = 1.0
    assert not m._fused_embeddings(ids)
    m.position.max_norm = None
    m.embedding.to(torch.bfloat16)
    assert not m._fused_embeddings(ids)
    m.embedding.to(torch.float32)
    assert not m._fused_embeddings(ids.cpu())

    class Mine(torch.nn.Embedding):
        pass
    m.position = Mine(256, 192).to(DEV)
    assert not m._fused_embeddings(ids)


@pytest.mark.parametrize("kind", ["swiglu", "geglu"])
def test_gated_model_against_torchs_products(kind):
    """One training step's loss and gradients of a gated model against the same weights with the feed-forward in torch's fp32
    operations: as far apart as bf16 operands leave them, a few roundings of 2^-8 along each path."""
    m = _model(ffn=kind)
    inputs, targets = _tokens(2, 200)
    loss, grads = _step(m, inputs, targets)
    loss0, grads0 = None, None
    for b in m.blocks:
        b.ff.fused = False
    loss0, grads0 = _step(m, inputs, targets)  # torch's bf16 products under autocast
    assert abs(float(loss - loss0)) < 2e-2
    for n in grads:
        d = float((grads[n] - grads0[n]).norm() / grads0[n].norm())
        assert d < 16 * 2.0 ** -8, (n, d)


def test_feed_forward_of_a_half_precision_model():
    """Weights and input in bf16 without autocast, as a server holds them: one token and many, the same rows."""
    from llattn_amd.config import ModelConfig
    from llattn_amd.lm import GatedFeedForward
    torch.manual_seed(0)
    ff = GatedFeedForward(ModelConfig(d_model=136, d_ff=264, ffn="swiglu")).to(DEV, torch.bfloat16)
    x = torch.randn(3, 40, 136, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    with torch.no_grad():
        y = ff(x)
        ff.fused = False
        want = ff.float()(x.float())
    assert y.dtype is torch.bfloat16 and y.shape == x.shape
    assert float((y.float() - want).norm() / want.norm()) < 4 * 2.0 ** -8


def test_training_steps_together():
    """Lookups, gated blocks, head loss, clipping and the update, as the trainer runs them: steps repeat bit for bit, and
    checkpointed blocks take the same way."""
    from llattn_amd.lm import make_optimizer, train_step
    inputs, targets = _tokens(2, 200)

    def run(**kw):
        m = _model(ffn="swiglu", fused_embeddings=True, **kw)
        opt = make_optimizer(m, lr=1e-3)
        losses = [train_step(m, opt, inputs, targets, grad_clip=0.25, fused_clip=True) for _ in range(3)]
        return torch.stack(losses), [p.detach().clone() for p in m.parameters()]
    a, b = run(), run()
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))
    c = run(checkpoint_blocks=True)
    assert torch.allclose(a[0], c[0], rtol=1e-3)
    assert bool(a[0].isfinite().all())


def test_clipping_of_a_models_gradients():
    from llattn_amd import clip_grad_norm_
    m = _model()
    _, grads = _step(m, *_tokens(2, 100))
    norm = clip_grad_norm_(m.parameters(), 0.1)
    got = [p.grad.clone() for p in m.parameters()]
    for p, g in zip(m.parameters(), grads.values()):
        p.grad = g
    want = torch.nn.utils.clip_grad_norm_(m.parameters(), 0.1)
    assert abs(float(norm - want)) <= 1e-6 * float(want)
    assert all(torch.allclose(a, p.grad, rtol=2e-6, atol=0) for a, p in zip(got, m.parameters()))


def test_generation_with_a_gated_model():
    m = _model(ffn="geglu").eval()
    prompt = _tokens(1, 9)[0]
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        out = m.generate(prompt, 4)
        again = m.generate(prompt, 4)
    assert out.shape == (1, 13) and torch.equal(out, again) and torch.equal(out[:, :9], prompt)


@pytest.mark.parametrize("name", ["w1", "w3", "w2"])
def test_projections_with_something_around_them(name):
    """An adapter, or a hook, on one projection shows in the result: the model's is that of its layers called one by one."""
    from llattn_amd.config import ModelConfig
    from llattn_amd.lm import GatedFeedForward
    torch.manual_seed(0)
    ff = GatedFeedForward(ModelConfig(d_model=64, d_ff=136, ffn="swiglu")).to(DEV, torch.bfloat16)
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    one_by_one = lambda: ff.w2(torch.nn.functional.silu(ff.w1(x)) * ff.w3(x))  # noqa: E731
    with torch.no_grad():
        clean = ff(x)
        hook = getattr(ff, name).register_forward_hook(lambda m, a, y: y * 3)
        assert torch.equal(ff(x), one_by_one()) and not torch.allclose(ff(x), clean, rtol=0.1)
        hook.remove()
        assert torch.equal(ff(x), clean)

        class Adapter(torch.nn.Linear):
            def forward(self, v):
                return super().forward(v) * 3
        m = Adapter(*reversed(getattr(ff, name).weight.shape)).to(DEV, torch.bfloat16)
        m.load_state_dict(getattr(ff, name).state_dict())
        setattr(ff, name, m)
        assert torch.equal(ff(x), one_by_one()) and not torch.allclose(ff(x), clean, rtol=0.1)


@pytest.mark.parametrize("name", ["w1", "w2"])
def test_ungated_projections_with_something_around_them(name):
    from llattn_amd.config import ModelConfig
    from llattn_amd.lm import FeedForward
    torch.manual_seed(0)
    ff = FeedForward(ModelConfig(d_model=64, d_ff=136)).to(DEV)
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    one_by_one = lambda: ff.w2(torch.nn.functional.gelu(ff.w1(x)))  # noqa: E731
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        clean = ff(x)
        hook = getattr(ff, name).register_forward_hook(lambda m, a, y: y * 3)
        assert torch.equal(ff(x), one_by_one()) and not torch.allclose(ff(x), clean, rtol=0.1)
        hook.remove()
        assert torch.equal(ff(x), clean)
        layer = getattr(ff, name)
        layer.forward = lambda v: torch.nn.functional.linear(v, layer.weight, layer.bias) * 3
        assert torch.equal(ff(x), one_by_one()) and not torch.allclose(ff(x), clean, rtol=0.1)
        del layer.forward
        ff.dropout = torch.nn.Identity()
        assert torch.equal(ff(x), one_by_one())


@pytest.mark.parametrize("what", ["x", "w3", "bias"])
def test_types_that_autocast_takes(what):
    """Half-precision inputs or layers under bf16 autocast, which the operator refuses: torch's products, as without it."""
    from llattn_amd.config import ModelConfig
    from llattn_amd.lm import GatedFeedForward
    torch.manual_seed(0)
    ff = GatedFeedForward(ModelConfig(d_model=64, d_ff=136, ffn="swiglu")).to(DEV)
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    if what == "x":
        x = x.half()
    elif what == "w3":
        ff.w3.half()
    else:
        ff.w1.bias = torch.nn.Parameter(ff.w1.bias.detach().half())
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        y = ff(x)
        assert y.dtype is torch.bfloat16 and torch.equal(y, ff.w2(torch.nn.functional.silu(ff.w1(x)) * ff.w3(x)))


def test_fp32_biases_of_a_half_precision_layer():
    """Without autocast the operator takes them, which torch's products do not."""
    from llattn_amd.config import ModelConfig
    from llattn_amd.lm import GatedFeedForward
    ff = GatedFeedForward(ModelConfig(d_model=64, d_ff=136, ffn="swiglu")).to(DEV, torch.bfloat16)
    x = torch.randn(40, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    with torch.no_grad():
        want = ff(x)
        for m in (ff.w1, ff.w3, ff.w2):
            m.bias = torch.nn.Parameter(m.bias.detach().float())
        assert torch.equal(ff(x), want)


@pytest.mark.parametrize("name", ["embedding", "position"])
def test_tables_whose_call_is_replaced(name):
    """A forward put on one table itself is what the model calls, with gradients and without."""
    m = _model(fused_embeddings=True)
    ids, table = _tokens(1, 20)[0], getattr(m, name)
    with torch.no_grad():
        clean = m.hidden(ids)
    table.forward = lambda i: 3 * torch.nn.functional.embedding(i, table.weight)
    assert not m._fused_embeddings(ids)
    with torch.no_grad():
        assert not m._fused_embeddings(ids) and not torch.allclose(m.hidden(ids), clean, rtol=0.1)
    del table.forward
    assert m._fused_embeddings(ids)
