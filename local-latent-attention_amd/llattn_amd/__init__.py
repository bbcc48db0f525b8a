"""MI355X-native (gfx950 HIP) local+latent attention: drop-in for the reference's fused block.

Public surface:

* :class:`LocalLatentAttentionTriton` -- the attention module (reference
  llattn_triton.py:33-176 surface, reference models.py:61-462 math);
* :class:`LLAttnFunction` -- the autograd op surface (reference kernels/llattn_op.py:184-238);
* :func:`build_attention` -- the dispatcher (reference models.py:465-488);
* :func:`pool` -- segment pooling op;
* :func:`piecewise_head_loss` -- LM head and cross entropy over a vocabulary of any size, no logits kept;
* :func:`embed` -- token rows, scaled, plus position rows;
* :func:`gated_feed_forward` -- ``w2(act(w1 x) * w3 x)``;
* :func:`grad_norm`, :func:`clip_grad_norm`, :func:`clip_grad_norm_`, :func:`clip_grads_with_norm_` -- the norm over all
  gradients, and clipping;
* :func:`orthogonalize`, :func:`muon_update`, :class:`Muon`, :class:`MuonAdamW` -- orthogonalised weight updates.
"""
from ._lib import DIV_COUNT, DIV_ONE, DIV_SEG, Layout, resolve_layout
from .clip import clip_grad_norm, clip_grad_norm_, clip_grads_with_norm_, grad_norm
from .config import ModelConfig, build_attention
from .embedding import embed
from .gated import gated_feed_forward
from .module import LocalLatentAttentionHIP, LocalLatentAttentionTriton
from .muon import Muon, MuonAdamW, muon_update, orthogonalize
from .ops import LLAttnCore, LLAttnFunction, pool
from .xent import piecewise_head_loss

__all__ = [
    "DIV_COUNT", "DIV_ONE", "DIV_SEG", "Layout", "resolve_layout", "ModelConfig", "build_attention",
    "LocalLatentAttentionHIP", "LocalLatentAttentionTriton", "LLAttnCore", "LLAttnFunction", "pool",
    "piecewise_head_loss", "orthogonalize", "muon_update", "Muon", "MuonAdamW",
    "embed", "gated_feed_forward", "grad_norm", "clip_grad_norm", "clip_grad_norm_", "clip_grads_with_norm_",
]
