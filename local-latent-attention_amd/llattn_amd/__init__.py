"""MI355X-native (gfx950 HIP) local+latent attention: drop-in for the reference's fused block.

Public surface:

* :class:`LocalLatentAttentionTriton` -- the attention module (reference
  llattn_triton.py:33-176 surface, reference models.py:61-462 math);
* :class:`LLAttnFunction` -- the autograd op surface (reference kernels/llattn_op.py:184-238);
* :func:`build_attention` -- the dispatcher (reference models.py:465-488);
* :func:`pool` -- segment pooling op;
* :func:`piecewise_head_loss` -- LM head and cross entropy over a vocabulary of any size, no logits kept;
* :func:`orthogonalize`, :func:`muon_update`, :class:`Muon`, :class:`MuonAdamW` -- orthogonalised weight updates.
"""
from ._lib import DIV_COUNT, DIV_ONE, DIV_SEG, Layout, resolve_layout
from .config import ModelConfig, build_attention
from .module import LocalLatentAttentionHIP, LocalLatentAttentionTriton
from .muon import Muon, MuonAdamW, muon_update, orthogonalize
from .ops import LLAttnCore, LLAttnFunction, pool
from .xent import piecewise_head_loss

__all__ = [
    "DIV_COUNT", "DIV_ONE", "DIV_SEG", "Layout", "resolve_layout", "ModelConfig", "build_attention",
    "LocalLatentAttentionHIP", "LocalLatentAttentionTriton", "LLAttnCore", "LLAttnFunction", "pool",
    "piecewise_head_loss", "orthogonalize", "muon_update", "Muon", "MuonAdamW",
]
