"""Differentiable rotary positions and block-sparse attention.

    table = video_rope(geometry, device=q.device)
    q, k = rotary(q, k, table)
    with torch.no_grad():
        csr = kernels.pool_topk(q, k, block_m=128, block_n=128, topk=14, text_blocks_q=2, text_blocks_k=2)
    out = sparse_attention(q, k, v, csr, sm_scale)
    out.backward(dout)

The block list is a constant of the step: no gradient passes through the
selection.  ``special_attentions.block_mask_attn.BlockSparseAttention`` does
this when one of its inputs requires a gradient.  Second derivatives are not
available.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import kernels
from .rope import RopeTable


class _SparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, csr, sm_scale):
        out, lse = kernels.bsa_fwd_lse(q, k, v, csr, sm_scale)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.csr, ctx.sm_scale = csr, sm_scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse = ctx.saved_tensors
        dq, dk, dv = kernels.bsa_bwd(dout, q, k, v, out, lse, ctx.csr, ctx.sm_scale)
        return dq, dk, dv, None, None


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, cos, sin, text_len, layout):
        ctx.save_for_backward(cos, sin)
        ctx.how = dict(text_len=text_len, layout=layout)
        return kernels.rope(q, k, cos, sin, **ctx.how)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        cos, sin = ctx.saved_tensors
        dq, dk = kernels.rope(dq, dk, cos, sin, inverse=True, **ctx.how)
        return dq, dk, None, None, None, None


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, csr: kernels.BlockCSR,
                     sm_scale: float) -> torch.Tensor:
    """Differentiable ``kernels.bsa_fwd_lse`` (its output alone): gradients to
    q, k and v by ``kernels.bsa_bwd``."""
    return _SparseAttention.apply(q, k, v, csr, float(sm_scale))


def rotary(q: torch.Tensor, k: torch.Tensor, table: RopeTable):
    """Differentiable ``kernels.rope`` on q and k with the table's layout and
    text length."""
    return _Rotary.apply(q, k, table.cos, table.sin, table.text_len, table.layout)
