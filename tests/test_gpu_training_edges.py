"""Edges of the training-side operators on the GPU: empty work items, layouts,
overlapping launches, magnitudes far apart, values that are not finite.

Tolerances as in test_gpu_training.py unless a test derives its own.
"""
import math

import pytest
import torch

from oracle import training as otr
from sparseattnfunctions_b200 import kernels
from test_gpu_training import BF16, F16, U, _check_fwd, _check_grad, _mask, _randn  # noqa: F401

pytestmark = pytest.mark.gpu


def _fill(like, value):
    """Leaves freed blocks of ``like``'s sizes full of ``value`` to the allocator."""
    for x in [torch.empty_like(t).fill_(value) for t in like]:
        del x


@pytest.mark.parametrize("dtype,bm,bn", [(BF16, 64, 64), (BF16, 128, 128), (F16, 64, 128)])
def test_empty_lines_between_listed_ones(cuda_device, dtype, bm, bn):
    """Most key blocks in no list and most row blocks empty, over many heads, so
    that a CTA takes empty and non-empty items in a row: every gradient row is
    written (the outputs' memory held a pattern), as the oracle has it, and in
    the same bits call after call."""
    B, H, S = 2, 40, 1500
    q, k, v, dout = (_randn(200 + i, B, H, S, 64, dtype=dtype) for i in range(4))
    nbq, nbk = math.ceil(S / bm), math.ceil(S / bn)
    g = torch.Generator().manual_seed(204)
    mask = torch.rand(B, H, nbq, nbk, generator=g) < 0.5
    mask &= torch.rand(B, H, nbq, 1, generator=g) < 0.3
    mask &= torch.rand(B, H, 1, nbk, generator=g) < 0.3
    csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bn)
    gq, gk, gv, gd = (t.to(cuda_device) for t in (q, k, v, dout))
    out, lse = kernels.bsa_fwd_lse(gq, gk, gv, csr, 0.125)
    _fill((gq, gk, gv), 7.0)
    first = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)
    live = otr.token_mask(mask, S, S, bm, bn)
    _check_grad(first, dout, q, k, v, out.cpu(), lse.cpu(), live, 0.125)
    for _ in range(40):
        _fill((gq, gk, gv), 7.0)
        again = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)
        assert all(torch.equal(a, b) for a, b in zip(again, first))
