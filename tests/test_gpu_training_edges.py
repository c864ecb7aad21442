"""Edges of the training-side operators on the GPU: empty work items, layouts,
overlapping launches, magnitudes far apart, values that are not finite.

Tolerances as in test_gpu_training.py unless a test derives its own.
"""
import math

import numpy as np
import pytest
import torch

from oracle import training as otr
from oracle.selection import to_f64
from sparseattnfunctions_b200 import kernels, training
from sparseattnfunctions_b200.geometry import VideoGeometry
from sparseattnfunctions_b200.special_attentions.block_mask_attn import BlockSparseAttention
from test_gpu_training import BF16, F16, F32, U, _check_grad, _mask, _near, _randn

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


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_out_needs_a_contiguous_last_dimension(cuda_device, dtype):
    """A destination whose channels are apart is refused, not written as if they
    were side by side; rows that are apart are fine."""
    q, k = (_randn(210 + i, 1, 2, 200, 64, dtype=dtype).to(cuda_device) for i in range(2))
    csr = kernels.mask_to_csr(torch.ones(1, 2, 2, 2, dtype=torch.bool, device=cuda_device), 128, 128)
    table = torch.ones(200, 32, device=cuda_device), torch.zeros(200, 32, device=cuda_device)
    good = torch.empty_like(q)
    apart = torch.full((1, 2, 200, 128), 5.0, dtype=dtype, device=cuda_device)
    turned = torch.full((1, 2, 64, 200), 5.0, dtype=dtype, device=cuda_device)
    for bad in (apart[..., ::2], turned.transpose(2, 3)):
        for call in (lambda: kernels.bsa_fwd_lse(q, k, k, csr, 0.125, out=bad),
                     lambda: kernels.rope(q, k, *table, out=(bad, good)),
                     lambda: kernels.rope(q, k, *table, out=(good, bad)),
                     lambda: kernels.rope(q, None, *table, out=bad),
                     lambda: kernels.rope(bad, k, *table, out=(bad, good))):
            with pytest.raises(ValueError):
                call()
    assert bool((apart == 5).all()) and bool((turned == 5).all())
    kernels.rope(q, k, *table, out=(apart[..., :64], good))
    assert torch.equal(apart[..., :64], q) and torch.equal(good, k) and bool((apart[..., 64:] == 5).all())
    ref = kernels.bsa_fwd_lse(q, k, k, csr, 0.125)[0]
    kernels.bsa_fwd_lse(q, k, k, csr, 0.125, out=apart[..., 64:])
    assert torch.equal(apart[..., 64:], ref)


@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32])
def test_gradient_expanded_over_heads_or_batch(cuda_device, dtype):
    """What autograd hands over behind a sum over heads or batch rows: a stride
    of 0 in those dimensions, whole rows inside."""
    q, k, v, d = (_randn(220 + i, 2, 3, 200, 64, dtype=dtype).to(cuda_device) for i in range(4))
    csr = kernels.mask_to_csr(torch.ones(2, 3, 2, 2, dtype=torch.bool, device=cuda_device), 128, 128)
    out, lse = kernels.bsa_fwd_lse(q, k, v, csr, 0.125)
    for dout in (d[:, :1].expand(d.shape), d[:1].expand(d.shape), d[:1, :1].expand(d.shape)):
        got = kernels.bsa_bwd(dout, q, k, v, out, lse, csr, 0.125)
        ref = kernels.bsa_bwd(dout.contiguous(), q, k, v, out, lse, csr, 0.125)
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    x = [t.clone().requires_grad_() for t in (q, k, v)]
    training.sparse_attention(*x, csr, 0.125).sum(1).mul(d[:, 0]).sum().backward()
    ref = kernels.bsa_bwd(d[:, :1].expand(d.shape).contiguous(), q, k, v, out, lse, csr, 0.125)
    assert all(torch.equal(a.grad, b) for a, b in zip(x, ref))


@pytest.mark.parametrize("lead", [0, 2])
def test_replays_beside_other_forwards(cuda_device, lead):
    """Replays of a captured training forward on one stream beside more than 64
    direct ones on another, more query tiles each than the GPU takes at once:
    no launch shares a counter with another, so all give the bits of one alone."""
    H, S = 20, 4000
    q, k, v = (_randn(230 + i, 1, H, S, 64, dtype=BF16).to(cuda_device) for i in range(3))
    mask = _mask(233, 1, H, 32, 32, 0.3)
    mask[:, :, :lead] = True
    csr = kernels.mask_to_csr(mask.to(cuda_device), 128, 128, dense_rows=lead)
    ref = kernels.bsa_fwd_lse(q, k, v, csr, 0.125)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.bsa_fwd_lse(q, k, v, csr, 0.125)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = [kernels.bsa_fwd_lse(q, k, v, csr, 0.125) for _ in range(8)]
    direct = []
    for _ in range(20):
        with torch.cuda.stream(side):
            graph.replay()
        direct += [kernels.bsa_fwd_lse(q, k, v, csr, 0.125) for _ in range(8)]
    torch.cuda.synchronize()
    for out, lse in held + direct:
        assert torch.equal(out, ref[0]) and torch.equal(lse, ref[1])


def _row_errors(got, ref):
    """Largest error of a row over the row's own size (2-norms)."""
    got = got.double().cpu().numpy()
    size = np.linalg.norm(ref, axis=-1)
    return float((np.linalg.norm(got - ref, axis=-1)[size > 0] / size[size > 0]).max())


@pytest.mark.parametrize("bm,bn", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("large", [2.0 ** 4, 2.0 ** 8, 2.0 ** 12])
@pytest.mark.parametrize("H,S", [(4, 1500), (1, 4000)])
def test_f16_rows_of_unlike_size(cuda_device, bm, bn, large, H, S):
    """One row block's gradients ``large`` times the others': every row of dq is
    good to its own size, and so are dk and dv of every key.

    A row's error is made of the rounding of the result and those of its terms
    ds or p, each at most u / sqrt(3) of the power of two above it in the mean
    square: 0.816 u together for values without a common part.  The rms of 64
    channels spreads by 1 / sqrt(128), 1.4 at 4.5 of it; what falls below f16's
    normal range is 2^-25 beside terms of 2^-9 and the fp32 sums 4e-5 of them,
    0.05 u."""
    q, k, v, dout = (_randn(240 + i, 1, H, S, 64, dtype=torch.float32) for i in range(4))
    dout[:, :, 2 * bm:3 * bm] *= large
    q, k, v, dout = (t.to(F16) for t in (q, k, v, dout))
    nbq, nbk = math.ceil(S / bm), math.ceil(S / bn)
    mask = _mask(244, 1, H, nbq, nbk, 0.3)
    mask[..., 1] = True
    mask[:, :, 2, nbk // 2:] = False
    csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bn)
    gq, gk, gv, gd = (t.to(cuda_device) for t in (q, k, v, dout))
    out, lse = kernels.bsa_fwd_lse(gq, gk, gv, csr, 0.125)
    grads = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)
    live = otr.token_mask(mask, S, S, bm, bn)
    ref = otr.attention_grad(dout, q, k, v, out.cpu(), lse.cpu(), live, 0.125)
    off = {n: _row_errors(x, ref[n][0]) / U[F16] for n, x in zip(("dq", "dk", "dv"), grads)}
    assert max(off.values()) <= 1.2, off


@pytest.mark.parametrize("H,Sq,Sk,bm,bn", [(2, 300, 700, 64, 64), (2, 500, 333, 128, 128), (1, 200, 5000, 64, 128)])
def test_f16_keys_with_a_common_part(cuda_device, H, Sq, Sk, bm, bn):
    """Keys that share a component eight times their spread: a row of ds sums to
    nearly zero, so dq hardly sees it, but a rounding of ds alone would show
    eight times over.  The result's rounding is 0.577 u at most in the mean
    square; ds in two parts is good to 2^-25 beside terms of 2^-9 (2500 keys),
    eight times over 0.15 u; 0.03 u for fp32's part (2e-6 of p, eight times
    over)."""
    q, k, v, dout = (_randn(250 + i, 1, H, s, 64, dtype=torch.float32) for i, s in enumerate((Sq, Sk, Sk, Sq)))
    q, k, v, dout = q.to(F16), (k + 8.0).to(F16), v.to(F16), dout.to(F16)
    mask = _mask(254, 1, H, math.ceil(Sq / bm), math.ceil(Sk / bn), 0.5)
    csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bn)
    gq, gk, gv, gd = (t.to(cuda_device) for t in (q, k, v, dout))
    out, lse = kernels.bsa_fwd_lse(gq, gk, gv, csr, 0.125)
    dq = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)[0]
    live = otr.token_mask(mask, Sq, Sk, bm, bn)
    ref = otr.attention_grad(dout, q, k, v, out.cpu(), lse.cpu(), live, 0.125)["dq"][0]
    off = np.linalg.norm(dq.double().cpu().numpy() - ref) / np.linalg.norm(ref)
    assert off <= 0.65 * U[F16], f"{off / U[F16]:.3f} U"


@pytest.mark.parametrize("bn", [64, 128])
@pytest.mark.parametrize("mode", ["plain", "lead", "bias", "ranges", "frames", "pool", "keys", "train", "processor"])
def test_f16_scores_that_grow_along_the_keys(cuda_device, mode, bn):
    """Later key blocks exceed a row's first ones by far more than f16's range
    (2^16): finite, and right, in every form of the 16-bit forward."""
    geo = VideoGeometry(64, 4, 10, 16)
    H, S = 2, geo.seq_len
    q, k, v = (_randn(260 + i, 1, H, S, 64, dtype=torch.float32) for i in range(3))
    k[:, :, :bn] *= 0.05
    k[:, :, bn:] *= 6.0
    q, k, v = (t.to(F16) for t in (q, k, v))
    gq, gk, gv = (t.to(cuda_device) for t in (q, k, v))
    nb = math.ceil(S / bn)
    csr = kernels.mask_to_csr(torch.ones(1, H, nb, nb, dtype=torch.bool, device=cuda_device), bn, bn,
                              dense_rows=2 if mode == "lead" else 0)
    live = np.ones((1, H, S, S), dtype=bool)
    lse = None
    if mode in ("plain", "lead"):
        out = kernels.bsa_fwd(gq, gk, gv, csr, 0.125)
    elif mode == "bias":
        out = kernels.bsa_fwd(gq, gk, gv, csr, 0.125, kv_bias=torch.zeros(S, device=cuda_device))
    elif mode == "ranges":
        live[..., S - 30:] = False
        ranges = torch.tensor([[0, S - 30, 0, 0]], dtype=torch.int32, device=cuda_device).repeat(S, 1)
        out = kernels.bsa_fwd(gq, gk, gv, csr, 0.125, row_ranges=ranges)
    elif mode == "frames":
        bits = torch.full((H, geo.frames), 15, dtype=torch.int32, device=cuda_device)
        fm = kernels.FrameMask(bits, None, None, geo.text_len, geo.frames, geo.frame_len)
        out = kernels.bsa_fwd_frames(gq, gk, gv, kernels.frame_csr(fm, 1, H, bn, bn), fm, 0.125)
    elif mode == "pool":
        out = kernels.bsa_fwd_pool(gq, gk, gv, csr, 0.125)[0]
    elif mode == "keys":
        keys = torch.arange(S, dtype=torch.int32, device=cuda_device)[None]
        out = kernels.bsa_fwd_keys(gq, gk, gv, keys, torch.zeros(1, dtype=torch.int32, device=cuda_device), 0.125)
    elif mode == "train":
        out, lse = kernels.bsa_fwd_lse(gq, gk, gv, csr, 0.125)
    else:
        out = BlockSparseAttention(block_size=bn, density=1.0, geometry=geo)(gq, gk, gv)
    ref, ref_lse = otr.attention(q, k, v, live, 0.125)
    # as test_gpu_training.py bounds the forward: the output's rounding, and P's
    # with an exponential good to 1e-4, doubled for the second order
    tol = U[F16] * np.abs(ref) + 2 * (U[F16] + 1e-4) * np.abs(to_f64(v)).max(axis=2, keepdims=True) + 1e-6
    _near("out", out, ref, tol)
    if lse is not None:
        _near("lse", lse, ref_lse, 1e-4)


@pytest.mark.parametrize("dtype,bm,S,lead", [(BF16, 128, 600, 0), (F16, 64, 600, 0), (BF16, 128, 3500, 2), (F16, 64, 3500, 3),
                                             (F32, 64, 600, 0), (F32, 128, 3500, 0)])
def test_nan_reaches_every_row_that_sees_it(cuda_device, dtype, bm, S, lead):
    """A query row of NaN, and a NaN among the keys of a listed block: the rows
    that see it have NaN output, log-sum-exp and dq, whether their keys are
    walked in one piece or in several, and the other rows keep their bits."""
    H = 2
    q, k, v, dout = (_randn(270 + i, 1, H, S, 64, dtype=dtype).to(cuda_device) for i in range(4))
    nb = math.ceil(S / bm)
    mask = _mask(274, 1, H, nb, nb, 0.4)
    mask[:, :, :lead] = True
    mask[:, :, lead:, nb - 1] = False
    mask[:, 1, lead:lead + 2, nb - 1] = True
    csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bm, dense_rows=lead)
    clean, clean_lse = kernels.bsa_fwd_lse(q, k, v, csr, 0.125)
    clean_dq = kernels.bsa_bwd(dout, q, k, v, clean, clean_lse, csr, 0.125)[0]

    def check(q, k, seen):
        out, lse = kernels.bsa_fwd_lse(q, k, v, csr, 0.125)
        assert bool(torch.isnan(lse[seen]).all()) and bool(torch.isnan(out[seen]).all())
        assert torch.equal(lse[~seen], clean_lse[~seen]) and torch.equal(out[~seen], clean[~seen])
        dq = kernels.bsa_bwd(dout, q, k, v, out, lse, csr, 0.125)[0]
        assert bool(torch.isnan(dq[seen]).all())
        return dq

    rows = torch.zeros(1, H, S, dtype=torch.bool, device=cuda_device)
    rows[0, 0, 5] = rows[0, 1, S - 1] = True
    bad = q.clone()
    bad[rows] = float("nan")
    dq = check(bad, k, rows)
    assert torch.equal(dq[~rows], clean_dq[~rows])
    seen = mask[..., nb - 1].to(cuda_device).repeat_interleave(bm, 2)[:, :, :S]
    bad = k.clone()
    bad[:, :, S - 1] = float("nan")
    check(q, bad, seen)


@pytest.mark.parametrize("bm,bn", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("dtype,H,S,lead", [(BF16, 3, 640, 0), (F16, 2, 640, 0), (F32, 2, 640, 0), (BF16, 1, 4000, 2)])
def test_values_in_another_blocks_lists(cuda_device, dtype, H, S, lead, bm, bn):
    """NaN and infinities in a key block that one row block lists, and in that
    row block's q and dout: what does not see them keeps its bits, 64-row
    neighbours in the same 128-row tile included."""
    q, k, v, d = (_randn(280 + i, 1, H, S, 64, dtype=dtype).to(cuda_device) for i in range(4))
    nbq, nbk = math.ceil(S / bm), math.ceil(S / bn)
    for row, x, y in ((lead, nbk - 2, 1), (lead + 1, nbk - 1, 0), (nbq - 1, 2, nbk - 1)):
        mask = _mask(284, 1, H, nbq, nbk, 0.4)
        mask[:, :, :lead] = True
        mask[..., x] = mask[:, :, row] = False
        mask[:, :, row, x] = mask[:, :, row, y] = True
        csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bn)
        out, lse = kernels.bsa_fwd_lse(q, k, v, csr, 0.125)
        clean = kernels.bsa_bwd(d, q, k, v, out, lse, csr, 0.125)
        rows = torch.zeros(S, dtype=torch.bool, device=cuda_device)
        rows[row * bm:(row + 1) * bm] = True
        keys = torch.zeros(S, dtype=torch.bool, device=cuda_device)
        for c in (x, y):
            keys[c * bn:(c + 1) * bn] = True
        q2, k2, v2, d2 = (t.clone() for t in (q, k, v, d))
        for t, at, value in ((k2, x * bn + 3, "nan"), (v2, x * bn + 9, "inf"), (v2, x * bn + 4, "nan"),
                             (q2, row * bm + 7, "inf"), (d2, row * bm + 1, "nan"), (d2, row * bm + 2, "inf")):
            t[:, :, at] = float(value)
        out2, lse2 = kernels.bsa_fwd_lse(q2, k2, v2, csr, 0.125)
        dirty = kernels.bsa_bwd(d2, q2, k2, v2, out2, lse2, csr, 0.125)
        assert torch.equal(out2[:, :, ~rows], out[:, :, ~rows]) and torch.equal(lse2[:, :, ~rows], lse[:, :, ~rows])
        assert torch.equal(dirty[0][:, :, ~rows], clean[0][:, :, ~rows])
        assert torch.equal(dirty[1][:, :, ~keys], clean[1][:, :, ~keys])
        assert torch.equal(dirty[2][:, :, ~keys], clean[2][:, :, ~keys])
        assert bool(torch.isnan(out2[:, :, row * bm:row * bm + bm]).any()) and bool(torch.isnan(dirty[1][:, :, keys]).any())


@pytest.mark.parametrize("Sk,size", [(2, 4000.0), (2, 60000.0), (70, 60000.0), (300, 3e-6)])
@pytest.mark.parametrize("bm", [64, 128])
def test_f16_values_of_any_size(cuda_device, Sk, size, bm):
    """Values at both ends of f16, all channels of one sign with dout's, so that
    dout . v is as large as it can be beside them: finite gradients, as exact as
    for values near 1 (the same tolerances), and infinite where f16 ends."""
    H, Sq = 2, 200
    sign = _randn(290, 1, 1, 1, 64).sign()
    flip = _randn(291, 1, H, Sk, 1).sign()
    q = _randn(292, 1, H, Sq, 64, dtype=F16)
    k = _randn(293, 1, H, Sk, 64, dtype=F16, scale=0.05 if size > 1 else 4.0)
    v = (sign * flip * (0.7 + 0.3 * torch.rand(1, H, Sk, 64, generator=torch.Generator().manual_seed(294))) * size).to(F16)
    dout = (sign * (0.5 + 0.5 * torch.rand(1, H, Sq, 64, generator=torch.Generator().manual_seed(295))) *
            (1.0 if size > 1 else 2.0 ** 12)).to(F16)
    nbq, nbk = math.ceil(Sq / bm), math.ceil(Sk / bm)
    mask = torch.ones(1, H, nbq, nbk, dtype=torch.bool)
    csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bm)
    gq, gk, gv, gd = (t.to(cuda_device) for t in (q, k, v, dout))
    out, lse = kernels.bsa_fwd_lse(gq, gk, gv, csr, 0.125)
    grads = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)
    live = otr.token_mask(mask, Sq, Sk, bm, bm)
    ref = otr.attention_grad(dout, q, k, v, out.cpu(), lse.cpu(), live, 0.125)
    for name, got in zip(("dq", "dk", "dv"), grads):
        value, by_term, by_size = ref[name]
        fits = np.abs(value) < 60000.0
        # one rounding of the result (2^-25 below the normal range), two of each term, fp32 sums
        tol = U[F16] * np.abs(value) * 1.01 + 2.0 ** -25 + 2 * (U[F16] + 1e-4) * by_term + 4e-5 * by_size
        off = np.abs(got.double().cpu().numpy() - value)
        assert fits.any() and bool((off[fits] <= tol[fits]).all()), f"{name}: {np.nanmax(off[fits] / tol[fits])}"
        past = np.abs(value) > 70000.0
        assert np.array_equal(got.double().cpu().numpy()[past], np.copysign(np.inf, value[past]))
