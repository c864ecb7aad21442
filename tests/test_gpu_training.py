"""GPU parity of the training-side operators (rotary positions, attention with
its log-sum-exp, the attention gradient) against the fp64 oracle.

Tolerances, from the number formats.  u is the unit roundoff of the stored
type (2^-8 bf16, 2^-11 f16, 2^-24 fp32).

* An output is rounded once: u |x|.
* In the 16-bit gradient p and ds pass through the 16-bit type on their way
  into a matrix product (u each, relative) and 2^x is good to 1e-4: each term
  of a sum is off by (u + 1e-4) of its size, doubled below for the terms of
  second order.  The f16 products keep p and ds scaled into the type's normal
  range, so what falls below it (2^-25 of the largest) is covered by e_small.
* fp32 sums of n terms, exponents off by 64 or 128 roundings of |s| <= 20, and
  the difference dp - delta are off by at most e32 = 4e-5 of the sizes summed.
"""
import math

import numpy as np
import pytest
import torch

from oracle import training as otr
from oracle.selection import to_f64
from sparseattnfunctions_b200 import kernels, training, workloads
from sparseattnfunctions_b200.geometry import VideoGeometry
from sparseattnfunctions_b200.rope import RopeScaling, video_rope
from sparseattnfunctions_b200.special_attentions.block_mask_attn import BlockSparseAttention

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = {dt: torch.finfo(dt).eps / 2 for dt in (BF16, F16, F32)}
E32 = 4e-5


def _randn(seed, *shape, dtype=F32, strided=False, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    if strided:
        B, H, S, D = shape
        return (torch.randn(B, S, H, D, generator=g) * scale).to(dtype).transpose(1, 2)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _mask(seed, B, H, nbq, nbk, density, empty=()):
    g = torch.Generator().manual_seed(seed)
    m = torch.rand(B, H, nbq, nbk, generator=g) < density
    m[..., 0] = True
    for i in empty:
        m[:, :, i] = False
    return m


def _near(name, got, value, tol):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isfinite(got), np.isfinite(value)), f"{name}: finite values differ"
    fine = np.isfinite(value)
    assert np.array_equal(got[~fine], value[~fine])
    excess = np.abs(got - np.where(fine, value, 0.0))[fine] - np.broadcast_to(tol, value.shape)[fine]
    assert excess.size == 0 or excess.max() <= 0, f"{name}: off by {excess.max():.3e} more than the bound"


def _check_fwd(out, lse, q, k, v, live, scale):
    dt = out.dtype
    ref, ref_lse = otr.attention(q, k, v, live, scale)
    vmax = np.abs(to_f64(v)).max(axis=2, keepdims=True)
    _near("out", out, ref, U[dt] * np.abs(ref) + ((U[dt] + 1e-4) * 2 if dt != F32 else E32) * vmax + 1e-6)
    _near("lse", lse, ref_lse, 1e-4 if dt != F32 else 2e-5)
    return ref, ref_lse


def _check_grad(grads, dout, q, k, v, out, lse, live, scale):
    dt = q.dtype
    u = U[dt]
    ref = otr.attention_grad(dout, q, k, v, out, lse, live, scale)
    for name, got in zip(("dq", "dk", "dv"), grads):
        value, by_term, by_size = ref[name]
        assert got.dtype == dt and got.shape == value.shape
        term = 2 * (u + 1e-4) if dt != F32 else E32
        # f16: a factor below the normal range loses 2^-25 of the largest, for every live pair
        e_small = 0.0 if dt != F16 else 2.0 ** -25 * max(q.shape[2], k.shape[2]) * float(dout.abs().max())
        _near(name, got, value, u * np.abs(value) * 1.01 + term * by_term + E32 * by_size + e_small + 1e-7)


def _run(dev, B, H, Sq, Sk, D, dtype, bm, bn, density, seed, empty=(), strided=False, scale=None, lead=0, mask=None,
         qscale=1.0, dscale=1.0):
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q = _randn(seed, B, H, Sq, D, dtype=dtype, strided=strided, scale=qscale)
    k = _randn(seed + 1, B, H, Sk, D, dtype=dtype, strided=strided)
    v = _randn(seed + 2, B, H, Sk, D, dtype=dtype, strided=strided)
    dout = _randn(seed + 3, B, H, Sq, D, dtype=dtype, strided=strided, scale=dscale)
    nbq, nbk = math.ceil(Sq / bm), math.ceil(Sk / bn)
    if mask is None:
        mask = _mask(seed + 4, B, H, nbq, nbk, density, empty)
    if lead:
        mask[:, :, :lead] = True
    csr = kernels.mask_to_csr(mask.to(dev), bm, bn, dense_rows=lead)
    live = otr.token_mask(mask, Sq, Sk, bm, bn)
    gq, gk, gv, gd = (t.to(dev) for t in (q, k, v, dout))
    out, lse = kernels.bsa_fwd_lse(gq, gk, gv, csr, scale)
    _check_fwd(out, lse, q, k, v, live, scale)
    grads = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, scale)
    _check_grad(grads, dout, q, k, v, out.cpu(), lse.cpu(), live, scale)
    return (gq, gk, gv, gd), out, lse, csr, grads


@pytest.mark.parametrize("bm,bn", [(128, 128), (64, 64), (64, 128), (128, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_block_sizes_and_types(cuda_device, bm, bn, dtype):
    _run(cuda_device, 2, 2, 1000, 900, 64, dtype, bm, bn, 0.35, seed=bm + 3 * bn, empty=(2,))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 200), (200, 1), (63, 65), (64, 64), (128, 128), (129, 257), (1500, 300)])
def test_lengths(cuda_device, Sq, Sk, dtype):
    _run(cuda_device, 1, 2, Sq, Sk, 64, dtype, 128, 128, 0.5, seed=Sq * 7 + Sk)


@pytest.mark.parametrize("D,bm,bn", [(128, 64, 64), (64, 192, 256), (128, 128, 192)])
def test_fp32_sizes(cuda_device, D, bm, bn):
    _run(cuda_device, 1, 2, 500, 700, D, F32, bm, bn, 0.5, seed=D + bm)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_strided_storage(cuda_device, dtype):
    (gq, gk, gv, gd), out, _, _, grads = _run(cuda_device, 2, 3, 400, 400, 64, dtype, 128, 128, 0.6, seed=9, strided=True)
    assert out.stride() == gq.stride() and [g.stride() for g in grads] == [x.stride() for x in (gq, gk, gv)]


@pytest.mark.parametrize("bm", [64, 128])
def test_dense_lead_rows(cuda_device, bm):
    """Dense leading rows and columns (text): the longest lists, split over work items."""
    nb = math.ceil(3000 / bm)
    mask = _mask(5, 1, 3, nb, nb, 0.1)
    mask[..., :3] = True
    _run(cuda_device, 1, 3, 3000, 3000, 64, BF16, bm, bm, 0.1, seed=11, lead=3, mask=mask)


def test_every_block_live(cuda_device):
    _run(cuda_device, 1, 1, 2500, 2500, 64, BF16, 128, 128, 1.1, seed=12)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_and_keys_in_no_list(cuda_device, dtype):
    """Nothing at all, one row alone, a key block nobody lists: zeros and -inf."""
    mask = torch.zeros(1, 2, 4, 5, dtype=torch.bool)
    mask[0, 1, 2, 3] = True
    _, out, lse, _, grads = _run(cuda_device, 1, 2, 470, 600, 64, dtype, 128, 128, 0, seed=13, mask=mask)
    assert not out[:, 0].any() and bool(torch.isneginf(lse[:, 0]).all())
    assert not grads[0][:, 0].any() and not grads[1][:, 0].any() and not grads[2][:, 0].any()
    assert not grads[1][0, 1, :384].any() and not grads[2][0, 1, 512:].any()


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_logits(cuda_device, dtype):
    """Logits of +-40: one key takes almost all of a row, and for f16 the sums
    taken against the first block's maximum pass the type's range."""
    _run(cuda_device, 1, 2, 512, 1024, 64, dtype, 128, 128, 0.7, seed=14, qscale=5.0)


@pytest.mark.parametrize("dscale", [2.0 ** -14, 1.0, 2.0 ** 8])
def test_f16_gradient_scales(cuda_device, dscale):
    """Loss scales that would leave the f16 range if ds were stored as it is."""
    _run(cuda_device, 1, 2, 700, 700, 64, F16, 128, 128, 0.5, seed=15, dscale=dscale)


@pytest.mark.parametrize("dtype,bm", [(BF16, 128), (BF16, 64), (F16, 128), (F32, 64)])
def test_equal_inputs_give_equal_bits(cuda_device, dtype, bm):
    (gq, gk, gv, gd), out, lse, csr, grads = _run(cuda_device, 1, 4, 1100, 1100, 64, dtype, bm, bm, 0.4, seed=16, lead=1)
    for _ in range(3):
        again = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)
        assert all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_values_in_unlisted_places_are_never_read(cuda_device, dtype):
    """NaN and infinities in key blocks that no row lists, and in the rows of q,
    dout and out that see nothing, change no bit of the other gradients."""
    B, H, S, bm = 1, 2, 640, 128
    mask = _mask(17, B, H, 5, 5, 0.5)
    mask[..., 3] = False
    mask[:, :, 1] = False
    x = {n: _randn(18 + i, B, H, S, 64, dtype=dtype).to(cuda_device) for i, n in enumerate("qkvd")}
    csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bm)
    out, lse = kernels.bsa_fwd_lse(x["q"], x["k"], x["v"], csr, 0.125)
    clean = kernels.bsa_bwd(x["d"], x["q"], x["k"], x["v"], out, lse, csr, 0.125)
    for n, rows in (("k", 3), ("v", 3), ("q", 1), ("d", 1)):
        x[n][:, :, rows * bm:(rows + 1) * bm] = float("nan")
        x[n][:, :, rows * bm + 5] = float("inf")
    out2, lse2 = kernels.bsa_fwd_lse(x["q"], x["k"], x["v"], csr, 0.125)
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    out2[:, :, bm:2 * bm] = float("nan")
    dirty = kernels.bsa_bwd(x["d"], x["q"], x["k"], x["v"], out2, lse, csr, 0.125)
    assert all(torch.equal(a, b) for a, b in zip(clean, dirty))
    assert not clean[0][:, :, bm:2 * bm].any() and not clean[1][:, :, 3 * bm:4 * bm].any()


def test_gradient_against_differences(cuda_device):
    """The fp32 gradient against central differences of the fp64 forward:
    directional derivatives agree to the gradient's own error (E32 of the sums
    of sizes; 2e-3 relative to the gradient's norm is far above it)."""
    B, H, Sq, Sk, D = 1, 2, 130, 150, 64
    q, k, v, w = (_randn(30 + i, B, H, n, D) for i, n in enumerate((Sq, Sk, Sk, Sq)))
    mask = _mask(34, B, H, 3, 3, 0.5, empty=(1,))
    live = otr.token_mask(mask, Sq, Sk, 64, 64)
    csr = kernels.mask_to_csr(mask.to(cuda_device), 64, 64)
    dev = [t.to(cuda_device) for t in (q, k, v, w)]
    out, lse = kernels.bsa_fwd_lse(*dev[:3], csr, 0.125)
    grads = kernels.bsa_bwd(dev[3], *dev[:3], out, lse, csr, 0.125)
    for i in range(3):
        way = to_f64(_randn(40 + i, *grads[i].shape))
        side = []
        for sign in (1, -1):
            x = [to_f64(t) for t in (q, k, v)]
            x[i] = x[i] + sign * 1e-4 * way
            side.append(float((otr.attention(*x, live, 0.125)[0] * to_f64(w)).sum()))
        g = to_f64(grads[i])
        assert abs((side[0] - side[1]) / 2e-4 - float((g * way).sum())) <= 2e-3 * np.linalg.norm(g)


def test_gradients_of_any_layout(cuda_device):
    """dout as autograd hands it over: expanded, offset by one element, transposed."""
    (gq, gk, gv, gd), out, lse, csr, _ = _run(cuda_device, 1, 2, 300, 300, 64, BF16, 128, 128, 0.6, seed=50)
    ones = torch.ones_like(gd)
    ref = kernels.bsa_bwd(ones, gq, gk, gv, out, lse, csr, 0.125)
    odd = torch.ones(gd.numel() + 1, dtype=BF16, device=cuda_device)[1:].view(gd.shape)
    for dout in (ones[:1, :1, :1, :1].expand(gd.shape), ones[:, :, :1].expand(gd.shape), odd,
                 ones.transpose(2, 3).contiguous().transpose(2, 3)):
        assert all(torch.equal(a, b) for a, b in zip(kernels.bsa_bwd(dout, gq, gk, gv, out, lse, csr, 0.125), ref))


def test_padded_log_sum_exp(cuda_device):
    """lse as a slice of a padded buffer, and in a layout that has to be copied."""
    (gq, gk, gv, gd), out, lse, csr, grads = _run(cuda_device, 2, 2, 300, 300, 64, BF16, 128, 128, 0.6, seed=51)
    padded = torch.full((2, 2, 384), float("nan"), device=cuda_device)
    padded[:, :, :300] = lse
    apart = torch.stack([lse, lse], dim=-1)[..., 0]
    for x in (padded[:, :, :300], apart):
        assert all(torch.equal(a, b) for a, b in zip(kernels.bsa_bwd(gd, gq, gk, gv, out, x, csr, 0.125), grads))


def test_offsets_past_32_bits(cuda_device):
    """Rows more than 2^31 elements apart (two batch rows of one large buffer)."""
    far, S = 2 ** 31 + 64, 200
    base = torch.empty(far + 8 * S * 64, dtype=BF16, device=cuda_device)
    views, small = [], []
    for i in range(4):
        x = base[i * S * 64:].as_strided((2, 1, S, 64), (far, S * 64, 64, 1))
        y = _randn(60 + i, 2, 1, S, 64, dtype=BF16).to(cuda_device)
        x.copy_(y)
        views.append(x)
        small.append(y)
    csr = kernels.mask_to_csr(_mask(64, 2, 1, 2, 2, 0.5).to(cuda_device), 128, 128)
    out, lse = kernels.bsa_fwd_lse(*small[:3], csr, 0.125)
    ref = kernels.bsa_bwd(small[3], *small[:3], out, lse, csr, 0.125)
    out2, lse2 = kernels.bsa_fwd_lse(*views[:3], csr, 0.125, out=torch.empty_like(out))
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    got = kernels.bsa_bwd(views[3], *views[:3], out2, lse2, csr, 0.125)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    table = video_rope(VideoGeometry(0, 1, 10, 20), 64, device=cuda_device)
    a = kernels.rope(small[0], small[1], table.cos, table.sin)
    b = kernels.rope(views[0], views[1], table.cos, table.sin, out=tuple(views[2:]))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_another_stream(cuda_device):
    """On a side stream, after work queued there, beside the same calls on the default one."""
    (gq, gk, gv, gd), out, lse, csr, grads = _run(cuda_device, 1, 3, 900, 900, 64, BF16, 128, 128, 0.5, seed=70, lead=2)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        q2 = gq * 1.0
        out2, lse2 = kernels.bsa_fwd_lse(q2, gk, gv, csr, 0.125)
        got = kernels.bsa_bwd(gd, q2, gk, gv, out2, lse2, csr, 0.125)
    here = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)
    torch.cuda.synchronize()
    assert torch.equal(out2, out) and torch.equal(lse2, lse)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(grads, got, here))


def test_zero_lengths(cuda_device):
    x = torch.zeros(1, 2, 0, 64, dtype=BF16, device=cuda_device)
    y = _randn(80, 1, 2, 70, 64, dtype=BF16).to(cuda_device)
    none = torch.zeros(2, 1, dtype=torch.int32, device=cuda_device)
    idx = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    csr = kernels.BlockCSR(none, idx, 1, 2, 0, 1, 128, 128)
    out, lse = kernels.bsa_fwd_lse(x, y, y, csr, 0.125)
    assert out.shape == x.shape and lse.shape == (1, 2, 0)
    dq, dk, dv = kernels.bsa_bwd(x, x, y, y, out, lse, csr, 0.125)
    assert dq.shape == x.shape and not dk.any() and not dv.any()
    csr = kernels.BlockCSR(torch.zeros(2, 2, dtype=torch.int32, device=cuda_device), idx, 1, 2, 1, 0, 128, 128)
    out, lse = kernels.bsa_fwd_lse(y, x, x, csr, 0.125)
    assert not out.any() and bool(torch.isneginf(lse).all())
    assert not kernels.bsa_bwd(y, y, x, x, out, lse, csr, 0.125)[0].any()
    table = torch.zeros(0, 32, device=cuda_device)
    assert kernels.rope(x, x, table, table)[0].shape == x.shape


def test_refusals(cuda_device):
    x = _randn(90, 1, 2, 200, 64, dtype=BF16).to(cuda_device)
    csr = kernels.mask_to_csr(torch.ones(1, 2, 2, 2, dtype=torch.bool, device=cuda_device), 128, 128)
    out, lse = kernels.bsa_fwd_lse(x, x, x, csr, 0.125)
    wide = torch.zeros(1, 2, 200, 128, dtype=BF16, device=cuda_device)
    for call in (lambda: kernels.bsa_fwd_lse(x, x[:, :1], x, csr, 0.125),
                 lambda: kernels.bsa_fwd_lse(x[:, :, :100], x, x, csr, 0.125),
                 lambda: kernels.bsa_fwd_lse(x, x.half(), x.half(), csr, 0.125),
                 lambda: kernels.bsa_fwd_lse(x, x, x, csr, -0.125),
                 lambda: kernels.bsa_fwd_lse(x, x, x, csr, 0.125, out=out.float()),
                 lambda: kernels.bsa_bwd(x, x, x, x, out, lse.half(), csr, 0.125),
                 lambda: kernels.bsa_bwd(x, x, x, x, out, lse[:, :, :100], csr, 0.125),
                 lambda: kernels.bsa_bwd(x[:, :, :100], x, x, x, out, lse, csr, 0.125),
                 lambda: kernels.bsa_bwd(x.float(), x, x, x, out, lse, csr, 0.125),
                 lambda: kernels.bsa_bwd(x, x, x, x, out, lse, csr, 0.0)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        kernels.bsa_fwd_lse(wide, wide, wide, csr, 0.125)
    t = torch.zeros(200, 32, device=cuda_device)
    for call in (lambda: kernels.rope(x, x, t, t, layout="quarter"), lambda: kernels.rope(x, x, t, t, text_len=3),
                 lambda: kernels.rope(x, x, t.half(), t.half()), lambda: kernels.rope(x, x[:, :, :100], t, t),
                 lambda: kernels.rope(x, x.float(), t, t), lambda: kernels.rope(x, x, t.repeat(1, 2), t.repeat(1, 2)),
                 lambda: kernels.rope(x, x, t, t, out=(x,))):
        with pytest.raises(ValueError):
            call()


# --------------------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,R,text,strided", [(64, 64, 7, False), (64, 32, 0, True), (64, 24, 5, False), (128, 128, 3, True),
                                              (72, 44, 2, False), (65, 10, 1, False)])
def test_rope(cuda_device, layout, dtype, D, R, text, strided):
    """Two products and a sum in fp32 (2^-22 of their sizes), one rounding."""
    B, Hq, Hk, n = 2, 5, 3, 77
    q = _randn(100, B, Hq, text + n, D, dtype=dtype, strided=strided)
    k = _randn(101, B, Hk, text + n, D, dtype=dtype, strided=strided)
    angle = _randn(102, n, R // 2) * 10
    cos, sin = angle.cos(), angle.sin()
    for inverse in (False, True):
        got = kernels.rope(q.to(cuda_device), k.to(cuda_device), cos.to(cuda_device), sin.to(cuda_device), text_len=text,
                           layout=layout, inverse=inverse)
        for x, y in zip((q, k), got):
            ref = otr.rope(x, cos, sin, text, layout, inverse)
            size = float(np.abs(to_f64(x)).max()) * 2
            _near("rope", y, ref, U[dtype] * np.abs(ref) * 1.01 + 2.0 ** -22 * size + (2.0 ** -25 if dtype == F16 else 0))
            assert torch.equal(y[:, :, :text].cpu(), x[:, :, :text]) and torch.equal(y[..., R:].cpu(), x[..., R:])


def test_rope_forms(cuda_device):
    """q alone, in place, a table per batch row, one token, no rotated token, unaligned rows."""
    q = _randn(110, 2, 3, 40, 64, dtype=BF16).to(cuda_device)
    k = _randn(111, 2, 2, 40, 64, dtype=BF16).to(cuda_device)
    angle = _randn(112, 2, 36, 32).to(cuda_device)
    cos, sin = angle.cos(), angle.sin()
    a, b = kernels.rope(q, k, cos, sin, text_len=4)
    for i in range(2):
        one = kernels.rope(q[i:i + 1], None, cos[i], sin[i], text_len=4)
        assert torch.equal(one, a[i:i + 1])
    x, y = q.clone(), k.clone()
    kernels.rope(x, y, cos, sin, text_len=4, out=(x, y))
    assert torch.equal(x, a) and torch.equal(y, b)
    assert torch.equal(kernels.rope(q[:, :, 4:5], None, cos[:, :1], sin[:, :1]), a[:, :, 4:5])
    assert torch.equal(kernels.rope(q, None, cos[0, :0], sin[0, :0], text_len=40), q)
    odd = torch.empty(2 * 3 * 40 * 65 + 1, dtype=BF16, device=cuda_device)[1:].as_strided((2, 3, 40, 64),
                                                                                         (7800, 2600, 65, 1))
    odd.copy_(q)
    assert torch.equal(kernels.rope(odd, None, cos, sin, text_len=4), a)
    back = kernels.rope(a.float(), None, cos, sin, text_len=4, inverse=True)
    assert float((back - q.float()).abs().max()) <= 2 * U[BF16] * float(q.abs().max()) * 1.5


# --------------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype,layout", [(BF16, "interleaved"), (F32, "half")])
def test_processor_trains(cuda_device, dtype, layout):
    """rotary -> selection -> attention -> gradients through the processor, on a
    short clip with text, against the oracle on the rotated values it used."""
    geo = VideoGeometry(70, 2, 10, 16)
    table = video_rope(geo, 64, layout=layout, scaling=RopeScaling("linear", 2.0), device=cuda_device)
    x = [t.to(cuda_device).requires_grad_() for t in workloads.video_qkv(geo, B=2, H=2, dtype=dtype, seed=5)]
    attn = BlockSparseAttention(block_size=64, density=0.3, geometry=geo, rope=table)
    out = attn(*x)
    w = _randn(120, *out.shape, dtype=dtype).to(cuda_device)
    (out * w).sum().backward()
    q, k = kernels.rope(x[0].detach(), x[1].detach(), table.cos, table.sin, text_len=70, layout=layout)
    live = otr.token_mask(attn.last_csr.to_dense().cpu(), geo.seq_len, geo.seq_len, 64, 64)
    plain, lse = kernels.bsa_fwd_lse(q, k, x[2].detach(), attn.last_csr, 0.125)
    assert torch.equal(plain, out)
    _check_fwd(plain, lse, q.cpu(), k.cpu(), x[2].detach().cpu(), live, 0.125)
    dq, dk, dv = kernels.bsa_bwd(w, q, k, x[2].detach(), plain, lse, attn.last_csr, 0.125)
    _check_grad((dq, dk, dv), w.cpu(), q.cpu(), k.cpu(), x[2].detach().cpu(), plain.cpu(), lse.cpu(), live, 0.125)
    dq, dk = kernels.rope(dq, dk, table.cos, table.sin, text_len=70, layout=layout, inverse=True)
    assert torch.equal(x[0].grad, dq) and torch.equal(x[1].grad, dk) and torch.equal(x[2].grad, dv)
    with torch.no_grad():  # the inference kernel; it may split dense text rows where the training forward does not
        infer = attn(*x)
    _check_fwd(infer, lse, q.cpu(), k.cpu(), x[2].detach().cpu(), live, 0.125)
    here = torch.empty_like(out)
    assert attn(*x, out=here) is here and torch.equal(here, infer)


def test_autograd_of_sums(cuda_device):
    """Expanded gradients and inputs of which only one wants a gradient."""
    q, k, v = (_randn(130 + i, 1, 2, 256, 64, dtype=BF16).to(cuda_device) for i in range(3))
    csr = kernels.mask_to_csr(torch.ones(1, 2, 2, 2, dtype=torch.bool, device=cuda_device), 128, 128)
    v.requires_grad_()
    training.sparse_attention(q, k, v, csr, 0.125).sum().backward()
    # every column of p sums over all queries, and the rows of p sum to 1: dv sums to 256 a channel
    assert torch.allclose(v.grad.float().sum(2), torch.full((1, 2, 64), 256.0, device=cuda_device), rtol=2e-2)
    table = video_rope(VideoGeometry(0, 1, 16, 16), 64, device=cuda_device)
    q.requires_grad_()
    a, _ = training.rotary(q, k, table)
    a.sum().backward()
    ref = kernels.rope(torch.ones_like(a), None, table.cos, table.sin, inverse=True)
    assert torch.equal(q.grad, ref)


@pytest.mark.parametrize("dtype,bm,H,Sq,Sk", [(BF16, 128, 1, 5000, 5000), (F16, 64, 1, 3000, 4000), (BF16, 128, 3, 4700, 3900),
                                              (BF16, 64, 1, 100, 6000)])
def test_long_lists_of_few_heads(cuda_device, dtype, bm, H, Sq, Sk):
    """Few heads with dense rows and columns: their lists are cut into parts
    that are summed afterwards (same tolerances), and give equal bits again."""
    nbq, nbk = math.ceil(Sq / bm), math.ceil(Sk / bm)
    mask = _mask(140, 1, H, nbq, nbk, 0.08)
    mask[..., :2] = True
    (gq, gk, gv, gd), out, lse, csr, grads = _run(cuda_device, 1, H, Sq, Sk, 64, dtype, bm, bm, 0, seed=141, lead=2, mask=mask)
    for _ in range(3):
        again = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)
        assert all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.parametrize("H,Sq,Sk,bm,bn", [(2, 300, 700, 64, 64), (2, 500, 333, 128, 128), (1, 200, 5000, 64, 128)])
def test_keys_with_a_common_part(cuda_device, H, Sq, Sk, bm, bn):
    """bf16 keys that share a component eight times their spread.  The rows of
    ds sum to nearly zero, so dq hardly sees it, but a rounding of ds alone
    would show eight times over (3 U).  A value rounded to nearest is off by
    2 U / sqrt(12) of its power of two in the mean square, 0.577 U of itself at
    most; 0.02 U for fp32's part (2e-6 of p, eight times over, and the sums)."""
    q, k, v, dout = (_randn(150 + i, 1, H, s, 64, dtype=F32) for i, s in enumerate((Sq, Sk, Sk, Sq)))
    q, k, v, dout = q.to(BF16), (k + 8.0).to(BF16), v.to(BF16), dout.to(BF16)
    mask = _mask(154, 1, H, math.ceil(Sq / bm), math.ceil(Sk / bn), 0.5)
    csr = kernels.mask_to_csr(mask.to(cuda_device), bm, bn)
    gq, gk, gv, gd = (t.to(cuda_device) for t in (q, k, v, dout))
    out, lse = kernels.bsa_fwd_lse(gq, gk, gv, csr, 0.125)
    dq = kernels.bsa_bwd(gd, gq, gk, gv, out, lse, csr, 0.125)[0]
    live = otr.token_mask(mask, Sq, Sk, bm, bn)
    ref = otr.attention_grad(dout, q, k, v, out.cpu(), lse.cpu(), live, 0.125)["dq"][0]
    off = np.linalg.norm(dq.double().cpu().numpy() - ref) / np.linalg.norm(ref)
    assert off <= 0.6 * U[BF16], f"{off / U[BF16]:.3f} U"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_replayed_from_a_graph(cuda_device, dtype):
    """Rotation, forward and gradient captured once and replayed on new values
    give the bits of direct calls."""
    H, S = 2, 700
    q, k, v, dout = (_randn(160 + i, 1, H, S, 64, dtype=dtype).to(cuda_device) for i in range(4))
    mask = _mask(164, 1, H, 11, 11, 0.4).to(cuda_device)
    csr = kernels.mask_to_csr(mask, 64, 64)
    table = video_rope(VideoGeometry(60, 4, 10, 16), 64, device=cuda_device)

    def step():
        a, b = kernels.rope(q, k, table.cos, table.sin, text_len=60)
        out, lse = kernels.bsa_fwd_lse(a, b, v, csr, 0.125)
        return (out, *kernels.bsa_bwd(dout, a, b, v, out, lse, csr, 0.125))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (170, 180):
        for i, x in enumerate((q, k, v, dout)):
            x.copy_(_randn(seed + i, 1, H, S, 64, dtype=dtype))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))
