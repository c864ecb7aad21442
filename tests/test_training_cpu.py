"""Rotary tables, refusals and host-side argument checks of the training-side
operators (no GPU), and the fp64 oracle's gradient against differences."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import training as otr
from sparseattnfunctions_b200 import _lib, kernels
from sparseattnfunctions_b200.geometry import VideoGeometry
from sparseattnfunctions_b200.rope import RopeScaling, rope_freqs, rope_table, video_rope


def test_video_table_follows_the_grid():
    geo = VideoGeometry(3, 2, 3, 4)
    t = video_rope(geo, 64)
    assert t.cos.shape == t.sin.shape == (24, 32) and t.cos.dtype == torch.float32
    assert (t.text_len, t.layout) == (3, "interleaved")
    for f in range(2):
        for h in range(3):
            for w in range(4):
                row = (f * 3 + h) * 4 + w
                for start, d, pos in ((0, 16, f), (8, 24, h), (20, 24, w)):
                    for m in range(d // 2):
                        angle = pos * 10000.0 ** (-2 * m / d)
                        # the stored value is the 64-bit one rounded once
                        assert float(t.cos[row, start + m]) == pytest.approx(math.cos(angle), abs=2 ** -24)
                        assert float(t.sin[row, start + m]) == pytest.approx(math.sin(angle), abs=2 ** -24)


def test_far_positions_keep_their_angle():
    pos = torch.tensor([[1_000_003]])
    cos, sin = rope_table(pos, (8,))
    assert float(cos[0, 0]) == pytest.approx(math.cos(1_000_003), abs=1e-7)
    assert float(sin[0, 1]) == pytest.approx(math.sin(1_000_003 * 10000.0 ** -0.25), abs=1e-7)


def test_scaling_rules():
    base = rope_freqs(24)
    assert torch.equal(rope_freqs(24, scaling=RopeScaling("linear", 4.0)), base / 4.0)
    ntk = rope_freqs(24, scaling=RopeScaling("ntk", 4.0))
    assert float(ntk[0]) == 1.0 and float(ntk[-1]) == pytest.approx(float(base[-1]) / 4.0, rel=1e-12)
    yarn = rope_freqs(64, scaling=RopeScaling("yarn", 4.0, trained_len=4096))
    ratio = rope_freqs(64) / yarn
    turns = 4096 * rope_freqs(64) / (2 * math.pi)
    assert torch.allclose(ratio[turns > 32], torch.ones(1, dtype=torch.float64))
    assert torch.allclose(ratio[turns < 1], torch.full((1,), 4.0, dtype=torch.float64))
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and bool(((ratio[mid] > 1) & (ratio[mid] < 4)).all())
    cos, sin = rope_table(torch.arange(5)[:, None], (64,), scaling=RopeScaling("yarn", 4.0, trained_len=4096))
    amp = 0.1 * math.log(4.0) + 1.0
    assert torch.allclose(cos * cos + sin * sin, torch.full_like(cos, amp * amp), rtol=1e-6)
    for kind in ("linear", "ntk"):
        assert torch.equal(rope_freqs(24, scaling=RopeScaling(kind, 1.0)), base)


@pytest.mark.parametrize("bad", [
    lambda: RopeScaling("cubic", 2.0), lambda: RopeScaling("linear", 0.5), lambda: RopeScaling("yarn", 2.0),
    lambda: RopeScaling("yarn", 2.0, 128, low=4, high=4), lambda: rope_freqs(7), lambda: rope_freqs(8, theta=0),
    lambda: rope_table(torch.zeros(4, 2), (8,)), lambda: video_rope(VideoGeometry(0, 1, 1, 1), 72),
    lambda: video_rope(VideoGeometry(0, 1, 1, 1), 64, dims=(32, 32, 32))])
def test_table_refusals(bad):
    with pytest.raises(ValueError):
        bad()


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 1, 64, 64)
    csr = kernels.BlockCSR(torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 1, 1, 1, 1, 64, 64)
    with pytest.raises(ValueError):
        kernels.bsa_fwd_lse(x, x, x, csr, 0.125)
    with pytest.raises(ValueError):
        kernels.bsa_bwd(x, x, x, x, x, torch.zeros(1, 1, 64), csr, 0.125)
    with pytest.raises(ValueError):
        kernels.rope(x, x, torch.zeros(64, 32), torch.zeros(64, 32))


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from sparseattnfunctions_b200 import build

        build.build()
    return _lib.load()


def _t4(dtype=_lib.SAF_BF16, data=0x10000, B=1, H=2, S=256, D=64):
    t = _lib.Tensor4()
    t.data, t.dtype = data, dtype
    t.B, t.H, t.S, t.D = B, H, S, D
    t.stride_s, t.stride_h, t.stride_b = D, S * D, H * S * D
    return t


def test_gradient_rejects_bad_arguments_on_host(lib):
    """Every call fails before the device is touched."""
    p = 0x10000

    def call(change=None, lse=p, rp=p, scale=0.125, ws=p, ws_bytes=1 << 40, bm=128, bn=128, cap=16, dtype=_lib.SAF_BF16, stride=256):
        t = {n: _t4(dtype) for n in ("dout", "q", "k", "v", "out", "dq", "dk", "dv")}
        t.update(change or {})
        r = {n: ctypes.byref(x) for n, x in t.items()}
        return lib.saf_bsa_bwd(r["dout"], r["q"], r["k"], r["v"], r["out"], lse, stride, r["dq"], r["dk"], r["dv"], rp, p, cap,
                               bm, bn, scale, ws, ws_bytes, None)

    assert call({"q": _t4(data=0)}) == _lib.SAF_ERR_ARG
    assert call(lse=None) == call(rp=None) == call(cap=-1) == _lib.SAF_ERR_ARG
    assert call(scale=0.0) == call(scale=-1.0) == call(scale=math.inf) == call(scale=math.nan) == _lib.SAF_ERR_ARG
    assert call({"dk": _t4(_lib.SAF_F16)}) == _lib.SAF_ERR_DTYPE
    assert call({"dout": _t4(S=128)}) == call({"dv": _t4(S=128)}) == call({"k": _t4(H=1)}) == _lib.SAF_ERR_SHAPE
    assert call({"dout": _t4(data=0x10008)}) == _lib.SAF_ERR_STRIDE
    odd = _t4()
    odd.stride_s = 68
    assert call({"dq": odd}) == _lib.SAF_ERR_STRIDE
    assert call(stride=255) == _lib.SAF_ERR_STRIDE
    assert call(bm=32) == call(bn=192) == _lib.SAF_ERR_UNSUPPORTED
    wide = {n: _t4(D=128) for n in ("dout", "q", "k", "v", "out", "dq", "dk", "dv")}
    assert call(wide) == _lib.SAF_ERR_UNSUPPORTED
    assert call(ws=None) == call(ws_bytes=64) == _lib.SAF_ERR_WORKSPACE
    q = _t4()
    assert lib.saf_bsa_bwd_workspace_bytes(ctypes.byref(q), ctypes.byref(q), 128, 128) > 0
    assert lib.saf_bsa_bwd_workspace_bytes(ctypes.byref(q), ctypes.byref(q), 32, 128) == 0
    long = _t4(S=16384 * 64 + 1)
    assert lib.saf_bsa_bwd_workspace_bytes(ctypes.byref(long), ctypes.byref(q), 64, 64) == 0


def test_training_forward_rejects_bad_arguments_on_host(lib):
    p, q, o = 0x10000, _t4(), _t4()

    def call(k=q, lse=p, scale=0.125, bm=128, lead=0):
        return lib.saf_bsa_fwd_lse(ctypes.byref(q), ctypes.byref(k), ctypes.byref(k), ctypes.byref(o), p, p, 16, bm, 128,
                                   scale, lead, lse, None, 0, None)

    assert call(lse=None) == call(scale=0.0) == call(scale=math.nan) == call(bm=0) == call(lead=-1) == _lib.SAF_ERR_ARG
    assert call(_t4(_lib.SAF_F16)) == _lib.SAF_ERR_DTYPE
    assert call(_t4(D=128)) == _lib.SAF_ERR_SHAPE


def test_rope_rejects_bad_arguments_on_host(lib):
    p = 0x10000

    def call(q=None, k=None, oq=None, ok=None, R=64, text=0, table=p):
        q, k, oq, ok = (x or _t4() for x in (q, k, oq, ok))
        return lib.saf_rope(ctypes.byref(q), ctypes.byref(k), ctypes.byref(oq), ctypes.byref(ok), table, table, 0, text,
                            R, 0, 0, None)

    assert call(R=0) == call(R=7) == call(R=66) == _lib.SAF_ERR_SHAPE
    assert call(text=-1) == call(text=257) == _lib.SAF_ERR_SHAPE
    assert call(k=_t4(S=128), ok=_t4(S=128)) == call(oq=_t4(H=1)) == _lib.SAF_ERR_SHAPE
    assert call(ok=_t4(_lib.SAF_F32)) == _lib.SAF_ERR_DTYPE
    assert call(table=None) == _lib.SAF_ERR_ARG
    q = _t4()
    assert lib.saf_rope(ctypes.byref(q), None, ctypes.byref(q), ctypes.byref(q), p, p, 0, 0, 64, 0, 0,
                        None) == _lib.SAF_ERR_ARG


def test_oracle_gradient_against_differences():
    """d/dx of sum(out * w) along random directions, by central differences of
    the fp64 forward, equals the formula's gradient: both have relative errors
    near h^2 = 1e-8 and 2^-53 / h = 1e-12."""
    g = torch.Generator().manual_seed(3)
    B, H, Sq, Sk, D = 1, 2, 9, 11, 8
    q, k, v, w = (torch.randn(B, H, n, D, generator=g, dtype=torch.float64).numpy() for n in (Sq, Sk, Sk, Sq))
    live = (torch.rand(B, H, Sq, Sk, generator=g) < 0.6).numpy()
    live[:, :, 4] = False
    out, lse = otr.attention(q, k, v, live, 0.4)
    grads = otr.attention_grad(w, q, k, v, out, lse, live, 0.4)
    assert np.all(out[:, :, 4] == 0) and np.all(np.isneginf(lse[:, :, 4]))
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn((q, k, v)[i].shape, generator=g, dtype=torch.float64).numpy()
        h = 1e-4
        side = []
        for sign in (1, -1):
            x = [q, k, v]
            x[i] = x[i] + sign * h * way
            side.append(float((otr.attention(*x, live, 0.4)[0] * w).sum()))
        assert (side[0] - side[1]) / (2 * h) == pytest.approx(float((grads[name][0] * way).sum()), rel=1e-6, abs=1e-8)
