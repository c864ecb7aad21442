"""fp64 restatement of the training-side operators (test infrastructure; see
``oracle/__init__.py``): block-sparse attention with its row log-sum-exp, its
gradient, and rotary positions.  Dense token masks, one head at a time, with
the error scales that the tests' tolerances are made of.
"""
from __future__ import annotations

import numpy as np

from .selection import to_f64


def token_mask(mask, Sq: int, Sk: int, bm: int, bn: int) -> np.ndarray:
    """bool ``[B, H, Sq, Sk]`` from a block mask ``[B, H, nbq, nbk]``."""
    m = np.asarray(to_f64(mask) != 0)
    return m.repeat(bm, axis=2).repeat(bn, axis=3)[:, :, :Sq, :Sk]


def attention(q, k, v, live, scale: float):
    """``(out, lse)`` under a token mask; a row that sees nothing gives zeros and -inf."""
    q, k, v = to_f64(q), to_f64(k), to_f64(v)
    s = np.where(live, (q @ k.swapaxes(-1, -2)) * scale, -np.inf)
    top = s.max(-1, keepdims=True)
    top = np.where(np.isfinite(top), top, 0.0)
    e = np.where(live, np.exp(s - top), 0.0)
    total = e.sum(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        lse = (top + np.log(total))[..., 0]
    return e @ v / np.where(total > 0, total, 1.0), lse


def attention_grad(dout, q, k, v, out, lse, live, scale: float):
    """Gradients and, for each, the sums of absolute terms that rounding errors
    scale with: ``{"dq": (value, by ds, by p), ...}``: ``by ds`` sums |ds| (or
    |p| for dv) times the other factor, ``by p`` sums p (|do||v| + |delta|)
    times it, the size of what ds is the difference of."""
    do, q, k, v, out, lse = (to_f64(x) for x in (dout, q, k, v, out, lse))
    s = (q @ k.swapaxes(-1, -2)) * scale
    p = np.where(live, np.exp(np.where(live, s - np.where(np.isfinite(lse), lse, 0.0)[..., None], 0.0)), 0.0)
    dp = do @ v.swapaxes(-1, -2)
    delta = (do * out).sum(-1, keepdims=True)
    ds = p * (dp - delta)
    size = p * (np.abs(do) @ np.abs(v).swapaxes(-1, -2) + np.abs(delta))
    t = lambda x: x.swapaxes(-1, -2)  # noqa: E731
    return {
        "dq": (scale * (ds @ k), scale * (np.abs(ds) @ np.abs(k)), scale * (size @ np.abs(k))),
        "dk": (scale * (t(ds) @ q), scale * (t(np.abs(ds)) @ np.abs(q)), scale * (t(size) @ np.abs(q))),
        "dv": (t(p) @ do, t(p) @ np.abs(do), t(p) @ np.abs(do)),
    }


def rope(x, cos, sin, text_len: int, layout: str, inverse: bool) -> np.ndarray:
    x, cos, sin = to_f64(x), to_f64(cos), to_f64(sin)
    y = x.copy()
    half = cos.shape[-1]
    cos, sin = (c[:, None] if c.ndim == 3 else c for c in (cos, -sin if inverse else sin))
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if layout == "interleaved" else \
        (slice(0, half), slice(half, 2 * half))
    a, b = x[:, :, text_len:, first], x[:, :, text_len:, second]
    y[:, :, text_len:, first] = a * cos - b * sin
    y[:, :, text_len:, second] = b * cos + a * sin
    return y
