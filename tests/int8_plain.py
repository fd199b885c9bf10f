"""The INT8 cache in plain numpy, 64 bits: what a row stands for, and attention over such rows with the bound its
kernels' roundings stay within."""
from __future__ import annotations

import numpy as np

AMAX_MIN, AMAX_MAX = 2.0 ** -40, 2.0 ** 64
EPS = {"bf16": 2.0 ** -7, "fp16": 2.0 ** -10, "fp32": 2.0 ** -23}          # torch.finfo(t).eps


def quantise(x):
    """Rows [..., D] -> (codes, float32 scales).  For 16-bit inputs 127 x / amax is a half-integer, exact in 64 bits, or
    more than 2^-19 of itself away from every one, so rint sees the definition's value."""
    x = np.asarray(x, dtype=np.float64)
    amax = np.clip(np.abs(x).max(axis=-1, keepdims=True), AMAX_MIN, AMAX_MAX)
    with np.errstate(invalid="ignore", over="ignore"):
        codes = np.clip(np.rint(127.0 * x / amax), -127, 127)
    return codes, (amax[..., 0].astype(np.float32) / np.float32(127.0)).astype(np.float32)


def stands_for(x):
    """The values of rows that went through the cache: code * scale, the float32 product that a read in FP32 returns."""
    codes, scale = quantise(x)
    return codes.astype(np.float32) * scale[..., None]


def attention(q, k, v, limits, out_type):
    """q [T, H, D], k and v [L, Hkv, D] (values as read back), token t sees positions < limits[t].
    -> (out [T, H, D] in 64 bits, bound on |kernel - out|).

    The kernel multiplies 16-bit probabilities with integer codes: each probability is rounded once, to fp16, by at most half
    an eps (2^-11) of itself, and what multiplies the values carries a relative error r in all, so the result is off by at
    most 2 r sum(p |v|) / sum(p) (numerator and denominator).  r adds up: 2^-11 for that rounding; the error of a score,
    (D + 8) products, sums and scalings of at most 2^-24 of sum |q k| / sqrt(D) each, which moves exp by as much; 2^-20 for
    the exponentials (two units in the last place each, a handful of factors) and the FP32 sums of the split and merged
    rows.  The result is rounded to its type once more: half an eps of it.
    What is rounded to fp16 is w_j = p_j vs_j / 2^m (vs the value's scale), 2^m at most the largest p_j vs_j: where w_j is
    below fp16's normal range its error is not 2^-11 of itself but half of fp16's smallest step, 2^-25.  It multiplies the
    code, v_j / vs_j, and 2^m: at most 2^-25 max(p vs) sum |v_j / vs_j| / sum(p) in all."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    T, H, D = q.shape
    G = H // k.shape[1]
    out, bound = np.zeros((T, H, D)), np.zeros((T, H, D))
    vs = np.maximum(np.abs(v).max(axis=-1), 127.0 * 2.0 ** -48) / 127.0     # a row's largest code is 127 (or the row is zero)
    for h in range(H):
        s = q[:, h] @ k[:, h // G].T / np.sqrt(D)
        mag = np.abs(q[:, h]) @ np.abs(k[:, h // G]).T / np.sqrt(D)
        seen = np.arange(k.shape[0])[None, :] < np.asarray(limits)[:, None]
        s = np.where(seen, s, -np.inf)
        top = s.max(axis=-1, keepdims=True, initial=-1e30)
        p = np.where(seen, np.exp(np.minimum(s - top, 0.0)), 0.0)
        total = p.sum(axis=-1, keepdims=True) + 1e-8
        out[:, h] = p @ v[:, h // G] / total
        r = 2.0 ** -11 + (D + 8) * 2.0 ** -24 * np.where(seen, mag, 0.0).max(axis=-1, keepdims=True, initial=0.0) + 2.0 ** -20
        w, codes = (p * vs[:, h // G]).max(axis=-1, keepdims=True, initial=0.0), np.abs(v[:, h // G]) / vs[:, h // G, None]
        bound[:, h] = 2.0 * r * (p @ np.abs(v[:, h // G]) / total) + 2.0 ** -25 * w * (seen @ codes) / total
    return out, bound + EPS[out_type] / 2 * (np.abs(out) + bound) + 1e-30


def check(got, want, bound, what=""):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == want.shape, f"{what}: shape {got.shape} vs {want.shape}"
    assert np.isfinite(got).all(), f"{what}: non-finite values"
    over = np.abs(got - want) / bound
    assert (over <= 1.0).all(), f"{what}: error is {over.max():.2f} of its bound at {np.unravel_index(over.argmax(), over.shape)}"
