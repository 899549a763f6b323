"""Float64 oracle for the RMS norm, the 8-bit rows and their matrix product (TEST INFRASTRUCTURE ONLY).

Written from the definitions; the operators have no counterpart in the reference.
  rms_norm       y = s r w with r = 1 / sqrt(mean(s^2) + eps), s = x or x + residual held in 16 bits
  rms_norm_bwd   g = dy w, xh = s r: ds = r (g - xh mean(g xh)) + dsum, dw = sum over rows of dy xh
  quotients      127 t / a of each row t with largest magnitude a: 8-bit rows hold its nearest
                 integers, and a / 127 as their scale
  nearest        those integers of fp32 values, ties to even, exactly
  hidden         x, relu(x), or swish of x's first half times its second
  project        (q w^T) sx sw + b + residual, the sum of integers exact

Pinned by (tests/test_rows8.py): the gradients against central differences of rms_norm, the rounding to
16 bits against torch's conversions, the matrix product against an explicit sum and the
nearest integers against fractions.
"""
import numpy as np

TINY = 2.0 ** -119  # rows whose largest magnitude is below it are zeros with scale 0


def round16(v, kind):
    """v rounded to fp16 or bf16 (kind "f16" or "bf16"), ties to even, as float64."""
    v = np.asarray(v, np.float64)
    if kind == "f16":
        with np.errstate(over="ignore"):
            return v.astype(np.float16).astype(np.float64)
    _, e = np.frexp(np.where(np.isfinite(v), v, 0.0))
    step = np.ldexp(1.0, np.maximum(e, -125) - 8)
    out = np.where(np.isfinite(v), np.rint(v / step) * step, v)
    return np.where(np.abs(out) > 3.3895313892515355e38, np.copysign(np.inf, out), out)


def rms_norm(s, w, eps):
    """(y, rstd) of s [M,C]."""
    s = np.asarray(s, np.float64)
    r = 1.0 / np.sqrt((s * s).mean(1) + eps)
    return s * r[:, None] * np.asarray(w, np.float64), r


def rms_norm_bwd(s, w, dy, dsum, eps):
    """(ds, dw)."""
    s, w, dy = (np.asarray(t, np.float64) for t in (s, w, dy))
    r = 1.0 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
    xh, g = s * r, dy * w
    ds = r * (g - xh * (g * xh).mean(1, keepdims=True))
    return (ds if dsum is None else ds + np.asarray(dsum, np.float64)), (dy * xh).sum(0)


def quotients(t):
    """(127 t / a, a / 127) of rows t: zeros where a is under TINY, zeros and NaN where a row is not finite."""
    t = np.asarray(t, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.abs(t).max(1)
        finite = np.isfinite(t).all(1)
        live = finite & (a >= TINY)
        q = np.where(live[:, None], 127.0 * np.where(live[:, None], t, 0.0) / np.where(live, a, 1.0)[:, None], 0.0)
    return q, np.where(finite, np.where(live, a / 127.0, 0.0), np.nan)


def hidden(x, activation):
    x = np.asarray(x, np.float64)
    if activation == 1:
        return np.where(x < 0, 0.0, x)
    if activation == 2:
        g, u = np.split(x, 2, axis=1)
        with np.errstate(over="ignore"):
            return g / (1.0 + np.exp(-g)) * u
    return x


def project(q, sx, w, sw, b=None, residual=None):
    """(out, sum of the terms' magnitudes) for integers q [M,K], w [N,K]."""
    s = (np.asarray(q, np.float64) @ np.asarray(w, np.float64).T) * np.asarray(sx, np.float64)[:, None] * np.asarray(
        sw, np.float64)
    out, mag = s, np.abs(s)
    for t in (b, residual):
        if t is not None:
            out = out + np.asarray(t, np.float64)
            mag = mag + np.abs(np.asarray(t, np.float64))
    return out, mag


def nearest(t):
    """127 t / a of rows t of fp32 values to the nearest integer, ties to even, without a rounding before it: 127 t and
    (n + 1/2) a are exact in float64."""
    t = np.asarray(t, np.float64)
    a = np.abs(t).max(1, keepdims=True)
    live = a >= TINY
    num, a = np.where(live, 127.0 * t, 0.0), np.where(live, a, 1.0)
    n = np.rint(num / a)
    odd = n % 2 == 1
    up, down = num - (n + 0.5) * a, num - (n - 0.5) * a
    return n + ((up > 0) | (odd & (up == 0))) - ((down < 0) | (odd & (down == 0)))
