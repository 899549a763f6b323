"""Float64 oracle for the heads' norm and rotation, the key-value cache and its attention (TEST INFRASTRUCTURE ONLY).

Written from the definitions; the operators have no counterpart in the reference.
  rotate         pairs (a, b) of a head's first R channels -> (a cos - b sin, a sin + b cos)
  norm_rope      x r w rotated, r = 1 / sqrt(mean(x^2) + eps), and a bound of what each value is summed from
  norm_rope_bwd  its gradients, and what each is summed from
  blocked        one page's head [page, d] in the cache's order, place by place
  attend         softmax(scale q K^T) V of one token, its lse in the log2 domain, sum p |v| and the largest sum |q k|

Pinned by (tests/test_heads.py): the gradients against central differences, the rotation against complex numbers, the
order against hip's documented places, attention against a direct sum.
"""
import numpy as np


def pairs(r, interleaved):
    """The channels of the r / 2 pairs: (first of each, second of each)."""
    i = np.arange(r // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)


def rotate(x, cos, sin, interleaved):
    """x [T, H, D] by cos, sin [T, r / 2]."""
    a, b = pairs(2 * cos.shape[1], interleaved)
    y = np.array(x, np.float64)
    c, s = cos[:, None], sin[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def partner_sum(x, r, interleaved):
    """|x| of each channel plus that of the one that it is rotated with."""
    y = np.abs(np.asarray(x, np.float64))
    a, b = pairs(r, interleaved)
    both = y[..., a] + y[..., b]
    y[..., a] = both
    y[..., b] = both
    return y


def _angles(rope, positions):
    rows = np.asarray(rope, np.float64)[positions]
    return np.split(rows, 2, axis=1)


def norm_rope(x, w, rope, positions, eps, interleaved):
    """(y, terms) of heads x [T, H, D]."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    cos, sin = _angles(rope, positions)
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    return rotate(n, cos, sin, interleaved), partner_sum(n, 2 * cos.shape[1], interleaved)


def norm_rope_bwd(x, w, rope, positions, dy, eps, interleaved):
    """(dx, its terms, dw, its terms)."""
    x, w, dy = (np.asarray(t, np.float64) for t in (x, w, dy))
    cos, sin = _angles(rope, positions)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh = x * r
    back = rotate(dy, cos, -sin, interleaved)
    size = partner_sum(dy, 2 * cos.shape[1], interleaved)
    g = back * w
    dx = r * (g - xh * (g * xh).mean(-1, keepdims=True))
    terms = r * (size * np.abs(w) + np.abs(xh) * (size * np.abs(w * xh)).mean(-1, keepdims=True))
    return dx, terms, (back * xh).sum((0, 1)), (size * np.abs(xh)).sum((0, 1))


def blocked(x, values, eight_bit):
    """x [page, d] as the cache holds it, [page, d] too."""
    n, d = x.shape
    out = np.empty_like(x).reshape(n // 16, 16 * d)
    c = 4 if eight_bit and d % 64 == 0 else 2
    w = 16 if eight_bit else 8
    for t in range(n):
        for ch in range(d):
            s = t % 16
            if values:
                b, e, i = ch // (16 * c), ch // 16 % c, ch % 16
                at = (((b * 4 + s // 4) * 16 + i) * c + e) * 4 + s % 4
            else:
                at = (ch // w * 16 + s) * w + ch % w
            out[t // 16, at] = x[t, ch]
    return out.reshape(n, d)


def attend(q, k, v, scale):
    """(out [G, D], lse [G], sum of p |v| / sum of p, largest sum of |q k| over the keys) of q [G, D] over k, v [n, D]."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    if len(k) == 0:
        return np.zeros_like(q), np.full(len(q), -np.inf), np.zeros_like(q), np.zeros(len(q))
    x = q @ k.T * scale
    m = x.max(1, keepdims=True)
    p = np.exp(x - m)
    total = p.sum(1, keepdims=True)
    return (p @ v / total, (m + np.log(total))[:, 0] / np.log(2.0), p @ np.abs(v) / total,
            (np.abs(q) @ np.abs(k).T).max(1) * abs(scale))
