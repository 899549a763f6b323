"""Weight re-layouts between the callers' natural weight shapes and the FFI targets' layouts.

The reference's FFI targets take their weights transposed or blocked; the callers' wrappers
(colabfold_kernels.fused_ops, not part of the reference repository) re-lay them out before each
call. The target layouts are fixed by the reference's FFI comments and kernels:

  ln_gated_dual_proj  wp, wg [K, P] -> wpT, wgT [P, K]          (cuda/volta_fused_ffi.h:42-43)
  trimul_epilogue     wo [C, O] -> woT [O, C]; wg [CA, O] -> wgT [O, CA]   (volta_fused_ffi.h:82-91)
  ln_projection       w [slots, K, n] -> wT [slots n, K], slot major;
                      wb [K, heads] -> wbT [heads, K]            (volta_fused_ffi.h:135-136)
  output_projection   w [K, N] -> wT [N, K]                      (volta_fused_ffi.h:178)
  transition          w1 [C, H] -> w1T [H, C]; w2 [H, C] -> w2T [H/64][C][64] with
                      w2T[j][c][i] = w2[64 j + i][c]             (volta_fused_ffi.h:216-217)

and the layout of the 8-bit projection's weights, which has no counterpart there:

  q8_projection       q [N, Kp] (8-bit rows of w^T, Kp a multiple of 64) ->
                      wq [ceil(N/64), Kp/64, 4, 4, 16, 16]

and what the heads' rotation and the key-value cache hold, which have none either:

  rope_table          [positions, r]: the cosines and sines of each position's angles
  keys_blocked, values_blocked  [pages, heads, page, d] in the order of the tokens -> in the cache's

Each function takes and returns torch tensors (any device) or numpy arrays, and returns a
contiguous result of the input's dtype (rope_table makes a torch tensor).
"""

HIDDEN_CHUNK = 64  # rows of w2 per block of the transition's blocked layout


def _contig(x):
    if hasattr(x, "contiguous"):
        return x.contiguous()
    import numpy as np
    return np.ascontiguousarray(x)


def _t(x):
    """The 2-D transpose, contiguous."""
    if x.ndim != 2:
        raise ValueError("expected a 2-D weight, got shape %s" % (tuple(x.shape),))
    return _contig(x.T)


def proj_pair_T(wp, wg):
    """wp, wg [K, P] -> wpT, wgT [P, K] (ln_gated_dual_proj)."""
    return _t(wp), _t(wg)


def linear_T(w):
    """w [K, N] -> wT [N, K] (output_projection, trimul_epilogue's wo and wg, transition's w1)."""
    return _t(w)


def slot_major(w):
    """w [slots, K, n] -> wT [slots n, K], slot major: wT[s n + j, k] = w[s, k, j] (ln_projection)."""
    if w.ndim != 3:
        raise ValueError("expected w [slots, K, n], got shape %s" % (tuple(w.shape),))
    slots, k, n = w.shape
    if hasattr(w, "permute"):
        return w.permute(0, 2, 1).reshape(slots * n, k).contiguous()
    return _contig(w.transpose(0, 2, 1).reshape(slots * n, k))


def heads_T(wb):
    """wb [K, heads] -> wbT [heads, K] (ln_projection's head bias)."""
    return _t(wb)


def w2_blocked(w2):
    """w2 [H, C] -> w2T [H/64][C][64], w2T[j][c][i] = w2[64 j + i][c] (transition)."""
    if w2.ndim != 2 or w2.shape[0] % HIDDEN_CHUNK:
        raise ValueError("expected w2 [H, C] with H a multiple of 64, got shape %s" % (tuple(w2.shape),))
    h, c = w2.shape
    blocks = w2.reshape(h // HIDDEN_CHUNK, HIDDEN_CHUNK, c)
    if hasattr(blocks, "permute"):
        return blocks.permute(0, 2, 1).contiguous()
    return _contig(blocks.transpose(0, 2, 1))


def w2_unblocked(w2T):
    """The inverse of w2_blocked: [H/64][C][64] -> w2 [H, C]."""
    j, c, i = w2T.shape
    if hasattr(w2T, "permute"):
        return w2T.permute(0, 2, 1).reshape(j * i, c).contiguous()
    return _contig(w2T.transpose(0, 2, 1).reshape(j * i, c))


Q8_BLOCK = 64  # channels and inputs of a block of the 8-bit weights


def q8_blocked(q):
    """q [N, Kp] -> wq [ceil(N/64), Kp/64, 4, 4, 16, 16] (q8_projection): blocks of 64 channels by 64
    inputs, wq[., ., b, c, 4 g + i, j] = q[channel 16 g + 4 b + i, input 16 c + j] of the block, zeros
    for channels past N."""
    if q.ndim != 2 or q.shape[1] % Q8_BLOCK:
        raise ValueError("expected q [N, Kp] with Kp a multiple of 64, got shape %s" % (tuple(q.shape),))
    n, kp = q.shape
    blocks = -(-n // Q8_BLOCK)
    if hasattr(q, "new_zeros"):
        p = q.new_zeros((blocks * Q8_BLOCK, kp))
        p[:n] = q
        return p.view(blocks, 4, 4, 4, kp // 64, 4, 16).permute(0, 4, 2, 5, 1, 3, 6).reshape(
            blocks, kp // 64, 4, 4, 16, 16).contiguous()
    import numpy as np
    p = np.zeros((blocks * Q8_BLOCK, kp), q.dtype)
    p[:n] = q
    return np.ascontiguousarray(p.reshape(blocks, 4, 4, 4, kp // 64, 4, 16).transpose(
        0, 4, 2, 5, 1, 3, 6).reshape(blocks, kp // 64, 4, 4, 16, 16))


def q8_unblocked(wq, n):
    """The inverse of q8_blocked: wq -> q [n, Kp]."""
    blocks, kbs = wq.shape[:2]
    p = wq.reshape(blocks, kbs, 4, 4, 4, 4, 16)
    p = p.permute(0, 4, 2, 5, 1, 3, 6) if hasattr(p, "permute") else p.transpose(0, 4, 2, 5, 1, 3, 6)
    return _contig(p.reshape(blocks * Q8_BLOCK, kbs * Q8_BLOCK)[:n])


def rope_table(positions, r, base=10000.0, device="cpu"):
    """rope [positions, r] fp32 (hip.qk_norm_rope): row p holds cos(p f_i), i < r / 2, then sin(p f_i), f_i = base^(-2 i / r),
    computed in float64."""
    import torch
    f = float(base) ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * f
    return torch.cat([angles.cos(), angles.sin()], 1).to(torch.float32).to(device)


CACHE_BLOCK = 16  # tokens of a block of the cache


def _cache_dims(x):
    if x.ndim != 4 or x.shape[2] % CACHE_BLOCK or x.shape[3] % 32:
        raise ValueError("expected [pages, heads, page, d], page a multiple of 16 and d of 32, got shape %s" % (tuple(x.shape),))
    item = x.element_size() if hasattr(x, "element_size") else x.dtype.itemsize
    p, h, n, d = x.shape
    return p, h, n // CACHE_BLOCK, d, 16 if item == 1 else 8, 4 if item == 1 and d % 64 == 0 else 2


def _reordered(x, shape, order):
    y = x.reshape(shape)
    return _contig((y.permute(*order) if hasattr(y, "permute") else y.transpose(order)).reshape(x.shape))


def keys_blocked(k):
    """k [pages, heads, page, d] -> the cache's order: blocks of 16 tokens as [d / w][16][w], w = 8 (16 bits) or 16 (8 bits)
    channels."""
    p, h, blocks, d, w, _ = _cache_dims(k)
    return _reordered(k, (p, h, blocks, 16, d // w, w), (0, 1, 2, 4, 3, 5))


def keys_unblocked(k):
    """The inverse of keys_blocked."""
    p, h, blocks, d, w, _ = _cache_dims(k)
    return _reordered(k, (p, h, blocks, d // w, 16, w), (0, 1, 2, 4, 3, 5))


def values_blocked(v):
    """v [pages, heads, page, d] -> the cache's order: blocks of 16 tokens as [d / (16 c)][4 g][16 i][c e][4 j], token 4 g + j,
    channel 16 (c b + e) + i; c = 2, or 4 for 8 bits where d is a multiple of 64."""
    p, h, blocks, d, _, c = _cache_dims(v)
    return _reordered(v, (p, h, blocks, 4, 4, d // (16 * c), c, 16), (0, 1, 2, 5, 3, 7, 6, 4))


def values_unblocked(v):
    """The inverse of values_blocked."""
    p, h, blocks, d, _, c = _cache_dims(v)
    return _reordered(v, (p, h, blocks, d // (16 * c), 4, 16, c, 4), (0, 1, 2, 4, 7, 3, 6, 5))
