"""Caller glue for PyTorch: what the reference's callers wrap around the FFI targets.

The reference repository ships the FFI targets only; its callers (the external
colabfold_kernels package) wire them into the framework. Its tests show the pieces this module
provides on top of `hip` (the C ABI binding):

  attention        the forward + backward pair as one differentiable op: VoltaMma with want_lse,
                   its lse kept for VoltaMmaBwd, and dbias cast to the bias dtype
                   (tests/test_attn_bwd.py:262-281, the custom_vjp wiring)
  gated_attention  attention times sigmoid(gate + gate_bias), the gated packed forward's
                   epilogue (cuda/volta_attn.h:46-52) as a differentiable op, so the gate gets
                   its gradient
  trim_limits      each batch row's last live key + 1, then the largest: the lims of
                   VoltaMmaPackedTrim (tests/test_packed_attention.py:53-57)
  ln_gated_dual_proj, trimul_epilogue_ln, ln_projection, output_projection, transition
                   the fused targets with the callers' natural weight shapes, re-laid out by
                   colabfold_legacy_kernels.layouts, and leading batch dimensions folded into
                   the row count (tests/test_fused.py:96-229 calls them so)
  fused_available  whether a fused target takes a width and dtype (tests/test_fused.py:223-229:
                   other widths and dtypes decline to the caller's own path)
  rms_norm         RMS norm with the residual's addition, differentiable in the input, the residual
                   and the scale
  rms_norm_q8, quantize_rows, dequantize_rows, q8_weights, q8_projection, q8_transition
                   the 8-bit serving path: norms and activations as 8-bit rows, weights quantised
                   once, projections and an MLP in 8-bit products (no counterpart in the reference)
  qk_norm_rope     a projection's queries, keys and values apart, queries and keys with each head's RMS norm and the
                   position rotation, differentiable
  cache_slots, qk_norm_rope_cache, kv_cache_write, kv_cache_read, paged_attention
                   attention over a paged key-value cache, in 16 or 8 bits, one new token a sequence (no counterpart
                   in the reference)

Everything runs on the GPU through the built library; there is no CPU path. The fused and the
8-bit wrappers are forward only (the reference's callers take their gradients from jnp references). They take
fp16 or bf16 activations, with weights and biases cast to fp16 for the kernels.
"""
import torch
from torch.autograd import forward_ad

from . import hip
from . import layouts

# (D, block_q, block_k) each head dim runs with by default: an entry of the reference's forward
# dispatch set (cuda/volta_mma_attn.cu:508-517), (64, 64) where D = 64 has no (64, 32)
_DEFAULT_BLOCKS = {8: (64, 32), 16: (64, 32), 24: (64, 32), 32: (64, 32), 48: (64, 32),
                   64: (64, 64), 96: (64, 32)}


def default_blocks(d):
    if d not in _DEFAULT_BLOCKS:
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "attention: unsupported head dim %d" % d)
    return _DEFAULT_BLOCKS[d]


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, kmask, scale, block_q, block_k):
        q, k, v, bias, kmask = (t.contiguous() for t in (q, k, v, bias, kmask))
        out, lse = hip.attention_fwd(q, k, v, bias, kmask, scale, block_q, block_k, want_lse=True)
        ctx.save_for_backward(q, k, v, bias, kmask, out, lse)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, bias, kmask, out, lse = ctx.saved_tensors
        want_dbias = bool(ctx.needs_input_grad[3])
        dq, dk, dv, dbias = hip.attention_bwd(q, k, v, bias, kmask, out,
                                              dout.to(torch.float16).contiguous(), lse, ctx.scale,
                                              want_dbias=want_dbias)
        return dq, dk, dv, (dbias.to(bias.dtype) if want_dbias else None), None, None, None, None


def attention(q, k, v, bias, kmask, scale=None, block_q=None, block_k=None):
    """Biased, masked attention [N,H,Sq,D] fp16, differentiable in q, k, v and bias.

    q [N,H,Sq,D], k, v [N,H,Sk,D], bias [H,Sq,Sk] fp16; kmask [N,Sk] (nonzero keeps a key).
    scale defaults to D^-1/2. The backward is VoltaMmaBwd with want_dbias only where bias needs
    a gradient; dbias (fp32, summed over the N rows) is cast to the bias dtype.
    """
    d = q.shape[-1]
    bq, bk = default_blocks(d) if block_q is None else (block_q, block_k)
    if kmask.dtype != torch.uint8:
        kmask = (kmask != 0).to(torch.uint8)
    return _Attention.apply(q, k, v, bias, kmask, float(d ** -0.5 if scale is None else scale),
                            int(bq), int(bk))


def gated_attention(q, k, v, bias, kmask, gate, gate_bias=None, scale=None):
    """attention(...) * sigmoid(gate + gate_bias), differentiable in the gate too.

    gate [N,H,Sq,D]; gate_bias [H,D] or [H*D] (zeros if None). The attention output o comes back
    from the kernel already rounded to fp16; the product o * sigmoid(g) is taken in fp32 and
    rounded to fp16 again. The result therefore carries two roundings, where the reference's gated
    packed forward gates the fp32 output and rounds once (cuda/volta_attn.h:46-52): the two
    differ by at most about one fp16 ulp of the result (|sigmoid| <= 1, so o's rounding error of
    half an ulp of o is at most half an ulp of the product's scale, plus the product's own half
    ulp). VoltaMmaPacked with G = 4 (attention_packed) is the single-rounding forward."""
    o = attention(q, k, v, bias, kmask, scale)
    g = gate.float()
    if gate_bias is not None:
        h, d = q.shape[1], q.shape[3]
        g = g + gate_bias.float().reshape(1, h, 1, d)
    return (o.float() * torch.sigmoid(g)).to(torch.float16)


def trim_limits(kmask):
    """lims [N+1] int32 on kmask's device: for each batch row its last live key + 1 (0 when the
    row has none), then the largest of them (tests/test_packed_attention.py:53-57)."""
    live = kmask != 0
    n, s = live.shape
    pos = torch.arange(1, s + 1, device=kmask.device, dtype=torch.int32)
    last = torch.where(live, pos, torch.zeros((), dtype=torch.int32, device=kmask.device))
    last = last.amax(dim=1) if s > 0 else torch.zeros(n, dtype=torch.int32, device=kmask.device)
    top = last.amax().reshape(1) if n > 0 else torch.zeros(1, dtype=torch.int32, device=kmask.device)
    return torch.cat([last, top]).to(torch.int32).contiguous()


# ---- fused pair-stack ops with natural weight shapes ----------------------------------------

def fused_available(kernel, dtype, *widths):
    """True if `kernel` takes these widths and this activation dtype: ln_gated_dual_proj (a, ci),
    trimul_epilogue (a, ci), ln_projection (a, n), output_projection (k, c), transition (c,
    hidden). fp16 is the reference's F16 contract; bf16 activations are this library's addition
    (the reference's wrappers decline them, tests/test_fused.py:223-229)."""
    if dtype not in (torch.float16, torch.bfloat16):
        return False
    w2 = {64, 128}
    if kernel in ("ln_gated_dual_proj", "trimul_epilogue"):
        a, ci = widths
        return a in w2 and ci in w2
    if kernel == "ln_projection":
        a = widths[0]
        n = widths[1] if len(widths) > 1 else 0
        return a in w2 and (n == 0 or n % 64 == 0)
    if kernel == "output_projection":
        k, c = widths
        return k in w2 and c in w2
    if kernel == "transition":
        c, hd = widths
        return c in (64, 128, 256) and hd in (2 * c, 4 * c)
    raise KeyError(kernel)


def _rows(x):
    """x [..., C] -> ([M, C] contiguous, leading shape)."""
    return x.reshape(-1, x.shape[-1]).contiguous(), tuple(x.shape[:-1])


def _keep_rows(keep):
    return None if keep is None else keep.reshape(-1).to(torch.float16).contiguous()


def _w16(w):
    """Weights and biases go to the kernels as fp16."""
    return w.to(torch.float16)


def ln_gated_dual_proj(x, scale, offset, wp, bp, wg, bg, mask, eps=1e-5):
    """left, right [ci, M] (channel major) = the halves of mask (LN(x)@wp + bp) sigmoid(LN(x)@wg
    + bg), with wp, wg [a, 2 ci] (tests/test_fused.py:96-103)."""
    x2, _ = _rows(x)
    wpT, wgT = layouts.proj_pair_T(_w16(wp), _w16(wg))
    return hip.ln_gdp(x2, scale.float().contiguous(), offset.float().contiguous(), wpT,
                      _w16(bp).contiguous(), wgT, _w16(bg).contiguous(), _keep_rows(mask), eps)


def trimul_epilogue_ln(x_cm, x, in_scale, in_offset, ln_scale, ln_offset, wo, bo, wg, bg,
                       keep=None, add_input=False, eps=1e-5):
    """out [..., a] = (LN(x_cm^T)@wo + bo) sigmoid(LN_in(x)@wg + bg) (+ x), with x_cm [ci, M]
    fp32, wo [ci, a], wg [a, a] (tests/test_fused.py:104-121). With add_input the result is
    written over x, as the target's output aliases its input."""
    x2, lead = _rows(x)
    out = hip.trimul_epilogue(x_cm.float().contiguous(), x2, in_scale.float().contiguous(),
                              in_offset.float().contiguous(), ln_scale.float().contiguous(),
                              ln_offset.float().contiguous(), layouts.linear_T(_w16(wo)),
                              _w16(bo).contiguous(), layouts.linear_T(_w16(wg)),
                              _w16(bg).contiguous(), keep=_keep_rows(keep), eps=eps,
                              add_input=add_input, out=x2 if add_input else None)
    return out.reshape(lead + (out.shape[-1],))


def ln_projection(x, scale, offset, w=None, wb=None, keep=None, eps=1e-5):
    """p [..., slots, n] = LN(x)@w[s] for each slot (no bias term) and the head bias
    [heads, ...] = (LN(x)@wb)^T, with w [slots, a, n] and wb [a, heads]; either may be None
    (tests/test_fused.py:180-199)."""
    x2, lead = _rows(x)
    wT = None if w is None else layouts.slot_major(_w16(w))
    wbT = None if wb is None else layouts.heads_T(_w16(wb))
    p, b = hip.ln_projection(x2, scale.float().contiguous(), offset.float().contiguous(), wT, wbT,
                             keep=_keep_rows(keep), eps=eps)
    if p is not None:
        p = p.reshape(lead + (w.shape[0], w.shape[2]))
    if b is not None:
        b = b.reshape((b.shape[0],) + lead)
    return p, b


def output_projection(o, w, b, residual=None, keep=None):
    """out [..., c] = o@w + b (+ residual), w [k, c]; with a residual the result is written over
    it, as the target aliases them (tests/test_fused.py:201-213)."""
    o2, lead = _rows(o)
    r2 = None if residual is None else residual.reshape(-1, residual.shape[-1]).contiguous()
    out = hip.output_projection(o2, layouts.linear_T(_w16(w)), _w16(b).contiguous(), residual=r2,
                                keep=_keep_rows(keep), out=r2)
    return out.reshape(lead + (out.shape[-1],))


def transition(x, scale, offset, w1, b1, w2, b2, keep=None, add_input=False, eps=1e-5):
    """out [..., c] = relu(LN(x)@w1 + b1)@w2 + b2 (+ x), w1 [c, hidden], w2 [hidden, c]
    (tests/test_fused.py:215-229); with add_input the result is written over x."""
    x2, lead = _rows(x)
    out = hip.transition(x2, scale.float().contiguous(), offset.float().contiguous(),
                         layouts.linear_T(_w16(w1)), _w16(b1).contiguous(),
                         layouts.w2_blocked(_w16(w2)), _w16(b2).contiguous(),
                         keep=_keep_rows(keep), eps=eps, add_input=add_input,
                         out=x2 if add_input else None)
    return out.reshape(lead + (out.shape[-1],))


# ---- RMS norm and the 8-bit path (no counterpart in the reference) ----------------------------

class _RmsNorm(torch.autograd.Function):
    """x and residual come in as the caller has them and are flattened in here: reshaped around this
    node, their gradients would reach the leaves as two views of ds, each of which autograd takes for
    a leaf's own and adds to in place. As one tensor for both inputs it is copied where a leaf keeps
    it, as an addition's gradient is."""

    @staticmethod
    def forward(ctx, x, scale, residual, eps):
        x = x.contiguous()
        residual = None if residual is None else residual.contiguous()
        if x.dim() == 2:
            out, total, rstd = hip.rms_norm(x, scale, residual, eps, True)
        else:  # results of x's own shape: as views of rows they could not be changed in place
            out, total = torch.empty_like(x), None if residual is None else torch.empty_like(x)
            rstd = hip.rms_norm(_matrix(x), scale, None if residual is None else _matrix(residual), eps, True,
                                _matrix(out), None if residual is None else _matrix(total))[2]
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if residual is None else total, scale, rstd)
        return out if residual is None else (out, total)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dsum=None):
        s, scale, rstd = ctx.saved_tensors
        _refuse_capture(s)
        dsum = None if dsum is None else dsum.to(s.dtype).contiguous()
        if dout is None:  # only the sum was used
            ds, dscale = dsum, torch.zeros_like(scale)
        else:
            dout = dout.to(s.dtype).contiguous()
            if s.dim() == 2:
                ds, dscale = hip.rms_norm_bwd(s, scale, rstd, dout, dsum)
            else:
                ds, dscale = torch.empty_like(s), torch.empty_like(scale)
                hip.rms_norm_bwd(_matrix(s), scale, rstd, _matrix(dout), None if dsum is None else _matrix(dsum),
                                 grads=(_matrix(ds), dscale))
        need = ctx.needs_input_grad
        return ds if need[0] else None, dscale if need[1] else None, ds if need[2] else None, None


def rms_norm(x, scale, residual=None, eps=1e-5):
    """y [..., c] = s / sqrt(mean(s^2) + eps) * scale with s = x, or (y, s) with s = x + residual
    rounded to x's type: the residual stream, which the next block adds to. x and residual fp16 or
    bf16, one shape; scale [c]. Differentiable in x, residual and scale (once, in reverse mode; a dual tensor is
    refused).

    While a HIP graph is being captured, a call that needs gradients is refused, and so is the backward of an
    earlier one on the capturing stream: a leaf that an eager pass has used keeps that pass's stream, torch makes it
    wait for the capture's work when the gradient reaches it, and nothing in a call tells whether one of its leaves
    is such a one. Capture hip.rms_norm and hip.rms_norm_bwd instead, which take their buffers."""
    _residual_like("rms_norm", "x", residual, x.shape)
    differentiated = torch.is_grad_enabled() and (x.requires_grad or scale.requires_grad or (
        residual is not None and residual.requires_grad))
    if differentiated:
        _refuse_capture(x)
    w = scale.float().contiguous()
    if differentiated or _any_tangent(x, scale, residual):
        return _RmsNorm.apply(x, w, residual, float(eps))
    out, total, _ = hip.rms_norm(_matrix(x), w, None if residual is None else _matrix(residual), eps)
    if x.dim() != 2:
        out, total = out.reshape(x.shape), None if total is None else total.reshape(x.shape)
    return out if residual is None else (out, total)


def _residual_like(name, what, residual, shape):
    if residual is not None and residual.shape != shape:
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "%s: residual must be like %s, got %s and %s"
                                  % (name, what, tuple(residual.shape), tuple(shape)))


def _residual_rows(name, what, residual, shape):
    """residual as rows: of `shape`, or given as rows [M, C] or a row (whose M and C the entry point checks)"""
    if residual is None:
        return None
    if residual.dim() > 2:
        _residual_like(name, what, residual, shape)
    return _rows(residual)[0]


def _capturing(t):
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


def _refuse_capture(t, name="rms_norm"):
    if _capturing(t):
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "%s: a differentiated call cannot be captured into a "
                                  "graph; capture hip.%s and hip.%s_bwd" % (name, name, name))


def _any_tangent(*tensors):
    """Whether one of them is a dual tensor of the open forward-mode level: the autograd node refuses those,
    which have no requires_grad. (Three looks with no level open are 1 us of a call's 9: the level first, where
    torch has it under this name.)"""
    return getattr(forward_ad, "_current_level", 0) >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _matrix(x):
    """x [..., C] as [M, C], contiguous; x itself where it is that"""
    return x.contiguous() if x.dim() == 2 else _rows(x)[0]


def _q8_lead(q, q_scale, lead):
    return q.reshape(lead + (q.shape[-1],)), q_scale.reshape(lead)


def rms_norm_q8(x, scale, residual=None, eps=1e-5):
    """(q, q_scale, s): rms_norm with its result as 8-bit rows, q [..., hip.padded_k(c)] int8 and
    q_scale [...] fp32; s as in rms_norm, None without a residual."""
    x2, lead = _rows(x)
    r2 = _residual_rows("rms_norm_q8", "x", residual, x.shape)
    q, q_scale, total = hip.rms_norm_q8(x2, scale.float().contiguous(), r2, eps)
    return _q8_lead(q, q_scale, lead) + (None if total is None else total.reshape(x.shape),)


_ACTIVATIONS = {None: 0, "relu": 1, "swish_gate": 2}


def quantize_rows(x, activation=None):
    """(q, q_scale): the 8-bit rows of x [..., k] (fp16, bf16 or fp32), of relu(x) ("relu"), or of
    swish(x[..., :k]) * x[..., k:] ("swish_gate", x [..., 2k])."""
    if activation not in _ACTIVATIONS:
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "quantize_rows: activation is None, 'relu' or 'swish_gate', got %r"
                                  % (activation,))
    x2, lead = _rows(x)
    return _q8_lead(*hip.quantize_rows(x2, _ACTIVATIONS[activation]), lead)


def dequantize_rows(q, q_scale, k=None, dtype=torch.float16):
    """What 8-bit rows stand for: [..., k] of `dtype` (k: all of q's columns)."""
    q2, lead = _rows(q)
    out = hip.dequantize_rows(q2, q_scale.reshape(-1).contiguous(), k, dtype)
    return out.reshape(lead + (out.shape[-1],))


def q8_weights(w):
    """(wq, w_scale) of w [k, n]: each output channel quantised with a scale of its own and laid out for
    q8_projection, once, when a program loads its weights."""
    q, w_scale = hip.quantize_rows(layouts.linear_T(w))
    return layouts.q8_blocked(q), w_scale


def q8_projection(q, q_scale, weights, b=None, residual=None, dtype=torch.float16):
    """out [..., n] = x@w (+ b) (+ residual) for the 8-bit rows q, q_scale of x and weights =
    q8_weights(w); in residual's type, or `dtype` without one."""
    wq, w_scale = weights
    q2, lead = _rows(q)
    r2 = _residual_rows("q8_projection", "the result", residual, q.shape[:-1] + w_scale.shape[:1])
    out = hip.q8_projection(q2, q_scale.reshape(-1).contiguous(), wq, w_scale, None if b is None else b.float().contiguous(),
                            r2, dtype if r2 is None else r2.dtype)
    return out.reshape(lead + (out.shape[-1],))


def q8_transition(x, scale, w1, b1, w2, b2, residual=None, activation="relu", add_input=False, eps=1e-5):
    """out [..., c] = h@w2 + b2 (+ s), h the activation ("relu", or "swish_gate" over w1's two halves) of
    RMS(s)@w1 + b1, s = x or x + residual: the transition with an RMS norm and 8-bit products. w1, w2 =
    q8_weights of [c, hidden] (or [c, 2 hidden]) and [hidden, c]; b1, b2 may be None. With a residual
    (out, s)."""
    q, q_scale, total = rms_norm_q8(x, scale, residual, eps)
    s = x if total is None else total
    h = q8_projection(q, q_scale, w1, b1, dtype=x.dtype)
    out = q8_projection(*quantize_rows(h, activation), w2, b2, residual=s if add_input else None, dtype=x.dtype)
    return out if residual is None else (out, s)


# ---- heads, the key-value cache and its attention (no counterpart in the reference) -----------

class _QkNormRope(torch.autograd.Function):
    """qkv [..., H, D] is flattened in here, as in _RmsNorm."""

    @staticmethod
    def forward(ctx, qkv, q_norm, k_norm, rope, positions, kv_heads, eps, interleaved):
        qkv = qkv.contiguous()
        out = hip.qk_norm_rope(_heads(qkv), q_norm, k_norm, rope, positions, kv_heads, eps, interleaved)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(qkv, q_norm, k_norm, rope, positions)
        ctx.rule = kv_heads, eps, interleaved
        return out if qkv.dim() == 3 else tuple(t.view(qkv.shape[:-2] + t.shape[1:]) for t in out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        qkv, q_norm, k_norm, rope, positions = ctx.saved_tensors
        kv_heads, eps, interleaved = ctx.rule
        _refuse_capture(qkv, "qk_norm_rope")
        lead, (h, d) = qkv.shape[:-2], qkv.shape[-2:]
        grads = [qkv.new_zeros(lead + (n, d)) if g is None else g.to(qkv.dtype).contiguous()
                 for g, n in zip(grads, (h - 2 * kv_heads, kv_heads, kv_heads))]
        dqkv, dq_norm, dk_norm = hip.qk_norm_rope_bwd(_heads(qkv), q_norm, k_norm, rope, positions, *map(_heads, grads), eps, interleaved)
        need = ctx.needs_input_grad
        return (dqkv.view(qkv.shape) if need[0] else None, dq_norm if need[1] else None, dk_norm if need[2] else None) + (None,) * 5


def _heads(x):
    """x [..., H, D] as [T, H, D]; x itself where it is that"""
    return x if x.dim() == 3 else x.reshape((-1,) + x.shape[-2:])


def _tokens(name, what, t, lead, shared=True):
    """One value a token: of the leading shape, or one that broadcasts to it (without `shared`: by dimensions of 1 alone, each
    token having its own), as [T]"""
    if len(lead) == 1 and t.shape == lead:
        return t.contiguous()
    try:
        flat = t.expand(lead).reshape(-1)
    except RuntimeError:
        flat = None
    if flat is None or not (shared or flat.numel() == t.numel()):
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "%s: %s must be of the tokens' shape %s, got %s"
                                  % (name, what, tuple(lead), tuple(t.shape)))
    return flat


def _check_heads(name, x, what):
    if x.dim() < 3:
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "%s: %s must be [..., heads, D], got shape %s" % (name, what, tuple(x.shape)))


def _head_rows(name, x, what):
    _check_heads(name, x, what)
    return _heads(x.contiguous())


def qk_norm_rope(qkv, q_norm, k_norm, rope, positions, kv_heads, eps=1e-5, interleaved=False):
    """(q [..., Hq, D], k, v [..., kv_heads, D]): the heads of a projection's result qkv [..., Hq + 2 kv_heads, D], apart;
    queries and keys with each head's RMS norm, weights q_norm, k_norm [D], then the first R channels rotated by the
    angles of positions [...] int32 (or a shape that broadcasts to it) in rope [P, R] fp32 = layouts.rope_table(P, R): channels
    i and i + R / 2 as pairs, or neighbours (interleaved). fp16 or bf16. Differentiable in qkv, q_norm and
    k_norm (once, in reverse mode; a dual tensor is refused); like rms_norm, not while a HIP graph is captured: capture
    hip.qk_norm_rope and hip.qk_norm_rope_bwd instead."""
    _check_heads("qk_norm_rope", qkv, "qkv")
    h = qkv.shape[-2]
    if not 0 < 2 * kv_heads < h:
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "qk_norm_rope: qkv has %d heads, of which 2 * %d cannot be keys and values"
                                  % (h, kv_heads))
    positions = _tokens("qk_norm_rope", "positions", positions, qkv.shape[:-2])
    wq, wk = q_norm.float().contiguous(), k_norm.float().contiguous()
    differentiated = torch.is_grad_enabled() and (qkv.requires_grad or q_norm.requires_grad or k_norm.requires_grad)
    if differentiated:
        _refuse_capture(qkv, "qk_norm_rope")
    if differentiated or _any_tangent(qkv, q_norm, k_norm, rope):
        return _QkNormRope.apply(qkv, wq, wk, rope, positions, int(kv_heads), float(eps), bool(interleaved))
    out = hip.qk_norm_rope(_head_rows("qk_norm_rope", qkv, "qkv"), wq, wk, rope, positions, int(kv_heads), eps, interleaved)
    return out if qkv.dim() == 3 else tuple(t.reshape(qkv.shape[:-2] + t.shape[1:]) for t in out)


def cache_slots(page_table, positions, page):
    """The slots [B] or [B, S] int32 of positions [B] or [B, S] of B sequences whose pages are page_table [B, N], `page` tokens
    a page: -1 for a negative position (a padded row), one past the table, or a page that is negative or past what int32
    slots reach."""
    if page_table.dim() != 2 or positions.dim() not in (1, 2) or positions.shape[0] != page_table.shape[0] or page < 1:
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "cache_slots: expected page_table [B, N], positions [B] or [B, S] and a page "
                                  "of 1 token at least, got %s, %s and %d" % (tuple(page_table.shape), tuple(positions.shape), page))
    if page_table.shape[1] == 0:
        return torch.full_like(positions, -1, dtype=torch.int32)
    at = (positions if positions.dim() == 2 else positions[:, None]).long()
    col = at.div(page, rounding_mode="floor")
    known = (at >= 0) & (col < page_table.shape[1])
    pages = page_table.long().gather(1, torch.where(known, col, torch.zeros_like(col)))
    known &= (pages >= 0) & (pages < 2 ** 31 // page)
    slots = torch.where(known, pages * page + at % page, torch.full_like(at, -1))
    return slots.to(torch.int32).reshape(positions.shape)


def qk_norm_rope_cache(qkv, q_norm, k_norm, rope, positions, slots, cache, eps=1e-5, interleaved=False):
    """q [..., Hq, D]: qk_norm_rope with keys and values written into `cache` = hip.kv_cache(...), each token at its slot
    (cache_slots; positions and slots [...] int32). A token with a slot that the cache does not have is not written;
    the slots of a call must differ from one another. Forward only."""
    rows = _head_rows("qk_norm_rope_cache", qkv, "qkv")
    lead = qkv.shape[:-2]
    q = hip.qk_norm_rope_cache(rows, q_norm.float().contiguous(), k_norm.float().contiguous(), rope,
                               _tokens("qk_norm_rope_cache", "positions", positions, lead),
                               _tokens("qk_norm_rope_cache", "slots", slots, lead, False), cache, eps, interleaved)
    return q if len(lead) == 1 else q.reshape(lead + q.shape[1:])


def kv_cache_write(k, v, slots, cache):
    """k, v [..., heads, D] into the cache as they are, each token at its slot (qk_norm_rope_cache's rules)."""
    if k.shape != v.shape:
        raise hip.InvalidArgument(hip.INVALID_ARGUMENT, "kv_cache_write: k and v must be alike, got %s and %s"
                                  % (tuple(k.shape), tuple(v.shape)))
    k, v, lead = _head_rows("kv_cache_write", k, "k"), _head_rows("kv_cache_write", v, "v"), k.shape[:-2]
    hip.kv_cache_write(k, v, _tokens("kv_cache_write", "slots", slots, lead, False), cache)


def kv_cache_read(cache, slots, dtype=None):
    """(k, v) [..., heads, D]: what slots [...] int32 of the cache hold, zeros for a slot that it does not have."""
    k, v = hip.kv_cache_read(cache, slots.reshape(-1), dtype)
    if slots.dim() == 1:
        return k, v
    return k.reshape(slots.shape + k.shape[1:]), v.reshape(slots.shape + v.shape[1:])


def paged_attention(q, cache, page_table, lengths, scale=None, want_lse=False):
    """softmax(scale q K^T) V for one new token a sequence, q [B, Hq, D], over the lengths[b] tokens that the pages
    page_table[b] of the cache hold (both int32); with want_lse (out, lse [B, Hq] fp32, log2 domain). scale defaults to
    D^-1/2. Forward only."""
    out, lse = hip.paged_attention(q.contiguous(), cache, page_table.contiguous(), lengths.contiguous(), scale, want_lse)
    return (out, lse) if want_lse else out
