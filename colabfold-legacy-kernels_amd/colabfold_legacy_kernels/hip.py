"""PyTorch-ROCm front end of the gfx950 library: each function is one XLA FFI target of the
reference, called through the library's C ABI (include/colabfold_gfx950.h) on the current HIP
stream, with the FFI binding's buffer order, attributes, result shapes and error behaviour.

  attention_fwd       VoltaMma            (reference cuda/volta_mma_attn.cu:625-640)
  attention_packed    VoltaMmaPacked[Trim] (volta_mma_attn.cu:594-623)
  attention_bwd       VoltaMmaBwd         (cuda/volta_mma_attn_bwd.cu:455-473)
  ln_gdp              VoltaLnGdp          (cuda/volta_fused_ffi.h:337-351)
  trimul_epilogue     VoltaTrimulEpilogue (volta_fused_ffi.h:353-371)
  ln_projection       VoltaLnProj         (volta_fused_ffi.h:373-388)
  output_projection   VoltaOutProj        (volta_fused_ffi.h:390-401)
  transition          VoltaTransition     (volta_fused_ffi.h:403-418)
  layer_norm          VoltaLayerNorm      (cuda/volta_ops.cu:86-94)
  gated_dual_proj     VoltaGdp            (volta_ops.cu:258-269)

and, without a counterpart in the reference, the RMS norm and the 8-bit serving path beside them:

  rms_norm, rms_norm_bwd      RMS norm with the residual's addition, and its gradients
  rms_norm_q8                 the same norm with 8-bit rows as its result
  quantize_rows, dequantize_rows  8-bit rows of a matrix (or of its relu or swish gate), and back
  q8_projection               8-bit rows times 8-bit weights, scales, bias and residual
  qk_norm_rope, qk_norm_rope_bwd  RMS norm of each query and key head with the position rotation, and its gradients
  qk_norm_rope_cache          the same with keys and values written into a paged cache, in 16 or 8 bits
  kv_cache, kv_cache_write, kv_cache_read  that cache, and keys and values into it and back
  paged_attention             one new token's attention over the cache

Results are allocated here with torch (as XLA preallocates them) unless passed in, which is how a
caller aliases an output to its residual / input. The fused ops take fp16 or bf16 activations
(all of a call's activations and results one type; weights, biases and keep fp16); results come
back in the activation type. A rejected call raises InvalidArgument (the
FFI's InvalidArgument) and a launch failure KernelError (Internal), with the library's message.
There is no CPU fallback: without the built library every call raises.
"""
import collections
import ctypes
import functools
import struct

import torch

from . import library_path

CLK_S8, CLK_S32, CLK_U8, CLK_F16, CLK_F32, CLK_BF16 = 2, 4, 6, 10, 11, 16
_DTYPES = {torch.int8: CLK_S8, torch.int32: CLK_S32, torch.uint8: CLK_U8, torch.float16: CLK_F16,
           torch.float32: CLK_F32, torch.bfloat16: CLK_BF16}
INVALID_ARGUMENT, INTERNAL = 3, 13


class KernelError(RuntimeError):
    def __init__(self, code, message):
        super().__init__(message)
        self.code = code


class InvalidArgument(KernelError, ValueError):
    pass


class Buffer(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("dtype", ctypes.c_int32), ("rank", ctypes.c_int32),
                ("dims", ctypes.POINTER(ctypes.c_int64))]


_P = ctypes.c_void_p  # a Buffer by reference (byref), or its address
_lib = None

_SIGNATURES = {
    "clk_attention_fwd": [ctypes.c_void_p, ctypes.c_int32] + [_P] * 7 +
                         [ctypes.c_float, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32],
    "clk_attention_packed": [ctypes.c_void_p, ctypes.c_int32] + [_P] * 5 +
                            [ctypes.c_float, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32],
    "clk_attention_packed_trim": [ctypes.c_void_p, ctypes.c_int32] + [_P] * 6 +
                                 [ctypes.c_float, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32],
    "clk_attention_bwd": [ctypes.c_void_p, ctypes.c_int32] + [_P] * 12 +
                         [ctypes.c_float, ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t],
    "clk_attention_bwd_noalloc": [ctypes.c_void_p, ctypes.c_int32] + [_P] * 12 +
                                 [ctypes.c_float, ctypes.c_int32],
    "clk_ln_gdp": [ctypes.c_void_p] + [_P] * 10 + [ctypes.c_float],
    "clk_trimul_epilogue": [ctypes.c_void_p] + [_P] * 12 +
                           [ctypes.c_float, ctypes.c_int32, ctypes.c_int32],
    "clk_ln_projection": [ctypes.c_void_p] + [_P] * 8 +
                         [ctypes.c_float, ctypes.c_int64, ctypes.c_int64, ctypes.c_int32],
    "clk_output_projection": [ctypes.c_void_p] + [_P] * 6 + [ctypes.c_int32, ctypes.c_int32],
    "clk_transition": [ctypes.c_void_p] + [_P] * 9 +
                      [ctypes.c_float, ctypes.c_int32, ctypes.c_int32],
    "clk_layer_norm": [ctypes.c_void_p] + [_P] * 4 + [ctypes.c_float],
    "clk_gated_dual_proj": [ctypes.c_void_p, ctypes.c_int32] + [_P] * 7 + [ctypes.c_int64],
    "clk_opm_update": [ctypes.c_void_p] + [_P] * 6 + [ctypes.c_float, ctypes.c_int32],
    "clk_opm_outer": [ctypes.c_void_p] + [_P] * 4,
    "clk_rms_norm": [ctypes.c_void_p] + [_P] * 6 + [ctypes.c_float, ctypes.c_int32, ctypes.c_int32],
    "clk_rms_norm_q8": [ctypes.c_void_p] + [_P] * 6 + [ctypes.c_float, ctypes.c_int32],
    "clk_rms_norm_bwd": [ctypes.c_void_p] + [_P] * 7 +
                        [ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t],
    "clk_quantize_rows": [ctypes.c_void_p] + [_P] * 3 + [ctypes.c_int64],
    "clk_dequantize_rows": [ctypes.c_void_p] + [_P] * 3,
    "clk_q8_projection": [ctypes.c_void_p] + [_P] * 7 + [ctypes.c_int32, ctypes.c_int32],
    "clk_qk_norm_rope": [ctypes.c_void_p] + [_P] * 8 + [ctypes.c_float, ctypes.c_int32],
    "clk_qk_norm_rope_bwd": [ctypes.c_void_p] + [_P] * 11 +
                            [ctypes.c_float, ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t],
    "clk_qk_norm_rope_cache": [ctypes.c_void_p] + [_P] * 11 + [ctypes.c_float, ctypes.c_int32],
    "clk_kv_cache_write": [ctypes.c_void_p] + [_P] * 7,
    "clk_kv_cache_read": [ctypes.c_void_p] + [_P] * 7,
    "clk_paged_attention": [ctypes.c_void_p] + [_P] * 9 +
                           [ctypes.c_float, ctypes.c_int32, ctypes.c_void_p, ctypes.c_size_t],
}


def lib():
    """The loaded gfx950 library (raises FileNotFoundError when it is not built)."""
    global _lib
    if _lib is None:
        handle = ctypes.CDLL(library_path("attention", 950))
        for name, args in _SIGNATURES.items():
            fn = getattr(handle, name)  # a library missing an entry point fails here, loudly
            fn.argtypes = args
            fn.restype = ctypes.c_int
        handle.clk_last_error.restype = ctypes.c_char_p
        handle.clk_version.restype = ctypes.c_char_p
        handle.clk_attention_bwd_workspace_size.argtypes = [ctypes.c_int32, _P, _P]
        handle.clk_attention_bwd_workspace_size.restype = ctypes.c_size_t
        handle.clk_attention_bwd_plan.argtypes = [ctypes.c_int32] + [ctypes.c_int64] * 5 + \
            [ctypes.POINTER(ctypes.c_int64), ctypes.c_int32]
        handle.clk_attention_bwd_plan.restype = ctypes.c_int
        handle.clk_rms_norm_bwd_workspace_size.argtypes = [_P]
        handle.clk_rms_norm_bwd_workspace_size.restype = ctypes.c_size_t
        handle.clk_qk_norm_rope_bwd_workspace_size.argtypes = [_P, _P]
        handle.clk_qk_norm_rope_bwd_workspace_size.restype = ctypes.c_size_t
        handle.clk_paged_attention_workspace_size.argtypes = [_P, _P, _P]
        handle.clk_paged_attention_workspace_size.restype = ctypes.c_size_t
        handle.clk_attention_bwd_noalloc_scratch_size.argtypes = []
        handle.clk_attention_bwd_noalloc_scratch_size.restype = ctypes.c_size_t
        _lib = handle
    return _lib


def buffer(t):
    """A clk_buffer describing tensor t (contiguous, on a HIP device)."""
    if t.dtype not in _DTYPES:
        raise TypeError("unsupported dtype %s" % t.dtype)
    if not t.is_contiguous():
        raise ValueError("tensors must be contiguous")
    dims = (ctypes.c_int64 * max(t.dim(), 1))(*t.shape)
    b = Buffer(ctypes.c_void_p(t.data_ptr()), _DTYPES[t.dtype], t.dim(), dims)
    b._keep = dims
    return b


def _ref(b):
    return ctypes.byref(b)


# The same descriptions for a whole call, as the calls below pass them: packed at once into one array,
# with the dimension arrays of shapes met before reused (they depend on the shape alone). A call of
# eight tensors spent 18 us in buffer(), half of it on the dimension arrays, where the smallest
# kernels take 5 us.
_PACKED = [struct.Struct("<" + "QiiQ" * n) for n in range(16)]
_FRAMES = [ctypes.c_char * (24 * n) for n in range(16)]
assert ctypes.sizeof(Buffer) == 24
_DIMS = {}
_DIMS_MAX = 4096


def _dims(shape):
    if len(_DIMS) >= _DIMS_MAX:
        _DIMS.clear()  # calls in flight hold the arrays they use
    arr = (ctypes.c_int64 * max(len(shape), 1))(*shape)
    d = _DIMS[shape] = (ctypes.addressof(arr), arr)
    return d


def _frame(*tensors):
    """The addresses of the clk_buffers of `tensors`, and what the caller keeps until its call is
    over; the tensors' checks are buffer()'s."""
    vals, keep = [], []
    for t in tensors:
        code = _DTYPES.get(t.dtype)
        if code is None:
            raise TypeError("unsupported dtype %s" % t.dtype)
        if not t.is_contiguous():
            raise ValueError("tensors must be contiguous")
        shape = t.shape
        d = _DIMS.get(shape) or _dims(shape)
        keep.append(d)
        vals += (t.data_ptr(), code, len(shape), d[0])
    n = len(tensors)
    frame = _FRAMES[n]()
    _PACKED[n].pack_into(frame, 0, *vals)
    keep.append(frame)
    base = ctypes.addressof(frame)
    return range(base, base + 24 * n, 24), keep


def _check(status):
    if status != 0:
        msg = lib().clk_last_error().decode()
        if status == INVALID_ARGUMENT:
            raise InvalidArgument(status, msg)
        raise KernelError(status, msg)


def _stream(t):
    if t.is_cuda:
        return torch._C._cuda_getCurrentRawStream(t.device.index)
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


_ONES = {}


def _one(like, dtype):
    """The one-element buffer the FFI takes for an absent optional input, or for a result that is
    not produced (never written, never returned). One zero buffer per device and dtype is kept for
    the process, so a call adds no allocation or fill of its own."""
    key = (like.device, dtype)
    t = _ONES.get(key)
    if t is None:
        t = _ONES[key] = torch.zeros(1, dtype=dtype, device=like.device)
    return t


def attention_fwd(q, k, v, bias, kmask, scale, block_q=64, block_k=32, want_lse=True, out=None,
                  lse=None):
    """VoltaMma: out [N,H,Sq,D] F16 and lse [N,H,Sq] F32 (log2 domain), or a one-element lse
    left untouched without want_lse (tests/test_attn_bwd.py:47-57)."""
    n, h, sq, d = q.shape
    out = torch.empty_like(q) if out is None else out
    if lse is None:
        lse = (torch.empty((n, h, sq), dtype=torch.float32, device=q.device) if want_lse
               else torch.zeros(1, dtype=torch.float32, device=q.device))
    bufs, hold = _frame(q, k, v, bias, kmask, out, lse)
    _check(lib().clk_attention_fwd(_stream(q), q.device.index, *bufs, float(scale),
                                   int(block_q), int(block_k), int(bool(want_lse))))
    return out, lse


def attention_packed(p, bias, kmask, gate_bias, scale, block_q=64, block_k=32, column=False,
                     lims=None, out=None):
    """VoltaMmaPacked (lims None) or VoltaMmaPackedTrim: out [X,Y,H,D] F16 from p [X,Y,G,H,D]."""
    x, y, _, h, d = p.shape
    out = torch.empty((x, y, h, d), dtype=torch.float16, device=p.device) if out is None else out
    if lims is None:
        bufs, hold = _frame(p, bias, kmask, gate_bias, out)
        fn = lib().clk_attention_packed
    else:
        bufs, hold = _frame(p, bias, kmask, gate_bias, lims, out)
        fn = lib().clk_attention_packed_trim
    _check(fn(_stream(p), p.device.index, *bufs, float(scale), int(block_q),
              int(block_k), int(bool(column))))
    return out


def attention_bwd_workspace(q, k):
    bufs, hold = _frame(q, k)
    return int(lib().clk_attention_bwd_workspace_size(q.device.index, *bufs))


def attention_bwd_plan(n, h, sq, sk, d, device=0):
    """The backward's launch plan on `device` (a diagnostic for tests and the bench)."""
    vals = (ctypes.c_int64 * 6)()
    _check(lib().clk_attention_bwd_plan(device, n, h, sq, sk, d, vals, 6))
    return dict(zip(("row_groups", "chunk", "chunks", "passes", "windows", "registers"), list(vals)))


def attention_bwd(q, k, v, bias, kmask, out, dout, lse, scale, want_dbias=True, workspace=None,
                  grads=None):
    """VoltaMmaBwd: dq, dk, dv F16 and dbias [H,Sq,Sk] F32 (zeros without want_dbias), written
    into `grads` = (dq, dk, dv, dbias) when given, as into XLA's preallocated results."""
    if grads is None:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dbias = torch.empty(bias.shape, dtype=torch.float32, device=q.device)
    else:
        dq, dk, dv, dbias = grads
    if workspace is None:
        need = attention_bwd_workspace(q, k)
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    bufs, hold = _frame(q, k, v, bias, kmask, out, dout, lse, dq, dk, dv, dbias)
    _check(lib().clk_attention_bwd(_stream(q), q.device.index, *bufs, float(scale),
                                   int(bool(want_dbias)), ctypes.c_void_p(workspace.data_ptr()),
                                   workspace.numel()))
    return dq, dk, dv, dbias


def attention_bwd_noalloc(q, k, v, bias, kmask, out, dout, lse, scale, want_dbias=True,
                          grads=None):
    """VoltaMmaBwd without a workspace: the library's static per-GPU scratch serves instead
    (clk_attention_bwd_noalloc; calls that overlap on one GPU race for it)."""
    if grads is None:
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dbias = torch.empty(bias.shape, dtype=torch.float32, device=q.device)
    else:
        dq, dk, dv, dbias = grads
    bufs, hold = _frame(q, k, v, bias, kmask, out, dout, lse, dq, dk, dv, dbias)
    _check(lib().clk_attention_bwd_noalloc(_stream(q), q.device.index, *bufs,
                                           float(scale), int(bool(want_dbias))))
    return dq, dk, dv, dbias


def ln_gdp(x, scale, offset, wpT, bp, wgT, bg, mask, eps=1e-5):
    """VoltaLnGdp: left, right [P/2, M] F16, channel major."""
    m, p = x.shape[0], wpT.shape[0]
    left = x.new_empty((p // 2, m))
    right = x.new_empty((p // 2, m))
    bufs, hold = _frame(x, scale, offset, wpT, bp, wgT, bg, mask, left, right)
    _check(lib().clk_ln_gdp(_stream(x), *bufs, float(eps)))
    return left, right


def trimul_epilogue(x_cm, x, in_scale, in_offset, ln_scale, ln_offset, woT, bo, wgT, bg,
                    keep=None, eps=1e-5, add_input=False, out=None):
    """VoltaTrimulEpilogue: out [M,O] F16. out may be x itself with add_input."""
    m, o = x.shape[0], woT.shape[0]
    out = x.new_empty((m, o)) if out is None else out
    has_keep = keep is not None
    keep = keep if has_keep else _one(x, torch.float16)
    bufs, hold = _frame(x_cm, x, in_scale, in_offset, ln_scale, ln_offset, woT, bo, wgT, bg, keep, out)
    _check(lib().clk_trimul_epilogue(_stream(x), *bufs, float(eps),
                                     int(bool(add_input)), int(has_keep)))
    return out


def ln_projection(x, scale, offset, wT=None, wbT=None, keep=None, eps=1e-5):
    """VoltaLnProj: p [M,n] = LN(x)@w and bias [heads,M]; a missing weight gives n or heads 0
    and a one-element (untouched) result in its place."""
    m = x.shape[0]
    n = 0 if wT is None else wT.shape[0]
    heads = 0 if wbT is None else wbT.shape[0]
    p = x.new_empty((m, n)) if n else _one(x, x.dtype)
    bias = (x.new_empty((heads, m)) if heads
            else _one(x, x.dtype))
    has_keep = keep is not None
    keep = keep if has_keep else _one(x, torch.float16)
    wT = wT if n else _one(x, torch.float16)
    wbT = wbT if heads else _one(x, torch.float16)
    bufs, hold = _frame(x, scale, offset, wT, wbT, keep, p, bias)
    _check(lib().clk_ln_projection(_stream(x), *bufs, float(eps), n, heads,
                                   int(has_keep)))
    return (p if n else None), (bias if heads else None)


def output_projection(o, wT, b, residual=None, keep=None, out=None):
    """VoltaOutProj: out [M,N] = o@w + b [+ residual]; out may be residual itself."""
    m, n = o.shape[0], wT.shape[0]
    out = o.new_empty((m, n)) if out is None else out
    has_residual = residual is not None
    residual = residual if has_residual else _one(o, o.dtype)
    has_keep = keep is not None
    keep = keep if has_keep else _one(o, torch.float16)
    bufs, hold = _frame(o, wT, b, residual, keep, out)
    _check(lib().clk_output_projection(_stream(o), *bufs, int(has_residual),
                                       int(has_keep)))
    return out


def transition(x, scale, offset, w1T, b1, w2T, b2, keep=None, eps=1e-5, add_input=False,
               out=None):
    """VoltaTransition: out [M,C] = relu(LN(x)@w1 + b1)@w2 + b2 [+ x], w2T blocked
    [H/64][C][64]; out may be x itself with add_input."""
    out = torch.empty_like(x) if out is None else out
    has_keep = keep is not None
    keep = keep if has_keep else _one(x, torch.float16)
    bufs, hold = _frame(x, scale, offset, w1T, b1, w2T, b2, keep, out)
    _check(lib().clk_transition(_stream(x), *bufs, float(eps), int(bool(add_input)),
                                int(has_keep)))
    return out


def layer_norm(x, scale, offset, eps=1e-5, out=None):
    """VoltaLayerNorm: out [M,C] F16, one-pass fp32 statistics."""
    out = torch.empty_like(x) if out is None else out
    bufs, hold = _frame(x, scale, offset, out)
    _check(lib().clk_layer_norm(_stream(x), *bufs, float(eps)))
    return out


def gated_dual_proj(x, wp, bp, wg, bg, mask, activation=0, out=None):
    """VoltaGdp: out [M,N] = mask * (x@wp + bp) * act(x@wg + bg); wp, wg [K,N];
    activation 0 sigmoid, 1 swish."""
    m, n = x.shape[0], wp.shape[1]
    out = torch.empty((m, n), dtype=torch.float16, device=x.device) if out is None else out
    bufs, hold = _frame(x, wp, bp, wg, bg, mask, out)
    _check(lib().clk_gated_dual_proj(_stream(x), x.device.index, *bufs, int(activation)))
    return out


def opm_update(lhs, t, bias, norm, residual=None, eps=1e-3, out=None):
    """VoltaOpmUpdate: out [B,D,F] = (lhs@t[:, d] + bias) / (eps + norm[b, d]) (+ residual);
    lhs [B,K], t [K,D,F] fp16, bias [F], norm [B,D] fp32. residual may be `out` itself."""
    b, (d, f) = lhs.shape[0], t.shape[1:]
    out = torch.empty((b, d, f), dtype=torch.float16, device=lhs.device) if out is None else out
    res = residual if residual is not None else _one(lhs, torch.float16)
    bufs, hold = _frame(lhs, t, bias, norm, res, out)
    _check(lib().clk_opm_update(_stream(lhs), *bufs, float(eps), int(residual is not None)))
    return out


def opm_outer(left, right, wT, out=None):
    """VoltaOpmOuter: out [B,D,F] = sum_c,e f16(sum_a left[a,b,c] right[a,d,e]) wT[f, c*32 + e];
    left [16,B,C], right [16,D,32], wT [F, 32 C], all fp16."""
    b, d, f = left.shape[1], right.shape[1], wT.shape[0]
    out = torch.empty((b, d, f), dtype=torch.float16, device=left.device) if out is None else out
    bufs, hold = _frame(left, right, wT, out)
    _check(lib().clk_opm_outer(_stream(left), *bufs))
    return out


# ---- RMS norm and 8-bit rows (no counterpart in the reference) --------------------------------

_FUNCTIONS = {}


def _call(name, tensors, *attrs):
    """One entry point on the current stream of the tensors' GPU, whichever GPU is the current one. An
    absent optional buffer is given as any tensor of its type. One loop does buffer()'s checks and
    _frame()'s packing: a call of seven tensors spends 2 us here, of the 8 that it takes the host."""
    index = tensors[0].get_device()
    vals, keep = [], []
    for t in tensors:
        if t.get_device() != index or index < 0:
            raise InvalidArgument(INVALID_ARGUMENT, "%s: all tensors must be on one GPU, got %s and %s"
                                  % (name[4:], tensors[0].device, t.device))
        code = _DTYPES.get(t.dtype)
        if code is None:
            raise TypeError("unsupported dtype %s" % t.dtype)
        if not t.is_contiguous():
            raise ValueError("tensors must be contiguous")
        shape = t.shape
        d = _DIMS.get(shape) or _dims(shape)
        keep.append(d)
        vals += (t.data_ptr(), code, len(shape), d[0])
    n = len(tensors)
    frame = _FRAMES[n]()
    _PACKED[n].pack_into(frame, 0, *vals)
    base = ctypes.addressof(frame)
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(lib(), name)
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        status = fn(stream, *range(base, base + 24 * n, 24), *attrs)
    else:
        with torch.cuda.device(index):
            status = fn(stream, *range(base, base + 24 * n, 24), *attrs)
    if status:
        _check(status)


def _matrix(name, t):
    if t.dim() != 2:
        raise InvalidArgument(INVALID_ARGUMENT, "%s: expected a matrix, got shape %s" % (name, tuple(t.shape)))
    return t.shape


def padded_k(k):
    """The columns of 8-bit rows of k values: k rounded up to a multiple of 64."""
    return (k + 63) // 64 * 64


def rms_norm(x, scale, residual=None, eps=1e-5, want_rstd=False, out=None, sum_out=None, rstd=None):
    """(out, sum, rstd): out [M,C] = s / sqrt(mean(s^2) + eps) * scale with s = x, or s = x + residual
    rounded to x's type, which is the returned sum (None without a residual); rstd [M] F32 for the
    backward, None without want_rstd. x, residual F16 or BF16, scale [C] F32. sum_out may be x or
    residual itself, out may be x."""
    m, _ = _matrix("rms_norm", x)
    out = torch.empty_like(x) if out is None else out
    if residual is not None and sum_out is None:
        sum_out = torch.empty_like(x)
    want_rstd = want_rstd or rstd is not None
    if want_rstd and rstd is None:
        rstd = x.new_empty(m, dtype=torch.float32)
    has_residual = residual is not None
    _call("clk_rms_norm", (x, residual if has_residual else x, scale, sum_out if has_residual else x, out,
                           rstd if want_rstd else scale), float(eps), int(has_residual), int(want_rstd))
    return out, (sum_out if has_residual else None), rstd


def rms_norm_q8(x, scale, residual=None, eps=1e-5, q=None, q_scale=None, sum_out=None):
    """(q, q_scale, sum): rms_norm with its result as 8-bit rows, q [M,Kp] S8 (Kp = padded_k(C), zeros
    past C) and q_scale [M] F32; sum as in rms_norm."""
    m, c = _matrix("rms_norm_q8", x)
    if q is None:
        q = x.new_empty((m, padded_k(c)), dtype=torch.int8)
    if q_scale is None:
        q_scale = x.new_empty(m, dtype=torch.float32)
    has_residual = residual is not None
    if has_residual and sum_out is None:
        sum_out = torch.empty_like(x)
    _call("clk_rms_norm_q8", (x, residual if has_residual else x, scale, sum_out if has_residual else x, q, q_scale),
          float(eps), int(has_residual))
    return q, q_scale, (sum_out if has_residual else None)


@functools.lru_cache(maxsize=1024)
def _rms_norm_bwd_workspace(shape):
    dims = (ctypes.c_int64 * max(len(shape), 1))(*shape)
    return int(lib().clk_rms_norm_bwd_workspace_size(ctypes.byref(Buffer(None, CLK_F16, len(shape), dims))))


def rms_norm_bwd_workspace(s):
    """Bytes of workspace rms_norm_bwd needs for s [M,C]."""
    return _rms_norm_bwd_workspace(tuple(s.shape))


def rms_norm_bwd(s, scale, rstd, dout, dsum=None, workspace=None, grads=None):
    """(ds, dscale): the gradients of rms_norm from its s (x, or the returned sum) and rstd; dsum is the
    gradient that reaches sum itself. ds [M,C] is the gradient of x and of residual alike, dscale [C]
    F32; written into `grads` = (ds, dscale) when given."""
    ds, dscale = grads if grads is not None else (torch.empty_like(s), torch.empty_like(scale))
    if workspace is None:
        workspace = s.new_empty(max(rms_norm_bwd_workspace(s), 1), dtype=torch.uint8)
    elif workspace.device != s.device or not workspace.is_contiguous():
        raise InvalidArgument(INVALID_ARGUMENT, "rms_norm_bwd: workspace must be contiguous, on the tensors' GPU")
    _call("clk_rms_norm_bwd", (s, scale, rstd, dout, s if dsum is None else dsum, ds, dscale),
          int(dsum is not None), ctypes.c_void_p(workspace.data_ptr()), workspace.numel() * workspace.element_size())
    return ds, dscale


def quantize_rows(x, activation=0, q=None, q_scale=None):
    """(q, q_scale): the 8-bit rows of h [M,K], q [M,Kp] S8 (Kp = padded_k(K), zeros past K) and q_scale
    [M] F32. activation 0: h = x; 1: h = relu(x); 2: h = swish(x[:, :K]) * x[:, K:] with x [M,2K]. x F16,
    BF16 or F32."""
    m, k = _matrix("quantize_rows", x)
    k = k // 2 if activation == 2 else k
    if q is None:
        q = x.new_empty((m, padded_k(k)), dtype=torch.int8)
    if q_scale is None:
        q_scale = x.new_empty(m, dtype=torch.float32)
    _call("clk_quantize_rows", (x, q, q_scale), int(activation))
    return q, q_scale


def dequantize_rows(q, q_scale, k=None, dtype=torch.float16, out=None):
    """out [M,k]: what the 8-bit rows stand for; k defaults to all of q's columns."""
    m, kp = _matrix("dequantize_rows", q)
    if out is None:
        out = q.new_empty((m, kp if k is None else k), dtype=dtype)
    _call("clk_dequantize_rows", (q, q_scale, out))
    return out


def q8_projection(q, q_scale, wq, w_scale, b=None, residual=None, dtype=torch.float16, out=None):
    """out [M,N] = (q @ w^T) * q_scale[m] * w_scale[n] [+ b[n]] [+ residual]: 8-bit rows times 8-bit
    weights, wq laid out by layouts.q8_blocked; b [N] F32; residual and out of `dtype`, F16 or BF16. out
    may be residual itself."""
    m, _ = _matrix("q8_projection", q)
    if out is None:
        out = q.new_empty((m, w_scale.shape[0]), dtype=dtype)
    _call("clk_q8_projection", (q, q_scale, wq, w_scale, w_scale if b is None else b, out if residual is None else residual,
                                out), int(b is not None), int(residual is not None))
    return out


# ---- heads, the key-value cache and its attention (no counterpart in the reference) -----------

KVCache = collections.namedtuple("KVCache", "k v k_scale v_scale")
KVCache.__doc__ = """A paged cache: k, v [pages, heads, page, D] in the order that layouts.keys_blocked and values_blocked make, F16, BF16
or S8; k_scale, v_scale [pages, heads, page] F32 for S8, else None. Any such four in a tuple serve."""


def kv_cache(pages, heads, page, d, dtype=torch.int8, device="cuda"):
    """A cache of `pages` pages of `page` tokens, a multiple of 16, filled with zeros; d a multiple of 32. dtype:
    float16, bfloat16, or int8 for 8-bit rows."""
    k, v = (torch.zeros((pages, heads, page, d), dtype=dtype, device=device) for _ in range(2))
    if dtype != torch.int8:
        return KVCache(k, v, None, None)
    return KVCache(k, v, *(torch.zeros((pages, heads, page), dtype=torch.float32, device=device) for _ in range(2)))


def _cache_buffers(name, cache):
    k, v, k_scale, v_scale = cache
    if (k_scale is None) != (v_scale is None) or (k_scale is None) == (k.dtype is torch.int8):
        raise InvalidArgument(INVALID_ARGUMENT, "%s: an 8-bit cache has scales, and no other has" % name)
    if k_scale is None:
        k_scale = v_scale = _one(k, torch.float32)
    return k, v, k_scale, v_scale


def _rank3(name, t):
    if t.dim() != 3:
        raise InvalidArgument(INVALID_ARGUMENT, "%s: expected [tokens, heads, D], got shape %s" % (name, tuple(t.shape)))
    return t.shape


def _scratch(name, workspace, like, need):
    """(workspace, its address, its bytes): the caller's, or one of `need` bytes"""
    if workspace is None:
        if need == 0:
            return None, None, 0
        workspace = like.new_empty(need, dtype=torch.uint8)
    elif workspace.device != like.device or not workspace.is_contiguous():
        raise InvalidArgument(INVALID_ARGUMENT, "%s: workspace must be contiguous, on the tensors' GPU" % name)
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def qk_norm_rope(qkv, q_norm, k_norm, rope, positions, kv_heads, eps=1e-5, interleaved=False, out=None):
    """(q, k, v): the heads of a projection's result qkv [T, Hq + 2 kv_heads, D], apart: q [T,Hq,D], k, v
    [T,kv_heads,D]. Queries and keys have each head's RMS norm with the weights q_norm, k_norm [D] F32, then the first R
    channels rotated by the angles of positions [T] S32 in rope [P,R] F32 (layouts.rope_table): halves as pairs, or
    neighbours (interleaved). Written into `out` = (q, k, v) when given."""
    t, h, d = _rank3("qk_norm_rope", qkv)
    if out is None:
        if not 0 < 2 * kv_heads < h:
            raise InvalidArgument(INVALID_ARGUMENT, "qk_norm_rope: qkv has %d heads, of which 2 * %d cannot be keys and values"
                                  % (h, kv_heads))
        out = qkv.new_empty((t, h - 2 * kv_heads, d)), qkv.new_empty((t, kv_heads, d)), qkv.new_empty((t, kv_heads, d))
    elif _rank3("qk_norm_rope", out[1])[1] != kv_heads:
        raise InvalidArgument(INVALID_ARGUMENT, "qk_norm_rope: out has %d key heads, not %d" % (out[1].shape[1], kv_heads))
    _call("clk_qk_norm_rope", (qkv, q_norm, k_norm, rope, positions) + tuple(out), float(eps), int(bool(interleaved)))
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_of(name, *shapes):
    arrays = [(ctypes.c_int64 * max(len(s), 1))(*s) for s in shapes]
    bufs = [Buffer(None, CLK_F16, len(s), a) for s, a in zip(shapes, arrays)]
    return int(getattr(lib(), name)(*(ctypes.byref(b) for b in bufs)))


def qk_norm_rope_bwd_workspace(qkv, dk):
    """Bytes of workspace qk_norm_rope_bwd needs for qkv [T,H,D] and dk [T,Hkv,D]."""
    return _workspace_of("clk_qk_norm_rope_bwd_workspace_size", tuple(qkv.shape), tuple(dk.shape))


def qk_norm_rope_bwd(qkv, q_norm, k_norm, rope, positions, dq, dk, dv, eps=1e-5, interleaved=False, workspace=None, grads=None):
    """(dqkv, dq_norm, dk_norm): the gradients of qk_norm_rope; written into `grads` when given."""
    if grads is None:
        grads = torch.empty_like(qkv), torch.empty_like(q_norm), torch.empty_like(k_norm)
    workspace, at, size = _scratch("qk_norm_rope_bwd", workspace, qkv, qk_norm_rope_bwd_workspace(qkv, dk))
    _call("clk_qk_norm_rope_bwd", (qkv, q_norm, k_norm, rope, positions, dq, dk, dv) + tuple(grads), float(eps),
          int(bool(interleaved)), at, size)
    return grads


def qk_norm_rope_cache(qkv, q_norm, k_norm, rope, positions, slots, cache, eps=1e-5, interleaved=False, q=None):
    """q [T,Hq,D]: qk_norm_rope with keys and values written into the cache, token t at slot slots[t] (S32: page * tokens of a
    page + place in the page). A token whose slot the cache does not have, a negative one for a padded row, is not
    written; slots of a call must differ from one another."""
    t, h, d = _rank3("qk_norm_rope_cache", qkv)
    bufs = _cache_buffers("qk_norm_rope_cache", cache)
    if q is None:
        heads = h - 2 * bufs[0].shape[1] if bufs[0].dim() == 4 else 1
        q = qkv.new_empty((t, max(heads, 1), d))
    _call("clk_qk_norm_rope_cache", (qkv, q_norm, k_norm, rope, positions, slots, q) + bufs, float(eps), int(bool(interleaved)))
    return q


def kv_cache_write(k, v, slots, cache):
    """k, v [T,heads,D] into the cache as they are, token t at slot slots[t], with qk_norm_rope_cache's rules."""
    _call("clk_kv_cache_write", (k, v, slots) + _cache_buffers("kv_cache_write", cache))


def kv_cache_read(cache, slots, dtype=None, out=None):
    """(k, v) [T,heads,D]: what the slots hold, zeros for a slot that the cache does not have. dtype: the cache's, or F16
    (the default) or BF16 for an 8-bit cache."""
    bufs = _cache_buffers("kv_cache_read", cache)
    if out is None:
        if bufs[0].dim() != 4:
            raise InvalidArgument(INVALID_ARGUMENT, "kv_cache_read: a cache must be [pages,heads,page,D]")
        if dtype is None:
            dtype = torch.float16 if bufs[0].dtype is torch.int8 else bufs[0].dtype
        shape = (slots.shape[0], bufs[0].shape[1], bufs[0].shape[3])
        out = bufs[0].new_empty(shape, dtype=dtype), bufs[0].new_empty(shape, dtype=dtype)
    _call("clk_kv_cache_read", bufs + (slots,) + tuple(out))
    return out


def paged_attention_workspace(q, cache, page_table):
    """Bytes of workspace paged_attention needs."""
    return _workspace_of("clk_paged_attention_workspace_size", tuple(q.shape), tuple(cache[0].shape), tuple(page_table.shape))


def paged_attention(q, cache, page_table, lengths, scale=None, want_lse=False, out=None, lse=None, workspace=None):
    """(out, lse): attention of one new token a sequence, q [B,Hq,D], over the lengths[b] (S32) tokens that the pages
    page_table[b,:] (S32 [B,N]) of the cache hold; lse [B,Hq] F32 in the log2 domain, None without want_lse. scale
    defaults to D^-1/2. A sequence of no tokens gives zeros and -inf."""
    b, h, d = _rank3("paged_attention", q)
    bufs = _cache_buffers("paged_attention", cache)
    out = torch.empty_like(q) if out is None else out
    want_lse = want_lse or lse is not None
    if want_lse and lse is None:
        lse = q.new_empty((b, h), dtype=torch.float32)
    workspace, at, size = _scratch("paged_attention", workspace, q, paged_attention_workspace(q, cache, page_table))
    _call("clk_paged_attention", (q,) + bufs + (page_table, lengths, out, lse if want_lse else _one(q, torch.float32)),
          float(d ** -0.5 if scale is None else scale), int(want_lse), at, size)
    return out, (lse if want_lse else None)
