"""The 8-bit and RMS-norm operators as cases that can be timed and checked.

A case is one pass through one operator, as the layers of a residual stream call it: a norm that
also adds the block's output to the stream, rows held in 8 bits with a scale each, and the integer
matrix product that reads them. Weights are quantised and laid out once, when a program loads them.
Row counts run from a single token to the 384 x 384 positions of a pair stack; widths from the pair
stack's 64 to 8192 (16384 for a norm alone); both are odd as often as round.

Kinds, and the range each stands for (`draw` covers it):

  norm     RMS norm with or without the residual's addition, 16-bit results ("half"), 8-bit rows
           ("q8"), or forward and backward ("train"); 1 to 262144 rows of 64 to 16384 channels
  quantize rows to 8 bits: as they are, through relu (the transition's activation) or through a
           swish gate over pairs of columns; 1 to 262144 rows of 64 to 16384 columns
  project  8-bit rows times 8-bit weights, with or without bias and residual; 1 to 262144 rows,
           64 to 8192 in and out

8-bit results are returned as the values that they stand for, in the activations' type, beside their
scales.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-5
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_NORM, _QUANT, _PRODUCT = 1 << 27, 1 << 27, 1 << 39  # most elements or products of a case


def listed():
    return [
        # One token's norm on its way into an 8-bit projection: the smallest call, latency alone.
        dict(name="norm_q8_token", kind="norm", form="q8", m=1, c=4096, residual=True, dtype="f16"),
        # A prompt of an odd length, the block's output added to the stream first.
        dict(name="norm_q8_prompt", kind="norm", form="q8", m=4099, c=5120, residual=True, dtype="bf16"),
        # The pair stack of 384 residues: very many short rows.
        dict(name="norm_half_pair", kind="norm", form="half", m=147456, c=128, residual=False, dtype="f16"),
        # A training step's norm at an odd width, few rows: launches and the weights' gradient.
        dict(name="norm_train_odd", kind="norm", form="train", m=1531, c=1025, residual=True, dtype="f16"),
        # A training step's norm over a large batch.
        dict(name="norm_train_large", kind="norm", form="train", m=16384, c=8192, residual=True, dtype="bf16"),
        # The hidden activation of the pair stack's transition between its two products.
        dict(name="quantize_relu_pair", kind="quantize", act="relu", m=147456, k=512, dtype="f16"),
        # A gated transition's hidden activation for a handful of tokens.
        dict(name="quantize_gate_few", kind="quantize", act="gate", m=7, k=8192, dtype="bf16"),
        # One token through a square projection: the weights' bytes are all there is.
        dict(name="project_token", kind="project", m=1, k=4096, n=4096, b=True, residual=True, dtype="f16"),
        # A batch of single tokens through a wide projection.
        dict(name="project_batch", kind="project", m=48, k=4096, n=8192, b=False, residual=False, dtype="bf16"),
        # The transition's first product on the pair stack: short rows, all output.
        dict(name="project_pair", kind="project", m=147456, k=128, n=512, b=True, residual=False, dtype="f16"),
        # Sizes that fill no tile.
        dict(name="project_ragged", kind="project", m=1531, k=1100, n=2050, b=True, residual=True, dtype="bf16"),
        # A large prompt through a wide layer.
        dict(name="project_large", kind="project", m=8192, k=8192, n=8192, b=False, residual=True, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width of the range: half of them multiples of 64, the others as they fall."""
    w = _log_int(rng, lo, hi)
    return max(lo, w // 64 * 64) if rng.random() < 0.5 else w


def draw(rng):
    kind = rng.choice(("norm", "norm", "quantize", "project", "project", "project"))
    dtype = rng.choice(("f16", "bf16"))
    if kind == "norm":
        c = _width(rng, 64, 16384)
        return dict(kind=kind, form=rng.choice(("half", "q8", "train")), m=_log_int(rng, 1, min(262144, _NORM // c)), c=c,
                    residual=rng.random() < 0.6, dtype=dtype)
    if kind == "quantize":
        act, k = rng.choice(("none", "relu", "gate")), _width(rng, 64, 16384)
        return dict(kind=kind, act=act, m=_log_int(rng, 1, min(262144, _QUANT // (2 * k if act == "gate" else k))), k=k, dtype=dtype)
    k, n = _width(rng, 64, 8192), _width(rng, 64, 8192)
    return dict(kind=kind, m=_log_int(rng, 1, min(262144, _PRODUCT // (k * n), _NORM // n)), k=k, n=n, b=rng.random() < 0.5,
                residual=rng.random() < 0.5, dtype=dtype)


# ---- inputs -----------------------------------------------------------------------------------

class _Draws:
    """Values from the seed alone, drawn on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return (t * std + mean).to(dtype)

    def stream(self, m, c, dtype):
        """Activations as a residual stream has them: every channel with a spread of its own."""
        spread = torch.exp(self.normal(c, std=0.5))
        return (self.normal(m, c) * spread).to(dtype)

    def rows8(self, r, k, std=1.0):
        """r rows of k values in 8 bits, the row padded with zeros to a multiple of 64, and their scales."""
        t = self.normal(r, k, std=std)
        a = t.abs().amax(1, keepdim=True)
        q = torch.zeros((r, -(-k // 64) * 64), dtype=torch.int8, device="cuda")
        q[:, :k] = torch.round(t * (127.0 / a)).to(torch.int8)
        return q, (a / 127.0).reshape(r).contiguous()


def _blocks(q):
    """Weights [N, Kp] in the projection's layout, as a program keeps them: blocks of 64 channels by
    64 inputs, [ceil(N/64), Kp/64, 4, 4, 16, 16], where entry [., ., b, c, 4 g + i, j] is channel
    16 g + 4 b + i, input 16 c + j of its block; channels past N are zeros."""
    n, kp = q.shape
    p = torch.zeros((-(-n // 64) * 64, kp), dtype=q.dtype, device=q.device)
    p[:n] = q
    return p.view(-1, 4, 4, 4, kp // 64, 4, 16).permute(0, 4, 2, 5, 1, 3, 6).reshape(-1, kp // 64, 4, 4, 16, 16).contiguous()


def prepare(case, seed):
    r, kind, dt = _Draws(seed), case["kind"], _TYPES[case["dtype"]]
    s = dict(case, dt=dt)
    m = case["m"]
    if kind == "norm":
        c = case["c"]
        s["x"] = r.stream(m, c, dt)
        s["res"] = r.stream(m, c, dt) if case["residual"] else None
        s["w"] = r.normal(c, std=0.1, mean=1.0)
        if case["form"] == "train":
            s["dy"] = r.normal(m, c, dtype=dt)
            s["ds"] = r.normal(m, c, dtype=dt) if case["residual"] else None
            for name in ("x", "res", "w"):
                if s[name] is not None:
                    s[name].requires_grad_()
    elif kind == "quantize":
        s["x"] = r.stream(m, case["k"] * (2 if case["act"] == "gate" else 1), dt)
    else:
        n, k = case["n"], case["k"]
        s["q"], s["qs"] = r.rows8(m, k)
        s["w"], s["ws"] = r.rows8(n, k, std=k ** -0.5)
        s["wq"] = _blocks(s["w"])
        s["bias"] = r.normal(n, std=0.1) if case["b"] else None
        s["res"] = r.normal(m, n, dtype=dt) if case["residual"] else None
    return s


# ---- one pass ---------------------------------------------------------------------------------

_kit = None


def _own():
    """The framework's entry points."""
    global _kit
    if _kit is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "colabfold-legacy-kernels_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from colabfold_legacy_kernels import hip, torch_ops
        _kit = hip, torch_ops
    return _kit


_ACTS = {"none": 0, "relu": 1, "gate": 2}


def _run_own(s):
    hip, torch_ops = _own()
    if s["kind"] == "norm":
        if s["form"] == "half":
            y, total, _ = hip.rms_norm(s["x"], s["w"], s["res"], EPS)
            return y, total
        if s["form"] == "q8":
            q, scale, total = hip.rms_norm_q8(s["x"], s["w"], s["res"], EPS)
            return hip.dequantize_rows(q, scale, s["c"], s["dt"]), scale, total
        if s["residual"]:
            y, total = torch_ops.rms_norm(s["x"], s["w"], s["res"], EPS)
            grads = torch.autograd.grad((y, total), (s["x"], s["res"], s["w"]), (s["dy"], s["ds"]))
            return (y.detach(), total.detach()) + grads
        y = torch_ops.rms_norm(s["x"], s["w"], None, EPS)
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    if s["kind"] == "quantize":
        q, scale = hip.quantize_rows(s["x"], _ACTS[s["act"]])
        return hip.dequantize_rows(q, scale, s["k"], s["dt"]), scale
    return hip.q8_projection(s["q"], s["qs"], s["wq"], s["ws"], s["bias"], s["res"], s["dt"])


def _eight_bits(t, dt, r=1.0):
    """Rows t to 8 bits, and what they stand for with their scale times r."""
    a = t.abs().amax(1, keepdim=True)
    scale = a * r / 127.0
    q = torch.round(t * torch.where(a > 0, 127.0 / a, a))
    return (q * scale).to(dt), scale.reshape(-1)


def _run_plain(s):
    dt = s["dt"]
    if s["kind"] == "norm":
        with torch.no_grad():
            total = s["x"] if s["res"] is None else (s["x"].float() + s["res"].float()).to(dt)
            x, w = total.float(), s["w"]
            r = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
            if s["form"] == "q8":
                values, scale = _eight_bits(x * w, dt, r)
                return values, scale, (None if s["res"] is None else total)
            y = (x * r * w).to(dt)
            if s["form"] == "half":
                return y, (None if s["res"] is None else total)
            dy = s["dy"].float()
            g, xh = dy * w, x * r
            dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
            dw = (dy * xh).sum(0)
            if s["res"] is None:
                return y, dx.to(dt), dw
            dx = (dx + s["ds"].float()).to(dt)
            return y, total, dx, dx, dw
    if s["kind"] == "quantize":
        x, k = s["x"].float(), s["k"]
        if s["act"] == "relu":
            x = torch.where(x > 0, x, torch.zeros_like(x))
        elif s["act"] == "gate":
            x = x[:, :k] / (1.0 + torch.exp(-x[:, :k])) * x[:, k:]
        return _eight_bits(x, dt)
    out = torch.matmul(s["q"].float(), s["w"].float().t())
    out = out * s["qs"][:, None] * s["ws"]
    if s["bias"] is not None:
        out = out + s["bias"]
    if s["res"] is not None:
        out = out + s["res"].float()
    return out.to(dt)


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    m = case["m"]
    if case["kind"] == "norm":
        mc, res = m * case["c"], case["residual"]
        if case["form"] == "q8":
            return {"bytes": 2 * mc * (3 if res else 1) + mc + 4 * m + 4 * case["c"], "flops": 6 * mc}
        if case["form"] == "half":
            return {"bytes": 2 * mc * (4 if res else 2) + 4 * case["c"], "flops": 5 * mc}
        # forward: x (and residual) in, y (and the sum) out; backward: the sum, dy (and its own
        # gradient) in, the inputs' gradient out
        return {"bytes": 2 * mc * ((4 if res else 2) + (4 if res else 3)) + 12 * case["c"], "flops": 16 * mc}
    if case["kind"] == "quantize":
        mk = m * case["k"]
        return {"bytes": 2 * mk * (2 if case["act"] == "gate" else 1) + mk + 4 * m, "flops": (8 if case["act"] == "gate" else 3) * mk}
    k, n = case["k"], case["n"]
    return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["b"] else 0) + 2 * m * n * (2 if case["residual"] else 1),
            "flops": 2 * m * n * k}


# ---- the same in 64 bits ----------------------------------------------------------------------

def _rows8_64(t):
    """(integers, a / 127) of rows t, the integers as the definition has them: 127 t / a to the nearest, ties to even."""
    a = t.abs().max(dim=1).values
    q = torch.where(a[:, None] > 0, (127.0 * t / a[:, None]).round(), torch.zeros_like(t))
    return q, a / 127.0


def exact(case, seed):
    s, dt = prepare(case, seed), _TYPES[case["dtype"]]
    with torch.no_grad():
        if case["kind"] == "norm":
            w = s["w"].double()
            total = s["x"].double()
            if case["residual"]:
                total = (total + s["res"].double()).to(dt).double()  # the stream is held in 16 bits
            var = total.square().sum(1) / case["c"]
            inv = torch.rsqrt(var + EPS)[:, None]
            stream = total if case["residual"] else None
            if case["form"] == "q8":
                q, scale = _rows8_64(total * w)
                scale = scale * inv[:, 0]
                return q * scale[:, None], scale, stream
            norm = total * inv
            if case["form"] == "half":
                return norm * w, stream
            dy = s["dy"].double()
            dw = torch.einsum("mc,mc->c", dy, norm)
            dn = dy * w
            dx = inv * dn - norm * inv * ((dn * norm).sum(1, keepdim=True) / case["c"])
            if not case["residual"]:
                return norm * w, dx, dw
            dx = dx + s["ds"].double()
            return norm * w, stream, dx, dx, dw
        if case["kind"] == "quantize":
            x = s["x"].double()
            if case["act"] == "relu":
                x = x.clamp(min=0)
            elif case["act"] == "gate":
                gate, up = x.split(case["k"], dim=1)
                x = gate * torch.sigmoid(gate) * up
            q, scale = _rows8_64(x)
            return q * scale[:, None], scale
        a = s["q"].double() * s["qs"].double()[:, None]
        out = a @ (s["w"].double() * s["ws"].double()[:, None]).t()
        if s["bias"] is not None:
            out += s["bias"].double()
        if s["res"] is not None:
            out += s["res"].double()
        return out
