"""The operators of attention with a key-value cache as cases that can be timed and checked.

A case is one pass through one operator, as a serving or training program calls it between the
projection that makes queries, keys and values and the one that takes attention's result.

Kinds, and the range each stands for (`draw` covers it):

  heads   a training step's RMS norm of each query and key head with the position rotation, forward
          and backward; 1 to 65536 tokens, 1 to 72 query heads, head widths 32 to 256
  step    the same pass in serving, which writes keys and values into the cache: single tokens of
          many sequences, or whole prompts; 1 to 65536 tokens, caches of 16 and 8 bits
  cache   keys and values into the cache and back out of it, as they are
  attend  one new token's attention for each of 1 to 256 sequences over 0 to 131072 cached keys,
          1 to 16 heads of keys with 1 to 72 query heads each

The cache is paged: keys and values [pages, heads, page, d]. Within a page's head, blocks of 16 tokens
lie one after another, each in the order in which the matrix instruction takes its operands:

  keys    [d / w][16 tokens][w], w = 8 values of 16 bits or 16 of 8 bits
  values  [d / (16 c)][4][16][c][4]: token 4 g + j, channel 16 (c b + e) + i at [b][g][i][e][j], c = 2
          (4 for 8 bits where d is a multiple of 64)

An 8-bit cache holds each token's head as round(127 x / a), a its largest magnitude, beside scales
a / 127, [pages, heads, page]. What is written to it is read back for the comparison, as the values that
it stands for.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
_HEADS, _CACHE, _ATTEND = 1 << 27, 1 << 27, 1 << 31  # most values of a case
_LOG2E = 1.4426950408889634


def listed():
    return [
        # A training step at an odd number of tokens and heads, half of each head rotated, neighbours in pairs.
        dict(name="heads_train_odd", kind="heads", t=1531, hq=7, hkv=7, d=96, r=48, interleaved=True, dtype="f16"),
        # A training step over a large batch, eight query heads to a head of keys.
        dict(name="heads_train_large", kind="heads", t=16384, hq=48, hkv=6, d=128, r=128, interleaved=False, dtype="bf16"),
        # One token of one sequence: the smallest call, latency alone.
        dict(name="step_token", kind="step", t=1, prompt=False, hq=32, hkv=8, d=128, r=128, interleaved=False, page=16,
             bits=16, dtype="bf16"),
        # One token of each sequence of a batch, into an 8-bit cache.
        dict(name="step_batch_q8", kind="step", t=61, prompt=False, hq=20, hkv=4, d=96, r=96, interleaved=False, page=32,
             bits=8, dtype="f16"),
        # A prompt of an odd length into an 8-bit cache.
        dict(name="step_prompt_q8", kind="step", t=4099, prompt=True, hq=32, hkv=8, d=128, r=64, interleaved=False, page=64,
             bits=8, dtype="bf16"),
        # Keys and values of a batch's tokens in and out of an 8-bit cache.
        dict(name="cache_batch_q8", kind="cache", t=48, prompt=False, hkv=8, d=64, page=16, bits=8, dtype="bf16"),
        # A long shared prefix in and out of a 16-bit cache.
        dict(name="cache_prefix", kind="cache", t=32771, prompt=True, hkv=8, d=128, page=64, bits=16, dtype="f16"),
        # The first tokens of one sequence's answer: latency.
        dict(name="attend_short", kind="attend", b=1, longest=77, ragged=False, hq=32, hkv=8, d=128, page=16, bits=16, lse=False,
             dtype="bf16"),
        # One sequence with a very long context: the cache's length is all there is to split.
        dict(name="attend_long", kind="attend", b=1, longest=131071, ragged=False, hq=32, hkv=8, d=128, page=64, bits=16, lse=True,
             dtype="bf16"),
        # A batch of lengths from none to 8192 over an 8-bit cache.
        dict(name="attend_ragged_q8", kind="attend", b=61, longest=8192, ragged=True, hq=32, hkv=4, d=128, page=32, bits=8,
             lse=False, dtype="f16"),
        # All query heads on one head of keys.
        dict(name="attend_one_head", kind="attend", b=16, longest=4097, ragged=True, hq=71, hkv=1, d=64, page=16, bits=16, lse=False,
             dtype="f16"),
        # A full batch at a common length: the cache's bytes are all there is.
        dict(name="attend_large", kind="attend", b=256, longest=4096, ragged=False, hq=32, hkv=8, d=128, page=64, bits=16, lse=False,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads_of(rng):
    hkv = _log_int(rng, 1, 16)
    group = rng.choice((1, 1, 2, 3, 4, 4, 5, 7, 8, 8, 16))
    if hkv <= 2 and rng.random() < 0.4:
        group = _log_int(rng, 8, 72 // hkv)
    return min(hkv * group, 72 // hkv * hkv), hkv


def draw(rng):
    kind = rng.choice(("heads", "step", "step", "cache", "attend", "attend", "attend", "attend"))
    dtype, bits, page = rng.choice(("f16", "bf16")), rng.choice((8, 16)), rng.choice((16, 32, 48, 64, 128))
    d = rng.choice((32, 64, 64, 96, 128, 128, 128, 160, 192, 256))
    hq, hkv = _heads_of(rng)
    r, interleaved = rng.choice((d, d, d // 2, 16)), rng.random() < 0.3
    if kind == "heads":
        t = _log_int(rng, 1, min(65536, _HEADS // ((hq + 2 * hkv) * d)))
        return dict(kind=kind, t=t, hq=hq, hkv=hkv, d=d, r=r, interleaved=interleaved, dtype=dtype)
    if kind in ("step", "cache"):
        prompt = rng.random() < 0.5
        t = _log_int(rng, 1, 256 if not prompt else min(65536, _CACHE // ((hq + 2 * hkv) * d)))
        c = dict(kind=kind, t=t, prompt=prompt, hkv=hkv, d=d, page=page, bits=bits, dtype=dtype)
        return dict(c, hq=hq, r=r, interleaved=interleaved) if kind == "step" else c
    b = _log_int(rng, 1, 256)
    longest = _log_int(rng, 1, min(131072, _ATTEND // (b * hkv * 2 * d), 2 * _ATTEND // (b * hq * d)))
    return dict(kind=kind, b=b, longest=longest, ragged=rng.random() < 0.6, hq=hq, hkv=hkv, d=d, page=page, bits=bits,
                lse=rng.random() < 0.3, dtype=dtype)


# ---- inputs -----------------------------------------------------------------------------------

def _lengths(case):
    """The sequences' lengths, without their order: alike, or from next to nothing to the longest, every
    sixteenth a row of a padded batch, which has none."""
    b, longest = case["b"], case["longest"]
    part = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(b)]
    if case["ragged"]:
        n = [max(1, int(longest * p * p)) if i % 16 != 15 else 0 for i, p in enumerate(part)]
    else:
        n = [longest - int(0.05 * longest * p) for p in part]
    return [longest] + n[1:]


class _Draws:
    """Values from the seed alone, drawn on the GPU."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda")
        self.gen.manual_seed(seed)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return (t * std + mean).to(dtype)

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")

    def uniform(self, *shape, lo, hi):
        return torch.rand(shape, generator=self.gen, device="cuda") * (hi - lo) + lo

    def projected(self, t, h, d, dtype):
        """What a projection gives: every channel with a spread of its own."""
        spread = torch.exp(self.normal(h, d, std=0.4))
        return (self.normal(t, h, d) * spread).to(dtype)

    def filled(self, shape, bits, dtype):
        """A cache in use: keys or values, and scales where it holds 8 bits."""
        if bits == 16:
            return torch.randn(shape, generator=self.gen, device="cuda", dtype=dtype), None
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float16)
        return t.mul_(40).round_().clamp_(-127, 127).to(torch.int8), self.uniform(*shape[:3], lo=0.015, hi=0.04)


def _rope(r, positions):
    """[positions, r]: the cosines of each position's r / 2 angles, then the sines."""
    f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(case, seed):
    g, dt, kind = _Draws(seed), _TYPES[case["dtype"]], case["kind"]
    s, d = dict(case, dt=dt), case["d"]
    if kind in ("heads", "step"):
        t, hq, hkv = case["t"], case["hq"], case["hkv"]
        s["qkv"] = g.projected(t, hq + 2 * hkv, d, dt)
        s["qn"], s["kn"] = g.normal(d, std=0.1, mean=1.0), g.normal(d, std=0.1, mean=1.0)
        span = 4096 if kind == "heads" or not case["prompt"] else max(t, 16)
        s["rope"] = _rope(case["r"], span)
        at = torch.arange(t, device="cuda") % span
        if kind == "step" and not case["prompt"]:
            at = (g.uniform(t, lo=0.0, hi=1.0) * span).long().clamp_(max=span - 1)
        s["pos"] = at.to(torch.int32)
    if kind == "heads":
        s["dq"], s["dk"], s["dv"] = g.normal(t, hq, d, dtype=dt), g.normal(t, hkv, d, dtype=dt), g.normal(t, hkv, d, dtype=dt)
        for name in ("qkv", "qn", "kn"):
            s[name].requires_grad_()
    if kind in ("step", "cache"):
        t, hkv, page = case["t"], case["hkv"], case["page"]
        if kind == "cache":
            s["k"], s["v"] = g.projected(t, hkv, d, dt), g.projected(t, hkv, d, dt)
        # a prompt's tokens fill pages from their start, single tokens go where their sequences end
        pages = -(-t // page) + 3 if case["prompt"] else t + 3
        at = torch.arange(t, device="cuda")
        where = g.order(pages)
        if case["prompt"]:
            slots = where[at // page] * page + at % page
        else:
            slots = where[at] * page + (g.uniform(t, lo=0.0, hi=1.0) * page).long().clamp_(max=page - 1)
            slots = torch.where(at % 16 == 15, torch.full_like(slots, -1), slots)  # a padded batch's rows
        s["slots"] = slots.to(torch.int32)
        shape = (pages, hkv, page, d)
        if case["bits"] == 16:
            s["cache"] = (torch.zeros(shape, dtype=dt, device="cuda"), torch.zeros(shape, dtype=dt, device="cuda"), None, None)
        else:
            s["cache"] = tuple(torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in range(2)) + tuple(
                torch.zeros(shape[:3], device="cuda") for _ in range(2))
    if kind == "attend":
        b, page = case["b"], case["page"]
        n = torch.tensor(_lengths(case), device="cuda")[g.order(b)]
        per = -(-case["longest"] // page)
        pages = int(sum(-(-x // page) for x in _lengths(case))) + 3
        shape = (pages, case["hkv"], page, d)
        k, ks = g.filled(shape, case["bits"], dt)
        v, vs = g.filled(shape, case["bits"], dt)
        s["cache"] = (k, v, ks, vs)
        used = (n + page - 1) // page
        first = torch.cumsum(used, 0) - used
        col = torch.arange(per, device="cuda")[None, :]
        live = col < used[:, None]
        table = g.order(pages)[torch.where(live, first[:, None] + col, torch.zeros_like(col))]
        s["table"] = torch.where(live, table, torch.full_like(table, -1)).to(torch.int32).contiguous()
        s["len"] = n.to(torch.int32)
        s["q"] = g.normal(b, case["hq"], d, dtype=dt)
        s["scale"] = d ** -0.5
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


def _run_own(s):
    hip, torch_ops = _own()
    if s["kind"] == "heads":
        y = torch_ops.qk_norm_rope(s["qkv"], s["qn"], s["kn"], s["rope"], s["pos"], s["hkv"], EPS, s["interleaved"])
        grads = torch.autograd.grad(y, (s["qkv"], s["qn"], s["kn"]), (s["dq"], s["dk"], s["dv"]))
        return tuple(t.detach() for t in y) + grads
    if s["kind"] == "attend":
        return hip.paged_attention(s["q"], s["cache"], s["table"], s["len"], s["scale"], want_lse=s["lse"])
    q = None
    if s["kind"] == "step":
        q = hip.qk_norm_rope_cache(s["qkv"], s["qn"], s["kn"], s["rope"], s["pos"], s["slots"], s["cache"], EPS, s["interleaved"])
    else:
        hip.kv_cache_write(s["k"], s["v"], s["slots"], s["cache"])
    if s["kind"] == "step" and s["bits"] == 16:
        return q, s["cache"][0], s["cache"][1]
    k, v = hip.kv_cache_read(s["cache"], s["slots"], s["dt"])
    return q, k, v, s["cache"][2], s["cache"][3]


def _pairs(x, r, interleaved):
    """The channels that are rotated together: the first r, halves or neighbours."""
    if interleaved:
        return x[..., 0:r:2], x[..., 1:r:2]
    return x[..., :r // 2], x[..., r // 2:r]


def _turned(x, cos, sin, r, interleaved):
    a, b = _pairs(x, r, interleaved)
    y = x.clone()
    ya, yb = _pairs(y, r, interleaved)
    ya.copy_(a * cos - b * sin)
    yb.copy_(a * sin + b * cos)
    return y


def _angles(s):
    rows = s["rope"][s["pos"].long()][:, None]
    return rows[..., :s["r"] // 2], rows[..., s["r"] // 2:]


def _normed(s):
    """Queries and keys after norm and rotation, in 32 bits."""
    x, hq, hkv = s["qkv"].float(), s["hq"], s["hkv"]
    cos, sin = _angles(s)
    x = x[:, :hq + hkv]
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * r
    q = _turned(xh[:, :hq] * s["qn"], cos, sin, s["r"], s["interleaved"])
    k = _turned(xh[:, hq:] * s["kn"], cos, sin, s["r"], s["interleaved"])
    return q, k, xh, r, cos, sin


def _run_heads(s):
    dt, hq, hkv = s["dt"], s["hq"], s["hkv"]
    q, k, xh, r, cos, sin = _normed(s)
    grads, ws = [], []
    for dy, w, lo, hi in ((s["dq"], s["qn"], 0, hq), (s["dk"], s["kn"], hq, hq + hkv)):
        g = _turned(dy.float(), cos, -sin, s["r"], s["interleaved"])
        h = xh[:, lo:hi]
        ws.append((g * h).sum((0, 1)))
        g = g * w
        grads.append(r[:, lo:hi] * (g - h * (g * h).mean(-1, keepdim=True)))
    dqkv = torch.cat(grads + [s["dv"].float()], 1).to(dt)
    return q.to(dt), k.to(dt), s["qkv"][:, hq + hkv:].clone(), dqkv, ws[0], ws[1]


def _channels(d, bits, device):
    """Where channels lie in a block of 16 tokens, and how far apart its tokens do: keys, then values."""
    c = torch.arange(d, device=device)
    w = 8 if bits == 16 else 16
    e = 2 if bits == 16 or d % 64 else 4
    block = c // 16
    return c // w * 16 * w + c % w, w, block // e * 256 * e + c % 16 * 4 * e + block % e * 4, e


def _places(s):
    """The flat places in the cache of each token's heads: keys', values', scales' [t, hkv, d], and the tokens that have one."""
    k, ks = s["cache"][0], s["cache"][2]
    pages, hkv, page, d = k.shape
    kc, w, vc, e = _channels(d, 16 if ks is None else 8, k.device)
    slots = s["slots"].long()
    live = (slots >= 0) & (slots < pages * page)
    at = torch.where(live, slots, torch.zeros_like(slots))
    row = (at // page)[:, None] * hkv + torch.arange(hkv, device=k.device)
    o = (at % page)[:, None]
    base = (row * page + o // 16 * 16) * d
    i = o % 16
    kp = (base + i * w)[..., None] + kc
    vp = (base + i // 4 * 64 * e + i % 4)[..., None] + vc
    return kp, vp, row * page + o, live


def _eight_bits(t):
    a = t.abs().amax(-1)
    return torch.round(t * torch.where(a > 0, 127.0 / a, a)[..., None]), a / 127.0


def _write(s, k, v):
    kp, vp, sp, live = _places(s)
    kc, vc, ks, vs = s["cache"]
    for x, c, sc, p in ((k, kc, ks, kp), (v, vc, vs, vp)):
        if sc is not None:
            x, a = _eight_bits(x)
            sc.view(-1)[sp[live]] = a[live]
        c.view(-1)[p[live]] = x[live].to(c.dtype)


def _read(s):
    kp, vp, sp, live = _places(s)
    kc, vc, ks, vs = s["cache"]
    out = []
    for c, sc, p in ((kc, ks, kp), (vc, vs, vp)):
        x = c.view(-1)[p].float()
        if sc is not None:
            x = x * sc.view(-1)[sp][..., None]
        out.append(torch.where(live[:, None, None], x, torch.zeros_like(x)).to(s["dt"]))
    return out


def _run_step(s):
    q = None
    if s["kind"] == "step":
        q, k, *_ = _normed(s)
        q, v = q.to(s["dt"]), s["qkv"][:, s["hq"] + s["hkv"]:].float()
    else:
        k, v = s["k"].float(), s["v"].float()
    _write(s, k, v)
    if s["kind"] == "step" and s["bits"] == 16:
        return q, s["cache"][0], s["cache"][1]
    k, v = _read(s)
    return q, k, v, s["cache"][2], s["cache"][3]


def _dense(c, values, sc):
    """Cached keys or values as [pages, heads, page, d], in 32 bits."""
    p, h, n, d = c.shape
    if values:
        e = 2 if sc is None or d % 64 else 4
        x = c.view(p, h, n // 16, d // 16 // e, 4, 16, e, 4).permute(0, 1, 2, 4, 7, 3, 6, 5)
    else:
        w = 8 if sc is None else 16
        x = c.view(p, h, n // 16, d // w, 16, w).permute(0, 1, 2, 4, 3, 5)
    x = x.reshape(p, h, n, d).float()
    return x if sc is None else x * sc[..., None]


def _run_attend(s):
    (kc, vc, ks, vs), b, hkv, d = s["cache"], s["b"], s["hkv"], s["d"]
    table = s["table"].long().clamp(min=0)
    take = lambda c, sc, values: _dense(c[table.view(-1)], values, None if sc is None else sc[table.view(-1)]).view(  # noqa: E731
        b, -1, hkv, s["page"], d).transpose(1, 2).reshape(b, hkv, -1, d)
    k = take(kc, ks, False)
    live = (torch.arange(k.shape[2], device=k.device) < s["len"][:, None])[:, None, None]
    q = s["q"].float().view(b, hkv, -1, d)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    del k
    x = torch.where(live, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    v = take(vc, vs, True)
    v = torch.where(live.transpose(2, 3), v, torch.zeros_like(v))
    out = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)) * _LOG2E
    return out.view(b, -1, d).to(s["dt"]), (lse.view(b, -1) if s["lse"] else None)


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"heads": _run_heads, "step": _run_step, "cache": _run_step, "attend": _run_attend}[s["kind"]](s)


# ---- what a pass cannot do without ------------------------------------------------------------

def work(case):
    d, kind = case["d"], case["kind"]
    if kind == "heads":
        t, h = case["t"], case["hq"] + 2 * case["hkv"]
        table = 4 * case["r"] * min(t, 4096)
        return {"bytes": 2 * 5 * t * h * d + table + 4 * t + 16 * d, "flops": 25 * t * h * d}
    if kind in ("step", "cache"):
        t, n = case["t"], 2 * case["t"] * case["hkv"]
        cached = n * d * 2 if case["bits"] == 16 else n * (d + 4)
        if kind == "cache":  # in, held, and out again
            return {"bytes": 2 * 2 * n * d + cached + 4 * t, "flops": (1 if case["bits"] == 16 else 6) * n * d}
        back = 0 if case["bits"] == 16 else 2 * n * d
        x = t * (case["hq"] + 2 * case["hkv"]) * d
        return {"bytes": 2 * x + 2 * t * case["hq"] * d + cached + back + t * (4 * case["r"] + 8), "flops": 12 * x}
    n = sum(_lengths(case))
    row = 2 * d * 2 if case["bits"] == 16 else 2 * (d + 4)
    b = case["b"]
    return {"bytes": n * case["hkv"] * row + 4 * b * case["hq"] * d + 4 * b + 4 * -(-n // case["page"]),
            "flops": 4 * n * case["hq"] * d}


# ---- the same in 64 bits ----------------------------------------------------------------------

def _rotation(x, table, r, neighbours):
    """x [t, h, d] with each token's pairs multiplied by its complex unit numbers."""
    z = torch.complex(table[:, :r // 2], table[:, r // 2:])[:, None]
    head, tail = x[..., :r], x[..., r:]
    if neighbours:
        y = torch.view_as_real(torch.view_as_complex(head.reshape(*head.shape[:2], r // 2, 2).contiguous()) * z).flatten(2)
    else:
        c = torch.complex(*head.chunk(2, -1)) * z
        y = torch.cat([c.real, c.imag], -1)
    return torch.cat([y, tail], -1)


def _heads64(s):
    with torch.enable_grad():
        x = s["qkv"].detach().double().requires_grad_()
        wq, wk = (s[n].detach().double().requires_grad_() for n in ("qn", "kn"))
        table = s["rope"].double()[s["pos"].long()]
        q, k, v = x.split([s["hq"], s["hkv"], s["hkv"]], 1)
        q, k = (_rotation(h * torch.rsqrt(h.square().sum(-1, keepdim=True) / s["d"] + EPS) * w, table, s["r"], s["interleaved"])
                for h, w in ((q, wq), (k, wk)))
        return x, wq, wk, q, k, v


def _held64(t, bits):
    """What the cache holds of t [t, h, d], and the scales."""
    if bits == 16:
        return t, None
    a = t.abs().max(-1, keepdim=True).values
    n = torch.where(a > 0, (t * 127.0 / a).round(), torch.zeros_like(t))
    return n * a / 127.0, a[..., 0] / 127.0


def _rows64(c, sc, pages, values):
    """The cached rows of some pages [pages, heads, page, d], out of the operands' order."""
    p, h, n, d = c.shape
    blocks, small = c.double().reshape(p * h * (n // 16), 16 * d), sc is not None
    token, channel = torch.meshgrid(torch.arange(16, device=c.device), torch.arange(d, device=c.device), indexing="ij")
    if values:
        e = 4 if small and d % 64 == 0 else 2
        group, rest = channel // (16 * e), channel % (16 * e)
        at = ((((group * 4 + token // 4) * 16 + rest % 16) * e + rest // 16) * 4) + token % 4
    else:
        w = 16 if small else 8
        at = (channel // w * 16 + token) * w + channel % w
    rows = blocks[:, at.flatten()].view(p, h, n, d)
    return rows * sc[pages].double()[..., None] if small else rows


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "heads":
        x, wq, wk, q, k, v = _heads64(s)
        g = torch.autograd.grad((q, k, v), (x, wq, wk), (s["dq"].double(), s["dk"].double(), s["dv"].double()))
        return (q.detach(), k.detach(), v.detach()) + g
    with torch.no_grad():
        if case["kind"] in ("step", "cache"):
            q = None
            if case["kind"] == "step":
                _, _, _, q, k, v = (t.detach() for t in _heads64(s))
            else:
                k, v = s["k"].double(), s["v"].double()
            live = (s["slots"] >= 0)[:, None]
            (k, ks), (v, vs) = _held64(k, case["bits"]), _held64(v, case["bits"])
            if case["kind"] == "step" and case["bits"] == 16:
                pages, hkv, page, d = s["cache"][0].shape
                slots = s["slots"].long()[s["slots"] >= 0]
                out = [q]
                for t, values in ((k, False), (v, True)):
                    full = torch.zeros((pages * page, hkv, d), dtype=torch.float64, device=t.device)
                    full[slots] = t[live[:, 0]]
                    full = full.view(pages, page // 16, 16, hkv, d).permute(0, 3, 1, 2, 4)  # pages, heads, blocks, tokens, d
                    if values:
                        full = full.reshape(pages, hkv, page // 16, 4, 4, d // 32, 2, 16).permute(0, 1, 2, 5, 3, 7, 6, 4)
                    else:
                        full = full.reshape(pages, hkv, page // 16, 16, d // 8, 8).transpose(3, 4)
                    out.append(full.reshape(pages, hkv, page, d))
                return tuple(out)
            k, v = (t * live[..., None] for t in (k, v))
            scales = [None, None]
            if case["bits"] == 8:
                pages, hkv, page, _ = s["cache"][0].shape
                slots = s["slots"].long()[s["slots"] >= 0]
                scales = []
                for t in (ks, vs):
                    full = torch.zeros((pages * page, hkv), dtype=torch.float64, device=t.device)
                    full[slots] = t[live[:, 0]]
                    scales.append(full.view(pages, page, hkv).transpose(1, 2).contiguous())
            return q, k, v, scales[0], scales[1]
        out, lse = [], []
        kc, vc, ks, vs = s["cache"]
        group, page = case["hq"] // case["hkv"], case["page"]
        for q, pages, n in zip(s["q"].double(), s["table"].long(), s["len"].tolist()):
            if n == 0:
                out.append(torch.zeros_like(q))
                lse.append(torch.full_like(q[:, 0], -math.inf))
                continue
            pages = pages[:-(-n // page)]
            k, v = _rows64(kc[pages], ks, pages, False), _rows64(vc[pages], vs, pages, True)
            k, v = (t.transpose(1, 2).reshape(-1, case["hkv"], case["d"])[:n].transpose(0, 1) for t in (k, v))
            x = torch.bmm(q.view(case["hkv"], group, -1), k.transpose(1, 2).contiguous()) * s["scale"]
            out.append(torch.bmm(torch.softmax(x, -1), v.contiguous()).view(case["hq"], -1))
            lse.append(torch.logsumexp(x, -1).view(-1) / math.log(2.0))
        return torch.stack(out), (torch.stack(lse) if case["lse"] else None)
