"""Heads, the key-value cache and its attention on the CPU: the float64 oracle against independent statements, the cache's
order place by place, and every refusal of the entry points, none of which touches a device. No kernel is launched here."""
import numpy as np
import pytest
import torch

from colabfold_legacy_kernels import hip as H
from colabfold_legacy_kernels import layouts, torch_ops
from oracle import heads as oh
from test_capi import F16, F32, S32, buf, lib  # noqa: F401

S8, BF16 = 2, 16


# ---- the oracle ---------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_complex_multiplication(interleaved):
    rng = np.random.default_rng(0)
    x, angle = rng.standard_normal((3, 2, 10)), rng.uniform(-9, 9, (3, 4))
    y = oh.rotate(x, np.cos(angle), np.sin(angle), interleaved)
    a, b = oh.pairs(8, interleaved)
    z = (x[..., a] + 1j * x[..., b]) * np.exp(1j * angle)[:, None]
    assert np.allclose(y[..., a], z.real) and np.allclose(y[..., b], z.imag) and np.array_equal(y[..., 8:], x[..., 8:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients_against_differences(interleaved):
    """By central differences with steps of 1e-5: about 1e-10 from the third derivative, 1e-16 / 1e-5 from the subtraction."""
    rng = np.random.default_rng(1)
    x, w, dy = rng.standard_normal((2, 3, 8)), rng.standard_normal(8), rng.standard_normal((2, 3, 8))
    rope, pos, eps, h = layouts.rope_table(7, 4, 10.0).numpy(), np.array([6, 2]), 1e-3, 1e-5

    def loss(x, w):
        return (oh.norm_rope(x, w, rope, pos, eps, interleaved)[0] * dy).sum()

    dx, _, dw, _ = oh.norm_rope_bwd(x, w, rope, pos, dy, eps, interleaved)
    for i in np.ndindex(x.shape):
        d = np.zeros(x.shape)
        d[i] = h
        assert abs((loss(x + d, w) - loss(x - d, w)) / (2 * h) - dx[i]) < 1e-8
    for j in range(8):
        d = np.zeros(8)
        d[j] = h
        assert abs((loss(x, w + d) - loss(x, w - d)) / (2 * h) - dw[j]) < 1e-8


def test_attend_is_a_weighted_sum():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((2, 4)), rng.standard_normal((5, 4)), rng.standard_normal((5, 4))
    out, lse, _, _ = oh.attend(q, k, v, 0.7)
    for g in range(2):
        e = [np.exp(0.7 * float(q[g] @ k[j])) for j in range(5)]
        assert np.allclose(out[g], sum(e[j] * v[j] for j in range(5)) / sum(e)) and np.isclose(lse[g], np.log2(sum(e)))
    out, lse, _, _ = oh.attend(q, k[:0], v[:0], 0.7)
    assert (out == 0).all() and (lse == -np.inf).all()


# ---- layouts ------------------------------------------------------------------------------

@pytest.mark.parametrize("lib_", ("numpy", "torch"))
@pytest.mark.parametrize("dtype", ("float16", "int8"))
@pytest.mark.parametrize("d", (32, 64, 96, 128))
def test_cache_order(lib_, dtype, d):
    x = np.random.default_rng(d).integers(-127, 128, (2, 3, 48, d)).astype(dtype)
    arg = torch.from_numpy(x) if lib_ == "torch" else x
    for values, there, back in ((False, layouts.keys_blocked, layouts.keys_unblocked),
                                (True, layouts.values_blocked, layouts.values_unblocked)):
        y = there(arg)
        for p in range(2):
            for h in range(3):
                assert np.array_equal(np.asarray(y)[p, h], oh.blocked(x[p, h], values, dtype == "int8"))
        assert np.array_equal(np.asarray(back(y)), x)


def test_cache_order_refuses_other_shapes():
    for shape in ((1, 1, 16, 40), (1, 1, 24, 32), (1, 16, 32)):
        with pytest.raises(ValueError, match="page a multiple of 16"):
            layouts.keys_blocked(torch.zeros(shape, dtype=torch.int8))


def test_rope_table():
    t = layouts.rope_table(100001, 6, 500.0)
    assert t.shape == (100001, 6) and t.dtype == torch.float32
    for p in (0, 1, 77, 100000):
        for i in range(3):
            angle = p * 500.0 ** (-2 * i / 6)
            assert abs(float(t[p, i]) - np.cos(angle)) < 1e-7 and abs(float(t[p, 3 + i]) - np.sin(angle)) < 1e-7


def test_cache_slots():
    table = torch.tensor([[5, 2, -1], [0, 7, 3]], dtype=torch.int32)
    s = torch_ops.cache_slots(table, torch.tensor([[0, 15, 16, 31, 32, -1], [47, 48, 20, 0, -7, 1]]), 16)
    assert s.dtype == torch.int32
    assert s.tolist() == [[80, 95, 32, 47, -1, -1], [63, -1, 116, 0, -1, 1]]
    assert torch_ops.cache_slots(table, torch.tensor([17, 33]), 16).tolist() == [33, 49]


def test_cache_slots_at_the_edges():
    pos = torch.tensor([[0, 63], [64, 127]])
    # pages whose slots would come round to slots of other pages in int32, and the largest that do not
    table = torch.tensor([[2 ** 26, 0], [2 ** 31 - 1, 2 ** 25 - 1]], dtype=torch.int32)
    assert torch_ops.cache_slots(table, pos, 64).tolist() == [[-1, -1], [2 ** 31 - 64, 2 ** 31 - 1]]
    assert torch_ops.cache_slots(table[:, :0], pos, 64).tolist() == [[-1, -1], [-1, -1]]
    assert torch_ops.cache_slots(table[:0], pos[:0], 64).shape == (0, 2)
    assert torch_ops.cache_slots(table[:0], pos[:0, 0], 64).shape == (0,)
    assert torch_ops.cache_slots(table, pos[:, :0], 64).shape == (2, 0)
    for bad in ((table, pos[:1], 64), (table[0], pos, 64), (table, pos[None], 64), (table, pos, 0), (table, torch.tensor(3), 16)):
        with pytest.raises(H.InvalidArgument, match="cache_slots"):
            torch_ops.cache_slots(*bad)


def test_kv_cache():
    c = H.kv_cache(3, 2, 16, 64, device="cpu")
    assert c.k.shape == c.v.shape == (3, 2, 16, 64) and c.k.dtype == torch.int8 and c.k_scale.shape == (3, 2, 16)
    c = H.kv_cache(3, 2, 16, 64, torch.bfloat16, device="cpu")
    assert c.v.dtype == torch.bfloat16 and c.k_scale is None and c.v_scale is None


# ---- refusals of the C entry points ----------------------------------------------------------

T, HQ, HKV, D, R, P = 6, 4, 2, 64, 32, 100


def refs(args):
    return [a[0] for a in args]


def refused(lib, status, message):
    assert status == 3 and message in lib.clk_last_error().decode(), (status, message, lib.clk_last_error())


def head_args(act=F16, t=T, d=D):
    return dict(qkv=buf(act, t, HQ + 2 * HKV, d), qn=buf(F32, d), kn=buf(F32, d), rope=buf(F32, P, R), pos=buf(S32, t))


HEADS = [
    (dict(qkv=buf(F16, T, 8 * D)), "qkv must be [T,Hq+2*Hkv,D]"),
    (dict(qkv=buf(F32, T, 8, D)), "must be F16, got F32"),
    (dict(qkv=buf(F16, T, 4, D)), "at least one query and one key head"),
    (dict(qkv=buf(F16, T, 8, 60)), "D must be a multiple of 8 up to 256"),
    (dict(qkv=buf(F16, T, 8, 264)), "D must be a multiple of 8 up to 256"),
    (dict(qkv=buf(F16, T, 8, D, data=0x100008)), "16-byte aligned"),
    (dict(qkv=buf(F16, 1 << 31, 8, D)), "too large"),
    (dict(qkv=buf(F16, T, 16385, D)), "too large"),
    (dict(qn=buf(F32, D + 1)), "q_norm and k_norm must be [D]"),
    (dict(kn=buf(F32, D - 1)), "q_norm and k_norm must be [D]"),
    (dict(kn=buf(F16, D)), "must be F32, got F16"),
    (dict(rope=buf(F32, 0, R)), "rope must be [P,R]"),
    (dict(rope=buf(F32, P, D + 8)), "rope must be [P,R]"),
    (dict(rope=buf(F32, P, 12)), "rope must be [P,R]"),
    (dict(rope=buf(F32, P, 0)), "rope must be [P,R]"),
    (dict(rope=buf(F32, P * R)), "rope must be [P,R]"),
    (dict(rope=buf(F32, P, R, data=0x100004)), "16-byte aligned"),
    (dict(pos=buf(S32, T + 1)), "positions must be [T]"),
    (dict(pos=buf(F32, T)), "must be S32"),
]


def forward_args(act=F16, t=T, d=D):
    return dict(head_args(act, t, d), q=buf(act, t, HQ, d), k=buf(act, t, HKV, d), v=buf(act, t, HKV, d))


@pytest.mark.parametrize("other,message", HEADS + [
    (dict(q=buf(F16, T, HQ + 1, D)), "q must be [T,Hq,D]"),
    (dict(k=buf(F16, T, HKV - 1, D)), "q must be [T,Hq,D]"),
    (dict(k=buf(F16, T, 0, D)), "at least one query and one key head"),
    (dict(k=buf(F16, T, HKV * D)), "k [T,Hkv,D]"),
    (dict(v=buf(F16, T - 1, HKV, D)), "q must be [T,Hq,D]"),
    (dict(v=buf(BF16, T, HKV, D)), "must be F16, got BF16"),
    (dict(v=buf(F16, T, HKV, D, data=0x100002)), "16-byte aligned"),
])
def test_qk_norm_rope_refusals(lib, other, message):
    refused(lib, lib.clk_qk_norm_rope(None, *refs({**forward_args(), **other}.values()), 1e-5, 0), message)


def test_qk_norm_rope_eps_and_empty(lib):
    for eps in (-1.0, float("nan")):
        refused(lib, lib.clk_qk_norm_rope(None, *refs(forward_args().values()), eps, 0), "eps must not be negative")
    assert lib.clk_qk_norm_rope(None, *refs(forward_args(t=0).values()), 1e-5, 0) == 0


def bwd_args():
    return dict(head_args(), dq=buf(F16, T, HQ, D), dk=buf(F16, T, HKV, D), dv=buf(F16, T, HKV, D),
                dqkv=buf(F16, T, HQ + 2 * HKV, D), dqn=buf(F32, D), dkn=buf(F32, D))


@pytest.mark.parametrize("other,message", HEADS[1:] + [
    (dict(dq=buf(F16, T, HQ, D + 8)), "dq must be [T,Hq,D]"),
    (dict(dk=buf(F16, T, HKV, D - 8)), "dq must be [T,Hq,D]"),
    (dict(dv=buf(F16, T, HKV + 1, D)), "dq must be [T,Hq,D]"),
    (dict(dqkv=buf(F16, T, HQ + 2 * HKV, D + 8)), "dqkv must be like qkv"),
    (dict(dqn=buf(F32, 1)), "dq_norm and dk_norm must be [D]"),
    (dict(dkn=buf(F32, D + 1)), "dq_norm and dk_norm must be [D]"),
    (dict(dqkv=buf(F16, T, HQ + 2 * HKV, D, data=0x100008)), "16-byte aligned"),
])
def test_qk_norm_rope_bwd_refusals(lib, other, message):
    refused(lib, lib.clk_qk_norm_rope_bwd(None, *refs({**bwd_args(), **other}.values()), 1e-5, 0, 0x100000, 1 << 30), message)


def test_qk_norm_rope_bwd_workspace(lib):
    a = bwd_args()
    need = lib.clk_qk_norm_rope_bwd_workspace_size(a["qkv"][0], a["dk"][0])
    assert need >= 2 * 4 * D and need % 256 == 0
    for ws, size, message in ((0x100000, need - 1, "workspace of"), (None, need, "workspace of"), (0x100010, need, "256-byte aligned")):
        refused(lib, lib.clk_qk_norm_rope_bwd(None, *refs(a.values()), 1e-5, 0, ws, size), message)
    for qkv, dk in ((buf(F16, 0, 8, D), a["dk"]), (buf(F16, T, 8, 60), a["dk"]), (buf(F16, T, 4, D), a["dk"]), (buf(F16, T), a["dk"])):
        assert lib.clk_qk_norm_rope_bwd_workspace_size(qkv[0], dk[0]) == 0
    assert lib.clk_qk_norm_rope_bwd_workspace_size(None, a["dk"][0]) == 0


def cache_args(dtype=F16, pages=5, heads=HKV, page=16, d=D):
    scales = (pages, heads, page) if dtype == S8 else (1,)
    return dict(kc=buf(dtype, pages, heads, page, d), vc=buf(dtype, pages, heads, page, d, data=0x200000), ks=buf(F32, *scales),
                vs=buf(F32, *scales))


CACHE = [
    (cache_args(F32), "must be F16, got F32"),
    (cache_args(BF16), "must be F16, got BF16"),
    (dict(cache_args(S8), vc=buf(F16, 5, HKV, 16, D, data=0x200000)), "must be S8, got F16"),
    (dict(cache_args(), vc=buf(F16, 5, HKV, 32, D, data=0x200000)), "must be [pages,heads,page,D], alike"),
    (dict(cache_args(), kc=buf(F16, 5, HKV, 16 * D)), "must be [pages,heads,page,D], alike"),
    (cache_args(d=48), "a cache's D must be a multiple of 32"),
    (cache_args(d=288), "a cache's D must be a multiple of 32"),
    (cache_args(page=24), "a cache's page must be a multiple of 16"),
    (cache_args(page=0), "a cache's page must be a multiple of 16"),
    (cache_args(pages=0), "a page and a head at least"),
    (cache_args(pages=1 << 27), "too large"),
    (dict(cache_args(S8), ks=buf(F32, 5, HKV)), "scales must be [pages,heads,page]"),
    (dict(cache_args(S8), vs=buf(F32, 5, HKV, 32)), "scales must be [pages,heads,page]"),
    (dict(cache_args(S8), vs=buf(F16, 5, HKV, 16)), "must be F32"),
    (dict(cache_args(), vc=buf(F16, 5, HKV, 16, D)), "must not be the same buffer"),
    (dict(cache_args(), vc=buf(F16, 5, HKV, 16, D, data=0x200008)), "16-byte aligned"),
    (dict(cache_args(S8), ks=buf(F32, 5, HKV, 16, data=0x200004)), "16-byte aligned"),
]


def step_args(cache=F16):
    return dict(head_args(), slots=buf(S32, T), q=buf(F16, T, HQ, D), **cache_args(cache))


@pytest.mark.parametrize("other,message", HEADS + CACHE + [
    (dict(slots=buf(S32, T - 1)), "slots must be [T]"),
    (dict(slots=buf(F32, T)), "must be S32"),
    (dict(q=buf(F16, T, HQ + 2, D)), "q must be [T,Hq,D]"),
    (cache_args(heads=4), "at least one query and one key head"),
    (cache_args(d=96), "the same D"),
    (dict(q=buf(F16, T, HQ, D, data=0x100004)), "16-byte aligned"),
])
def test_qk_norm_rope_cache_refusals(lib, other, message):
    refused(lib, lib.clk_qk_norm_rope_cache(None, *refs({**step_args(), **other}.values()), 1e-5, 0), message)


@pytest.mark.parametrize("other,message", CACHE + [
    (dict(k=buf(F16, T, HKV + 1, D)), "k and v must be [T,heads,D]"),
    (dict(k=buf(F16, T, HKV * D)), "k and v must be [T,heads,D]"),
    (dict(v=buf(F16, T + 1, HKV, D)), "k and v must be [T,heads,D]"),
    (dict(v=buf(BF16, T, HKV, D)), "must be F16, got BF16"),
    (dict(slots=buf(S32, T, 1)), "slots must be [T]"),
    (dict(k=buf(F16, T, HKV, D, data=0x100008)), "16-byte aligned"),
])
def test_moves_refuse(lib, other, message):
    a = {**dict(k=buf(F16, T, HKV, D), v=buf(F16, T, HKV, D), slots=buf(S32, T)), **cache_args(), **other}
    w = [a[n] for n in ("k", "v", "slots", "kc", "vc", "ks", "vs")]
    refused(lib, lib.clk_kv_cache_write(None, *refs(w)), message)
    r = [a[n] for n in ("kc", "vc", "ks", "vs", "slots", "k", "v")]
    refused(lib, lib.clk_kv_cache_read(None, *refs(r)), message)


def attend_args(cache=F16, b=3, n=7):
    return dict(q=buf(F16, b, HQ, D), **cache_args(cache), table=buf(S32, b, n), len=buf(S32, b), out=buf(F16, b, HQ, D),
                lse=buf(F32, b, HQ))


@pytest.mark.parametrize("other,message", CACHE + [
    (dict(q=buf(F16, 3, 5, D), out=buf(F16, 3, 5, D)), "Hq a multiple of the cache's heads"),
    (dict(q=buf(F16, 3, HQ, 96), out=buf(F16, 3, HQ, 96)), "D its D"),
    (dict(q=buf(F16, 3, 0, D), out=buf(F16, 3, 0, D)), "q must be [B,Hq,D]"),
    (dict(q=buf(F16, 3, HQ * D)), "q must be [B,Hq,D]"),
    (dict(q=buf(F32, 3, HQ, D)), "must be F16, got F32"),
    (dict(table=buf(S32, 4, 7)), "page_table must be"),
    (dict(table=buf(S32, 3, 0)), "page_table must be"),
    (dict(table=buf(S32, 21)), "page_table must be"),
    (dict(table=buf(F32, 3, 7)), "must be S32"),
    (dict(table=buf(S32, 3, 1 << 27)), "too large"),
    (dict(len=buf(S32, 2)), "lengths must be [B]"),
    (dict(out=buf(F16, 3, HQ, 32)), "out must be like q"),
    (dict(out=buf(BF16, 3, HQ, D)), "must be F16, got BF16"),
    (dict(lse=buf(F32, 3)), "lse must be [B,Hq]"),
    (dict(out=buf(F16, 3, HQ, D, data=0x100008)), "16-byte aligned"),
])
def test_paged_attention_refusals(lib, other, message):
    a = {**attend_args(), **other}
    refused(lib, lib.clk_paged_attention(None, *refs(a.values()), 0.1, 1, 0x100000, 1 << 40), message)


def test_paged_attention_scale_past_its_range(lib):
    a = attend_args()
    for scale in (3e38, -3e38):  # times log2(e) it is infinite
        refused(lib, lib.clk_paged_attention(None, *refs(a.values()), scale, 1, 0x100000, 1 << 40), "scale must be finite")


def test_paged_attention_scale_workspace_and_empty(lib):
    a = attend_args()
    for scale in (float("nan"), float("inf")):
        refused(lib, lib.clk_paged_attention(None, *refs(a.values()), scale, 1, 0x100000, 1 << 40), "scale must be finite")
    big = {**attend_args(b=61, n=512), **cache_args(S8, pages=5)}
    need = lib.clk_paged_attention_workspace_size(big["q"][0], big["kc"][0], big["table"][0])
    if need:
        for ws, size, message in ((0x100000, need - 1, "workspace of"), (None, need, "workspace of"),
                                  (0x100010, need, "256-byte aligned")):
            refused(lib, lib.clk_paged_attention(None, *refs(big.values()), 0.1, 1, ws, size), message)
    assert lib.clk_paged_attention_workspace_size(None, a["kc"][0], a["table"][0]) == 0
    assert lib.clk_paged_attention_workspace_size(buf(F16, 3, 5, D)[0], a["kc"][0], a["table"][0]) == 0
    assert lib.clk_paged_attention(None, *refs(attend_args(b=0).values()), 0.1, 1, None, 0) == 0


# ---- refusals of the Python entry points -------------------------------------------------------

def test_cpu_tensors_are_refused():
    qkv, w, rope = torch.zeros((4, 8, 64), dtype=torch.float16), torch.ones(64), layouts.rope_table(10, 64)
    pos = torch.zeros(4, dtype=torch.int32)
    c = H.kv_cache(3, 2, 16, 64, device="cpu")
    q, k = qkv[:, :4].contiguous(), qkv[:, :2].contiguous()
    table = torch.zeros((4, 2), dtype=torch.int32)
    for call in (lambda: H.qk_norm_rope(qkv, w, w, rope, pos, 2), lambda: H.qk_norm_rope_bwd(qkv, w, w, rope, pos, q, k, k),
                 lambda: H.qk_norm_rope_cache(qkv, w, w, rope, pos, pos, c), lambda: H.kv_cache_write(k, k, pos, c),
                 lambda: H.kv_cache_read(c, pos), lambda: H.paged_attention(q, c, table, pos),
                 lambda: torch_ops.qk_norm_rope(qkv, w, w, rope, pos, 2), lambda: torch_ops.kv_cache_write(k, k, pos, c),
                 lambda: torch_ops.qk_norm_rope(qkv.requires_grad_(), w, w, rope, pos, 2)):
        with pytest.raises(H.InvalidArgument, match="must be on one GPU"):
            call()


def test_shapes_and_caches_are_refused():
    x, w, rope = torch.zeros((4, 64), dtype=torch.float16), torch.ones(64), layouts.rope_table(10, 64)
    pos = torch.zeros(4, dtype=torch.int32)
    c = H.kv_cache(3, 2, 16, 64, device="cpu")
    for call in (lambda: H.qk_norm_rope(x, w, w, rope, pos, 2), lambda: H.qk_norm_rope_cache(x, w, w, rope, pos, pos, c),
                 lambda: H.paged_attention(x, c, pos, pos)):
        with pytest.raises(H.InvalidArgument, match="expected .tokens, heads, D."):
            call()
    y = torch.zeros((4, 8, 64), dtype=torch.float16)
    for n in (0, 4, 5, -1):
        for module in (H, torch_ops):
            with pytest.raises(H.InvalidArgument, match="cannot be keys and values"):
                module.qk_norm_rope(y, w, w, rope, pos, n)
    with pytest.raises(H.InvalidArgument, match="8-bit cache has scales"):
        H.paged_attention(y, (c.k, c.v, None, None), pos, pos)
    with pytest.raises(H.InvalidArgument, match="8-bit cache has scales"):
        H.kv_cache_write(y, y, pos, (y, y, c.k_scale, c.v_scale))
    with pytest.raises(H.InvalidArgument, match="positions must be of the tokens' shape"):
        torch_ops.qk_norm_rope(y, w, w, rope, pos[:3], 2)
    with pytest.raises(H.InvalidArgument, match="must be .*heads, D"):
        torch_ops.qk_norm_rope(x, w, w, rope, pos, 2)
    with pytest.raises(H.InvalidArgument, match="k and v must be alike"):
        torch_ops.kv_cache_write(y, y[:2], pos, c)
