"""bf16 results near the type's largest from the RMS norm, its gradients, the 8-bit rows and the output projection: bit patterns that, read as fp16, are
signalling NaNs (bf16 values of 2^121 to 2^125) come out as the numbers that they are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def patterns(least):
    """Every finite bf16 value of a magnitude of `least` or more, both signs, 8 of a kind (sign and exponent) at a time."""
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    x = bits.view(torch.bfloat16)
    return x[x.isfinite() & (x.abs().float() >= least)]


@pytest.mark.parametrize("c", (5, 8, 240, 1001, 4096, 16384, 20000))
def test_sums(hip, c):
    x = patterns(0.0)
    x = x.repeat(-(-2 * c // len(x)) + 1)
    x = x[:len(x) // c * c].view(-1, c).cuda()
    _, s, _ = hip.rms_norm(x, torch.ones(c, device="cuda"), torch.full_like(x, -0.0))
    assert torch.equal(s.view(torch.int16), x.view(torch.int16))


@pytest.mark.parametrize("c", (5, 8, 240, 1001, 4096, 16384, 20000))
def test_products(hip, c):
    """Rows of +-1 have r = 1, to the rounding of a division and a square root: results are the weights."""
    w = patterns(2.0 ** 100)
    for first in range(0, len(w), c):
        part = w[first:first + c].float()
        part = torch.nn.functional.pad(part, (0, c - len(part)), value=1.0).cuda()
        x = torch.where(torch.arange(3 * c, device="cuda").view(3, c) % 2 == 0, 1.0, -1.0).to(torch.bfloat16)
        out, _, _ = hip.rms_norm(x, part, eps=0.0)
        want = x.double() * part.double()
        # half a step and fp32's own roundings; the largest may round past the type, as any value that is a step off would
        assert ((out.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -20) * want.abs()).all()


@pytest.mark.parametrize("c", (8, 240, 1000, 4096, 16384, 20000))
def test_gradients(hip, c):
    """Equal gradients of values +1 and -1 side by side: the mean over the row is 0, and ds = dy."""
    dy = patterns(2.0 ** 100)
    dy = dy[dy.abs().float() < 2.0 ** 126].repeat_interleave(2)
    dy = torch.nn.functional.pad(dy.float(), (0, -len(dy) % c), value=1.0).to(torch.bfloat16).view(-1, c).cuda()
    s = torch.where(torch.arange(dy.numel(), device="cuda").view(dy.shape) % 2 == 0, 1.0, -1.0).to(torch.bfloat16)
    ds, _ = hip.rms_norm_bwd(s, torch.ones(c, device="cuda"), torch.ones(len(s), device="cuda"), dy)
    assert ((ds.double() - dy.double()).abs() <= 2.0 ** -8 * dy.double().abs()).all()


@pytest.mark.parametrize("k", (5, 64, 255, 2048))
def test_rows_back(hip, k):
    q = (torch.arange(4 * hip.padded_k(k)) % 255 - 127).to(torch.int8).view(4, -1)
    scale = 2.0 ** torch.tensor([114.0, 116.0, 118.0, 120.0])
    out = hip.dequantize_rows(q.cuda(), scale.cuda(), k, torch.bfloat16)
    assert torch.equal(out.double().cpu(), q[:, :k].double() * scale[:, None].double())


@pytest.mark.parametrize("n", (64, 128))
@pytest.mark.parametrize("k", (64, 128))
def test_output_projection_keeps_its_residual(hip, k, n):
    x = patterns(0.0)
    x = x[x.abs().float() >= 2.0 ** -126]  # (sums of subnormal values may round to zero)
    x = torch.nn.functional.pad(x.float(), (0, -len(x) % n), value=1.0).to(torch.bfloat16).view(-1, n).cuda()
    o = torch.zeros(len(x), k, dtype=torch.bfloat16, device="cuda")
    w, b = torch.ones(n, k, dtype=torch.float16, device="cuda"), torch.zeros(n, dtype=torch.float16, device="cuda")
    assert torch.equal(hip.output_projection(o, w, b, x), x)
