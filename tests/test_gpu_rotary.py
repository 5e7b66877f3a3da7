"""Rotary positions on the GPU against 64 bits: layouts, part of the head, odd
sizes, strides, types, the gradient, and what the call refuses."""
import math

import pytest
import torch

from kv_reference import assert_close, rotate64

from conftest import GAMMA_FP32

pytestmark = pytest.mark.gpu


def _check(x, angles, positions, layout, inverse=False, **kw):
    from rdna2_ops.rotary import rotary
    want, size = rotate64(x, angles, positions, layout, inverse)
    got = rotary(x, angles, positions, layout=layout, inverse=inverse, **kw)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert_close(got, want, GAMMA_FP32 * size, x.dtype)
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot", [
    (1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 64, 32), (37, 24, 128, 64), (7, 3, 80, 80), (5, 2, 96, 32),
    (2, 9, 256, 128), (4, 3, 33, 10), (6, 1, 130, 128), (300, 17, 64, 64), (1, 1, 1024, 1000)])
def test_rotary(dtype, layout, tokens, heads, dim, rot):
    from rdna2_ops.rotary import rope_table
    g = torch.Generator().manual_seed(tokens * 1000 + dim)
    x = torch.randn(tokens, heads, dim, generator=g).mul(20).to(dtype).cuda()
    positions = torch.randint(0, 5000, (tokens,), generator=g).cuda()
    angles = rope_table(5000, rot)
    _check(x, angles, positions, layout)
    _check(x, angles, positions.int(), layout, inverse=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32), (33, 10)])
def test_bit_by_bit_with_elementwise_products_and_sums(dtype, layout, dim, rot):
    """Every product and sum is rounded to fp32 on its own, in any layout."""
    from rdna2_ops.rotary import rope_table, rotary
    g = torch.Generator().manual_seed(dim)
    x = torch.randn(500, 7, dim, generator=g).mul(20).to(dtype).cuda()
    angles, positions = rope_table(3000, rot), torch.randint(0, 3000, (500,), generator=g).cuda()
    row = angles[positions][:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:]
    f = x.float()
    a, b = (f[..., :rot // 2], f[..., rot // 2:rot]) if layout == "half" else (f[..., 0:rot:2], f[..., 1:rot:2])
    for inverse in (False, True):
        s = -sin if inverse else sin
        y, z = a * cos - b * s, b * cos + a * s
        turned = torch.cat([y, z], -1) if layout == "half" else torch.stack([y, z], -1).flatten(-2)
        want = torch.cat([turned, f[..., rot:]], -1).to(dtype)
        assert torch.equal(rotary(x, angles, positions, layout=layout, inverse=inverse), want)


def test_strided_in_place_and_out():
    from rdna2_ops.rotary import rope_table, rotary
    torch.manual_seed(0)
    fused = torch.randn(19, 3 * 8, 64, device="cuda").half()
    angles, positions = rope_table(64, 64), torch.arange(19, device="cuda")
    q = fused[:, 8:16]
    want = _check(q, angles, positions, "half")
    _check(fused[:, ::3], angles, positions, "interleaved")
    _check(fused.transpose(1, 2).contiguous().transpose(1, 2), angles, positions, "half")  # channels not contiguous
    _check(fused.flatten()[1:1 + 18 * 1536].view(18, 24, 64), angles, positions[:18], "half")  # 2-byte aligned
    out = torch.zeros(19, 16, 64, device="cuda", dtype=torch.half)
    assert rotary(q, angles, positions, out=out[:, ::2]).data_ptr() == out.data_ptr()
    assert torch.equal(out[:, ::2], want) and not out[:, 1::2].any()
    k0, v0 = fused[:, :8].clone(), fused[:, 16:].clone()
    rotary(q, angles, positions, out=q)
    assert torch.equal(q, want) and torch.equal(fused[:, :8], k0) and torch.equal(fused[:, 16:], v0)


def test_positions_outside_the_table_are_nan():
    from rdna2_ops.rotary import rope_table, rotary
    x = torch.ones(4, 2, 64, device="cuda")
    got = rotary(x, rope_table(8, 32), torch.tensor([0, 8, -1, 2 ** 40], device="cuda"))
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1:, :, :32]).all() and (got[1:, :, 32:] == 1).all()


def test_empty():
    from rdna2_ops.rotary import rope_table, rotary
    none = torch.empty(0, dtype=torch.long, device="cuda")
    assert rotary(torch.empty(0, 4, 64, device="cuda"), rope_table(4, 64), none).shape == (0, 4, 64)
    assert rotary(torch.empty(2, 0, 64, device="cuda"), rope_table(4, 64), torch.arange(2, device="cuda")).numel() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_inverse_rotation(layout):
    """d/dx of sum(w * rotary(x)) is rotary(w, inverse): against the formula's
    own gradient in 64 bits, and against differences of the kernel (the map is
    linear, so a difference of step h is exact but for fp32 rounding, 2^-22 *
    |values| / h)."""
    from rdna2_ops.rotary import rope_table, rotary
    torch.manual_seed(1)
    x, w = torch.randn(5, 3, 32, device="cuda"), torch.randn(5, 3, 32, device="cuda")
    angles, positions = rope_table(100, 16), torch.randint(0, 100, (5,), device="cuda")
    got = rotary(w, angles, positions, layout=layout, inverse=True)
    x64 = x.cpu().double().requires_grad_()
    row = angles.cpu().double()[positions.cpu()][:, None]
    z = torch.complex(row[..., :8].contiguous(), row[..., 8:].contiguous())
    a, b = (x64[..., :8], x64[..., 8:16]) if layout == "half" else (x64[..., 0:16:2], x64[..., 1:16:2])
    y = torch.complex(a, b) * z
    pairs = torch.cat([y.real, y.imag], -1) if layout == "half" else torch.stack([y.real, y.imag], -1).flatten(-2)
    (torch.cat([pairs, x64[..., 16:]], -1) * w.cpu().double()).sum().backward()
    assert_close(got, x64.grad, GAMMA_FP32 * rotate64(w, angles, positions, layout)[1], torch.float32)
    for t, h, i in ((0, 0, 0), (1, 2, 9), (4, 1, 15), (2, 0, 20)):
        up, down = x.clone(), x.clone()
        up[t, h, i] += 0.5
        down[t, h, i] -= 0.5
        step = (up[t, h, i].double() - down[t, h, i].double()).item()
        slope = ((rotary(up, angles, positions, layout=layout).double()
                  - rotary(down, angles, positions, layout=layout).double()) * w.double()).sum().item() / step
        room = 2.0 ** -22 * (8 * w[t, h].abs().max().item() * x[t, h].abs().max().item() * 4)
        assert abs(slope - got[t, h, i].item()) <= room + 2.0 ** -20


def test_table_scalings():
    """rope_table against its formulas: fp32 of 64-bit cosines (half a unit of
    values up to the gain, 2^-24 * 2, and the 64-bit angle's own error)."""
    from rdna2_ops.rotary import rope_table
    n, rot, base, factor, original = 300, 32, 500.0, 4.0, 64
    pair = torch.arange(rot // 2, dtype=torch.float64)
    plain = base ** (-2 * pair / rot)
    at = torch.arange(n, dtype=torch.float64)[:, None]
    low = max(math.floor(rot * math.log(original / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
    high = min(math.ceil(rot * math.log(original / (2 * math.pi)) / (2 * math.log(base))), rot - 1)
    ramp = ((pair - low) / (high - low)).clamp(0, 1)
    for kw, freq, gain in (
            (dict(), plain, 1.0), (dict(scaling="linear", factor=factor), plain / factor, 1.0),
            (dict(scaling="ntk", factor=factor), (base * factor ** (rot / (rot - 2))) ** (-2 * pair / rot), 1.0),
            (dict(scaling="yarn", factor=factor, original_positions=original),
             plain * (1 - ramp) + plain / factor * ramp, 0.1 * math.log(factor) + 1)):
        got = rope_table(n, rot, base=base, **kw).cpu().double()
        want = torch.cat([torch.cos(at * freq), torch.sin(at * freq)], 1) * gain
        assert (got - want).abs().max() <= 2.0 ** -23, kw


def test_refusals():
    from rdna2_ops.rotary import rope_table, rotary
    x, angles, at = torch.zeros(4, 2, 64, device="cuda"), rope_table(8, 64), torch.arange(4, device="cuda")
    for exc, args, kw in [
            (TypeError, (x.int(), angles, at), {}), (TypeError, (x, angles.half(), at), {}),
            (TypeError, (x, angles, at.float()), {}), (ValueError, (x, angles, at[:3]), {}),
            (ValueError, (x[0], angles, at), {}), (ValueError, (x, angles[:, :63], at), {}),
            (ValueError, (x, angles, at), dict(layout="rows")), (ValueError, (x.cpu(), angles, at), {}),
            (ValueError, (x, angles.cpu(), at), {}), (ValueError, (x, rope_table(8, 66), at), {}),
            (ValueError, (x, angles, at), dict(out=x.half())), (ValueError, (x, angles, at), dict(out=x[:2])),
            (ValueError, (x.clone().requires_grad_(), angles, at), {})]:
        with pytest.raises(exc):
            rotary(*args, **kw)
    for bad in (dict(rotary_dim=3), dict(scaling="log"), dict(factor=0.5), dict(scaling="yarn", factor=2.0)):
        with pytest.raises(ValueError):
            rope_table(**{"positions": 8, "rotary_dim": 64, **bad})
