"""Rotary positions: a table of angles, and the rotation itself.

  rope_table(positions, rotary_dim, ...)        -> angles [positions, rotary_dim] fp32
  rotary(x, angles, positions, ...)             -> x with its first channels rotated

A pair of channels (a, b) at position p turns by t = p * f_i:
(a cos t - b sin t, b cos t + a sin t), products and sums each rounded to fp32
and the result once to x's type.  The map is orthogonal up to the table's own
scaling, so its gradient is the rotation by -t: rotary(grad, ..., inverse=True).
"""
from __future__ import annotations

import math

import torch

from . import _args
from . import _native as nat

LAYOUTS = {"half": 0, "interleaved": 1}


def rope_table(positions, rotary_dim, *, base=10000.0, scaling=None, factor=1.0, original_positions=None,
               beta_fast=32.0, beta_slow=1.0, device="cuda"):
    """cos | sin of every position below `positions`, [positions, rotary_dim] fp32,
    computed in 64 bits.  Channel pair i turns by p * base ** (-2i / rotary_dim).

    For contexts longer than the `original_positions` a model was trained on,
    `factor` times as long, `scaling` is one of

      "linear"  positions divided by `factor`;
      "ntk"     base * factor ** (rotary_dim / (rotary_dim - 2));
      "yarn"    (Peng et al., arXiv 2309.00071) pairs that turn fewer than
                beta_slow times in the original context are interpolated,
                those that turn more than beta_fast times are kept, with a
                ramp between them, and cos and sin are multiplied by
                0.1 ln(factor) + 1.
    """
    _args.require(positions >= 1 and rotary_dim >= 2 and rotary_dim % 2 == 0, ValueError,
                  "rope_table needs at least one position and an even rotary_dim")
    _args.require(scaling in (None, "linear", "ntk", "yarn"), ValueError,
                  "scaling must be None, 'linear', 'ntk' or 'yarn'")
    _args.require(factor >= 1.0, ValueError, "factor must be at least 1")
    gain = 1.0
    if scaling == "ntk":
        _args.require(rotary_dim > 2, ValueError, "'ntk' needs rotary_dim > 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    exponent = torch.arange(0, rotary_dim, 2, device=device, dtype=torch.float64) / rotary_dim
    freq = base ** -exponent
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        _args.require(original_positions is not None and original_positions >= 1, ValueError,
                      "'yarn' needs original_positions")

        def pair_of(turns):
            return rotary_dim * math.log(original_positions / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        pair = torch.arange(rotary_dim // 2, device=device, dtype=torch.float64)
        ramp = ((pair - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        gain = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos() * gain, angle.sin() * gain], 1).float()


def angle_table(angles, dim, device):
    """Checks a table of angles for heads of `dim` channels."""
    if not isinstance(angles, torch.Tensor) or angles.dtype != torch.float32:
        raise TypeError("angles must be an fp32 tensor")
    shape = angles.shape
    if len(shape) != 2 or shape[0] < 1 or not angles.is_contiguous() or angles.device != device:
        raise ValueError(f"angles must be contiguous [positions, rotary_dim] on {device}")
    if shape[1] < 2 or shape[1] % 2 or shape[1] > dim:
        raise ValueError(f"rotary_dim must be even and at most {dim}, got {shape[1]}")


def rotary(x, angles, positions, *, layout="half", inverse=False, out=None):
    """x [tokens, heads, dim] (fp32, fp16 or bf16, any strides) rotated by
    angles[positions] in its first angles.shape[1] channels.

    layout "half" pairs channel i with channel i + rotary_dim / 2,
    "interleaved" pairs neighbours.  positions: int32 or int64 [tokens]; one
    outside the table makes NaN.  inverse rotates back (the gradient).  out
    may be x itself."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _args.FLOAT_DTYPES:
        raise TypeError("x must be an fp32, fp16 or bf16 tensor")
    if layout not in LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved'")
    if x.ndim != 3:
        raise ValueError(f"x must be [tokens, heads, dim], got {tuple(x.shape)}")
    dev = nat.require_device(x, positions)
    nat.eager_only(x)
    tokens, heads, dim = x.shape
    angle_table(angles, dim, dev)
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError("positions must be int32 or int64")
    if positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError(f"positions must be contiguous [{tokens}], got {tuple(positions.shape)}")
    if out is None:
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
    elif out.shape != x.shape or out.dtype != x.dtype or out.device != dev or out.stride(2) != 1:
        raise ValueError("out must have x's shape, type and device, and contiguous channels")
    if x.stride(2) != 1:
        x = x.contiguous()
    nat.launch(
        dev, "b2_rotary", x.data_ptr(), nat.DTYPE_CODE[x.dtype], tokens, heads, dim, x.stride(0), x.stride(1),
        angles.data_ptr(), angles.shape[0], angles.shape[1], LAYOUTS[layout], int(inverse), positions.data_ptr(),
        int(positions.dtype == torch.int64), out.data_ptr(), out.stride(0), out.stride(1))
    return out
