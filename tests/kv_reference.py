"""64-bit restatements of the cached-attention operators, for the tests: written
row by row from the formulas, on the CPU, with the bounds that the kernels'
32-bit arithmetic is held to."""
import math

import torch

from conftest import GAMMA_FP32, ulp_of

KIND = {torch.float32: "fp32", torch.float16: "fp16", torch.bfloat16: "bf16"}
TOP = {"int8": 127.0, "e4m3": 448.0}
FLOOR = 2.0 ** -100


def rotate64(x, angles, positions, layout, inverse=False):
    """(rotated [T, H, D] in 64 bits, sum of the products' magnitudes)."""
    x = x.cpu().double()
    out, size = x.clone(), x.abs()
    rot = angles.shape[1]
    row = angles.cpu().double()[positions.cpu().long()][:, None]
    cos, sin = row[..., :rot // 2], row[..., rot // 2:] * (-1 if inverse else 1)
    ia = torch.arange(rot // 2) if layout == "half" else torch.arange(0, rot, 2)
    ib = ia + (rot // 2 if layout == "half" else 1)
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * cos - b * sin, b * cos + a * sin
    size[..., ia] = (a * cos).abs() + (b * sin).abs()
    size[..., ib] = (b * cos).abs() + (a * sin).abs()
    return out, size


def places(lengths, offsets, tokens):
    """[(sequence, position)] of every token of the call."""
    lengths = lengths.tolist()
    if offsets is None:
        each = tokens // len(lengths) if lengths else 0
        offsets = [each * b for b in range(len(lengths) + 1)]
    else:
        offsets = offsets.tolist()
    got = []
    for b in range(len(lengths)):
        n = offsets[b + 1] - offsets[b]
        got += [(b, lengths[b] - n + i) for i in range(n)]
    return got


def code_step(value, code):
    """Distance between the codes around `value` (in units of the scale)."""
    if code == "int8":
        return torch.ones_like(value)
    power = torch.floor(torch.log2(value.abs().clamp_min(2.0 ** -12))).clamp(-6, 8)
    return torch.exp2(power - 3)


def check_append(before, after, x, size, where, table, code):
    """Codes and scales after an append of x [T, H, D] (64 bits; `size` bounds
    the magnitudes its rounding errors go with) at the places `where`.
    before, after: (codes, scales) on the CPU, codes as float64 numbers.

    Bounds: a 32-bit scale is within 2 roundings of the 64-bit one beside x's
    own error; code = RNE(x * fp32(1/s)) is within half a step of x / s plus
    the roundings of x, of 1/s, of the product and of s, 2^-20 * |x| / s
    together."""
    (codes0, scale0), (codes1, scale1) = before, after
    page = codes0.shape[2]
    blocks = {}
    for i, (b, pos) in enumerate(where):
        if pos < 0 or pos // page >= table.shape[1]:
            continue
        pid = int(table[b, pos // page])
        if 0 <= pid < codes0.shape[0]:
            blocks.setdefault((pid, b, pos // page), []).append((pos % page, i))
    untouched = set(range(codes0.shape[0])) - {k[0] for k in blocks}
    for pid in untouched:
        assert torch.equal(codes0[pid], codes1[pid]) and torch.equal(scale0[pid], scale1[pid]), pid
    for (pid, b, _), rows in blocks.items():
        slots = [s for s, _ in rows]
        new, room = x[[i for _, i in rows]], size[[i for _, i in rows]]  # [n, H, D]
        first = min(slots)
        s = (new.abs().amax((0, 2)) / TOP[code]).clamp_min(FLOOR)
        if first > 0:
            s = torch.maximum(s, scale0[pid])
        got = scale1[pid]
        slack = GAMMA_FP32 * (room.amax((0, 2)) / TOP[code] + s)
        assert ((got - s).abs() <= slack).all(), (pid, got, s)
        for slot in range(page):
            c1 = codes1[pid, :, slot]
            if slot in slots:
                want = new[slots.index(slot)] / got[:, None]
                slack = room[slots.index(slot)] / got[:, None]
            elif slot < first:
                want = codes0[pid, :, slot] * (scale0[pid] / got)[:, None]
                slack = want.abs()
            else:
                assert torch.equal(c1, codes0[pid, :, slot]), (pid, slot)
                continue
            want = want.clamp(-TOP[code], TOP[code])
            step = torch.maximum(code_step(want, code), code_step(c1, code))
            assert ((c1 - want).abs() <= 0.5 * step + GAMMA_FP32 * slack).all(), (pid, slot, b)


def attend64(q, cache, lengths, table, offsets, causal, window, scale=None):
    """(out, lse, bound of out, bound of lse) in 64 bits.  cache: (k, v,
    v_scale) values [P, H, page, D] and scales [P, H] on the CPU.

    With w_j = softmax, e = the error of a score: scores are sums of exact
    products in fp32, e <= 2^-20 * sum|q k| * scale, plus the exponential's and
    the logarithm's own 2^-21 relative or absolute.  The weights that multiply
    the codes are fp16, relative to the largest w_j vs_j: each is off by 2^-11
    of itself or by 2^-25 of that largest one, and codes are at most TOP."""
    k, v, v_scale = cache
    tokens, heads, dim = q.shape
    group = heads // k.shape[1]
    page = k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    q = q.cpu().double()
    out, lse = torch.zeros_like(q), torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    out_tol, lse_tol = torch.zeros_like(q), torch.zeros(tokens, heads, dtype=torch.float64)
    top = 127.0 * 256.0  # the largest code of either kind is below it
    for i, (b, pos) in enumerate(places(lengths, offsets, tokens)):
        length = int(lengths[b])
        hi = min(length, table.shape[1] * page)
        hi = min(hi, pos + 1) if causal else hi
        lo = max(0, pos - window + 1) if window else 0
        at = torch.arange(lo, max(lo, hi))
        pid = table[b, at // page].long()
        at, pid = at[(pid >= 0) & (pid < k.shape[0])], pid[(pid >= 0) & (pid < k.shape[0])]
        if not len(at):
            continue
        kk, vv = k[pid, :, at % page], v[pid, :, at % page]  # [n, H, D]
        vs = v_scale[pid]
        for h in range(heads):
            s = kk[:, h // group] @ q[i, h] * scale
            e = GAMMA_FP32 * (kk[:, h // group].abs() @ q[i, h].abs()).max() * scale + 2.0 ** -20
            lse[i, h] = torch.logsumexp(s, 0)
            w = torch.exp(s - lse[i, h])
            out[i, h] = w @ vv[:, h // group]
            largest = (w * vs[:, h // group]).max()
            out_tol[i, h] = (2.0 ** -11 + 4 * e) * (w @ vv[:, h // group].abs()) + len(at) * 2.0 ** -25 * top * largest
            lse_tol[i, h] = 2 * e + 2.0 ** -22 * lse[i, h].abs()
    return out, lse, out_tol, lse_tol


def assert_close(got, want, tol, dtype, what=""):
    """|got - want| <= half a unit in the last place of either + tol; the same
    infinities and NaN."""
    got, want = got.cpu().double(), want
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), what
    got, want, tol = got[~odd], want[~odd], tol[~odd]
    ulp = torch.from_numpy(ulp_of(torch.maximum(got.abs(), want.abs()).numpy(), KIND[dtype]))
    off = (got - want).abs() - (0.5 * ulp + tol)
    assert (off <= 0).all(), f"{what}: off by up to {off.max().item():.3g} more than allowed"
