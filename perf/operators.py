"""Timed cases of the cached-attention operators: rotary positions, the append
to a paged 8-bit key/value cache, and attention over that cache.

`listed()` names the cases, `draw(rng)` makes more of the same ranges,
`prepare(case, seed)` builds what a serving program holds before the call,
`run(state)` makes one pass, `work(case)` counts the bytes and operations the
pass cannot do without and `exact(case, seed)` gives its results in 64 bits.
With `own` false, run() computes in elementary 32-bit torch operations; with
`own` true it calls this repository's operators.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
SCALE_FLOOR = 2.0 ** -100  # the scale of a block that holds only zeros


def _ops():
    root = str(Path(__file__).resolve().parents[1] / "rdna2-gfx1030-ai-handbook_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from rdna2_ops import kv_cache, rotary
    return rotary, kv_cache


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one generated token's queries, rotated on their own: launch latency
        dict(name="rotary_token", op="rotary", tokens=1, heads=32, head_dim=128, rotary_dim=128, layout="half",
             dtype="bf16", fused=False, inverse=False),
        # the gradient of a partial, interleaved rotation: an odd number of
        # tokens, read in place out of a fused projection's rows
        dict(name="rotary_partial_grad", op="rotary", tokens=4061, heads=40, head_dim=128, rotary_dim=64,
             layout="interleaved", dtype="fp16", fused=True, inverse=True),
        # the queries of a long prompt: memory bandwidth
        dict(name="rotary_prompt", op="rotary", tokens=65536, heads=32, head_dim=128, rotary_dim=128, layout="half",
             dtype="bf16", fused=False, inverse=False),
        # one token joins one sequence's cache, its queries rotated on the way
        dict(name="append_token", op="append", batch=1, new=1, length=1001, mix=0, q_heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, page=64, code="int8", dtype="bf16", layout="half"),
        # a generation step of a full batch: one token each, every page at
        # another fill, some blocks requantized
        dict(name="append_step", op="append", batch=128, new=1, length=4096, mix=3, q_heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, page=16, code="e4m3", dtype="fp16", layout="half"),
        # ragged prompts behind earlier turns, every query head with its own keys
        dict(name="append_prompts", op="append", batch=7, new=2048, length=5000, mix=5, q_heads=40, kv_heads=40,
             head_dim=128, rotary_dim=64, page=64, code="int8", dtype="bf16", layout="interleaved"),
        # a whole long document in one call
        dict(name="append_document", op="append", batch=1, new=65536, length=65536, mix=0, q_heads=32, kv_heads=8,
             head_dim=128, rotary_dim=128, page=128, code="e4m3", dtype="bf16", layout="half"),
        # one token over a short history: launch latency
        dict(name="attend_token", op="attend", batch=1, new=1, length=300, mix=0, q_heads=32, kv_heads=8,
             head_dim=128, page=64, code="int8", dtype="bf16", window=0, causal=True),
        # a generation step of a batch with histories of every length
        dict(name="attend_step", op="attend", batch=64, new=1, length=8192, mix=7, q_heads=64, kv_heads=8,
             head_dim=128, page=64, code="int8", dtype="bf16", window=0, causal=True),
        # one token over one very long history: the history has to be split
        dict(name="attend_long", op="attend", batch=1, new=1, length=262131, mix=0, q_heads=32, kv_heads=8,
             head_dim=128, page=128, code="e4m3", dtype="fp16", window=0, causal=True),
        # chunks of ragged prompts over long histories behind a sliding window,
        # small heads and small pages
        dict(name="attend_chunks", op="attend", batch=4, new=512, length=16384, mix=11, q_heads=32, kv_heads=4,
             head_dim=64, page=16, code="e4m3", dtype="fp16", window=4096, causal=True),
        # a whole prompt at once, causal: the tensor cores
        dict(name="attend_prompt", op="attend", batch=1, new=8192, length=8192, mix=0, q_heads=32, kv_heads=8,
             head_dim=128, page=128, code="int8", dtype="bf16", window=0, causal=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attend step", "attend step", "attend chunk", "attend chunk"])
    dim = rng.choice([64, 128])
    code, dtype = rng.choice(["int8", "e4m3"]), rng.choice(["fp16", "bf16"])
    layout, page = rng.choice(["half", "interleaved"]), rng.choice([16, 32, 64, 128])
    rotary_dim = rng.choice([dim, dim, dim // 2])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if kind == "rotary":
        heads = rng.choice([1, 8, 24, 32, 40])
        return dict(op="rotary", tokens=_log_int(rng, 1, 65536 * 32 * 128 // (heads * dim * 2)), heads=heads,
                    head_dim=dim, rotary_dim=rotary_dim, layout=layout, dtype=rng.choice(["fp32", "fp16", "bf16"]),
                    fused=rng.random() < 0.5, inverse=rng.random() < 0.5)
    if kind == "append":
        batch = _log_int(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(4, 32768 // batch))
        return dict(op="append", batch=batch, new=new, length=new + _log_int(rng, 1, 4096), mix=rng.randrange(1, 1000),
                    q_heads=q_heads, kv_heads=kv_heads, head_dim=dim, rotary_dim=rotary_dim, page=page, code=code,
                    dtype=dtype, layout=layout)
    window = rng.choice([0, 0, _log_int(rng, 16, 8192)])
    if kind == "attend step":
        batch = _log_int(rng, 1, 128)
        new = rng.choice([1, 1, 1, 2, 5])
        most = max(64, 262144 * 8 // (batch * max(kv_heads, q_heads // 4)))
        length = new + _log_int(rng, 16, min(131072, most))
        causal = rng.random() < 0.8
        return dict(op="attend", batch=batch, new=new, length=length, mix=rng.randrange(1, 1000), q_heads=q_heads,
                    kv_heads=kv_heads, head_dim=dim, page=page, code=code, dtype=dtype, window=window, causal=causal)
    batch = rng.randrange(1, 5)
    new = _log_int(rng, 9, 2048)
    most = 8192 * 8192 * 32 // (batch * new * q_heads)
    length = new + _log_int(rng, 16, max(17, min(most // 2, 32768)))
    return dict(op="attend", batch=batch, new=new, length=length, mix=rng.randrange(1, 1000), q_heads=q_heads,
                kv_heads=kv_heads, head_dim=dim, page=page, code=code, dtype=dtype, window=window,
                causal=rng.random() < 0.8)


def _sequences(case):
    """[(new tokens, tokens cached once they are in)] of each sequence; mix 0:
    all alike, else ragged, the first one the longest and, among four or more
    with more than one new token, the last one absent from this call."""
    if not case["mix"]:
        return [(case["new"], case["length"])] * case["batch"]
    rng = random.Random(case["mix"])
    got = [(case["new"], case["length"])]
    for _ in range(case["batch"] - 1):
        new = rng.randint(max(1, case["new"] // 4), case["new"])
        got.append((new, new + int((case["length"] - case["new"]) * rng.random())))
    if case["batch"] >= 4 and case["new"] > 1:
        got[-1] = (0, 0)
    return got


# ------------------------------------------------------------------ the inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _angles(rotary_dim, positions):
    """cos | sin of every position, [positions, rotary_dim] in 32 bits."""
    inv = 10000.0 ** (-torch.arange(0, rotary_dim, 2, device="cuda", dtype=torch.float64) / rotary_dim)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def _outliers(gen, heads, dim):
    """One channel in a hundred, at least one in all, is twenty times as large."""
    gain = torch.ones(heads * dim, device="cuda")
    at = torch.randperm(heads * dim, generator=gen, device="cuda")[: max(1, heads * dim // 100)]
    gain[at] = 20.0
    return gain.view(heads, dim)


def _cache(gen, case, pages):
    """Codes [pages, kv_heads, page, head_dim] and scales [pages, kv_heads] of earlier tokens."""
    heads, dim, page, code = case["kv_heads"], case["head_dim"], case["page"], case["code"]
    x = _normal(gen, pages, heads, page, dim)
    scale = (x.abs().amax((2, 3)) / CODE_MAX[code]).clamp_min(SCALE_FLOOR)
    x = (x / scale[:, :, None, None]).clamp_(-CODE_MAX[code], CODE_MAX[code])
    x = x.round_().to(torch.int8) if code == "int8" else x.to(CODES[code])
    # blocks of differing loudness
    scale = scale * torch.exp(0.5 * _normal(gen, pages, heads))
    return x, scale


def _paging(gen, case):
    """Lengths, offsets of the new tokens and block table: pages scattered
    over a pool with some left over, -1 where a sequence has none."""
    seqs, page = _sequences(case), case["page"]
    lengths = torch.tensor([s[1] for s in seqs], dtype=torch.int32)
    counts = torch.tensor([s[0] for s in seqs], dtype=torch.int32)
    cu = torch.cat([torch.zeros(1, dtype=torch.int32), counts.cumsum(0).int()])
    need = (lengths + page - 1) // page
    width = max(1, int(need.max()))
    total = int(need.sum())
    pool = total + 3
    table = torch.full((len(seqs), width), -1, dtype=torch.int32)
    table[torch.arange(width)[None] < need[:, None]] = torch.arange(total, dtype=torch.int32)
    order = torch.randperm(pool, generator=gen, device="cuda").int()
    table = table.cuda()
    table = torch.where(table >= 0, order[table.clamp_min(0).long()], table)
    return lengths.cuda(), cu.cuda(), table, pool


def prepare(case, seed):
    gen = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    heads, dim = case.get("q_heads", case.get("heads")), case["head_dim"]
    if case["op"] == "rotary":
        row = heads * 3 if case["fused"] else heads  # queries, keys and values side by side
        x = (_normal(gen, case["tokens"], row, dim) * _outliers(gen, row, dim)).to(dtype)[:, :heads]
        top = max(4096, case["tokens"])
        positions = torch.arange(case["tokens"], device="cuda") + int(torch.randint(
            0, top - case["tokens"] + 1, (1,), generator=gen, device="cuda"))
        return dict(case=case, x=x, positions=positions, angles=_angles(case["rotary_dim"], top))
    lengths, cu, table, pool = _paging(gen, case)
    tokens = sum(s[0] for s in _sequences(case))
    k_codes, k_scale = _cache(gen, case, pool)
    v_codes, v_scale = _cache(gen, case, pool)
    q = (_normal(gen, tokens, heads, dim) * _outliers(gen, heads, dim)).to(dtype)
    state = dict(case=case, q=q, lengths=lengths, offsets=cu if case["new"] > 1 else None, table=table,
                 most=case["new"], k_codes=k_codes, k_scale=k_scale, v_codes=v_codes, v_scale=v_scale)
    if case["op"] == "append":
        kv = case["kv_heads"]
        state["k"] = (_normal(gen, tokens, kv, dim) * _outliers(gen, kv, dim)).to(dtype)
        state["v"] = _normal(gen, tokens, kv, dim).to(dtype)
        state["angles"] = _angles(case["rotary_dim"], case["length"])
        # the pages that the new tokens fall on; what no token holds yet is zero
        seq, position = _places(state)
        state["pages"] = table[seq, position // case["page"]].unique()
        held = torch.zeros(pool, case["page"], dtype=torch.bool, device="cuda")
        at = torch.arange(table.shape[1] * case["page"], device="cuda")
        start = lengths - (cu[1:] - cu[:-1])
        live = (at[None] < start[:, None]) & (table.repeat_interleave(case["page"], 1) >= 0)
        held[table.repeat_interleave(case["page"], 1)[live].long(), at.expand_as(live)[live] % case["page"]] = True
        for name in ("k_codes", "v_codes"):
            bits = state[name].view(torch.uint8)
            bits *= held[:, None, :, None].to(torch.uint8)
    if own:
        state["cache"] = _ops()[1].PagedKVCache.wrap(k_codes, v_codes, k_scale, v_scale)
    return state


# ---------------------------------------------------------- one pass, plain form
def _values(state, name, pages):
    """The 32-bit values of the keys ("k") or values ("v") on `pages`."""
    codes, scale = state[name + "_codes"], state[name + "_scale"]
    return codes.view(torch.uint8)[pages].view(codes.dtype).float() * scale[pages][..., None, None]


def _places(state):
    """Each new token's sequence and position."""
    lengths, cu, tokens = state["lengths"].long(), state["offsets"], state["q"].shape[0]
    if cu is None:
        per = tokens // lengths.shape[0]
        seq = torch.arange(tokens, device="cuda") // per
        return seq, lengths[seq] - per + torch.arange(tokens, device="cuda") % per
    cu = cu.long()
    seq = torch.repeat_interleave(cu[1:] - cu[:-1], output_size=tokens)
    return seq, lengths[seq] - cu[seq + 1] + torch.arange(tokens, device="cuda")


def _rotated(x, angles, positions, layout, inverse=False):
    """x [tokens, heads, dim] in 32 bits with its first channels rotated."""
    x = x.float()
    half = angles.shape[1] // 2
    row = angles[positions][:, None]
    cos, sin = row[..., :half], row[..., half:]
    sin = -sin if inverse else sin
    turned, rest = x[..., : 2 * half], x[..., 2 * half:]
    if layout == "half":
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, rest], -1)


def _plain_append_one(x, codes, scale, page_of, slot, pages, old, code):
    """Joins x [tokens, heads, dim] to the blocks `page_of`, whose scales grow
    to hold it; earlier codes of a block are requantized to its new scale."""
    top = CODE_MAX[code]
    cast = (lambda v: v.round().clamp(-top, top).to(torch.int8)) if code == "int8" else (
        lambda v: v.clamp(-top, top).to(CODES[code]))
    amax = torch.zeros_like(scale).index_reduce_(0, page_of, x.abs().amax(-1), "amax")
    was = torch.where(old[:, None], scale, torch.zeros_like(scale))
    now = torch.maximum(was, (amax / torch.full_like(amax, top)).clamp_min(SCALE_FLOOR))[pages]
    bits = codes.view(torch.uint8)
    earlier = bits[pages].view(codes.dtype).float()
    bits[pages] = cast(earlier * (was[pages] / now)[:, :, None, None]).view(torch.uint8)
    scale[pages] = now
    bits[page_of, :, slot] = cast(x * (1.0 / scale[page_of])[:, :, None]).view(torch.uint8)


def _plain_append(state):
    case = state["case"]
    seq, position = _places(state)
    page_of = state["table"][seq, position // case["page"]].long()
    slot = position % case["page"]
    pages = state["pages"].long()
    # blocks that begin before the first new token
    start = state["lengths"].long() - torch.zeros_like(state["lengths"], dtype=torch.long).index_add_(
        0, seq, torch.ones_like(seq))
    first = torch.zeros(state["k_scale"].shape[0], dtype=torch.bool, device="cuda")
    old = first.index_put((page_of,), (position // case["page"] * case["page"] < start[seq]))
    keys = _rotated(state["k"], state["angles"], position, case["layout"])
    _plain_append_one(keys, state["k_codes"], state["k_scale"], page_of, slot, pages, old, case["code"])
    _plain_append_one(state["v"].float(), state["v_codes"], state["v_scale"], page_of, slot, pages, old, case["code"])
    q = _rotated(state["q"], state["angles"], position, case["layout"]).to(state["q"].dtype)
    k, v = (_values(state, name, pages).to(q.dtype) for name in "kv")
    return q, k, v, state["k_scale"][pages], state["v_scale"][pages]


def _plain_attend(state):
    case = state["case"]
    heads, kv, dim = case["q_heads"], case["kv_heads"], case["head_dim"]
    table = state["table"].clamp_min(0).long()
    batch, length, most = table.shape[0], table.shape[1] * case["page"], state["most"]
    keys, values = (_values(state, name, table).transpose(1, 2).reshape(batch, kv, length, dim) for name in "kv")
    seq, position = _places(state)
    lengths = state["lengths"].long()
    counts = torch.zeros_like(lengths).index_add_(0, seq, torch.ones_like(seq))
    index = position - (lengths - counts)[seq]
    q = torch.zeros(batch, most, heads, dim, device="cuda")
    q[seq, index] = state["q"].float()
    q = q.view(batch, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(batch, kv, -1, dim)
    logits = (q @ keys.transpose(-1, -2) * dim ** -0.5).view(batch, kv, -1, most, length)
    at = torch.arange(length, device="cuda")
    mine = (lengths - counts)[:, None, None] + torch.arange(most, device="cuda")[:, None]
    seen = at < lengths[:, None, None]
    seen = seen & (at <= mine) if case["causal"] else seen.expand(-1, most, -1)
    if case["window"]:
        seen = seen & (at > mine - case["window"])
    logits = logits.masked_fill(~seen[:, None, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    out = p.view(batch, kv, -1, length) @ values
    out = out.view(batch, kv, -1, most, dim) / total.clamp_min(1e-30)
    lse = (total.log() + top)[..., 0]
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)[seq, index]
    lse = lse.permute(0, 3, 1, 2).reshape(batch, most, heads)[seq, index]
    return out.to(state["q"].dtype), lse


def run(state):
    case = state["case"]
    if own:
        rotary, _ = _ops()
        if case["op"] == "rotary":
            return rotary.rotary(state["x"], state["angles"], state["positions"], layout=case["layout"],
                                 inverse=case["inverse"])
        cache = state["cache"]
        if case["op"] == "append":
            q = cache.append(state["k"], state["v"], state["lengths"], state["table"], offsets=state["offsets"],
                             q=state["q"], angles=state["angles"], layout=case["layout"])
            k, v, k_scale, v_scale = cache.read(state["pages"], dtype=q.dtype, return_scales=True)
            return q, k, v, k_scale, v_scale
        return cache.attend(state["q"], state["lengths"], state["table"], offsets=state["offsets"],
                            max_new=state["most"], causal=case["causal"], window=case["window"] or None,
                            return_lse=True)
    if case["op"] == "rotary":
        x = state["x"]
        return _rotated(x, state["angles"], state["positions"], case["layout"], case["inverse"]).to(x.dtype)
    return _plain_append(state) if case["op"] == "append" else _plain_attend(state)


# ---------------------------------------------------------------- what it needs
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    dim = case["head_dim"]
    if case["op"] == "rotary":
        values = case["tokens"] * case["heads"] * dim
        return {"bytes": 2 * size * values + case["tokens"] * (8 + 4 * case["rotary_dim"]),
                "flops": 3 * case["tokens"] * case["heads"] * case["rotary_dim"]}
    seqs, page, kv, heads = _sequences(case), case["page"], case["kv_heads"], case["q_heads"]
    tokens = sum(n for n, _ in seqs)
    if case["op"] == "append":
        blocks = sum((have - 1) // page - (have - n) // page + 1 for n, have in seqs if n)
        read = tokens * (heads + 2 * kv) * dim * size + tokens * case["rotary_dim"] * 4
        wrote = tokens * heads * dim * size + tokens * 2 * kv * dim + blocks * 2 * kv * 4
        back = blocks * 2 * kv * page * dim * (1 + size) + blocks * 2 * kv * 8
        return {"bytes": read + wrote + back,
                "flops": tokens * (3 * (heads + kv) * case["rotary_dim"] + 4 * kv * dim)}
    pairs = touched = 0
    for n, have in seqs:
        first = have - n
        begin = max(0, first - case["window"] + 1) if case["window"] else 0
        touched += max(0, have - begin) if n else 0
        if case["causal"] and not case["window"]:
            pairs += n * first + n * (n + 1) // 2
        elif case["causal"]:
            full = max(0, min(n, case["window"] - first))  # rows whose window reaches the beginning
            pairs += full * first + full * (full + 1) // 2 + (n - full) * case["window"]
        elif case["window"]:
            pairs += sum(have - max(0, first + i - case["window"] + 1) for i in range(n))
        else:
            pairs += n * have
    blocks = touched / page
    return {"bytes": int(2 * tokens * heads * dim * size + tokens * heads * 4 + 2 * touched * kv * dim
                         + 2 * blocks * kv * 4),
            "flops": 4 * pairs * heads * dim}


# --------------------------------------------------------- the results in 64 bits
def _turn64(x, angles, positions, layout, sign=1.0):
    """The rotation as a product of complex numbers."""
    half = angles.shape[1] // 2
    row = angles[positions].double()[:, None]
    z = torch.complex(row[..., :half].contiguous(), sign * row[..., half:].contiguous())
    out = x.double().clone()
    if layout == "half":
        w = torch.complex(out[..., :half].contiguous(), out[..., half: 2 * half].contiguous()) * z
        out[..., :half], out[..., half: 2 * half] = w.real, w.imag
    else:
        w = torch.complex(out[..., 0: 2 * half: 2].contiguous(), out[..., 1: 2 * half: 2].contiguous()) * z
        out[..., 0: 2 * half: 2], out[..., 1: 2 * half: 2] = w.real, w.imag
    return out


def _grid64(x, code):
    """x at the nearest value that the code has (ties to even)."""
    if code == "int8":
        return torch.round(x).clamp(-127, 127)
    power = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp(-6, 8)
    step = torch.exp2(power - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _append64(state):
    case, page = state["case"], state["case"]["page"]
    cu = state["offsets"].tolist() if state["offsets"] is not None else list(range(case["batch"] + 1))
    lengths = state["lengths"].tolist()
    positions = torch.cat([torch.arange(lengths[b] - (cu[b + 1] - cu[b]), lengths[b]) for b in range(case["batch"])])
    positions = positions.cuda()
    keys = _turn64(state["k"], state["angles"], positions, case["layout"])
    where = {p: i for i, p in enumerate(state["pages"].tolist())}
    table = state["table"].tolist()
    got = []
    for x, codes, scale in ((keys, state["k_codes"], state["k_scale"]),
                            (state["v"].double(), state["v_codes"], state["v_scale"])):
        scales = scale[state["pages"].long()].double()
        values = codes.view(torch.uint8)[state["pages"].long()].view(codes.dtype).double() * scales[:, :, None, None]
        parts, rows, spans = [], [], []
        for b in range(case["batch"]):
            at = lengths[b] - (cu[b + 1] - cu[b])
            while at < lengths[b]:
                end = min(lengths[b], at - at % page + page)
                token = cu[b] + at - (lengths[b] - (cu[b + 1] - cu[b]))
                rows.append(where[table[b][at // page]])
                spans.append((token, end - at, at % page))
                at = end
        sizes = torch.tensor([s[1] for s in spans], device="cuda")
        firsts = torch.tensor([s[2] for s in spans], device="cuda")
        peak = torch.segment_reduce(x.abs().amax(-1), "max", lengths=sizes)
        row = torch.tensor(rows, device="cuda")
        now = (peak / CODE_MAX[case["code"]]).clamp_min(SCALE_FLOOR)
        was = torch.where((firsts > 0)[:, None], scales[row], torch.zeros_like(now))
        now = torch.maximum(now, was)
        slots = torch.arange(page, device="cuda")
        for c in range(0, len(rows), 256):
            r, n, f = row[c: c + 256], sizes[c: c + 256], firsts[c: c + 256]
            fill = slots[None] - f[:, None]
            is_new = (fill >= 0) & (fill < n[:, None])
            base = torch.tensor([s[0] for s in spans[c: c + 256]], device="cuda")
            source = (base[:, None] + fill).clamp(0, x.shape[0] - 1)
            new = x[source].transpose(1, 2)
            both = torch.where(is_new[:, None, :, None], new, values[r])
            s = now[c: c + 256][:, :, None, None]
            parts.append(_grid64(both / s, case["code"]) * s)
        out = torch.empty_like(values)
        out[row] = torch.cat(parts)
        scales[row] = now
        got.append((out, scales))
    q = _turn64(state["q"], state["angles"], positions, case["layout"])
    return q, got[0][0], got[1][0], got[0][1], got[1][1]


def _attend64(state):
    case, page = state["case"], state["case"]["page"]
    heads, group = case["q_heads"], case["q_heads"] // case["kv_heads"]
    q = state["q"].double()
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    cu = state["offsets"].tolist() if state["offsets"] is not None else list(range(case["batch"] + 1))
    for b, have in enumerate(state["lengths"].tolist()):
        n = cu[b + 1] - cu[b]
        if not n or not have:
            continue
        own_pages = state["table"][b, : (have + page - 1) // page].long()
        mine = torch.arange(have - n, have, device="cuda")[:, None]
        at = torch.arange(have, device="cuda")
        hidden = torch.zeros(n, have, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= at > mine
        if case["window"]:
            hidden |= at <= mine - case["window"]
        for h in range(heads):
            k, v = ((codes.view(torch.uint8)[own_pages, h // group].view(codes.dtype).double()
                     * scale[own_pages, h // group].double()[:, None, None]).reshape(-1, case["head_dim"])[:have]
                    for codes, scale in ((state["k_codes"], state["k_scale"]), (state["v_codes"], state["v_scale"])))
            logits = q[cu[b]: cu[b + 1], h] @ k.T / math.sqrt(case["head_dim"])
            logits[hidden] = -math.inf
            total = torch.logsumexp(logits, -1)
            weight = torch.exp(logits - torch.nan_to_num(total, neginf=0.0)[:, None])
            out[cu[b]: cu[b + 1], h] = weight @ v
            lse[cu[b]: cu[b + 1], h] = total
    return out, lse


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        sign = -1.0 if case["inverse"] else 1.0
        return _turn64(state["x"], state["angles"], state["positions"], case["layout"], sign)
    return _append64(state) if case["op"] == "append" else _attend64(state)
