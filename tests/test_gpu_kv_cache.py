"""The paged 8-bit cache on the GPU against 64 bits: append, read and attention
over ragged batches, odd lengths, absent pages, windows, strides, streams, long
offsets, odd values, and what the calls refuse."""
import math
import random

import pytest
import torch

from kv_reference import assert_close, attend64, check_append, places, rotate64

from conftest import GAMMA_FP32

pytestmark = pytest.mark.gpu


def _paging(lengths, page, rng, width=None, spare=2):
    """A block table over scattered pages, and the number of pages."""
    need = [(n + page - 1) // page for n in lengths]
    width = max(1, *need) if width is None else width
    total = sum(need) + spare
    order = rng.sample(range(total), total)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        for i in range(min(n, width)):
            table[b, i] = order[at]
            at += 1
    return table, total


def _values(cache):
    """(k, v) of every page in 64 bits, from the codes and scales themselves."""
    return tuple(c.cpu().double() * s.cpu().double()[..., None, None]
                 for c, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)))


def _filled(pages, heads, dim, page, code, seed, spread=1.0):
    """A cache with every code in use and scales of differing size."""
    from rdna2_ops.kv_cache import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    cache = PagedKVCache(pages, heads, dim, page_size=page, code=code)
    for codes, scale in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        if code == "int8":
            codes.copy_(torch.randint(-127, 128, codes.shape, generator=g, dtype=torch.int8))
        else:
            bits = torch.randint(0, 256, codes.shape, generator=g, dtype=torch.uint8)
            bits[(bits & 127) == 127] = 126  # no NaN
            codes.view(torch.uint8).copy_(bits)
        scale.copy_(torch.exp(spread * torch.randn(scale.shape, generator=g)) * (0.01 if code == "int8" else 0.004))
    return cache


def _offsets(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)


def _attend(cache, counts, lengths, table, heads, dtype, *, offsets=True, seed=0, q=None, gain=1.0, scale=None, **kw):
    tokens = sum(counts)
    if q is None:
        g = torch.Generator().manual_seed(seed)
        q = (torch.randn(tokens, heads, cache.head_dim, generator=g) * gain).to(dtype).cuda()
    off = _offsets(counts) if offsets else None
    lens = torch.tensor(lengths, dtype=torch.int32)
    k, v = _values(cache)
    want = attend64(q, (k, v, cache.v_scale.cpu().double()), lens, table, off, kw.get("causal", True),
                    kw.get("window"), scale)
    out, lse = cache.attend(q, lens.cuda(), table.cuda(), offsets=None if off is None else off.cuda(), scale=scale,
                            return_lse=True, **kw)
    assert_close(out, want[0], want[2], dtype, "out")
    assert_close(lse, want[1], want[3], torch.float32, "lse")
    return out, lse


# ------------------------------------------------------------------- attention
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 4), (3, 8), (1, 16)])
def test_one_token_each(code, dim, page, kv, group):
    rng = random.Random(dim + page + kv)
    lengths = [1, 15, 16, 17, 0, 127, 128, 129, 300, 1000]
    table, pages = _paging(lengths, page, rng)
    cache = _filled(pages, kv, dim, page, code, seed=page)
    _attend(cache, [1] * len(lengths), lengths, table, kv * group, torch.bfloat16, offsets=False)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,page,group", [(64, 16, 3), (128, 64, 4), (128, 128, 1), (64, 32, 8)])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 7), (True, 100), (False, None), (False, 50)])
def test_ragged_rows(dtype, code, dim, page, group, causal, window):
    rng = random.Random(page + group)
    counts, lengths = [5, 0, 1, 33, 2, 0, 140], [5, 0, 400, 33, 257, 30, 300]
    table, pages = _paging(lengths, page, rng)
    cache = _filled(pages, 2, dim, page, code, seed=group)
    _attend(cache, counts, lengths, table, 2 * group, dtype, causal=causal, window=window, max_new=140)


@pytest.mark.parametrize("max_new", [None, 1, 64, 1000])
def test_max_new_only_chooses_the_kernel(max_new):
    rng = random.Random(3)
    counts, lengths = [1, 64, 9], [200, 64, 90]
    table, pages = _paging(lengths, 32, rng)
    cache = _filled(pages, 2, 128, 32, "int8", seed=5)
    _attend(cache, counts, lengths, table, 8, torch.float16, max_new=max_new)


@pytest.mark.parametrize("dim,count", [(64, 300), (128, 511), (128, 129)])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_a_long_prompt(dim, count, code):
    rng = random.Random(count)
    table, pages = _paging([count + 130], 64, rng)
    cache = _filled(pages, 1, dim, 64, code, seed=count)
    _attend(cache, [count], [count + 130], table, 2, torch.bfloat16, offsets=False)


def test_rows_that_see_nothing():
    """Positions below zero, absent pages, windows past the end, no tokens at
    all: zeros and -inf, and rows beside them are as ever."""
    rng = random.Random(4)
    lengths = [3, 0, 40, 200]
    table, pages = _paging(lengths, 16, rng)
    cache = _filled(pages, 2, 64, 16, "int8", seed=1)
    out, lse = _attend(cache, [6, 4, 3, 2], lengths, table, 4, torch.bfloat16)
    assert (lse[:3] == -math.inf).all() and not out[:3].any() and torch.isfinite(lse[3:6]).all()
    assert (lse[6:10] == -math.inf).all() and not out[6:10].any()
    gone = table.clone()
    gone[2], gone[3, 3:9] = -1, 10 ** 6
    _attend(cache, [6, 4, 3, 2], lengths, gone, 4, torch.bfloat16)
    _attend(cache, [6, 4, 3, 2], lengths, gone, 4, torch.bfloat16, causal=False, window=5)
    narrow = table[:, :2].contiguous()  # sequences longer than the table
    _attend(cache, [6, 4, 3, 2], lengths, narrow, 4, torch.bfloat16)
    _attend(cache, [6, 4, 3, 2], lengths, narrow, 4, torch.bfloat16, causal=False, window=20)


@pytest.mark.parametrize("batch", [257, 700])
def test_many_sequences(batch):
    rng = random.Random(batch)
    lengths = [rng.choice([0, 1, 5, 40, 130]) for _ in range(batch)]
    table, pages = _paging(lengths, 16, rng)
    cache = _filled(pages, 1, 64, 16, "int8", seed=2)
    _attend(cache, [1] * batch, lengths, table, 2, torch.float16, offsets=False)


def test_a_history_split_over_many_blocks():
    rng = random.Random(6)
    lengths = [30011, 13]
    table, pages = _paging(lengths, 128, rng)
    cache = _filled(pages, 1, 128, 128, "e4m3", seed=3)
    first = _attend(cache, [1, 1], lengths, table, 4, torch.float16, offsets=False, gain=0.2)
    again = _attend(cache, [1, 1], lengths, table, 4, torch.float16, offsets=False, gain=0.2)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])  # sums have one order
    _attend(cache, [9, 5], lengths, table, 4, torch.float16, gain=0.2, max_new=9)
    _attend(cache, [70, 13], lengths, table, 4, torch.float16, gain=0.2, window=20000, max_new=70)


@pytest.mark.parametrize("gain,scale", [(1e-30, None), (1e30, 1e-30), (3e38, 1e-38), (1.0, 100.0), (0.0, None)])
@pytest.mark.parametrize("counts", [[1, 1], [40, 80]])
def test_queries_of_any_size(gain, scale, counts):
    rng = random.Random(7)
    lengths = [90, 100]
    table, pages = _paging(lengths, 32, rng)
    cache = _filled(pages, 1, 64, 32, "int8", seed=4)
    q = (torch.rand(sum(counts), 4, 64, generator=torch.Generator().manual_seed(1)) * 2 - 1) * gain
    _attend(cache, counts, lengths, table, 4, torch.bfloat16, q=q.bfloat16().cuda(), scale=scale)


@pytest.mark.parametrize("counts", [[1, 1], [40, 80]])
def test_blocks_of_very_different_scale(counts):
    """Values' scales over forty powers of ten: weights go with the largest
    contribution, and the sum of the weights does not."""
    rng = random.Random(8)
    lengths = [256, 100]
    table, pages = _paging(lengths, 32, rng)
    cache = _filled(pages, 2, 128, 32, "int8", seed=5)
    cache.v_scale.copy_(torch.tensor([1e-20, 1.0, 1e20, 1e-3, 1e5])[torch.arange(cache.v_scale.numel()) % 5].view(
        cache.v_scale.shape))
    _attend(cache, counts, lengths, table, 4, torch.bfloat16)
    cache.v_scale.zero_()  # pages that nothing was appended to
    out, lse = cache.attend(torch.ones(2, 4, 128, device="cuda").half(),
                            torch.tensor(lengths, dtype=torch.int32).cuda(), table.cuda(), return_lse=True)
    assert not out.any() and torch.isfinite(lse).all()


@pytest.mark.parametrize("counts", [[1, 1], [40, 80]])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_masked_blocks_do_not_leak(counts, bad):
    """What lies past a sequence's end or outside its window may be anything;
    a block with a NaN scale shows in the rows that see it and no others."""
    rng = random.Random(9)
    lengths, page = [200, 100], 16
    table, pages = _paging(lengths, page, rng, width=16)
    cache = _filled(pages, 1, 64, page, "e4m3", seed=6)
    used = set(table[table >= 0].tolist())
    (loose,) = [p for p in range(pages) if p not in used][:1]
    cache.k_scale[loose] = cache.v_scale[loose] = bad
    cache.k_codes.view(torch.uint8)[loose] = 127
    table[0, 13:], table[1, 7:] = loose, loose  # past the ends
    clean = _attend(cache, counts, lengths, table, 2, torch.float16)
    tail = cache.k_codes.view(torch.uint8)[int(table[1, 6]), :, 4:], cache.v_codes.view(torch.uint8)[
        int(table[1, 6]), :, 4:]
    for t in tail:
        t.fill_(127)  # the NaN byte, behind the last token of the second sequence
    again = cache.attend(*_same(counts, lengths, table), return_lse=True, offsets=_offsets(counts).cuda())
    q = _same(counts, lengths, table)[0]
    assert torch.equal(again[0], clean[0]) and torch.equal(again[1], clean[1]) and q.shape[0] == sum(counts)
    cache.v_scale[int(table[0, 0])] = bad  # only the first sequence's first tokens
    seen = cache.attend(*_same(counts, lengths, table), return_lse=True, offsets=_offsets(counts).cuda())
    assert not torch.isfinite(seen[0][:counts[0]]).any()
    assert torch.equal(seen[0][counts[0]:], clean[0][counts[0]:])
    window = cache.attend(*_same(counts, lengths, table), offsets=_offsets(counts).cuda(), window=16)
    assert torch.isfinite(window).all()


def _same(counts, lengths, table):
    q = torch.randn(sum(counts), 2, 64, generator=torch.Generator().manual_seed(0)).half().cuda()
    return q, torch.tensor(lengths, dtype=torch.int32).cuda(), table.cuda()


@pytest.mark.parametrize("counts", [[1, 1], [40, 80]])
def test_odd_queries_stay_in_their_rows(counts):
    rng = random.Random(10)
    lengths = [90, 100]
    table, pages = _paging(lengths, 32, rng)
    cache = _filled(pages, 1, 64, 32, "int8", seed=4)
    q, lens, tab = _same(counts, lengths, table)
    off = _offsets(counts).cuda()
    clean = cache.attend(q, lens, tab, offsets=off)
    q[0, 1, 3], q[-1, 0, 5] = math.nan, math.inf
    got = cache.attend(q, lens, tab, offsets=off)
    keep = torch.ones(q.shape[:2], dtype=torch.bool)
    keep[0, 1] = keep[-1, 0] = False
    assert torch.equal(got[keep.cuda()], clean[keep.cuda()])
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[-1, 0]).all()


@pytest.mark.parametrize("counts", [[1, 1], [40, 80]])
def test_strided_queries_and_another_stream(counts):
    rng = random.Random(11)
    lengths = [190, 100]
    table, pages = _paging(lengths, 64, rng)
    cache = _filled(pages, 2, 128, 64, "int8", seed=7)
    fused = torch.randn(sum(counts), 12, 128, generator=torch.Generator().manual_seed(2)).half().cuda()
    for q in (fused[:, 3:7], fused[:, ::3], fused.transpose(0, 1).contiguous().transpose(0, 1)[:, :4],
              fused.transpose(1, 2).contiguous().transpose(1, 2)[:, :4],
              fused.flatten()[1:-127].view(-1)[: (sum(counts) - 1) * 1536].view(-1, 12, 128)[:, :4]):
        n = list(counts)
        n[1] -= sum(counts) - q.shape[0]
        _attend(cache, n, lengths, table, 4, torch.float16, q=q)
    want, _ = _attend(cache, counts, lengths, table, 4, torch.float16, q=fused[:, :4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [cache.attend(fused[:, :4], torch.tensor(lengths, dtype=torch.int32, device="cuda"), table.cuda(),
                            offsets=_offsets(counts).cuda()) for _ in range(3)]
    here = [cache.attend(fused[:, :4], torch.tensor(lengths, dtype=torch.int32, device="cuda"), table.cuda(),
                         offsets=_offsets(counts).cuda()) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got + here)


@pytest.mark.parametrize("counts", [[1], [40]])
def test_offsets_past_32_bits(counts):
    """Pages that begin more than 2^32 bytes into the codes."""
    from rdna2_ops.kv_cache import PagedKVCache
    pages, heads, page, dim = 36000, 8, 128, 128
    assert pages * heads * page * dim > 2 ** 32
    cache = PagedKVCache(pages, heads, dim, page_size=page)
    table = torch.tensor([[35999, 1, 35001, 33333]], dtype=torch.int32)
    some = table[0].tolist()
    g = torch.Generator().manual_seed(12)
    k, v = (torch.randn(500, heads, dim, generator=g).half().cuda() for _ in range(2))
    lens = torch.tensor([500], dtype=torch.int32)
    cache.append(k, v, lens.cuda(), table.cuda())
    small = PagedKVCache(4, heads, dim, page_size=page)
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        getattr(small, name).copy_(getattr(cache, name)[some])
    local = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32)
    want = small.read(local[0].cuda(), dtype=torch.float32)
    assert all(torch.equal(a, b) for a, b in zip(want, cache.read(table[0].cuda(), dtype=torch.float32)))
    assert (want[0].transpose(1, 2).reshape(-1, heads, dim)[:500] - k.float()).abs().max() < 0.03
    q = torch.randn(counts[0], 16, dim, generator=g).half().cuda()
    got = cache.attend(q, lens.cuda(), table.cuda())
    assert torch.equal(got, small.attend(q, lens.cuda(), local.cuda()))
    _attend(small, counts, [500], local, 16, torch.float16, q=q, offsets=False)


# ---------------------------------------------------------------------- append
def _state(cache):
    return tuple((c.cpu().double(), s.cpu().double())
                 for c, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)))


def _append(cache, counts, lengths, table, dtype, *, offsets=True, angles=None, layout="half", q_heads=0, seed=0,
            k=None, v=None, gain=1.0):
    tokens = sum(counts)
    g = torch.Generator().manual_seed(seed)
    shape = (tokens, cache.kv_heads, cache.head_dim)
    k = (torch.randn(shape, generator=g) * gain).to(dtype).cuda() if k is None else k
    v = (torch.randn(shape, generator=g) * gain).to(dtype).cuda() if v is None else v
    q = torch.randn(tokens, q_heads, cache.head_dim, generator=g).to(dtype).cuda() if q_heads else None
    off = _offsets(counts) if offsets else None
    lens = torch.tensor(lengths, dtype=torch.int32)
    before = _state(cache)
    got = cache.append(k, v, lens.cuda(), table.cuda(), offsets=None if off is None else off.cuda(), q=q, angles=angles,
                       layout=layout)
    after = _state(cache)
    where = places(lens, off, tokens)
    positions = torch.tensor([p for _, p in where], dtype=torch.long)
    inside = positions.clamp(0, None if angles is None else angles.shape[0] - 1)
    kk, size = (k.cpu().double(), k.cpu().double().abs()) if angles is None else rotate64(k, angles, inside, layout)
    check_append(before[0], after[0], kk, size, where, table, cache.code)
    check_append(before[1], after[1], v.cpu().double(), v.cpu().double().abs(), where, table, cache.code)
    if q_heads:
        want, size = rotate64(q, angles, inside, layout)
        held = positions >= 0
        assert_close(got[held.cuda()], want[held], GAMMA_FP32 * size[held], dtype, "q")
    else:
        assert got is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dim,page,rot,layout", [
    (64, 16, 64, "half"), (64, 32, 32, "interleaved"), (128, 64, 128, "interleaved"), (128, 128, 48, "half"),
    (128, 16, 0, "half")])
def test_append(dtype, code, dim, page, rot, layout):
    """Prompts, then a few single tokens, then a chunk, onto pages at every
    fill; loud tokens make blocks grow."""
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table
    rng = random.Random(page)
    counts = [page + 3, 1, 0, 2 * page, 5]
    table, pages = _paging([n + 40 for n in counts], page, rng)
    cache = PagedKVCache(pages, 3, dim, page_size=page, code=code)
    angles = rope_table(4096, rot) if rot else None
    lengths = list(counts)
    _append(cache, counts, lengths, table, dtype, angles=angles, layout=layout, q_heads=6 if rot else 0)
    for step in range(4):
        lengths = [n + 1 for n in lengths]
        _append(cache, [1] * 5, lengths, table, dtype, offsets=step % 2 == 0, angles=angles, layout=layout,
                q_heads=7 if rot else 0, seed=step + 1, gain=0.3 + step)
    counts = [7, 0, 20, 1, 33]
    lengths = [a + b for a, b in zip(lengths, counts)]
    _append(cache, counts, lengths, table, dtype, angles=angles, layout=layout, q_heads=1 if rot else 0, seed=9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("layout,counts", [("half", [100, 33]), ("interleaved", [2, 1])])
def test_append_bit_by_bit(dtype, code, layout, counts):
    """Scales, codes and queries against the formulas in elementwise 32-bit torch."""
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table, rotary
    cache = PagedKVCache(10, 3, 64, page_size=32, code=code)
    table = torch.tensor([[4, 9, 0, 2], [7, 1, 3, 8]], dtype=torch.int32)
    g = torch.Generator().manual_seed(2)
    k, v, q = (torch.randn(sum(counts), n, 64, generator=g).to(dtype).cuda() for n in (3, 3, 5))
    lengths, angles = torch.tensor(counts, dtype=torch.int32), rope_table(128, 64)
    got = cache.append(k, v, lengths.cuda(), table.cuda(), offsets=_offsets(counts).cuda(), q=q, angles=angles,
                       layout=layout)
    where = places(lengths, _offsets(counts), sum(counts))
    at = torch.tensor([p for _, p in where]).cuda()
    assert torch.equal(got, rotary(q, angles, at, layout=layout))
    top = torch.tensor(127.0 if code == "int8" else 448.0, device="cuda")
    keys = rotary(k.float(), angles, at, layout=layout)  # held bit by bit to torch elsewhere
    for x, codes, scales in ((keys, cache.k_codes, cache.k_scale), (v.float(), cache.v_codes, cache.v_scale)):
        blocks = {}
        for i, (b, pos) in enumerate(where):
            blocks.setdefault(int(table[b, pos // 32]), []).append((i, pos % 32))
        for page, rows in blocks.items():
            new = x[[i for i, _ in rows]]
            s = (new.abs().amax((0, 2)) / top).clamp_min(2.0 ** -100)
            assert torch.equal(scales[page], s)
            want = new * (1.0 / s)[:, None]
            want = want.round().to(torch.int8) if code == "int8" else want.clamp(-top, top).to(torch.float8_e4m3fn)
            held = codes.view(torch.uint8)[page][:, [slot for _, slot in rows]].transpose(0, 1)
            assert torch.equal(held, want.view(torch.uint8))


def test_append_skips_what_has_no_place():
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table
    rng = random.Random(13)
    lengths = [3, 40, 100, 0]
    table, pages = _paging(lengths, 16, rng)
    table[1, 1], table[2, 4] = -1, 10 ** 6
    cache = _filled(pages, 2, 64, 16, "int8", seed=8)
    _append(cache, [6, 40, 70, 3], lengths, table, torch.float16, angles=rope_table(128, 64), q_heads=3)
    _append(cache, [6, 40, 70, 3], lengths, table[:, :3].contiguous(), torch.float16)
    cache.append(torch.empty(0, 2, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda"),
                 torch.tensor(lengths, dtype=torch.int32, device="cuda"), table.cuda())


def test_append_strided():
    from rdna2_ops.kv_cache import PagedKVCache
    rng = random.Random(14)
    table, pages = _paging([50, 30], 32, rng)
    fused = torch.randn(80, 8, 64, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    for k, v in ((fused[:, 4:6], fused[:, 6:]), (fused[:, ::4], fused[:, 1::4]),
                 (fused.transpose(1, 2).contiguous().transpose(1, 2)[:, :2], fused[:, 2:4])):
        cache = PagedKVCache(pages, 2, 64, page_size=32)
        _append(cache, [50, 30], [50, 30], table, torch.bfloat16, k=k, v=v)


def test_zero_tokens_and_small_ones():
    """A block of zeros has the smallest scale, and its first real token sets it."""
    from rdna2_ops.kv_cache import PagedKVCache
    cache = PagedKVCache(1, 1, 64, page_size=16)
    table = torch.zeros(1, 1, dtype=torch.int32)
    _append(cache, [2], [2], table, torch.float32, gain=0.0)
    assert (cache.k_scale == 2.0 ** -100).all()
    _append(cache, [1], [3], table, torch.float32, gain=1e-20, seed=1)
    _append(cache, [1], [4], table, torch.float32, gain=1e-38, seed=2)
    _append(cache, [1], [5], table, torch.float32, gain=3.0, seed=3)
    assert 0.001 < cache.k_scale.item() < 0.1


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_odd_values_show_in_their_block(code, bad):
    from rdna2_ops.kv_cache import PagedKVCache
    cache = PagedKVCache(3, 2, 64, page_size=16, code=code)
    table = torch.tensor([[0, 2]], dtype=torch.int32).cuda()
    k = torch.randn(20, 2, 64, device="cuda")
    v = torch.randn(20, 2, 64, device="cuda")
    k[3, 1, 5] = bad
    cache.append(k, v, torch.tensor([20], dtype=torch.int32, device="cuda"), table)
    got_k, got_v = cache.read(torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda"), dtype=torch.float32)
    assert not torch.isfinite(got_k[0, 1, 3, 5]) and not torch.isfinite(cache.k_scale[0, 1])
    assert torch.isfinite(got_k[0, 0]).all() and torch.isfinite(got_k[1:]).all() and torch.isfinite(got_v).all()
    out = cache.attend(torch.randn(20, 2, 64, device="cuda").half(),
                       torch.tensor([20], dtype=torch.int32, device="cuda"), table)
    assert torch.isfinite(out[:, 0]).all() and not torch.isfinite(out[3:, 1]).any()


def test_positions_past_the_angles_are_nan():
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table
    cache = PagedKVCache(2, 1, 64, page_size=16)
    table = torch.tensor([[0, 1]], dtype=torch.int32).cuda()
    x = torch.ones(20, 1, 64, device="cuda")
    q = cache.append(x, x, torch.tensor([20], dtype=torch.int32, device="cuda"), table, q=x, angles=rope_table(16, 64))
    assert torch.isfinite(q[:16]).all() and torch.isnan(q[16:]).all()
    assert torch.isfinite(cache.k_scale[0]).all() and torch.isnan(cache.k_scale[1]).all()


# ------------------------------------------------------------------------ read
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128)])
def test_read(dtype, code, page, dim):
    cache = _filled(5, 3, dim, page, code, seed=9)
    pages = torch.tensor([4, 0, 4, -1, 5], dtype=torch.int32)
    k, v, ks, vs = cache.read(pages.cuda(), dtype=dtype, return_scales=True)
    for got, scales, codes, scale in ((k, ks, cache.k_codes, cache.k_scale), (v, vs, cache.v_codes, cache.v_scale)):
        want = (codes.float() * scale[..., None, None]).to(dtype)  # one fp32 product, rounded once
        assert torch.equal(got[:3], want[pages[:3].long().cuda()]) and torch.isnan(got[3:]).all()
        assert torch.equal(scales[:3], scale[pages[:3].long().cuda()]) and torch.isnan(scales[3:]).all()
    assert cache.read(pages[:0].cuda(), dtype=dtype)[0].shape == (0, 3, page, dim)


# -------------------------------------------------------------------- refusals
def test_refusals():
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table
    for exc, args, kw in [(ValueError, (4, 2, 96), {}), (ValueError, (4, 2, 64), dict(page_size=48)),
                          (ValueError, (4, 2, 64), dict(code="int4")), (ValueError, (4, 0, 64), {})]:
        with pytest.raises(exc):
            PagedKVCache(*args, **kw)
    cache = PagedKVCache(4, 2, 64, page_size=16)
    parts = cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale
    for exc, bad in [(TypeError, (parts[0].float(), *parts[1:])), (ValueError, (parts[0][:2], *parts[1:])),
                     (TypeError, (*parts[:2], parts[2].half(), parts[3])), (ValueError, (*parts[:3], parts[3].t())),
                     (ValueError, (parts[0].cpu(), *parts[1:]))]:
        with pytest.raises(exc):
            PagedKVCache.wrap(*bad)
    x, lens = torch.zeros(4, 2, 64, device="cuda").half(), torch.tensor([4, 4], dtype=torch.int32, device="cuda")
    table, off = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 4], dtype=torch.int32).cuda()
    ok = dict(lengths=lens, table=table)
    for exc, kw in [
            (TypeError, dict(q=x.float())), (ValueError, dict(q=x[:, :1])), (ValueError, dict(q=x[:3])),
            (ValueError, dict(q=x[..., :32])), (TypeError, dict(lengths=lens.long())),
            (TypeError, dict(table=table.long())), (ValueError, dict(lengths=lens[:1])),
            (ValueError, dict(table=table.t())), (ValueError, dict(offsets=off[:2])),
            (TypeError, dict(offsets=off.long())), (ValueError, dict(window=0)), (ValueError, dict(scale=0.0)),
            (ValueError, dict(scale=math.inf)), (ValueError, dict(lengths=lens.cpu())), (ValueError, dict(q=x.cpu())),
            (ValueError, dict(offsets=off, max_new=0)), (ValueError, dict(q=x.clone().requires_grad_()))]:
        with pytest.raises(exc):
            cache.attend(**{"q": x, **ok, **kw})
    angles = rope_table(8, 64)
    for exc, kw in [
            (TypeError, dict(k=x.int(), v=x.int())), (ValueError, dict(v=x.float())), (ValueError, dict(v=x[:, :1])),
            (ValueError, dict(k=x[:, :1], v=x[:, :1])), (ValueError, dict(q=x)),
            (TypeError, dict(q=x.float(), angles=angles)),
            (ValueError, dict(q=x[:2], angles=angles)), (ValueError, dict(angles=rope_table(8, 24))),
            (TypeError, dict(angles=angles.half())), (ValueError, dict(angles=angles, layout="other")),
            (ValueError, dict(offsets=off[:2])), (ValueError, dict(k=x[:3], v=x[:3]))]:
        with pytest.raises(exc):
            cache.append(**{"k": x, "v": x, **ok, **kw})
    for exc, args, kw in [(TypeError, (off.long(),), {}), (ValueError, (table,), {}), (ValueError, (off.cpu(),), {}),
                          (TypeError, (off,), dict(dtype=torch.int8))]:
        with pytest.raises(exc):
            cache.read(*args, **kw)
