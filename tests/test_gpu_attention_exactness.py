"""Attention over the cache against 64 bits, with bounds that follow from its
arithmetic term by term, and where its kernels' pipelines could go wrong."""
import math
import random

import pytest
import torch

from kv_reference import assert_close, places
from test_gpu_kv_cache import _filled, _offsets, _paging, _values

from conftest import GAMMA_FP32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def no_wait_gave_up():
    from rdna2_ops import _native as nat
    yield
    assert nat.device_status() == 0


def _cuda(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _run(cache, q, counts, lengths, table, **kw):
    return cache.attend(q, _cuda(lengths), table.cuda(), offsets=_offsets(counts).cuda(), max_new=max(counts),
                        return_lse=True, **kw)


# --------------------------------------------------------- the tiles' pipeline
@pytest.mark.parametrize("dim,page", [(64, 16), (64, 128), (128, 32), (128, 64)])
@pytest.mark.parametrize("count", [20, 100, 200])
def test_long_walks_repeat_themselves(dim, page, count):
    """Every tile of a long history in one CTA (many heads, so that nothing is
    split) and in parts, with one row tile and with two: no wait gives up, and
    the same call gives the same bits."""
    for heads, length in ((160, 6000), (1, 20000)):
        table, pages = _paging([length], page, random.Random(page))
        cache = _filled(pages, heads, dim, page, "int8", seed=count)
        q = torch.randn(count, heads, dim, generator=torch.Generator().manual_seed(1)).half().cuda()
        first = _run(cache, q, [count], [length], table)
        assert torch.isfinite(first[0]).all() and torch.isfinite(first[1]).all()
        for _ in range(10):
            again = _run(cache, q, [count], [length], table)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ------------------------------------------------------------ 64 bits, bounds
TOP = {"int8": 127.0, "e4m3": 448.0}


def _exact(cache, q, counts, lengths, table, causal=True, window=None, scale=None, only=None):
    """(out, lse, bound of out, bound of lse) in 64 bits, of the heads `only`
    or all, and the pages that each row sees.

    With w_j the softmax of a row and R the largest w_j vs_j in it:

    * A score's products are exact and summed in fp32, GAMMA_FP32 of the sum of
      their magnitudes, int8 keys as c + 128; a query channel below fp16's
      normal numbers is off by 2^-25 of the row's largest.  The exponent, its
      argument and the logarithms add 2^-20: e in all, relative to w_j and
      absolute in the log-sum-exp.
    * A weight that multiplies a code is fp16: off by 2^-11 of itself or, below
      fp16's normal numbers, by 2^-25 of its unit, where the largest is
      2^6 units at least, so by 2^-31 R / vs_j.
    """
    k, v = _values(cache)
    vs, ks = cache.v_scale.cpu().double(), cache.k_scale.cpu().double()
    tokens, heads, dim = q.shape
    group, page = heads // k.shape[1], k.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    q = q.cpu().double()
    out, lse = torch.zeros_like(q), torch.full((tokens, heads), -math.inf, dtype=torch.float64)
    out_tol, lse_tol, seen = torch.zeros_like(q), torch.zeros(tokens, heads, dtype=torch.float64), []
    for i, (b, pos) in enumerate(places(torch.tensor(lengths), _offsets(counts), tokens)):
        hi = min(lengths[b], table.shape[1] * page)
        at = torch.arange(max(0, pos - window + 1) if window else 0, max(0, min(hi, pos + 1) if causal else hi))
        pid = table[b, at // page].long()
        at, pid = at[pid >= 0], pid[pid >= 0]
        seen.append(set(pid.tolist()))
        if not len(at):
            continue
        for h in range(heads) if only is None else only:
            g = h // group
            kk, vv, units = k[pid, g, at % page], v[pid, g, at % page], vs[pid, g].clamp_min(2.0 ** -100)
            s = kk @ q[i, h] * scale
            size = kk.abs() @ q[i, h].abs() + q[i, h].abs().sum() * 128 * ks[pid, g] * (cache.code == "int8")
            e = ((GAMMA_FP32 * size + 2.0 ** -25 * q[i, h].abs().max() * kk.abs().sum(1)) * scale).max() + 2.0 ** -20
            lse[i, h] = torch.logsumexp(s, 0)
            w = torch.exp(s - lse[i, h])
            out[i, h] = w @ vv
            out_tol[i, h] = (2.0 ** -11 + 4 * e) * (w @ vv.abs()) + 2.0 ** -31 * (w * units).max() * (
                vv.abs() / units[:, None]).sum(0)
            lse_tol[i, h] = 2 * e + 2.0 ** -22 * lse[i, h].abs()
    return out, lse, out_tol, lse_tol, seen


def _check(cache, q, counts, lengths, table, only=None, **kw):
    want = _exact(cache, q, counts, lengths, table, only=only, **kw)
    out, lse = _run(cache, q, counts, lengths, table, **kw)
    some = list(range(q.shape[1])) if only is None else only
    assert_close(out[:, some], want[0][:, some], want[2][:, some], q.dtype, "out")
    assert_close(lse[:, some], want[1][:, some], want[3][:, some], torch.float32, "lse")


def _queries(counts, heads, dim, dtype=torch.float16, seed=0):
    return torch.randn(sum(counts), heads, dim, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("code,dtype", [("int8", torch.float16), ("e4m3", torch.float16), ("int8", torch.bfloat16)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (64, 128), (128, 64)])
@pytest.mark.parametrize("counts", [[1, 4], [60, 33]])
@pytest.mark.parametrize("kw", [{}, dict(window=77), dict(causal=False)])
def test_within_the_bounds(code, dtype, dim, page, counts, kw):
    lengths = [700, 333]
    table, pages = _paging(lengths, page, random.Random(dim + page))
    cache = _filled(pages, 2, dim, page, code, seed=page)
    _check(cache, _queries(counts, 6, dim, dtype), counts, lengths, table, **kw)


# ------------------------------------------------------ many small weights
@pytest.mark.parametrize("code,dim", [("int8", 64), ("int8", 128), ("e4m3", 64), ("e4m3", 128)])
@pytest.mark.parametrize("count,heads,length", [(1, 1, 8192), (40, 1, 8192), (1, 300, 1024), (40, 160, 512)])
@pytest.mark.parametrize("log2", [-12, -20, -22, -26])
@pytest.mark.parametrize("last", [False, True])
def test_many_small_weights_beside_a_large_one(code, dim, count, heads, length, log2, last):
    """One token takes nearly all of the weight and has no value; many others,
    2^log2 of it each, are all that comes out.  With many heads a CTA walks the
    whole of a history."""
    lengths = [length + count]
    at = length - 2 if last else 0
    table, pages = _paging(lengths, 64, random.Random(2))
    cache = _filled(pages, heads, dim, 64, code, seed=4)
    cache.k_codes.view(torch.uint8).zero_()
    cache.v_scale.fill_(0.01)
    cache.k_scale.fill_(0.125)
    sink = int(table[0, at // 64])
    # a score of -log2 * ln 2 for queries of one channel: scale * q * code * ks
    cache.k_codes[sink, :, at % 64, 0] = 64
    cache.v_codes.view(torch.uint8)[sink, :, at % 64] = 0
    q = torch.zeros(count, heads, dim)
    q[..., 0] = -log2 * math.log(2) / (8.0 * dim ** -0.5)
    _check(cache, q.half().cuda(), [count], lengths, table, only=[0, heads - 1])


# ----------------------------------------------- masked blocks of no numbers
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("code,dim,page", [("int8", 64, 16), ("e4m3", 128, 16), ("e4m3", 64, 32), ("int8", 128, 32),
                                           ("int8", 128, 64), ("e4m3", 64, 64)])
@pytest.mark.parametrize("counts,kw", [([8], {}), ([8], dict(window=3)), ([4], dict(window=8, causal=False)),
                                       ([12], {}), ([12], dict(window=5)),
                                       ([180], {}), ([180], dict(window=20)), ([300], dict(window=40, causal=False))])
def test_a_block_of_no_numbers_shows_in_the_rows_that_see_it_alone(bad, which, code, dim, page, counts, kw):
    """As an append of a NaN or an infinity leaves it: its scale is no number
    and its codes are 0.  Rows on earlier pages, and rows whose window begins
    behind it, are as if it were any other block."""
    lengths = [324 if counts == [8] else 330]
    table, pages = _paging(lengths, page, random.Random(page))
    cache = _filled(pages, 2, dim, page, code, seed=dim)
    odd = int(table[0, (lengths[0] - counts[0] // 2) // page - (1 if kw else 0)])
    for codes in (cache.k_codes, cache.v_codes):
        codes.view(torch.uint8)[odd] = 0
    q = _queries(counts, 4, dim)
    want = _exact(cache, q, counts, lengths, table, **kw)
    getattr(cache, which)[odd, 1] = bad  # of the second kv head
    out, lse = _run(cache, q, counts, lengths, table, **kw)
    sees = torch.tensor([[odd in s and h >= 2 for h in range(4)] for s in want[4]])
    assert sees.any() and not sees[:, 2:].all()
    assert not torch.isfinite(out[sees.cuda()]).any()
    assert_close(out[~sees.cuda()], want[0][~sees], want[2][~sees], q.dtype, "out")
    assert_close(lse[~sees.cuda()], want[1][~sees], want[3][~sees], torch.float32, "lse")


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("counts", [[3], [100]])
def test_a_row_that_sees_nothing_of_no_numbers_is_zero(bad, counts):
    """Positions below zero, with a query or the only block of no numbers."""
    lengths = [2]
    table, pages = _paging(lengths, 16, random.Random(1))
    cache = _filled(pages, 1, 64, 16, "int8", seed=1)
    cache.k_scale[int(table[0, 0])] = cache.v_scale[int(table[0, 0])] = bad
    q = _queries(counts, 2, 64)
    q[0, 1, 7] = bad
    out, lse = _run(cache, q, counts, lengths, table)
    assert not out[:counts[0] - 2].any() and (lse[:counts[0] - 2] == -math.inf).all()
    assert not torch.isfinite(out[counts[0] - 2:]).any()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("counts", [[8], [12], [150]])
def test_a_masked_block_that_would_overflow_stays_masked(code, counts):
    """Queries near 1e30 over keys near 1e-30, and, where it is masked, a block
    whose scores would be infinite."""
    lengths, page = [324], 16
    table, pages = _paging(lengths, page, random.Random(3))
    cache = _filled(pages, 1, 64, page, code, seed=6)
    cache.k_scale.mul_(1e-30)
    q = (_queries(counts, 2, 64).float() * 1e30).bfloat16()
    odd = int(table[0, lengths[0] // page])
    want = _exact(cache, q, counts, lengths, table)
    cache.k_scale[odd] = 1e20
    out, lse = _run(cache, q, counts, lengths, table)
    free = torch.tensor([odd not in s for s in want[4]])
    assert free.any() and not free.all()
    assert_close(out[free.cuda()], want[0][free], want[2][free], q.dtype, "out")
    assert_close(lse[free.cuda()], want[1][free], want[3][free], torch.float32, "lse")


# ------------------------------------------------------- value scales far apart
@pytest.mark.parametrize("counts,page", [([2], 16), ([2], 64), ([100], 16), ([100], 128)])
@pytest.mark.parametrize("order", [1, -1])
@pytest.mark.parametrize("apart", [2.0 ** -30, 2.0 ** -64, 2.0 ** -70, 2.0 ** -90])
@pytest.mark.parametrize("hide", ["score", "window", "none"])
def test_quiet_blocks_that_the_softmax_favours(counts, page, order, apart, hide):
    """Blocks whose values are `apart` of the others', where those have next to
    no weight, or are hidden: the quiet values come out as they are, whichever
    blocks come first."""
    blocks, dim = 512 // page, 64
    lengths = [512]
    table, pages = _paging(lengths, page, random.Random(page))
    cache = _filled(pages, 1, dim, page, "int8", seed=3, spread=0.1)
    row = table[0].long().cuda()
    late = torch.arange(blocks).cuda() * page >= 256  # the last 256 tokens
    quiet = row[late if order == 1 else ~late]
    loud = row[~late if order == 1 else late]
    cache.v_scale[loud], cache.v_scale[quiet] = 0.25, 0.25 * apart
    kw = {}
    q = _queries(counts, 2, dim, torch.bfloat16)
    if hide == "score":  # about -150 for the loud ones
        q = q * 0.05 + 18.75
        cache.k_codes[loud] = -100
        cache.k_scale[loud] = 0.01
        cache.k_codes[quiet] //= 16
    elif hide == "window" and order == 1:
        kw = dict(window=256 if counts == [2] else 200)  # the last rows see quiet ones alone
    elif hide == "window":  # every row ends in the quiet half
        lengths = [250]
    q = q.bfloat16()
    _check(cache, q, counts, lengths, table, **kw)
