"""The layer that runs the cached-attention operators between INT8 projections,
and the attention kernels where their variants meet and their references move."""
import random

import pytest
import torch

from test_gpu_kv_cache import _attend, _filled, _offsets, _paging

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def no_wait_gave_up():
    from rdna2_ops import _native as nat
    yield
    assert nat.device_status() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,count", [
    (1, 8), (1, 9), (8, 1), (9, 1), (4, 4), (1, 17), (17, 1), (2, 64), (1, 129), (5, 26), (1, 256), (1, 257), (3, 86),
    (16, 16), (7, 40)])
def test_where_the_variants_meet(dim, group, count):
    """Rows of a kv head at, below and above 8, 16, 128 and 256."""
    lengths = [count + 70, count]
    table, pages = _paging(lengths, 16 if dim == 64 else 64, random.Random(count))
    cache = _filled(pages, 2, dim, 16 if dim == 64 else 64, "int8" if group % 2 else "e4m3", seed=count)
    _attend(cache, [count, count], lengths, table, 2 * group, torch.float16, offsets=False)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (64, 128)])
@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [40, 80]])
@pytest.mark.parametrize("rate", [1.25, 0.8])
def test_scores_that_grow_and_fall(dim, page, counts, rate):
    """Keys a quarter louder, or quieter, with every block: references are
    raised again and again, or never again."""
    lengths = [1500, 700]
    rng = random.Random(page)
    table, pages = _paging(lengths, page, rng)
    cache = _filled(pages, 1, dim, page, "int8", seed=3, spread=0.0)
    for row in table:
        steps = 64 * torch.arange(len(row)) / len(row)  # the same range whatever the page
        held = row >= 0
        cache.k_scale[row[held].long().cuda()] = (1e-5 * rate ** steps * (1.0 if rate > 1 else 1e6)).cuda()[
            held.cuda(), None]
    _attend(cache, counts, lengths, table, 2, torch.float16)
    _attend(cache, counts, lengths, table, 2, torch.float16, window=600)


def test_one_workspace_serves_calls_of_any_shape():
    """Calls of every variant in turn on one stream: each leaves the counters as it found them."""
    lengths = [2000, 1]
    table, pages = _paging(lengths, 32, random.Random(2))
    cache = _filled(pages, 2, 128, 32, "int8", seed=8)
    first = {}
    for turn in range(3):
        for counts in ([1, 1], [9, 1], [200, 1], [2, 0]):
            got = _attend(cache, counts, lengths, table, 8, torch.bfloat16, max_new=max(counts))
            if turn:
                assert torch.equal(got[0], first[tuple(counts)])
            first[tuple(counts)] = got[0]


@pytest.mark.parametrize("offsets", [[0, 300, 100, 400], [50, 60, 70, 80], [0, -5, 1000, 7], [400, 0, 0, 0]])
def test_offsets_that_make_no_sense_stay_inside(offsets):
    """Decreasing, beyond the tokens, or not from 0: no result is promised, but
    what lies around the outputs, the cache's other pages and its codes behind
    them are as they were."""
    lengths = [500, 30, 90]
    table, pages = _paging(lengths, 32, random.Random(5))
    cache = _filled(pages + 2, 2, 64, 32, "int8", seed=4)
    used = set(table[table >= 0].tolist())
    loose = torch.tensor([p for p in range(pages + 2) if p not in used]).cuda()
    before = [t[loose].clone() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)]
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    lens, tab = torch.tensor(lengths, dtype=torch.int32).cuda(), table.cuda()
    x = torch.randn(400, 6, 64, device="cuda").half()
    for most in (1, 400):
        out, lse = cache.attend(x, lens, tab, offsets=off, max_new=most, return_lse=True)
        assert out.shape == x.shape and lse.shape == (400, 6)
    cache.append(x[:, :2], x[:, 2:4], lens, tab, offsets=off)
    torch.cuda.synchronize()
    for a, t in zip(before, (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)):
        assert torch.equal(a, t[loose])


def _layer(window=None, code="int8"):
    from rdna2_ops.cached_attention import CachedAttention
    from rdna2_ops.convrot_checkpoint import quantize_convrot
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table
    torch.manual_seed(4)
    features, q_heads, kv, dim = 512, 8, 2, 64
    qkv, out = (quantize_convrot(torch.randn(n, k, device="cuda") * 0.04, rotation_block=128)
                for n, k in (((q_heads + 2 * kv) * dim, features), (features, q_heads * dim)))
    table = torch.tensor([[3, 0, 5, 7], [1, 6, 2, 4]], dtype=torch.int32).cuda()
    return CachedAttention(qkv, out, PagedKVCache(8, kv, dim, page_size=32, code=code), rope_table(256, dim),
                           q_heads=q_heads, window=window), table


@pytest.mark.parametrize("window", [None, 20])
def test_layer_is_its_operators(window):
    """A prompt and three tokens through the layer and through its parts, bit by bit."""
    layer, table = _layer(window)
    parts, _ = _layer(window)
    counts = [50, 7]
    lengths, offsets = torch.tensor(counts, dtype=torch.int32).cuda(), _offsets(counts).cuda()
    x = torch.randn(57, 512, device="cuda").half()
    for step in range(4):
        got = layer(x, lengths, table, offsets=offsets, max_new=50 if step == 0 else None)
        both = parts.qkv(x, rotation_block=128).view(-1, 12, 64)
        q = parts.cache.append(both[:, 8:10], both[:, 10:], lengths, table, offsets=offsets, q=both[:, :8],
                               angles=parts.angles)
        y = parts.cache.attend(q, lengths, table, offsets=offsets, window=window)
        want = parts.out(y.reshape(-1, 512), rotation_block=128)
        assert got.shape == x.shape and torch.equal(got, want)
        x, offsets = torch.randn(2, 512, device="cuda").half(), None
        lengths += 1


@pytest.mark.parametrize("code,room", [("int8", 0.02), ("e4m3", 0.06)])
def test_layer_against_whole_precision_attention(code, room):
    """The cache's own error: a value is off by half a step of its block, 1/254
    of the block's largest (int8), or by 1/16 of itself (e4m3), uniformly: about
    0.6 % and 2 % of a typical value; the attention and the output projection's
    INT8 (1 %) pass that on.  Three times that is allowed."""
    layer, table = _layer(code=code)
    x = torch.randn(120, 512, device="cuda").half()
    got = layer(x, torch.tensor([60, 60], dtype=torch.int32).cuda(), table)
    both = layer.qkv(x, rotation_block=128, out_dtype=torch.float32).view(2, 60, 12, 64).double()
    row = layer.angles.double()[:60][:, None]
    cos, sin = row[..., :32], row[..., 32:]
    a, b = both[..., :10, :32], both[..., :10, 32:]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    q, k, v = turned[..., :8, :], turned[..., 8:, :].repeat_interleave(4, 2), both[..., 10:, :].repeat_interleave(4, 2)
    s = torch.einsum("bihd,bjhd->bhij", q, k) / 8
    s = s.masked_fill(torch.ones(60, 60, device="cuda").triu(1).bool(), -torch.inf).softmax(-1)
    y = torch.einsum("bhij,bjhd->bihd", s, v).reshape(120, 512).float()
    want = layer.out(y, rotation_block=128, out_dtype=torch.float32)
    assert (got.float() - want).norm() <= 3 * room * want.norm()


def test_layer_refusals():
    from rdna2_ops.cached_attention import CachedAttention
    from rdna2_ops.convrot_checkpoint import quantize_convrot
    layer, _ = _layer()
    narrow = quantize_convrot(torch.randn(512, 256, device="cuda"), rotation_block=128)
    for exc, args, kw in [(TypeError, (layer.qkv.weight, layer.out, layer.cache), dict(q_heads=8)),
                          (TypeError, (layer.qkv, layer.out, None), dict(q_heads=8)),
                          (ValueError, (layer.qkv, layer.out, layer.cache), dict(q_heads=4)),
                          (ValueError, (layer.qkv, narrow, layer.cache), dict(q_heads=8))]:
        with pytest.raises(exc):
            CachedAttention(*args, **kw)


def test_example_runs(capsys):
    from rdna2_ops import cached_attention
    cached_attention.main()
    assert "lengths [320, 65, 21, 190]" in capsys.readouterr().out
