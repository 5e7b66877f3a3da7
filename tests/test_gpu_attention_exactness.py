"""Attention over the cache where its kernels' pipelines could go wrong: long
walks over the cache."""
import random

import pytest
import torch

from test_gpu_kv_cache import _filled, _offsets, _paging

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
