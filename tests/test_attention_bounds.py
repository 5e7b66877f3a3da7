"""Windows and bounds on new tokens far beyond any sequence mean what a large
enough one means."""
import random

import pytest
import torch

import rdna2_ops._native as nat


@pytest.mark.parametrize("most", [401, 2 ** 31, 2 ** 62, 2 ** 63 - 1])
def test_workspaces(most):
    need = nat.library().b2_kv_attention_workspace_bytes
    for heads, window in ((8, 0), (32, 0), (32, 100)):
        want = need(400, 2, 400, heads, 8, 128, 64, 64, window)
        assert want > 0 and need(400, 2, most, heads, 8, 128, 64, 64, window) == want
    assert need(400, 2, 400, 32, 8, 128, 64, 64, max(most, 2 ** 20)) == need(400, 2, 400, 32, 8, 128, 64, 64, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 62, 2 ** 63 - 1])
@pytest.mark.parametrize("counts", [[7, 3], [60, 30]])
@pytest.mark.parametrize("causal", [True, False])
def test_a_window_over_everything(window, counts, causal):
    from test_gpu_kv_cache import _filled, _offsets, _paging
    lengths = [counts[0] - 5, 100]  # five rows at positions below zero
    table, pages = _paging(lengths, 16, random.Random(1))
    cache = _filled(pages, 2, 64, 16, "int8", seed=1)
    q = torch.randn(sum(counts), 4, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    args = q, torch.tensor(lengths, dtype=torch.int32).cuda(), table.cuda()
    off = _offsets(counts).cuda()
    for most in (max(counts), window):
        want = cache.attend(*args, offsets=off, causal=causal, max_new=min(most, sum(counts)), return_lse=True)
        got = cache.attend(*args, offsets=off, causal=causal, window=window, max_new=most, return_lse=True)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("counts,page,dim", [([1, 1, 1], 16, 128), ([40, 1, 7], 16, 64), ([300, 130, 0], 64, 128)])
def test_tables_far_wider_than_their_sequences(counts, page, dim):
    """As wide as the longest context that a server allows: parts of the tile
    kernel go by the width, and most of them find no tokens."""
    from test_gpu_attention_exactness import _check, _queries
    from test_gpu_kv_cache import _filled, _paging
    lengths = [400, 31, 130]
    narrow, pages = _paging(lengths, page, random.Random(4))
    table = torch.full((3, 131072 // page), -1, dtype=torch.int32)
    table[:, :narrow.shape[1]] = narrow
    cache = _filled(pages, 2, dim, page, "int8", seed=9)
    for kw in ({}, dict(window=90), dict(causal=False)):
        _check(cache, _queries(counts, 8, dim), counts, lengths, table, **kw)
