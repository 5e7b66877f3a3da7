"""A cache of no pages: its codes and scales are empty tensors without memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _int32(*values):
    return torch.tensor(values, dtype=torch.int32).cuda()


@pytest.mark.parametrize("tokens", [2, 80])
def test_a_cache_of_no_pages(tokens):
    """Nothing is stored, and rows see nothing."""
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table, rotary
    cache = PagedKVCache(0, 2, 64, page_size=16)
    x = torch.randn(tokens, 2, 64, device="cuda").half()
    lengths, angles = _int32(tokens // 2, tokens // 2), rope_table(64, 64)
    for table in (_int32([-1], [0]), torch.empty(2, 0, dtype=torch.int32, device="cuda")):
        q = cache.append(x, x, lengths, table, q=x, angles=angles)
        at = torch.arange(tokens, device="cuda") % (tokens // 2)
        assert torch.equal(q, rotary(x, angles, at))
        out, lse = cache.attend(x, lengths, table, return_lse=True)
        assert not out.any() and torch.isneginf(lse).all()
    k, v = cache.read(_int32(0, -1))
    assert torch.isnan(k).all() and torch.isnan(v).all() and k.shape == (2, 2, 16, 64)
