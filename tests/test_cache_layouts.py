"""Keys, values and queries whose strides say nothing, since a dimension has one
entry."""
import pytest
import torch


def _int32(*values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _one_token(heads, gen, device="cuda"):
    """[1, heads, 64] in a buffer whose rows are 129 apart."""
    buf = torch.randn(3, heads * 64 + 1, generator=gen).half().to(device)
    return buf[:, :heads * 64].unflatten(1, (heads, 64))[:1]


def _one_head(tokens, gen, device="cuda"):
    """[tokens, 1, 64] with a head stride of 1."""
    return torch.randn(tokens, 64, generator=gen).half().to(device).unsqueeze(-1).transpose(1, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("make,heads,tokens", [(_one_token, 2, 1), (_one_head, 1, 5), (_one_head, 1, 40)])
def test_strides_of_dimensions_of_one(make, heads, tokens):
    from rdna2_ops.kv_cache import PagedKVCache
    from rdna2_ops.rotary import rope_table
    g = torch.Generator().manual_seed(0)
    k, v, q = (make(heads if make is _one_token else tokens, g) for _ in range(3))
    assert k.shape == (tokens, heads, 64) and k.is_contiguous() and (k.stride(0) % 8 or k.stride(1) % 8)
    table, lengths, angles = _int32([0, 1, 2]), _int32(tokens), rope_table(64, 64)
    a, b = (PagedKVCache(3, heads, 64, page_size=16) for _ in range(2))
    got = a.append(k, v, lengths, table, q=q, angles=angles)
    want = b.append(k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format),
                    lengths, table, q=q.clone(memory_format=torch.contiguous_format), angles=angles)
    assert torch.equal(got, want)
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        assert torch.equal(getattr(a, name), getattr(b, name))
    assert torch.equal(a.attend(q, lengths, table), b.attend(q.clone(memory_format=torch.contiguous_format), lengths,
                                                            table))


@pytest.mark.parametrize("make,n", [(_one_token, 2), (_one_token, 1), (_one_head, 5), (_one_head, 1)])
def test_rows_as_the_kernels_take_them(make, n):
    from rdna2_ops import kv_cache
    x = make(n, torch.Generator().manual_seed(1), "cpu")
    got = kv_cache._rows(x)
    assert torch.equal(got, x) and got.data_ptr() % 16 == 0
    assert got.stride(2) == 1 and got.stride(0) % 8 == 0 and got.stride(1) % 8 == 0


def test_rows_that_the_kernels_read_as_they_are():
    from rdna2_ops import kv_cache
    x = torch.randn(6, 4, 64).half()
    for y in (x, x[:, 1:3], x[::2], x[:0], x[:, :1], x[:1]):
        assert kv_cache._rows(y).data_ptr() == y.data_ptr()
    for y in (x.transpose(1, 2).contiguous().transpose(1, 2), x.flatten()[1:257].view(1, 4, 64)):
        got = kv_cache._rows(y)
        assert torch.equal(got, y) and got.is_contiguous() and got.data_ptr() != y.data_ptr()
