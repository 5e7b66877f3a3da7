"""The C entry points of the cached-attention operators refuse bad arguments
with a status before they touch a GPU.  CPU only."""
import pytest
import torch

import rdna2_ops._native as nat

EINVAL = 1  # cudaErrorInvalidValue


def _rotary(**kw):
    args = dict(x=16, dtype=1, tokens=2, heads=4, dim=64, xt=256, xh=64, angles=16, rows=8, rot=64, layout=0, inverse=0,
                positions=16, p64=1, out=16, ot=256, oh=64, stream=None)
    args.update(kw)
    return nat.library().b2_rotary(*args.values())


@pytest.mark.parametrize("bad", [
    dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(dim=0), dict(rot=3), dict(rot=0), dict(rot=66), dict(rows=0),
    dict(layout=2), dict(xt=-1), dict(oh=-1), dict(x=None), dict(angles=None), dict(positions=None), dict(out=None)])
def test_rotary_rejects_bad_arguments(bad):
    assert _rotary(**bad) == EINVAL


def _append(**kw):
    args = dict(k=16, v=16, dtype=1, tokens=4, kv=2, dim=64, kt=128, kh=64, vt=128, vh=64, lengths=16, offsets=None,
                batch=2, table=16, width=3, q=16, qh=4, qt=256, qhs=64, q_out=16, angles=16, rows=8, rot=64, layout=0,
                code=0, kc=16, vc=16, ks=16, vs=16, pages=4, page=16, stream=None)
    args.update(kw)
    return nat.library().b2_kv_append(*args.values())


@pytest.mark.parametrize("bad", [
    dict(dtype=4), dict(tokens=-1), dict(tokens=5), dict(tokens=2 ** 31), dict(kv=0), dict(dim=96), dict(k=24),
    dict(kt=129), dict(vh=-8), dict(lengths=None), dict(batch=0), dict(batch=2 ** 21), dict(table=None), dict(qh=0),
    dict(q_out=None), dict(angles=None), dict(angles=20), dict(rot=24), dict(rot=80), dict(rows=0), dict(layout=2),
    dict(code=2), dict(kc=None), dict(kc=24), dict(vs=None), dict(pages=-1), dict(page=48), dict(page=256)])
def test_append_rejects_bad_arguments(bad):
    assert _append(**bad) == EINVAL


def _attend(**kw):
    args = dict(q=16, dtype=1, tokens=4, qh=4, qt=256, qhs=64, lengths=16, offsets=None, batch=2, most=2, table=16,
                width=3, code=0, kc=16, vc=16, ks=16, vs=16, pages=4, kv=2, page=16, dim=64, scale=0.125, causal=1,
                window=0, out=16, lse=None, work=256, bytes=0, stream=None)
    args.update(kw)
    return nat.library().b2_kv_attention(*args.values())


@pytest.mark.parametrize("bad", [
    dict(), dict(dtype=0), dict(dtype=3), dict(tokens=-1), dict(tokens=5), dict(qh=3), dict(qh=0), dict(qt=257),
    dict(qhs=-8), dict(q=24), dict(lengths=None), dict(batch=0), dict(most=0), dict(most=1), dict(table=None),
    dict(width=2 ** 30), dict(code=2), dict(vc=None), dict(pages=-1), dict(pages=2 ** 31 - 1), dict(kv=0),
    dict(page=24), dict(dim=80), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(window=-1), dict(out=None), dict(out=8), dict(work=None), dict(work=128)])
def test_attention_rejects_bad_arguments(bad):
    """dict(): a workspace that is too small."""
    assert _attend(**bad) == EINVAL


@pytest.mark.parametrize("bad", [
    dict(code=2), dict(num_pages=-1), dict(kv=0), dict(page=8), dict(dim=32), dict(n=-1), dict(dtype=3), dict(kc=None),
    dict(kc=24), dict(k_out=None), dict(pages=None)])
def test_read_rejects_bad_arguments(bad):
    args = dict(kc=16, vc=16, ks=16, vs=16, code=0, num_pages=4, kv=2, page=16, dim=64, pages=16, n=2, dtype=1,
                k_out=16, v_out=16, scales=None, stream=None)
    args.update(bad)
    assert nat.library().b2_kv_read(*args.values()) == EINVAL


def test_nothing_to_do_is_no_error():
    assert _rotary(tokens=0) == 0 and _rotary(heads=0) == 0
    assert _append(tokens=0) == 0 and _attend(tokens=0) == 0
    assert nat.library().b2_kv_attention_workspace_bytes(0, 2, 1, 4, 2, 64, 3, 16, 0) == 0
    assert nat.library().b2_kv_attention_workspace_bytes(4, 2, 1, 3, 2, 64, 3, 16, 0) == 0  # heads do not divide


def test_workspace_does_not_grow_without_end():
    """The most that any call needs: the split row blocks of 128-channel heads."""
    need = nat.library().b2_kv_attention_workspace_bytes
    most = max(need(t, b, t, 64, 8, 128, 4096, 128, 0) for t in (1, 8, 64, 512, 4096, 65536) for b in (1, 7, 64))
    assert most <= 4 * 160 * 256 * 131 * 4 + (1 << 20)


def test_operators_refuse_cpu_tensors():
    from rdna2_ops import kv_cache, rotary
    table = rotary.rope_table(4, 64, device="cpu")
    assert table.shape == (4, 64) and table.dtype == torch.float32
    with pytest.raises(ValueError):
        rotary.rotary(torch.zeros(2, 1, 64), table, torch.arange(2))
    cache = kv_cache.PagedKVCache(2, 1, 64, page_size=16, device="cpu")
    lengths, pages = torch.ones(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64)
    with pytest.raises(ValueError):
        cache.append(x, x, lengths, pages)
    with pytest.raises(ValueError):
        cache.attend(x.half(), lengths, pages)
    with pytest.raises(ValueError):
        cache.read(pages[0])
