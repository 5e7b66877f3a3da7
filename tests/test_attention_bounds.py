"""Bounds far beyond any sequence mean what a large enough one means."""
import pytest

import rdna2_ops._native as nat


@pytest.mark.parametrize("most", [401, 2 ** 31, 2 ** 62, 2 ** 63 - 1])
def test_workspaces(most):
    need = nat.library().b2_kv_attention_workspace_bytes
    for heads, window in ((8, 0), (32, 0), (32, 100)):
        want = need(400, 2, 400, heads, 8, 128, 64, 64, window)
        assert want > 0 and need(400, 2, most, heads, 8, 128, 64, 64, window) == want
