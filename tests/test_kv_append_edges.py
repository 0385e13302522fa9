"""The appends' C entries without tokens, and tables without rows."""

from __future__ import annotations

import numpy as np
import pytest

from tests.kv_cases import back, normal16, to


def _calls():
    """Each entry with no pointer but the table, the queries' weights and what else is given."""
    from retrieve_amd import _native as nat

    lib = nat.lib()

    def plain(t, cos_sin, length, weight=None):
        return lib.rt_kv_append(None, 0, 0, None, 0, 0, None, 0, 0, t, 4, 2, 64, 0, cos_sin, length, 64,
                                0, None, None, None, 1, 4, None, None, 3, 16, None, None, None, None)

    def norm(t, cos_sin, length, weight=None):
        return lib.rt_kv_append_norm(None, 0, 0, None, 0, 0, None, 0, 0, t, 4, 2, 64, 0, weight, None, 0,
                                     1e-6, cos_sin, length, 64, 0, None, None, None, 1, 4, None, None, 3,
                                     16, None, None, None, None)

    def int8(t, cos_sin, length, weight=None):
        return lib.rt_kv_append_int8(None, 0, 0, None, 0, 0, None, 0, 0, t, 4, 2, 64, 0, weight, None, 0,
                                     1e-6, cos_sin, length, 64, 0, None, None, None, 1, 4, None, None,
                                     None, None, None, None, 3, 16, None, None, None, None)

    return lib, {"plain": plain, "norm": norm, "int8": int8}


@pytest.mark.parametrize("name", ["plain", "norm", "int8"])
def test_no_pointer_is_looked_at_without_tokens(name):
    """(No GPU: such a call launches nothing, and the refusals come before any launch.)"""
    lib, calls = _calls()
    call = calls[name]
    assert call(0, None, 5) == 0 and call(0, 4, 5) == 0 and call(0, None, 0) == 0
    assert call(0, None, 5, 8) == 0
    assert call(1, None, 5) == 1 and b"null" in lib.rt_last_error()
    assert call(1, 4, 5) == 1 and call(1, None, 0) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("small", [False, True])
def test_a_table_without_rows(dev, small):
    """Every token is past it: zero rows, and nothing is written."""
    import torch

    from retrieve_amd import kv

    kind = kv.Int8PagedCache if small else kv.PagedCache
    cache = kind(4, 2, 64, 16, 1, 4, torch.bfloat16, dev)
    cache.reserve(0, 40)
    held = [x for x in vars(cache).values() if isinstance(x, torch.Tensor)]
    for x in held:
        if x is not cache.page_table:
            x.copy_(torch.ones_like(x))
    before = [back(x) for x in held]
    x = to(dev, normal16(1, (40, 8, 64), "bf16"), "bf16")
    pos = torch.arange(40, dtype=torch.int32, device=dev)
    q = cache.append(x[:, :4], x[:, 4:6], x[:, 6:], torch.empty((0, 64), device=dev), pos,
                     torch.zeros_like(pos))
    assert (back(q) == 0).all()
    assert all(np.array_equal(back(a), b) for a, b in zip(held, before))
