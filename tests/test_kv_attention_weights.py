"""Attention weights far below a row's largest, in fp16."""

from __future__ import annotations

import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,heads_kv,count", [(512, 128, 8, 1024), (600, 16, 8, 256),
                                                         (1, 16, 8, 1024), (700, 8, 8, 1024)])
def test_many_small_weights_beside_a_large_one(dev, tokens, heads, heads_kv, count):
    """One key of weight 1 and all others of about 2^-25.1, values of 1: the output is 1, as the small
    weights are in the sum of the values as they are in the sum of the weights (together 0.4 % of it
    for 131071 keys).

    Tolerance: every weight is rounded once to fp16, where it is held 2^5 times as large at least:
    2^-11 relative, or 2^-25 / 2^5 of the largest; the output once, 2^-11; fp32 sums 2^-18."""
    import torch

    from retrieve_amd import kv

    print(f"{tokens} tokens, {heads}/{heads_kv} heads, {count} blocks", flush=True)
    page, d = 128, 64
    k = torch.zeros((count, heads_kv, page, d), dtype=torch.float16, device=dev)
    k[..., 0] = -17.40625
    k[0, :, 3, 0] = 0.0
    v = torch.ones_like(k)
    q = torch.zeros((tokens, heads, d), dtype=torch.float16, device=dev)
    q[..., 0] = 1.0
    tab = torch.arange(count, dtype=torch.int32, device=dev)[None]
    blocks = tab.expand(tokens, heads_kv, count).contiguous()
    pos = torch.full((tokens,), count * page - 1, dtype=torch.int32, device=dev)
    out, _ = kv.block_attention(q, k, v, blocks, pos, torch.zeros_like(pos), tab, 1.0)
    off = float((out.float() - 1).abs().max())
    assert off <= 2 * 2.0**-11 + count * page * 2.0**-30 + 2.0**-18
