"""Captured calls that use scratch: the two-launch selection, its slabs, the attention's parts."""

from __future__ import annotations

import pytest

from retrieve_amd import _native as nat


def _replay(dev, step, change, times=5):
    """Captures ``step``, then replays it ``times`` times behind ``change(i)``, with eager work of the
    same kind between; every replay's results are the eager step's."""
    import torch

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    last = None
    for i in range(times):
        change(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in held]
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        assert last is None or not torch.equal(last, got[0]), "the inputs do not reach the replay"
        last = got[0]


def _inputs(dev, tokens, blocks, columns, heads, heads_kv, d, page=16, pages=400):
    """Tokens at the end of one long sequence whose blocks share the pages (a plain cache of so many
    blocks is not needed for the selection)."""
    import torch

    g = torch.Generator(device=dev).manual_seed(5)
    tab = torch.full((1, columns), -1, dtype=torch.int32, device=dev)
    tab[0, :blocks] = torch.randint(0, pages, (blocks,), generator=g, device=dev, dtype=torch.int32)
    codes = torch.randint(-127, 128, (pages, heads_kv, 2 * d), generator=g, device=dev,
                          dtype=torch.int8)
    scales = torch.rand((pages, heads_kv), generator=g, device=dev) + 0.1
    q = torch.randn((tokens, heads, d), generator=g, device=dev).to(torch.bfloat16)
    pos = page * blocks - 1 - torch.arange(tokens, dtype=torch.int32, device=dev).flip(0)
    return g, tab, codes, scales, q, pos, torch.zeros_like(pos)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,blocks,columns,heads_kv", [(1, 3000, 3001, 1), (3, 20000, 20000, 2),
                                                            (400, 700, 1200, 2), (700, 900, 300000, 1)])
def test_selection_in_two_launches(dev, tokens, blocks, columns, heads_kv):
    """Single tokens over more blocks than one launch takes, prompts, and prompts in slabs."""
    import torch

    from retrieve_amd import kv

    print(f"{tokens} tokens, {blocks} blocks of {columns} columns", flush=True)
    g, tab, codes, scales, q, pos, seq = _inputs(dev, tokens, blocks, columns, 4 * heads_kv, heads_kv,
                                                 64)
    need = nat.lib().rt_kv_select_workspace(tokens, heads_kv, 1, columns, 32, 1, 2)
    whole = 4 * tokens * heads_kv * (columns + 63 & ~63)
    assert 0 < need <= whole and (need < whole) == (columns == 300000)

    def step():
        return (kv.select_blocks(q, codes, scales, pos, seq, tab, 16, 32, 1, 2),)

    def change(i):
        q.copy_(torch.randn(q.shape, generator=g, device=dev))

    _replay(dev, step, change)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,heads_kv,count,page", [(1, 8, 2, 64, 16), (7, 32, 4, 40, 64),
                                                              (2, 40, 1, 300, 16)])
def test_attention_in_parts(dev, tokens, heads, heads_kv, count, page):
    import torch

    from retrieve_amd import kv

    print(f"{tokens} tokens, {heads}/{heads_kv} heads, {count} blocks of {page}", flush=True)
    d, blocks = 128, 400
    g, tab, _, _, q, pos, seq = _inputs(dev, tokens, blocks, blocks, heads, heads_kv, d, page, blocks)
    tab[0] = torch.randperm(blocks, generator=g, device=dev)
    k = torch.randn((blocks, heads_kv, page, d), generator=g, device=dev).to(torch.bfloat16)
    v = torch.randn((blocks, heads_kv, page, d), generator=g, device=dev).to(torch.bfloat16)
    need = nat.lib().rt_kv_attention_workspace(tokens, heads, heads_kv, d, page, count)
    assert need > 0
    chosen = torch.zeros((tokens, heads_kv, count), dtype=torch.int32, device=dev)

    def step():
        return kv.block_attention(q, k, v, chosen, pos, seq, tab)

    def change(i):
        q.copy_(torch.randn(q.shape, generator=g, device=dev))
        order = torch.rand((tokens, heads_kv, blocks), generator=g, device=dev).argsort(-1)
        chosen.copy_(order[..., :count])

    change(-1)
    _replay(dev, step, change)
