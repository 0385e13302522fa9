"""Forms of the 8-bit cache's calls: weights of either kind, one or both or none, long prompts; the
attention's workspace, whatever number of sequences a call names."""

from __future__ import annotations

import numpy as np
import pytest

from tests.kv_cases import back, table, to
from tests.kv_int8_cases import append, on_gpu, same, start, want, weights
from tests.test_kv_int8_attention import _case

RUNS = [(3, 40), (0, 21), (30, 2), (15, 1), (40, 24)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d,page,rot,inter", [("bf16", 128, 16, 128, False),
                                                   ("fp16", 64, 32, 64, True),
                                                   ("bf16", 96, 16, 40, False),
                                                   ("fp16", 256, 64, 256, False),
                                                   ("bf16", 192, 16, 0, False)])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("which", ["q", "k", "both"])
def test_append_with_weights(dev, kind, d, page, rot, inter, wide, which):
    """Weights of the rows' type and of 32 bits (whose last bits no 16-bit number has), for the
    queries, the keys or both, with a rotation and without: bit for bit the oracle's."""
    print(f"int8 append {kind} d={d} page={page} rot={rot} wide={wide} {which}", flush=True)
    c, qkv, pos, seq, tab = start(d + rot, page, RUNS, 6, 2, d, kind)
    w = weights(d, d, kind)
    if wide:
        w = [x + np.float32(2.0**-20) * (1 + np.arange(d, dtype=np.float32) % 7) for x in w]
    w = [x if which in (n, "both") else None for x, n in zip(w, "qk")]
    state = on_gpu(dev, c)
    args = (qkv, 6, 2, table(400, rot) if rot else None, pos, seq, tab, inter, *w, 1e-5)
    got = append(dev, c, state, *args, wide=wide)
    assert np.array_equal(got, want(c, *args))
    same(state, c)


@pytest.mark.gpu
@pytest.mark.parametrize("heads_kv,runs", [(6, [(5, 1000), (0, 700)]), (8, [(5, 1500), (40, 640)])])
def test_append_of_long_prompts(dev, heads_kv, runs):
    """Tiles of 32 and of 64 tokens a workgroup (T * Hkv above 8192 and above 16384)."""
    print(f"int8 append of {runs}", flush=True)
    c, qkv, pos, seq, tab = start(heads_kv, 16, runs, heads_kv, heads_kv, 64, "bf16")
    state = on_gpu(dev, c)
    args = (qkv, heads_kv, heads_kv, table(1600, 64), pos, seq, tab, False, *weights(7, 64, "bf16"))
    assert np.array_equal(append(dev, c, state, *args), want(c, *args))
    same(state, c)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,heads,heads_kv,count", [(1, 4, 1, 200), (7, 8, 2, 64), (63, 20, 1, 40),
                                                         (64, 4, 4, 40), (300, 2, 2, 33),
                                                         (520, 8, 2, 8), (1100, 8, 8, 5)])
def test_nothing_behind_the_workspace(dev, tokens, heads, heads_kv, count):
    """A call is given as many bytes as the size function asks for, before a region that stays as it
    was, whatever number of sequences the call names (it chooses among forms); the same call again
    gives the same bits."""
    import torch

    from retrieve_amd import _native as nat

    page, d = 16, 64
    c, q, blocks, pos, seq, tab = _case(tokens, "bf16", heads, heads_kv, d, page,
                                        [(page * 40, tokens)], count)
    lib = nat.lib()
    need = lib.rt_kv_attention_int8_workspace(tokens, heads, heads_kv, d, page, count)
    guard = 1 << 22
    space = torch.full((need + guard,), 0x5A, dtype=torch.uint8, device=dev)
    cache = on_gpu(dev, c)[0]
    gq = to(dev, q, "bf16")
    gb, gp, gs, gt = (to(dev, x) for x in (blocks, pos, seq, tab))
    for sequences in (0, 1, 2, tokens // 3, tokens // 2, tokens - 1, tokens, tokens + 1, 100000):
        print(f"{tokens} tokens of {sequences} sequences, {need} bytes", flush=True)
        results = []
        for _ in range(2):
            out, lse = torch.empty_like(gq), torch.empty((tokens, heads), device=dev)
            st = lib.rt_kv_attention_int8(
                gq.data_ptr(), gq.stride(0), gq.stride(1), tokens, heads, heads_kv, d, 0,
                *(x.data_ptr() for x in cache), c.k.shape[0], page, gb.data_ptr(), count,
                gp.data_ptr(), gs.data_ptr(), gt.data_ptr(), *gt.shape, 0.125, sequences,
                out.data_ptr(), lse.data_ptr(), space.data_ptr(), need,
                torch.cuda.current_stream().cuda_stream)
            assert st == 0
            assert bool((space[need:] == 0x5A).all()), sequences
            results.append((back(out), back(lse)))
        assert all(np.array_equal(a, b) for a, b in zip(*results)), sequences
