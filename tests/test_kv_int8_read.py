"""Reading the 8-bit cache back: bit for bit, runs and scattered tokens, open blocks, padding."""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import rng
from tests.kv_cases import back, to
from tests.kv_int8_cases import on_gpu, start


def _read(dev, c, state, pos, seq, tab):
    from retrieve_amd import kv

    return [back(x) for x in kv.read_int8(*state[0], to(dev, pos), to(dev, seq), to(dev, tab))]


def _check(dev, c, pos, seq, tab):
    got = _read(dev, c, on_gpu(dev, c), pos, seq, tab)
    for name, a, b in zip("kv", got, c.read(pos, seq, tab)):
        assert np.array_equal(a, b), name


SHAPES = [("bf16", 2, 128, 64), ("fp16", 3, 64, 16), ("bf16", 1, 96, 32), ("fp16", 2, 192, 16),
          ("bf16", 1, 256, 128), ("fp16", 5, 96, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads_kv,d,page", SHAPES)
def test_whole_sequences(dev, kind, heads_kv, d, page):
    """From their first token on, up to an open block or a full one; runs that start inside 16 slots."""
    held = [(0, 1), (0, page), (0, 3 * page + 5), (0, 2 * page - 1), (7, page), (17, 200)]
    c, _, pos, seq, tab = start(d, page, held, 1, heads_kv, d, kind)
    for s, (had, new) in enumerate(held):
        for i in tab[s]:
            if i >= 0:
                c.ks[i] = c.vs[i] = 0.02 + 0.01 * s
        if (had + new) % page:
            i = tab[s, (had + new) // page]
            c.ks[i] = c.vs[i] = 0.0
    print(f"read {kind} {heads_kv} d={d} page={page}", flush=True)
    _check(dev, c, pos, seq, tab)
    order = rng(3).permutation(len(pos))
    _check(dev, c, pos[order], seq[order], tab)
    _check(dev, c, pos[::-1].copy(), seq[::-1].copy(), tab)
    _check(dev, c, np.repeat(pos, 2), np.repeat(seq, 2), tab)
    _check(dev, c, pos[5:6], seq[5:6], tab)


@pytest.mark.gpu
def test_padding(dev):
    """Rows without a token are zeros, whatever stands beside them."""
    c, _, pos, seq, tab = start(5, 16, [(0, 50), (0, 33)], 1, 2, 64, "bf16")
    pos, seq, tab = pos.copy(), seq.copy(), tab.copy()
    c.ks[:], c.vs[:] = 0.03, 0.02
    pos[3], pos[20], seq[40], tab[0, 2] = -1, 2**31 - 1, -5, 99
    got = _read(dev, c, on_gpu(dev, c), pos, seq, tab)
    expected = c.read(pos, seq, tab)
    assert np.array_equal(got[0], expected[0]) and np.array_equal(got[1], expected[1])
    assert (got[0][[3, 20, 40, 35]] == 0).all() and (got[1][[3, 20, 40, 35]] == 0).all()
    empty = _read(dev, c, on_gpu(dev, c), pos[:0], seq[:0], tab)
    assert empty[0].shape == empty[1].shape == (0, 2, 64)


@pytest.mark.gpu
def test_the_largest_numbers(dev):
    """Scales at which codes leave fp16, and the least ones."""
    c, _, pos, seq, tab = start(7, 16, [(0, 48)], 1, 1, 64, "fp16")
    c.ks[tab[0]] = np.float32([[65504 / 127], [1e-8 / 127], [600.0]])
    c.vs[tab[0]] = np.float32([[1e-8 / 127], [65504 / 127], [2e-7]])
    with np.errstate(over="ignore"):
        _check(dev, c, pos, seq, tab)


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    import torch

    from retrieve_amd import kv

    pages, page, d = 18400, 128, 128
    shape = (pages, 8, page, d)
    k, v = (torch.zeros(shape, dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.full((pages, 8), 0.5, device=dev) for _ in range(2))
    kt, vt = (torch.zeros((1, 8, page, d), dtype=torch.bfloat16, device=dev) for _ in range(2))
    g = torch.Generator(device=dev).manual_seed(1)
    where = [0, pages - 1, pages - 2]
    for i in where:
        k[i] = torch.randint(-127, 128, shape[1:], generator=g, device=dev, dtype=torch.int8)
        v[i] = torch.randint(-127, 128, shape[1:], generator=g, device=dev, dtype=torch.int8)
    pos = torch.arange(3 * page, dtype=torch.int32, device=dev)
    tab = torch.tensor([where], dtype=torch.int32, device=dev)
    gk, gv = kv.read_int8(k, v, ks, vs, kt, vt, pos, torch.zeros_like(pos), tab)
    assert torch.equal(gk, (k[where] * 0.5).transpose(1, 2).flatten(0, 1).bfloat16())
    assert torch.equal(gv, (v[where] * 0.5).permute(0, 3, 1, 2).flatten(0, 1).bfloat16())
