"""Appending against the formulas in 64 bits: what is stored, and the bounds of what is stored.

Tolerances: a rotated value is two products and a sum rounded to fp32 and once to 16 bits: ``u |x| +
3 2^-24 (|a| + |b|)`` (a cosine or sine is 1 at most; 2^-25 for fp16's least step). A bound's code
is the quotient by the row's largest, times 127, rounded: half a code, and the fp32 roundings of the
middle, the quotient, the product and the scale, each 2^-24 of at most 127 codes.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from tests.kv_cases import back, layout, normal16, table, to

HALF_CODE = 0.5 + 4 * 127 * 2.0**-24


def test_the_two_oracles_agree():
    """The complex product is the rotation's formula; the codes stand for the range in 64 bits."""
    x = normal16(1, (30, 3, 64), "bf16")
    pos = np.arange(30) * 7
    for rot, inter in ((64, False), (20, True)):
        cs = table(300, rot)
        assert np.allclose(okv.append64(x, cs, pos, inter), okv.rotate(x, cs[pos], inter, np.float64),
                           rtol=0, atol=1e-14)
    for size in (1.0, 1e-12, 1e4):
        stored = normal16(2, (64, 96), "bf16", size)
        codes, scale = okv.bounds_of(stored)
        row, step = okv.bounds64(stored)
        assert abs(scale - step) <= step * 2.0**-22
        assert (np.abs(codes * np.float64(scale) - row) <= HALF_CODE * step).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,rot,interleaved,size", [
    ("bf16", 8, 2, 128, 64, 128, False, 1.0), ("fp16", 3, 3, 64, 16, 32, True, 1.0),
    ("bf16", 4, 1, 96, 32, 20, False, 300.0), ("fp16", 2, 2, 256, 128, 256, True, 0.01),
    ("bf16", 5, 5, 192, 16, 192, True, 1e-9)])
def test_stored_keys_and_their_bounds(dev, kind, heads, heads_kv, d, page, rot, interleaved, size):
    import torch

    from retrieve_amd import kv

    print(f"{kind} {heads}/{heads_kv} d={d} page={page} rot={rot}", flush=True)
    pos, seq, tab, pages = layout(d + page, page, [(0, 3 * page + 5), (0, page), (0, 2 * page - 1)])
    x = normal16(d, (len(pos), heads + 2 * heads_kv, d), kind, size)
    cs = table(400, rot)
    g = to(dev, x, kind)
    caches = [torch.zeros((pages, heads_kv, page, d), dtype=g.dtype, device=dev) for _ in range(2)]
    bounds = torch.zeros((pages, heads_kv, 2 * d), dtype=torch.int8, device=dev)
    scales = torch.zeros((pages, heads_kv), device=dev)
    q = kv.append(g[:, :heads], g[:, heads:heads + heads_kv], g[:, heads + heads_kv:], to(dev, cs),
                  to(dev, pos), to(dev, seq), to(dev, tab), *caches, bounds, scales, interleaved)
    exact = okv.append64(x[:, :heads + heads_kv], cs, pos, interleaved)
    stored = back(caches[0])
    got = np.concatenate([back(q), stored[tab[seq, pos // page], :, pos % page]], 1)
    u = 2.0**-8 if kind == "bf16" else 2.0**-11
    rough = 2 * np.abs(x[:, :heads + heads_kv]).max(-1, keepdims=True)
    least = 2.0**-25 if kind == "fp16" else 0.0
    assert (np.abs(got - exact) <= u * np.abs(exact) + 3 * 2.0**-24 * rough + least).all()
    codes, scales = bounds.cpu().numpy().astype(np.float64), back(scales).astype(np.float64)
    full = [tab[s, b] for s, n in enumerate(np.bincount(seq)) for b in range(n // page)]
    assert len(full) == 5
    for i in full:
        for h in range(heads_kv):
            row, step = okv.bounds64(stored[i, h])
            assert abs(scales[i, h] - step) <= step * 2.0**-22
            assert (np.abs(codes[i, h] * scales[i, h] - row) <= HALF_CODE * step).all()
