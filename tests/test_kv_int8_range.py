"""Attention over the 8-bit cache where scores are large: one key holds a row's weight."""

from __future__ import annotations

import numpy as np
import pytest

from tests.kv_int8_cases import UNIT
from tests.test_kv_int8_attention import _case, _run

# times that a case's five tokens are taken: few rows (lists split), 1200 and 2400 tokens of four query
# heads a key/value head (four tokens a workgroup in one tile, eight in two)
FORMS = [1, 240, 480]


def _five(seed, kind, d=128, page=16):
    return _case(seed, kind, 8, 2, d, page, [(200, 1), (90, 4)], 6)


def _repeated(dev, n, c, q, blocks, pos, seq, tab, scale=None):
    """The first and the last of each token's ``n`` results."""
    out, lse = _run(dev, c, *(np.repeat(x, n, 0) for x in (q, blocks, pos, seq)), tab, scale)
    pick = np.sort(np.r_[0:len(pos) * n:n, n - 1:len(pos) * n:n])
    return out[pick], lse[pick], pick // n


def _row(c, blocks, p, s, h, tab):
    """A row's keys and values in 64 bits."""
    keys, values = [], []
    for b in blocks:
        if not 0 <= b <= p // c.page:
            continue
        i, n = tab[s, b], min(c.page, p - b * c.page + 1)
        if c.ks[i, h] > 0:
            k = c.k[i, h] * np.float64(c.ks[i, h])
            v = c.v[i, h].T * np.float64(c.vs[i, h])
        elif b == p // c.page:
            k, v = c.kt[s, h].astype(np.float64), c.vt[s, h].T.astype(np.float64)
        else:
            continue
        keys.append(k[:n])
        values.append(v[:n])
    return np.concatenate(keys), np.concatenate(values)


def _check_winners(got, c, q, blocks, pos, seq, tab, scale=None):
    """Scores are so large that the best key has all the weight wherever it leads by more than twice what
    a score may be off (``off``, as ``kv_int8_cases.check_attention`` derives it) and 30 more (weights of
    at most e^-30 beside it, below the 2^-25 allowed): the output is its value, its weight rounded
    once (``w``) and the output once (``u``). Nearly every row's does."""
    out, lse, of = got
    d, group = q.shape[2], q.shape[1] // c.k.shape[1]
    scale, u = 1 / np.sqrt(d) if scale is None else scale, UNIT[c.kind]
    w = max(u, 2.0**-11)
    decided = 0
    for row, t in enumerate(of):
        for g in range(q.shape[1]):
            h, x = g // group, q[t, g].astype(np.float64)
            kk, vv = _row(c, blocks[t, h], pos[t], seq[t], h, tab)
            scores = kk @ x * scale
            off = (d + 16) * 2.0**-24 * (np.abs(kk) @ np.abs(x)).max() * abs(scale) + 2.0**-17
            off += 2.0**-24 * (d / 32 + 8) * 255 * c.ks.max() * abs(scale) * np.abs(x).sum()
            best = scores.argmax()
            ahead = scores[best] - np.partition(scores, -2)[-2] > 2 * off + 30
            assert np.isfinite(out[row, g]).all() and np.isfinite(lse[row, g]), (t, g)
            slack = off + 2.0**-20 * max(1, abs(scores[best])) + (0 if ahead else np.log(len(scores)))
            assert abs(lse[row, g] - scores[best]) <= slack, (t, g)
            if not ahead:
                continue
            decided += 1
            v = vv[best]
            keys = c.page * blocks.shape[2]
            tol = (u + w) * np.abs(v) * (1 + u) + 2.0**-24 * (keys / 32 + 16) * 255 * c.vs.max()
            assert (np.abs(out[row, g] - v) <= tol + 2.0**-25).all(), (t, g)
    assert decided >= 0.9 * len(of) * q.shape[1]


@pytest.mark.gpu
@pytest.mark.parametrize("n", FORMS)
@pytest.mark.parametrize("kind,scale", [("bf16", 2.0**18), ("fp16", 2.0**22), ("bf16", 2.0**30),
                                        ("fp16", -(2.0**40)), ("bf16", -(2.0**90)),
                                        ("fp16", 2.0**96)])
def test_far_scores(dev, kind, scale, n):
    """Scores that are rounded by whole powers of e, of both signs and all below 0."""
    print(f"{kind} scale {scale} x{n}", flush=True)
    c, q, *rest = _five(69, kind)
    _check_winners(_repeated(dev, n, c, q, *rest, scale), c, q, *rest, scale)
    c.k = -np.maximum(np.abs(c.k), 1).astype(np.int8)
    c.kt = -np.abs(c.kt)
    q = np.abs(q) * np.float32(np.sign(scale))
    _check_winners(_repeated(dev, n, c, q, *rest, scale), c, q, *rest, scale)
