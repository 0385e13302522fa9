"""Attention over chosen blocks where scores are so large that one key holds a row's weight."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_kv_attention import UNIT, _case, _run


def _check_winners(got, of, kind, q, kc, vc, blocks, pos, seq, tab, scale):
    """The best key has all the weight wherever it leads by more than twice what a score may be off
    (``off``: fp32 sums of exact products, and the two products behind them) and 30 more (weights of
    at most e^-30 beside it, below the 2^-25 allowed): the output is its value, its weight rounded
    once and the output once (``u`` each). Nearly every row's does."""
    out, lse = got
    d, page, u = q.shape[2], kc.shape[2], UNIT[kind]
    group = q.shape[1] // kc.shape[1]
    decided = 0
    for row, t in enumerate(of):
        for h in range(kc.shape[1]):
            keys, values = [], []
            for b in blocks[t, h]:
                if 0 <= b <= pos[t] // page:
                    n = min(page, pos[t] - b * page + 1)
                    keys.append(kc[tab[seq[t], b], h, :n])
                    values.append(vc[tab[seq[t], b], h, :n])
            kk, vv = (np.concatenate(x).astype(np.float64) for x in (keys, values))
            for g in range(h * group, (h + 1) * group):
                x = q[t, g].astype(np.float64)
                scores = kk @ x * scale
                off = (d + 8) * 2.0**-24 * (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                best = scores.argmax()
                ahead = scores[best] - np.partition(scores, -2)[-2] > 2 * off + 30
                assert np.isfinite(out[row, g]).all() and np.isfinite(lse[row, g]), (t, g)
                slack = off + 2.0**-20 * max(1, abs(scores[best]))
                slack += 0 if ahead else np.log(len(scores))
                assert abs(lse[row, g] - scores[best]) <= slack, (t, g)
                if ahead:
                    decided += 1
                    tol = 2 * u * np.abs(vv[best]) * (1 + u) + 2.0**-25
                    assert (np.abs(out[row, g] - vv[best]) <= tol).all(), (t, g)
    assert decided >= 0.9 * len(of) * q.shape[1]


@pytest.mark.gpu
@pytest.mark.parametrize("heads,n", [(8, 1), (8, 480), (40, 300)])
@pytest.mark.parametrize("kind,scale", [("bf16", 2.0**18), ("fp16", 2.0**22), ("bf16", 2.0**30),
                                        ("fp16", -(2.0**40)), ("bf16", -(2.0**90)),
                                        ("fp16", 2.0**96)])
def test_far_scores(dev, kind, scale, heads, n):
    """Scores that are rounded by whole powers of e, of both signs and all below 0: a few rows, many
    joined by workgroup, many of more heads than are joined."""
    print(f"{kind} scale {scale} x{n}", flush=True)
    q, kc, vc, blocks, pos, seq, tab = _case(69, kind, heads, 2, 128, 16, [(200, 1), (90, 4)], 6)
    pick = np.sort(np.r_[0:len(pos) * n:n, n - 1:len(pos) * n:n])
    for below in (False, True):
        if below:
            kc, q = -np.abs(kc), np.abs(q) * np.float32(np.sign(scale))
        many = [np.repeat(x, n, 0) for x in (q, blocks, pos, seq)]
        out, lse = _run(dev, kind, many[0], kc, vc, *many[1:], tab, scale)
        _check_winners((out[pick], lse[pick]), pick // n, kind, q, kc, vc, blocks, pos, seq, tab, scale)
