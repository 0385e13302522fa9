"""Attention over chosen blocks where scores are so large that one key holds a row's weight."""

from __future__ import annotations

import numpy as np
import pytest

from tests.test_kv_attention import UNIT, _case, _check, _run


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


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,count", [("bf16", 20, 1, 64, 16, 128),
                                                              ("fp16", 4, 2, 128, 64, 60),
                                                              ("bf16", 3, 1, 256, 32, 70)])
def test_far_scores_of_long_lists(dev, kind, heads, heads_kv, d, page, count):
    """Single tokens whose lists are split over workgroups."""
    case = _case(81, kind, heads, heads_kv, d, page, [(page * 150 + 5, 1), (40, 1)], count)
    _check_winners(_run(dev, kind, *case, 2.0**40), np.arange(2), kind, *case, 2.0**40)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 480])
def test_rows_beside_far_ones(dev, n):
    """Tokens of far scores beside padding, rows without a list and tokens of ordinary scores: each as
    it is alone."""
    q, kc, vc, blocks, pos, seq, tab = _case(83, "bf16", 8, 2, 64, 16, [(200, 2), (90, 6)], 6)
    q[0] *= np.float32(2.0**60)
    pos[1], blocks[2] = -1, -1
    many = [np.repeat(x, n, 0) for x in (q, blocks, pos, seq)]
    out, lse = _run(dev, "bf16", many[0], kc, vc, *many[1:], tab)
    pick = np.sort(np.r_[0:len(pos) * n:n, n - 1:len(pos) * n:n])
    of = pick // n
    out, lse = out[pick], lse[pick]
    none, first, rest = (of == 1) | (of == 2), of == 0, of > 2
    assert (out[none] == 0).all() and np.isneginf(lse[none]).all()
    _check_winners((out[first], lse[first]), of[first], "bf16", q, kc, vc, blocks, pos, seq, tab, 0.125)
    _check((out[rest], lse[rest]), "bf16", q[of[rest]], kc, vc, blocks[of[rest]], pos[of[rest]],
           seq[of[rest]], tab)
