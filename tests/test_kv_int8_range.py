"""Attention over the 8-bit cache where scores are large, or a query's size or the scale is near the
end of 32 bits while the scores are not: one key holds a row's weight, or several keys of equal score
share it."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from tests.kv_int8_cases import UNIT
from tests.test_kv_int8_attention import _case, _run

# times that a case's five tokens are taken: few rows (lists split), 1200 and 2400 tokens of four
# query heads a key/value head (four tokens a workgroup in one tile, eight in two)
FORMS = [1, 240, 480]
MOST = {"bf16": float.fromhex("0x1.fep127"), "fp16": 65504.0}


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
    """Scores are so large that the best key has all the weight wherever it leads by more than twice
    what a score may be off (``off``, as ``kv_int8_cases.check_attention`` derives it) and 30 more
    (weights of at most e^-30 beside it, below the 2^-25 allowed): the output is its value, its weight
    rounded once (``w``) and the output once (``u``). Nearly every row's does."""
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
            slack = off + 2.0**-20 * max(1, abs(scores[best]))
            slack += 0 if ahead else np.log(len(scores))
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


@pytest.mark.gpu
@pytest.mark.parametrize("n", FORMS)
@pytest.mark.parametrize("size", [2.0**112, 2.0**119, 2.0**121, 2.0**123, 2.0**125, 2.0**126])
def test_large_queries(dev, size, n):
    """bf16 queries up to the type's largest number beside keys that leave the scores finite, of
    both signs and all below 0."""
    print(f"queries of {size} x{n}", flush=True)
    c, q, *rest = _five(71, "bf16")
    most = np.float64(MOST["bf16"])
    q = okv.round16(np.clip(q * np.float64(size), -most, most).astype(np.float32), "bf16")
    small = np.float32(2.0**110 / size)
    c.ks *= small
    c.kt = okv.round16(c.kt * small, "bf16")
    _check_winners(_repeated(dev, n, c, q, *rest), c, q, *rest)
    c.k = -np.maximum(np.abs(c.k), 1).astype(np.int8)
    c.kt = -np.abs(c.kt)
    q = np.abs(q)
    _check_winners(_repeated(dev, n, c, q, *rest), c, q, *rest)


@pytest.mark.gpu
@pytest.mark.parametrize("n", FORMS)
@pytest.mark.parametrize("d,page", [(64, 64), (96, 16), (96, 128), (128, 32), (192, 64), (256, 16)])
def test_large_queries_of_every_shape(dev, d, page, n):
    print(f"queries of {d} channels over pages of {page}, x{n}", flush=True)
    c, q, *rest = _five(75, "bf16", d, page)
    q = q * np.float32(2.0**124)
    small = np.float32(2.0**-14)
    c.ks *= small
    c.kt = okv.round16(c.kt * small, "bf16")
    _check_winners(_repeated(dev, n, c, q, *rest), c, q, *rest)


@pytest.mark.gpu
@pytest.mark.parametrize("n", FORMS)
@pytest.mark.parametrize("kind,size,scale", [("bf16", 2.0**127, None), ("bf16", -(2.0**127), None),
                                             ("bf16", 1.0, 2.0**122), ("fp16", 1.0, 2.0**122),
                                             ("fp16", 65504.0, -(2.0**107)),
                                             ("bf16", 2.0**100, 2.0**-126)])
def test_scores_of_zero_beside_large_ones(dev, kind, size, scale, n):
    """Queries of one channel, so that every score is one product (exact but for the three behind it,
    and for the 2^-17 that the logarithm of a block's scale and its sum are off): keys that do not hold
    the channel score 0 and share the weight evenly where all others are below 0; then one key holds a
    code of 1, and the weight. With a scale of the least size all scores are next to 0."""
    print(f"{kind} {size} x {scale}, x{n}", flush=True)
    c, q, blocks, pos, seq, tab = _five(73, kind)
    sign = 1.0 if scale is None else np.sign(scale)
    at, down = 37, -np.sign(size) * sign
    q[:] = 0
    q[:, :, at] = size
    c.k[..., at] = down * np.where(np.arange(16) % 3 == 0, 0, np.abs(c.k[..., at].astype(np.int32)))
    c.kt[..., at] = down * np.where(np.arange(16) % 5 == 0, 0, np.abs(c.kt[..., at]))
    q[1] = q[1] if scale == 2.0**-126 else 0 * q[1]  # (a row of nothing: all scores 0)
    rest = blocks, pos, seq, tab
    used = 1 / np.sqrt(128) if scale is None else scale
    for one in (False, True):
        if one:
            c.k[:, :, 3, at] = -down
        got_out, got_lse, of = _repeated(dev, n, c, q, *rest, scale)
        with np.errstate(under="ignore"):
            out, lse, spread, _ = c.attention(q, *rest, used)
        u, w = UNIT[kind], max(UNIT[kind], 2.0**-11)
        keys = c.page * blocks.shape[2]
        most = max(np.abs(c.v * c.vs[..., None, None]).max(), np.abs(c.vt).max())
        least = 2.0**-32 * keys * most + 2.0**-24 * (keys / 32 + 16) * 255 * c.vs.max()
        tol = u * np.abs(out) + (w + 2.0**-16) * spread * (1 + u) + least + 2.0**-25
        assert np.isfinite(got_out).all() and np.isfinite(got_lse).all()
        off = 2.0**-17 + 2.0**-20 * np.maximum(1, np.abs(lse))
        assert (np.abs(got_lse - lse[of]) <= off[of]).all()
        assert (np.abs(got_out - out[of]) <= tol[of]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", FORMS)
@pytest.mark.parametrize("kind,page,size,scale", [("bf16", 16, 1.0, 2.0**20), ("fp16", 64, 1.0, 2.0**24),
                                                  ("fp16", 32, -1.0, 2.0**36),
                                                  ("bf16", 128, 2.0**123, None),
                                                  ("bf16", 16, -(2.0**123), None)])
def test_equal_far_scores(dev, kind, page, size, scale, n):
    """Keys that are all alike, so that every score of a row is the same number, over full blocks whose
    values are of unlike size: each weighs the same, and the output is the values' mean. (Off: its
    rounding, the weights' and the 2^-17 of a scale's logarithm and its sum; the sums' roundings beside
    the largest block's as ``kv_int8_cases.check_attention`` has them.)"""
    print(f"{kind} page={page} {size} x {scale}, x{n}", flush=True)
    c, q, blocks, pos, seq, tab = _case(77, kind, 8, 2, 128, page, [(9 * page + 3, 1), (7 * page, 4)], 6)
    last = pos // page
    for t in range(len(pos)):
        blocks[t][blocks[t] == last[t]] = -1  # (the open block has no codes)
    g = np.random.Generator(np.random.PCG64(78))
    c.k[:] = c.k[:1, :1, :1]
    c.ks[c.ks > 0] = 0.01 if abs(size) == 1 else 1e-4
    c.vs[c.vs > 0] = np.exp2(g.uniform(-12, 3, c.vs.shape)).astype(np.float32)[c.vs > 0]
    q = okv.round16((np.abs(q) + 1) * np.sign(c.k[0, 0, 0]) * np.float32(size), kind)
    used = 1 / np.sqrt(128) if scale is None else scale
    out, lse, of = _repeated(dev, n, c, q, blocks, pos, seq, tab, scale)
    u, w = UNIT[kind], max(UNIT[kind], 2.0**-11)
    assert np.isfinite(out).all() and np.isfinite(lse).all()
    for row, t in enumerate(of):
        for g in range(8):
            kk, vv = _row(c, blocks[t, g // 4], pos[t], seq[t], g // 4, tab)
            mean, spread, x = vv.mean(0), np.abs(vv).mean(0), q[t, g].astype(np.float64)
            score = kk[0] @ x * used
            assert abs(score) > 2.0**24
            off = (128 + 16) * 2.0**-24 * (np.abs(kk[0]) @ np.abs(x)) * used
            off += 2.0**-24 * (128 / 32 + 8) * 255 * c.ks.max() * used * np.abs(x).sum()
            assert abs(lse[row, g] - score - np.log(len(kk))) <= off + 2.0**-20 * abs(score)
            tol = u * np.abs(mean) + (w + 2.0**-16) * spread * (1 + u) + 2.0**-25
            tol += 2.0**-24 * (len(kk) / 32 + 16) * 255 * c.vs.max()
            assert (np.abs(out[row, g] - mean) <= tol).all(), (t, g, np.abs(out[row, g] - mean).max())


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,count", [("bf16", 20, 1, 64, 16, 128),
                                                              ("fp16", 4, 2, 128, 64, 60),
                                                              ("bf16", 3, 1, 256, 32, 70)])
def test_far_scores_of_long_lists(dev, kind, heads, heads_kv, d, page, count):
    """Single tokens whose lists are split over workgroups, more heads than one tile has."""
    print(f"{kind} {heads}/{heads_kv} d={d} page={page} count={count}", flush=True)
    c, q, *rest = _case(81, kind, heads, heads_kv, d, page, [(page * 150 + 5, 1), (40, 1)], count)
    got = (*_run(dev, c, q, *rest, 2.0**40), np.arange(2))
    _check_winners(got, c, q, *rest, 2.0**40)


@pytest.mark.gpu
@pytest.mark.parametrize("n", FORMS)
def test_rows_beside_far_ones(dev, n):
    """Tokens of far scores beside padding, rows without a list, queries that are not finite and tokens
    of ordinary scores: each as it is alone; captured, replayed and the same bits every time."""
    import torch

    from retrieve_amd import kv
    from tests.kv_cases import back, to
    from tests.kv_int8_cases import check_attention, on_gpu

    c, q, blocks, pos, seq, tab = _case(83, "bf16", 8, 2, 64, 16, [(200, 2), (90, 6)], 6)
    q[0] = okv.round16(q[0] * np.float32(2.0**60), "bf16")
    pos[1], blocks[2], q[3, 5, 7] = -1, -1, np.nan
    case = [np.repeat(x, n, 0) for x in (q, blocks, pos, seq)]
    gq, gb, gp, gs, gt = to(dev, case[0], "bf16"), *(to(dev, x) for x in (*case[1:], tab))
    cache = on_gpu(dev, c)[0]

    def call():
        return kv.block_attention_int8(gq, *cache, gb, gp, gs, gt)

    out, lse = (back(x) for x in call())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(3):
        for x in held:
            x.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(back(held[0]), out, equal_nan=True)
        assert np.array_equal(back(held[1]), lse, equal_nan=True)
    pick = np.sort(np.r_[0:len(pos) * n:n, n - 1:len(pos) * n:n])
    of = pick // n
    out, lse = out[pick], lse[pick]
    none = (of == 1) | (of == 2)
    assert (out[none] == 0).all() and np.isneginf(lse[none]).all()
    assert np.isnan(out[of == 3, 5]).all() and np.isnan(lse[of == 3, 5]).all()
    first = of == 0
    _check_winners((out[first], lse[first], of[first]), c, q, blocks, pos, seq, tab)
    rest = of > 3
    check_attention((out[rest], lse[rest]), c, *(x[of[rest]] for x in (q, blocks, pos, seq)), tab)
