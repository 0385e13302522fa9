"""The 8-bit paged cache's tests: the oracle's state on the GPU, calls, and comparisons."""

from __future__ import annotations

import numpy as np

from oracle import kv as okv
from oracle import kv_int8 as o8
from tests.kv_cases import KINDS, back, layout, normal16, to

UNIT = {"bf16": 2.0**-8, "fp16": 2.0**-11}
NAMES = ("k", "v", "ks", "vs", "kt", "vt")


def on_gpu(dev, c: o8.Cache):
    """(the six tensors of the cache, bounds and their scales)"""
    kind = {"kt": c.kind, "vt": c.kind}
    return ([to(dev, getattr(c, n), kind.get(n)) for n in NAMES],
            [to(dev, c.bounds), to(dev, c.bound_scales)])


def append(dev, c, state, qkv, heads, heads_kv, cos_sin, pos, seq, tab, interleaved=False,
           q_weight=None, k_weight=None, eps=1e-6, wide=False):
    from retrieve_amd import kv

    x = to(dev, qkv, c.kind)
    w = [None if y is None else to(dev, y, None if wide else c.kind) for y in (q_weight, k_weight)]
    out = kv.append_int8(x[:, :heads], x[:, heads:heads + heads_kv], x[:, heads + heads_kv:],
                         None if cos_sin is None else to(dev, cos_sin), to(dev, pos), to(dev, seq),
                         to(dev, tab), *state[0], *state[1], interleaved, *w, eps)
    return back(out)


def want(c, qkv, heads, heads_kv, cos_sin, pos, seq, tab, interleaved=False, q_weight=None,
         k_weight=None, eps=1e-6):
    """The oracle's cache updated in place: the queries."""
    return c.append(qkv[:, :heads], qkv[:, heads:heads + heads_kv], qkv[:, heads + heads_kv:],
                    cos_sin, pos, seq, tab, interleaved, q_weight, k_weight, eps)


def same(state, c: o8.Cache, before: o8.Cache | None = None):
    """Everything that is held, bit for bit: codes of full pages, scales, bounds, the rows of open
    blocks that count (all of them where a sequence has had no tokens)."""
    got = {n: back(x) for n, x in zip(NAMES, state[0])}
    bounds, scales = (back(x) for x in state[1])
    for n in ("ks", "vs"):
        assert np.array_equal(got[n], getattr(c, n)), n
    full = c.ks[:, 0] > 0
    for n in ("k", "v"):
        assert np.array_equal(got[n][full], getattr(c, n)[full]), n
    assert np.array_equal(bounds, c.bounds)
    assert np.array_equal(scales, c.bound_scales, equal_nan=True)  # (what was never written)
    for s, n in enumerate(c.open_of):
        n = c.page if n is None else n
        assert np.array_equal(got["kt"][s, :, :n], c.kt[s, :, :n], equal_nan=True), ("k_tail", s)
        assert np.array_equal(got["vt"][s, :, :, :n], c.vt[s, :, :, :n], equal_nan=True), ("v_tail", s)


def start(seed, page, had_new, heads, heads_kv, d, kind, spare=2):
    """Sequences that hold some tokens already (blocks before their last in codes, the last one open),
    and the packed new tokens' inputs."""
    pos, seq, tab, pages = layout(seed, page, had_new, spare)
    c = o8.Cache(seed + 1, pages, heads_kv, page, d, len(had_new), kind)
    for s, (had, _) in enumerate(had_new):
        if had % page:
            i = tab[s, had // page]
            c.ks[i] = c.vs[i] = 0.0
            c.open_of[s] = had % page
    qkv = normal16(seed + 2, (len(pos), heads + 2 * heads_kv, d), kind)
    return c, qkv, pos, seq, tab


def weights(seed, d, kind):
    return [okv.round16(normal16(seed + i, (d,), kind, 0.3) + np.float32(1), kind) for i in range(2)]


def check_attention(got, c: o8.Cache, q, blocks, pos, seq, tab, scale=None):
    """Tolerances: an output is rounded once (``u |out|``). Weights are rounded once before their
    product with the values: to fp16 beside codes, to the type beside the open block (``w`` relative;
    fp16 also has a least step, 2^-32 of the row's largest weight times value, at most). Scores are
    fp32 sums of D products, exact each: off by ``(D + 16) 2^-24 scale sum |q k|`` with the three
    products behind them; the exponent adds the logarithm of a block's scale (below 2^6 in size, its
    rounding and the sum's 2^-18).

    The products are taken of ``code + 128``, and 128 times the sum of the other factor taken off
    again: every addition to a sum (one for 32 products) rounds a number of up to 255 times that
    factor's sum, by 2^-24. For a score that is ``2^-24 (D / 32 + 8) 255 s_k scale sum |q|``, for an
    output ``2^-24 (keys / 32 + 16) 255 s_v``: 2^-15 to 2^-12 of a code's step."""
    d = q.shape[2]
    scale = 1 / np.sqrt(d) if scale is None else scale
    out, lse, spread, slack = c.attention(q, blocks, pos, seq, tab, scale)
    u, w = UNIT[c.kind], max(UNIT[c.kind], 2.0**-11)
    off = (d + 16) * 2.0**-24 * slack + 2.0**-17
    off += 2.0**-24 * (d / 32 + 8) * 255 * c.ks.max() * abs(scale) * np.abs(q.astype(np.float64)).sum(-1)
    most = max(np.abs(c.v * c.vs[..., None, None]).max(initial=0), np.abs(np.nan_to_num(c.vt)).max())
    keys = c.page * blocks.shape[2]
    least = 2.0**-32 * keys * most + 2.0**-24 * (keys / 32 + 16) * 255 * c.vs.max()
    tol = u * np.abs(out) + (w + 2 * off[..., None]) * spread * (1 + u) + least + 2.0**-25
    bad = ~(np.abs(got[0] - out) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[0][bad][:5], out[bad][:5], tol[bad][:5])
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got[1]), empty) and (got[0][empty] == 0).all()
    with np.errstate(invalid="ignore"):
        assert (empty | (np.abs(got[1] - lse) <= off + 2.0**-20 * np.maximum(1, np.abs(lse)))).all()


__all__ = ["KINDS", "NAMES", "UNIT", "append", "check_attention", "on_gpu", "same", "start", "want",
           "weights"]
