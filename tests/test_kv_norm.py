"""Appending with normed heads: bit for bit against the oracle, and the formula in 64 bits.

``y = x r w`` has three roundings to fp32 (``r``, ``x r``, the product with ``w``) and the rotation two
more (a product, the sum): off by ``5 2^-24`` of the sum of both products' sizes, then one rounding to
16 bits."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from oracle import kv_int8 as o8
from tests.kv_cases import back, layout, normal16, table, to
from tests.kv_int8_cases import UNIT, weights

HAD_NEW = [(0, 70), (5, 60), (127, 1), (16, 1), (31, 33)]


def _call(dev, kind, qkv, heads, heads_kv, cos_sin, pos, seq, tab, state, inter, w, eps, wide=False):
    from retrieve_amd import kv

    x = to(dev, qkv, kind)
    state = [to(dev, state[0], kind), to(dev, state[1], kind), to(dev, state[2]), to(dev, state[3])]
    w = [None if y is None else to(dev, y, None if wide else kind) for y in w]
    out = kv.append(x[:, :heads], x[:, heads:heads + heads_kv], x[:, heads + heads_kv:],
                    None if cos_sin is None else to(dev, cos_sin), to(dev, pos), to(dev, seq),
                    to(dev, tab), *state, inter, *w, eps)
    return [back(y) for y in (out, *state)]


def _want(kind, qkv, heads, heads_kv, cos_sin, pos, seq, tab, state, inter, w, eps):
    kc, vc, bo, sc = (x.copy() for x in state)
    out = okv.append(o8.norm(qkv[:, :heads], w[0], eps),
                     o8.norm(qkv[:, heads:heads + heads_kv], w[1], eps), qkv[:, heads + heads_kv:],
                     cos_sin, pos, seq, tab, kc, vc, bo, sc, kind, inter)
    return [out, kc, vc, bo, sc]


def _case(seed, kind, heads, heads_kv, d, page, had_new=HAD_NEW, size=1.0):
    pos, seq, tab, pages = layout(seed, page, had_new)
    qkv = normal16(seed + 1, (len(pos), heads + 2 * heads_kv, d), kind, size)
    state = (normal16(seed + 2, (pages, heads_kv, page, d), kind),
             normal16(seed + 3, (pages, heads_kv, page, d), kind),
             np.zeros((pages, heads_kv, 2 * d), np.int8), np.zeros((pages, heads_kv), np.float32))
    return pos, seq, tab, qkv, state


def _same(got, want):
    for name, g, w in zip(("q", "k_cache", "v_cache", "bounds", "scales"), got, want):
        assert np.array_equal(g, w), name


def test_the_oracle_norms():
    """A normed head has a mean square of 1 (with weights of 1 and no eps); both oracles agree."""
    x = okv.round16(np.random.Generator(np.random.PCG64(1)).standard_normal((5, 96)), "bf16")
    one = np.ones(96, np.float32)
    assert np.allclose((o8.norm64(x, one, 0.0) ** 2).mean(-1), 1, rtol=0, atol=1e-14)
    assert np.allclose(o8.norm(x, one * 3, 1e-3), o8.norm64(x, one * 3, 1e-3), rtol=4 * 2.0**-24)
    assert o8.norm(x, None, 0.0) is x


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,rot,inter", [
    ("bf16", 8, 2, 128, 64, 128, False), ("fp16", 7, 1, 96, 32, 48, False),
    ("bf16", 4, 2, 96, 128, 20, False), ("fp16", 4, 2, 64, 16, 6, True),
    ("bf16", 5, 5, 192, 32, 192, True), ("fp16", 2, 1, 256, 128, 128, False),
    ("bf16", 3, 3, 64, 16, 32, True), ("fp16", 6, 3, 192, 16, 64, False)])
def test_matches_the_oracle(dev, kind, heads, heads_kv, d, page, rot, inter):
    print(f"norm {kind} {heads}/{heads_kv} d={d} page={page} rot={rot} {inter}", flush=True)
    pos, seq, tab, qkv, state = _case(rot + d, kind, heads, heads_kv, d, page)
    w = weights(d, d, kind)
    args = (qkv, heads, heads_kv, table(400, rot), pos, seq, tab, state, inter, w, 1e-5)
    got = _call(dev, kind, *args)
    _same(got, _want(kind, *args))
    x = o8.norm64(qkv[:, :heads], w[0], 1e-5)
    cs = args[3][pos]
    exact = okv.rotate(x, cs, inter, np.float64)
    size = np.abs(x).max(-1, keepdims=True) * 2
    u = UNIT[kind]
    assert (np.abs(got[0] - exact) <= u * np.abs(exact) + 5 * 2.0**-24 * size + 2.0**-25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["q", "k", "wide", "no rotation"])
def test_parts(dev, which):
    """Queries alone, keys alone, weights of 32 bits, no rotation."""
    pos, seq, tab, qkv, state = _case(3, "bf16", 4, 2, 128, 16)
    w = weights(4, 128, "bf16")
    if which == "wide":
        w = [x + np.float32(2.0**-20) for x in w]
    w = [w[0] if which != "k" else None, w[1] if which != "q" else None]
    cs = None if which == "no rotation" else table(400, 128)
    args = (qkv, 4, 2, cs, pos, seq, tab, state, False, w, 1e-6)
    _same(_call(dev, "bf16", *args, wide=which == "wide"), _want("bf16", *args))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_sizes(dev, kind):
    """Rows of zeros with and without eps (0 and not a number), rows whose squares leave fp32."""
    pos, seq, tab, qkv, state = _case(5, kind, 4, 2, 64, 16, [(0, 20), (7, 1)])
    w = weights(6, 64, kind)
    qkv[3] = 0
    big = np.float32(1e30 if kind == "bf16" else 6e4)
    qkv[5] = okv.round16(qkv[5] * big / 8, kind)
    qkv[6] = okv.round16(qkv[6] / big, kind)
    args = (qkv, 4, 2, table(30, 64), pos, seq, tab, state, False, w, 1e-6)
    got = _call(dev, kind, *args)
    assert (got[0][3] == 0).all() and np.isfinite(got[0]).all()
    _same(got, _want(kind, *args))
    got = _call(dev, kind, *args[:-1], 0.0)
    assert np.isnan(got[0][3]).all() and np.isfinite(np.delete(got[0], 3, 0)).all()


@pytest.mark.gpu
def test_prompts_and_single_tokens_agree(dev):
    """The same bits whether a sequence comes as one prompt or token by token."""
    import torch

    from retrieve_amd import kv

    heads, heads_kv, d, n = 4, 2, 96, 37
    qkv = to(dev, normal16(7, (n, heads + 2 * heads_kv, d), "bf16"), "bf16")
    w = [to(dev, x, "bf16") for x in weights(8, d, "bf16")]
    cs = to(dev, table(64, 48))
    out = []
    for step in (n, 1, 5):
        c = kv.PagedCache(4, heads_kv, d, 16, device=dev)
        c.bounds.zero_(), c.bound_scales.zero_()
        c.reserve(0, n)
        q = []
        for t in range(0, n, step):
            x = qkv[t:t + step]
            pos = torch.arange(t, t + len(x), dtype=torch.int32, device=dev)
            q.append(c.append(x[:, :4], x[:, 4:6], x[:, 6:], cs, pos, torch.zeros_like(pos),
                              q_weight=w[0], k_weight=w[1]))
        pages = c.page_table[0, :3].long()
        rows = c.k[pages].transpose(1, 2).flatten(0, 1)[:n]
        out.append((torch.cat(q), rows, c.bounds[pages[:2]], c.bound_scales[pages[:2]]))
    for other in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], other))


@pytest.mark.gpu
def test_refusals(dev):
    import torch

    from retrieve_amd import kv

    pos, seq, tab, qkv, state = _case(9, "bf16", 4, 2, 64, 16, [(0, 3)])
    x = to(dev, qkv, "bf16")
    cache = (to(dev, state[0], "bf16"), to(dev, state[1], "bf16"), to(dev, state[2]),
             to(dev, state[3]))

    def call(**k):
        return kv.append(x[:, :4], x[:, 4:6], x[:, 6:], None, to(dev, pos), to(dev, seq),
                         to(dev, tab), *cache, **k)

    w = torch.ones(64, device=dev, dtype=torch.bfloat16)
    call(q_weight=w, k_weight=w)
    call(q_weight=w.float())
    # (a view of odd alignment and one with gaps are read as they are)
    odd = torch.ones(65, device=dev, dtype=torch.bfloat16)[1:]
    assert torch.equal(call(q_weight=odd), call(q_weight=w))
    assert torch.equal(call(q_weight=torch.ones(128, device=dev, dtype=torch.bfloat16)[::2]),
                       call(q_weight=w))
    for error, wrong in [(ValueError, dict(q_weight=w[:32])), (ValueError, dict(k_weight=w[None])),
                         (TypeError, dict(q_weight=w.half())), (TypeError, dict(k_weight=w.double())),
                         (TypeError, dict(q_weight=w, k_weight=w.float())),
                         (ValueError, dict(q_weight=w.cpu())),
                         (ValueError, dict(q_weight=w, eps=-1e-6)),
                         (ValueError, dict(q_weight=w, eps=float("nan"))),
                         (ValueError, dict(k_weight=w, eps=float("inf")))]:
        with pytest.raises(error):
            call(**wrong)
