"""Appending to the paged cache: slots, rotations, bounds and padding, bit for bit against the
oracle."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, table, to

# one token a sequence at every place of a page, prompts that start and end inside pages, an empty
# call
DECODE = [(p, 1) for p in (0, 1, 14, 15, 16, 31, 47, 63, 64, 127, 128, 255)]
PROMPTS = [(0, 16), (5, 60), (0, 1), (130, 200), (127, 1), (1, 127)]


def _state(seed, page, had_new, heads, heads_kv, d, kind):
    pos, seq, tab, pages = layout(seed, page, had_new)
    t = len(pos)
    qkv = normal16(seed + 1, (t, heads + 2 * heads_kv, d), kind)
    k_cache = normal16(seed + 2, (pages, heads_kv, page, d), kind)
    v_cache = normal16(seed + 3, (pages, heads_kv, page, d), kind)
    bounds = rng(seed + 4).integers(-127, 128, (pages, heads_kv, 2 * d), dtype=np.int8)
    scales = rng(seed + 5).random((pages, heads_kv), dtype=np.float32)
    return pos, seq, tab, qkv, k_cache, v_cache, bounds, scales


def _run(dev, kind, qkv, heads, heads_kv, cos_sin, pos, seq, tab, kc, vc, bo, sc, interleaved):
    from retrieve_amd import kv

    x = to(dev, qkv, kind)
    state = [to(dev, kc, kind), to(dev, vc, kind), to(dev, bo), to(dev, sc)]
    out = kv.append(x[:, :heads], x[:, heads:heads + heads_kv], x[:, heads + heads_kv:],
                    None if cos_sin is None else to(dev, cos_sin), to(dev, pos), to(dev, seq),
                    to(dev, tab), *state, interleaved)
    return [back(y) for y in (out, *state)]


def _want(kind, qkv, heads, heads_kv, cos_sin, pos, seq, tab, kc, vc, bo, sc, interleaved):
    kc, vc, bo, sc = kc.copy(), vc.copy(), bo.copy(), sc.copy()
    out = okv.append(qkv[:, :heads], qkv[:, heads:heads + heads_kv], qkv[:, heads + heads_kv:],
                     cos_sin, pos, seq, tab, kc, vc, bo, sc, kind, interleaved)
    return out, kc, vc, bo, sc


def _same(got, want):
    for name, g, w in zip(("q", "k_cache", "v_cache", "bounds", "scales"), got, want):
        assert np.array_equal(g, w), name


def test_rotation_turns_pairs():
    """The oracle's rotation is the complex product, and keeps a pair's length."""
    x = rng(1).standard_normal((3, 2, 8))
    angle = rng(2).standard_normal((3, 3))
    cs = np.concatenate([np.cos(angle), np.sin(angle)], 1)
    for inter in (False, True):
        y = okv.rotate(x, cs, inter, np.float64)
        a, b = okv._pairs(6, inter)
        z = (x[..., a] + 1j * x[..., b]) * np.exp(1j * angle)[:, None]
        assert np.allclose(y[..., a] + 1j * y[..., b], z, rtol=0, atol=1e-14)
        assert np.array_equal(y[..., 6:], x[..., 6:])


def test_bounds_hold_every_key():
    """q . mid + |q| . half is the most a block's keys can score, up to half a code a channel."""
    stored = okv.round16(rng(3).standard_normal((16, 64)), "bf16")
    codes, scale = okv.bounds_of(stored)
    for q in rng(4).standard_normal((20, 64)):
        score = (np.concatenate([q, np.abs(q)]) @ codes) * scale
        exact = okv.most_a_block_can_score(q.astype(np.float64), stored.astype(np.float64))
        assert exact >= (stored.astype(np.float64) @ q).max() - 1e-9
        assert abs(score - exact) <= np.abs(q).sum() * scale * (1 + 1e-5) + 1e-9


@pytest.mark.gpu
@pytest.mark.parametrize("had_new", [DECODE, PROMPTS], ids=["decode", "prompts"])
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,rot,interleaved", [
    ("bf16", 8, 2, 128, 64, 128, False),
    ("fp16", 8, 2, 128, 64, 128, True),
    ("bf16", 3, 3, 64, 16, 32, False),
    ("fp16", 7, 1, 96, 32, 48, False),   # halves of whole chunks
    ("bf16", 4, 2, 96, 128, 20, False),  # halves of 10: partners across chunks
    ("fp16", 4, 2, 64, 16, 6, True),     # a chunk half turned
    ("bf16", 5, 5, 192, 32, 192, True),
    ("fp16", 2, 1, 256, 128, 128, False),
    ("bf16", 8, 8, 64, 64, 2, False),
])
def test_matches_the_oracle(dev, had_new, kind, heads, heads_kv, d, page, rot, interleaved):
    print(f"append {kind} {heads}/{heads_kv} d={d} page={page} rot={rot} {interleaved}", flush=True)
    pos, seq, tab, qkv, *state = _state(rot + d, page, had_new, heads, heads_kv, d, kind)
    args = (qkv, heads, heads_kv, table(400, rot), pos, seq, tab, *state, interleaved)
    got, want = _run(dev, kind, *args), _want(kind, *args)
    _same(got, want)
    # the formula in 64 bits: a product's, a sum's and the 16-bit rounding
    cs = args[3][pos]
    exact = okv.rotate(qkv[:, :heads], cs, interleaved, np.float64)
    size = np.abs(okv.rotate(np.abs(qkv[:, :heads]), np.abs(cs), interleaved, np.float64))
    # (|a| |c| + |b| |s| of the second of each pair is the sum; the first's is bounded by both)
    size = np.maximum(size, np.abs(qkv[:, :heads]).max(-1, keepdims=True) * 2)
    u = 2.0**-8 if kind == "bf16" else 2.0**-11
    assert (np.abs(got[0] - exact) <= u * np.abs(exact) + 2.0**-22 * size + 2.0**-25).all()


@pytest.mark.gpu
def test_many_tokens_share_a_workgroup(dev):
    """More tokens and heads than are given a workgroup each: the bounds' tiles of 64 tokens, with
    blocks that begin in one tile and end in the next."""
    had_new = [(3, 700), (0, 65), (60, 1)] + [(i, 1) for i in range(7, 200, 16)]
    pos, seq, tab, qkv, *state = _state(7, 16, had_new, 12, 6, 64, "bf16")
    args = (qkv, 12, 6, table(800, 64), pos, seq, tab, *state, False)
    _same(_run(dev, "bf16", *args), _want("bf16", *args))


@pytest.mark.gpu
def test_without_rotation(dev):
    pos, seq, tab, qkv, *state = _state(9, 16, PROMPTS, 4, 2, 64, "fp16")
    args = (qkv, 4, 2, None, pos, seq, tab, *state, False)
    got = _run(dev, "fp16", *args)
    _same(got, _want("fp16", *args))
    assert np.array_equal(got[0], qkv[:, :4])


@pytest.mark.gpu
def test_padding_writes_nothing(dev):
    """Negative and too large positions, sequences and pages out of range, positions past the
    table."""
    pos, seq, tab, qkv, *state = _state(11, 16, [(0, 40), (15, 1), (30, 20)], 4, 2, 64, "bf16")
    pos, seq, tab = pos.copy(), seq.copy(), tab.copy()
    pos[3], pos[20], seq[5], seq[41] = -1, 2**31 - 1, -2, 3
    tab[0, 1], tab[2, 2] = -1, 10**6
    cos_sin = table(45, 64)
    args = (qkv, 4, 2, cos_sin, pos, seq, tab, *state, False)
    got, want = _run(dev, "bf16", *args), _want("bf16", *args)
    _same(got, want)
    assert (got[0][3] == 0).all() and (got[0][20] == 0).all() and (got[0][5] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cuts", [[40], [1] * 40, [15, 1, 1, 7, 16]])
def test_split_calls_leave_the_same_cache(dev, cuts):
    """The same 40 tokens in one call, token by token, or in pieces: one cache, one set of
    bounds."""
    import torch

    from retrieve_amd import kv

    pos, seq, tab, qkv, kc, vc, bo, sc = _state(13, 16, [(0, 40)], 4, 2, 128, "bf16")
    want = _want("bf16", qkv, 4, 2, table(64, 128), pos, seq, tab, kc, vc, bo, sc, False)
    x, cs, tab = to(dev, qkv, "bf16"), to(dev, table(64, 128)), to(dev, tab)
    state = [to(dev, kc, "bf16"), to(dev, vc, "bf16"), to(dev, bo), to(dev, sc)]
    parts, at = [], 0
    for n in cuts:
        i = slice(at, at + n)
        parts.append(kv.append(x[i, :4], x[i, 4:6], x[i, 6:], cs, to(dev, pos[i]),
                               to(dev, seq[i]), tab, *state))
        at += n
    _same([back(y) for y in (torch.cat(parts), *state)], want)


@pytest.mark.gpu
def test_no_tokens(dev):
    import torch

    from retrieve_amd import kv

    _, _, tab, _, *state = _state(15, 16, [(0, 5)], 4, 2, 64, "bf16")
    state = [to(dev, state[0], "bf16"), to(dev, state[1], "bf16"), to(dev, state[2]),
             to(dev, state[3])]
    x = torch.empty((0, 8, 64), dtype=torch.bfloat16, device=dev)
    none = torch.empty((0,), dtype=torch.int32, device=dev)
    out = kv.append(x[:, :4], x[:, 4:6], x[:, 6:], to(dev, table(4, 64)), none, none, to(dev, tab),
                    *state)
    assert out.shape == (0, 4, 64)


@pytest.mark.gpu
def test_rows_off_the_alignment_are_copied(dev):
    """Views whose rows do not start on 16 bytes, or whose channels are strided."""
    from retrieve_amd import kv
    import torch

    pos, seq, tab, qkv, kc, vc, bo, sc = _state(17, 16, [(3, 30)], 4, 2, 64, "bf16")
    want = _want("bf16", qkv, 4, 2, table(64, 64), pos, seq, tab, kc, vc, bo, sc, False)
    x = to(dev, qkv, "bf16")
    wide = torch.zeros((30, 8, 67), dtype=torch.bfloat16, device=dev)
    wide[..., 3:] = x
    turned = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    state = [to(dev, kc, "bf16"), to(dev, vc, "bf16"), to(dev, bo), to(dev, sc)]
    out = kv.append(wide[:, :4, 3:], turned[:, 4:6], x.transpose(0, 1).contiguous()[6:].transpose(0, 1),
                    to(dev, table(64, 64)), to(dev, pos), to(dev, seq), to(dev, tab), *state)
    _same([back(y) for y in (out, *state)], want)


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """A cache of 2.4 G elements: the last pages' slots, and only they, are written."""
    import torch

    from retrieve_amd import kv

    pages, heads_kv, page, d = 18400, 8, 128, 128
    kc = torch.zeros((pages, heads_kv, page, d), dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    bo = torch.zeros((pages, heads_kv, 2 * d), dtype=torch.int8, device=dev)
    sc = torch.zeros((pages, heads_kv), device=dev)
    assert kc.numel() > 2**31
    x = torch.randn((page, 24, d), device=dev).to(torch.bfloat16)
    pos = torch.arange(page, dtype=torch.int32, device=dev)
    seq = torch.zeros_like(pos)
    tab = torch.tensor([[pages - 1]], dtype=torch.int32, device=dev)
    kv.append(x[:, :8], x[:, 8:16], x[:, 16:], None, pos, seq, tab, kc, vc, bo, sc)
    assert torch.equal(kc[-1], x[:, 8:16].transpose(0, 1))
    assert torch.equal(vc[-1], x[:, 16:].transpose(0, 1))
    assert not kc[:-1].any() and not vc[:-1].any() and not bo[:-1].any()
    codes, scale = okv.bounds_of(back(kc[-1, 7]))
    assert np.array_equal(bo[-1, 7].cpu().numpy(), codes) and float(sc[-1, 7]) == scale


@pytest.mark.gpu
def test_values_that_are_not_finite(dev):
    """NaN and infinities are stored as they are; their block's codes stay in range, other blocks'
    are untouched."""
    pos, seq, tab, qkv, *state = _state(19, 16, [(0, 32)], 2, 1, 64, "bf16")
    qkv[3, 2, 5], qkv[4, 2, 6], qkv[5, 3, 7] = np.nan, np.inf, -np.inf
    args = (qkv, 2, 1, None, pos, seq, tab, *state, False)
    got, want = _run(dev, "bf16", *args), _want("bf16", *args)
    for g, w in zip(got[:3], want[:3]):
        assert np.array_equal(g, w, equal_nan=True)
    second = tab[0, 1]
    assert np.array_equal(got[3][second], want[3][second])
    assert got[4][second] == want[4][second]


@pytest.mark.gpu
def test_refusals(dev):
    import torch

    from retrieve_amd import kv

    pos, seq, tab, qkv, kc, vc, bo, sc = _state(21, 16, [(0, 8)], 4, 2, 64, "bf16")
    x = to(dev, qkv, "bf16")
    good = dict(q=x[:, :4], k=x[:, 4:6], v=x[:, 6:], cos_sin=to(dev, table(16, 64)),
                positions=to(dev, pos), seq_ids=to(dev, seq), page_table=to(dev, tab),
                k_cache=to(dev, kc, "bf16"), v_cache=to(dev, vc, "bf16"), bounds=to(dev, bo),
                bound_scales=to(dev, sc))
    kv.append(**good)
    odd = to(dev, table(16, 64))
    for error, wrong in [
        (ValueError, {"q": x[:, :3]}), (ValueError, {"k": x[:, 4:7]}), (ValueError, {"v": x[:4, 6:]}),
        (TypeError, {"q": x[:, :4].half()}), (TypeError, {"k": x[:, 4:6].float()}),
        (ValueError, {"positions": good["positions"][:4]}),
        (TypeError, {"positions": good["positions"].long()}),
        (TypeError, {"page_table": good["page_table"].long()}),
        (ValueError, {"page_table": good["page_table"][0]}),
        (ValueError, {"cos_sin": odd[:, :3]}), (TypeError, {"cos_sin": odd.double()}),
        (ValueError, {"cos_sin": odd[:, :32]}),
        (ValueError, {"cos_sin": torch.cat([odd, odd], 1)}),
        (ValueError, {"bounds": good["bounds"][:, :1]}),
        (TypeError, {"bounds": good["bounds"].short()}),
        (ValueError, {"bound_scales": good["bound_scales"][:1]}),
        (ValueError, {"k_cache": good["k_cache"].transpose(0, 1)}),
        (ValueError, {"v_cache": good["v_cache"][:1]}),
        (ValueError, {"positions": good["positions"].cpu()}),
        (TypeError, {n: good[n][..., :32].contiguous() for n in ("q", "k", "v", "k_cache", "v_cache")}),
        (ValueError, {n: good[n][:, :, :8].contiguous() for n in ("k_cache", "v_cache")}),
    ]:
        with pytest.raises(error):
            kv.append(**{**good, **wrong})
