"""Appending to the 8-bit cache: codes, scales, open blocks and bounds, bit for bit against the oracle
(which goes token by token)."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv as okv
from oracle import kv_int8 as o8
from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, table, to
from tests.kv_int8_cases import append, on_gpu, same, start, want, weights

# one token a sequence at every place of a page; prompts that start and end inside pages, fill several
# blocks and leave one open, begin in an open block and end in it
DECODE = [(p, 1) for p in (0, 1, 14, 15, 16, 31, 47, 63, 64, 127, 128, 255)]
PROMPTS = [(0, 16), (5, 60), (0, 1), (130, 200), (127, 1), (1, 127), (3, 4), (17, 300), (0, 0)]
SHAPES = [("bf16", 8, 2, 128, 64, 128, False), ("fp16", 8, 2, 128, 64, 128, True),
          ("bf16", 3, 3, 64, 16, 32, False), ("fp16", 7, 1, 96, 32, 48, False),
          ("bf16", 4, 2, 96, 128, 20, False), ("fp16", 4, 2, 64, 16, 6, True),
          ("bf16", 5, 5, 192, 32, 192, True), ("fp16", 2, 1, 256, 128, 128, False)]


def test_codes():
    """Codes of the oracle: off by half a step, ties to even, the largest at 127, oddities."""
    x = okv.round16(rng(1).standard_normal((16, 64)), "bf16")
    codes, scale = o8.codes_of(x)
    assert np.abs(codes).max() == 127
    # (the scale is rounded once: 2^-24 of at most 127 steps)
    assert (np.abs(codes * np.float64(scale) - x) <= scale * (0.5 + 127 * 2.0**-24)).all()
    codes, scale = o8.codes_of(np.float32([1, 0.5, -0.5, 0, np.nan, np.inf, -np.inf]))
    assert codes.tolist() == [127, 64, -64, 0, 0, 127, -127] and scale == np.float32(1) / 127
    assert o8.codes_of(np.zeros(3, np.float32))[1] == np.float32(1e-8) / np.float32(127)


@pytest.mark.gpu
@pytest.mark.parametrize("had_new", [DECODE, PROMPTS], ids=["decode", "prompts"])
@pytest.mark.parametrize("kind,heads,heads_kv,d,page,rot,inter", SHAPES)
def test_matches_the_oracle(dev, had_new, kind, heads, heads_kv, d, page, rot, inter):
    print(f"int8 {kind} {heads}/{heads_kv} d={d} page={page} rot={rot} {inter}", flush=True)
    c, qkv, pos, seq, tab = start(rot + d, page, had_new, heads, heads_kv, d, kind)
    state = on_gpu(dev, c)
    w = weights(d, d, kind) if rot != d else [None, None]
    args = (qkv, heads, heads_kv, table(400, rot), pos, seq, tab, inter, *w)
    got = append(dev, c, state, *args)
    assert np.array_equal(got, want(c, *args))
    same(state, c)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d,page", [("bf16", 128, 64), ("fp16", 64, 16), ("bf16", 256, 32)])
def test_sequences_grow(dev, kind, d, page):
    """Calls of many sizes, one after the other, three sequences in turn or together; the same bits as
    one prompt."""
    c, *_ = start(11, page, [(0, 700)] * 3, 4, 2, d, kind)
    _, _, tab, _ = layout(11, page, [(0, 700)] * 3)
    state = on_gpu(dev, c)
    cs = table(800, d)
    at = [0, 0, 0]
    rows = normal16(12, (3, 700, 8, d), kind)
    for sizes in [(1, 0, 5), (1, 3, 0), (page - 2, 1, 2 * page), (1, page, 1), (3 * page + 7, 1, 0),
                  (1, 1, 1), (2 * page, 4 * page - 3, page + 1), (0, 5, 1), (page - 1, 1, 1)]:
        pos = np.concatenate([np.arange(a, a + n) for a, n in zip(at, sizes)]).astype(np.int32)
        seq = np.repeat(np.arange(3), sizes).astype(np.int32)
        qkv = rows[seq, pos]
        args = (qkv, 4, 2, cs, pos, seq, tab)
        assert np.array_equal(append(dev, c, state, *args), want(c, *args))
        same(state, c)
        at = [a + n for a, n in zip(at, sizes)]
    whole, *_ = start(13, page, [(0, 700)] * 3, 4, 2, d, kind)
    other = on_gpu(dev, whole)
    pos = np.concatenate([np.arange(a) for a in at]).astype(np.int32)
    seq = np.repeat(np.arange(3), at).astype(np.int32)
    append(dev, whole, other, rows[seq, pos], 4, 2, cs, pos, seq, tab)
    for s, n in enumerate(at):
        full = tab[s, :n // page]
        for x, y in zip(state[0][:4] + state[1], other[0][:4] + other[1]):
            assert np.array_equal(back(x)[full], back(y)[full])


@pytest.mark.gpu
@pytest.mark.parametrize("kind,page", [("bf16", 16), ("fp16", 64)])
def test_sequences_cut_back(dev, kind, page):
    """Tokens at positions that were held already: inside the open block, into a full block (which is
    opened again from its codes), over its end."""
    c, *_ = start(21, page, [(0, 6 * page)] * 4, 4, 2, 64, kind)
    _, _, tab, _ = layout(21, page, [(0, 6 * page)] * 4)
    state = on_gpu(dev, c)
    cs = table(7 * page, 64)
    for i, runs in enumerate([[(0, 3 * page + 9), (0, 2 * page), (0, 2 * page + 1), (0, 5)],
                              [(3 * page + 4, 2), (page + 3, 1), (page + 5, 3), (2, 1)],
                              [(2 * page + 7, 1), (page + 4, page), (page + 8, page - 8), (3, page)],
                              [(2 * page + 8, 2 * page), (7, 3 * page), (2 * page, 1), (1, 4)]]):
        pos = np.concatenate([np.arange(a, a + n) for a, n in runs]).astype(np.int32)
        seq = np.repeat(np.arange(4), [n for _, n in runs]).astype(np.int32)
        qkv = normal16(30 + i, (len(pos), 8, 64), kind)
        args = (qkv, 4, 2, cs, pos, seq, tab)
        assert np.array_equal(append(dev, c, state, *args), want(c, *args))
        same(state, c)


@pytest.mark.gpu
def test_many_tokens_share_a_workgroup(dev):
    had_new = [(3, 700), (0, 65), (60, 1)] + [(i, 1) for i in range(7, 200, 16)]
    c, qkv, pos, seq, tab = start(7, 16, had_new, 12, 6, 64, "bf16")
    state = on_gpu(dev, c)
    args = (qkv, 12, 6, table(800, 64), pos, seq, tab)
    assert np.array_equal(append(dev, c, state, *args), want(c, *args))
    same(state, c)


@pytest.mark.gpu
def test_a_long_prompt_behind_an_open_block(dev):
    """A run of more blocks than a workgroup has threads: its last, open block is found in steps."""
    had_new = [(5, 16 * 300 + 6), (9, 3)]
    c, qkv, pos, seq, tab = start(41, 16, had_new, 1, 1, 64, "fp16")
    state = on_gpu(dev, c)
    args = (qkv, 1, 1, None, pos, seq, tab)
    assert np.array_equal(append(dev, c, state, *args), want(c, *args))
    same(state, c)


@pytest.mark.gpu
def test_padding(dev):
    """Positions below 0 and past the table or the angles, sequences outside it, missing pages: a zero
    row and nothing written, also between tokens that count."""
    had_new = [(3, 40), (0, 20), (30, 2), (15, 1), (40, 9)]
    c, qkv, pos, seq, tab = start(51, 16, had_new, 4, 2, 64, "bf16")
    pos, seq, tab = pos.copy(), seq.copy(), tab.copy()
    pos[60:62] = [-1, 2**31 - 1]
    seq[62] = 7
    tab[4, 2:] = -1
    state = on_gpu(dev, c)
    args = (qkv, 4, 2, table(41, 64), pos, seq, tab)
    got = append(dev, c, state, *args)
    assert np.array_equal(got, want(c, *args)) and (got[60:63] == 0).all()
    same(state, c)
    empty = append(dev, c, state, qkv[:0], 4, 2, None, pos[:0], seq[:0], tab)
    assert empty.shape == (0, 4, 64)
    same(state, c)


@pytest.mark.gpu
def test_numbers_that_are_not_finite(dev):
    """Infinities become +-127 of the finite ones' scale, NaN 0; blocks of zeros; the type's largest
    and least numbers."""
    c, qkv, pos, seq, tab = start(61, 16, [(0, 16 * 7)], 2, 2, 64, "bf16")
    state = on_gpu(dev, c)
    kv = qkv[:, 2:]
    kv[3, 0, 5], kv[4, 2, 6], kv[17, 1, 7], kv[18, 3, 8] = np.inf, -np.inf, np.nan, np.nan
    kv[32:48] = 0
    kv[48:64] *= np.float32(2.0**120)
    kv[64:80] *= np.float32(2.0**-126)
    kv[80:96, :, :] = np.nan
    qkv[:] = okv.round16(qkv, "bf16")
    args = (qkv, 2, 2, None, pos, seq, tab)
    append(dev, c, state, *args)
    with np.errstate(all="ignore"):
        want(c, *args)
    got = [back(x) for x in state[0]]
    for a, b in zip(got[:4], (c.k, c.v, c.ks, c.vs)):
        assert np.array_equal(a, b)
    first = tab[0, 0]
    assert got[0][first, 0, 3, 5] == 127 and got[1][first, 0, 6, 4] == -127
    assert np.isfinite(got[2]).all() and (got[2] > 0).all() and (got[0][tab[0, 5]] == 0).all()


@pytest.mark.gpu
def test_ties(dev):
    """Quotients halfway between two codes go to the even one; every significand against every
    largest one of 8 bits."""
    m = np.arange(128, 256, dtype=np.float32)
    x = np.zeros((128, 1, 256), np.float32)
    x[:, 0, 0] = m * 2  # a block's largest
    for e in range(1, 8):
        x[:, 0, 32 * (e - 1) + 1:32 * e] = (m[:, None] + 4 * np.arange(31)) % 128 + 128
        x[:, 0, 32 * (e - 1) + 1:32 * e] *= np.float32(2.0 ** (1 - e))
    x = np.minimum(x, x[:, :, :1])
    c, _, pos, seq, tab = start(71, 16, [(0, 16 * 128)], 1, 1, 256, "bf16")
    qkv = np.zeros((16 * 128, 3, 256), np.float32)
    qkv[::16, 1], qkv[::16, 2] = x[:, 0], -x[:, 0]
    state = on_gpu(dev, c)
    args = (qkv, 1, 1, None, pos, seq, tab)
    append(dev, c, state, *args)
    want(c, *args)
    same(state, c)


@pytest.mark.gpu
def test_strided_rows(dev):
    import torch

    from retrieve_amd import kv

    c, qkv, pos, seq, tab = start(81, 32, [(3, 70), (9, 1)], 4, 2, 64, "fp16")
    ref = c.copy()
    expected = want(ref, qkv, 4, 2, None, pos, seq, tab)
    x = to(dev, qkv, "fp16")
    odd = torch.zeros((len(pos), 8, 71), dtype=torch.float16, device=dev)
    odd[..., 7:] = x
    for q, k, v in [(odd[:, :4, 7:], odd[:, 4:6, 7:], odd[:, 6:, 7:]),
                    [y.transpose(0, 1).contiguous().transpose(0, 1)
                     for y in (x[:, :4], x[:, 4:6], x[:, 6:])]]:
        state = on_gpu(dev, c)
        got = kv.append_int8(q, k, v, None, to(dev, pos), to(dev, seq), to(dev, tab), *state[0],
                             *state[1])
        assert np.array_equal(back(got), expected)
        same(state, ref)


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """A cache of 2.4 G codes: a prompt and single tokens on its last pages."""
    import torch

    from retrieve_amd import kv

    pages, page, d = 18400, 128, 128
    shape = (pages, 8, page, d)
    k, v = (torch.zeros(shape, dtype=torch.int8, device=dev) for _ in range(2))
    ks, vs = (torch.zeros((pages, 8), device=dev) for _ in range(2))
    kt, vt = (torch.zeros((1, 8, page, d), dtype=torch.bfloat16, device=dev) for _ in range(2))
    bounds, scales = torch.zeros((pages, 8, 2 * d), dtype=torch.int8, device=dev), ks.clone()
    c, qkv, pos, seq, tab = start(91, page, [(0, 2 * page + 5)], 8, 8, d, "bf16", spare=0)
    where = torch.tensor([pages - 1, 0, pages - 2], device=dev)
    x = to(dev, qkv, "bf16")
    kv.append_int8(x[:, :8], x[:, 8:16], x[:, 16:], None, to(dev, pos), to(dev, seq),
                   where.int()[None], k, v, ks, vs, kt, vt, bounds, scales)
    want(c, qkv, 8, 8, None, pos, seq, tab)
    order = tab[0]
    for got, expected in ((k, c.k), (v, c.v), (ks, c.ks), (vs, c.vs), (bounds, c.bounds)):
        assert np.array_equal(back(got[where[:2]]), expected[order[:2]])
    assert np.array_equal(back(kt)[0, :, :5], c.kt[0, :, :5])
    assert int((ks > 0).sum()) == 16


@pytest.mark.gpu
@pytest.mark.parametrize("kind,d,page", [("bf16", 64, 16), ("fp16", 256, 128)])
def test_open_rows_behind_the_end_stay(dev, kind, d, page):
    """A run that completes a block its sequence was cut back into (the earlier rows come from the
    codes) and ends in the next one, and a run that completes an open block: the open block's rows
    from the end on are as they were."""
    had_new = [(page - 3, 5), (2 * page + 9, page - 5), (page // 2, page // 2 + 2)]
    c, qkv, pos, seq, tab = start(d, page, had_new, 4, 2, d, kind)
    for i in (tab[0, 0], tab[1, 2]):  # full so far
        c.ks[i] = c.vs[i] = 0.03
        c.open_of[0] = c.open_of[1] = None
    print(f"append int8 {kind} d={d} page={page}: rows behind the end", flush=True)
    state, before = on_gpu(dev, c), c.copy()
    got = append(dev, c, state, qkv, 4, 2, None, pos, seq, tab)
    assert np.array_equal(got, want(c, qkv, 4, 2, None, pos, seq, tab))
    same(state, c)
    kt, vt = back(state[0][4]), back(state[0][5])
    for s, (had, new) in enumerate(had_new):
        end = (had + new) % page
        assert 0 < end < had % page
        assert np.array_equal(kt[s, :, end:], before.kt[s, :, end:]), s
        assert np.array_equal(vt[s, :, :, end:], before.vt[s, :, :, end:]), s
