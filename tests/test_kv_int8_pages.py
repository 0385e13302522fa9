"""Pages of the 8-bit cache that pass from one sequence to another."""

from __future__ import annotations

import numpy as np
import pytest

from tests.kv_cases import back, normal16, to


def _cache(device, pages=8, sequences=2):
    import torch

    from retrieve_amd import kv

    return kv.Int8PagedCache(pages, 2, 64, 16, sequences, 6, torch.bfloat16, device)


def test_reserved_pages_are_not_full():
    """Whatever a page's scales were, it holds no block once a sequence takes it; pages that others
    hold keep theirs."""
    c = _cache("cpu")
    c.reserve(0, 40)
    c.reserve(1, 33)
    for scales in (c.k_scales, c.v_scales):
        scales.fill_(0.5)
    c.free(0)
    c.reserve(0, 17)
    mine, others = (c.page_table[s][c.page_table[s] >= 0].long() for s in (0, 1))
    assert len(mine) == 2 and len(others) == 3
    for scales in (c.k_scales, c.v_scales):
        assert not scales[mine].any() and (scales[others] == 0.5).all()
    for scales in (c.k_scales, c.v_scales):
        scales[mine] = 0.5
    c.reserve(0, 60)  # (two more: those that it had stay as they are)
    new = c.page_table[0, 2:4].long()
    for scales in (c.k_scales, c.v_scales):
        assert not scales[new].any() and (scales[mine] == 0.5).all()
    c.reserve(0, 60)
    assert (c.k_scales[mine] == 0.5).all()


@pytest.mark.gpu
def test_a_sequence_does_not_see_the_last_owner(dev):
    """A sequence whose pages were another's, before it has written them: blocks before its token's
    own are skipped. Written, it gives what it gives in a cache of its own."""
    import torch

    rows = to(dev, normal16(3, (96, 8, 64), "bf16"), "bf16")
    pos = torch.arange(96, dtype=torch.int32, device=dev)
    results = []
    for used in (False, True):
        c = _cache(dev, pages=6, sequences=2)
        c.k_tail.zero_(), c.v_tail.zero_()
        if used:
            c.reserve(0, 96)
            c.append(rows[:, :4], rows[:, 4:6], rows[:, 6:], None, pos, torch.zeros_like(pos))
            assert bool((c.k_scales > 0).all())
            c.free(0)
        c.reserve(1, 90)
        one = torch.ones_like(pos)
        blocks = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev).expand(1, 2, 3).contiguous()
        at = torch.tensor([60], dtype=torch.int32, device=dev)
        out, lse = c.attend_to(rows[:1, :4], blocks, at, one[:1])
        assert (back(out) == 0).all() and np.isneginf(back(lse)).all()
        got = []
        for a, b in ((0, 70), (70, 71), (71, 90)):
            new = rows[a:b].flip(0).contiguous()
            q = c.append(new[:, :4], new[:, 4:6], new[:, 6:], None, pos[a:b], one[a:b])
            blocks = torch.arange(6, dtype=torch.int32, device=dev).expand(b - a, 2, 6).contiguous()
            got += [q, *c.attend_to(q, blocks, pos[a:b], one[a:b])]
        results.append([back(x) for x in (*got, *c.read(pos[:90], one[:90]))])
    assert all(np.array_equal(a, b) for a, b in zip(*results))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_a_shared_page_is_copied_before_it_is_cut_into(dev, kind):
    """Two sequences share a prompt's full pages; one is cut back into the last of them, after that
    page was copied to one of its own: it goes on as a sequence alone does that is cut back there, and
    the other one's results stay the same bits."""
    import torch

    from retrieve_amd import kv

    page, at = 16, 41
    dtype = getattr(torch, {"bf16": "bfloat16", "fp16": "float16"}[kind])
    rows = to(dev, normal16(5, (60, 8, 64), kind), kind)
    more = to(dev, normal16(6, (20, 8, 64), kind), kind)

    def append(c, s, x, first):
        pos = torch.arange(first, first + len(x), dtype=torch.int32, device=dev)
        seq = torch.full_like(pos, s)
        q = c.append(x[:, :4], x[:, 4:6], x[:, 6:], None, pos, seq)
        return [q, *c.attend(q, pos, seq, 6, 0, 6)]

    def held(c, s, n):
        pos = torch.arange(n, dtype=torch.int32, device=dev)
        return c.read(pos, torch.full_like(pos, s))

    alone = kv.Int8PagedCache(8, 2, 64, page, 1, 4, dtype, dev)
    alone.reserve(0, 64)
    append(alone, 0, rows[:48], 0)
    expected = [*append(alone, 0, more, at), *held(alone, 0, at + 20)]

    c = kv.Int8PagedCache(8, 2, 64, page, 2, 4, dtype, dev)
    c.reserve(0, 64)
    c.reserve(1, 64)
    append(c, 0, rows[:48], 0)
    before = held(c, 0, 48)
    own = int(c.page_table[1, 2])
    c.page_table[1, :2] = c.page_table[0, :2]
    shared = int(c.page_table[0, 2])
    for x in (c.k_codes, c.v_codes, c.k_scales, c.v_scales, c.bounds, c.bound_scales):
        x[own] = x[shared]
    got = [*append(c, 1, more, at), *held(c, 1, at + 20)]
    assert all(torch.equal(a, b) for a, b in zip(got, expected))
    assert all(torch.equal(a, b) for a, b in zip(held(c, 0, 48), before))
