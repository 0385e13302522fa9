"""The paged cache as a layer uses it: the rotary tables, the page book-keeping, the three calls
together, their schemas, graph capture, other streams."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import kv as okv
from tests.conftest import rng
from tests.kv_cases import back, normal16, to


# --- on the host --------------------------------------------------------------------------------


def test_rotary_table_turns_by_position():
    from retrieve_amd import kv

    t = kv.rotary_table(50, 8, device="cpu").numpy()
    for p in (0, 1, 49):
        for i in range(4):
            angle = p * 10000.0 ** (-2 * i / 8)
            assert t[p, i] == np.float32(math.cos(angle)) and t[p, 4 + i] == np.float32(math.sin(angle))


def test_rotary_scalings():
    from retrieve_amd import kv

    plain = kv.rotary_table(64, 16, device="cpu")
    linear = kv.rotary_table(64, 16, scaling="linear", factor=4.0, device="cpu")
    assert np.array_equal(linear[::4].numpy(), plain[:16].numpy())
    base = kv.rotary_table(2, 16, scaling="base", factor=4.0, device="cpu").double().numpy()
    want = kv.rotary_table(2, 16, device="cpu").double().numpy()
    angle, slow = np.arctan2(base[1, 8:], base[1, :8]), np.arctan2(want[1, 8:], want[1, :8])
    assert np.isclose(angle[0], slow[0], rtol=1e-6) and np.isclose(angle[7] * 4, slow[7], rtol=1e-4)
    ramp = kv.rotary_table(2, 16, scaling="ramp", factor=4.0, original=2048, device="cpu")
    ramp = ramp.double().numpy()
    size = 0.1 * math.log(4.0) + 1
    assert np.allclose(np.hypot(ramp[1, :8], ramp[1, 8:]), size, rtol=1e-6)
    ratio = np.arctan2(ramp[1, 8:], ramp[1, :8]) / slow
    assert np.isclose(ratio[0], 1, rtol=1e-6) and np.isclose(ratio[7], 0.25, rtol=1e-4)
    assert (np.diff(ratio) <= 1e-6).all()


def test_rotary_table_refusals():
    from retrieve_amd import kv

    for wrong in ({"rot": 7}, {"rot": 0}, {"factor": 0.5}, {"scaling": "other"},
                  {"scaling": "ramp", "factor": 2.0}, {"scaling": "base", "rot": 2}):
        with pytest.raises(ValueError):
            kv.rotary_table(4, **{"rot": 8, "device": "cpu", **wrong})


def test_pages_are_reserved_and_freed():
    from retrieve_amd import kv

    c = kv.PagedCache(pages=10, heads=2, dim=64, page=16, sequences=3, max_pages=6, device="cpu")
    c.reserve(0, 17)
    c.reserve(1, 16)
    c.reserve(0, 32)
    table = c.page_table.numpy()
    assert (table >= 0).sum(1).tolist() == [2, 1, 0]
    assert len(set(table[table >= 0])) == 3
    c.reserve(2, 96)
    with pytest.raises(RuntimeError, match="free"):
        c.reserve(1, 40)
    with pytest.raises(ValueError, match="at most 6"):
        c.reserve(0, 97)
    c.free(2)
    assert (c.page_table[2] == -1).all()
    c.reserve(1, 40)
    assert sorted(c._free + sum(c._held, [])) == list(range(10))
    for error, wrong in ((ValueError, {"page": 20}), (TypeError, {"dim": 80})):
        with pytest.raises(error):
            kv.PagedCache(**{"pages": 4, "heads": 1, "dim": 64, "device": "cpu", **wrong})


def test_schemas_and_fakes():
    """Three ops of a namespace of their own; ``append`` says which arguments it writes; shapes come
    from the fakes without a GPU."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    import retrieve_amd.kv  # noqa: F401

    names = {s.name.removeprefix("retrieve_kv::"): s for s in torch._C._jit_get_all_schemas()
             if s.name.startswith("retrieve_kv::")}
    assert sorted(names) == ["append", "block_attention", "select_blocks"]
    written = [a.name for a in names["append"].arguments if a.alias_info and a.alias_info.is_write]
    assert written == ["k_cache", "v_cache", "bounds", "bound_scales"]
    assert not names["select_blocks"].is_mutable and not names["block_attention"].is_mutable
    ops = torch.ops.retrieve_kv
    with FakeTensorMode():
        q = torch.empty((5, 8, 64), dtype=torch.bfloat16)
        i = torch.empty((5,), dtype=torch.int32)
        tab = torch.empty((2, 4), dtype=torch.int32)
        cache = torch.empty((9, 2, 16, 64), dtype=torch.bfloat16)
        b, s = torch.empty((9, 2, 128), dtype=torch.int8), torch.empty((9, 2))
        assert ops.append(q, q[:, :2], q[:, :2], None, i, i, tab, cache, cache, b, s).shape == q.shape
        blocks = ops.select_blocks(q, b, s, i, i, tab, 16, 3)
        assert blocks.shape == (5, 2, 3) and blocks.dtype == torch.int32
        out, lse = ops.block_attention(q, cache, cache, blocks, i, i, tab)
        assert out.shape == q.shape and lse.shape == (5, 8) and lse.dtype == torch.float32


def test_cpu_tensors_are_refused():
    import torch

    from retrieve_amd import kv

    c = kv.PagedCache(pages=4, heads=1, dim=64, page=16, device="cpu")
    q = torch.zeros((1, 1, 64), dtype=torch.bfloat16)
    i = torch.zeros((1,), dtype=torch.int32)
    for call in (lambda: c.append(q, q, q, None, i, i), lambda: c.select(q, i, i, 2),
                 lambda: c.attend(q, i, i, 2)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_argument_errors_need_no_gpu():
    import torch  # noqa: F401

    from retrieve_amd import _native as nat

    lib = nat.lib()

    def select(t=1, heads=4, heads_kv=2, d=64, dtype=0, page=16, count=4, sink=1, recent=1):
        return lib.rt_kv_select(None, 0, 0, t, heads, heads_kv, d, dtype, None, None, 0, page, None,
                                None, None, 0, 0, count, sink, recent, None, None, 0, None)

    for status, how, word in [(1, {}, b"null"), (1, {"heads": 3}, b"multiple"), (2, {"d": 72}, b"channels"),
                              (2, {"dtype": 2}, b"dtype"), (1, {"page": 48}, b"page"),
                              (1, {"count": 2000}, b"count"), (1, {"recent": 0}, b"recent"),
                              (1, {"sink": 4}, b"fit"), (1, {"t": -1}, b"tokens"),
                              (1, {"t": 2**31}, b"tokens"), (1, {"heads_kv": 0}, b"multiple")]:
        assert select(**how) == status and word in lib.rt_last_error(), how
    assert select(t=0) == 0
    st = lib.rt_kv_attention(None, 0, 0, 1, 4, 2, 64, 0, None, None, 0, 16, None, 3, None, None, None,
                             0, 0, 1.0, None, None, None, 0, None)
    assert st == 1 and b"null" in lib.rt_last_error()
    st = lib.rt_kv_append(None, 0, 0, None, 0, 0, None, 0, 0, 1, 4, 2, 64, 0, None, 0, 65, 0, None, None,
                          None, 0, 0, None, None, 0, 16, None, None, None, None)
    assert st == 1 and b"rotated part" in lib.rt_last_error()


# --- on the GPU ---------------------------------------------------------------------------------


def _layer(dev, kind="bf16", steps=70, heads=8, heads_kv=2, d=64, page=16):
    """A cache of two sequences filled by a prompt, then single tokens: the layer's inputs."""
    from retrieve_amd import kv

    import torch

    cache = kv.PagedCache(pages=80, heads=heads_kv, dim=d, page=page, sequences=2, max_pages=40,
                          dtype=getattr(torch, {"bf16": "bfloat16", "fp16": "float16"}[kind]),
                          device=dev)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    cache.bound_scales.fill_(float("nan"))
    lens = [260, 131]
    x = [normal16(200 + i, (n + steps, heads + 2 * heads_kv, d), kind) for i, n in enumerate(lens)]
    return cache, lens, x, kv.rotary_table(400, d, device=dev)


@pytest.mark.gpu
def test_prompt_then_tokens(dev):
    """Prompt, then decode steps, each step held to the oracle on the oracle's own cache: chosen
    blocks equal, outputs within the attention's tolerance, over pages that start as NaN."""
    from tests.test_kv_attention import _check

    kind = "bf16"
    cache, lens, x, cs = _layer(dev)
    table = cs.cpu().numpy()
    mirror = [np.zeros(cache.k.shape, np.float32), np.zeros(cache.v.shape, np.float32),
              np.zeros(cache.bounds.shape, np.int8), np.zeros(cache.bound_scales.shape, np.float32)]
    at = [0, 0]
    for step in [lens] + [[1, 1]] * 40 + [[17, 0], [0, 13]]:
        rows, pos, seq = [], [], []
        for s, n in enumerate(step):
            cache.reserve(s, at[s] + n)
            rows.append(x[s][at[s]:at[s] + n])
            pos += range(at[s], at[s] + n)
            seq += [s] * n
            at[s] += n
        rows, pos, seq = np.concatenate(rows), np.array(pos, np.int32), np.array(seq, np.int32)
        tab = back(cache.page_table)
        g = to(dev, rows, kind)
        q = cache.append(g[:, :8], g[:, 8:10], g[:, 10:], cs, to(dev, pos), to(dev, seq))
        want_q = okv.append(rows[:, :8], rows[:, 8:10], rows[:, 10:], table, pos, seq, tab, *mirror, kind)
        assert np.array_equal(back(q), want_q)
        if len(pos) > 100:
            continue
        blocks = cache.select(q, to(dev, pos), to(dev, seq), 6, 1, 2)
        want = okv.select(want_q, mirror[2], mirror[3], pos, seq, tab, 16, 6, 1, 2)
        assert np.array_equal(back(blocks), want)
        got = cache.attend(q, to(dev, pos), to(dev, seq), 6, 1, 2)
        _check([back(y) for y in got], kind, want_q, mirror[0], mirror[1], want, pos, seq, tab)


@pytest.mark.gpu
def test_every_block_kept_is_full_attention(dev):
    """With as many places as blocks the layer is plain causal attention."""
    cache, lens, x, cs = _layer(dev, "fp16", 0)
    from tests.test_kv_attention import _check

    for s, n in enumerate(lens):
        cache.reserve(s, n)
    rows = np.concatenate(x)
    pos = np.concatenate([np.arange(n) for n in lens]).astype(np.int32)
    seq = np.repeat([0, 1], lens).astype(np.int32)
    g = to(dev, rows, "fp16")
    q = cache.append(g[:, :8], g[:, 8:10], g[:, 10:], cs, to(dev, pos), to(dev, seq))
    out, lse = cache.attend(q, to(dev, pos), to(dev, seq), 40)
    pick = np.r_[0:5, 250:260, 260, 300, 390]
    every = np.broadcast_to(np.arange(17, dtype=np.int32), (len(pick), 2, 17))
    kc, vc = np.nan_to_num(back(cache.k)), np.nan_to_num(back(cache.v))
    _check((back(out)[pick], back(lse)[pick]), "fp16", back(q)[pick], kc, vc, every, pos[pick],
           seq[pick], back(cache.page_table))


@pytest.mark.gpu
@pytest.mark.parametrize("sequences,blocks", [(1, 300), (2, 12)])
def test_graph_replays(dev, sequences, blocks):
    """A captured decode step, replayed with new inputs and positions between eager work, gives the
    eager step's results every time (the split forms' scratch among them)."""
    import torch

    from retrieve_amd import kv

    page, heads, heads_kv, d = 16, 8, 2, 64
    pages = sequences * (blocks + 2)
    cache = kv.PagedCache(pages, heads_kv, d, page, sequences, blocks + 2, device=dev)
    cs = kv.rotary_table(page * (blocks + 2), d, device=dev)
    for s in range(sequences):
        cache.reserve(s, page * (blocks + 2))
    g = torch.Generator(device=dev).manual_seed(3)
    n = page * blocks - 3
    for s in range(sequences):
        x = torch.randn((n, 12, d), generator=g, device=dev).to(torch.bfloat16)
        pos = torch.arange(n, dtype=torch.int32, device=dev)
        cache.append(x[:, :8], x[:, 8:10], x[:, 10:], cs, pos, torch.full_like(pos, s))
    seq = torch.arange(sequences, dtype=torch.int32, device=dev)
    x = torch.zeros((sequences, 12, d), dtype=torch.bfloat16, device=dev)
    pos = torch.full((sequences,), n, dtype=torch.int32, device=dev)

    def step():
        q = cache.append(x[:, :8], x[:, 8:10], x[:, 10:], cs, pos, seq)
        return (q, *cache.attend(q, pos, seq, 8, 1, 2))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(5):
        x.copy_(torch.randn(x.shape, generator=g, device=dev))
        pos.fill_(n + i)
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in held]
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


@pytest.mark.gpu
def test_on_another_stream(dev):
    """Calls enqueue on the current stream: a step behind a long product on a side stream."""
    import torch

    cache, lens, x, cs = _layer(dev, "bf16", 0)
    cache.reserve(0, lens[0])
    rows, pos = to(dev, x[0], "bf16"), torch.arange(lens[0], dtype=torch.int32, device=dev)
    seq = torch.zeros_like(pos)

    def step(y):
        q = cache.append(y[:, :8], y[:, 8:10], y[:, 10:], cs, pos, seq)
        return q, *cache.attend(q, pos, seq, 5)

    want = step(rows)
    late = torch.zeros_like(rows)
    big = torch.randn((4096, 4096), device=dev)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            big = big @ big * 1e-3
        late.copy_(rows)
        got = step(late)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_opcheck(dev):
    import torch

    cache, lens, x, cs = _layer(dev, "bf16", 0)
    cache.reserve(0, lens[0])
    for y in (cache.k, cache.v, cache.bound_scales):
        y.zero_()
    cache.bounds.zero_()
    rows, pos = to(dev, x[0], "bf16"), torch.arange(lens[0], dtype=torch.int32, device=dev)
    seq = torch.zeros_like(pos)
    ops = torch.ops.retrieve_kv
    how = ("test_schema", "test_faketensor")
    q, k, v = rows[:, :8].contiguous(), rows[:, 8:10].contiguous(), rows[:, 10:].contiguous()
    torch.library.opcheck(ops.append.default, (
        q, k, v, cs, pos, seq, cache.page_table, cache.k, cache.v, cache.bounds,
        cache.bound_scales), test_utils=how)
    cache.append(q, k, v, cs, pos, seq)
    torch.library.opcheck(ops.select_blocks.default, (
        q, cache.bounds, cache.bound_scales, pos, seq, cache.page_table, 16, 5), test_utils=how)
    blocks = cache.select(q, pos, seq, 5)
    torch.library.opcheck(ops.block_attention.default, (
        q, cache.k, cache.v, blocks, pos, seq, cache.page_table), test_utils=how)


@pytest.mark.gpu
def test_recall_of_the_heaviest_blocks(dev):
    """On keys with structure (each block around its own centre) the chosen blocks hold nearly all
    the attention's weight: log-sums over 16 of 128 blocks close to those over all."""
    import torch

    from retrieve_amd import kv

    g = rng(300)
    blocks, page, d = 128, 16, 64
    centre = g.standard_normal((blocks, 1, 1, d)) * 1.5
    keys = okv.round16((centre + 0.5 * g.standard_normal((blocks, page, 1, d))).reshape(-1, 1, d), "bf16")
    cache = kv.PagedCache(blocks, 1, d, page, 1, blocks, device=dev)
    cache.reserve(0, blocks * page)
    pos = torch.arange(blocks * page, dtype=torch.int32, device=dev)
    seq = torch.zeros_like(pos)
    k = to(dev, keys, "bf16")
    cache.append(k, k, k, None, pos, seq)
    q = to(dev, okv.round16(2.0 * centre[5:25, 0] + g.standard_normal((20, 1, d)), "bf16"), "bf16")
    at, one = torch.full((20,), blocks * page - 1, dtype=torch.int32, device=dev), seq[:20]
    _, few = cache.attend(q, at, one, 16)
    _, every = cache.attend(q, at, one, blocks)
    assert float((every - few).max()) < 0.05
