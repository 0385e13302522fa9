"""The 8-bit cache's functions as they are called: schemas, refusals (none needs a GPU), calls that
are recorded or transformed."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kv_int8 as o8
from tests.kv_cases import back, layout, normal16, table, to
from tests.kv_int8_cases import on_gpu

OPS = {"append_int8": "append", "read_int8": "read", "block_attention_int8": "block_attention"}
NAMES = tuple(OPS)
LIVE = {"append_int8": 0, "read_int8": 4, "block_attention_int8": 0}  # an input of 16 bits
CACHE = {"append_int8": 7, "read_int8": 0, "block_attention_int8": 1}  # where the cache begins


def _inputs(dev, seed=1, page=16, heads=4, heads_kv=2, d=64):
    """One call's arguments of each function, over a cache of three sequences."""
    pos, seq, tab, pages = layout(seed, page, [(40, 1), (3, 20), (100, 2)])
    c = o8.Cache(seed + 1, pages, heads_kv, page, d, 3, "bf16")
    for i in (tab[0, 2], tab[1, 1], tab[2, 6]):
        c.ks[i] = c.vs[i] = 0.0
    t = len(pos)
    qkv = to(dev, normal16(seed + 2, (t, heads + 2 * heads_kv, d), "bf16"), "bf16")
    q = qkv[:, :heads].contiguous()
    cache, bounds = on_gpu(dev, c)
    blocks = to(dev, np.tile(np.array([2, 0, 1], np.int32), (t, heads_kv, 1)))
    where = [to(dev, x) for x in (pos, seq, tab)]
    return {"append_int8": (q, qkv[:, heads:heads + heads_kv], qkv[:, heads + heads_kv:],
                            to(dev, table(200, d)), *where, *cache, *bounds),
            "read_int8": (*cache, *where),
            "block_attention_int8": (q, *cache, blocks, *where)}


def _with(name, args, x):
    i = LIVE[name]
    return (*args[:i], x, *args[i + 1:])


def test_schemas_and_fakes():
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    import retrieve_amd.kv  # noqa: F401

    names = {s.name.removeprefix("retrieve_kv_int8::"): s for s in torch._C._jit_get_all_schemas()
             if s.name.startswith("retrieve_kv_int8::")}
    assert sorted(names) == ["append", "block_attention", "read"]
    written = [a.name for a in names["append"].arguments if a.alias_info and a.alias_info.is_write]
    assert written == ["k_codes", "v_codes", "k_scales", "v_scales", "k_tail", "v_tail", "bounds",
                       "bound_scales"]
    assert not names["read"].is_mutable and not names["block_attention"].is_mutable
    ops = torch.ops.retrieve_kv_int8
    with FakeTensorMode():
        q = torch.empty((5, 8, 64), dtype=torch.float16)
        i = torch.empty((5,), dtype=torch.int32)
        tab = torch.empty((3, 4), dtype=torch.int32)
        scales = torch.empty((9, 2))
        cache = (torch.empty((9, 2, 16, 64), dtype=torch.int8),
                 torch.empty((9, 2, 64, 16), dtype=torch.int8), scales, scales,
                 torch.empty((3, 2, 16, 64), dtype=torch.float16),
                 torch.empty((3, 2, 64, 16), dtype=torch.float16))
        bounds = torch.empty((9, 2, 128), dtype=torch.int8)
        got = ops.append(q, q[:, :2], q[:, :2], None, i, i, tab, *cache, bounds, scales)
        assert got.shape == q.shape and got.dtype == q.dtype
        k, v = ops.read(*cache, i, i, tab)
        assert k.shape == v.shape == (5, 2, 64) and k.dtype == v.dtype == torch.float16
        blocks = torch.empty((5, 2, 3), dtype=torch.int32)
        out, lse = ops.block_attention(q, *cache, blocks, i, i, tab)
        assert out.shape == q.shape and lse.shape == (5, 8) and lse.dtype == torch.float32


@pytest.mark.parametrize("name", NAMES)
def test_cache_refusals(name):
    """Shapes, dtypes and layouts that the kernels do not read, then CPU tensors."""
    import torch

    from retrieve_amd import kv

    args, at = _inputs("cpu")[name], CACHE[name]
    k, v, ks, vs, kt, vt = range(at, at + 6)

    def turned(x):
        return x.transpose(-1, -2).contiguous().transpose(-1, -2)

    def refused(error, word=None, **change):
        new = list(args)
        for i, f in change.items():
            i = int(i[1:])
            new[i] = f(new[i])
        with pytest.raises(error, match=word):
            getattr(kv, name)(*new)

    for i, how, error in [
            (k, lambda x: x[0], ValueError), (k, lambda x: x[:-1], ValueError),
            (k, lambda x: x.to(torch.uint8), TypeError), (k, turned, ValueError),
            (v, lambda x: x.transpose(2, 3).contiguous(), ValueError),
            (v, lambda x: x.float(), TypeError), (v, turned, ValueError),
            (ks, lambda x: x[:, :1], ValueError), (ks, lambda x: x.double(), TypeError),
            (ks, lambda x: x.t().contiguous().t(), ValueError),
            (vs, lambda x: x[:-1], ValueError), (vs, lambda x: x.half(), TypeError),
            (kt, lambda x: x[:-1], ValueError), (kt, turned, ValueError),
            (kt, lambda x: x.half(), TypeError), (kt, lambda x: x.float(), TypeError),
            (vt, lambda x: x.transpose(2, 3).contiguous(), ValueError),
            (vt, lambda x: x.half(), TypeError), (vt, lambda x: x[:, :1], ValueError)]:
        refused(error, **{f"_{i}": how})
    refused(TypeError, **{f"_{kt}": lambda x: x.float(), f"_{vt}": lambda x: x.float()})
    where = 4 if name == "append_int8" else len(args) - 3
    refused(TypeError, "int32", **{f"_{where}": lambda x: x.long()})
    refused(ValueError, None, **{f"_{where + 1}": lambda x: x[:-1]})
    refused(ValueError, "contiguous", **{f"_{where + 2}": lambda x: x.t().contiguous().t()})
    # (one open block for each row of the table)
    refused(ValueError, "page_table", **{f"_{where + 2}": lambda x: x[:2]})
    refused(ValueError, "GPU", **{})
    # sizes that no kernel has
    for size, error in [(dict(d=80), TypeError), (dict(page=8), ValueError),
                        (dict(heads=3), ValueError)]:
        if name == "read_int8" and "heads" in size:
            continue
        with pytest.raises(error):
            getattr(kv, name)(*_inputs("cpu", **size)[name])


def test_more_refusals():
    import torch

    from retrieve_amd import kv

    every = _inputs("cpu")
    q, k, v, cs, pos, seq, tab, *rest = every["append_int8"]
    for error, new in [(TypeError, (q.half(), k, v)), (TypeError, (q, k.half(), v)),
                       (ValueError, (q[..., :32], k, v)), (ValueError, (q, k[:, :1], v)),
                       (ValueError, (q, k, v[:-1])), (ValueError, (q[:-1], k[:-1], v[:-1])),
                       (ValueError, (q[0], k, v))]:
        with pytest.raises(error):
            kv.append_int8(*new, cs, pos, seq, tab, *rest)
    w = torch.ones(64, dtype=torch.bfloat16)
    for error, how in [(TypeError, dict(cos_sin=cs.half())), (ValueError, dict(cos_sin=cs[:, :63])),
                       (ValueError, dict(q_weight=w[:32])), (TypeError, dict(k_weight=w.half())),
                       (TypeError, dict(q_weight=w, k_weight=w.float())),
                       (ValueError, dict(q_weight=w, eps=-1.0)),
                       (ValueError, dict(q_weight=w, eps=float("nan")))]:
        with pytest.raises(error):
            kv.append_int8(q, k, v, how.pop("cos_sin", cs), pos, seq, tab, *rest, **how)
    for error, bounds in [(ValueError, (rest[6][..., :64], rest[7])),
                          (TypeError, (rest[6].float(), rest[7])),
                          (TypeError, (rest[6], rest[7].half())), (ValueError, (rest[6], rest[7][:1]))]:
        with pytest.raises(error):
            kv.append_int8(q, k, v, cs, pos, seq, tab, *rest[:6], *bounds)
    args = every["block_attention_int8"]
    for error, blocks in [(ValueError, args[7][:-1]), (ValueError, args[7][:, :1]),
                          (TypeError, args[7].long())]:
        with pytest.raises(error):
            kv.block_attention_int8(*args[:7], blocks, *args[8:])
    with pytest.raises(ValueError, match="sequences"):
        kv.block_attention_int8(*args, sequences=0)


def test_int8_paged_cache_on_the_host():
    import torch

    from retrieve_amd import kv

    c = kv.Int8PagedCache(pages=10, heads=2, dim=64, page=16, sequences=3, max_pages=6,
                          dtype=torch.float16, device="cpu")
    assert c.k_codes.shape == (10, 2, 16, 64) and c.v_codes.shape == (10, 2, 64, 16)
    assert c.k_tail.shape == (3, 2, 16, 64) and c.v_tail.dtype == torch.float16
    assert not c.k_scales.any() and not c.v_scales.any()
    c.reserve(0, 17)
    assert (c.page_table >= 0).sum(1).tolist() == [2, 0, 0]
    c.free(0)
    assert sorted(c._free) == list(range(10))
    for error, wrong in ((ValueError, {"page": 20}), (TypeError, {"dim": 80}),
                         (TypeError, {"dtype": torch.float32})):
        with pytest.raises(error):
            kv.Int8PagedCache(**{"pages": 4, "heads": 1, "dim": 64, "device": "cpu", **wrong})
    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    i = torch.zeros((1,), dtype=torch.int32)
    for call in (lambda: c.append(q, q, q, None, i, i), lambda: c.attend(q, i, i, 2),
                 lambda: c.read(i, i)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_argument_errors_need_no_gpu():
    from retrieve_amd import _native as nat

    lib = nat.lib()

    def append(t=1, heads=4, heads_kv=2, d=64, dtype=0, page=16, pages=3, rot=0, eps=1e-6, length=0,
               weight=None, b=1):
        return lib.rt_kv_append_int8(None, 0, 0, None, 0, 0, None, 0, 0, t, heads, heads_kv, d, dtype,
                                     weight, None, 0, eps, None, length, rot, 0, None, None, None, b,
                                     4, None, None, None, None, None, None, pages, page, None, None,
                                     None, None)

    def read(t=1, heads_kv=2, d=64, dtype=0, page=16, pages=3, b=1):
        return lib.rt_kv_read_int8(None, None, None, None, None, None, t, heads_kv, d, dtype, pages,
                                   page, None, None, None, b, 4, None, None, None)

    def attend(t=1, heads=4, heads_kv=2, d=64, dtype=0, page=16, pages=3, count=3, scale=1.0,
               sequences=1, b=1):
        return lib.rt_kv_attention_int8(None, 0, 0, t, heads, heads_kv, d, dtype, None, None, None,
                                        None, None, None, pages, page, None, count, None, None, None,
                                        b, 4, scale, sequences, None, None, None, 0, None)

    for call in (append, read, attend):
        for status, how, word in [(1, {}, b"null"), (2, {"d": 72}, b"channels"),
                                  (2, {"dtype": 2}, b"dtype"), (1, {"page": 48}, b"page"),
                                  (1, {"t": -1}, b"tokens"), (1, {"t": 2**31}, b"tokens"),
                                  (1, {"heads_kv": 0}, b"head")]:
            assert call(**how) == status and word in lib.rt_last_error(), (call, how)
        assert call(t=0) == 0
    assert append(heads=3) == 1 and b"multiple" in lib.rt_last_error()
    assert attend(heads=3) == 1 and b"multiple" in lib.rt_last_error()
    assert append(rot=65) == 1 and b"rotated part" in lib.rt_last_error()
    assert append(weight=64, eps=-1.0) == 1 and b"eps" in lib.rt_last_error()
    assert attend(scale=float("inf")) == 1 and b"scale" in lib.rt_last_error()
    assert lib.rt_kv_attention_int8_workspace(-1, 4, 2, 64, 16, 3) == 0
    assert lib.rt_kv_attention_int8_workspace(1, 4, 0, 64, 16, 3) == 0


# --- recorded and transformed -------------------------------------------------------------------


@pytest.fixture
def straight(monkeypatch):
    """The functions that were taken straight to their kernels."""
    from retrieve_amd import kv

    seen = []
    for name, attr in zip(NAMES, ("_append_int8", "_read_int8", "_attention_int8")):
        monkeypatch.setattr(kv, attr, lambda *a, name=name, **k: seen.append(name))
    return seen


@pytest.mark.parametrize("name", NAMES)
def test_plain_calls_go_straight(straight, name):
    import torch

    from retrieve_amd import kv

    getattr(kv, name)(*_inputs("cpu")[name])
    with torch.no_grad():
        getattr(kv, name)(*_inputs("cpu")[name])
    with torch.inference_mode():
        getattr(kv, name)(*_inputs("cpu")[name])
    assert straight == [name] * 3


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("how", ["make_fx", "jit", "mode", "vmap", "grad", "requires_grad"])
def test_recorded_calls_reach_the_op(straight, name, how):
    """(On the CPU the op itself refuses: that it was reached is what is looked at.)"""
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    from retrieve_amd import kv

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    if (name, how) == ("append_int8", "vmap"):
        pytest.skip("an op that writes its arguments is not batched")
    args = _inputs("cpu")[name]
    x = args[LIVE[name]]

    def call(x):
        return getattr(kv, name)(*_with(name, args, x))

    with pytest.raises(ValueError, match="retrieve_kv ops run on the GPU only"):
        if how == "make_fx":
            make_fx(call)(x)
        elif how == "jit":
            torch.jit.trace(call, (x,), check_trace=False)
        elif how == "mode":
            with Mode():
                call(x)
        elif how == "vmap":
            torch.vmap(call)(x[None])
        elif how == "grad":
            torch.func.grad(call)(x)
        else:
            call(x.clone().requires_grad_())
    assert straight == []


@pytest.mark.parametrize("name", NAMES)
def test_the_graph_holds_the_op(name):
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx

    from retrieve_amd import kv

    args = _inputs("cpu")[name]
    graph = make_fx(lambda x: getattr(kv, name)(*_with(name, args, x)), tracing_mode="fake",
                    _allow_non_fake_inputs=True)(args[LIVE[name]])
    op = getattr(torch.ops.retrieve_kv_int8, OPS[name]).default
    assert [n.target for n in graph.graph.nodes if "retrieve_kv" in str(n.target)] == [op]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    import torch
    from torch.autograd import forward_ad

    from retrieve_amd import kv

    args = _inputs("cpu")[name]
    x = args[LIVE[name]]
    with forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
        getattr(kv, name)(*_with(name, args, forward_ad.make_dual(x, torch.ones_like(x))))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_recorded_graphs_run_the_kernels(dev, name):
    """A graph recorded on one input gives, on another, what an eager call gives, the cache that it
    writes among it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from retrieve_amd import kv

    args, other = _inputs(dev)[name], _inputs(dev, 11)[name][LIVE[name]]
    graph = make_fx(lambda x: getattr(kv, name)(*_with(name, args, x)))(args[LIVE[name]])
    results = []
    for call in (graph, lambda x: getattr(kv, name)(*_with(name, args, x))):
        if name == "append_int8":
            for x, y in zip(args[7:], _inputs(dev)[name][7:]):
                x.copy_(y)
        got = call(other)
        got = list(got) if isinstance(got, (tuple, list)) else [got]
        results.append([back(x) for x in got + (list(args[7:]) if name == "append_int8" else [])])
    assert len(results[0]) == len(results[1])
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(*results))


@pytest.mark.gpu
def test_opcheck(dev):
    import torch

    how = ("test_schema", "test_faketensor")
    for name, args in _inputs(dev).items():
        torch.library.opcheck(getattr(torch.ops.retrieve_kv_int8, OPS[name]).default, args,
                              test_utils=how)


@pytest.mark.gpu
def test_a_backward_pass_warns(dev):
    from retrieve_amd import kv

    args = _inputs(dev)["block_attention_int8"]
    q = args[0].clone().requires_grad_()
    out, _ = kv.block_attention_int8(*_with("block_attention_int8", args, q))
    assert out.requires_grad
    assert (back(out.detach()) == back(kv.block_attention_int8(*args)[0])).all()
    with pytest.warns(UserWarning, match="retrieve_kv_int8::block_attention"):
        out.float().sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_calls_without_tokens(dev, name):
    from retrieve_amd import kv

    args = list(_inputs(dev)[name])
    at = 4 if name == "append_int8" else len(args) - 3
    for i in {"append_int8": (0, 1, 2), "read_int8": (),
              "block_attention_int8": (0, 7)}[name] + (at, at + 1):
        args[i] = args[i][:0]
    before = [x.clone() for x in args]
    got = getattr(kv, name)(*args)
    for x in got if isinstance(got, tuple) else (got,):
        assert x.shape[0] == 0
    assert all(np.array_equal(back(a), back(b)) for a, b in zip(args, before))


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("heads,heads_kv", [(1, 1), (32, 8), (20, 20), (40, 1)])
def test_the_workspace_holds_every_form(heads, heads_kv, d):
    """Rows that are split have their parts in the workspace, and the calls of one size have one
    workspace, however many sequences they name: 16 columns of ``d`` sums, a maximum and a sum for
    each part, of enough parts for 512 workgroups or as many as the lists have units for."""
    from retrieve_amd import _native as nat

    need = nat.lib().rt_kv_attention_int8_workspace
    tiles = -(-(heads // heads_kv) // 16)
    for tokens in (1, 2, 15, 16, 63, 64, 65, 200, 511, 512, 2000):
        for count, page in ((1, 16), (16, 64), (96, 16), (600, 128)):
            rows = tokens * heads_kv * tiles
            parts = max(1, min(-(-512 // rows), -(-count * page // 256)))
            want = 4 * rows * parts * 16 * (d + 2) if parts > 1 else 0
            assert need(tokens, heads, heads_kv, d, page, count) == want, (tokens, count, page)
