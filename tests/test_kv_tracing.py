"""The paged cache's functions where calls are recorded or transformed: the registered op is what is
seen, never the allocations around a launch."""

from __future__ import annotations

import numpy as np
import pytest

from tests.conftest import rng
from tests.kv_cases import back, layout, normal16, table, to

NAMES = ("append", "select_blocks", "block_attention")


def _inputs(dev, seed=1):
    """One call's arguments of each function, over a cache of three sequences."""
    pos, seq, tab, pages = layout(seed, 16, [(40, 1), (3, 20), (100, 2)])
    t = len(pos)
    qkv = to(dev, normal16(seed + 1, (t, 8, 64), "bf16"), "bf16")
    q = qkv[:, :4].contiguous()
    caches = [to(dev, normal16(seed + i, (pages, 2, 16, 64), "bf16"), "bf16") for i in (2, 3)]
    codes = to(dev, rng(seed + 4).integers(-127, 128, (pages, 2, 128), dtype="int8"))
    scales = to(dev, rng(seed + 5).random((pages, 2), dtype="float32"))
    blocks = to(dev, np.tile(np.array([2, 0, 1], np.int32), (t, 2, 1)))
    where = [to(dev, x) for x in (pos, seq, tab)]
    return {"append": (q, qkv[:, 4:6], qkv[:, 6:], to(dev, table(200, 64)), *where, *caches, codes,
                       scales),
            "select_blocks": (q, codes, scales, *where, 16, 4),
            "block_attention": (q, *caches, blocks, *where)}


@pytest.fixture
def straight(monkeypatch):
    """The functions that were taken straight to their kernels."""
    from retrieve_amd import kv

    seen = []
    for name, attr in zip(NAMES, ("_append", "_select", "_attention")):
        monkeypatch.setattr(kv, attr, lambda *a, name=name, **k: seen.append(name))
    return seen


def _first(args, x):
    return (x, *args[1:])


@pytest.mark.parametrize("name", NAMES)
def test_plain_calls_go_straight(straight, name):
    import torch

    from retrieve_amd import kv

    getattr(kv, name)(*_inputs("cpu")[name])
    with torch.no_grad(), torch.device("cpu"):
        getattr(kv, name)(*_inputs("cpu")[name])
    with torch.inference_mode():
        getattr(kv, name)(*_inputs("cpu")[name])
    assert straight == [name] * 3


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("how", ["make_fx", "pre_dispatch", "jit", "mode", "vmap", "grad",
                                 "requires_grad", "parameter"])
def test_recorded_calls_reach_the_op(straight, name, how):
    """(On the CPU the op itself refuses: that it was reached is what is looked at.)"""
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    from retrieve_amd import kv

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    if (name, how) == ("append", "vmap"):
        pytest.skip("an op that writes its arguments is not batched")
    args = _inputs("cpu")[name]

    def call(x):
        return getattr(kv, name)(*_first(args, x))

    with pytest.raises(ValueError, match="retrieve_kv ops run on the GPU only"):
        if how == "make_fx":
            make_fx(call)(args[0])
        elif how == "pre_dispatch":
            make_fx(call, pre_dispatch=True)(args[0])
        elif how == "jit":
            torch.jit.trace(call, (args[0],), check_trace=False)
        elif how == "mode":
            with Mode():
                call(args[0])
        elif how == "vmap":
            torch.vmap(call)(args[0][None])
        elif how == "grad":
            torch.func.grad(call)(args[0])
        elif how == "parameter":
            with torch.no_grad():
                call(torch.nn.Parameter(args[0]))
        else:
            call(args[0].clone().requires_grad_())
    assert straight == []


@pytest.mark.parametrize("name", NAMES)
def test_the_graph_holds_the_op(name):
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx

    from retrieve_amd import kv

    args = _inputs("cpu")[name]
    graph = make_fx(lambda x: getattr(kv, name)(*_first(args, x)), tracing_mode="fake",
                    _allow_non_fake_inputs=True)(args[0])
    op = getattr(torch.ops.retrieve_kv, name).default
    assert [n.target for n in graph.graph.nodes if "retrieve_kv" in str(n.target)] == [op]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    import torch
    from torch.autograd import forward_ad

    from retrieve_amd import kv

    args = _inputs("cpu")[name]
    with forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
        getattr(kv, name)(*_first(args, forward_ad.make_dual(args[0], torch.ones_like(args[0]))))
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda x: getattr(kv, name)(*_first(args, x)), (args[0],), (args[0],))


# --- on the GPU ---------------------------------------------------------------------------------


def _outputs(got):
    return [back(x) for x in (got if isinstance(got, tuple) else (got,))]


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("how", ["make_fx", "jit"])
def test_recorded_graphs_run_the_kernels(dev, name, how):
    """A graph recorded on some queries gives, on others, what an eager call gives, the caches that
    it writes among it."""
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx

    from retrieve_amd import kv

    args, other = _inputs(dev)[name], _inputs(dev, 11)[name][0]

    def call(x):
        return getattr(kv, name)(*_first(args, x))

    if how == "make_fx":
        graph = make_fx(call)(args[0])
        targets = [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]
        assert [t for t in targets if "retrieve_kv" in t or "empty" in t] == [
            f"retrieve_kv.{name}.default"]
    else:
        graph = torch.jit.trace(call, (args[0],), check_trace=False)
        assert [n.kind() for n in graph.graph.nodes() if "retrieve_kv" in n.kind()] == [
            f"retrieve_kv::{name}"]
    if name == "append":
        for x in args[7:]:
            x.zero_()
    got = _outputs(graph(other)) + ([back(x) for x in args[7:]] if name == "append" else [])
    if name == "append":
        for x in args[7:]:
            x.zero_()
    want = _outputs(call(other)) + ([back(x) for x in args[7:]] if name == "append" else [])
    assert len(got) == len(want) and all((a == b).all() for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_backward_pass_warns(dev):
    from retrieve_amd import kv

    args = _inputs(dev)["block_attention"]
    q = args[0].clone().requires_grad_()
    out, _ = kv.block_attention(*_first(args, q))
    assert out.requires_grad
    assert (back(out.detach()) == back(kv.block_attention(*args)[0])).all()
    with pytest.warns(UserWarning, match="retrieve_kv::block_attention"):
        out.float().sum().backward()
