"""Inputs of the paged-cache tests: packed tokens of ragged sequences over a shuffled page pool, as
numpy arrays whose values the 16-bit types hold exactly."""

from __future__ import annotations

import numpy as np

from oracle import kv as okv
from tests.conftest import rng

KINDS = {"bf16": "bfloat16", "fp16": "float16"}


def layout(seed, page, had_new, spare=2, max_pages=None):
    """(positions, seq_ids, page_table, pages) of sequences with ``(tokens before, new tokens)``."""
    g = rng(seed)
    need = [-(-(h + n) // page) for h, n in had_new]
    pages = sum(need) + spare
    order = g.permutation(pages)
    table = np.full((len(had_new), max_pages or max(need, default=0)), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    pos = np.concatenate([np.arange(h, h + n) for h, n in had_new] or [[]]).astype(np.int32)
    seq = np.repeat(np.arange(len(had_new)), [n for _, n in had_new]).astype(np.int32)
    return pos, seq, table, pages


def normal16(seed, shape, kind, size=1.0):
    return okv.round16(rng(seed).standard_normal(shape, dtype=np.float32) * np.float32(size), kind)


def table(length, rot, seed=5):
    """Angles of a rotation (any numbers serve): ``[length, rot]`` cosines then sines."""
    freq = 100.0 ** -(np.arange(rot // 2) / max(1, rot // 2))
    angle = np.arange(length)[:, None] * freq
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


def to(dev, x, kind=None):
    import torch

    x = torch.from_numpy(np.ascontiguousarray(x))
    return x.to(dev) if kind is None else x.to(getattr(torch, KINDS[kind])).to(dev)


def back(x):
    import torch

    return (x.float() if x.dtype in (torch.bfloat16, torch.float16) else x).cpu().numpy()
