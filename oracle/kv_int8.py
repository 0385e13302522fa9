"""The paged cache in 8 bits in numpy (test infrastructure; see ``oracle/__init__``): token by token,
as the documentation states it. Values of 16-bit types are float32 arrays, as in ``oracle.kv``."""

from __future__ import annotations

import numpy as np

from oracle import kv as okv


def norm(x, weight, eps):
    """Heads ``[..., D]`` normed: the sum in 64 bits, each step behind it rounded to float32."""
    if weight is None:
        return x
    r = 1.0 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + eps)
    with np.errstate(invalid="ignore", over="ignore"):
        return (x * r.astype(np.float32)) * weight.astype(np.float32)


def norm64(x, weight, eps):
    x = x.astype(np.float64)
    if weight is None:
        return x
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight


def codes_of(block):
    """int8 codes of one head's block (any shape) and the scale."""
    a = np.abs(block.astype(np.float64))
    top = max(np.where(np.isfinite(a), a, 0.0).max(), np.float64(np.float32(1e-8)))
    x = np.clip(np.nan_to_num(block.astype(np.float64), nan=0.0, posinf=top, neginf=-top), -top, top)
    return np.rint(127 * x / top).astype(np.int8), np.float32(top) / np.float32(127)


class Cache:
    """What an 8-bit cache holds; ``open_of[b]`` is how many rows of sequence ``b``'s open block count
    (None where the calls so far do not say)."""

    def __init__(self, seed, pages, heads_kv, page, dim, sequences, kind):
        g = np.random.Generator(np.random.PCG64(seed))
        self.kind, self.page = kind, page
        self.k = g.integers(-127, 128, (pages, heads_kv, page, dim), dtype=np.int8)
        self.v = g.integers(-127, 128, (pages, heads_kv, dim, page), dtype=np.int8)
        self.ks = g.random((pages, heads_kv), dtype=np.float32) * np.float32(0.05) + np.float32(0.01)
        self.vs = g.random((pages, heads_kv), dtype=np.float32) * np.float32(0.05) + np.float32(0.01)
        self.kt = okv.round16(g.standard_normal((sequences, heads_kv, page, dim), np.float32), kind)
        self.vt = okv.round16(g.standard_normal((sequences, heads_kv, dim, page), np.float32), kind)
        self.bounds = g.integers(-127, 128, (pages, heads_kv, 2 * dim), dtype=np.int8)
        self.bound_scales = g.random((pages, heads_kv), dtype=np.float32)
        self.open_of = [None] * sequences

    def copy(self):
        other = object.__new__(Cache)
        other.__dict__ = {n: x.copy() if isinstance(x, np.ndarray) else
                          list(x) if isinstance(x, list) else x for n, x in self.__dict__.items()}
        return other

    def held(self, i):
        """Page ``i``'s keys and values in 16 bits, ``[Hkv, page, D]`` and ``[Hkv, D, page]``."""
        return (okv.round16(self.k[i] * self.ks[i][:, None, None], self.kind),
                okv.round16(self.v[i] * self.vs[i][:, None, None], self.kind))

    def append(self, q, k, v, cos_sin, positions, seq_ids, page_table, interleaved=False,
               q_weight=None, k_weight=None, eps=1e-6):
        out = np.zeros(q.shape, np.float32)
        pages, page = len(self.k), self.page
        for t, at in enumerate(okv.place(positions, seq_ids, page_table, pages, page)):
            if at is None or (cos_sin is not None and at[0] >= len(cos_sin)):
                continue
            i, s = okv._page(at, at[1], pages), int(seq_ids[t])
            if i < 0:
                continue
            row = np.zeros((1, 0), np.float32) if cos_sin is None else cos_sin[at[0]][None]
            out[t] = okv.round16(okv.rotate(norm(q[t][None], q_weight, eps), row, interleaved),
                                 self.kind)[0]
            slot = at[0] % page
            if slot and self.ks[i, 0] > 0:  # (full so far: cut back)
                self.kt[s], self.vt[s] = self.held(i)
            self.ks[i] = self.vs[i] = 0.0
            self.kt[s, :, slot] = okv.round16(
                okv.rotate(norm(k[t][None], k_weight, eps), row, interleaved), self.kind)[0]
            self.vt[s, :, :, slot] = v[t]
            self.open_of[s] = slot + 1
            if slot == page - 1:
                self.open_of[s] = 0
                for h in range(self.k.shape[1]):
                    self.bounds[i, h], self.bound_scales[i, h] = okv.bounds_of(self.kt[s, h])
                    self.k[i, h], self.ks[i, h] = codes_of(self.kt[s, h])
                    self.v[i, h], self.vs[i, h] = codes_of(self.vt[s, h])
        return out

    def read(self, positions, seq_ids, page_table):
        heads, dim = self.k.shape[1], self.k.shape[3]
        k = np.zeros((len(positions), heads, dim), np.float32)
        v = np.zeros_like(k)
        for t, at in enumerate(okv.place(positions, seq_ids, page_table, len(self.k), self.page)):
            i = -1 if at is None else okv._page(at, at[1], len(self.k))
            if i < 0:
                continue
            slot, s = at[0] % self.page, int(seq_ids[t])
            kb, vb = self.held(i) if self.ks[i, 0] > 0 else (self.kt[s], self.vt[s])
            k[t], v[t] = kb[:, slot], vb[:, :, slot]
        return k, v

    def attention(self, q, blocks, positions, seq_ids, page_table, scale):
        """As ``oracle.kv.attention``, over what the codes stand for; ``spread`` in two parts, of the
        codes and of the open block."""
        pages = len(self.k)
        k = np.concatenate([self.k * self.ks.astype(np.float64)[..., None, None],
                            self.kt.astype(np.float64)])
        v = np.concatenate([self.v * self.vs.astype(np.float64)[..., None, None],
                            self.vt.astype(np.float64)]).swapaxes(2, 3)
        # (a block that is not full is its sequence's open one, or nothing)
        table = np.where((page_table >= 0) & (page_table < pages), page_table, -1)
        unfilled = (table >= 0) & (self.ks[:, 0][np.maximum(table, 0)] == 0)
        table = np.where(unfilled, pages + np.arange(len(table))[:, None], table).astype(np.int32)
        blocks = blocks.copy()
        for t, at in enumerate(okv.place(positions, seq_ids, page_table, pages, self.page)):
            if at is not None:
                gone = np.zeros(table.shape[1], bool)
                gone[:at[1]] = unfilled[int(seq_ids[t]), :at[1]]
                b = blocks[t]
                inside = (b >= 0) & (b < table.shape[1])
                b[inside & gone[np.where(inside, b, 0)]] = -1
        return okv.attention(q, k, v, blocks, positions, seq_ids, table, scale)
