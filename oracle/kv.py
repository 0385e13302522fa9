"""The paged cache's operators in numpy (test infrastructure; see ``oracle/__init__``).

Values of 16-bit types are held as float32 arrays; ``round16`` rounds to them. ``append`` follows
the kernels' single fp32 roundings (bit-exact), ``append64``, ``bounds64`` and ``attention`` the
formulas in 64 bits, ``select`` integers. ``blocks_by_bounds`` states the selection a second time,
over exact rationals.
"""

from __future__ import annotations

from fractions import Fraction

import numpy as np

from oracle import quantize as oq


def round16(x: np.ndarray, kind: str) -> np.ndarray:
    """float32 or float64 values to the nearest ``"bf16"`` or ``"fp16"`` (ties to even), as
    float32."""
    if kind == "fp16":
        with np.errstate(over="ignore"):
            return np.asarray(x).astype(np.float16).astype(np.float32)
    x = np.asarray(x, np.float32)
    bits = x.view(np.uint32)
    up = (((bits >> 16) & 1) + np.uint32(0x7FFF)).astype(np.uint32)
    out = ((bits + up) & np.uint32(0xFFFF0000)).view(np.float32)
    return np.where(np.isnan(x), x, out)


def _pairs(rot: int, interleaved: bool) -> tuple[np.ndarray, np.ndarray]:
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def rotate(x: np.ndarray, cos_sin: np.ndarray, interleaved: bool, dtype=np.float32) -> np.ndarray:
    """``x [T, H, D]`` turned by each token's row ``cos_sin [T, rot]``, every step in ``dtype``."""
    out = x.astype(dtype)
    rot = cos_sin.shape[1]
    a, b = _pairs(rot, interleaved)
    c = cos_sin[:, None, :rot // 2].astype(dtype)
    s = cos_sin[:, None, rot // 2:].astype(dtype)
    xa, xb = out[..., a], out[..., b]
    out[..., a], out[..., b] = xa * c - xb * s, xb * c + xa * s
    return out


def place(positions, seq_ids, page_table, pages: int, page: int):
    """(position, own block, the sequence's page-table row) of each token, None for padding."""
    b, most = page_table.shape
    return [(int(p), int(p) // page, page_table[s]) if p >= 0 and 0 <= s < b and p // page < most
            else None for p, s in zip(positions, seq_ids)]


def _page(at, block: int, pages: int) -> int:
    i = int(at[2][block])
    return i if 0 <= i < pages else -1


def bounds_of(stored: np.ndarray) -> tuple[np.ndarray, np.float32]:
    """The codes ``[2 D]`` and scale of a block's stored keys ``[page, D]``."""
    low, high = stored.min(0).astype(np.float32), stored.max(0).astype(np.float32)
    half = np.float32(0.5)
    row = np.concatenate([(low + high) * half, (high - low) * half]).astype(np.float32)
    codes, scales = oq.quantize_int8(row[None], divide=True)
    return codes[0], scales[0]


def append64(x, cos_sin, positions, interleaved=False):
    """Queries or keys ``[T, H, D]`` turned by their positions' angles in 64 bits: each pair as a
    complex number times ``c + i s``."""
    out = np.array(x, np.float64)
    rot = cos_sin.shape[1]
    a, b = _pairs(rot, interleaved)
    row = cos_sin[positions].astype(np.float64)[:, None]
    z = (out[..., a] + 1j * out[..., b]) * (row[..., :rot // 2] + 1j * row[..., rot // 2:])
    out[..., a], out[..., b] = z.real, z.imag
    return out


def bounds64(stored):
    """``(row [2 D], scale)`` of a block's stored keys ``[page, D]``: the middle and half the width
    of each channel's range, and what one code of the row stands for."""
    low, high = stored.astype(np.float64).min(0), stored.astype(np.float64).max(0)
    row = np.concatenate([low + (high - low) / 2, (high - low) / 2])
    return row, max(np.abs(row).max(), 1e-8) / 127


def append(q, k, v, cos_sin, positions, seq_ids, page_table, k_cache, v_cache, bounds, scales, kind,
           interleaved=False):
    """Updates the caches and bounds in place, token by token; returns the rotated queries."""
    pages, _, page, _ = k_cache.shape
    out = np.zeros(q.shape, np.float32)
    for t, at in enumerate(place(positions, seq_ids, page_table, pages, page)):
        if at is None or (cos_sin is not None and at[0] >= len(cos_sin)):
            continue
        i = _page(at, at[1], pages)
        if i < 0:
            continue
        row = np.zeros((1, 0), np.float32) if cos_sin is None else cos_sin[at[0]][None]
        out[t] = round16(rotate(q[t][None], row, interleaved), kind)[0]
        k_cache[i, :, at[0] % page] = round16(rotate(k[t][None], row, interleaved), kind)[0]
        v_cache[i, :, at[0] % page] = v[t]
        if at[0] % page == page - 1:
            for h in range(k_cache.shape[1]):
                bounds[i, h], scales[i, h] = bounds_of(k_cache[i, h])
    return out


def scores(q, bounds, scales, pages_of_blocks, heads_kv):
    """fp32 scores ``[Hkv, blocks]`` of one token's ``q [Hq, D]`` with the listed pages."""
    codes, qs = oq.quantize_int8(q, divide=True)
    codes = codes.astype(np.int64)
    both = np.concatenate([codes, np.abs(codes)], 1).reshape(heads_kv, -1, 2 * q.shape[1])
    rows = bounds[pages_of_blocks].astype(np.int64)  # [blocks, Hkv, 2 D]
    dots = np.einsum("hgd,bhd->hgb", both, rows).astype(np.float32)
    best = (dots * qs.reshape(heads_kv, -1, 1)).max(1)
    return best * scales[pages_of_blocks].T


def select(q, bounds, scales, positions, seq_ids, page_table, page, count, sink=1, recent=1):
    """int32 ``[T, Hkv, count]``."""
    pages, heads_kv, _ = bounds.shape
    out = np.full((len(q), heads_kv, count), -1, np.int32)
    for t, at in enumerate(place(positions, seq_ids, page_table, pages, page)):
        if at is None:
            continue
        last = at[1]
        middle = [b for b in range(sink, last - recent + 1) if _page(at, b, pages) >= 0]
        forced = [b for b in range(last + 1) if b < sink or b > last - recent]
        s = scores(q[t], bounds, scales, [_page(at, b, pages) for b in middle], heads_kv)
        s = np.where(np.isnan(s), -np.inf, s)
        for h in range(heads_kv):
            order = np.lexsort((middle, -s[h]))[:count - sink - recent]
            kept = sorted(forced + [middle[i] for i in order])
            out[t, h, :len(kept)] = kept
    return out


def most_a_block_can_score(q, stored) -> np.ndarray:
    """sum over channels of the larger of q lo and q hi: what no key of the block exceeds."""
    return np.maximum(q * stored.min(0), q * stored.max(0)).sum()


def attention(q, k_cache, v_cache, blocks, positions, seq_ids, page_table, scale):
    """``(out, lse, spread, slack)`` in 64 bits: ``spread`` = the weights' sum over ``|v|`` (what a
    relative error of every weight can move an output by), ``slack [T, Hq]`` = the largest ``|scale|
    sum |q k|``."""
    pages, heads_kv, page, d = k_cache.shape
    t, heads, _ = q.shape
    out, spread = np.zeros((t, heads, d)), np.zeros((t, heads, d))
    lse, slack = np.full((t, heads), -np.inf), np.zeros((t, heads))
    for i, at in enumerate(place(positions, seq_ids, page_table, pages, page)):
        if at is None:
            continue
        for h in range(heads_kv):
            rows_k, rows_v = [], []
            for b in blocks[i, h]:
                if b < 0 or b > at[1] or _page(at, b, pages) < 0:
                    continue
                n = min(page, at[0] - int(b) * page + 1)
                rows_k.append(k_cache[_page(at, b, pages), h, :n])
                rows_v.append(v_cache[_page(at, b, pages), h, :n])
            if not rows_k:
                continue
            kk = np.concatenate(rows_k).astype(np.float64)
            vv = np.concatenate(rows_v).astype(np.float64)
            for g in range(h * heads // heads_kv, (h + 1) * heads // heads_kv):
                x = kk @ q[i, g].astype(np.float64) * scale
                w = np.exp(x - x.max())
                lse[i, g] = x.max() + np.log(w.sum())
                w /= w.sum()
                out[i, g], spread[i, g] = w @ vv, w @ np.abs(vv)
                slack[i, g] = (np.abs(kk) @ np.abs(q[i, g].astype(np.float64))).max() * abs(scale)
    return out, lse, spread, slack


def blocks_by_bounds(q_codes, q_scales, codes, scale, want):
    """The ``want`` best blocks of one head group over exact rationals (no fp32 rounding), ties to
    the lower block: what ``select`` gives wherever no two scores are within fp32 rounding."""
    def score(b):
        return max(Fraction(int(sum(int(c) * int(m) for c, m in zip(row, codes[b][:len(row)]))
                                + sum(abs(int(c)) * int(m)
                                      for c, m in zip(row, codes[b][len(row):]))))
                   * Fraction(float(s)) for row, s in zip(q_codes, q_scales)) \
            * Fraction(float(scale[b]))
    return sorted(sorted(range(len(codes)), key=lambda b: (-score(b), b))[:want])
