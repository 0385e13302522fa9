"""A language model's paged key/value cache searched by block, as ``torch.ops.retrieve_kv.*``.

At long contexts a token attends to the few blocks of the cache whose keys can score highest with
its query, found the way the scans find items: int8 codes, int32 sums, exact selection with ties
to the lower index. Three ops over one layer's cache, in the order a model's layer calls them:

- :func:`append`: new tokens' queries, keys and values rotated, keys and values written to their
  pages, int8 bounds of the blocks that become full;
- :func:`select_blocks`: the best blocks of each token and key/value head by those bounds;
- :func:`block_attention`: softmax attention over the chosen blocks.

Tokens are packed: token ``t`` is at ``positions[t]`` of sequence ``seq_ids[t]``, a row of
``page_table [B, max_pages]`` (the physical page of each block of ``page`` tokens, -1 for none), all
int32. One token a sequence is a decode step, many a prompt; a call may mix them. Caches are ``[P,
Hkv, page, D]`` (a block of one head is contiguous), bounds int8 ``[P, Hkv, 2 D]`` with scales fp32
``[P, Hkv]``. :class:`PagedCache` holds them and makes the three calls; :func:`rotary_table` builds
the table of cosines and sines. No counterpart in the reference; serving only: the ops have no
gradients (a backward pass through one warns and stops there, a forward-mode tangent is refused).

The ops check their arguments here (``ValueError`` on shapes, ``TypeError`` on dtypes), allocate
from torch's caching allocator and enqueue on torch's current stream, without a host
synchronization.
"""

from __future__ import annotations

import contextlib
import math

import torch
from torch import Tensor
from torch.autograd import forward_ad

from retrieve_amd import _native as nat

DTYPES = {torch.bfloat16: 0, torch.float16: 1}
HEAD_DIMS = (64, 96, 128, 192, 256)
PAGE_SIZES = (16, 32, 64, 128)
MAX_COUNT = 1024

_lib = torch.library.Library("retrieve_kv", "DEF")
_lib.define("append(Tensor q, Tensor k, Tensor v, Tensor? cos_sin, Tensor positions, "
            "Tensor seq_ids, Tensor page_table, Tensor(a!) k_cache, Tensor(b!) v_cache, "
            "Tensor(c!) bounds, Tensor(d!) bound_scales, bool interleaved=False) -> Tensor")
_lib.define("select_blocks(Tensor q, Tensor bounds, Tensor bound_scales, Tensor positions, "
            "Tensor seq_ids, Tensor page_table, int page_size, int count, int sink=1, "
            "int recent=1, int? sequences=None) -> Tensor")
_lib.define("block_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor blocks, "
            "Tensor positions, Tensor seq_ids, Tensor page_table, float? scale=None, "
            "int? sequences=None) -> (Tensor, Tensor)")


# --- checks -----------------------------------------------------------------------------------


def _check_tokens(t: int, positions: Tensor, seq_ids: Tensor, page_table: Tensor) -> None:
    if positions.shape != (t,) or seq_ids.shape != (t,) or page_table.dim() != 2:
        raise ValueError(f"positions and seq_ids must be [{t}] and page_table [B, max_pages]")
    if not (positions.dtype is seq_ids.dtype is page_table.dtype is torch.int32):
        raise TypeError("positions, seq_ids and page_table must be int32")
    if not (positions.is_contiguous() and seq_ids.is_contiguous() and page_table.is_contiguous()):
        raise ValueError("positions, seq_ids and page_table must be contiguous")


def _check_heads(dtype: torch.dtype, heads: int, heads_kv: int, dim: int, page: int) -> int:
    """The dtype's number, after the checks of the numbers that every call has."""
    if dtype not in DTYPES:
        raise TypeError(f"q must be bfloat16 or float16, got {dtype}")
    if dim not in HEAD_DIMS:
        raise TypeError(f"heads have {HEAD_DIMS} channels, got {dim}")
    if page not in PAGE_SIZES:
        raise ValueError(f"a page holds {PAGE_SIZES} tokens, got {page}")
    if heads_kv < 1 or heads < 1 or heads % heads_kv:
        raise ValueError(f"{heads} query heads do not share {heads_kv} key/value heads evenly")
    return DTYPES[dtype]


def _check_caches(q: Tensor, k_cache: Tensor, v_cache: Tensor):
    """``(T, Hq, P, Hkv, page, D, dtype's number)``"""
    shape = k_cache.shape
    if len(shape) != 4 or v_cache.shape != shape:
        raise ValueError("k_cache and v_cache must both be [P, Hkv, page, D]")
    pages, heads_kv, page, dim = shape
    if q.dim() != 3 or q.shape[2] != dim:
        raise ValueError(f"q must be [T, Hq, {dim}], got {list(q.shape)}")
    t, heads, _ = q.shape
    if not (q.dtype is k_cache.dtype is v_cache.dtype):
        raise TypeError("q and the caches must have one dtype")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache and v_cache must be contiguous")
    return t, heads, pages, heads_kv, page, dim, _check_heads(q.dtype, heads, heads_kv, dim, page)


def _check_bounds(bounds: Tensor, bound_scales: Tensor, dim: int) -> tuple[int, int]:
    """``(P, Hkv)``"""
    shape = bounds.shape
    if len(shape) != 3 or shape[2] != 2 * dim or bound_scales.shape != shape[:2]:
        raise ValueError("bounds must be [P, Hkv, 2 D] and bound_scales [P, Hkv]")
    if bounds.dtype is not torch.int8 or bound_scales.dtype is not torch.float32:
        raise TypeError("bounds must be int8 and bound_scales float32")
    if not (bounds.is_contiguous() and bound_scales.is_contiguous()):
        raise ValueError("bounds and bound_scales must be contiguous")
    return shape[0], shape[1]


def _sequences(sequences: int | None, page_table: Tensor) -> int:
    """How many sequences a call's tokens belong to at most."""
    if sequences is None:
        return page_table.shape[0]
    if sequences < 1:
        raise ValueError(f"sequences must be at least 1, got {sequences}")
    return sequences


def _rows(x: Tensor) -> tuple[Tensor, int, int]:
    """``x [T, H, D]`` with its token and head strides, where its rows lie as the kernels read them
    (16-byte chunks of contiguous channels: the views of a fused projection do), else a copy."""
    token, head, channel = x.stride()
    if channel != 1 or token % 8 or head % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        _, h, d = x.shape
        token, head = h * d, d
    return x, token, head


def _device(*tensors: Tensor) -> int:
    """The GPU that holds all of them."""
    at = tensors[0].get_device()
    for t in tensors:
        if t.get_device() != at or at < 0:
            nat.require_device(*tensors)
    return at


def _on(device: int):
    """The tensors' GPU as the current one, where it is not already."""
    return _HERE if device == _current() else torch.cuda.device(device)


def _out(q: Tensor, t: int, heads: int, dim: int) -> Tensor:
    """A contiguous tensor of the queries' shape."""
    return torch.empty_like(q) if q.is_contiguous() else q.new_empty((t, heads, dim))


_HERE = contextlib.nullcontext()
_current = torch._C._cuda_getDevice  # (torch is initialised there: the tensors are on a GPU)
_stream = torch._C._cuda_getCurrentRawStream  # (the current stream's handle, without an object)


# What a thread that traces nothing and transforms nothing has among the dispatcher's included keys.
# The modes that see or rewrite calls (make_fx, torch.jit.trace, dispatch modes, vmap, grad, jvp)
# each add their own.
_included = torch._C._dispatch_tls_local_include_set
_PLAIN_KEYS = (torch._C.DispatchKeySet(torch._C.DispatchKey.BackendSelect)
               | torch._C.DispatchKeySet(torch._C.DispatchKey.ADInplaceOrView)).raw_repr()
_PLAIN_TYPES = frozenset((Tensor, type(None)))


def _eager(*tensors: Tensor | None) -> bool:
    """Whether a call can go straight to its kernels: plain tensors that carry no gradients, nothing
    being traced or transformed. Elsewhere it goes through the registered op (the dispatcher's 3 to
    5 us a call are a third of a small one; these checks take 1)."""
    if torch.compiler.is_compiling():
        return False
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError("retrieve_kv ops have no derivatives: an input has a tangent")
    if _included().raw_repr() & ~_PLAIN_KEYS or not _PLAIN_TYPES.issuperset(map(type, tensors)):
        return False
    return not (torch.is_grad_enabled() and torch._C._any_requires_grad(*tensors))


# --- append -----------------------------------------------------------------------------------


def _append(q, k, v, cos_sin, positions, seq_ids, page_table, k_cache, v_cache, bounds,
            bound_scales, interleaved=False):
    t, heads, pages, heads_kv, page, dim, dtype = _check_caches(q, k_cache, v_cache)
    if k.shape != (t, heads_kv, dim) or v.shape != k.shape:
        raise ValueError(f"k and v must be [{t}, {heads_kv}, {dim}]")
    if not (k.dtype is v.dtype is q.dtype):
        raise TypeError("q, k and v must have one dtype")
    _check_tokens(t, positions, seq_ids, page_table)
    if _check_bounds(bounds, bound_scales, dim) != (pages, heads_kv):
        raise ValueError("bounds must be [P, Hkv, 2 D] and bound_scales [P, Hkv]")
    length = rot = 0
    if cos_sin is not None:
        if cos_sin.dim() != 2 or cos_sin.shape[1] % 2 or cos_sin.shape[1] > dim:
            raise ValueError(f"cos_sin must be [length, rot], rot even and at most {dim}")
        if cos_sin.dtype is not torch.float32:
            raise TypeError("cos_sin must be float32")
        if not cos_sin.is_contiguous():
            raise ValueError("cos_sin must be contiguous")
        if cos_sin.get_device() != q.get_device():
            nat.require_device(q, cos_sin)
        length, rot = cos_sin.shape
        if cos_sin.data_ptr() % 16:
            cos_sin = cos_sin.clone()
    dev = _device(q, k, v, positions, seq_ids, page_table, k_cache, v_cache, bounds, bound_scales)
    q, q_token, q_head = _rows(q)
    k, k_token, k_head = _rows(k)
    v, v_token, v_head = _rows(v)
    out = _out(q, t, heads, dim)
    with _on(dev):
        st = nat.lib().rt_kv_append(
            q.data_ptr(), q_token, q_head, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token,
            v_head, t, heads, heads_kv, dim, dtype, nat.ptr(cos_sin), length, rot, interleaved,
            positions.data_ptr(), seq_ids.data_ptr(), page_table.data_ptr(), *page_table.shape,
            k_cache.data_ptr(), v_cache.data_ptr(), pages, page, bounds.data_ptr(),
            bound_scales.data_ptr(), out.data_ptr(), _stream(dev))
    if st:
        nat.check(st)
    return out


def append(q: Tensor, k: Tensor, v: Tensor, cos_sin: Tensor | None, positions: Tensor,
           seq_ids: Tensor, page_table: Tensor, k_cache: Tensor, v_cache: Tensor, bounds: Tensor,
           bound_scales: Tensor, interleaved: bool = False) -> Tensor:
    """Rotates the new tokens' queries ``q [T, Hq, D]`` and keys ``k [T, Hkv, D]`` and writes keys
    and values ``v [T, Hkv, D]`` to their slots; returns the rotated queries. Any token and head
    strides (the views of a fused projection are read where they lie).

    ``cos_sin [length, rot]`` fp32 holds a position's ``rot / 2`` cosines, then its sines
    (:func:`rotary_table`); channels ``(i, i + rot / 2)`` turn together, ``(2 i, 2 i + 1)`` with
    ``interleaved``; channels from ``rot`` on stay as they are; None (or ``rot`` 0) rotates nothing.
    A token at the last slot of its block fills the block's ``bounds``: ``[mid | half]`` of its
    stored keys' least and largest values per channel, quantised as ``quantize_int8``'s rows. For
    that a sequence's tokens come in order, side by side. Tokens that are padding (a position below
    0, or past the page table or ``cos_sin``; a sequence outside it; no page) write nothing and
    return a zero row."""
    args = (q, k, v, cos_sin, positions, seq_ids, page_table, k_cache, v_cache, bounds,
            bound_scales)
    call = _append if _eager(*args) else torch.ops.retrieve_kv.append
    return call(*args, interleaved)


# --- select -----------------------------------------------------------------------------------


def _select(q, bounds, bound_scales, positions, seq_ids, page_table, page_size, count, sink=1,
            recent=1, sequences=None):
    if q.dim() != 3:
        raise ValueError("q must be [T, Hq, D]")
    t, heads, dim = q.shape
    pages, heads_kv = _check_bounds(bounds, bound_scales, dim)
    dtype = _check_heads(q.dtype, heads, heads_kv, dim, page_size)
    _check_tokens(t, positions, seq_ids, page_table)
    if not 1 <= count <= MAX_COUNT:
        raise ValueError(f"count must be in [1, {MAX_COUNT}], got {count}")
    if sink < 0 or recent < 1 or sink + recent > count:
        raise ValueError(f"sink >= 0 and recent >= 1 must fit in count, got {sink}, {recent}")
    sequences = _sequences(sequences, page_table)
    dev = _device(q, bounds, bound_scales, positions, seq_ids, page_table)
    q, q_token, q_head = _rows(q)
    out = positions.new_empty((t, heads_kv, count))
    lib = nat.lib()
    b, max_pages = page_table.shape
    with _on(dev):
        need = lib.rt_kv_select_workspace(t, heads_kv, sequences, max_pages, count, sink, recent)
        ws = bounds.new_empty((need,)) if need else None
        st = lib.rt_kv_select_of(
            q.data_ptr(), q_token, q_head, t, heads, heads_kv, dim, dtype, bounds.data_ptr(),
            bound_scales.data_ptr(), pages, page_size, positions.data_ptr(), seq_ids.data_ptr(),
            page_table.data_ptr(), b, max_pages, count, sink, recent, sequences, out.data_ptr(),
            nat.ptr(ws), need, _stream(dev))
    if st:
        nat.check(st)
    return out


def select_blocks(q: Tensor, bounds: Tensor, bound_scales: Tensor, positions: Tensor,
                  seq_ids: Tensor, page_table: Tensor, page_size: int, count: int, sink: int = 1,
                  recent: int = 1, sequences: int | None = None) -> Tensor:
    """The blocks that each token and key/value head attends to, int32 ``[T, Hkv, count]``,
    ascending, -1 at the end. The first ``sink`` blocks and the last ``recent`` ones up to the
    token's own are always among them; the other places go to the best blocks between by ``(score
    desc, block asc)``. A score is the largest, over the heads that share the key/value head, of
    ``c . mid + |c| . half`` (int32; ``c`` the rotated query's int8 codes) times the query's and the
    block's scales: an upper bound on what the block's keys can score, up to the codes' rounding.
    Blocks between without a page are left out; padding tokens get -1 throughout.

    ``sequences``: how many sequences the tokens belong to at most, where that is known to be fewer
    than the page table has rows. It chooses among kernels (prompts share a pass over their
    sequence's blocks), never what is chosen."""
    args = (q, bounds, bound_scales, positions, seq_ids, page_table)
    call = _select if _eager(*args) else torch.ops.retrieve_kv.select_blocks
    return call(*args, page_size, count, sink, recent, sequences)


# --- attention ----------------------------------------------------------------------------------


def _attention(q, k_cache, v_cache, blocks, positions, seq_ids, page_table, scale=None,
               sequences=None):
    t, heads, pages, heads_kv, page, dim, dtype = _check_caches(q, k_cache, v_cache)
    _check_tokens(t, positions, seq_ids, page_table)
    if blocks.dim() != 3 or blocks.shape[:2] != (t, heads_kv):
        raise ValueError(f"blocks must be [{t}, {heads_kv}, count]")
    if blocks.dtype is not torch.int32:
        raise TypeError("blocks must be int32")
    if not blocks.is_contiguous():
        raise ValueError("blocks must be contiguous")
    sequences = _sequences(sequences, page_table)
    dev = _device(q, k_cache, v_cache, blocks, positions, seq_ids, page_table)
    q, q_token, q_head = _rows(q)
    count = blocks.shape[2]
    out = _out(q, t, heads, dim)
    lse = q.new_empty((t, heads), dtype=torch.float32)
    lib = nat.lib()
    with _on(dev):
        need = lib.rt_kv_attention_workspace(t, heads, heads_kv, dim, page, count)
        ws = blocks.new_empty((need // 4,)) if need else None  # (floats)
        st = lib.rt_kv_attention_of(
            q.data_ptr(), q_token, q_head, t, heads, heads_kv, dim, dtype, k_cache.data_ptr(),
            v_cache.data_ptr(), pages, page, blocks.data_ptr(), count, positions.data_ptr(),
            seq_ids.data_ptr(), page_table.data_ptr(), *page_table.shape,
            1.0 / math.sqrt(dim) if scale is None else scale, sequences, out.data_ptr(),
            lse.data_ptr(), nat.ptr(ws), need, _stream(dev))
    if st:
        nat.check(st)
    return out, lse


def block_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, blocks: Tensor, positions: Tensor,
                    seq_ids: Tensor, page_table: Tensor, scale: float | None = None,
                    sequences: int | None = None) -> tuple[Tensor, Tensor]:
    """Softmax attention of ``q [T, Hq, D]`` (rotated) over the keys of the listed ``blocks`` (int32
    ``[T, Hkv, count]``, each at most once a row, in any order) at positions up to the token's own,
    with scores ``scale * q . k`` (``1 / sqrt(D)`` by default): ``(out [T, Hq, D], lse fp32 [T,
    Hq])``, ``lse`` the natural logarithm of the weights' sum. Entries below 0, past the token's
    block or without a page are skipped; a row without a key is zeros and ``-inf``. Slots past a
    token's position are not used, whatever they hold. ``sequences`` as in :func:`select_blocks`."""
    args = (q, k_cache, v_cache, blocks, positions, seq_ids, page_table)
    call = _attention if _eager(*args) else torch.ops.retrieve_kv.block_attention
    return call(*args, scale, sequences)


_lib.impl("append", _append, "CUDA")
_lib.impl("select_blocks", _select, "CUDA")
_lib.impl("block_attention", _attention, "CUDA")


@torch.library.register_fake("retrieve_kv::append", lib=_lib)
def _(q, k, v, cos_sin, positions, seq_ids, page_table, k_cache, v_cache, bounds, bound_scales,
      interleaved=False):
    return q.new_empty(q.shape)


@torch.library.register_fake("retrieve_kv::select_blocks", lib=_lib)
def _(q, bounds, bound_scales, positions, seq_ids, page_table, page_size, count, sink=1, recent=1,
      sequences=None):
    return q.new_empty((q.shape[0], bounds.shape[1], count), dtype=torch.int32)


@torch.library.register_fake("retrieve_kv::block_attention", lib=_lib)
def _(q, k_cache, v_cache, blocks, positions, seq_ids, page_table, scale=None, sequences=None):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


def _no_cpu(*args, **kwargs):
    raise ValueError("retrieve_kv ops run on the GPU only")


for _name in ("append", "select_blocks", "block_attention"):
    _lib.impl(_name, _no_cpu, "CPU")


# --- the rotation's table ------------------------------------------------------------------------


def rotary_table(length: int, rot: int, *, base: float = 10000.0, scaling: str | None = None,
                 factor: float = 1.0, original: int | None = None, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, device: str | torch.device = "cuda") -> Tensor:
    """``cos_sin [length, rot]`` fp32 for :func:`append`, computed in 64 bits: position ``p`` turns
    pair ``i`` by ``p * base ** (-2 i / rot)``. ``scaling`` stretches a model trained on
    ``original`` positions to ``factor`` times as many:

    - ``"linear"``: every position divided by ``factor``;
    - ``"base"``: a larger base, ``base * factor ** (rot / (rot - 2))``: the fastest pair as it was,
      the slowest slowed by ``factor``;
    - ``"ramp"``: pairs that turn more than ``beta_fast`` times over ``original`` as they were,
      those below ``beta_slow`` divided by ``factor``, a linear ramp over the pairs between (from
      the pair where the turns pass ``beta_fast``, rounded down, to the one where they pass
      ``beta_slow``, rounded up), cosines and sines scaled by ``0.1 ln(factor) + 1``.
    """
    if rot < 2 or rot % 2 or length < 0:
        raise ValueError(f"rot must be even and at least 2, length at least 0: {rot}, {length}")
    if factor < 1.0:
        raise ValueError(f"factor must be at least 1, got {factor}")
    half = rot // 2
    if scaling == "base":
        if rot < 4:
            raise ValueError("scaling the base needs rot of 4 or more")
        base = base * factor ** (rot / (rot - 2))
    pair = torch.arange(half, dtype=torch.float64)
    freq = base ** (-pair / half)
    size = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ramp":
        if original is None or original < 1:
            raise ValueError("scaling 'ramp' needs the original length")

        def at(turns: float) -> float:  # the pair that turns so often over the original length
            return half * math.log(original / (turns * 2 * math.pi)) / math.log(base)

        low, high = math.floor(at(beta_fast)), math.ceil(at(beta_slow))
        slow = ((pair - low) / max(high - low, 1)).clamp(0, 1)
        freq = freq * (1 - slow) + freq / factor * slow
        size = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'ramp', got {scaling!r}")
    angle = torch.arange(length, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos() * size, angle.sin() * size], 1).float().to(device)


# --- one layer's cache ---------------------------------------------------------------------------


class PagedCache:
    """One layer's cache and the three calls over it, for a fixed set of sequences' slots.

    >>> cache = PagedCache(pages=4096, heads=8, dim=128, page=64, sequences=16, max_pages=2048)
    >>> cache.reserve(seq, tokens)                    # pages for a sequence (host)
    >>> q = cache.append(q, k, v, cos_sin, positions, seq_ids)
    >>> out, lse = cache.attend(q, positions, seq_ids, count=64)

    ``reserve`` and ``free`` keep the page table on the host and send a sequence's row to the GPU;
    ``append`` and ``attend`` only launch kernels. These are chosen by how many sequences a call's
    tokens belong to: ``sequences``, or the slots that hold pages where it is not said (say it for a
    prompt beside many held slots)."""

    def __init__(self, pages: int, heads: int, dim: int, page: int = 64, sequences: int = 1,
                 max_pages: int | None = None, dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device = "cuda"):
        if page not in PAGE_SIZES:
            raise ValueError(f"a page holds {PAGE_SIZES} tokens, got {page}")
        if dim not in HEAD_DIMS or dtype not in DTYPES:
            raise TypeError(f"heads have {HEAD_DIMS} channels in bfloat16 or float16")
        max_pages = pages if max_pages is None else max_pages
        self.page = page
        shape = (pages, heads, page, dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.bounds = torch.empty((pages, heads, 2 * dim), dtype=torch.int8, device=device)
        self.bound_scales = torch.empty((pages, heads), dtype=torch.float32, device=device)
        self.page_table = torch.full((sequences, max_pages), -1, dtype=torch.int32, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._held: list[list[int]] = [[] for _ in range(sequences)]
        self._active = 0  # slots that hold pages

    def reserve(self, seq: int, tokens: int) -> None:
        """Pages for the sequence's first ``tokens`` tokens, those that it has already among
        them."""
        held, need = self._held[seq], -(-tokens // self.page)
        if need > self.page_table.shape[1]:
            raise ValueError(f"{need} pages: a sequence has at most {self.page_table.shape[1]}")
        more = need - len(held)
        if more > len(self._free):
            raise RuntimeError(f"{more} pages wanted, {len(self._free)} free")
        if more > 0:
            new = [self._free.pop() for _ in range(more)]
            self.page_table[seq, len(held):need] = torch.tensor(new, dtype=torch.int32)
            self._active += not held
            held += new

    def free(self, seq: int) -> None:
        """Returns the sequence's pages."""
        self._free += reversed(self._held[seq])
        self._active -= bool(self._held[seq])
        self._held[seq] = []
        self.page_table[seq] = -1

    def append(self, q: Tensor, k: Tensor, v: Tensor, cos_sin: Tensor | None, positions: Tensor,
               seq_ids: Tensor, interleaved: bool = False) -> Tensor:
        """:func:`append` into this cache: the rotated queries."""
        return append(q, k, v, cos_sin, positions, seq_ids, self.page_table, self.k, self.v,
                      self.bounds, self.bound_scales, interleaved)

    def _sequences(self, sequences: int | None) -> int | None:
        return self._active or None if sequences is None else sequences

    def select(self, q: Tensor, positions: Tensor, seq_ids: Tensor, count: int, sink: int = 1,
               recent: int = 1, sequences: int | None = None) -> Tensor:
        """:func:`select_blocks` over this cache."""
        return select_blocks(q, self.bounds, self.bound_scales, positions, seq_ids,
                             self.page_table, self.page, count, sink, recent,
                             self._sequences(sequences))

    def attend(self, q: Tensor, positions: Tensor, seq_ids: Tensor, count: int, sink: int = 1,
               recent: int = 1, scale: float | None = None, sequences: int | None = None
               ) -> tuple[Tensor, Tensor]:
        """The selection and the attention over what it chose: ``(out, lse)``."""
        blocks = self.select(q, positions, seq_ids, count, sink, recent, sequences)
        return block_attention(q, self.k, self.v, blocks, positions, seq_ids, self.page_table,
                               scale, self._sequences(sequences))


__all__ = ["PagedCache", "append", "block_attention", "rotary_table", "select_blocks"]
