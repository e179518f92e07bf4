"""A paged cache of 4-bit keys and values for many requests at once.

``create_kv_cache`` serves one batch whose sequences have equal lengths and
lie in memory of their own.  Here requests of different lengths share a pool
of pages, keys and values are both held in 4 bits (no codec to fit), and a
step runs without the host knowing any length:

``build_block_tables``  pages, slots and positions of a step from the
                        requests' lengths, on the GPU
``append_paged``        quantise the new tokens into their slots
``append_rotated_paged``  the same with the norms and the rotation of queries
                        and keys on the way (``rotary_table``)
``read_paged``          what slots hold
``paged_attention``     the new tokens' queries over their requests
``build_shared_plan``   which requests continue others, for ``paged_attention``
``PagedKVCache``        the four tied together; ``sunshape_sdpa`` and the SDPA
                        router take it as they take the other caches

A row of ``head_dim`` values is held in groups of ``group_size``: zero = the
group's smallest value, scale = (largest - smallest) / 15 in the cache's
16-bit type, and a 4-bit code per value, the nearest of 0 .. 15 to
(x - zero) / scale; the held value is zero + code * scale.  A group with an
infinity or NaN, or whose range passes float32, is held as NaN.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _hip
from .cache import DeferredTensor

_HALF = (torch.float16, torch.bfloat16)
_MAX_REQUESTS = 4096  # of build_block_tables


class _Store(ctypes.Structure):
    """``ss_paged_store``."""

    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("k_meta", ctypes.c_void_p), ("v_meta", ctypes.c_void_p),
                ("n_pages", ctypes.c_int64), ("n_kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("group_size", ctypes.c_int),
                ("page_size", ctypes.c_int), ("dtype", ctypes.c_int)]


class _Rotation(ctypes.Structure):
    """``ss_rotation``."""

    _fields_ = [("table", ctypes.c_void_p), ("n_positions", ctypes.c_int64),
                ("rotary_dim", ctypes.c_int), ("neighbours", ctypes.c_int),
                ("q_weight", ctypes.c_void_p), ("k_weight", ctypes.c_void_p),
                ("eps", ctypes.c_double), ("weight_dtype", ctypes.c_int)]


class _Scores(ctypes.Structure):
    """``ss_paged_scores``."""

    _fields_ = [("softcap", ctypes.c_float), ("slopes", ctypes.c_void_p),
                ("window", ctypes.c_int64), ("prefix_lengths", ctypes.c_void_p),
                ("group_starts", ctypes.c_void_p), ("group_rows", ctypes.c_void_p),
                ("parents", ctypes.c_void_p), ("n_groups", ctypes.c_int64),
                ("max_shared", ctypes.c_int64)]


class PagedKVStore(NamedTuple):
    """The pool's pages:

    ``k_codes`` int32 (n_pages, H, P, D/8): word w of a token holds its dims
    8w .. 8w+7; ``v_codes`` int32 (n_pages, H, P/8, D): word (w, d) holds dim
    d of tokens 8w .. 8w+7; element j of a word at bit 4*(j//2) + 16*(j%2).
    ``k_meta``, ``v_meta`` float16 or bfloat16 (n_pages, H, D/group, P, 2):
    scale and zero.  Slot s is token s % P of page s // P.
    """

    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_meta: torch.Tensor
    v_meta: torch.Tensor

    @classmethod
    def zeros(cls, n_pages: int, n_kv_heads: int, head_dim: int, *, page_size: int = 64,
              group_size: int = 64, dtype: torch.dtype = torch.float16,
              device=None) -> "PagedKVStore":
        """An empty pool."""
        if dtype not in _HALF:
            raise TypeError(f"a paged cache is float16 or bfloat16, not {dtype}")
        if head_dim not in (64, 128) or group_size not in (32, 64, 128) or group_size > head_dim:
            raise ValueError(f"head_dim must be 64 or 128 and group_size 32, 64 or 128 and at most "
                             f"head_dim (got {head_dim}, {group_size})")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 16 to 1024, got {page_size}")
        if n_pages < 1 or n_kv_heads < 1:
            raise ValueError("n_pages and n_kv_heads must be positive")
        if max(n_pages * page_size, n_pages * n_kv_heads) >= 2 ** 31:
            raise ValueError(f"a pool of {n_pages} pages of {page_size} tokens and {n_kv_heads} heads: "
                             f"slots, and heads of pages, are counted in 32 bits")
        dev = torch.device("cuda") if device is None else torch.device(device)
        meta = (n_pages, n_kv_heads, head_dim // group_size, page_size, 2)
        return cls(
            torch.zeros((n_pages, n_kv_heads, page_size, head_dim // 8), dtype=torch.int32, device=dev),
            torch.zeros((n_pages, n_kv_heads, page_size // 8, head_dim), dtype=torch.int32, device=dev),
            torch.zeros(meta, dtype=dtype, device=dev), torch.zeros(meta, dtype=dtype, device=dev))

    @property
    def page_size(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return self.v_codes.shape[3]

    @property
    def n_kv_heads(self) -> int:
        return self.k_codes.shape[1]

    @property
    def dtype(self) -> torch.dtype:
        return self.k_meta.dtype


class BlockPlan(NamedTuple):
    """What ``build_block_tables`` gives: the requests' lengths and the free
    pages after the step, where each request's new tokens start in the packed
    order, each packed token's slot and position (-1 behind the last), and
    ``status`` (0, or why the step changed nothing: ``check_plan``)."""

    lengths: torch.Tensor
    n_free: torch.Tensor
    token_starts: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    status: torch.Tensor


class SharedPlan(NamedTuple):
    """What ``build_shared_plan`` gives: the rows that see the tokens of request
    p, ``rows[group_starts[p]:group_starts[p + 1]]`` (token, position among its
    request's own tokens); each request's parent or -1; the packed tokens'
    positions, which follow their parents' tokens (-1 behind the last); and
    what the caller knows of the sizes."""

    group_starts: torch.Tensor
    rows: torch.Tensor
    parents: torch.Tensor
    positions: torch.Tensor
    n_groups: int = 1
    max_shared: int | None = None


def _struct(store: PagedKVStore) -> _Store:
    """The store's C form, its tensors checked (every call: they may have been
    given other memory in place)."""
    kc, vc, km, vm = store
    if not (kc.is_cuda and vc.is_cuda and km.is_cuda and vm.is_cuda):
        _hip.require_gpu(kc, vc, km, vm)
    shape, meta = kc.shape, km.shape
    if len(shape) != 4 or len(meta) != 5:
        raise ValueError("a paged store has 4-dim codes and 5-dim scales")
    n, h, p, w = shape
    d, g = 8 * w, meta[2]
    if vc.shape != (n, h, p // 8, d) or meta != (n, h, g, p, 2) or vm.shape != meta or \
            g < 1 or d % g or p % 8:
        raise ValueError(f"store shapes do not agree: {tuple(shape)}, {tuple(vc.shape)}, "
                         f"{tuple(meta)}, {tuple(vm.shape)}")
    dtype = km.dtype
    if kc.dtype is not torch.int32 or vc.dtype is not torch.int32 or dtype not in _HALF or \
            vm.dtype is not dtype:
        raise TypeError("a paged store has int32 codes and float16 or bfloat16 scales")
    dev = kc.get_device()
    if vc.get_device() != dev or km.get_device() != dev or vm.get_device() != dev or not (
            kc.is_contiguous() and vc.is_contiguous() and km.is_contiguous() and
            vm.is_contiguous()):
        raise ValueError("store tensors must be contiguous and on one device")
    return _Store(kc.data_ptr(), vc.data_ptr(), km.data_ptr(), vm.data_ptr(), n, h, d, d // g, p,
                  _CODE[dtype])


# names of the dispatch counters (get_kernel_stats)
_STATS = {f"ss_{n}": f"{n}_hip" for n in ("block_tables", "append_paged", "append_rotated_paged",
                                          "read_paged", "paged_attn", "paged_attn_scored",
                                          "shared_plan")}
_CODE = {torch.float32: _hip.SS_F32, torch.float16: _hip.SS_F16, torch.bfloat16: _hip.SS_BF16}


def _index(name: str, t: torch.Tensor, shape, dev: int) -> int:
    """The address of an int32 tensor of the tables, checked."""
    if not t.is_cuda:
        _hip.require_gpu(t)
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, not {t.dtype}")
    if t.shape != shape or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{name} must be contiguous {tuple(shape)} on cuda:{dev}, got "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _launch(name: str, dev: int, *args) -> None:
    """A C-ABI call on the current stream of device ``dev``, which need not be
    the current device."""
    fn = getattr(_hip.load_library(), name)
    if dev == torch._C._cuda_getDevice():
        rc = fn(*args, _hip.stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _hip.stream_handle(dev))
    _hip._launched(_STATS[name], rc)


def _capturing(t: torch.Tensor) -> bool:
    """Whether calls on this tensor go into a graph."""
    return t.is_cuda and torch.cuda.is_current_stream_capturing()


def build_block_tables(lengths: torch.Tensor, new_lengths: torch.Tensor,
                       block_table: torch.Tensor, free_pages: torch.Tensor,
                       n_free: torch.Tensor, page_size: int, n_tokens: int, *,
                       lengths_out: torch.Tensor | None = None,
                       n_free_out: torch.Tensor | None = None) -> BlockPlan:
    """A scheduling step: request r holds ``lengths[r]`` tokens and adds
    ``new_lengths[r]`` (negative: gives its last ones back).  Pages no longer
    needed go onto the stack ``free_pages[:n_free]``, new ones come from its
    top; ``block_table`` (R, W) and ``free_pages`` are updated in place.  The
    new tokens are packed request after request into ``n_tokens`` places (at
    least as many as are added).  ``lengths_out`` / ``n_free_out``: where the
    counts after the step go (``lengths`` / ``n_free`` themselves to step in
    place; new tensors by default).  All tensors int32 on one device; nothing
    waits for the GPU: a step that is impossible (too few pages, say) changes
    nothing, gives no token a slot and says why in ``status``."""
    if lengths.dim() != 1 or block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("lengths (R,), block_table (R, W) and free_pages (n_pages,) expected")
    if n_tokens < 0:
        raise ValueError("n_tokens must not be negative")
    if not lengths.is_cuda:
        _hip.require_gpu(lengths)
    dev, size = lengths.get_device(), lengths.shape
    r, width = size[0], block_table.shape[1]
    args = (_index("lengths", lengths, size, dev), _index("new_lengths", new_lengths, size, dev), r,
            _index("block_table", block_table, (r, width), dev), width,
            _index("free_pages", free_pages, free_pages.shape, dev), free_pages.shape[0],
            _index("n_free", n_free, (1,), dev), page_size, n_tokens)
    # one allocation for everything that is new
    buf = torch.empty(2 * r + 3 + 2 * n_tokens, dtype=torch.int32, device=lengths.device)
    starts, slots, positions, len_out, free_out, status = buf.split_with_sizes(
        (r + 1, n_tokens, n_tokens, r, 1, 1))
    at = buf.data_ptr()
    at_len = at + 4 * (r + 1 + 2 * n_tokens)
    at_free, at_status = at_len + 4 * r, at_len + 4 * r + 4
    if lengths_out is not None:
        len_out, at_len = lengths_out, _index("lengths_out", lengths_out, size, dev)
    if n_free_out is not None:
        free_out, at_free = n_free_out, _index("n_free_out", n_free_out, (1,), dev)
    at_slots = at + 4 * (r + 1)
    _launch("ss_block_tables", dev, *args, at_len, at_free, at, at_slots, at_slots + 4 * n_tokens,
            at_status)
    return BlockPlan(len_out, free_out, starts, slots, positions, status)


_STATUS = ((1, "a negative length"), (2, "more tokens than a block table row holds"),
           (4, "too few free pages"), (8, "more new tokens than n_tokens"),
           (16, "a count of free pages out of range"))


def check_plan(plan: BlockPlan) -> None:
    """Raise if the step of ``plan`` was impossible (waits for the GPU)."""
    status = int(plan.status.item())
    if status:
        raise RuntimeError("block tables: " + ", ".join(t for b, t in _STATUS if status & b))


def build_shared_plan(parents: torch.Tensor, lengths: torch.Tensor, token_starts: torch.Tensor,
                      n_tokens: int, *, n_groups: int = 1,
                      max_shared: int | None = None) -> SharedPlan:
    """Which of the packed tokens continue which request.  Request r continues
    ``parents[r]`` where that is another request, else (-1, say) none: its
    tokens follow all of the parent's, which the cache holds once for all that
    continue it.  A parent's own parent is not followed.  ``lengths`` and
    ``token_starts`` are the step's (``build_block_tables``); all int32 on one
    device.  ``n_groups`` (how many parents) and ``max_shared`` (their longest
    length) size later launches: wrong ones cost time and change roundings
    only.  One plan serves every layer of the step."""
    if parents.dim() != 1:
        raise ValueError("parents (R,) expected")
    if n_tokens < 0 or n_groups < 1 or (max_shared is not None and max_shared < 0):
        raise ValueError("n_tokens and max_shared must not be negative, n_groups positive")
    if not parents.is_cuda:
        _hip.require_gpu(parents)
    dev, r = parents.get_device(), parents.shape[0]
    args = (_index("parents", parents, (r,), dev), _index("lengths", lengths, (r,), dev),
            _index("token_starts", token_starts, (r + 1,), dev), r, n_tokens)
    # one allocation for everything that is new
    buf = parents.new_empty(3 * n_tokens + 3 * r + 1)
    rows, starts, of, _, positions = buf.split_with_sizes((2 * n_tokens, r + 1, r, r, n_tokens))
    at = buf.data_ptr()
    at_starts = at + 8 * n_tokens
    at_of = at_starts + 4 * (r + 1)
    _launch("ss_shared_plan", dev, *args, at_starts, at, at_of, at_of + 4 * r, at_of + 8 * r)
    return SharedPlan(starts, rows.view(n_tokens, 2), of, positions, n_groups, max_shared)


def _rows(name: str, t: torch.Tensor, shape, dev: int) -> torch.Tensor:
    """(N, H, D) rows with unit last stride."""
    if not t.is_cuda:
        _hip.require_gpu(t)
    if t.shape != shape or t.get_device() != dev:
        raise ValueError(f"{name} must be {tuple(shape)} on cuda:{dev}, got {tuple(t.shape)} on "
                         f"{t.device}")
    return t if t.stride(2) == 1 else t.contiguous()


def _new_rows(keys: torch.Tensor, values: torch.Tensor, shape, dev: int):
    """(keys, values, type code) of new tokens, as the append takes them."""
    if keys.dtype is not values.dtype:
        raise TypeError("keys and values must share a dtype")
    code = _hip.dtype_code(keys.dtype)
    return _rows("keys", keys, shape, dev), _rows("values", values, shape, dev), code


def append_paged(store: PagedKVStore, keys: torch.Tensor, values: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Quantise ``keys`` and ``values`` (N, H, D), float16, bfloat16 or
    float32 (rounded to the store's type first), into ``slots`` (N,) int32.
    Tokens whose slot is negative or outside the pool are left out; the slots
    of the others have to differ from each other."""
    st = _struct(store)
    dev = store[0].get_device()
    n = slots.shape[0]
    at_slots = _index("slots", slots, (n,), dev)
    k, v, code = _new_rows(keys, values, (n, st.n_kv_heads, st.head_dim), dev)
    _launch("ss_append_paged", dev, ctypes.addressof(st), k.data_ptr(), v.data_ptr(), code, n,
            k.stride(0), k.stride(1), v.stride(0), v.stride(1), at_slots)


def rotary_table(n_positions: int, rotary_dim: int, base: float = 10000.0, *,
                 frequencies: torch.Tensor | None = None, device=None) -> torch.Tensor:
    """Cosines and sines of ``append_rotated_paged``, (n_positions,
    rotary_dim / 2, 2) float32: pair i of position p turns by p *
    frequencies[i] (by default base^(-2i / rotary_dim)), an angle in 64 bits."""
    if n_positions < 1 or rotary_dim < 16 or rotary_dim % 16:
        raise ValueError(f"n_positions must be positive and rotary_dim a multiple of 16 (got "
                         f"{n_positions}, {rotary_dim})")
    dev = torch.device("cuda") if device is None else torch.device(device)
    half = rotary_dim // 2
    if frequencies is None:
        if not 0.0 < base < float("inf"):
            raise ValueError(f"base must be positive, got {base}")
        freq = float(base) ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
    else:
        freq = torch.as_tensor(frequencies, dtype=torch.float64, device=dev)
        if freq.shape != (half,):
            raise ValueError(f"{half} frequencies expected, got {tuple(freq.shape)}")
    angle = torch.arange(n_positions, dtype=torch.float64, device=dev)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _like(q: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A new contiguous tensor of q's shape (empty_like takes half the time)."""
    if dtype is q.dtype and q.is_contiguous():
        return torch.empty_like(q)
    return torch.empty(q.shape, dtype=dtype, device=q.device)


def _no_derivative(name: str, *tensors) -> None:
    """Refuse tensors through which something is differentiated."""
    for t in tensors:
        if t is None:
            continue
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} has no backward pass: call it under torch.no_grad()")
        if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name} has no forward-mode derivative: unpack its dual tensors")


def append_rotated_paged(store: PagedKVStore, queries: torch.Tensor, keys: torch.Tensor,
                         values: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor,
                         rotary: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                         k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                         neighbours: bool = False,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """``append_paged`` of keys that are normalised and rotated on the way;
    returns the ``queries`` (N, Hq, D), normalised and rotated too, in their
    type (float32 ones in the store's).  All of one type, float16, bfloat16 or
    float32; keys and values (N, H, D).

    ``q_weight``, ``k_weight`` (D,): y = x / sqrt(mean(x^2) + eps) * weight, head
    by head (no norm without one).  ``rotary`` (n_positions, R/2, 2) float32:
    cosine and sine of each position (``rotary_table``); the first R dims turn,
    pairs are (i, i + R/2) or, with ``neighbours``, (2i, 2i + 1).  Each operation
    is rounded to float32 by itself, the result once.  ``positions`` (N,) int32,
    as ``build_block_tables`` gives them: a token with a negative one is not
    stored, and its query is zero, or, with ``out``, left as it was (``out`` may
    be contiguous ``queries``).  A position past the table makes the turned dims
    NaN.  Queries, weights or a table under autograd are refused; keys and values
    are stored without a derivative."""
    st = _struct(store)
    dev, d = store[0].get_device(), st.head_dim
    shape = queries.shape
    if len(shape) != 3 or shape[1] < 1 or slots.dim() != 1:
        raise ValueError("queries (N, Hq, D) and slots (N,) expected")
    n, hq, _ = shape
    if queries.dtype is not keys.dtype:
        raise TypeError("queries, keys and values must share a dtype")
    _no_derivative("append_rotated_paged", queries, q_weight, k_weight, rotary, out)
    at_slots = _index("slots", slots, (n,), dev)
    at_positions = _index("positions", positions, (n,), dev)
    k, v, code = _new_rows(keys, values, (n, st.n_kv_heads, d), dev)
    q = _rows("queries", queries, (n, hq, d), dev)
    if not rotary.is_cuda:
        _hip.require_gpu(rotary)
    if rotary.dtype is not torch.float32:
        raise TypeError(f"rotary must be float32, not {rotary.dtype}")
    turns = rotary.shape
    if len(turns) != 3 or turns[2] != 2 or not rotary.is_contiguous() or rotary.get_device() != dev:
        raise ValueError(f"rotary must be contiguous (n_positions, R/2, 2) on cuda:{dev}, got "
                         f"{tuple(rotary.shape)} on {rotary.device}")
    w_type, w_at = 0, []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            w_at.append(None)
            continue
        if not w.is_cuda:
            _hip.require_gpu(w)
        if w.shape != (d,) or not w.is_contiguous() or w.get_device() != dev:
            raise ValueError(f"{name} must be contiguous ({d},) on cuda:{dev}, got "
                             f"{tuple(w.shape)} on {w.device}")
        if w_at and w_at[0] is not None and w.dtype is not q_weight.dtype:
            raise TypeError("q_weight and k_weight must share a dtype")
        w_type = _hip.dtype_code(w.dtype)
        w_at.append(w.data_ptr())
    dtype = store[2].dtype if queries.dtype is torch.float32 else queries.dtype
    zero_rest = out is None
    if zero_rest:
        out = _like(q, dtype)
    elif out.shape != shape or out.dtype is not dtype or out.device != q.device or \
            not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} {(n, hq, d)} on {q.device}")
    ro = _Rotation(rotary.data_ptr(), turns[0], 2 * turns[1], neighbours, *w_at, eps, w_type)
    q_st, q_sh, _ = q.stride()
    k_st, k_sh, _ = k.stride()
    v_st, v_sh, _ = v.stride()
    _launch("ss_append_rotated_paged", dev, ctypes.addressof(st), q.data_ptr(), k.data_ptr(),
            v.data_ptr(), code, n, hq, q_st, q_sh, k_st, k_sh, v_st, v_sh, at_slots, at_positions,
            ctypes.addressof(ro), out.data_ptr(), zero_rest)
    if not zero_rest:  # (graphs that saved it refuse their backward pass)
        torch.autograd.graph.increment_version(out)
    return out


def read_paged(store: PagedKVStore, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(keys, values) that ``slots`` (N,) hold, (N, H, D) in the store's type
    (zeros for a slot outside the pool)."""
    st = _struct(store)
    n = slots.shape[0]
    dev = store[0].get_device()
    at_slots = _index("slots", slots, (n,), dev)
    shape = (n, st.n_kv_heads, st.head_dim)
    k = store[2].new_empty(shape)
    v = torch.empty_like(k)
    _launch("ss_read_paged", dev, ctypes.addressof(st), at_slots, n, k.data_ptr(), v.data_ptr())
    return k, v


@lru_cache(maxsize=4096)
def _workspace_bytes(dev: int, shape: tuple, n: int, r: int, hq: int, max_new: int,
                     max_length: int) -> int:
    """Workspace of a call of these sizes on device ``dev``."""
    like = _Store(1 << 20, 1 << 20, 1 << 20, 1 << 20, *shape)  # (addresses are not read)
    with torch.cuda.device(dev):
        return _hip.load_library().ss_paged_attn_workspace_bytes(
            ctypes.addressof(like), n, r, hq, max_new, max_length)


@lru_cache(maxsize=4096)
def _scored_workspace_bytes(dev: int, shape: tuple, n: int, r: int, hq: int, max_new: int,
                            max_length: int, window: int, n_groups: int, max_shared: int) -> int:
    """Workspace of a scored call of these sizes on device ``dev`` (n_groups 0:
    without shared tokens)."""
    like = _Store(1 << 20, 1 << 20, 1 << 20, 1 << 20, *shape)
    at = (1 << 20) if n_groups else None
    sc = _Scores(0.0, None, window, None, at, at, at, n_groups, max_shared)
    with torch.cuda.device(dev):
        return _hip.load_library().ss_paged_attn_scored_workspace_bytes(
            ctypes.addressof(like), n, r, hq, max_new, max_length, ctypes.addressof(sc))


def _scores(softcap, slopes, window, prefix_lengths, shared, n: int, r: int, hq: int, most: int,
            dev: int) -> _Scores:
    """The options of a scored call, checked."""
    sc = _Scores()
    if softcap is not None:
        if not 2.0 ** -60 <= softcap <= 2.0 ** 60:
            raise ValueError(f"softcap must be from 2^-60 to 2^60, got {softcap}")
        sc.softcap = softcap
    if slopes is not None:
        _no_derivative("paged_attention", slopes)
        if not slopes.is_cuda:
            _hip.require_gpu(slopes)
        if slopes.dtype is not torch.float32:
            raise TypeError(f"slopes must be float32, not {slopes.dtype}")
        if slopes.shape != (hq,) or not slopes.is_contiguous() or slopes.get_device() != dev:
            raise ValueError(f"slopes must be contiguous ({hq},) on cuda:{dev}, got "
                             f"{tuple(slopes.shape)} on {slopes.device}")
        sc.slopes = slopes.data_ptr()
    if window is not None:
        if window < 1:
            raise ValueError(f"window must be positive, got {window}")
        sc.window = min(window, 2 ** 31 - 1)
    if prefix_lengths is not None:
        sc.prefix_lengths = _index("prefix_lengths", prefix_lengths, (r,), dev)
    if shared is not None:
        if window is not None or prefix_lengths is not None:
            raise ValueError("shared tokens are not combined with window or prefix_lengths")
        sc.group_starts = _index("shared.group_starts", shared.group_starts, (r + 1,), dev)
        sc.group_rows = _index("shared.rows", shared.rows, (n, 2), dev)
        sc.parents = _index("shared.parents", shared.parents, (r,), dev)
        sc.n_groups = max(1, min(r, shared.n_groups))
        longest = most if shared.max_shared is None else shared.max_shared
        sc.max_shared = max(1, min(most, longest))
    return sc


def paged_attention(queries: torch.Tensor, store: PagedKVStore, block_table: torch.Tensor,
                    lengths: torch.Tensor, token_starts: torch.Tensor, scale: float, *,
                    causal: bool = True, max_new: int | None = None,
                    max_length: int | None = None, out: torch.Tensor | None = None,
                    softcap: float | None = None, slopes: torch.Tensor | None = None,
                    window: int | None = None, prefix_lengths: torch.Tensor | None = None,
                    shared: SharedPlan | None = None) -> torch.Tensor:
    """Attention of packed ``queries`` (N, Hq, D), float16 or bfloat16, over
    the pages of their requests.  Rows ``token_starts[r]`` to
    ``token_starts[r + 1]`` are the last of the ``lengths[r]`` tokens of
    request r (as ``build_block_tables`` counts them); with ``causal`` each
    sees the tokens up to its own, otherwise all of the request's.  A row
    that sees nothing is zero.  Rows of no request are zero, or, with ``out``,
    left as they were.

    ``max_new`` and ``max_length``, the most new tokens and the longest length
    if the caller knows them, size the launch (by default every request adds
    a token and a table row is full); wrong ones cost time and change roundings
    only.

    Other scores: with ``softcap`` c, a score s becomes c tanh(s / c); with
    ``slopes`` (Hq,) float32, a head's slope times the distance of the two
    tokens is taken off.  Other masks: with ``window`` w, a row sees none before
    the last w tokens up to its own; with ``prefix_lengths`` (R,) int32, all rows
    of request r see its first ``prefix_lengths[r]`` tokens (that the window
    leaves).  ``shared`` (``build_shared_plan`` for these starts and lengths): the
    rows of a request that continues another see all of that one's tokens
    first, which are read once for all of them; distances count them.  Not
    together with ``window`` or ``prefix_lengths``; ``max_length`` is then that
    that of the tokens that requests hold themselves.

    Scores, softmax statistics and sums are float32.  Probabilities, in prompts and
    over shared tokens values too, enter the products rounded to fp16 (2^-11; values
    below 2^-29 of a request's largest by 2^-40 of it); of bfloat16 queries the bits
    down to 2^-29 of a row's largest count; a capped score is off by 2^-21 of itself.
    Queries under autograd, forward mode too, are refused: there is no
    derivative."""
    st = _struct(store)
    dev = store[0].get_device()
    if queries.dim() != 3 or lengths.dim() != 1 or block_table.dim() != 2:
        raise ValueError("queries (N, Hq, D), lengths (R,) and block_table (R, W) expected")
    n, hq, _ = queries.shape
    r, width = block_table.shape
    dtype = queries.dtype
    if dtype not in _HALF:
        raise TypeError(f"queries must be float16 or bfloat16, not {dtype}")
    _no_derivative("paged_attention", queries, out)
    if hq < 1 or hq % st.n_kv_heads:
        raise ValueError(f"{hq} query heads do not share {st.n_kv_heads} KV heads")
    shape = (n, hq, st.head_dim)
    q = _rows("queries", queries, shape, dev)
    at_lengths = _index("lengths", lengths, (r,), dev)
    at_table = _index("block_table", block_table, (r, width), dev)
    at_starts = _index("token_starts", token_starts, (r + 1,), dev)
    zero_rest = out is None
    if zero_rest:
        out = _like(q, dtype)
    elif out.shape != shape or out.dtype is not dtype or out.device != q.device or \
            not out.is_contiguous():
        raise ValueError(f"out must be contiguous {dtype} {shape} on {q.device}")
    if n == 0:
        return out
    if r == 0:
        return out.zero_() if zero_rest else out
    most = width * st.page_size
    max_new = max(1, min(n, n - r + 1 if max_new is None else max_new))
    max_length = max(1, min(most, most if max_length is None else max_length))
    shape = (st.n_pages, st.n_kv_heads, st.head_dim, st.group_size, st.page_size, st.dtype)
    if softcap is not None or slopes is not None or window is not None or \
            prefix_lengths is not None or shared is not None:
        sc = _scores(softcap, slopes, window, prefix_lengths, shared, n, r, hq, most, dev)
        need = _scored_workspace_bytes(dev, shape, n, r, hq, max_new, max_length, sc.window,
                                       sc.n_groups, sc.max_shared)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _launch("ss_paged_attn_scored", dev, ctypes.addressof(st), q.data_ptr(), _CODE[dtype], n,
                q.stride(0), q.stride(1), hq, at_table, width, at_lengths, at_starts, r, scale,
                causal, max_new, max_length, out.data_ptr(), zero_rest, ctypes.addressof(sc),
                _hip.ptr(ws), need)
    else:
        need = _workspace_bytes(dev, shape, n, r, hq, max_new, max_length)
        # of this call alone: calls on other streams and captured graphs have their own
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        _launch("ss_paged_attn", dev, ctypes.addressof(st), q.data_ptr(), _CODE[dtype], n, q.stride(0),
                q.stride(1), hq, at_table, width, at_lengths, at_starts, r, scale, causal, max_new,
                max_length, out.data_ptr(), zero_rest, _hip.ptr(ws), need)
    if not zero_rest:  # (graphs that saved it refuse their backward pass)
        torch.autograd.graph.increment_version(out)
    return out


class PagedKVCache:
    """The keys and values of up to ``n_requests`` requests in one pool of
    ``n_pages`` pages (by default enough for ``max_tokens`` of each).

    A serving step is ``step`` (scheduling), ``append`` and ``attend`` on packed
    tokens, all requests together:

        cache.step(new_lengths, n_tokens)      # how many tokens each adds
        cache.append(keys, values)             # (N, H, D), request after request
        out = cache.attend(queries, scale)     # (N, Hq, D)

    Lengths, tables and the stack of free pages live on the GPU and are
    stepped there in place, so a step needs no synchronisation and can be
    captured in a graph.  ``share`` lets requests continue another, whose tokens are
    held and read once for all.  A batch whose sequences all add the same number of
    tokens may use ``update_and_fetch`` and ``sunshape_sdpa`` (or the SDPA
    router) instead, as with the other caches."""

    def __init__(self, *, n_requests: int, n_kv_heads: int = 1, head_dim: int = 128,
                 max_tokens: int, n_pages: int | None = None, page_size: int = 64,
                 group_size: int = 64, dtype: torch.dtype = torch.float16, device=None,
                 lazy_fetch: bool = True):
        if n_requests < 1 or max_tokens < 1:
            raise ValueError("n_requests and max_tokens must be positive")
        if n_requests > _MAX_REQUESTS or max_tokens > 2 ** 30:
            raise ValueError(f"at most {_MAX_REQUESTS} requests of at most 2^30 tokens (got "
                             f"{n_requests}, {max_tokens})")
        width = -(-max_tokens // max(1, page_size))
        if n_requests * width >= 2 ** 31:
            raise ValueError(f"a block table of {n_requests} rows of {width} pages")
        n_pages = n_requests * width if n_pages is None else n_pages
        self.store = PagedKVStore.zeros(n_pages, n_kv_heads, head_dim, page_size=page_size,
                                        group_size=group_size, dtype=dtype, device=device)
        dev = self.store.k_codes.device
        self.n_requests, self.n_kv_heads, self.head_dim = n_requests, n_kv_heads, head_dim
        self.page_size, self.group_size, self.dtype = page_size, group_size, dtype
        self.max_tokens = max_tokens
        self.lazy_fetch = lazy_fetch
        self.block_table = torch.full((n_requests, width), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros((n_requests,), dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(n_pages, dtype=torch.int32, device=dev)
        self.n_free = torch.full((1,), n_pages, dtype=torch.int32, device=dev)
        self.plan: BlockPlan | None = None  # of the last step
        self.shared: SharedPlan | None = None  # of it, where a request continues another
        self._kept: list[tuple] = []        # of steps that graphs go on reading
        self.parents: torch.Tensor | None = None  # on the GPU, once a request has one
        self._parent = [-1] * n_requests
        self._prefixes: frozenset[int] = frozenset()  # the requests that others continue
        self._version = 0                   # bumped by every change of the stored tokens
        # what the host knows of the lengths: all of them (steps given as
        # lists), or a bound
        self._host: list[int] | None = [0] * n_requests
        self._bound = 0
        self._max_new = self._longest = 1   # of the last step, for its attends' launches
        self._starts: tuple[int, torch.Tensor] | None = None

    # -------------------------------------------------------------- serving
    def step(self, new_lengths, n_tokens: int | None = None, *,
             max_new: int | None = None) -> BlockPlan:
        """Schedule a step in which request r adds ``new_lengths[r]`` tokens
        (negative: gives its last ones back; minus its length: ends).

        A list of ints raises here when the step is impossible, as long as the
        host knows the lengths: until a first step given as a tensor.  It
        cannot be captured.  A request that others continue gives tokens back only
        where all of these end in the same step; one that ends continues nothing
        any more.

        An int32 tensor on the GPU needs ``n_tokens``, at least the sum of what
        is added (``max_new``, the most one adds, sizes later launches).  It is
        held to what a row of the block table takes, ``max_tokens`` rounded up
        to whole pages; whether it was possible is seen by ``check``, as with a
        list whose lengths only the GPU knows.  Captured, it goes into the graph
        with its append and attend, and the plan holds what the last replay
        made of it; a graph with append or attend alone goes on with the slots
        and starts of the step that they were captured after.  The host sees neither
        what such a step ends nor, after one, what a list ends: requests that share
        have to end through ``release`` there."""
        return self._step(new_lengths, n_tokens, max_new)

    def _step(self, new_lengths, n_tokens: int | None = None, max_new: int | None = None,
              ended: set | None = None) -> BlockPlan:
        """``step``; ``ended``: the requests that end, whatever they add (by
        default those of a list that give back all they hold)."""
        host, bound, row = None, self._bound, self.block_table.shape[1] * self.page_size
        if isinstance(new_lengths, torch.Tensor):
            if n_tokens is None:
                raise ValueError("n_tokens is required with new_lengths on the GPU")
            new = new_lengths
            most = min(n_tokens, n_tokens if max_new is None else max_new)
            bound = min(row, bound + max(0, most))
            if _capturing(self.lengths):  # (replays add to the lengths too)
                bound = row
        else:
            if _capturing(self.lengths):
                raise RuntimeError("a step given as a list cannot be captured (its replays would not "
                                   "reach the host's lengths): give new_lengths on the GPU")
            adds = [int(x) for x in new_lengths]
            if len(adds) != self.n_requests:
                raise ValueError(f"{len(adds)} lengths for {self.n_requests} requests")
            total = sum(max(0, x) for x in adds)
            if n_tokens is not None and n_tokens < total:
                raise ValueError(f"{total} new tokens do not fit n_tokens {n_tokens}")
            n_tokens = total if n_tokens is None else n_tokens
            most = max(adds)
            if self._host is not None:
                host = [n + x for n, x in zip(self._host, adds)]
                pages = sum(-(-n // self.page_size) for n in host)
                if min(host) < 0 or max(host) > self.max_tokens:
                    raise ValueError(f"lengths {host} are not within 0 .. {self.max_tokens}")
                if pages > self.free_pages.shape[0]:
                    raise RuntimeError(f"{pages} pages needed, {self.free_pages.shape[0]} there")
                bound = max(host)
                if ended is None:
                    ended = {r for r, x in enumerate(adds) if x < 0 and not host[r]}
            else:
                bound = min(row, bound + max(0, most))
            for p in self._prefixes:
                if adds[p] < 0 and any(q == p and r not in (ended or ()) for r, q in enumerate(self._parent)):
                    raise ValueError(f"request {p}, which others continue, gives tokens back only where these "
                                     f"end too (see release)")
            new = torch.tensor(adds, dtype=torch.int32).to(self.lengths.device)
        plan = build_block_tables(self.lengths, new, self.block_table, self.free_pages,
                                  self.n_free, self.page_size, n_tokens,
                                  lengths_out=self.lengths, n_free_out=self.n_free)
        # (only now: a step that was refused has changed nothing here either)
        self._host, self._bound = host, bound
        self.shared, self._longest = None, max(1, bound)
        if self._prefixes:
            if host is not None:  # (rows are of those that add tokens: others' lengths do not matter)
                self._longest = max((n for n, x in zip(host, adds) if x > 0), default=1)
            longest = bound if host is None else max(host[p] for p in self._prefixes)
            self.shared = build_shared_plan(self.parents, self.lengths, plan.token_starts, n_tokens,
                                            n_groups=len(self._prefixes), max_shared=longest)
            plan = plan._replace(positions=self.shared.positions)
        self.plan, self._max_new = plan, max(1, most)
        self._version += 1
        if ended and self._prefixes:
            self._set_parents([-1 if r in ended else p for r, p in enumerate(self._parent)])
        return plan

    def check(self) -> None:
        """Raise if the last step was impossible (waits for the GPU)."""
        if self.plan is not None:
            check_plan(self.plan)

    def _last_plan(self, name: str) -> BlockPlan:
        if self.plan is None:
            raise RuntimeError(f"{name} needs a step first")
        if _capturing(self.lengths) and (not self._kept or self._kept[-1][0] is not self.plan):
            # the graph reads it after the next step has replaced it here
            self._kept.append((self.plan, self.shared))
        return self.plan

    def share(self, requests, parent: int | None) -> None:
        """From the next step on these requests continue ``parent``: their tokens
        follow all of its tokens, which the cache holds once; ``attend`` reads
        those once for all of them, and positions (``append_rotated``) count them
        (a parent that grows later moves them: keys rotated before that stay as
        they are).
        They hold no tokens yet; a request continues only one that continues none.
        ``parent`` None: they continue nothing; not while they hold tokens behind
        one.  (Where only the GPU knows the lengths, after a step given as a tensor,
        both are the caller's to see to.)  Graphs follow, but for those of a
        step that was captured while no request continued another."""
        at = [int(r) for r in requests]
        every = range(self.n_requests)
        if any(r not in every for r in at) or (parent is not None and parent not in every):
            raise ValueError(f"requests must be within 0 .. {self.n_requests - 1}")
        if _capturing(self.lengths):
            raise RuntimeError("share cannot be captured: the host keeps the parents")
        p = -1 if parent is None else int(parent)
        if p >= 0:
            if p in at or self._parent[p] >= 0:
                raise ValueError(f"request {p} continues another or itself")
            if not self._prefixes.isdisjoint(at):
                raise ValueError("a request that others continue cannot continue another")
            if self._host is not None and any(self._host[r] for r in at):
                raise ValueError("requests hold tokens already: share before their first step")
        elif self._host is not None and any(self._host[r] and self._parent[r] >= 0 for r in at):
            raise ValueError("requests hold tokens behind those of another: release ends them")
        new = list(self._parent)
        for r in at:
            new[r] = p
        self._set_parents(new)

    def _set_parents(self, new: list) -> None:
        if new == self._parent:
            return
        on_gpu = torch.tensor(new, dtype=torch.int32)
        if self.parents is None:
            self.parents = on_gpu.to(self.lengths.device)
        else:
            self.parents.copy_(on_gpu)
        self._parent, self._prefixes = new, frozenset(new) - {-1}

    def append(self, keys: torch.Tensor, values: torch.Tensor) -> None:
        """Store the keys and values (N, H, D) of the last step's tokens."""
        append_paged(self.store, keys, values, self._last_plan("append").slots)
        self._version += 1

    def append_rotated(self, queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor,
                       rotary: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                       k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                       neighbours: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
        """``append`` with the norms and the rotation of the last step's tokens
        on the way (``append_rotated_paged``); returns their queries for
        ``attend``."""
        plan = self._last_plan("append_rotated")
        out = append_rotated_paged(self.store, queries, keys, values, plan.slots, plan.positions,
                                   rotary, q_weight=q_weight, k_weight=k_weight, eps=eps,
                                   neighbours=neighbours, out=out)
        self._version += 1
        return out

    def attend(self, queries: torch.Tensor, scale: float, *, causal: bool = True,
               out: torch.Tensor | None = None, softcap: float | None = None,
               slopes: torch.Tensor | None = None, window: int | None = None,
               prefix_lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the last step's tokens' queries (N, Hq, D); scores and
        masks other than the causal ones as in ``paged_attention``."""
        starts = self._last_plan("attend").token_starts
        return paged_attention(queries, self.store, self.block_table, self.lengths, starts, scale,
                               causal=causal, max_new=self._max_new, max_length=self._longest, out=out,
                               softcap=softcap, slopes=slopes, window=window,
                               prefix_lengths=prefix_lengths, shared=self.shared)

    def release(self, requests) -> None:
        """End these requests: their pages go back to the pool, and they continue
        nothing any more.  One that others continue ends with them or after."""
        at = torch.as_tensor(list(requests), dtype=torch.int64)
        if at.numel() and (int(at.min()) < 0 or int(at.max()) >= self.n_requests):
            raise ValueError(f"requests must be within 0 .. {self.n_requests - 1}")
        gone = set(at.tolist())
        if not self._prefixes.isdisjoint(gone) and \
                any(p in gone and r not in gone for r, p in enumerate(self._parent)):
            raise ValueError("a request that others continue ends with them or after them")
        if self._host is not None:
            self._step([-n if r in gone else 0 for r, n in enumerate(self._host)], ended=gone)
        else:
            new = torch.zeros_like(self.lengths)
            at = at.to(new.device)
            new[at] = -self.lengths[at]
            self._step(new, 0, ended=gone)

    def trim(self, n: int) -> None:
        """Give the last ``n`` tokens of every request back (of those that others
        continue none).  A request of which none are left goes on where it was: it
        continues what it continued."""
        n = max(0, n)
        keep = self._prefixes
        if self._host is not None:
            self._step([0 if r in keep else -min(n, have) for r, have in enumerate(self._host)], ended=set())
        else:
            new = -self.lengths.clamp(max=n)
            for r in keep:
                new[r] = 0
            self.step(new, 0)

    # ------------------------------------------- batches of equal steps
    def _none_shared(self, name: str) -> None:
        if self._prefixes:
            raise RuntimeError(f"{name} steps all requests alike: where some continue others, use "
                               f"step, append and attend")

    def update_and_fetch(self, keys: torch.Tensor, values: torch.Tensor):
        """Append ``keys`` and ``values`` (B, H, T, D), T tokens to each of the
        cache's B requests.  Returns them as held, (B, H, offset, D) in the
        cache's type (read when used, with ``lazy_fetch``), where all requests
        have one length, else (None, None)."""
        self._none_shared("update_and_fetch")
        b_, h_, t_, d = keys.shape
        if (b_, h_, d) != (self.n_requests, self.n_kv_heads, self.head_dim) or \
                values.shape != keys.shape:
            raise ValueError(f"keys and values must be ({self.n_requests}, {self.n_kv_heads}, T, "
                             f"{self.head_dim}), got {tuple(keys.shape)}, {tuple(values.shape)}")
        rows = (b_ * t_, h_, d)
        # refused before the requests grow
        k, v, _ = _new_rows(keys.transpose(1, 2).reshape(rows), values.transpose(1, 2).reshape(rows),
                            rows, self.lengths.get_device())
        self.step([t_] * b_)
        self.append(k, v)
        if self._host is None or min(self._host) != max(self._host):
            return None, None
        shape = (b_, h_, self._host[0], d)
        if not self.lazy_fetch:
            return self._held()
        dev = self.lengths.device
        return tuple(DeferredTensor(lambda i=i: self._held()[i], shape, self.dtype, dev, self)
                     for i in range(2))

    def _held(self):
        """(keys, values) of requests of one length, (B, H, offset, D)."""
        n = self.offset
        pos = torch.arange(n, device=self.lengths.device)
        slots = self.block_table[:, pos // self.page_size] * self.page_size + pos % self.page_size
        k, v = read_paged(self.store, slots.to(torch.int32).reshape(-1))
        shape = (self.n_requests, n, self.n_kv_heads, self.head_dim)
        return k.view(shape).transpose(1, 2), v.view(shape).transpose(1, 2)

    def sdpa(self, queries: torch.Tensor, scale: float, mask=None) -> torch.Tensor:
        """``sunshape_sdpa`` over this cache: ``queries`` (B, Hq, T, D) are those
        of each request's last T tokens; ``mask`` is None (every query sees all
        of its request) or ``"causal"``.  Lengths make the padding masks of
        other caches unnecessary; arrays are refused."""
        if mask is not None and not (isinstance(mask, str) and mask in ("causal", "none")):
            raise ValueError("a paged cache takes no mask array: its requests have lengths of "
                             "their own (mask None or 'causal')")
        self._none_shared("sdpa")
        b_, hq, t_, d = queries.shape
        if b_ != self.n_requests:
            raise ValueError(f"queries of {b_} sequences, {self.n_requests} requests")
        dev = self.lengths.device
        if _capturing(self.lengths):  # (the graph's own, filled by its replays)
            starts = torch.arange(b_ + 1, dtype=torch.int32, device=dev) * t_
        else:
            if self._starts is None or self._starts[0] != t_:
                # copied from the host, which waits: any stream may read it
                self._starts = (t_, (torch.arange(b_ + 1, dtype=torch.int32) * t_).to(dev))
            starts = self._starts[1]
        out = paged_attention(queries.transpose(1, 2).reshape(b_ * t_, hq, d), self.store,
                              self.block_table, self.lengths, starts, scale,
                              causal=mask == "causal", max_new=max(1, t_),
                              max_length=max(1, self._bound))
        return out.view(b_, t_, hq, d).transpose(1, 2)

    @property
    def offset(self) -> int:
        """Tokens held by every request (raises where they differ or the host
        does not know them; ``lengths`` has them on the GPU)."""
        if self._host is None or min(self._host) != max(self._host):
            raise RuntimeError("the requests have no one length known to the host; see lengths")
        return self._host[0]

    # -------------------------------------------------------------- protocol
    def is_trimmable(self) -> bool:
        return True

    def empty(self) -> bool:
        """Whether no request holds a token (waits for the GPU where the host
        does not know the lengths)."""
        return not any(self._host) if self._host is not None else not bool(self.lengths.any())

    def make_mask(self, N: int, return_array: bool = False, window_size: int | None = None,
                  **kwargs):
        """``"causal"``, the mask of new queries (no array: see ``sdpa``)."""
        if return_array or window_size is not None:
            raise ValueError("a paged cache has no mask arrays")
        return "causal"

    @property
    def nbytes(self) -> int:
        """Bytes of the pool."""
        return sum(t.numel() * t.element_size() for t in self.store)

    def __repr__(self) -> str:
        return (f"PagedKVCache(n_requests={self.n_requests}, n_kv_heads={self.n_kv_heads}, "
                f"head_dim={self.head_dim}, pages={self.free_pages.shape[0]}x{self.page_size}, "
                f"group_size={self.group_size}, dtype={self.dtype})")
