"""A paged cache of 4-bit keys and values for many requests at once.

``create_kv_cache`` serves one batch whose sequences have equal lengths and
lie in memory of their own.  Here requests of different lengths share a pool
of pages, keys and values are both held in 4 bits (no codec to fit), and a
step runs without the host knowing any length:

``build_block_tables``  pages, slots and positions of a step from the
                        requests' lengths, on the GPU
``append_paged``        quantise the new tokens into their slots
``read_paged``          what slots hold
``paged_attention``     the new tokens' queries over their requests
``PagedKVCache``        the four tied together; ``sunshape_sdpa`` and the SDPA
                        router take it as they take the other caches

A row of ``head_dim`` values is held in groups of ``group_size``: zero = the
group's smallest value, scale = (largest - smallest) / 15 in the cache's
16-bit type, and a 4-bit code per value, the nearest of 0 .. 15 to
(x - zero) / scale; the held value is zero + code * scale.  A group with an
infinity or NaN is held as NaN.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _hip

_HALF = (torch.float16, torch.bfloat16)


class _Store(ctypes.Structure):
    """``ss_paged_store``."""

    _fields_ = [("k_codes", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("k_meta", ctypes.c_void_p), ("v_meta", ctypes.c_void_p),
                ("n_pages", ctypes.c_int64), ("n_kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int), ("group_size", ctypes.c_int),
                ("page_size", ctypes.c_int), ("dtype", ctypes.c_int)]


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


def _struct(store: PagedKVStore) -> _Store:
    """The store's C form, its tensors' shapes checked against each other."""
    kc, vc, km, vm = store
    if kc.dim() != 4 or vc.dim() != 4 or km.dim() != 5 or kc.shape[2] < 1:
        raise ValueError("a paged store has 4-dim codes and 5-dim scales")
    n, h, p, _ = kc.shape
    d = vc.shape[3]
    g = km.shape[2]
    meta = (n, h, g, p, 2)
    if kc.shape != (n, h, p, d // 8) or vc.shape != (n, h, p // 8, d) or km.shape != meta or \
            vm.shape != meta or g < 1 or d % g or d % 8:
        raise ValueError(f"store shapes do not agree: {tuple(kc.shape)}, {tuple(vc.shape)}, "
                         f"{tuple(km.shape)}, {tuple(vm.shape)}")
    if kc.dtype != torch.int32 or vc.dtype != torch.int32 or km.dtype not in _HALF or \
            vm.dtype != km.dtype:
        raise TypeError("a paged store has int32 codes and float16 or bfloat16 scales")
    _hip.require_gpu(*store)
    dev = kc.device
    for t in store:
        if not t.is_contiguous() or t.device != dev:
            raise ValueError("store tensors must be contiguous and on one device")
    return _Store(kc.data_ptr(), vc.data_ptr(), km.data_ptr(), vm.data_ptr(), n, h, d, d // g, p,
                  _hip.dtype_code(km.dtype))


def _index(name: str, t: torch.Tensor, shape, device) -> torch.Tensor:
    """An int32 tensor of the tables, checked."""
    _hip.require_gpu(t)
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, not {t.dtype}")
    if t.shape != shape or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be contiguous {tuple(shape)} on {device}, got "
                         f"{tuple(t.shape)} on {t.device}")
    return t


def _launch(name: str, device, *args) -> None:
    """A C-ABI call on the current stream of ``device``, which need not be
    the current device."""
    fn = getattr(_hip.load_library(), name)
    if device.index == torch.cuda.current_device():
        _hip.check(fn(*args, _hip.stream_handle(device)))
    else:
        with torch.cuda.device(device):
            _hip.check(fn(*args, _hip.stream_handle(device)))
    _hip.record_dispatch(name[3:] + "_hip")


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
    _hip.require_gpu(lengths)
    dev = lengths.device
    if lengths.dim() != 1 or block_table.dim() != 2 or free_pages.dim() != 1:
        raise ValueError("lengths (R,), block_table (R, W) and free_pages (n_pages,) expected")
    r = lengths.shape[0]
    _index("lengths", lengths, (r,), dev)
    _index("new_lengths", new_lengths, (r,), dev)
    _index("block_table", block_table, (r, block_table.shape[1]), dev)
    _index("free_pages", free_pages, free_pages.shape, dev)
    _index("n_free", n_free, (1,), dev)
    if n_tokens < 0:
        raise ValueError("n_tokens must not be negative")
    # one allocation for everything that is new
    buf = torch.empty(2 * r + 3 + 2 * n_tokens, dtype=torch.int32, device=dev)
    parts = buf.split_with_sizes((r + 1, n_tokens, n_tokens, r, 1, 1))
    starts, slots, positions, len_out, free_out, status = parts
    len_out = len_out if lengths_out is None else _index("lengths_out", lengths_out, (r,), dev)
    free_out = free_out if n_free_out is None else _index("n_free_out", n_free_out, (1,), dev)
    _launch("ss_block_tables", dev, lengths.data_ptr(), new_lengths.data_ptr(), r,
            block_table.data_ptr(), block_table.shape[1], free_pages.data_ptr(),
            free_pages.shape[0], n_free.data_ptr(), page_size, n_tokens, len_out.data_ptr(),
            free_out.data_ptr(), starts.data_ptr(), slots.data_ptr(), positions.data_ptr(),
            status.data_ptr())
    return BlockPlan(len_out, free_out, starts, slots, positions, status)


_STATUS = ((1, "a negative length"), (2, "more tokens than a block table row holds"),
           (4, "too few free pages"), (8, "more new tokens than n_tokens"),
           (16, "a count of free pages out of range"))


def check_plan(plan: BlockPlan) -> None:
    """Raise if the step of ``plan`` was impossible (waits for the GPU)."""
    status = int(plan.status.item())
    if status:
        raise RuntimeError("block tables: " + ", ".join(t for b, t in _STATUS if status & b))


def _rows(name: str, t: torch.Tensor, shape, device) -> torch.Tensor:
    """(N, H, D) rows of a kernel's type with unit last stride."""
    _hip.require_gpu(t)
    if t.shape != shape or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} on {device}, got {tuple(t.shape)} on "
                         f"{t.device}")
    return t if t.stride(2) == 1 else t.contiguous()


def append_paged(store: PagedKVStore, keys: torch.Tensor, values: torch.Tensor,
                 slots: torch.Tensor) -> None:
    """Quantise ``keys`` and ``values`` (N, H, D), float16, bfloat16 or
    float32 (rounded to the store's type first), into ``slots`` (N,) int32.
    Tokens whose slot is negative or outside the pool are left out; the slots
    of the others have to differ from each other."""
    st = _struct(store)
    dev = store.k_codes.device
    shape = (slots.shape[0], st.n_kv_heads, st.head_dim) if slots.dim() == 1 else None
    _index("slots", slots, slots.shape[:1], dev)
    if keys.dtype != values.dtype:
        raise TypeError("keys and values must share a dtype")
    code = _hip.dtype_code(keys.dtype)
    k, v = _rows("keys", keys, shape, dev), _rows("values", values, shape, dev)
    _launch("ss_append_paged", dev, ctypes.addressof(st), k.data_ptr(), v.data_ptr(), code,
            shape[0], k.stride(0), k.stride(1), v.stride(0), v.stride(1), slots.data_ptr())


def read_paged(store: PagedKVStore, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(keys, values) that ``slots`` (N,) hold, (N, H, D) in the store's type
    (zeros for a slot outside the pool)."""
    st = _struct(store)
    dev = store.k_codes.device
    _index("slots", slots, slots.shape[:1], dev)
    n = slots.shape[0]
    out = torch.empty((2, n, st.n_kv_heads, st.head_dim), dtype=store.dtype, device=dev)
    k, v = out.unbind(0)
    _launch("ss_read_paged", dev, ctypes.addressof(st), slots.data_ptr(), n, k.data_ptr(),
            v.data_ptr())
    return k, v


def paged_attention(queries: torch.Tensor, store: PagedKVStore, block_table: torch.Tensor,
                    lengths: torch.Tensor, token_starts: torch.Tensor, scale: float, *,
                    causal: bool = True, max_new: int | None = None,
                    max_length: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed ``queries`` (N, Hq, D), float16 or bfloat16, over
    the pages of their requests.  Rows ``token_starts[r]`` to
    ``token_starts[r + 1]`` are the last of the ``lengths[r]`` tokens of
    request r (as ``build_block_tables`` counts them); with ``causal`` each
    sees the tokens up to its own, otherwise all of the request's.  A row
    that sees nothing is zero.  Rows of no request are zero, or, with ``out``,
    left as they were.

    ``max_new`` and ``max_length``, the most new tokens and the longest length
    if the caller knows them, size the launch (by default every request adds
    a token and a table row is full); the result does not depend on them.
    Queries under autograd are refused: there is no backward pass."""
    st = _struct(store)
    dev = store.k_codes.device
    if queries.dim() != 3 or lengths.dim() != 1 or block_table.dim() != 2:
        raise ValueError("queries (N, Hq, D), lengths (R,) and block_table (R, W) expected")
    n, hq, _ = queries.shape
    r = lengths.shape[0]
    if queries.dtype not in _HALF:
        raise TypeError(f"queries must be float16 or bfloat16, not {queries.dtype}")
    if queries.requires_grad and torch.is_grad_enabled():
        raise ValueError("paged_attention has no backward pass: call it under torch.no_grad()")
    if hq < 1 or hq % st.n_kv_heads:
        raise ValueError(f"{hq} query heads do not share {st.n_kv_heads} KV heads")
    q = _rows("queries", queries, (n, hq, st.head_dim), dev)
    width = block_table.shape[1]
    _index("lengths", lengths, (r,), dev)
    _index("block_table", block_table, (r, width), dev)
    _index("token_starts", token_starts, (r + 1,), dev)
    zero_rest = out is None
    if out is None:
        out = torch.empty((n, hq, st.head_dim), dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or \
            not out.is_contiguous():
        raise ValueError(f"out must be contiguous {q.dtype} {tuple(q.shape)} on {dev}")
    if n == 0:
        return out
    if r == 0:
        return out.zero_() if zero_rest else out
    max_new = max(1, min(n, n - r + 1 if max_new is None else max_new))
    max_length = max(1, min(width * st.page_size, max_length or width * st.page_size))
    at = ctypes.addressof(st)
    need = _hip.load_library().ss_paged_attn_workspace_bytes(at, n, r, hq, max_new, max_length)
    # of this call alone: calls on other streams and captured graphs have their own
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _launch("ss_paged_attn", dev, at, q.data_ptr(), _hip.dtype_code(q.dtype), n, q.stride(0),
            q.stride(1), hq, block_table.data_ptr(), width, lengths.data_ptr(),
            token_starts.data_ptr(), r, float(scale), int(causal), max_new, max_length,
            out.data_ptr(), int(zero_rest), _hip.ptr(ws), need)
    return out
