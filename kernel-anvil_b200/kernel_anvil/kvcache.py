"""The paged key/value cache and the attention over it, on the libanvil C ABI (include/anvil.h).

What a decoder does between its k/v products and its output product:

  cache = PagedKVCache(num_pages, page_size, kv_heads, head_dim, "Q8_0")   one layer's cache
  kv_write(cache, k, v, page_table, q_start, kv_len)                       new tokens into their pages
  out = paged_attention(q, cache, page_table, q_start, kv_len)             new tokens over all cached ones
  k, v = kv_read(cache, page_table, start, rows)                           cached tokens as values again

A batch is ragged: sequence b has the packed rows q_start[b] .. q_start[b+1] of q, k and v (one
token of a decode step, a few to verify, a chunk of a prompt, or none), and kv_len[b] cached tokens,
the new ones included, in the pages page_table[b].  All of that stays on the device, so a captured
CUDA graph replays with other lengths.  Kernels run on torch's current stream of the tensors' device.
There is no CPU path and no backward pass.

An entry of page_table, q_start or kv_len that is out of range is cut or skipped, never followed, and
sets BAD_PAGE in ``kernel_anvil.mmvq.take_device_status()``.
"""
from __future__ import annotations

import ctypes

import torch

from kernel_anvil import _native
from kernel_anvil._native import ANVIL_ERR_INVALID, ANVIL_FLAG_ZERO_REST, AnvilError, check

# kind -> (ggml type id, dtype of the codes, codes per head value as a divisor, values per scale)
KINDS = {
    "F16": (1, torch.float16, 1, 0),
    "BF16": (30, torch.bfloat16, 1, 0),
    "Q8_0": (8, torch.int8, 1, 32),
    "Q4_0": (2, torch.uint8, 2, 32),
}
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
HEAD_DIMS = (64, 128, 256)
BAD_PAGE = 2  # bit of kernel_anvil.mmvq.take_device_status()


class _Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in ("kind", "num_pages", "kv_heads", "page_size", "head_dim")] + [
        (n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")]


class _Batch(ctypes.Structure):
    _fields_ = [("page_table", ctypes.c_void_p), ("page_table_stride", ctypes.c_int64)] + [
        (n, ctypes.c_int) for n in ("max_pages", "batch", "total")] + [
        ("start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p)]


def _bad(msg: str) -> AnvilError:
    return AnvilError(ANVIL_ERR_INVALID, msg)


class PagedKVCache:
    """One layer's keys and values in pages.

    k, v: (num_pages, kv_heads, page_size, head_dim) of float16 / bfloat16 / int8, or
    (..., head_dim / 2) uint8 for Q4_0; k_scale, v_scale: (num_pages, kv_heads, page_size,
    head_dim / 32) float16 for the quantised kinds, else None.  head_dim 64, 128 or 256;
    page_size a power of two up to 1024.
    """

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, kind: str = "Q8_0",
                 device="cuda"):
        if kind not in KINDS:
            raise _bad(f"cache kind {kind!r} is not one of {', '.join(KINDS)}")
        if head_dim not in HEAD_DIMS:
            raise _bad(f"head_dim={head_dim} is not one of {HEAD_DIMS}")
        _, dtype, div, per = KINDS[kind]
        shape = (num_pages, kv_heads, page_size)
        new = lambda last, dt: torch.zeros(shape + (last,), dtype=dt, device=device)  # noqa: E731
        self._take(kind, new(head_dim // div, dtype), new(head_dim // div, dtype),
                   new(head_dim // per, torch.float16) if per else None,
                   new(head_dim // per, torch.float16) if per else None)

    @classmethod
    def from_buffers(cls, kind: str, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache on tensors that the caller holds (used in place).

        Scales above 512 (Q8_0) or 8188 (Q4_0) in magnitude, which kv_write never makes, pass fp16's range with
        their codes: paged_attention takes such a block as NaN, kv_read gives its values.
        """
        self = cls.__new__(cls)
        self._take(kind, k, v, k_scale, v_scale)
        return self

    def _take(self, kind, k, v, k_scale, v_scale):
        if kind not in KINDS:
            raise _bad(f"cache kind {kind!r} is not one of {', '.join(KINDS)}")
        ggml, dtype, div, per = KINDS[kind]
        shape, device = k.shape, k.device
        if len(shape) != 4:
            raise _bad("k and v are (num_pages, kv_heads, page_size, row)")
        pages, heads, size, last = shape
        dim = last * div
        if dim not in HEAD_DIMS:
            raise _bad(f"head_dim={dim} is not one of {HEAD_DIMS}")
        if not 1 <= size <= 1024 or size & (size - 1):
            raise _bad(f"page_size={size} is not a power of two up to 1024")
        if pages < 1 or heads < 1:
            raise _bad("a cache has at least one page and one head")
        scales = (k_scale, v_scale) if per else ()
        for t in (k, v):
            if t.dtype != dtype or t.shape != shape or t.device != device or not t.is_contiguous():
                raise _bad(f"k and v of a {kind} cache are contiguous {dtype} tensors of one shape on one device")
        for t in scales:
            if t is None or t.dtype != torch.float16 or t.shape != (pages, heads, size, dim // per) or \
                    t.device != device or not t.is_contiguous():
                raise _bad(f"scales of a {kind} cache are contiguous float16 (num_pages, kv_heads, page_size, "
                           f"{dim // per}) tensors on its device")
        if not per and (k_scale is not None or v_scale is not None):
            raise _bad(f"a {kind} cache has no scales")
        self.kind, self.k, self.v, self.k_scale, self.v_scale = kind, k, v, k_scale, v_scale
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, dim
        self.device = device
        self._c = _Cache(ggml, pages, heads, size, dim, k.data_ptr(), v.data_ptr(),
                         k_scale.data_ptr() if per else None, v_scale.data_ptr() if per else None)
        self._ref = ctypes.byref(self._c)
        self._work: dict[tuple, int] = {}  # attention scratch by (batch, rows, pages, heads): it depends on these alone

    @property
    def bytes_per_token(self) -> int:
        """Bytes that one token's keys and values take in the cache."""
        per = KINDS[self.kind][3]
        row = self.k.shape[3] * self.k.element_size() + (2 * self.head_dim // per if per else 0)
        return 2 * self.kv_heads * row

    def __repr__(self):
        return (f"PagedKVCache(num_pages={self.num_pages}, page_size={self.page_size}, kv_heads={self.kv_heads}, "
                f"head_dim={self.head_dim}, kind={self.kind!r}, device={str(self.device)!r})")


_INT = torch.int32


def _batch(cache: PagedKVCache, page_table, start, kv_len, total: int) -> _Batch:
    dev = cache.device
    if dev.type != "cuda":
        raise _bad("the cache must be on a CUDA device (no CPU path)")
    shape = start.shape
    if len(shape) != 1 or shape[0] < 1 or start.dtype != _INT or not start.is_contiguous():
        raise _bad("the starts are a contiguous int32 tensor of batch + 1 values")
    n = shape[0] - 1
    shape = page_table.shape
    if len(shape) != 2 or shape[0] != n or page_table.dtype != _INT:
        raise _bad(f"page_table is an int32 tensor ({n}, pages) with contiguous rows")
    pages = shape[1]
    step, inner = page_table.stride()
    if pages > 1 and inner != 1:
        raise _bad(f"page_table is an int32 tensor ({n}, pages) with contiguous rows")
    if start.device != dev or page_table.device != dev:
        raise _bad("page_table, starts and lengths must be on the cache's device")
    lens = None
    if kv_len is not None:
        if kv_len.dtype != _INT or kv_len.shape != (n,) or not kv_len.is_contiguous():
            raise _bad(f"lengths and first positions are contiguous int32 tensors of {n} values")
        if kv_len.device != dev:
            raise _bad("page_table, starts and lengths must be on the cache's device")
        lens = kv_len.data_ptr()
    if total > 0x7FFFFFFF:
        raise _bad("more than 2^31 - 1 rows in one call")
    return _Batch(page_table.data_ptr(), step if n > 1 else pages, pages, n, total, start.data_ptr(), lens)


def _rows(name: str, x: torch.Tensor, cache: PagedKVCache, heads: int | None) -> torch.Tensor:
    """x as (rows, heads, head_dim) whose rows start on 16-byte boundaries (copied where they do not)."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    shape = x.shape
    if len(shape) != 3 or shape[2] != cache.head_dim or (heads is not None and shape[1] != heads):
        raise _bad(f"{name} is (rows, {heads or 'heads'}, {cache.head_dim}), got {tuple(shape)}")
    if x.device != cache.device:
        raise _bad(f"{name} must be on the cache's device {cache.device}, got {x.device}")
    if x.dtype not in DTYPES:
        raise _bad(f"{name} must be float32, float16 or bfloat16, got {x.dtype}")
    if x.requires_grad and torch.is_grad_enabled():
        raise _bad(f"{name} requires grad, and the cache's operators have no backward pass")
    if torch.autograd.forward_ad.unpack_dual(x).tangent is not None:
        raise _bad(f"{name} carries a tangent, and the cache's operators have no forward-mode derivative")
    row, head, inner = x.stride()
    n = 4 if x.dtype == torch.float32 else 8  # values in 16 bytes
    if inner != 1 or row % n or head % n or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
    return x


def _call(cache: PagedKVCache, fn, *args) -> None:
    """fn(*args, stream) on the cache's device and torch's current stream there.

    (By the functions behind torch.cuda.current_stream and current_device, which build objects: 2 us of a call's 17.
    Looked up here, since a torch without CUDA lacks them.)
    """
    index = cache.device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        status = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            status = fn(*args, stream)
    if status < 0:
        check(status)


def kv_write(cache: PagedKVCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
             q_start: torch.Tensor, kv_len: torch.Tensor) -> None:
    """Puts new tokens' keys and values into the cache, quantised by its kind's rule.

    k, v: (rows, kv_heads, head_dim), float32 / float16 / bfloat16, any row and head strides.  Row i of
    sequence b goes to position kv_len[b] - (q_start[b+1] - q_start[b]) + i.  Rows behind
    q_start[-1] are left out, and so is a sequence with an entry out of range: no cached token is lost to
    one.  Positions that two sequences of one call share (a common page) must not be
    among those written: both would write them.  The codes are those of the GGUF type for exact arithmetic
    (include/anvil.h); F16 and BF16 round.
    """
    k, v = _rows("k", k, cache, cache.kv_heads), _rows("v", v, cache, cache.kv_heads)
    if k.shape != v.shape or k.dtype != v.dtype:
        raise _bad("k and v must have one shape and type")
    b = _batch(cache, page_table, q_start, kv_len, k.shape[0])
    _call(cache, _native.lib().anvil_kv_write, cache._ref, ctypes.byref(b), DTYPES[k.dtype], k.data_ptr(),
          k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1))


def kv_read(cache: PagedKVCache, page_table: torch.Tensor, start: torch.Tensor, rows: int,
            first: torch.Tensor | None = None, dtype: torch.dtype = torch.float32,
            out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v) of cached tokens, each (rows, kv_heads, head_dim) of `dtype`: rows start[b] .. start[b+1]
    are the positions first[b], first[b] + 1, ... (first None: from 0) of sequence b.

    A position without a page reads as zeros; so do rows of no sequence (before start[0] and behind start[-1]),
    except in a given `out`, where they are left as they were.
    """
    if dtype not in DTYPES:
        raise _bad(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    b = _batch(cache, page_table, start, first, rows)
    b.kv_len = None
    shape = (rows, cache.kv_heads, cache.head_dim)
    flags = 0 if out is not None else ANVIL_FLAG_ZERO_REST
    if out is None:
        out = (torch.empty(shape, dtype=dtype, device=cache.device),
               torch.empty(shape, dtype=dtype, device=cache.device))
    for t in out:
        if t.shape != shape or t.dtype != dtype or t.device != cache.device or not t.is_contiguous() or \
                t.data_ptr() % 16:
            raise _bad(f"out is two contiguous 16-byte aligned {dtype} tensors {shape} on the cache's device")
    if abs(out[0].data_ptr() - out[1].data_ptr()) < out[0].numel() * out[0].element_size():
        raise _bad("the two tensors of out overlap")
    _call(cache, _native.lib().anvil_kv_read_ex, cache._ref, ctypes.byref(b),
          first.data_ptr() if first is not None else None, DTYPES[dtype], out[0].data_ptr(), out[1].data_ptr(),
          flags)
    return out


def paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor, q_start: torch.Tensor,
                    kv_len: torch.Tensor, scale: float | None = None, causal: bool = True,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of each row of q over its sequence's cached tokens, (rows, heads, head_dim).

    q: (rows, heads, head_dim), float16 or bfloat16 (an F16 / BF16 cache takes its own type), any row
    and head strides; heads a multiple of the cache's kv_heads, query head h reading key/value head
    h // (heads // kv_heads).  Row i of sequence b sees its kv_len[b] cached tokens, or, causal,
    those up to its own position kv_len[b] - q_len + i; a row that sees none (or whose scores are all -inf)
    is zeros.  scale
    defaults to head_dim ** -0.5.  Rows of no sequence (before q_start[0] and behind q_start[-1]: the padding of a
    captured step) are zeros, except in a given `out`, where they are left as they were.  out may be q itself, but not
    overlap it otherwise.
    """
    q = _rows("q", q, cache, None)
    heads = q.shape[1]
    if q.dtype == torch.float32:
        raise _bad("q must be float16 or bfloat16 (the products run in 16 bits)")
    if heads < 1 or heads % cache.kv_heads:
        raise _bad(f"heads={heads} is not a multiple of kv_heads={cache.kv_heads}")
    if cache.k_scale is None and q.dtype != cache.k.dtype:
        raise _bad(f"a {cache.kind} cache takes q of its own type, got {q.dtype}")
    b = _batch(cache, page_table, q_start, kv_len, q.shape[0])
    flags = 0 if out is not None else ANVIL_FLAG_ZERO_REST
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != cache.device or \
            not out.is_contiguous() or out.data_ptr() % 16:
        raise _bad("out is a contiguous 16-byte aligned tensor of q's shape and type on the cache's device")
    elif out.numel() and not (out.data_ptr() == q.data_ptr() and q.is_contiguous()):  # (q itself is: rows are read first)
        span = 1 + sum((n - 1) * step for n, step in zip(q.shape, q.stride()))
        at = (out.data_ptr() - q.data_ptr()) // q.element_size()
        if -out.numel() < at < span:
            raise _bad("out overlaps q without being q")
    if kv_len is None:
        raise _bad("kv_len is needed")
    lib, ref = _native.lib(), ctypes.byref(b)
    key = (b.batch, b.total, b.max_pages, heads)
    need = cache._work.get(key)
    if need is None:
        need = check(lib.anvil_paged_attention_workspace(cache._ref, ref, heads))
        if len(cache._work) > 4096:  # ragged totals of a long-lived server
            cache._work.clear()
        cache._work[key] = need
    # scratch of this call, from torch's allocator: its memory follows the stream and, in a capture, the graph
    work = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    _call(cache, lib.anvil_paged_attention_ex, cache._ref, ref, DTYPES[q.dtype], q.data_ptr(), q.stride(0),
          q.stride(1), heads, cache.head_dim ** -0.5 if scale is None else float(scale), int(bool(causal)),
          out.data_ptr(), work.data_ptr() if work is not None else None, need, flags)
    return out
