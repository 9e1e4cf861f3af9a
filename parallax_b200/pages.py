"""Pages of a paged KV cache: copying, forking rows, compacting, freeing.

The cache is the one :func:`parallax_attn_with_kvcache` reads: pools ``k_cache`` / ``v_cache`` ``(n_pages, page_size, H_kv, D)``
with a power-of-two ``page_size``, a ``page_table`` ``(B, max_num_blocks)`` int32 and ``seqused_k`` ``(B,)`` int32.  The ACTIVE
entries of a row are the first ``ceil(seqused_k / page_size)``; a page is live while some row's active entry names it, and free
otherwise.  There is no other bookkeeping: what a table holds beyond its active entries is never looked at.

Pools are written in place; tables and lengths come back as new tensors.  A model has a pair of pools per layer under ONE table: call
once a layer, each time with the table and lengths from BEFORE; every call returns the same new ones, to be used from then on (a layer
that is given the new table would fork or compact again).  Everything is decided on the device -- nothing here
waits for it, so the calls can be captured in a CUDA graph -- and numbers out of range (a page outside the pool, a row outside
the table) are passed over.  (The reference names paged caches but does not implement them:
parallax/cute/parallax_decode.py:1578-1580.)
"""
from __future__ import annotations

import ctypes as C
from typing import Tuple

import torch
from torch import Tensor

from . import _cabi
from .ops import _ptr, _stream, eager_host


def _pool(k: Tensor, v: Tensor) -> _cabi.PagePool:
    p = _cabi.PagePool()
    p.k, p.v = k.data_ptr(), v.data_ptr()
    p.n_pages, p.page_size, p.heads_kv, p.head_dim = k.shape
    p.k_stride_p, p.k_stride_t, p.k_stride_h = k.stride()[:3]
    p.v_stride_p, p.v_stride_t, p.v_stride_h = v.stride()[:3]
    return p


def _workspace(n_pages: int, batch: int, n_forks: int, device) -> Tensor:
    need = C.c_size_t(0)
    _cabi.check(_cabi.lib().plx_pages_workspace_bytes(n_pages, batch, n_forks, C.byref(need)), "plx_pages_workspace_bytes")
    return torch.empty(need.value, device=device, dtype=torch.uint8)


@torch.library.custom_op("plx::pages_copy", mutates_args=("k_cache", "v_cache"), device_types="cuda")
def pages_copy(k_cache: Tensor, v_cache: Tensor, src: Tensor, dst: Tensor) -> None:
    pool = _pool(k_cache, v_cache)
    with torch.cuda.device(k_cache.device):
        st = _cabi.lib().plx_pages_copy(C.byref(pool), _ptr(src), _ptr(dst), src.numel(), _stream(k_cache.device))
    _cabi.check(st, "plx_pages_copy")


@torch.library.custom_op("plx::pages_fork", mutates_args=("k_cache", "v_cache"), device_types="cuda")
def pages_fork(k_cache: Tensor, v_cache: Tensor, page_table: Tensor, seqused_k: Tensor, parents: Tensor,
               children: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    table, lens, missing = torch.empty_like(page_table), torch.empty_like(seqused_k), seqused_k.new_empty(1)
    pool = _pool(k_cache, v_cache)
    ws = _workspace(k_cache.shape[0], table.shape[0], parents.numel(), k_cache.device)
    with torch.cuda.device(k_cache.device):
        st = _cabi.lib().plx_pages_fork(C.byref(pool), _ptr(page_table), _ptr(seqused_k), table.shape[0], table.shape[1], _ptr(parents),
                                        _ptr(children), parents.numel(), _ptr(table), _ptr(lens), _ptr(missing), _ptr(ws),
                                        C.c_size_t(ws.numel()), _stream(k_cache.device))
    _cabi.check(st, "plx_pages_fork")
    return table, lens, missing


@pages_fork.register_fake
def _(k_cache, v_cache, page_table, seqused_k, parents, children):
    return torch.empty_like(page_table), torch.empty_like(seqused_k), seqused_k.new_empty(1)


@torch.library.custom_op("plx::pages_compact", mutates_args=("k_cache", "v_cache"), device_types="cuda")
def pages_compact(k_cache: Tensor, v_cache: Tensor, page_table: Tensor, seqused_k: Tensor) -> Tuple[Tensor, Tensor]:
    table, n_live = torch.empty_like(page_table), seqused_k.new_empty(1)
    pool = _pool(k_cache, v_cache)
    ws = _workspace(k_cache.shape[0], table.shape[0], 0, k_cache.device)
    with torch.cuda.device(k_cache.device):
        st = _cabi.lib().plx_pages_compact(C.byref(pool), _ptr(page_table), _ptr(seqused_k), table.shape[0], table.shape[1], _ptr(table),
                                           _ptr(n_live), _ptr(ws), C.c_size_t(ws.numel()), _stream(k_cache.device))
    _cabi.check(st, "plx_pages_compact")
    return table, n_live


@pages_compact.register_fake
def _(k_cache, v_cache, page_table, seqused_k):
    return torch.empty_like(page_table), seqused_k.new_empty(1)


@torch.library.custom_op("plx::pages_free", mutates_args=(), device_types="cuda")
def pages_free(page_table: Tensor, seqused_k: Tensor, rows: Tensor, n_pages: int, page_size: int) -> Tuple[Tensor, Tensor, Tensor]:
    lens, free, n_free = torch.empty_like(seqused_k), seqused_k.new_empty(n_pages), seqused_k.new_empty(1)
    need = C.c_size_t(0)
    _cabi.check(_cabi.lib().plx_pages_free_workspace_bytes(n_pages, C.byref(need)), "plx_pages_free_workspace_bytes")
    ws = torch.empty(need.value, device=page_table.device, dtype=torch.uint8)
    with torch.cuda.device(page_table.device):
        st = _cabi.lib().plx_pages_free(_ptr(page_table), _ptr(seqused_k), page_table.shape[0], page_table.shape[1], _ptr(rows), rows.numel(),
                                        n_pages, page_size, _ptr(lens), _ptr(free), _ptr(n_free), _ptr(ws), C.c_size_t(ws.numel()),
                                        _stream(page_table.device))
    _cabi.check(st, "plx_pages_free")
    return lens, free, n_free


@pages_free.register_fake
def _(page_table, seqused_k, rows, n_pages, page_size):
    return torch.empty_like(seqused_k), seqused_k.new_empty(n_pages), seqused_k.new_empty(1)


# --------------------------------------------------------------------------- #
# checks
# --------------------------------------------------------------------------- #
def _check_pool(name: str, k: Tensor, v: Tensor) -> None:
    if k.dtype not in (torch.bfloat16, torch.float16) or v.dtype != k.dtype:
        raise TypeError(f"{name} requires bf16 or fp16 pools of one type, got {k.dtype} and {v.dtype}")
    if k.ndim != 4 or v.shape != k.shape or k.numel() == 0:
        raise ValueError(f"{name}: k_cache and v_cache must both be (n_pages, page_size, H_kv, D), got {tuple(k.shape)} and {tuple(v.shape)}")
    _check_page_size(name, k.shape[1])
    if k.shape[3] % 8 != 0:
        raise NotImplementedError(f"{name}: head_dim must be a multiple of 8, got {k.shape[3]}")
    _check_cuda(name, k, v)
    for x in (k, v):
        # written in place: there is no copy that could be brought into another layout
        if x.stride(3) != 1 or any(s % 8 != 0 for s in x.stride()[:3]) or x.data_ptr() % 16 != 0:
            raise ValueError(f"{name}: pools need a contiguous head_dim axis, strides that are multiples of 8 and a 16-byte aligned base, got "
                             f"strides {tuple(x.stride())}")
        if any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
            raise ValueError(f"{name}: pools must not be expanded, got strides {tuple(x.stride())}")


def _check_page_size(name: str, page_size: int) -> None:
    if page_size < 1 or page_size & (page_size - 1):
        raise ValueError(f"{name}: page size must be a power of two, got {page_size}")


def _check_cuda(name: str, *tensors: Tensor) -> None:
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError(f"{name}: tensors must live on a CUDA device (there is no CPU path)")
        if t.device != tensors[0].device:
            raise ValueError(f"{name}: tensors live on {tensors[0].device} and {t.device}")


def _check_table(name: str, page_table: Tensor, seqused_k: Tensor) -> None:
    _check_ints(name, page_table=page_table, seqused_k=seqused_k)
    if page_table.ndim != 2 or page_table.numel() == 0:
        raise ValueError(f"{name}: page_table must have shape (B, max_num_blocks), got {tuple(page_table.shape)}")
    if tuple(seqused_k.shape) != (page_table.shape[0],):
        raise ValueError(f"{name}: seqused_k must have shape (B={page_table.shape[0]},), got {tuple(seqused_k.shape)}")


def _check_ints(name: str, **tensors: Tensor) -> None:
    for what, t in tensors.items():
        if t.dtype != torch.int32:
            raise TypeError(f"{name}: {what} must be int32, got {t.dtype}")


def _check_lists(name: str, **tensors: Tensor) -> None:
    _check_ints(name, **tensors)
    sizes = {t.numel() for t in tensors.values()}
    if any(t.ndim != 1 for t in tensors.values()) or len(sizes) != 1:
        raise ValueError(f"{name}: {' and '.join(tensors)} must be vectors of one length, got {[tuple(t.shape) for t in tensors.values()]}")


# --------------------------------------------------------------------------- #
# public calls
# --------------------------------------------------------------------------- #
def parallax_copy_pages(k_cache: Tensor, v_cache: Tensor, src: Tensor, dst: Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]``, of k and of v, for all i in one launch.

    ``src``, ``dst``: int32 vectors of one length.  Entries out of range (-1, say, to pad a list to a fixed length) are passed
    over.  No page may be a target twice, or a source and a target: what such a page holds afterwards is not defined.
    """
    host = eager_host()
    if host is not None and host.pages_copy(k_cache, v_cache, src, dst):
        return
    _check_pool("parallax_copy_pages", k_cache, v_cache)
    _check_lists("parallax_copy_pages", src=src, dst=dst)
    _check_cuda("parallax_copy_pages", k_cache, src, dst)
    if src.numel():
        pages_copy(k_cache, v_cache, src.contiguous(), dst.contiguous())


def parallax_fork_pages(k_cache: Tensor, v_cache: Tensor, page_table: Tensor, seqused_k: Tensor, parents: Tensor,
                        children: Tensor) -> Tuple[Tensor, Tensor, Tensor]:
    """Row ``children[i]`` becomes row ``parents[i]``, for parallel sampling and beams: ``(page_table, seqused_k, n_missing)``.

    ``parents``, ``children``: int32 vectors of row numbers.  Every parent is read as it was before the call; of a row mentioned twice
    among the children the last mention counts; pairs out of range are passed over.  A child shares the whole pages of its
    parent.  Where the last page is not full, its keys are copied to a page of the child's own: the lowest one that no row held
    before the call, in the order of the lists.  ``n_missing`` (one int32 on the device) counts the children for which there was
    none: their rows end with the whole pages (and the entry behind those is -1).
    """
    host = eager_host()
    res = None if host is None else host.pages_fork(k_cache, v_cache, page_table, seqused_k, parents, children)
    if res is not None:
        return res
    name = "parallax_fork_pages"
    _check_pool(name, k_cache, v_cache)
    _check_table(name, page_table, seqused_k)
    _check_lists(name, parents=parents, children=children)
    _check_cuda(name, k_cache, page_table, seqused_k, parents, children)
    if parents.numel() == 0:
        return page_table.clone(), seqused_k.clone(), seqused_k.new_zeros(1)
    return pages_fork(k_cache, v_cache, page_table.contiguous(), seqused_k.contiguous(), parents.contiguous(), children.contiguous())


def parallax_compact_pages(k_cache: Tensor, v_cache: Tensor, page_table: Tensor, seqused_k: Tensor) -> Tuple[Tensor, Tensor]:
    """Move the live pages to the front of the pool: ``(page_table, n_live)``.

    Of ``n_live`` live pages (one int32 on the device) the i-th from page ``n_live`` on goes to the i-th free page below it, and the
    tables follow; pages that are in place stay there, shared pages stay shared.  All pages from ``n_live`` on are free afterwards.
    """
    host = eager_host()
    res = None if host is None else host.pages_compact(k_cache, v_cache, page_table, seqused_k)
    if res is not None:
        return res
    name = "parallax_compact_pages"
    _check_pool(name, k_cache, v_cache)
    _check_table(name, page_table, seqused_k)
    _check_cuda(name, k_cache, page_table, seqused_k)
    return pages_compact(k_cache, v_cache, page_table.contiguous(), seqused_k.contiguous())


def parallax_free_pages(page_table: Tensor, seqused_k: Tensor, rows: Tensor, n_pages: int, page_size: int) -> Tuple[Tensor, Tensor, Tensor]:
    """Free rows: ``(seqused_k, free, n_free)``.

    The lengths of ``rows`` (int32 row numbers; none is fine, and only lists) become 0.  ``free`` ``(n_pages,)`` int32 holds the pages
    that are not live then, ascending, -1 behind the last; ``n_free`` (one int32 on the device) is their number.  A page that another
    row shares stays live.
    """
    host = eager_host()
    res = None if host is None else host.pages_free(page_table, seqused_k, rows, n_pages, page_size)
    if res is not None:
        return res
    name = "parallax_free_pages"
    _check_table(name, page_table, seqused_k)
    _check_lists(name, rows=rows)
    if n_pages < 1:
        raise ValueError(f"{name}: n_pages must be positive, got {n_pages}")
    _check_page_size(name, page_size)
    _check_cuda(name, page_table, seqused_k, rows)
    return pages_free(page_table.contiguous(), seqused_k.contiguous(), rows.contiguous(), int(n_pages), int(page_size))
