"""Pages of a latent cache: copying them, forking and ending sequences,
reserving pages for the tokens to come, compacting the pool.

No counterpart in the reference, which takes a block table that its caller
made (src/triton_mla/model.py:86-94 writes rows through one). What a serving
program keeps, all on the GPU:

    kv_cache     [num_pages, page_size, D] the pool (with kv_scale, if its
                 elements are fp8 codes)
    block_table  int32 [batch, width]: row b's pages in order. An entry outside
                 [0, num_pages) holds nothing; these functions write -1 there.
    cache_seqlens int32 [batch]
    page_refs    int32 [num_pages]: how many entries hold a page (a program may
                 add its own holds); a page with a count of 0 or less is free.

Tables, lengths and counts are returned as new tensors, the pool is written in
place. Choices go by order (the lowest free page first), so equal inputs give
equal results; nothing synchronises with the host, and every call can be
captured into a graph (csrc/cache_pages.hip).
"""

from __future__ import annotations

import functools

import torch

from . import _native
from . import kernel as _k


def _device_of(*tensors):
    dev = tensors[0].device
    if dev.type != "cuda" or any(t.device != dev for t in tensors):
        raise RuntimeError("triton_mla page operations run on the GPU only: all tensors on one HIP device")
    return dev


def _ints(t, name, device, shape=None):
    if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
        t = t.to(device=device, dtype=torch.int32).contiguous()
    if shape is not None:
        assert t.shape == shape, f"{name} must be {list(shape)}"
    return t


def _table(block_table):
    if block_table.dtype is not torch.int32:
        block_table = block_table.to(torch.int32)
    assert block_table.dim() == 2 and block_table.shape[1] >= 1, "block_table must be [batch, width]"
    return block_table if block_table.stride(1) == 1 else block_table.contiguous()


def _pool(kv_cache, kv_scale):
    """The pool's arguments of the C calls (and the tensors they point into)."""
    if kv_cache.dim() == 4:
        assert kv_cache.shape[2] == 1, "MLA uses a single shared latent KV head"
        kv_cache = kv_cache.squeeze(2)
    assert kv_cache.dim() == 3 and kv_cache.stride(-1) == 1, "kv_cache must be [num_pages, page_size, D]"
    pages, rows, dim = kv_cache.shape
    scale = (None, 0, 0, 0)
    if kv_scale is not None:
        assert kv_cache.element_size() == 1, "kv_scale applies to an fp8 (float8_e4m3fn) kv_cache only"
    if kv_scale is not None and torch.is_tensor(kv_scale) and kv_scale.numel() > 1:
        # written in place: as it lies, no copy of it
        if kv_scale.dtype != torch.float32 or kv_scale.device != kv_cache.device:
            raise ValueError("kv_scale must be float32 on the cache's device: its rows move with the pages")
        assert kv_scale.shape[0] == pages and (kv_scale.dim() == 1 or tuple(kv_scale.shape) == (pages, rows)), \
            f"kv_scale of shape [{pages}] or [{pages}, {rows}] expected"
        if pages > 1 and kv_scale.stride(0) == 0 or kv_scale.dim() == 2 and rows > 1 and kv_scale.stride(1) == 0:
            raise ValueError("kv_scale must not be an expanded tensor: its rows move with the pages")
        scale = (kv_scale.data_ptr(), kv_scale.stride(0), kv_scale.stride(1) if kv_scale.dim() == 2 else 0,
                 rows if kv_scale.dim() == 2 else 1)
    return (kv_cache.data_ptr(), kv_cache.stride(0), kv_cache.stride(1), pages, rows, dim, kv_cache.element_size(),
            *scale)


class _Space:
    """What kernel._workspace takes to hand out the stream's workspace."""

    __slots__ = ("dev_idx", "device", "ws_alloc", "ws_bytes")


@functools.lru_cache(maxsize=256)
def _space(device, pages, batch, pairs):
    space = _Space()
    space.device = device
    space.dev_idx = device.index
    space.ws_bytes = _native.load().tmla_pages_workspace_bytes(pages, batch, pairs)
    space.ws_alloc = max(space.ws_bytes, 16)
    return space


def _run(name, device, pages, batch, pairs, *args):
    """One C call on the current stream of `device`, with the stream's workspace
    (the GIL is held over its launches, as for the decode calls that share it)."""
    space = _space(device, pages, batch, pairs)
    with _k._OnDevice(space.dev_idx):
        stream = _k._raw_stream(space.dev_idx)
        ws, ws_ptr = _k._workspace(space, stream)
        rc = getattr(_native.load_gil_held(), name)(*args, ws_ptr, space.ws_bytes, stream)
    if rc:
        _native.check(rc, name)


def copy_pages(kv_cache, src, dst, kv_scale=None):
    """Page src[i] of the pool copied to page dst[i], for all i.

    Args:
        kv_cache: [num_pages, page_size, D] (or [..., 1, D]) of elements of 1,
            2 or 4 bytes, written in place.
        src, dst: [pairs] page ids.
        kv_scale: scales of an fp8 pool ([num_pages] or [num_pages,
            page_size]), which move with the pages; one scale for the whole
            pool (a number or one element) stays.

    Returns:
        int32 [1] on the device: the pairs that were refused. Refused, and
        left out, is a pair with an id outside the pool, one whose destination
        a later pair has too, and one whose source another pair writes (what
        it holds would depend on the order). A page may be copied onto itself.
    """
    device = _device_of(kv_cache)
    src, dst = _ints(src, "src", device), _ints(dst, "dst", device)
    assert src.dim() == 1 and src.shape == dst.shape, "src and dst must be [pairs]"
    pool = _pool(kv_cache, kv_scale)
    if pool[3] == 0:
        raise ValueError("kv_cache holds no pages")
    refused = torch.empty(1, dtype=torch.int32, device=device)
    _run("tmla_pages_copy", device, pool[3], 0, src.shape[0], *pool, src.data_ptr(), dst.data_ptr(), src.shape[0],
         refused.data_ptr())
    return refused


def fork_sequences(kv_cache, block_table, cache_seqlens, page_refs, parents, kv_scale=None):
    """Every row i of the batch becomes a copy of row parents[i].

    Forks a prompt into samples, draws beams anew and ends sequences in one
    call: the copies share their parent's full pages, and only a last page that
    is not full is copied, to the lowest free pages in the order of the rows.
    A parent's first copy keeps its last page and whatever it has reserved
    beyond it; a row that no row continues gives its pages back (also to the
    copies of this call).

    Args:
        kv_cache, kv_scale: the pool (``copy_pages``), written in place.
        block_table, cache_seqlens, page_refs: the state (this module's text).
        parents: int32 [batch]; a value outside [0, batch) leaves an empty row.

    Returns:
        (block_table, cache_seqlens, page_refs, missing): the new state and,
        int32 [1] on the device, how many free pages were lacking. If any
        were, nothing is done: the state returned is the one given.
    """
    device = _device_of(kv_cache, block_table, page_refs)
    table = _table(block_table)
    batch, width = table.shape
    pool = _pool(kv_cache, kv_scale)
    seqlens = _ints(cache_seqlens, "cache_seqlens", device, (batch,))
    parents = _ints(parents, "parents", device, (batch,))
    refs = _ints(page_refs, "page_refs", device, (pool[3],))
    new_table = torch.empty(batch, width, dtype=torch.int32, device=device)
    new_seqlens, new_refs = torch.empty_like(seqlens), torch.empty_like(refs)
    missing = torch.empty(1, dtype=torch.int32, device=device)
    _run("tmla_pages_fork", device, pool[3], batch, 0, *pool, table.data_ptr(), table.stride(0), batch, width,
         seqlens.data_ptr(), refs.data_ptr(), parents.data_ptr(), new_table.data_ptr(), new_seqlens.data_ptr(),
         new_refs.data_ptr(), missing.data_ptr())
    return new_table, new_seqlens, new_refs, missing


def free_sequences(block_table, cache_seqlens, page_refs, ended):
    """The sequences with ended[b] give their pages back: their rows hold
    nothing and have length 0 afterwards.

    Returns (block_table, cache_seqlens, page_refs), the new state."""
    device = _device_of(block_table, page_refs)
    table = _table(block_table)
    batch, width = table.shape
    seqlens = _ints(cache_seqlens, "cache_seqlens", device, (batch,))
    assert page_refs.dim() == 1, "page_refs must be [num_pages]"
    refs = _ints(page_refs, "page_refs", device)
    ended = ended.to(device=device, dtype=torch.bool).contiguous()
    assert ended.shape == (batch,), "ended must be [batch]"
    new_table = torch.empty(batch, width, dtype=torch.int32, device=device)
    new_seqlens, new_refs = torch.empty_like(seqlens), torch.empty_like(refs)
    _run("tmla_pages_free", device, refs.shape[0], batch, 0, table.data_ptr(), table.stride(0), batch, width,
         seqlens.data_ptr(), refs.data_ptr(), refs.shape[0], ended.data_ptr(), new_table.data_ptr(),
         new_seqlens.data_ptr(), new_refs.data_ptr())
    return new_table, new_seqlens, new_refs


def reserve_pages(block_table, cache_seqlens, page_refs, new_tokens, page_size):
    """Pages for new_tokens more tokens of every sequence: each entry of the
    first cdiv(length + new_tokens, page_size) of a row that holds no page gets
    one, the lowest free pages in the order of rows and columns.

    Args:
        new_tokens: an int, or int32 [batch] (below 0: none).
        page_size: tokens per page.

    Returns:
        (block_table, page_refs, missing): the new state and, int32 [1] on the
        device, how many pages were lacking: free ones, or columns of the
        table. If any were, nothing is done: the state returned is the one
        given.
    """
    device = _device_of(block_table, page_refs)
    table = _table(block_table)
    batch, width = table.shape
    seqlens = _ints(cache_seqlens, "cache_seqlens", device, (batch,))
    assert page_refs.dim() == 1, "page_refs must be [num_pages]"
    refs = _ints(page_refs, "page_refs", device)
    each, all_rows = None, 0
    if torch.is_tensor(new_tokens):
        each = _ints(new_tokens, "new_tokens", device, (batch,))
    else:
        all_rows = int(new_tokens)
        if not 0 <= all_rows < 1 << 31:
            raise ValueError("new_tokens must be in [0, 2^31)")
    new_table = torch.empty(batch, width, dtype=torch.int32, device=device)
    new_refs = torch.empty_like(refs)
    missing = torch.empty(1, dtype=torch.int32, device=device)
    _run("tmla_pages_reserve", device, refs.shape[0], batch, 0, table.data_ptr(), table.stride(0), batch, width,
         seqlens.data_ptr(), refs.data_ptr(), refs.shape[0], int(page_size), None if each is None else each.data_ptr(),
         all_rows, new_table.data_ptr(), new_refs.data_ptr(), missing.data_ptr())
    return new_table, new_refs, missing


def compact_pages(kv_cache, block_table, page_refs, kv_scale=None):
    """The pages in use brought to the front of the pool: with L pages in use,
    those behind the first L move, in order, to the free ones among them, and
    the table's entries follow.

    Returns:
        (block_table, page_refs, live): the new state and L, int32 [1] on the
        device: every page from L on is free.
    """
    device = _device_of(kv_cache, block_table, page_refs)
    table = _table(block_table)
    batch, width = table.shape
    pool = _pool(kv_cache, kv_scale)
    refs = _ints(page_refs, "page_refs", device, (pool[3],))
    new_table = torch.empty(batch, width, dtype=torch.int32, device=device)
    new_refs = torch.empty_like(refs)
    live = torch.empty(1, dtype=torch.int32, device=device)
    _run("tmla_pages_compact", device, pool[3], batch, 0, *pool, table.data_ptr(), table.stride(0), batch, width,
         refs.data_ptr(), new_table.data_ptr(), new_refs.data_ptr(), live.data_ptr())
    return new_table, new_refs, live
