"""Decode over shared prefixes: ``mla_decode_shared``.

No counterpart in the reference, which reads every sequence's cache on its
own (src/triton_mla/kernel.py:83-123). Where sequences begin with the same
pages (samples of one prompt, a system prompt), the rows of a whole group
attend to those pages once (csrc/mla_decode_shared.hip).
"""

from __future__ import annotations

import functools

import torch

from . import _native
from . import kernel as _k


def _sharing_pays(rows, batch, groups, capacity, fp8):
    """Whether attending to the prefixes once for their groups is faster than
    ``mla_decode``, which reads them per sequence: from what the host knows,
    the rows of a sequence (query tokens x heads) and the cache that a batch of
    full block tables would read. Measured (us, shared / mla_decode):

      * Sequences whose rows fill whole blocks of 128 leave no matrix work to
        save, and the bytes of shared pages come from the caches: 32 x 128 heads
        over 2K 49 / 42, 8K 95 / 87, 32K 294 / 272; 16 x 2 tokens x 128 heads
        93 / 86; fp8 over 32K 401 / 347.
      * Otherwise up to a certain number of bytes the merge of two more
        partials costs more than it saves. 16-bit caches, about 150 MB: 16
        heads, 41 MB 26 / 22, 153 MB 38 / 37, 155 MB 33 / 35, 317 MB 39 / 50, 2.4
        GB 94 / 263; 64 heads, 90 MB 43 / 34, 153 MB 44 / 47, 317 MB 66 / 68. fp8,
        about 75 MB: 32 heads, 45 MB 42 / 34, 76 MB 43 / 49, 158 MB 57 / 75; but
        more where 16 rows or fewer run the kernel that streams codes for 16
        heads: 77 MB 38 / 28, 158 MB 46 / 36 (it reads 4.8 TB/s).
      * Under 4,096 tokens (fp8: 8,192) a row has few partials, and mla_decode's,
        rounded to the 16-bit type, show in the result (1.5 to 1.9 times the error
        of its own rounding, 1.0 to 1.3 here): those calls share whatever their
        size, and so do those of several groups, whose sequences may be short in
        a long table.
    """
    if groups > 1 or capacity < (8192 if fp8 else 4096):
        return True
    if rows % 128 == 0:
        return False
    least = 150e6 if not fp8 else 350e6 if rows <= 16 else 75e6
    return batch * capacity * 576 * (1 if fp8 else 2) >= least


def _ints(t, device):
    if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
        t = t.to(device=device, dtype=torch.int32).contiguous()
    return t


@functools.lru_cache(maxsize=256)
def _space(device, batch, rows, groups, workers):
    """What kernel._workspace takes to hand out the stream's workspace."""
    space = _k._CallShape()
    space.dev_idx, space.device = device.index, device
    space.ws_bytes = _native.load().tmla_shared_workspace_bytes(batch, rows, groups, workers)
    space.ws_alloc = max(space.ws_bytes, 16)
    return space


def mla_decode_shared(
    q: torch.Tensor,
    kv_cache: torch.Tensor,
    cache_seqlens: torch.Tensor,
    block_table: torch.Tensor,
    prefix_lens,
    group_starts: torch.Tensor = None,
    head_dim_v: int = 512,
    softmax_scale: float = None,
    return_lse: bool = False,
    kv_scale=None,
    share: bool = None,
):
    """``mla_decode`` of a batch whose sequences share prefixes.

    The batch is cut into groups of consecutive sequences; the first tokens of
    a group's sequences lie in the same pages, and the group attends to them
    once. The result is ``mla_decode``'s, up to the rounding of split
    partials (finer here, see csrc/mla_decode_shared.hip).

    Args:
        q, kv_cache, cache_seqlens, head_dim_v, softmax_scale, return_lse:
            as ``mla_decode`` takes them (one query token a sequence, or
            [batch, q_len, num_heads, D]), at head_dim_v 512 and rope dim 64.
        block_table: [batch, max_blocks_per_seq] page indices (required: only
            pages can be shared).
        prefix_lens: tokens that the sequences of each group share: int32
            [groups], or one int for all. The first cdiv(prefix, page_size)
            entries of a group's rows of the block table name pages with the
            same contents in those tokens (the same pages, normally); they are
            read through the group's first sequence that holds a token. Less
            than the whole may be shared: whole 64-token tiles are, and no more
            than the shortest sequence of the group holds (sequences of length
            0 aside), so any value is safe, up to that promise.
        group_starts: int32 [groups + 1], ascending: group g is the sequences
            [group_starts[g], group_starts[g + 1]); sequences outside every
            group share nothing. None: the whole batch is one group.
        kv_scale: scales of an fp8 cache, as ``mla_decode`` takes them, one per
            page or one for the whole cache (scales per token are refused), on
            pages of a power of two of at least 32 tokens.
        share: True attends to every prefix once, False runs ``mla_decode``,
            None (default) chooses by the sizes: mla_decode where it is the
            faster of the two and its contexts are long (_sharing_pays).

    Returns:
        out [batch, num_heads, head_dim_v] in q.dtype (and lse [batch,
        num_heads] float32), with the q_len dim for a 4-D q. A head's row that
        meets a value of infinity or NaN within its tokens is NaN throughout
        (mla_decode: in that dim, where the score is -inf); behind them the
        cache may hold anything.
    """
    if kv_cache.dim() == 4:
        assert kv_cache.shape[2] == 1, "MLA uses a single shared latent KV head"
        kv_cache = kv_cache.squeeze(2)
    multi_token = q.dim() == 4
    q_len = 1
    if multi_token:
        q_len = q.shape[1]
        assert q_len >= 1, "q must hold at least one query token"
        if q.stride(1) != q.shape[2] * q.stride(2):
            q = q.contiguous()
        q = q.reshape(q.shape[0], q_len * q.shape[2], q.shape[3])
    assert q.dim() == 3 and kv_cache.dim() == 3
    batch, rows, d_qk = q.shape
    num_heads = rows // q_len
    d_rope = d_qk - head_dim_v
    assert kv_cache.shape[-1] == d_qk
    assert q.stride(-1) == 1 and kv_cache.stride(-1) == 1
    if block_table is None:
        raise ValueError("mla_decode_shared needs a paged cache (block_table): only pages can be shared")
    fp8 = kv_cache.dtype in _k._FP8_CACHE
    if fp8:
        if kv_scale is None:
            raise ValueError("an fp8 kv_cache needs kv_scale (its dequantisation scales)")
        kv_cache = kv_cache.view(torch.uint8)
        page = kv_cache.shape[1]
        if page % 32 or page & (page - 1):
            raise NotImplementedError("mla_decode_shared needs an fp8 cache's pages to be a power of two of at least "
                                      "32 tokens")
        if torch.is_tensor(kv_scale) and kv_scale.dim() == 2 and kv_scale.numel() > 1:
            raise NotImplementedError("mla_decode_shared takes one scale per page or per cache, not per token")
    else:
        assert kv_scale is None, "kv_scale applies to an fp8 (float8_e4m3fn) kv_cache only"
        assert q.dtype == kv_cache.dtype
    if q.device.type != "cuda" or kv_cache.device != q.device:
        raise RuntimeError("triton_mla.mla_decode_shared runs on the GPU only: q and kv_cache must be "
                           "on the same HIP device")
    if q.dtype not in _k._DTYPES:
        raise NotImplementedError(f"mla_decode_shared supports bf16 and fp16 inputs, got {q.dtype}")
    if (head_dim_v, d_rope) not in _k._SUPPORTED_DIMS:
        raise NotImplementedError(
            f"mla_decode_shared is built for head_dim_v=512, rope_dim=64; got {head_dim_v}, {d_rope}")
    if softmax_scale is None:
        softmax_scale = d_qk ** -0.5
    device = q.device
    cache_seqlens = _ints(cache_seqlens, device)
    assert cache_seqlens.shape == (batch,), "cache_seqlens must be [batch]"
    if block_table.dtype is not torch.int32 or block_table.device != device:
        block_table = block_table.to(device=device, dtype=torch.int32)
    if block_table.stride(-1) != 1:
        block_table = block_table.contiguous()
    assert block_table.dim() == 2 and block_table.shape[0] == batch
    groups, starts_ptr = 1, None
    if group_starts is not None:
        group_starts = _ints(group_starts, device)
        assert group_starts.dim() == 1 and group_starts.shape[0] >= 2, "group_starts must be [groups + 1]"
        groups, starts_ptr = group_starts.shape[0] - 1, group_starts.data_ptr()
    prefix_len, prefix_ptr = 0, None
    if torch.is_tensor(prefix_lens):
        prefix_lens = _ints(prefix_lens, device)
        assert prefix_lens.shape == (groups,), "prefix_lens must be [groups] (or one int)"
        prefix_ptr = prefix_lens.data_ptr()
    else:
        prefix_len = int(prefix_lens)
        if not 0 <= prefix_len < 1 << 31:
            raise ValueError("prefix_lens must be in [0, 2^31)")
    if share is None:
        share = _sharing_pays(rows, batch, groups, block_table.shape[1] * kv_cache.shape[1], fp8)
    if not share:
        return _k.mla_decode(q.unflatten(1, (q_len, num_heads)) if multi_token else q, kv_cache, cache_seqlens,
                             block_table, head_dim_v, softmax_scale, return_lse=return_lse, kv_scale=kv_scale)
    shape = (batch, q_len, num_heads) if multi_token else (batch, num_heads)
    out = torch.empty(*shape, head_dim_v, dtype=q.dtype, device=device)
    lse = torch.empty(*shape, dtype=torch.float32, device=device) if return_lse else None
    if batch:
        if kv_cache.shape[0] == 0 or kv_cache.shape[1] == 0:
            raise ValueError("kv_cache holds no tokens")
        if not _k._aligned(q):
            q = q.clone(memory_format=torch.contiguous_format)
        if not _k._aligned(kv_cache, 16 if fp8 else 8):
            kv_cache = kv_cache.clone(memory_format=torch.contiguous_format)
        scale_ptr, scale_stride = None, 0
        if fp8:
            kv_scale, scale_stride, _ = _k._scale_layout(kv_scale, kv_cache.shape[0], kv_cache.shape[1], device)
            scale_ptr = kv_scale.data_ptr()
        lib = _native.load_gil_held()  # the stream's workspace is shared by its calls
        workers = _k._num_sms(device)
        call = _space(device, batch, rows, groups, workers)
        with _k._OnDevice(call.dev_idx):
            stream = _k._raw_stream(call.dev_idx)
            ws, ws_ptr = _k._workspace(call, stream)
            rc = lib.tmla_mla_decode_shared(
                q.data_ptr(), q.stride(0), q.stride(1), kv_cache.data_ptr(), kv_cache.stride(0), kv_cache.stride(1),
                kv_cache.shape[0], kv_cache.shape[1], scale_ptr, scale_stride, block_table.data_ptr(), block_table.stride(0),
                block_table.shape[1], cache_seqlens.data_ptr(), prefix_ptr, prefix_len, starts_ptr, groups, batch,
                q_len, num_heads, head_dim_v, d_rope, _native.DTYPE_CODE[q.dtype], float(softmax_scale), workers,
                out.data_ptr(), out.stride(0), out.stride(-2), None if lse is None else lse.data_ptr(), ws_ptr,
                call.ws_bytes, stream)
        if rc:
            _native.check(rc, "tmla_mla_decode_shared")
    return (out, lse) if return_lse else out
