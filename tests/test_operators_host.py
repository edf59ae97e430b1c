"""What mla_decode_shared and the page operations refuse, before any GPU work
(no GPU needed): the Python checks and the C entry points'."""

import ctypes
import os

import pytest
import torch

I32 = torch.int32


@pytest.fixture(scope="module")
def lib():
    from triton_mla import _native

    if not os.path.exists(_native.LIB_PATH):
        pytest.fail(f"HIP library not built: {_native.LIB_PATH} (run __graft_entry__.build())")
    return _native.load()


def _decode_args(**kw):
    args = dict(q=torch.zeros(2, 16, 576, dtype=torch.bfloat16), kv_cache=torch.zeros(4, 64, 576, dtype=torch.bfloat16),
                cache_seqlens=torch.ones(2, dtype=I32), block_table=torch.zeros(2, 2, dtype=I32), prefix_lens=64)
    args.update(kw)
    return args


@pytest.mark.parametrize("kw,error", [
    ({}, RuntimeError),  # CPU tensors
    ({"block_table": None}, ValueError),  # a dense cache shares nothing
    ({"kv_cache": torch.zeros(4, 64, 2, 576, dtype=torch.bfloat16)}, AssertionError),  # two kv heads
    ({"kv_cache": torch.zeros(4, 64, 512, dtype=torch.bfloat16)}, AssertionError),  # rows of another width
    ({"kv_cache": torch.zeros(4, 64, 576, dtype=torch.float16)}, AssertionError),  # another type
    ({"q": torch.zeros(2, 0, 16, 576, dtype=torch.bfloat16)}, AssertionError),  # no query token
])
def test_decode_refusals(kw, error):
    import triton_mla

    with pytest.raises(error):
        triton_mla.mla_decode_shared(**_decode_args(**kw))


def test_page_operations_refuse_cpu_tensors():
    import triton_mla

    kv, table = torch.zeros(4, 2, 16), torch.zeros(2, 2, dtype=I32)
    two, refs = torch.zeros(2, dtype=I32), torch.zeros(4, dtype=I32)
    for call in (lambda: triton_mla.copy_pages(kv, two, two),
                 lambda: triton_mla.fork_sequences(kv, table, two, refs, two),
                 lambda: triton_mla.free_sequences(table, two, refs, two.bool()),
                 lambda: triton_mla.reserve_pages(table, two, refs, 1, 2),
                 lambda: triton_mla.compact_pages(kv, table, refs)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


FAKE = 1 << 20  # a non-null, aligned address that no refused call reads


def _shared(lib, **kw):
    a = dict(q=FAKE, q_sb=16 * 576, q_sh=576, kv=FAKE, s0=64 * 576, s1=576, blocks=4, page=64, kv_scale=None, sc_s0=0, bt=FAKE, bt_s=2,
             bt_cols=2, lens=FAKE, prefix=None, prefix_len=64, starts=None, groups=1, batch=2, q_len=1, heads=16,
             dv=512, dr=64, dtype=0, scale=0.1, workers=256, out=FAKE, out_sb=16 * 512, out_sh=512, lse=None, ws=FAKE,
             ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return lib.tmla_mla_decode_shared(*a.values())


@pytest.mark.parametrize("kw,status,text", [
    ({"batch": -1}, 1, b"batch"), ({"heads": 0}, 1, b"num_heads"), ({"q_len": 0}, 1, b"q_len"),
    ({"dtype": 2}, 1, b"dtype"), ({"dv": 256}, 2, b"512"), ({"dr": 32}, 2, b"64"),
    ({"groups": 0}, 1, b"num_groups"), ({"groups": 4097}, 2, b"4096"), ({"groups": 2}, 1, b"group_starts"),
    ({"workers": 0}, 1, b"num_workers"), ({"workers": 65536}, 1, b"num_workers"),
    ({"page": 0}, 1, b"page_size"), ({"blocks": 0}, 1, b"num_blocks"), ({"bt_cols": 0}, 1, b"bt_cols"),
    ({"s1": 0}, 2, b"stride"), ({"s1": (1 << 25) + 8}, 2, b"stride"), ({"s1": 577}, 1, b"multiples of 8"),
    ({"q": None}, 1, b"null"), ({"bt": None}, 1, b"null"), ({"lens": None}, 1, b"null"), ({"out": None}, 1, b"null"),
    ({"q": FAKE + 2}, 1, b"aligned"), ({"ws": FAKE + 4}, 1, b"aligned"), ({"out_sh": 513}, 1, b"multiples of 8"),
    ({"ws": None}, 3, b"workspace"), ({"ws_bytes": 1000}, 3, b"workspace"),
    ({"kv_scale": FAKE, "s1": 584}, 1, b"multiples of 16"), ({"kv_scale": FAKE + 2}, 1, b"aligned"),
    ({"kv_scale": FAKE, "page": 16}, 2, b"32 tokens"), ({"kv_scale": FAKE, "page": 96}, 2, b"32 tokens"),
    ({"heads": 262141}, 2, b"262140"), ({"batch": 1 << 28}, 2, b"too large"),
    ({"batch": 1 << 24, "heads": 1, "bt_cols": 1}, 2, b"too large"),
    ({"bt_cols": 1 << 30, "batch": 4096}, 2, b"too large"),
])
def test_shared_entry_refusals(lib, kw, status, text):
    assert _shared(lib, **kw) == status
    assert text in lib.tmla_last_error()


def test_shared_workspace(lib):
    need = lib.tmla_shared_workspace_bytes
    assert need(0, 16, 1, 256) > 0 and _shared(lib, batch=0, bt_cols=0, page=0) == 0  # nothing to do
    assert need(64, 16, 1, 256) < need(64, 128, 1, 256) < need(64, 128, 64, 256)
    for bad in ((-1, 16, 1, 256), (2, 0, 1, 256), (2, 16, 0, 256), (2, 16, 1, 0), (1 << 30, 128, 1, 256)):
        assert need(*bad) == 0


def _pool_args(**kw):
    a = dict(kv=FAKE, s0=2 * 16, s1=16, pages=4, page=2, dim=16, elem=2, scale=None, sc0=0, sc1=0, cols=0)
    a.update(kw)
    return list(a.values())


def _page_calls(lib, pool, ws=FAKE, ws_bytes=1 << 30, null=None, table=(FAKE, 3, 2, 3), pages=4, page=2):
    """Every page entry point's status for the same fault; null: the index of a
    pointer left out."""
    def p(i):
        return None if null == i else FAKE

    tail = (ws, ws_bytes, None)
    return {
        "copy": lib.tmla_pages_copy(*pool, p(0), FAKE, 3, FAKE, *tail),
        "fork": lib.tmla_pages_fork(*pool, *table, p(0), p(1), FAKE, FAKE, FAKE, FAKE, FAKE, *tail),
        "free": lib.tmla_pages_free(*table, p(0), p(1), pages, FAKE, FAKE, FAKE, FAKE, *tail),
        "reserve": lib.tmla_pages_reserve(*table, p(0), p(1), pages, page, None, 1, FAKE, FAKE, FAKE, *tail),
        "compact": lib.tmla_pages_compact(*pool, *table, p(1), FAKE, FAKE, FAKE, *tail),
    }


def test_page_entries_refuse_bad_pools(lib):
    for kw, status in (({"kv": None}, 1), ({"pages": 0}, 1), ({"pages": 2 ** 31 - 8192}, 1), ({"page": 0}, 1),
                       ({"dim": 0}, 1), ({"elem": 3}, 1), ({"elem": 8}, 1), ({"s1": 15}, 1), ({"s0": 31}, 1),
                       ({"s0": 0}, 1), ({"s1": -16}, 1), ({"page": 1 << 20, "dim": 1 << 11, "s1": 1 << 11,
                                                          "s0": 1 << 31}, 2),
                       ({"scale": FAKE}, 1), ({"scale": FAKE + 2, "cols": 1}, 1)):
        for name, got in _page_calls(lib, _pool_args(**kw)).items():
            if name in ("copy", "fork", "compact"):
                assert got == status, (name, kw, lib.tmla_last_error())


def test_page_entries_refuse_missing_pointers_and_workspaces(lib):
    for null in (0, 1):
        for name, got in _page_calls(lib, _pool_args(), null=null).items():
            if (name, null) not in (("copy", 1), ("compact", 0)):
                assert got == 1, (name, null)
    for ws, size in ((None, 1 << 30), (FAKE, 16)):
        assert set(_page_calls(lib, _pool_args(), ws=ws, ws_bytes=size).values()) == {3}
    assert set(_page_calls(lib, _pool_args(), ws=FAKE + 8).values()) == {1}


def test_page_entries_refuse_bad_tables(lib):
    for table, status in (((FAKE, 3, -1, 3), 1), ((FAKE, 3, 2, 0), 1), ((FAKE, 3, (1 << 20) + 1, 3), 2),
                          ((FAKE, 3, 1 << 20, 1 << 20), 2)):
        got = _page_calls(lib, _pool_args(), table=table)
        got.pop("copy")
        assert set(got.values()) == {status}, (table, lib.tmla_last_error())
    assert lib.tmla_pages_reserve(FAKE, 3, 2, 3, FAKE, FAKE, 4, 0, None, 1, FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == 1
    assert lib.tmla_pages_free(FAKE, 3, 2, 3, FAKE, FAKE, 0, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 30, None) == 1


def test_copies_beyond_a_launch_are_refused(lib):
    """2^32 threads or more along the grid (pages of 2^30 + 2^20 bytes in rows of an odd
    number are 1,049,600 workgroups each)."""
    pool = _pool_args(page=1 << 20, dim=1025, elem=1, s1=1025, s0=1025 << 20, pages=2048)
    tail = (FAKE, 1 << 40, None)
    assert lib.tmla_pages_copy(*pool, FAKE, FAKE, 253, FAKE, *tail) == 2
    assert b"pages of too many bytes" in lib.tmla_last_error()
    table = (FAKE, 3, 1 << 12, 3)
    assert lib.tmla_pages_fork(*pool, *table, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, *tail) == 2
    assert b"pages of too many bytes" in lib.tmla_last_error()


def test_pages_workspace(lib):
    need = lib.tmla_pages_workspace_bytes
    assert need(1, 0, 0) > 0 and need(1 << 20, 64, 0) > 3 * 4 << 20 and need(16, 0, 1000) >= need(16, 0, 0) + 8000
    assert need(0, 1, 1) == 0 and need(1, -1, 0) == 0 and need(1, 0, -1) == 0
    assert ctypes.sizeof(ctypes.c_size_t) == 8
