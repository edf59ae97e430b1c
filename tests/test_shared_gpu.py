"""mla_decode_shared on the GPU against softmax attention in float64.

Bounds. With A = sum_t p_t |v_t| per output element (float64) and u = eps / 2
of the element type (bf16 2^-8, fp16 2^-11), the output carries two
roundings to the type, each of relative size at most u: the probabilities
before the value product (u A) and the result (u |out| <= u A): 2 u A. The
partials are 16-bit fractions of their row's largest value, off by half of
1 / 32767 of it, and no value of a row exceeds its largest A: 2^-15 max A for a
convex combination of them (with some room for the product). A score's float32
accumulation is off by at most 576 * 2^-24 * sum_i |q_i k_i| * scale, which
moves a probability by as much, relatively, twice with the normaliser; the
same amount bounds the lse's error, beside the exponential's and logarithm's
(2^-20 relative). fp16 probabilities below 2^-14 (relative to the row's
reference maximum) are off by up to 2^-25 each.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SCALE = 192 ** -0.5


def build(sizes, prefixes, own, heads, page=64, dtype=torch.bfloat16, q_len=1, seed=0, empty=(), scale_q=1.0):
    """A paged cache in which group g's sequences share their first
    prefixes[g] // page pages; own: tokens of its own of every sequence, in
    order; empty: sequences set to length 0. Returns the call's arguments."""
    g = torch.Generator().manual_seed(seed)
    lens, shared = [], []
    b = 0
    for n, p in zip(sizes, prefixes):
        shared.append(p // page)
        for _ in range(n):
            lens.append(p + own[b])
            b += 1
    groups = [i for i, n in enumerate(sizes) for _ in range(n)]
    pages = [-(-n // page) for n in lens]
    total = sum(shared) + sum(p - shared[i] for p, i in zip(pages, groups)) + 3
    perm = torch.randperm(total, generator=g).tolist()
    width = max(max(pages), 1)
    heads_of, at = [], 0
    for s in shared:
        heads_of.append(perm[at:at + s])
        at += s
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    for b, i in enumerate(groups):
        mine = pages[b] - shared[i]
        row = heads_of[i] + perm[at:at + mine]
        at += mine
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    for b in empty:
        lens[b] = 0
        table[b] = -7  # what a padded row may hold
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    kv = torch.randn(total, page, 576, generator=g).to(dtype)
    shape = (len(lens), heads, 576) if q_len == 1 else (len(lens), q_len, heads, 576)
    q = (torch.randn(*shape, generator=g) * scale_q).to(dtype)
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(q=q.cuda(), kv_cache=kv.cuda(), cache_seqlens=torch.tensor(lens, **i32), block_table=table.cuda(),
                prefix_lens=torch.tensor([s * page for s in shared], **i32), group_starts=torch.tensor(starts, **i32))


def check(args, out, lse, scale=SCALE, kv=None):
    """Every row within the bounds above of the float64 result; kv: float64
    values of the cache (an fp8 one)."""
    q = args["q"]
    u = torch.finfo(q.dtype).eps / 2
    many = (q if q.dim() == 4 else q.unsqueeze(1)).double()
    got = (out if q.dim() == 4 else out.unsqueeze(1)).double()
    got_lse = (lse if q.dim() == 4 else lse.unsqueeze(1)).double()
    cache = args["kv_cache"].double() if kv is None else kv
    page, q_len = cache.shape[1], many.shape[1]
    assert torch.isfinite(got).all()
    for b, n in enumerate(args["cache_seqlens"].tolist()):
        ids = args["block_table"][b, :-(-max(n, 0) // page)].long()
        rows = cache[ids].reshape(-1, 576)[:max(n, 0)]
        for t in range(q_len):
            seen = rows[:max(n - (q_len - 1 - t), 0)]
            if seen.shape[0] == 0:
                assert (got[b, t] == 0).all() and (got_lse[b, t] == -math.inf).all()
                continue
            s = many[b, t] @ seen.t().contiguous() * scale
            ref_lse = torch.logsumexp(s, -1)
            p = torch.exp(s - ref_lse[:, None])
            val = seen[:, :512].contiguous()
            ref, mag = p @ val, p @ val.abs()
            ds = 576 * 2.0 ** -24 * (many[b, t].abs() @ seen.abs().t().contiguous()).amax(-1) * abs(scale) + 2.0 ** -20
            tol = (2 * u * 1.01 + 2 * ds[:, None]) * mag + 2.0 ** -15 * mag.amax(-1, keepdim=True)
            if q.dtype == torch.float16:
                # relative to the reference maximum, whose own term is at least 1 in the normaliser
                tol = tol + 2.0 ** -25 * val.abs().sum(0)[None] * p.amax(-1, keepdim=True) + 2.0 ** -24
            bad = (got[b, t] - ref).abs() - tol
            assert bad.max() <= 0, f"sequence {b} token {t}: {bad.max().item():.3e} beyond {tol.max().item():.3e}"
            dl = (got_lse[b, t] - ref_lse).abs() - (ds + 2.0 ** -20 * ref_lse.abs())
            assert dl.max() <= 0, f"sequence {b} token {t}: lse {dl.max().item():.3e} beyond its bound"


def run(args, **kw):
    import triton_mla

    return triton_mla.mla_decode_shared(**args, softmax_scale=SCALE, return_lse=True, **{"share": True, **kw})


CASES = {
    # name: (sizes, prefixes, own, heads, page, dtype, q_len, empty)
    "one_group": ([4], [256], [1, 64, 65, 130], 16, 64, torch.bfloat16, 1, ()),
    "odd_heads": ([5], [640], [3, 1, 77, 200, 64], 20, 64, torch.bfloat16, 1, ()),
    "one_head": ([3], [128], [1, 2, 3], 1, 64, torch.float16, 1, ()),
    "rows_past_a_block": ([9], [320], [10 * i + 1 for i in range(9)], 24, 32, torch.bfloat16, 1, ()),
    "all_heads": ([3], [448], [5, 64, 129], 128, 64, torch.bfloat16, 1, ()),
    "more_heads_than_a_block": ([2], [192], [33, 1], 200, 64, torch.float16, 1, ()),
    "groups": ([1, 3, 2, 4], [100, 700, 64, 1500], [9, 1, 50, 300, 7, 8, 2, 3, 4, 64], 16, 16, torch.bfloat16, 1, ()),
    "no_prefix": ([3], [0], [1, 63, 200], 16, 64, torch.bfloat16, 1, ()),
    "below_a_tile": ([3], [48], [1, 63, 200], 16, 16, torch.bfloat16, 1, ()),
    "nothing_of_its_own": ([3], [512], [0, 0, 70], 32, 64, torch.bfloat16, 1, ()),
    "page_of_one": ([3], [130], [1, 40, 90], 16, 1, torch.bfloat16, 1, ()),
    "page_of_48": ([4], [480], [1, 40, 90, 5], 40, 48, torch.float16, 1, ()),
    "large_pages": ([4], [1024], [1, 40, 300, 5], 40, 256, torch.bfloat16, 1, ()),
    "padded_rows": ([4, 2], [256, 192], [5, 6, 7, 8, 9, 10], 16, 64, torch.bfloat16, 1, (0, 3, 4, 5)),
    "all_empty": ([3], [64], [1, 1, 1], 16, 64, torch.bfloat16, 1, (0, 1, 2)),
    "two_tokens": ([3], [320], [2, 40, 90], 16, 64, torch.bfloat16, 2, ()),
    "five_tokens_short": ([2, 2], [0, 64], [1, 3, 6, 5], 20, 16, torch.float16, 5, ()),
    "tokens_reach_into_the_prefix": ([3], [256], [1, 2, 3], 16, 64, torch.bfloat16, 4, (1,)),
    "long": ([6], [9000], [1, 500, 20, 30, 40, 64], 16, 64, torch.bfloat16, 1, ()),
    "one_long_one_short": ([2, 1], [6400, 0], [1, 2, 20000], 64, 64, torch.bfloat16, 1, ()),
}


@pytest.mark.parametrize("name", CASES)
def test_against_float64(gpu, name):
    sizes, prefixes, own, heads, page, dtype, q_len, empty = CASES[name]
    args = build(sizes, prefixes, own, heads, page, dtype, q_len, empty=empty)
    check(args, *run(args))


@pytest.mark.parametrize("granularity", ["page", "tensor", "number"])
@pytest.mark.parametrize("name", ["one_group", "rows_past_a_block", "all_heads", "more_heads_than_a_block",
                                  "large_pages", "padded_rows", "two_tokens", "long", "nothing_of_its_own"])
def test_fp8_against_float64(gpu, name, granularity):
    """The codes stand for e4m3 * scale exactly, so the 16-bit bounds hold with
    the same roundings: the probabilities take the page's scale in float32, then
    their one."""
    import triton_mla

    sizes, prefixes, own, heads, page, dtype, q_len, empty = CASES[name]
    args = build(sizes, prefixes, own, heads, page, dtype, q_len, empty=empty)
    # pages of different magnitudes
    kv = args["kv_cache"].float() * torch.rand(args["kv_cache"].shape[0], 1, 1, device="cuda") + 0.01
    codes, scale = triton_mla.quantize_kv_fp8(kv, "page" if granularity == "page" else "tensor")
    values = triton_mla.dequantize_kv_fp8(codes, scale).double()
    out, lse = run({**args, "kv_cache": codes.view(torch.uint8) if granularity == "tensor" else codes},
                   kv_scale=float(scale) if granularity == "number" else scale)
    check({**args, "kv_cache": codes}, out, lse, kv=values)


def test_fp8_strides_and_zero_scales(gpu):
    import triton_mla

    args = build([3], [320], [1, 64, 100], 16)
    codes, scale = triton_mla.quantize_kv_fp8(args["kv_cache"], "page")
    scale[args["block_table"][0, 1].long()] = 0.0  # a page of zeros, for all of the group
    want = run({**args, "kv_cache": codes}, kv_scale=scale)
    check(args, *want, kv=triton_mla.dequantize_kv_fp8(codes, scale).double())
    wide = torch.zeros(codes.shape[0], 70, 592, dtype=torch.uint8, device="cuda")
    wide[:, :64, :576] = codes.view(torch.uint8)
    scales = torch.zeros(codes.shape[0], 3, device="cuda")
    scales[:, 1] = scale
    got = run({**args, "kv_cache": wide[:, :64, :576]}, kv_scale=scales[:, 1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_fp8_refusals(gpu):
    args = build([3], [320], [1, 64, 100], 16)
    codes = args["kv_cache"].to(torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        run({**args, "kv_cache": codes})
    with pytest.raises(NotImplementedError):  # per token
        run({**args, "kv_cache": codes}, kv_scale=torch.ones(codes.shape[:2], device="cuda"))
    with pytest.raises(NotImplementedError):  # small pages
        run({**args, "kv_cache": codes.view(-1, 16, 576)}, kv_scale=1.0)
    with pytest.raises(AssertionError):
        run(args, kv_scale=1.0)


def test_prefix_as_one_number_and_one_group(gpu):
    args = build([4], [320], [1, 64, 65, 130], 16)
    want = run(args)
    args["prefix_lens"], args["group_starts"] = 320, None
    got = run(args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    import triton_mla

    alone = triton_mla.mla_decode_shared(**args, softmax_scale=SCALE, share=True)
    assert torch.equal(alone, want[0])


@pytest.mark.parametrize("prefix", [0, 63, 64, 100, 320, 321, 10 ** 9])
def test_any_prefix_up_to_the_shared_tokens_gives_the_result(gpu, prefix):
    # all rows of the table the same: every token is shared
    args = build([3], [384], [0, 0, 0], 16)
    args["cache_seqlens"] = torch.tensor([384, 321, 0], dtype=torch.int32, device="cuda")
    args["prefix_lens"] = prefix
    check(args, *run(args))


@pytest.mark.parametrize("starts", [[0, 2, 5], [1, 3, 4], [0, 0, 5], [3, 2, 5], [-4, 9, 2], [5, 5, 5], [2, 2, 2]])
def test_groups_out_of_order_or_range_only_share_less(gpu, starts):
    args = build([5], [256], [1, 20, 64, 70, 3], 16)
    args["group_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    args["prefix_lens"] = torch.tensor([256, 256], dtype=torch.int32, device="cuda")
    check(args, *run(args))


def test_many_groups(gpu):
    sizes = [2] * 600 + [1] * 500  # more groups than the planning kernel has threads
    args = build(sizes, [64] * len(sizes), [1 + i % 5 for i in range(sum(sizes))], 4, 64)
    out, lse = run(args)
    check(args, out, lse)


def test_large_scores_and_negative_scale(gpu):
    import triton_mla

    args = build([3], [320], [1, 64, 100], 16, scale_q=30.0)
    check(args, *run(args))
    args = build([3], [320], [1, 64, 100], 16)
    for scale in (-SCALE, 0.0, 1.0):
        got = triton_mla.mla_decode_shared(**args, softmax_scale=scale, return_lse=True, share=True)
        check(args, *got, scale=scale)


def test_masked_places_may_hold_anything(gpu):
    args = build([3], [256], [5, 1, 70], 16)
    want = run(args)
    kv, page = args["kv_cache"], 64
    used = torch.zeros(kv.shape[0], page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(args["cache_seqlens"].tolist()):
        for t in range(n):
            used[args["block_table"][b, t // page], t % page] = True
    for bad in (math.nan, math.inf, torch.finfo(torch.bfloat16).min):
        kv[~used] = bad
        got = run(args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_strides_and_layouts(gpu):
    args = build([4], [320], [1, 64, 65, 130], 16, q_len=3)
    want = run(args)
    q = args["q"]
    wide = torch.zeros(4, 3, 16, 584, dtype=q.dtype, device="cuda")  # padded rows
    wide[..., :576] = q
    odd = torch.zeros(q.numel() + 1, dtype=q.dtype, device="cuda")[1:].view(q.shape)  # 2-byte aligned
    odd.copy_(q)
    for other in (wide[..., :576], q.transpose(1, 2).contiguous().transpose(1, 2), odd):
        got = run({**args, "q": other})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    kv = args["kv_cache"]
    big = torch.zeros(kv.shape[0], 80, 640, dtype=kv.dtype, device="cuda")
    big[:, :64, :576] = kv
    table = torch.zeros(4, 2 * args["block_table"].shape[1], dtype=torch.int32, device="cuda")
    table[:, ::2] = args["block_table"]
    got = run({**args, "kv_cache": big[:, :64, :576].unsqueeze(2), "block_table": table[:, ::2],
               "cache_seqlens": args["cache_seqlens"].long(), "prefix_lens": args["prefix_lens"].cpu()})
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits(gpu):
    # a page every 2^25 elements: the last page lies past 2^32 bytes
    args = build([3], [192], [1, 64, 65], 16)
    kv = args["kv_cache"]
    step = 1 << 25
    store = torch.zeros((kv.shape[0] - 1) * step * 16 + 64 * 576, dtype=kv.dtype, device="cuda")
    far = store.as_strided(kv.shape, (step * 16, 576, 1))
    assert far.stride(0) * (kv.shape[0] - 1) > 1 << 31
    far.copy_(kv)
    got, want = run({**args, "kv_cache": far}), run(args)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_bits_repeat_and_streams(gpu):
    args = build([6, 2], [1000, 300], [1, 500, 20, 30, 40, 64, 3, 9], 16)
    want = run(args)
    other = build([4], [320], [1, 64, 65, 130], 128, seed=3)
    want_other = run(other)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            results.append((i, run(args if i % 2 else other)))
    torch.cuda.synchronize()
    for i, got in results:
        for a, b in zip(got, want if i % 2 else want_other):
            assert torch.equal(a, b)


def test_graph_replays_with_new_lengths(gpu):
    args = build([4], [320], [1, 64, 65, 130], 16)
    lens, prefix = args["cache_seqlens"].clone(), args["prefix_lens"].clone()
    run(args)
    torch.cuda.synchronize()
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = run(args)
    with torch.cuda.graph(second):
        out2, lse2 = run(args)
    for i in range(4):
        args["cache_seqlens"].copy_(lens - i * torch.tensor([0, 20, 1, 30], dtype=torch.int32, device="cuda"))
        args["prefix_lens"].copy_(prefix - 70 * i)
        out.zero_(), out2.zero_()
        graph.replay()
        second.replay()
        eager = run(args)
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
        assert torch.equal(out2, eager[0]) and torch.equal(lse2, eager[1])


def test_empty_batch(gpu):
    import triton_mla

    q = torch.empty(0, 16, 576, dtype=torch.bfloat16, device="cuda")
    kv = torch.zeros(2, 64, 576, dtype=torch.bfloat16, device="cuda")
    out, lse = triton_mla.mla_decode_shared(q, kv, torch.empty(0, dtype=torch.int32, device="cuda"),
                                            torch.empty(0, 3, dtype=torch.int32, device="cuda"), 64, return_lse=True,
                                            share=True)
    assert out.shape == (0, 16, 512) and lse.shape == (0, 16)


@pytest.mark.parametrize("name", ["one_group", "all_heads", "padded_rows", "two_tokens", "five_tokens_short"])
def test_without_sharing_it_is_mla_decode(gpu, name):
    import triton_mla

    sizes, prefixes, own, heads, page, dtype, q_len, empty = CASES[name]
    args = build(sizes, prefixes, own, heads, page, dtype, q_len, empty=empty)
    plain = triton_mla.mla_decode(args["q"], args["kv_cache"], args["cache_seqlens"], args["block_table"],
                                  softmax_scale=SCALE, return_lse=True)
    got = run(args, share=False)
    assert torch.equal(got[0], plain[0]) and torch.equal(got[1], plain[1])
    got, shared = run(args, share=None), run(args)  # (short tables share)
    assert torch.equal(got[0], shared[0]) and torch.equal(got[1], shared[1])


def test_sharing_is_chosen_by_size(gpu):
    """Past the rule's sizes a call shares (the bits of share=True), a long
    table of few bytes or of rows that fill blocks does not."""
    for sizes, heads, shares in (([40], 16, True), ([2], 16, False), ([2], 128, False)):
        args = build(sizes, [4096], [1 + i for i in range(sizes[0])], heads)
        want = run(args, share=shares)
        got = run(args, share=None)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_values_of_one_row_far_apart(gpu):
    """Value dims of very different size: no row's small ones are lost beyond the
    16-bit fractions of its largest one."""
    args = build([3], [320], [1, 64, 100], 16, dtype=torch.float16)
    args["kv_cache"][..., :8] *= 200.0
    args["q"][..., :8] = 0
    check(args, *run(args))
    args["kv_cache"][..., :512] = 0
    out, lse = run(args)
    assert (out == 0).all()
    check(args, out, lse)


@pytest.mark.parametrize("sign", [1, -1])
def test_infinity_in_a_token_that_counts(gpu, sign):
    """The rows that meet it are NaN, whichever way their scores go."""
    args = build([3], [256], [5, 1, 70], 16)
    args["q"][..., 100] = sign * args["q"][..., 100].abs().clamp(min=0.1)
    args["kv_cache"][args["block_table"][1, 4].long(), 0, 100] = math.inf  # of the second sequence alone
    out, _ = run(args)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]]).all()


def test_negative_scales_of_an_fp8_cache(gpu):
    """Pages of scales of either sign and of far exponents."""
    import triton_mla

    args = build([3], [320], [70, 1, 130], 16)
    codes, scale = triton_mla.quantize_kv_fp8(args["kv_cache"], "page")
    factor = torch.tensor([1.0, -1.0, 2.0 ** -9, -0.75], device="cuda")[torch.arange(scale.numel(), device="cuda") % 4]
    scale = scale * factor.reshape(scale.shape)
    kv = codes.view(torch.float8_e4m3fn).double() * scale.double().reshape(-1, 1, 1)
    args["kv_cache"] = codes
    check(args, *run(args, kv_scale=scale), kv=kv)


def test_nan_in_a_token_that_counts(gpu):
    """A NaN that a row attends to is not lost."""
    args = build([3], [256], [5, 1, 70], 16)
    args["kv_cache"][args["block_table"][0, 1].long(), 3, 100] = math.nan  # in the prefix
    out, _ = run(args)
    assert torch.isnan(out).all()
    args = build([3], [256], [5, 1, 70], 16)
    args["kv_cache"][args["block_table"][1, 4].long(), 0, 511] = math.nan  # of the second sequence alone
    out, _ = run(args)
    assert torch.isnan(out[1]).all() and not torch.isnan(out[[0, 2]]).any()


def test_items_past_the_list_of_a_worker(gpu):
    """Many short ends behind one prefix: a worker's items do not fit its list."""
    import triton_mla

    args = build([200], [6400], [1 + i % 3 for i in range(200)], 4)
    check(args, *run(args))
    codes, scale = triton_mla.quantize_kv_fp8(args["kv_cache"], "page")
    check({**args, "kv_cache": codes}, *run({**args, "kv_cache": codes}, kv_scale=scale),
          kv=triton_mla.dequantize_kv_fp8(codes, scale).double())


@pytest.mark.parametrize("batch", [255, 256, 257])
def test_plans_by_the_workers_and_by_their_own_launch(gpu, batch):
    """Both sides of the size up to which the workers make the plan."""
    sizes = [batch - 2, 2]
    args = build(sizes, [192, 128], [1 + (7 * i) % 90 for i in range(batch)], 20, empty=(3, batch - 1))
    check(args, *run(args))


def test_one_worker_and_many(gpu):
    """The C entry with other worker counts than the device's."""
    from triton_mla import _native

    args = build([6, 3], [640, 200], [1, 70, 2, 130, 64, 65, 9, 8, 7], 24)
    q, kv, bt = args["q"], args["kv_cache"], args["block_table"]
    lib = _native.load()
    for workers in (1, 3, 1000):
        need = lib.tmla_shared_workspace_bytes(9, 24, 2, workers)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        out, lse = torch.empty(9, 24, 512, dtype=q.dtype, device="cuda"), torch.empty(9, 24, device="cuda")
        _native.check(lib.tmla_mla_decode_shared(
            q.data_ptr(), q.stride(0), q.stride(1), kv.data_ptr(), kv.stride(0), kv.stride(1), kv.shape[0], 64, None, 0,
            bt.data_ptr(), bt.stride(0), bt.shape[1], args["cache_seqlens"].data_ptr(), args["prefix_lens"].data_ptr(),
            0, args["group_starts"].data_ptr(), 2, 9, 1, 24, 512, 64, 0, SCALE, workers, out.data_ptr(), out.stride(0),
            out.stride(1), lse.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream), "shared")
        check(args, out, lse)
