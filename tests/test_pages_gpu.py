"""Page operations on the GPU against their definitions in plain Python: whole
numbers and moved bytes, so every comparison is for equality."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu

I32 = torch.int32


def held(e, pages):
    return 0 <= e < pages


def ref_copy(pages, src, dst):
    """(pairs that copy, refused) in terms of page ids."""
    valid = [held(a, pages) and held(b, pages) for a, b in zip(src, dst)]
    last = {b: i for i, (b, v) in enumerate(zip(dst, valid)) if v}
    done, refused = [], 0
    for i, (a, b) in enumerate(zip(src, dst)):
        if not valid[i] or last[b] != i or (a in last and src[last[a]] != dst[last[a]]):
            refused += 1
        elif a != b:
            done.append((a, b))
    return done, refused


def ref_fork(rows, lens, refs, parents, page):
    pages, width = len(refs), len(rows[0])
    new, new_lens, counts, copies, first = [], [], list(refs), [], set()
    for i, p in enumerate(parents):
        if not 0 <= p < len(rows):
            new.append([-1] * width)
            new_lens.append(0)
            continue
        full, n = min(max(lens[p], 0) // page, width), lens[p]
        row = [e if held(e, pages) else -1 for e in rows[p]]
        if p in first:
            last = row[full] if full < width and n > 0 and n % page else -1
            row = row[:full] + [-1] * (width - full)
            if last >= 0:
                copies.append((i, full, last))
        first.add(p)
        new.append(row)
        new_lens.append(n)
    for table, d in ((rows, -1), (new, 1)):
        for row in table:
            for e in row:
                if held(e, pages):
                    counts[e] += d
    free = [i for i, c in enumerate(counts) if c <= 0]
    if len(copies) > len(free):
        return [list(r) for r in rows], list(lens), list(refs), len(copies) - len(free), []
    moves = []
    for (i, j, e), page_id in zip(copies, free):
        new[i][j] = page_id
        counts[page_id] = 1
        moves.append((e, page_id))
    return new, new_lens, counts, 0, moves


def ref_reserve(rows, lens, refs, new_tokens, page):
    pages, width = len(refs), len(rows[0])
    want, beyond = [], 0
    for b, n in enumerate(lens):
        need = -(-(max(n, 0) + max(new_tokens[b], 0)) // page)
        beyond += max(need - width, 0)
        want += [(b, j) for j in range(min(need, width)) if not held(rows[b][j], pages)]
    free = [i for i, c in enumerate(refs) if c <= 0]
    missing = max(len(want) - len(free), 0) + beyond
    new, counts = [list(r) for r in rows], list(refs)
    if missing == 0:
        for (b, j), e in zip(want, free):
            new[b][j] = e
            counts[e] = 1
    return new, counts, missing


def ref_compact(rows, refs):
    live = sum(c > 0 for c in refs)
    holes = [i for i in range(live) if refs[i] <= 0]
    moves = list(zip([i for i in range(live, len(refs)) if refs[i] > 0], holes))
    to, counts = dict(moves), list(refs)
    for a, b in moves:
        counts[b], counts[a] = refs[a], 0
    return [[to.get(e, e) for e in r] for r in rows], counts, live, moves


def cuda(x, dtype=I32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def state(rng, pages, batch, width, page, share=True, junk=True):
    """A consistent random state: rows of distinct pages, some of them shared
    between rows, entries beyond them that hold nothing."""
    ids = list(range(pages))
    rng.shuffle(ids)
    rows, lens, refs = [], [], [0] * pages
    for b in range(batch):
        room = min(width, len(ids))
        n = rng.choice([0, 1, room // 2, room, rng.randint(0, max(room, 0))]) if room else 0
        n = min(n, max(1, pages // (batch + 1)))
        row, common = [], 0
        if share and rows and rng.random() < 0.4:
            other = rng.choice(rows)
            common = min(rng.randint(0, width), sum(held(e, pages) for e in other))
            common = next((j for j in range(common) if not held(other[j], pages)), common)
            row = other[:common]
        for _ in range(max(n - common, 0)):
            row.append(ids.pop())
        for e in row:
            refs[e] += 1
        lens.append(rng.randint(max(0, len(row) - 1) * page, len(row) * page) if row else 0)
        tail = [rng.choice([-1, -1, -7, pages, pages + 5, -2 ** 31, 2 ** 31 - 1] if junk else [-1])
                for _ in range(width - len(row))]
        rows.append(row + tail)
    return rows, lens, refs


def pool(pages, page, dim, dtype, seed=0, layout="packed"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    raw = torch.randint(0, 256, (pages, page, dim * torch.empty(0, dtype=dtype).element_size()), generator=g,
                        device="cuda", dtype=torch.uint8)
    kv = raw.view(dtype)
    if layout == "packed":
        return kv
    if layout == "padded":  # pages and rows apart
        big = torch.zeros(pages, page + 2, dim + 8, dtype=dtype, device="cuda")
    elif layout == "odd":  # rows on no boundary
        big = torch.zeros(pages, page, dim + 3, dtype=dtype, device="cuda")
    else:  # rows of the pages dealt out in turn
        big = torch.zeros(page, pages, dim, dtype=dtype, device="cuda").transpose(0, 1)
    view = big[:, :page, :dim]
    view.copy_(kv)
    return view


def moved(kv, moves):
    new = kv.clone()
    for a, b in moves:
        new[b] = kv[a]
    return new


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("pairs", [0, 1, 2, 7, 256, 257, 3000])
@pytest.mark.parametrize("kind", ["plain", "anything"])
def test_copy(gpu, pairs, kind):
    import triton_mla

    rng = random.Random(pairs)
    pages = max(2 * pairs, 4)
    if kind == "plain":
        ids = list(range(pages))
        rng.shuffle(ids)
        src, dst = ids[:pairs], ids[pairs:2 * pairs]
    else:  # chains, repeated destinations, ids outside, pages onto themselves
        pages = max(pairs, 4)
        src = [rng.randint(-1, pages) for _ in range(pairs)]
        dst = [rng.choice([rng.randint(-2, pages + 1), s]) if rng.random() < 0.2 else rng.randint(0, pages - 1)
               for s in src]
        if pairs:
            dst[-1] = 2 ** 31 - 1
    kv = pool(pages, 3, 32, torch.bfloat16)
    done, refused = ref_copy(pages, src, dst)
    want = moved(kv, done)
    got = triton_mla.copy_pages(kv, cuda(src), cuda(dst))
    assert got.item() == refused
    assert same(kv, want)


@pytest.mark.parametrize("page,dim,dtype,layout", [
    (64, 576, torch.bfloat16, "packed"), (64, 576, torch.float16, "padded"), (1, 576, torch.bfloat16, "packed"),
    (48, 576, torch.float32, "packed"), (16, 288, torch.uint8, "odd"), (5, 33, torch.uint8, "packed"),
    (7, 35, torch.float16, "odd"), (64, 576, torch.float8_e4m3fn, "packed"), (16, 64, torch.bfloat16, "in turn"),
    (256, 1280, torch.float32, "packed"), (1, 1, torch.uint8, "packed"),
])
@pytest.mark.parametrize("pairs", [5, 300])
def test_copy_layouts(gpu, page, dim, dtype, layout, pairs):
    import triton_mla

    pages = 2 * pairs + 1
    kv = pool(pages, page, dim, dtype, layout=layout)
    before = kv.clone()
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).tolist()
    src, dst = perm[:pairs], perm[pairs:2 * pairs]
    shaped = kv.unsqueeze(2) if layout == "packed" else kv
    triton_mla.copy_pages(shaped, torch.tensor(src), cuda(dst))
    assert same(kv, moved(before.view(torch.uint8) if dtype.itemsize == 1 else before, list(zip(src, dst))))


@pytest.mark.parametrize("granularity", ["page", "token", "tensor", "number"])
@pytest.mark.parametrize("pairs", [3, 300])
def test_copy_moves_the_scales(gpu, granularity, pairs):
    import triton_mla

    pages = 2 * pairs
    x = torch.randn(pages, 16, 64, device="cuda") * torch.rand(pages, 16, 1, device="cuda")
    kv, scale = triton_mla.quantize_kv_fp8(x, granularity if granularity != "number" else "tensor")
    if granularity == "number":
        scale = float(scale)
    src, dst = list(range(pairs)), list(range(pairs, 2 * pairs))
    want = moved(kv.view(torch.uint8), zip(src, dst))
    want_scale = moved(scale, zip(src, dst)) if granularity in ("page", "token") else scale
    triton_mla.copy_pages(kv, cuda(src), cuda(dst), kv_scale=scale)
    assert same(kv, want)
    assert torch.equal(scale, want_scale) if torch.is_tensor(scale) else scale == want_scale


FORKS = [  # pages, batch, width, page
    (40, 1, 3, 4), (60, 5, 4, 4), (300, 16, 9, 16), (5000, 64, 40, 64), (9000, 300, 17, 1), (700, 3, 300, 8),
]


@pytest.mark.parametrize("pages,batch,width,page", FORKS)
@pytest.mark.parametrize("how", ["one", "same", "random", "none", "beam"])
def test_fork(gpu, pages, batch, width, page, how):
    import triton_mla

    rng = random.Random(pages + batch)
    rows, lens, refs = state(rng, pages, batch, width, page)
    parents = {"one": [rng.randrange(batch)] * batch, "same": list(range(batch)),
               "random": [rng.randint(-2, batch + 1) for _ in range(batch)], "none": [-1] * batch,
               "beam": [min(i // 4 * 4 + rng.randrange(4), batch - 1) for i in range(batch)]}[how]
    kv = pool(pages, page, 16, torch.bfloat16)
    new, new_lens, counts, missing, moves = ref_fork(rows, lens, refs, parents, page)
    want = moved(kv, moves)
    got = triton_mla.fork_sequences(kv, cuda(rows), cuda(lens), cuda(refs), cuda(parents))
    assert got[3].tolist() == [missing]
    assert got[0].tolist() == new
    assert got[1].tolist() == new_lens
    assert got[2].tolist() == counts
    assert same(kv, want)


def test_fork_without_room_changes_nothing(gpu):
    import triton_mla

    rows, lens, refs = [[0, 1, -1], [-1, -5, 9], [2, -1, -1]], [6, 0, 4], [1, 1, 1]
    kv = pool(3, 4, 16, torch.bfloat16)
    before = kv.clone()
    got = triton_mla.fork_sequences(kv, cuda(rows), cuda(lens), cuda(refs), cuda([0, 0, 0]))
    # row 2 gives its page back: one of the two copies would find room
    assert got[3].tolist() == [1] and got[0].tolist() == rows and got[1].tolist() == lens
    assert got[2].tolist() == refs and same(kv, before)
    got = triton_mla.fork_sequences(kv, cuda(rows), cuda(lens), cuda(refs), cuda([0, 0, -1]))
    assert got[3].tolist() == [0] and got[0].tolist() == [[0, 1, -1], [0, 2, -1], [-1, -1, -1]]
    assert got[2].tolist() == [2, 1, 1] and same(kv[2], before[1]) and same(kv[:2], before[:2])


def test_fork_moves_the_scales(gpu):
    import triton_mla

    for granularity in ("page", "token"):
        kv, scale = triton_mla.quantize_kv_fp8(torch.randn(6, 4, 32, device="cuda"), granularity)
        want, want_scale = moved(kv.view(torch.uint8), [(4, 0)]), moved(scale, [(4, 0)])
        got = triton_mla.fork_sequences(kv, cuda([[5, 4], [-1, -1]]), cuda([7, 0]), cuda([0, 0, 0, 0, 1, 1]),
                                        cuda([0, 0]), kv_scale=scale)
        assert got[0].tolist() == [[5, 4], [5, 0]] and same(kv, want) and torch.equal(scale, want_scale)


@pytest.mark.parametrize("pages,batch,width,page", FORKS)
def test_free(gpu, pages, batch, width, page):
    import triton_mla

    rng = random.Random(pages)
    rows, lens, refs = state(rng, pages, batch, width, page)
    refs[rng.randrange(pages)] += 3  # holds of the program's own
    ended = [rng.random() < 0.5 for _ in range(batch)]
    want = list(refs)
    for b, end in enumerate(ended):
        for e in rows[b]:
            if end and held(e, pages):
                want[e] -= 1
    for flags in (torch.tensor(ended, device="cuda"), cuda([5 * e for e in ended])):
        got = triton_mla.free_sequences(cuda(rows), cuda(lens), cuda(refs), flags)
        assert got[0].tolist() == [[-1] * width if e else r for r, e in zip(rows, ended)]
        assert got[1].tolist() == [0 if e else n for n, e in zip(lens, ended)]
        assert got[2].tolist() == want


@pytest.mark.parametrize("pages,batch,width,page", FORKS)
@pytest.mark.parametrize("most", [0, 1, 9, 100])
def test_reserve(gpu, pages, batch, width, page, most):
    import triton_mla

    rng = random.Random(pages + most)
    rows, lens, refs = state(rng, pages, batch, width, page)
    new_tokens = [rng.randint(-1, most) for _ in range(batch)]
    want = ref_reserve(rows, lens, refs, new_tokens, page)
    got = triton_mla.reserve_pages(cuda(rows), cuda(lens), cuda(refs), cuda(new_tokens), page)
    assert (got[0].tolist(), got[1].tolist(), got[2].item()) == want
    want = ref_reserve(rows, lens, refs, [most] * batch, page)
    got = triton_mla.reserve_pages(cuda(rows), cuda(lens), cuda(refs), most, page)
    assert (got[0].tolist(), got[1].tolist(), got[2].item()) == want


def test_reserve_without_room_or_columns_changes_nothing(gpu):
    import triton_mla

    rows, lens, refs = [[0, -1], [-1, -1]], [4, 0], [1, 0, 0, -3]
    for new_tokens, missing in (([4, 8], 0), ([4, 9], 1), ([2 ** 31 - 1] * 2, 2 * (2 ** 29 - 2) + 1)):
        want = ref_reserve(rows, lens, refs, new_tokens, 4)
        assert want[2] == missing
        got = triton_mla.reserve_pages(cuda(rows), cuda(lens), cuda(refs), cuda(new_tokens), 4)
        assert (got[0].tolist(), got[1].tolist(), got[2].item()) == want
    got = triton_mla.reserve_pages(cuda(rows), cuda(lens), cuda([1, 1, 1, 0]), cuda([4, 8]), 4)
    assert got[2].item() == 2 and got[0].tolist() == rows and got[1].tolist() == [1, 1, 1, 0]


def test_reserve_more_than_31_bits_are_missing(gpu):
    import triton_mla

    rows = [[-1]] * 8
    got = triton_mla.reserve_pages(cuda(rows), cuda([2 ** 31 - 1] * 8), cuda([0] * 9), 2 ** 31 - 1, 1)
    assert got[2].item() == 2 ** 31 - 1 and got[0].tolist() == rows


@pytest.mark.parametrize("pages,every", [(20000, 1), (20001, 2), (14000, 3), (40000, 17), (5_000_000, 1000)])
def test_reserve_of_long_rows(gpu, pages, every):
    """Rows that are given many pages: more than a pass finds at once, spread over
    chunks, entered between entries that hold pages."""
    import triton_mla

    rng = random.Random(pages)
    refs = [0 if i % every == every // 2 else 1 + i % 2 for i in range(pages)]
    free = refs.count(0)
    counts = [1, 0, 1023, 1024, 1025, 300, 2049, 1]
    width = max(counts) + 700
    rows, lens, want_tokens = [], [], []
    for c in counts:
        c = min(c, max(free // 5 - 5, 0))
        keep = rng.randint(0, 600)
        row = [rng.randrange(pages) for _ in range(keep)] + [rng.choice([-1, -7, pages]) for _ in range(c)]
        rng.shuffle(row)
        rows.append(row + [-1] * (width - len(row)))
        lens.append(0)
        want_tokens.append(len(row) * 4)
    want = ref_reserve(rows, lens, refs, want_tokens, 4)
    assert want[2] == 0
    got = triton_mla.reserve_pages(cuda(rows), cuda(lens), cuda(refs), cuda(want_tokens), 4)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].item() == 0


@pytest.mark.parametrize("pages", [4096, 4097, 12288, 5_000_000])
def test_large_pools(gpu, pages):
    """Pools of several chunks: the free pages far apart, at the borders."""
    import triton_mla

    refs = torch.ones(pages, dtype=I32)
    free = sorted({0, 1, 4095, 4096 % pages, 4097 % pages, pages // 2, pages - 2, pages - 1})
    refs[free] = 0
    rows = torch.full((len(free) + 1, 2), -1, dtype=I32)
    rows[0, 0] = 2
    lens = cuda([1] + [0] * len(free))
    got = triton_mla.reserve_pages(rows.cuda(), lens, refs.cuda(), 1, 1)  # one row more than free pages
    assert got[2].item() == 1 and torch.equal(got[0].cpu(), rows) and torch.equal(got[1].cpu(), refs)
    got = triton_mla.reserve_pages(rows.cuda(), lens, refs.cuda(), cuda([1] * len(free) + [0]), 1)
    assert got[2].item() == 0
    assert got[0][:, 0].tolist() == [2] + free[1:] + [-1] and got[0][0, 1].item() == free[0]
    assert (got[1] == 1).all()
    table = torch.tensor([[pages - 3, 5, pages, -1]], dtype=I32)
    if pages > 100000:
        refs[pages // 3:] = 0
        refs[pages - 3] = 4
        refs[pages - 4096 * 3] = 1
    kv = torch.arange(pages, device="cuda", dtype=torch.float32).reshape(pages, 1, 1)
    want = kv.clone()
    new, counts, live, moves = ref_compact(table.tolist(), refs.tolist())
    for a, b in moves:
        want[b] = kv[a]
    got = triton_mla.compact_pages(kv, table.cuda(), refs.cuda())
    assert got[0].tolist() == new and got[1].tolist() == counts and got[2].item() == live and torch.equal(kv, want)


@pytest.mark.parametrize("pages,batch,width,page", FORKS)
@pytest.mark.parametrize("layout", ["packed", "odd"])
def test_compact(gpu, pages, batch, width, page, layout):
    import triton_mla

    rng = random.Random(batch)
    rows, lens, refs = state(rng, pages, batch, width, page)
    kv = pool(pages, page, 16, torch.bfloat16, layout=layout)
    new, counts, live, moves = ref_compact(rows, refs)
    want = moved(kv, moves)
    got = triton_mla.compact_pages(kv, cuda(rows), cuda(refs))
    assert got[0].tolist() == new and got[1].tolist() == counts and got[2].tolist() == [live]
    assert same(kv, want)


@pytest.mark.parametrize("refs", [[0] * 9, [1] * 9, [0] * 8 + [1], [1] + [0] * 8, [-1, 2, 0, 1]])
def test_compact_full_empty_and_borders(gpu, refs):
    import triton_mla

    pages = len(refs)
    rows = [[pages - 1, 0, -1, pages]]
    kv = pool(pages, 2, 16, torch.float32)
    new, counts, live, moves = ref_compact(rows, refs)
    want = moved(kv, moves)
    got = triton_mla.compact_pages(kv, cuda(rows), cuda(refs))
    assert got[0].tolist() == new and got[1].tolist() == counts and got[2].tolist() == [live] and same(kv, want)


def test_strided_tables_and_other_integer_types(gpu):
    import triton_mla

    rng = random.Random(2)
    rows, lens, refs = state(rng, 60, 5, 4, 4)
    wide = torch.full((5, 8), -1, dtype=I32, device="cuda")
    wide[:, ::2] = cuda(rows)
    tall = torch.full((5, 9), -1, dtype=I32, device="cuda")
    tall[:, :4] = cuda(rows)
    want = triton_mla.reserve_pages(cuda(rows), cuda(lens), cuda(refs), 3, 4)
    for table in (wide[:, ::2], tall[:, :4], cuda(rows).long().clamp(-9, 99)):
        got = triton_mla.reserve_pages(table.clamp(-9, 99), cuda(lens).long(), cuda(refs).long(),
                                       torch.full((5,), 3, device="cuda"), 4)
        assert torch.equal(got[0].clamp(-9, 99), want[0].clamp(-9, 99)) and torch.equal(got[1], want[1])


def test_offsets_past_32_bits(gpu):
    import triton_mla

    pages, step = 40, 1 << 28  # a page every 2^29 bytes: the last ones past 2^34
    store = torch.zeros((pages - 1) * (step // 2) + 64, dtype=torch.float16, device="cuda")
    kv = store.as_strided((pages, 2, 32), (step // 2, 32, 1))
    kv.copy_(torch.randn(pages, 2, 32).to(kv))
    want = moved(kv.contiguous(), [(3, 39), (38, 1)])
    triton_mla.copy_pages(kv, cuda([3, 38]), cuda([39, 1]))
    assert same(kv, want)


def test_empty_batch(gpu):
    import triton_mla

    kv = pool(4, 2, 16, torch.bfloat16)
    none = torch.empty(0, dtype=I32, device="cuda")
    table, refs = torch.empty(0, 3, dtype=I32, device="cuda"), cuda([0, 2, 0, 1])
    got = triton_mla.fork_sequences(kv, table, none, refs, none)
    assert got[0].shape == (0, 3) and torch.equal(got[2], refs) and got[3].item() == 0
    got = triton_mla.reserve_pages(table, none, refs, 1, 2)
    assert torch.equal(got[1], refs) and got[2].item() == 0
    got = triton_mla.free_sequences(table, none, refs, none.bool())
    assert torch.equal(got[2], refs)
    got = triton_mla.compact_pages(kv, table, refs)
    assert got[1].tolist() == [1, 2, 0, 0] and got[2].item() == 2


def test_streams_and_graphs(gpu):
    import triton_mla

    rng = random.Random(5)
    rows, lens, refs = state(rng, 5000, 64, 40, 64)
    parents = [rng.randrange(64) for _ in range(64)]
    kv = pool(5000, 64, 16, torch.bfloat16)
    args = (cuda(rows), cuda(lens), cuda(refs), cuda(parents))
    new, new_lens, counts, missing, moves = ref_fork(rows, lens, refs, parents, 64)
    assert missing == 0 and moves
    streams = [torch.cuda.Stream() for _ in range(3)]
    pools = [kv.clone() for _ in streams]
    torch.cuda.synchronize()
    results = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            results.append(triton_mla.fork_sequences(pools[i % 3], *args))
            triton_mla.reserve_pages(results[-1][0], results[-1][1], results[-1][2], 70, 64)
    torch.cuda.synchronize()
    want = moved(kv, moves)
    for got in results:
        assert got[0].tolist() == new and got[1].tolist() == new_lens and got[2].tolist() == counts
    assert all(same(p, want) for p in pools)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forked = triton_mla.fork_sequences(kv, *args)
        held_pages = triton_mla.reserve_pages(forked[0], forked[1], forked[2], 70, 64)
        packed = triton_mla.compact_pages(kv, held_pages[0], held_pages[1])
    for i in range(3):
        if i:
            parents = [rng.randrange(64) for _ in range(64)]
            args[3].copy_(cuda(parents))
        before = kv.clone()
        graph.replay()
        torch.cuda.synchronize()
        new, new_lens, counts, missing, moves = ref_fork(rows, lens, refs, parents, 64)
        assert missing == 0 and forked[0].tolist() == new
        content = moved(before, moves)
        new, counts, missing = ref_reserve(new, new_lens, counts, [70] * 64, 64)
        new, counts, live, moves = ref_compact(new, counts)
        assert packed[0].tolist() == new and packed[1].tolist() == counts and packed[2].item() == live
        assert same(kv, moved(content, moves))


@pytest.mark.parametrize("fp8", [False, True])
def test_serving_run(gpu, fp8):
    """A prompt in one row, forked into samples, decoded over the shared
    prefix while the samples grow, drawn anew as beams, some ended, the pool
    compacted: every step's decode equals the plain one of a program that
    keeps each sequence's rows on its own."""
    import triton_mla

    rng = random.Random(11)
    batch, heads, page, pages, width = 6, 16, 64, 64, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    kv = torch.zeros(pages, page, 576, dtype=torch.bfloat16, device="cuda")
    scale = None
    if fp8:  # codes of 1/8, and one scale a page that moves with it
        kv = torch.zeros(pages, page, 576, dtype=torch.uint8, device="cuda")
        scale = torch.full((pages,), 0.125, device="cuda")
    table = torch.full((batch, width), -1, dtype=I32, device="cuda")
    lens = torch.zeros(batch, dtype=I32, device="cuda")
    refs = torch.zeros(pages, dtype=I32, device="cuda")
    kept = [torch.empty(0, 576, dtype=torch.bfloat16, device="cuda") for _ in range(batch)]

    def append(counts):
        nonlocal table, lens, refs
        table, refs, missing = triton_mla.reserve_pages(table, lens, refs, cuda(counts), page)
        assert missing.item() == 0
        for b, n in enumerate(counts):
            rows = torch.randn(n, 576, generator=g, device="cuda", dtype=torch.bfloat16)
            codes = (rows.float() * 8).to(torch.float8_e4m3fn)
            for j in range(n):
                t = kept[b].shape[0] + j
                kv[table[b, t // page].long(), t % page] = codes[j].view(torch.uint8) if fp8 else rows[j]
            if fp8:  # (three bits and a power of two: exact in bf16)
                rows = (codes.float() / 8).to(torch.bfloat16)
            kept[b] = torch.cat([kept[b], rows])
        lens = lens + cuda(counts)

    def decode(prefix):
        q = torch.randn(batch, heads, 576, generator=g, device="cuda", dtype=torch.bfloat16)
        shared, lse = triton_mla.mla_decode_shared(q, kv, lens, table, prefix, softmax_scale=192 ** -0.5,
                                                   return_lse=True, kv_scale=scale, share=True)
        dense = torch.zeros(batch, max(k.shape[0] for k in kept), 576, dtype=torch.bfloat16, device="cuda")
        for b, k in enumerate(kept):
            dense[b, :k.shape[0]] = k
        plain, plain_lse = triton_mla.mla_decode(q, dense, lens, softmax_scale=192 ** -0.5, return_lse=True)
        # each is within 3 roundings of sum p |v| <= max |v| of the exact result
        assert (shared.float() - plain.float()).abs().max() <= 6 * 2.0 ** -8 * dense.float().abs().max()
        assert torch.equal(lse == -float("inf"), plain_lse == -float("inf"))
        assert torch.where(lens[:, None] > 0, lse - plain_lse, torch.zeros_like(lse)).abs().max() <= 1e-3
        return q, shared, lse

    append([331] + [0] * (batch - 1))
    parents = [0] * batch
    table, lens, refs, missing = triton_mla.fork_sequences(kv, table, lens, refs, cuda(parents), scale)
    assert missing.item() == 0
    kept = [kept[0].clone() for _ in range(batch)]
    assert refs.max().item() == batch
    for step in range(4):
        append([rng.choice([1, 1, 40]) for _ in range(batch)])
        decode(320)
        parents = [rng.randrange(batch) for _ in range(batch)]
        table, lens, refs, missing = triton_mla.fork_sequences(kv, table, lens, refs, cuda(parents), scale)
        assert missing.item() == 0
        kept = [kept[p].clone() for p in parents]
    ended = torch.tensor([True, False] * 3, device="cuda")
    table, lens, refs = triton_mla.free_sequences(table, lens, refs, ended)
    kept = [k[:0] if e else k for k, e in zip(kept, ended.tolist())]
    q, out, lse = decode(320)
    table, refs, live = triton_mla.compact_pages(kv, table, refs, scale)
    assert (refs[live.item():] == 0).all() and (refs[:live.item()] > 0).all()
    kv = kv[:live.item()].clone()  # the rest of the pool can go
    again = triton_mla.mla_decode_shared(q, kv, lens, table, 320, softmax_scale=192 ** -0.5, return_lse=True,
                                         kv_scale=scale[:live.item()] if fp8 else None, share=True)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_threads_and_streams_at_once(gpu):
    """Threads that share a stream (and so its workspace) and threads with their
    own: page operations and decodes give what they give alone."""
    import threading

    import triton_mla

    rng = random.Random(3)
    work = []
    for pages, batch, width in ((200, 4, 6), (20000, 30, 40), (300, 9, 8), (14000, 500, 64)):
        rows, lens, refs = state(rng, pages, batch, width, 4)
        rows, lens, refs, parents = cuda(rows), cuda(lens), cuda(refs), cuda([rng.randrange(batch) for _ in range(batch)])
        kv = torch.randn(pages, 4, 576, device="cuda").bfloat16()
        q = torch.randn(batch, 16, 576, device="cuda").bfloat16()
        table = torch.randint(0, pages, (batch, width), device="cuda", dtype=I32)
        common = width // 2
        table[:, :common] = table[0, :common]
        counts = torch.randint(4 * common, 4 * width, (batch,), device="cuda", dtype=I32)

        def calls(kv=kv, q=q, rows=rows, lens=lens, refs=refs, parents=parents, table=table, counts=counts,
                  prefix=4 * common):
            return (*triton_mla.mla_decode_shared(q, kv, counts, table, prefix, return_lse=True, share=True),
                    *triton_mla.reserve_pages(rows, lens, refs, 3, 4),
                    *triton_mla.fork_sequences(kv.clone(), rows, lens, refs, parents),
                    *triton_mla.compact_pages(kv.clone(), rows, refs))

        work.append((calls, calls()))
    torch.cuda.synchronize()
    wrong = []

    def run(i, stream):
        calls, want = work[i]
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = calls()
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(i)

    shared = torch.cuda.Stream()
    threads = [threading.Thread(target=run, args=(i, shared if i < 2 else torch.cuda.Stream())) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []
