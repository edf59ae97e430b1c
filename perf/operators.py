"""Decode over a shared prefix and the page operations that make one.

Five operators of a serving program that keeps its latent cache in pages:

  shared   ``mla_decode_shared``: decode of a batch whose sequences, in groups,
           begin with the same pages, each group's prefix attended to once;
  copy     ``copy_pages``: whole pages to other pages;
  fork     ``fork_sequences`` (and ``free_sequences``): rows of the block table
           become copies of others or end, with the pages' reference counts;
  reserve  ``reserve_pages``: pages for the tokens to come;
  compact  ``compact_pages``: the pages in use moved to the pool's front.

``listed`` holds the calls they are measured by, ``draw`` spreads over the same
ranges. Queries and caches are N(0, 1), pages lie shuffled in their pool, and
the lengths of a batch are spread evenly over [lo, hi] in a shuffled order, so
a case's work does not depend on the seed.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
WIDTH, VALUE = 576, 512  # latent + rope dims of a cached row, and the latent ones
SCALE = 192 ** -0.5


def _package():
    folder = os.path.abspath("triton-mla_amd")  # the package's folder in the tree under test
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import triton_mla

    return triton_mla


# --- cases -------------------------------------------------------------------


def _shared(name, groups, prefixes, heads, lo, hi, dtype="bf16", page=64, q_len=1, fp8=False, empty=0):
    """groups: sequences of each group; prefixes: tokens each group shares;
    [lo, hi]: the tokens that a sequence has of its own; empty: sequences at
    the batch's end that hold nothing (a padded batch)."""
    return {"name": name, "kind": "shared", "groups": groups, "prefixes": prefixes, "heads": heads, "lo": lo,
            "hi": hi, "dtype": dtype, "page": page, "q_len": q_len, "fp8": fp8, "empty": empty}


def _copy(name, pairs, pool, page=64, dtype="bf16"):
    return {"name": name, "kind": "copy", "pairs": pairs, "pool": pool, "page": page, "dtype": dtype}


def _fork(name, mode, batch, lo, hi, page=64, width=128):
    """mode "split": the first sequence becomes the whole batch; "beam": every
    eight rows are drawn anew from among themselves; "free": a third ends."""
    return {"name": name, "kind": "fork", "mode": mode, "batch": batch, "lo": lo, "hi": hi, "page": page,
            "width": width}


def _reserve(name, batch, lo, hi, most, pool, page=64):
    """most: up to this many new tokens a sequence (0 for some)."""
    return {"name": name, "kind": "reserve", "batch": batch, "lo": lo, "hi": hi, "most": most, "pool": pool,
            "page": page}


def _compact(name, batch, lo, hi, pool, page=64):
    return {"name": name, "kind": "compact", "batch": batch, "lo": lo, "hi": hi, "pool": pool, "page": page}


def listed():
    return [
        # Four samples of one short prompt on one rank of eight (16 heads):
        # the smallest call, its time is launches and latency.
        _shared("shared_b4_h16_2k", "4", "2048", 16, 1, 64),
        # 64 samples of one long document, 16 heads: a whole batch over one
        # 32K prefix, the largest gain over reading it 64 times.
        _shared("shared_b64_h16_32k", "64", "32768", 16, 17, 509),
        # A system prompt of 8K tokens under a full batch with all 128 heads.
        _shared("shared_b32_h128_8k", "32", "8192", 128, 33, 1021),
        # Several prompts, each with its samples, one alone, one that shares
        # nothing, prefixes of odd lengths, small pages, rows of padding.
        _shared("shared_groups_h64_fp16", "1,3,8,12,5", "700,4100,6011,1999,0", 64, 1, 900, "fp16", 16, empty=3),
        # The system prompt over an fp8 cache, two query tokens a sequence
        # (a draft token verified beside the next one).
        _shared("shared_fp8_spec2_b16_h128_8k", "16", "8192", 128, 33, 1021, q_len=2, fp8=True),
        # A few pages copied before they are written to: latency.
        _copy("copy_8", 8, 64),
        # A third of a pool moved at once (swap-in, a new layout): bytes.
        _copy("copy_4k", 4096, 12288),
        # One prompt becomes 16 samples.
        _fork("fork_split_b16", "split", 16, 1500, 1500),
        # Beam search: 256 beams drawn anew from their groups of eight.
        _fork("fork_beam_b256", "beam", 256, 500, 4000),
        # A decode step's pages for a batch of 64, and for a batch of 1,024
        # with drafts over the page table of a large pool.
        _reserve("reserve_b64", 64, 100, 4000, 1, 8192),
        _reserve("reserve_b1024", 1024, 1, 16000, 70, 524288),
        # A fragmented pool of 1.2 GB brought together.
        _compact("compact_16k", 192, 100, 6000, 16384),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "shared", "shared", "copy", "fork", "fork", "reserve", "compact"])
    page = rng.choice([16, 32, 64, 64, 64, 128])
    if kind == "copy":
        page = rng.choice([1, 16, 48, 64, 64, 128])
        pairs = _log_int(rng, 1, 4096 * 64 // max(page, 64))
        return _copy("", pairs, 2 * pairs + rng.randrange(1, 100), page, rng.choice(["bf16", "fp16"]))
    if kind == "fork":
        mode = rng.choice(["split", "beam", "free"])
        batch = _log_int(rng, 2, 256)
        hi = _log_int(rng, 20, 4000)
        lo = max(1, int(hi * rng.choice([0.05, 0.5, 1.0])))
        page = rng.choice([16, 64, 64, 48, 128])
        return _fork("", mode, batch, lo, hi, page, -(-hi // page) + rng.choice([0, 1, 37]))
    if kind == "reserve":
        batch = _log_int(rng, 1, 1024)
        hi = _log_int(rng, 20, 16000)
        pages = batch * (-(-hi // page) + 8)
        pool = min(524288, pages + _log_int(rng, 1, 200000))
        return _reserve("", batch, rng.choice([0, 1, hi // 2]), hi, rng.choice([1, 1, 5, 70]), max(pool, pages), page)
    if kind == "compact":
        page = rng.choice([16, 48, 64, 64, 128])
        batch = _log_int(rng, 1, 192)
        hi = _log_int(rng, 20, 6000)
        lo = max(1, int(hi * rng.choice([0.02, 0.5, 1.0])))
        pages = sum(-(-n // page) for n in _spread(batch, lo, hi))
        cap = 16384 * 64 // page  # (the listed pool's bytes)
        while pages > cap:
            batch = max(1, batch // 2)
            pages = sum(-(-n // page) for n in _spread(batch, lo, hi))
        return _compact("", batch, lo, hi, min(cap, pages + int(pages * rng.choice([0.0, 0.1, 0.9, 3.0]))), page)
    heads = rng.choice([8, 16, 16, 20, 32, 64, 128, 128])
    count = rng.choice([1, 1, 1, 2, 3, 6])
    q_len = rng.choice([1, 1, 1, 2, 3])
    fp8 = rng.random() < 0.25
    groups, prefixes, cost = [], [], 0
    budget = 64 * 16 * 32768  # rows times tokens, as in the largest listed case
    for _ in range(count):
        n = _log_int(rng, 1, max(1, 96 // count))
        prefix = _log_int(rng, 100, 32768) if rng.random() < 0.9 else 0
        n = max(1, min(n, (budget - cost) // (heads * q_len * (prefix + 1024))))
        prefix = min(prefix, max(0, (budget - cost) // (heads * q_len * n) - 1024))
        cost += heads * q_len * n * (prefix + 1024)
        groups.append(n)
        prefixes.append(prefix)
        if cost * 10 > budget * 9:
            break
    hi = _log_int(rng, q_len, 1000)
    return _shared("", ",".join(map(str, groups)), ",".join(map(str, prefixes)), heads, max(q_len, hi // 20), hi,
                   rng.choice(["bf16", "bf16", "fp16"]), rng.choice([32, 64, 128]) if fp8 else page, q_len, fp8,
                   rng.choice([0, 0, 0, 2]))


def _spread(count, lo, hi):
    return [lo + round((hi - lo) * (i + 0.5) / count) for i in range(count)]


def _numbers(text):
    return [int(x) for x in text.split(",")]


# --- inputs ------------------------------------------------------------------


def _shuffled(values, seed):
    order = torch.randperm(len(values), generator=torch.Generator().manual_seed(seed))
    return [values[int(i)] for i in order]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _fill(table, pages, perm, start=0):
    """Row b of the table gets pages[b] pages of the permutation, in order."""
    flat = perm.tolist()
    rows = []
    for n in pages:
        rows.append(flat[start:start + n] + [-1] * (table.shape[1] - n))
        start += n
    if rows:
        table.copy_(_ints(rows))
    return start


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"shared": _prepare_shared, "copy": _prepare_copy, "fork": _prepare_fork, "reserve": _prepare_reserve,
            "compact": _prepare_compact}[case["kind"]](case, seed, g)


def _prepare_shared(case, seed, g):
    sizes, page = _numbers(case["groups"]), case["page"]
    shared = [p // page if n > 1 else 0 for n, p in zip(sizes, _numbers(case["prefixes"]))]  # whole pages
    batch = sum(sizes)
    own_tokens = _shuffled(_spread(batch, case["lo"], case["hi"]), seed)
    lens, pages, b = [], [], 0
    for n, s, p in zip(sizes, shared, _numbers(case["prefixes"])):
        for _ in range(n):  # (a prefix's last tokens, short of a page, lie in every sequence's own pages)
            lens.append(p + own_tokens[b])
            pages.append(-(-lens[b] // page) - s)
            b += 1
    total = sum(pages) + sum(shared)
    perm = torch.randperm(total, generator=g, device="cuda").tolist()
    width = max(-(-n // page) for n in lens)
    rows, at, b = [], 0, 0
    for n, s in zip(sizes, shared):
        head = perm[at:at + s]
        at += s
        for _ in range(n):
            row = head + perm[at:at + pages[b]]
            at += pages[b]
            rows.append(row + [0] * (width - len(row)))
            b += 1
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    if case["empty"]:  # a group of sequences that hold nothing
        starts.append(batch + case["empty"])
        shared.append(0)
        lens += [0] * case["empty"]
        rows += [[0] * width] * case["empty"]
    dtype = DTYPES[case["dtype"]]
    kv = torch.randn(total, page, WIDTH, generator=g, device="cuda", dtype=dtype)
    shape = (len(lens), case["heads"], WIDTH) if case["q_len"] == 1 else \
        (len(lens), case["q_len"], case["heads"], WIDTH)
    q = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
    scale = None
    if case["fp8"]:  # one scale a page
        scale = kv.float().abs().amax(dim=(1, 2)) / 448.0
        kv = (kv.float() / scale[:, None, None]).to(torch.float8_e4m3fn)
    return {"kind": "shared", "q": q, "kv": kv, "kv_scale": scale, "seqlens": _ints(lens), "table": _ints(rows),
            "prefix_lens": _ints([s * page for s in shared]), "group_starts": _ints(starts), "lens": lens}


def _pool(case, g, pages):
    return torch.randn(pages, case["page"], WIDTH, generator=g, device="cuda",
                       dtype=DTYPES[case.get("dtype", "bf16")])


def _prepare_copy(case, seed, g):
    perm = torch.randperm(case["pool"], generator=g, device="cuda").to(torch.int32)
    n = case["pairs"]
    return {"kind": "copy", "kv": _pool(case, g, case["pool"]), "src": perm[:n].contiguous(),
            "dst": perm[n:2 * n].contiguous()}


def _prepare_fork(case, seed, g):
    batch, page, mode = case["batch"], case["page"], case["mode"]
    lens = _shuffled(_spread(batch, case["lo"], case["hi"]), seed)
    if mode == "split":
        lens = lens[:1] + [0] * (batch - 1)
    pages = [-(-n // page) for n in lens]
    total = sum(pages) + batch + 5  # room for the copies of the last pages
    perm = torch.randperm(total, generator=g, device="cuda")
    table = torch.full((batch, case["width"]), -1, dtype=torch.int32, device="cuda")
    used = _fill(table, pages, perm)
    refs = torch.zeros(total, dtype=torch.int32, device="cuda")
    refs[perm[:used]] = 1
    state = {"kind": "fork", "mode": mode, "table": table, "seqlens": _ints(lens), "refs": refs, "page": page}
    c = torch.Generator().manual_seed(seed)
    if mode == "free":
        state["ended"] = (torch.rand(batch, generator=c) < 0.33).cuda()
        return state
    if mode == "split":
        parents = [0] * batch
    else:
        pick = torch.randint(0, 8, (batch,), generator=c).tolist()
        parents = [i // 8 * 8 + pick[i] % min(8, batch - i // 8 * 8) for i in range(batch)]
    state["parents"] = _ints(parents)
    state["kv"] = _pool(case, g, total)
    return state


def _prepare_reserve(case, seed, g):
    batch, page = case["batch"], case["page"]
    lens = _shuffled(_spread(batch, case["lo"], case["hi"]), seed)
    pages = [-(-n // page) for n in lens]
    perm = torch.randperm(case["pool"], generator=g, device="cuda")
    table = torch.full((batch, -(-(case["hi"] + case["most"]) // page)), -1, dtype=torch.int32, device="cuda")
    used = _fill(table, pages, perm)
    refs = torch.zeros(case["pool"], dtype=torch.int32, device="cuda")
    refs[perm[:used]] = 1
    c = torch.Generator().manual_seed(seed)
    new = torch.randint(0, case["most"] + 1, (batch,), generator=c) if case["most"] > 1 else torch.ones(batch)
    return {"kind": "reserve", "table": table, "seqlens": _ints(lens), "refs": refs, "page": page,
            "new_tokens": new.to(torch.int32).cuda()}


def _prepare_compact(case, seed, g):
    page = case["page"]
    lens = _shuffled(_spread(case["batch"], case["lo"], case["hi"]), seed)
    pages = [-(-n // page) for n in lens]
    perm = torch.randperm(case["pool"], generator=g, device="cuda")
    table = torch.full((case["batch"], max(pages) + 3), -1, dtype=torch.int32, device="cuda")
    used = _fill(table, pages, perm)
    refs = torch.zeros(case["pool"], dtype=torch.int32, device="cuda")
    refs[perm[:used]] = 1
    # every second sequence's first page is the one of the sequence before it
    share = torch.arange(1, case["batch"], 2, device="cuda")
    refs[table[share, 0].long()] -= 1
    table[share, 0] = table[share - 1, 0]
    refs[table[share, 0].long()] += 1
    return {"kind": "compact", "table": table, "refs": refs, "kv": _pool(case, g, case["pool"])}


# --- one pass ----------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    tm = _package()
    if s["kind"] == "shared":
        out, lse = tm.mla_decode_shared(s["q"], s["kv"], s["seqlens"], s["table"], s["prefix_lens"], s["group_starts"],
                                        softmax_scale=SCALE, return_lse=True, kv_scale=s["kv_scale"])
        return {"out": out, "lse": lse}
    if s["kind"] == "copy":
        refused = tm.copy_pages(s["kv"], s["src"], s["dst"])
        return {"cache": s["kv"], "refused": refused}
    if s["kind"] == "fork":
        if s["mode"] == "free":
            table, lens, refs = tm.free_sequences(s["table"], s["seqlens"], s["refs"], s["ended"])
            return {"table": table, "seqlens": lens, "refs": refs}
        table, lens, refs, missing = tm.fork_sequences(s["kv"], s["table"], s["seqlens"], s["refs"], s["parents"])
        return {"table": table, "seqlens": lens, "refs": refs, "missing": missing, "cache": s["kv"]}
    if s["kind"] == "reserve":
        table, refs, missing = tm.reserve_pages(s["table"], s["seqlens"], s["refs"], s["new_tokens"], s["page"])
        return {"table": table, "refs": refs, "missing": missing}
    table, refs, live = tm.compact_pages(s["kv"], s["table"], s["refs"])
    return {"table": table, "refs": refs, "live": live, "cache": s["kv"]}


def _run_plain(s):
    return {"shared": _plain_shared, "copy": _plain_copy, "fork": _plain_fork, "reserve": _plain_reserve,
            "compact": _plain_compact}[s["kind"]](s)


def _plain_shared(s):
    q, kv, page = s["q"], s["kv"], s["kv"].shape[1]
    flat = q.unsqueeze(1) if q.dim() == 3 else q
    batch, q_len, heads, _ = flat.shape
    out = torch.zeros(batch, q_len, heads, VALUE, dtype=q.dtype, device=q.device)
    lse = torch.full((batch, q_len, heads), -math.inf, dtype=torch.float32, device=q.device)
    for b, n in enumerate(s["lens"]):
        if n == 0:
            continue
        ids = s["table"][b, :-(-n // page)].long()
        rows = kv[ids].float()
        if s["kv_scale"] is not None:
            rows = rows * s["kv_scale"][ids][:, None, None]
        rows = rows.reshape(-1, WIDTH)[:n]
        logits = (flat[b].reshape(-1, WIDTH).float() @ rows.t()) * SCALE  # [q_len * heads, n]
        if q_len > 1:  # query token t sees the first n - (q_len - 1 - t) tokens
            sees = n - (q_len - 1) + torch.arange(q_len, device=q.device).repeat_interleave(heads)
            logits = logits.masked_fill(torch.arange(n, device=q.device) >= sees[:, None], -math.inf)
        top = logits.amax(dim=1, keepdim=True)
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
        p = torch.exp(logits - top)
        total = p.sum(dim=1, keepdim=True)
        row = (p @ rows[:, :VALUE]) / torch.where(total == 0, torch.ones_like(total), total)
        out[b] = row.reshape(q_len, heads, VALUE).to(q.dtype)
        lse[b] = (top + torch.log(total)).reshape(q_len, heads)
    if q.dim() == 3:
        return {"out": out[:, 0], "lse": lse[:, 0]}
    return {"out": out, "lse": lse}


def _plain_copy(s):
    pages, n = s["kv"].shape[0], s["src"].shape[0]
    src, dst = s["src"].long(), s["dst"].long()
    good = (src >= 0) & (src < pages) & (dst >= 0) & (dst < pages)
    order = torch.arange(n, device=src.device)
    last = torch.full((pages + 1,), -1, dtype=torch.int64, device=src.device)
    last.scatter_reduce_(0, torch.where(good, dst, pages), order, "amax")  # the last pair that writes a page
    good &= (last[dst.clamp(0, pages - 1)] == order) & (last[src.clamp(0, pages - 1)] < 0)
    s["kv"][dst[good]] = s["kv"][src[good]]
    return {"cache": s["kv"], "refused": (n - good.sum()).to(torch.int32).reshape(1)}


def _held(table, pages):
    return (table >= 0) & (table < pages)


def _uses(table, mask, pages):
    """How often each page stands in the masked entries of a table."""
    index = torch.where(mask, table.long(), torch.full_like(table, pages, dtype=torch.int64)).flatten()
    count = torch.zeros(pages + 1, dtype=torch.int64, device=table.device)
    return count.scatter_add_(0, index, torch.ones_like(index))[:pages]


def _lowest_free(counts):
    """The free pages in ascending order (then the number of pages, repeated)."""
    pages = counts.shape[0]
    ids = torch.arange(pages, device=counts.device)
    return torch.where(counts == 0, ids, torch.full_like(ids, pages)).sort().values


def _plain_fork(s):
    table, lens, refs, page = s["table"], s["seqlens"], s["refs"], s["page"]
    batch, width = table.shape
    pages = refs.shape[0]
    if s["mode"] == "free":
        ended = s["ended"]
        gone = _uses(table, _held(table, pages) & ended[:, None], pages)
        return {"table": torch.where(ended[:, None], torch.full_like(table, -1), table),
                "seqlens": torch.where(ended, torch.zeros_like(lens), lens),
                "refs": (refs - gone).clamp(min=0).to(torch.int32)}
    parents, row = s["parents"].long(), torch.arange(batch, device=table.device)
    valid = (parents >= 0) & (parents < batch)
    p = parents.clamp(0, batch - 1)
    first = torch.full((batch,), batch, dtype=torch.int64, device=table.device)
    first.scatter_reduce_(0, p, torch.where(valid, row, torch.full_like(row, batch)), "amin")
    keeper = valid & (first[p] == row)  # the first child keeps the parent's last page and what it has reserved
    old, n = table[p], torch.where(valid, lens[p], torch.zeros_like(lens))
    held = _held(old, pages)
    full = (n // page).clamp(max=width).long()
    share = valid[:, None] & held & (keeper[:, None] | (torch.arange(width, device=table.device) < full[:, None]))
    new = torch.where(share, old, torch.full_like(old, -1))
    counts = (refs - _uses(table, _held(table, pages), pages) + _uses(new, share, pages)).clamp(min=0)
    last = full.clamp(max=width - 1)[:, None]
    copied = valid & ~keeper & (n % page > 0) & (full < width) & held.gather(1, last)[:, 0]
    free = _lowest_free(counts)
    missing = (copied.sum() - (counts == 0).sum()).clamp(min=0)
    done = missing == 0
    target = free[(copied.cumsum(0) - 1).clamp(0, pages - 1)]
    new = new.scatter(1, last, torch.where(copied, target.to(torch.int32), new.gather(1, last)[:, 0])[:, None])
    counts = counts + _uses(target[:, None], copied[:, None], pages)
    make = copied & done
    s["kv"][target[make]] = s["kv"][old.gather(1, last)[:, 0][make].long()]
    return {"table": torch.where(done, new, table), "seqlens": torch.where(done, n, lens),
            "refs": torch.where(done, counts, refs).to(torch.int32), "missing": missing.to(torch.int32).reshape(1),
            "cache": s["kv"]}


def _plain_reserve(s):
    table, refs, page = s["table"], s["refs"], s["page"]
    batch, width = table.shape
    pages = refs.shape[0]
    need = (s["seqlens"].clamp(min=0) + s["new_tokens"].clamp(min=0) + page - 1) // page
    lack = (torch.arange(width, device=table.device) < need[:, None]) & ~_held(table, pages)
    rank = (lack.flatten().cumsum(0) - 1).reshape(batch, width)
    beyond = (need - width).clamp(min=0).sum()  # pages the table has no column for
    missing = (lack.sum() - (refs == 0).sum()).clamp(min=0) + beyond
    done = missing == 0
    take = lack & done
    ids = _lowest_free(refs)[rank.clamp(0, pages - 1)]
    return {"table": torch.where(take, ids.to(torch.int32), table),
            "refs": (refs + _uses(ids, take, pages)).to(torch.int32), "missing": missing.to(torch.int32).reshape(1)}


def _plain_compact(s):
    table, refs, kv = s["table"], s["refs"], s["kv"]
    pages = refs.shape[0]
    ids = torch.arange(pages, device=refs.device)
    used = refs > 0
    live = used.sum()
    to = ids.clone()
    moved, holes = ids[used & (ids >= live)], ids[~used & (ids < live)]
    to[moved] = holes
    kv[holes] = kv[moved]
    counts = refs.clone()
    counts[holes] = refs[moved]
    counts[moved] = 0
    new = torch.where(_held(table, pages), to[table.clamp(0, pages - 1).long()].to(torch.int32), table)
    return {"table": new, "refs": counts, "live": live.to(torch.int32).reshape(1), "cache": kv}


# --- what one pass cannot do without -------------------------------------------


def work(case):
    page = case["page"]
    row = page * WIDTH * 2  # bytes of a page
    if case["kind"] == "shared":
        sizes, prefixes = _numbers(case["groups"]), _numbers(case["prefixes"])
        own_tokens = sum(_spread(sum(sizes), case["lo"], case["hi"]))
        tokens, seen = own_tokens, own_tokens  # tokens read, tokens attended to
        for n, p in zip(sizes, prefixes):
            whole = p // page * page if n > 1 else 0
            tokens += whole + n * (p - whole)
            seen += n * p
        rows = (sum(sizes) + case["empty"]) * case["heads"] * case["q_len"]
        cache = tokens * WIDTH * (1 if case["fp8"] else 2)
        return {"bytes": cache + rows * (2 * WIDTH + 2 * VALUE + 4),
                "flops": 2 * case["heads"] * case["q_len"] * seen * (WIDTH + VALUE)}
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pairs"] * row + 8 * case["pairs"], "flops": 0}
    if case["kind"] == "fork":
        batch = case["batch"]
        lens = _spread(batch, case["lo"], case["hi"])
        pool = sum(-(-n // page) for n in (lens[:1] if case["mode"] == "split" else lens)) + batch + 5
        # copies of last pages: all rows but one, or about the share of eight
        # draws that repeat one drawn before (the table and counts besides)
        copies = {"split": batch - 1, "beam": batch * 0.34, "free": 0}[case["mode"]]
        return {"bytes": 2 * int(copies) * row + 8 * batch * case["width"] + 8 * pool + 12 * batch, "flops": 0}
    if case["kind"] == "reserve":
        width = -(-(case["hi"] + case["most"]) // page)
        return {"bytes": 8 * case["batch"] * width + 8 * case["pool"] + 8 * case["batch"], "flops": 0}
    lens = _spread(case["batch"], case["lo"], case["hi"])
    live = sum(-(-n // page) for n in lens) - case["batch"] // 2
    pool = case["pool"]
    moves = live * (pool - live) // pool  # pages in use behind the live-th, expected
    return {"bytes": 2 * moves * row + 8 * case["batch"] * (-(-max(lens) // page) + 3) + 8 * pool, "flops": 0}


# --- the definition, apart from the forms above --------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "shared":
        return _exact_shared(s)
    if case["kind"] == "copy":
        pairs = list(zip(s["src"].tolist(), s["dst"].tolist()))
        return {"cache": _moved(s["kv"], pairs), "refused": _zero()}
    refs = s["refs"].tolist()
    rows = s["table"].tolist()
    if case["kind"] == "fork":
        return _exact_fork(s, rows, refs)
    if case["kind"] == "reserve":
        free = iter([i for i, c in enumerate(refs) if c == 0])
        new = s["new_tokens"].tolist()
        for b, n in enumerate(s["seqlens"].tolist()):
            for j in range(-(-(n + new[b]) // s["page"])):
                if rows[b][j] < 0:
                    rows[b][j] = next(free)
                    refs[rows[b][j]] = 1
        return {"table": _int_rows(rows), "refs": _int_rows(refs), "missing": _zero()}
    live = sum(c > 0 for c in refs)
    holes = [i for i in range(live) if refs[i] == 0]
    moves = dict(zip([i for i in range(live, len(refs)) if refs[i] > 0], holes))
    for a, b in moves.items():
        refs[b], refs[a] = refs[a], 0
    return {"table": _int_rows([[moves.get(e, e) for e in r] for r in rows]), "refs": _int_rows(refs),
            "live": _int_rows([live]), "cache": _moved(s["kv"], moves.items())}


def _int_rows(rows):
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def _zero():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _moved(kv, pairs):
    new = kv.clone()
    for a, b in pairs:
        new[b] = kv[a]
    return new


def _exact_fork(s, rows, refs):
    page, lens = s["page"], s["seqlens"].tolist()
    if s["mode"] == "free":
        for b, end in enumerate(s["ended"].tolist()):
            if end:
                for e in rows[b]:
                    if e >= 0:
                        refs[e] -= 1
                rows[b] = [-1] * len(rows[b])
                lens[b] = 0
        return {"table": _int_rows(rows), "seqlens": _int_rows(lens), "refs": _int_rows(refs)}
    parents = s["parents"].tolist()
    new, copies, kept = [], [], set()
    for i, p in enumerate(parents):
        row = list(rows[p])
        if p in kept:
            whole = lens[p] // page
            row = row[:whole] + [-1] * (len(row) - whole)
            if lens[p] % page:
                copies.append((i, whole, rows[p][whole]))
        kept.add(p)
        new.append(row)
    for r in rows:
        for e in r:
            if e >= 0:
                refs[e] -= 1
    for r in new:
        for e in r:
            if e >= 0:
                refs[e] += 1
    free = iter([i for i, c in enumerate(refs) if c == 0])
    moves = []
    for i, j, e in copies:
        new[i][j] = next(free)
        moves.append((e, new[i][j]))
    for _, b in moves:
        refs[b] = 1
    return {"table": _int_rows(new), "seqlens": _int_rows([lens[p] for p in parents]), "refs": _int_rows(refs),
            "missing": _zero(), "cache": _moved(s["kv"], moves)}


def _exact_shared(s):
    """Softmax attention in float64, one sequence and query token at a time."""
    q, kv = s["q"], s["kv"]
    many = q if q.dim() == 4 else q[:, None]
    out = torch.zeros(*many.shape[:3], VALUE, dtype=torch.float64, device=q.device)
    lse = torch.full(many.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["seqlens"].tolist()):
        if n == 0:
            continue
        ids = s["table"][b, :-(-n // kv.shape[1])].long()
        keys = kv[ids].double()
        if s["kv_scale"] is not None:
            keys *= s["kv_scale"][ids].double()[:, None, None]
        keys = keys.flatten(0, 1)[:n]
        for t in range(many.shape[1]):
            seen = keys[:n - (many.shape[1] - 1 - t)]
            logits = (seen @ many[b, t].double().t().contiguous()).t().contiguous() * SCALE
            lse[b, t] = torch.logsumexp(logits, dim=-1)
            out[b, t] = torch.softmax(logits, dim=-1) @ seen[:, :VALUE].contiguous()
    if q.dim() == 3:
        return {"out": out[:, 0], "lse": lse[:, 0]}
    return {"out": out, "lse": lse}
