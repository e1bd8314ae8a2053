"""Operators of decoding with several continuations of a text: cases, plain forms, 64-bit values and the work each cannot do without.

Five operators on the paged cache of one decoding step, in the order in which beam search runs them:

* ``select``  -- the best continuations over beams and vocabulary, from logits and the beams' scores;
* ``fork``    -- page tables reordered by the chosen parents: whole pages shared, partly filled ones given a
  page of their own, pages that nobody holds any more back in the pool;
* ``compact`` -- the pages in use moved to the lowest numbers, tables renamed;
* ``copy``    -- the moves that fork and compact ask for, in the caches of all layers;
* ``prefix``  -- attention of one new token per request where groups of requests share their first pages.

``run`` computes them with elementary torch operations, or, where ``own`` is set, with
manifesto_b200.beams and manifesto_b200.paged on the same tensors (torch's default stream is
the library's default stream, the legacy one).
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
      "e5m2": torch.float8_e5m2}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1, "e5m2": 1}


def listed():
    return [
        # one user's beam search, a small vocabulary: latency
        {"name": "select_one", "op": "select", "batch": 1, "beams": 4, "vocab": 32000, "out": 4, "dtype": "bf16",
         "ended": False},
        # a server's step: 64 prompts of 8 beams, twice as many candidates as beams
        {"name": "select_batch", "op": "select", "batch": 64, "beams": 8, "vocab": 128256, "out": 16, "dtype": "bf16",
         "ended": False},
        # rows of an odd length in 32 bits, some of the beams at their end already
        {"name": "select_odd", "op": "select", "batch": 7, "beams": 5, "vocab": 49999, "out": 10, "dtype": "f32",
         "ended": True},
        # 16 prompts of 8 beams, reordered between two tokens
        {"name": "fork_beams", "op": "fork", "before": 128, "after": 128, "beams": 8, "longest": 2000, "page": 16,
         "spare": 1000, "short": False},
        # many samples of many prompts, long ones, most pages shared, and a pool that does not suffice
        {"name": "fork_many", "op": "fork", "before": 1500, "after": 2048, "beams": 4, "longest": 8191, "page": 32,
         "spare": 20000, "short": True},
        # a small cache that shrinks to the pages it uses
        {"name": "compact_small", "op": "compact", "requests": 48, "longest": 700, "page": 16, "pages": 4096,
         "limit": "used"},
        # a large one, pages of a few tokens, two fifths of it given back
        {"name": "compact_large", "op": "compact", "requests": 2048, "longest": 3999, "page": 8, "pages": 1000000,
         "limit": "most"},
        # the partly filled pages of forked beams, in a few layers
        {"name": "copy_beams", "op": "copy", "moves": 56, "pages": 1024, "caches": 16, "kv_heads": 8, "dim": 128,
         "page": 16, "cache": "bf16", "order": "HND", "partial": True},
        # whole pages of an 8-bit cache moved by a compaction
        {"name": "copy_pages_fp8", "op": "copy", "moves": 2001, "pages": 4500, "caches": 8, "kv_heads": 8, "dim": 128,
         "page": 32, "cache": "e4m3", "order": "NHD", "partial": False},
        # four beams of one short prompt: latency
        {"name": "prefix_one", "op": "prefix", "groups": 1, "members": 4, "shared": 900, "own": 40, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "order": "HND", "softcap": 0.0,
         "idle": False},
        # 24 prompts of 8 beams, lengths of all sizes, an 8-bit cache in token order, capped scores
        {"name": "prefix_beams_fp8", "op": "prefix", "groups": 24, "members": 8, "shared": 6000, "own": 128, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 32, "order": "NHD", "softcap": 30.0,
         "idle": False},
        # a server whose requests all begin with the same long instructions
        {"name": "prefix_system", "op": "prefix", "groups": 1, "members": 250, "shared": 8192, "own": 700, "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "order": "HND", "softcap": 0.0,
         "idle": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["select", "fork", "compact", "copy", "prefix", "prefix"])
    if op == "select":
        beams, vocab = rng.choice([1, 2, 3, 4, 5, 8, 16]), _log(rng, 300, 200_000)
        return {"op": op, "batch": _log(rng, 1, max(1, min(256, 32_000_000 // (beams * vocab)))), "beams": beams,
                "vocab": vocab, "out": beams * rng.choice([1, 2]), "dtype": rng.choice(["bf16", "f16", "f32"]),
                "ended": rng.random() < 0.5}
    if op == "fork":
        before, page = _log(rng, 1, 1500), rng.choice([1, 7, 16, 24, 32, 64, 128])
        return {"op": op, "before": before, "after": _log(rng, 1, 2048), "beams": rng.choice([1, 2, 4, 5, 8]),
                "longest": _log(rng, 1, 256 * page), "page": page, "spare": _log(rng, 1, 20000),
                "short": rng.random() < 0.3}
    if op == "compact":
        requests, page, longest = _log(rng, 1, 2048), rng.choice([1, 7, 16, 24, 32, 64, 128]), _log(rng, 1, 400)
        held = requests * (longest // page + 1)
        return {"op": op, "requests": requests, "longest": longest, "page": page,
                "pages": held + _log(rng, 1, max(1, 1_000_000 - held)), "limit": rng.choice(["used", "most"])}
    kv_heads, dim, page = rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 80, 96, 128, 256]), rng.choice([1, 8, 16, 20, 32, 64, 128])
    dtype, order = rng.choice(["bf16", "f16"]), rng.choice(["HND", "NHD"])
    cache = rng.choice([dtype, dtype, "e4m3", "e5m2"])
    if op == "copy":
        moves = _log(rng, 1, max(1, min(3000, 100_000_000 // (kv_heads * dim * page * 16))))
        return {"op": op, "moves": moves, "pages": 2 * moves + _log(rng, 1, moves + 10), "caches": rng.choice([2, 6, 16]),
                "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache, "order": order,
                "partial": rng.random() < 0.5}
    group, groups = rng.choice([1, 2, 4, 5, 7, 8]), _log(rng, 1, 40)
    members = _log(rng, 2, max(2, 250 // groups))
    # no more than half of the largest listed case's products and bytes
    rows = groups * members * kv_heads * group * dim
    shared = _log(rng, 1, max(1, min(30_000, 4_000_000_000 // rows, 40_000_000 // (groups * kv_heads * dim))))
    return {"op": op, "groups": groups, "members": members, "shared": shared,
            "own": _log(rng, 1, max(1, min(1000, 40_000_000 // (groups * members * kv_heads * dim)))),
            "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cache": cache, "page": page,
            "order": order, "softcap": rng.choice([0.0, 0.0, 50.0]), "idle": rng.random() < 0.3}


# ------------------------------------------------------------------ what a case's numbers mean

def _book(case, rng):
    """Tables of requests in families that share their first pages, as earlier forks left them: lengths, table,
    holders of each page beyond the first, and the numbers of the pages in use."""
    n, page = case.get("before", case.get("requests")), case["page"]
    beams = case.get("beams", 4)
    i = np.arange(n)
    family = i // beams
    lens = np.maximum(1, (case["longest"] * (1 + family)) // (1 + family[-1])) - (i * 7) % 5
    lens = np.maximum(lens, 0)
    held = -(-lens // page)
    # a family shares the first three quarters of what its shortest member has in whole pages
    least = np.full(family[-1] + 1, 1 << 40)
    np.minimum.at(least, family, lens // page)
    common = (3 * least[family]) // 4
    lead = i % beams == 0
    fresh = np.where(lead, held, held - common)
    start = np.cumsum(fresh) - fresh
    width = max(1, -(-(case["longest"] + 1) // page))
    col = np.arange(width)[None, :]
    index = np.where(~lead[:, None] & (col < common[:, None]), start[family * beams][:, None] + col,
                     start[:, None] + col - np.where(lead, 0, common)[:, None])
    used = int(fresh.sum())
    pages = case["pages"] if "pages" in case else used + case["spare"]
    number = rng.permutation(pages).astype(np.int32)
    table = np.where(col < held[:, None], number[np.clip(index, 0, used - 1 if used else 0)], -1).astype(np.int32)
    holders = np.bincount(table[table >= 0], minlength=pages)
    return lens, table, np.maximum(holders - 1, 0).astype(np.int32), number[used:], pages


def _parents(case, rng):
    """Who continues whom: among the beams of a family some have several children and some none; families keep their
    places; rows past the families before (and a few others) begin empty."""
    i = np.arange(case["after"])
    beams, n = case["beams"], case["before"]
    family = (i * n // case["after"]) // beams
    first = family * beams
    size = np.minimum(beams, n - first)
    chosen = first + np.minimum(rng.geometric(0.4, len(i)) - 1, size - 1)
    return np.where(rng.random(len(i)) < 0.02, -1, chosen).astype(np.int32)


def _groups(case):
    """Members and shared tokens of each group; members own between 1 and `own` tokens besides, an idle one has none at all."""
    g, page = np.arange(case["groups"]), case["page"]
    members = np.full(case["groups"], case["members"])
    shared = np.maximum(1, case["shared"] * (g + 1) // case["groups"]) // page * page
    i = np.arange(int(members.sum()))
    lens = np.repeat(shared, members) + 1 + (i * 131 + 17) % case["own"]
    return members, shared, np.where(i % 50 == 3, 0, lens) if case["idle"] else lens


def _width(case):
    return -(-(case["shared"] + case["own"]) // case["page"])


def _tokens(case):
    """Tokens that each move copies."""
    if not case["partial"]:
        return np.full(case["moves"], case["page"])
    return 1 + (np.arange(case["moves"]) * 7) % max(1, case["page"] - 1)


def work(case):
    op = case["op"]
    if op == "select":
        rows = case["batch"] * case["beams"]
        return {"bytes": 1.0 * rows * case["vocab"] * SIZE[case["dtype"]] + 8.0 * rows + 16.0 * case["batch"] * case["out"],
                "flops": 3.0 * rows * case["vocab"]}
    if op in ("fork", "compact"):
        rng = np.random.default_rng(0)
        lens, table, _, free, pages = _book(case, rng)
        n = len(lens)
        rows = n + (case["after"] if op == "fork" else n)
        # tables, lengths and parents read and written; the holders of each page; the list of free pages
        return {"bytes": 4.0 * (rows * table.shape[1] + 2 * rows + 2 * pages + 2 * len(free)), "flops": 1.0 * rows * table.shape[1]}
    if op == "copy":
        row = case["kv_heads"] * case["dim"] * SIZE[case["cache"]]
        return {"bytes": 2.0 * int(_tokens(case).sum()) * row * case["caches"] + 16.0 * case["moves"], "flops": 0.0}
    d, hq, hkv, e, c = case["dim"], case["heads"], case["kv_heads"], SIZE[case["dtype"]], SIZE[case["cache"]]
    members, shared, lens = _groups(case)
    r = len(lens)
    seen = int(lens.sum())
    read = int(shared.sum()) + int(np.maximum(lens - np.repeat(shared, members), 0).sum())
    return {"bytes": 2.0 * read * hkv * d * c + 2.0 * r * hq * d * e + 4 * r * (hq + 1) + 4.0 * read / case["page"],
            "flops": 4.0 * seen * hq * d}


# ------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype, std=1.0):
    made = torch.float32 if dtype == torch.float32 or dtype.itemsize == 1 else dtype
    return torch.empty(shape, dtype=made, device="cuda").normal_(0.0, std, generator=gen).to(dtype)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _empty(*shape):
    return torch.full(shape, -1, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": case, "keep": {}}
    op = case["op"]
    if op == "select":
        batch, beams, vocab, out = case["batch"], case["beams"], case["vocab"], case["out"]
        s["logits"] = _normal(gen, (batch * beams, vocab), DT[case["dtype"]], 2.5)
        banned = torch.randint(0, vocab, (max(1, vocab // 100),), generator=gen, device="cuda")
        s["logits"][:, banned] = -math.inf
        s["end"] = int(rng.integers(0, vocab))
        s["logits"][:, s["end"]] = 9.0  # the end is likely
        s["scores"] = -(torch.rand(batch * beams, generator=gen, device="cuda") * 3.0 + 20.0)
        s["ended"] = _i32((rng.random(batch * beams) < 0.3) * 1) if case["ended"] else None
        s |= {"scores_after": torch.zeros(batch, out, device="cuda"), "tokens": _empty(batch, out),
              "parents": _empty(batch, out), "ended_after": _empty(batch, out)}
        return s
    if op in ("fork", "compact"):
        lens, table, shares, free, pages = _book(case, rng)
        n, width = table.shape
        rows = case["after"] if op == "fork" else n
        count = len(free)
        if op == "fork":
            s["parents"] = _i32(_parents(case, rng))
            if case["short"]:  # fewer free pages than the forks ask for
                count = min(count, max(1, case["after"] // 20))
        else:
            used = pages - len(free)
            s["limit"] = 0 if case["limit"] == "used" else used + (pages - used) // 2
        s |= {"lens": _i32(lens), "table": _i32(table), "shares": _i32(shares), "pages": pages, "count": count,
              "free": _i32(np.concatenate([np.zeros(3), free[:count], np.zeros(pages)])[:pages] if 3 + count <= pages
                           else np.concatenate([free[:count], np.zeros(pages)])[:pages]),
              "pool": _i32([3 if 3 + count <= pages else 0, count]), "table_after": _empty(rows, width),
              "lens_after": _empty(rows), "shares_after": _empty(pages), "free_after": _empty(pages),
              "pool_after": _empty(4), "moves": _empty(rows if op == "fork" else max(1, pages // 2), 4),
              "numbers": _empty(pages)}
        return s
    if op == "copy":
        pages, page = case["pages"], case["page"]
        shape = ((pages, case["kv_heads"], page, case["dim"]) if case["order"] == "HND" else
                 (pages, page, case["kv_heads"], case["dim"]))
        s["caches"] = [_normal(gen, shape, DT[case["cache"]]) for _ in range(case["caches"])]
        number = rng.permutation(pages)[:2 * case["moves"]]
        src = number[:case["moves"]]
        if case["partial"]:  # several forks of one page
            src = src[np.arange(case["moves"]) // 3 * 3]
        tokens = _tokens(case)
        tokens = tokens[np.arange(case["moves"]) // 3 * 3] if case["partial"] else tokens
        s["moves"] = _i32(np.stack([src, number[case["moves"]:], tokens, 0 * src], 1))
        s["count"] = _i32([case["moves"]])
        return s
    dtype, d, hq, hkv, page = DT[case["dtype"]], case["dim"], case["heads"], case["kv_heads"], case["page"]
    members, shared, lens = _groups(case)
    r, width = len(lens), _width(case)
    of_group = np.repeat(np.arange(len(members)), members)
    first = (shared // page)[of_group]                              # pages of the shared part
    held = np.maximum(-(-lens // page), first)
    common = np.cumsum(shared // page) - shared // page             # numbers of the shared pages start here
    mine = held - first
    start = int((shared // page).sum()) + np.cumsum(mine) - mine
    pages = int((shared // page).sum() + mine.sum()) + 3
    col = np.arange(width)[None, :]
    index = np.where(col < first[:, None], common[of_group][:, None] + col, start[:, None] + col - first[:, None])
    table = np.where(col < held[:, None], rng.permutation(pages)[np.clip(index, 0, pages - 1)], -1)
    shape = (pages, hkv, page, d) if case["order"] == "HND" else (pages, page, hkv, d)
    scaled = SIZE[case["cache"]] == 1
    for name in ("k", "v"):
        s[name + "_cache"] = _normal(gen, shape, DT[case["cache"]], 40.0 if scaled else 1.0)
        # what an 8-bit code of each head is multiplied by
        s[name + "_scale"] = (torch.rand(hkv, generator=gen, device="cuda") + 0.5) / 40.0 if scaled else None
    s |= {"lens": _i32(lens), "table": _i32(table), "starts": _i32(np.concatenate([[0], np.cumsum(members)])),
          "shared": _i32(shared), "q": _normal(gen, (r, hq, d), dtype), "requests": r,
          "out": torch.zeros(r, hq, d, dtype=dtype, device="cuda"), "lse": torch.zeros(r, hq, device="cuda")}
    return s


# ------------------------------------------------------------------ the plain forms

def _plain_select(s, case):
    batch, beams, vocab, out = case["batch"], case["beams"], case["vocab"], case["out"]
    # Candidates are ranked by scores in 64 bits: two that differ by less than the 32-bit rounding keep their order.
    x = s["logits"].double()
    score = x - torch.logsumexp(x, 1, keepdim=True) + s["scores"].double()[:, None]
    if s["ended"] is not None:  # a beam at its end goes on as it is, by the end's token alone
        gone = s["ended"].bool()[:, None]
        at_end = torch.arange(vocab, device="cuda") == s["end"]
        score = torch.where(gone, torch.where(at_end, s["scores"].double()[:, None], -math.inf), score)
    best, at = torch.sort(score.view(batch, beams * vocab), dim=1, descending=True, stable=True)
    best, at = best[:, :out], at[:, :out]
    there = best > -math.inf
    parent = at // vocab + torch.arange(batch, device="cuda")[:, None] * beams
    token = at % vocab
    over = token == s["end"]
    i32 = torch.int32
    return {"scores": best.float(), "tokens": torch.where(there, token, -1).to(i32),
            "parents": torch.where(there, parent, -1).to(i32), "ended": (there & over).to(i32)}


def _exclusive(x):
    return x.cumsum(0) - x


def _place(size, at, values, keep):
    """An int32 array of -1 with `values` at `at` where `keep`."""
    out = torch.full((size + 1,), -1, dtype=torch.int64, device="cuda")
    out[torch.where(keep, at, size)] = values
    return out[:size].to(torch.int32)


def _plain_fork(s, case):
    page, pages, width = case["page"], s["pages"], s["table"].shape[1]
    lens, table, n, rows = s["lens"].long(), s["table"].long(), case["before"], case["after"]
    parent = s["parents"].long()
    alive = (parent >= 0) & (parent < n)
    p = parent.clamp(0, n - 1)
    row = torch.arange(rows, device="cuda")
    first = torch.full((n,), rows, dtype=torch.int64, device="cuda")
    first.scatter_reduce_(0, p, torch.where(alive, row, rows), "amin")
    need = alive & (first[p] != row) & (lens[p] % page != 0)
    col = torch.arange(width, device="cuda")
    held = col < -(-lens // page)[:, None]
    childless = first == rows
    gone = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")
    gone.index_add_(0, torch.where(held & childless[:, None], table, pages).view(-1),
                    torch.ones(n * width, dtype=torch.int64, device="cuda"))
    left = s["shares"].long() - gone[:pages]
    freed = left < 0
    n_freed = freed.sum()
    page_no = torch.arange(pages, device="cuda")
    combined = _place(pages, _exclusive(freed.long()), page_no, freed).long()
    old = s["free"].long()[(s["pool"][0].long() + page_no).clamp(0, pages - 1)]
    combined = torch.where(page_no < n_freed, combined, old[(page_no - n_freed).clamp(0, pages - 1)])
    before = _exclusive(need.long())
    there = s["pool"][1] + n_freed
    fits = alive & (~need | (before < there))
    taken = torch.where(need & fits, before + 1, 0).amax()
    dst = combined[before.clamp(0, pages - 1)]
    full = (lens[p] // page)[:, None]
    after = torch.where(held[p] & fits[:, None], table[p], -1)
    after = torch.where((need & fits)[:, None] & (col == full), dst[:, None], after)
    extra = fits & (first[p] != row)
    more = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")
    more.index_add_(0, torch.where(extra[:, None] & (col < full), table[p], pages).view(-1),
                    torch.ones(rows * width, dtype=torch.int64, device="cuda"))
    moved = need & fits
    src = table[p].gather(1, full.clamp(max=width - 1))[:, 0]
    moves = torch.stack([_place(rows, before, x, moved) for x in (src, dst, lens[p] % page, 0 * src)], 1)
    count = there - taken
    listed_free = torch.where(page_no < count, combined[(page_no + taken).clamp(0, pages - 1)], -1)
    i32 = torch.int32
    return {"table": after.to(i32), "lens": torch.where(fits, lens[p], 0).to(i32),
            "shares": (left.clamp(min=0) + more[:pages]).to(i32), "free": listed_free.to(i32), "moves": moves,
            "pool": torch.stack([0 * taken, count, moved.sum(), (alive & ~fits).sum()]).to(i32)}


def _plain_compact(s, case):
    page, pages, width = case["page"], s["pages"], s["table"].shape[1]
    page_no = torch.arange(pages, device="cuda")
    listed_free = s["free"].long()[(s["pool"][0].long() + page_no).clamp(0, pages - 1)]
    free = torch.zeros(pages + 1, dtype=torch.bool, device="cuda")
    free[torch.where(page_no < s["pool"][1], listed_free, pages)] = True
    free = free[:pages]
    used = pages - s["pool"][1].long()
    limit = torch.clamp(used, min=s["limit"])
    leave, take = ~free & (page_no >= limit), free & (page_no < limit)
    rank_leave, rank_take = _exclusive(leave.long()), _exclusive(take.long())
    count = leave.sum()
    room = max(1, pages // 2)
    src = _place(room, rank_leave, page_no, leave).long()
    moved = page_no[:room] < count
    dst = torch.where(moved, _place(pages, rank_take, page_no, take).long()[:room], -1)
    numbers = page_no.clone()
    numbers = torch.cat([numbers, numbers[:1]])
    numbers[torch.where(moved, src, pages)] = dst
    numbers = numbers[:pages]
    shares = torch.zeros(pages, dtype=torch.int64, device="cuda")
    shares.index_add_(0, numbers, torch.where(free, 0, s["shares"].long()))
    now_free = (free & (page_no >= limit)) | leave | (take & (rank_take >= count))
    held = torch.arange(width, device="cuda") < -(-s["lens"].long() // page)[:, None]
    table = torch.where(held, numbers[s["table"].long().clamp(0, pages - 1)], -1)
    four = torch.stack([src, dst, torch.where(moved, page, -1), torch.where(moved, 0, -1)], 1)
    zero = 0 * count
    i32 = torch.int32
    return {"table": table.to(i32), "shares": shares.to(i32), "numbers": numbers.to(i32), "moves": four.to(i32),
            "free": _place(pages, _exclusive(now_free.long()), page_no, now_free),
            "pool": torch.stack([zero, s["pool"][1].long(), count, zero]).to(i32)}


def _plain_copy(s, case):
    """Each move's tokens, of every cache at once; 8-bit codes as the bytes that they are."""
    src, dst, tokens = (s["moves"][:, i].long() for i in range(3))
    token = torch.arange(case["page"], device="cuda")
    kept = token < tokens[:, None]                                     # [moves, page]
    move, at = torch.where(kept)
    pages, heads = s["caches"][0].shape[0], case["kv_heads"]
    h = torch.arange(heads, device="cuda")
    if case["order"] == "HND":
        here, there = ((x[move][:, None] * heads + h) * case["page"] + at[:, None] for x in (src, dst))
    else:
        here, there = ((x[move] * case["page"] + at)[:, None] * heads + h for x in (src, dst))
    here, there = here.reshape(-1), there.reshape(-1)
    kind = torch.uint8 if SIZE[case["cache"]] == 1 else DT[case["cache"]]
    flat = [c.view(kind).view(pages * heads * case["page"], case["dim"]) for c in s["caches"]]
    [x.index_copy_(0, there, x[here]) for x in flat]
    return s["caches"]


def _gathered(cache, table, case, scale):
    """[rows, kv_heads, tokens, dim] of the pages in the table, in 32 bits."""
    wide = cache.view(torch.uint8)[table].view(cache.dtype) if SIZE[case["cache"]] == 1 else cache[table]
    x = (wide.transpose(1, 2) if case["order"] == "HND" else wide.permute(0, 3, 1, 2, 4)).float()
    x = x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])
    return x if scale is None else x * scale[:, None, None]


def _capped(score, case):
    score = score * (1.0 / math.sqrt(case["dim"]))
    return case["softcap"] * torch.tanh(score / case["softcap"]) if case["softcap"] else score


def _plain_prefix(s, case):
    hq, hkv, d, page, groups, members = (case[x] for x in ("heads", "kv_heads", "dim", "page", "groups", "members"))
    each, r = hq // hkv, s["requests"]
    table, lens, shared = s["table"].long(), s["lens"].long(), s["shared"].long()
    of = torch.arange(r, device="cuda") // members
    q = s["q"].float().view(r, hkv, each, d)
    # the shared tokens: a group's queries against its first member's pages
    columns = max(1, case["shared"] // page)
    k = _gathered(s["k_cache"], table[::members, :columns].clamp(min=0), case, s["k_scale"])
    q_all = q.view(groups, members, hkv, each, d).permute(0, 2, 1, 3, 4).reshape(groups, hkv, members * each, d)
    common = _capped(q_all @ k.transpose(2, 3), case).view(groups, hkv, members, each, -1)
    common = common.permute(0, 2, 1, 3, 4).reshape(r, hkv, each, -1)
    token = torch.arange(columns * page, device="cuda")
    seen = token < torch.minimum(lens, shared[of])[:, None]
    common = common.masked_fill(~seen[:, None, None], -math.inf)
    # the tokens of its own
    mine = shared[of][:, None] // page + torch.arange(-(-case["own"] // page) + 1, device="cuda")
    own_table = table.gather(1, mine.clamp(max=table.shape[1] - 1)).clamp(min=0)
    alone = _capped(q @ _gathered(s["k_cache"], own_table, case, s["k_scale"]).transpose(2, 3), case)
    token = shared[of][:, None] + torch.arange(alone.shape[-1], device="cuda")
    alone = alone.masked_fill(~(token < lens[:, None])[:, None, None], -math.inf)
    score = torch.cat([common, alone], -1)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)  # a request without tokens: zeros, and the logarithm of none
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    w = p / torch.where(total == 0, 1.0, total)
    w_common = w[..., :common.shape[-1]].reshape(groups, members, hkv, each, -1).permute(0, 2, 1, 3, 4)
    v = _gathered(s["v_cache"], table[::members, :columns].clamp(min=0), case, s["v_scale"])
    out = (w_common.reshape(groups, hkv, members * each, -1) @ v).view(groups, hkv, members, each, d)
    out = out.permute(0, 2, 1, 3, 4).reshape(r, hkv, each, d)
    out = out + w[..., common.shape[-1]:] @ _gathered(s["v_cache"], own_table, case, s["v_scale"])
    return {"out": out.reshape(r, hq, d).to(s["q"].dtype), "lse": (total.log() + top).reshape(r, hq)}


# ------------------------------------------------------------------ the framework's

def _at(t):
    return 0 if t is None else t.data_ptr()


def _handle(s, case):
    """The operator's description, as a program makes it once and keeps it over its steps.  It is made on the first
    pass, since prepare() also runs where the operators are not there."""
    if "handle" in s["keep"]:
        return s["keep"]["handle"]
    from manifesto_b200 import CUDABackend, DType, beams, paged
    kinds = {"bf16": DType.BFLOAT16, "f16": DType.FLOAT16, "f32": DType.FLOAT32, "e4m3": DType.FLOAT8_E4M3,
             "e5m2": DType.FLOAT8_E5M2}
    CUDABackend(0)
    op = case["op"]
    if op == "select":
        h = beams.BeamSelect(kinds[case["dtype"]], case["vocab"], case["beams"], case["out"], max_batch=case["batch"],
                             end_token=s["end"])
    elif op in ("fork", "compact"):
        rows = max(case["before"], case["after"]) if op == "fork" else case["requests"]
        h = paged.PageBook(case["page"], s["table"].shape[1], s["pages"], max_requests=rows)
    else:
        cache = s["caches"][0] if op == "copy" else s["k_cache"]
        layout = paged.CacheLayout(cache.shape[0], case["page"], case["kv_heads"], case["dim"], kinds[case["cache"]],
                                   case["order"])
        if op == "copy":
            h = paged.PageCopy(layout, [_at(c) for c in s["caches"]])
        else:
            h = paged.PrefixAttention(layout, case["heads"], kinds[case["dtype"]], max_pages=s["table"].shape[1],
                                      max_requests=s["requests"], scale=1.0 / math.sqrt(case["dim"]),
                                      softcap=case["softcap"], k_scale_inv=_at(s["k_scale"]), v_scale_inv=_at(s["v_scale"]))
    s["keep"]["handle"] = h
    return h


def _own(s, case):
    op, h = case["op"], _handle(s, case)
    if op == "select":
        h.run(s["logits"].data_ptr(), s["scores"].data_ptr(), case["batch"], s["scores_after"].data_ptr(),
              s["tokens"].data_ptr(), s["parents"].data_ptr(), ended=_at(s["ended"]), ended_after=s["ended_after"].data_ptr())
        return {"scores": s["scores_after"], "tokens": s["tokens"], "parents": s["parents"], "ended": s["ended_after"]}
    if op == "fork":
        h.fork(s["table"].data_ptr(), s["lens"].data_ptr(), case["before"], s["parents"].data_ptr(), case["after"],
               s["shares"].data_ptr(), s["free"].data_ptr(), s["pool"].data_ptr(), s["table_after"].data_ptr(),
               s["lens_after"].data_ptr(), s["shares_after"].data_ptr(), s["free_after"].data_ptr(),
               s["pool_after"].data_ptr(), s["moves"].data_ptr())
        return {"table": s["table_after"], "lens": s["lens_after"], "shares": s["shares_after"], "free": s["free_after"],
                "moves": s["moves"], "pool": s["pool_after"]}
    if op == "compact":
        h.compact(s["table"].data_ptr(), s["lens"].data_ptr(), case["requests"], s["shares"].data_ptr(), s["free"].data_ptr(),
                  s["pool"].data_ptr(), s["limit"], s["table_after"].data_ptr(), s["shares_after"].data_ptr(),
                  s["free_after"].data_ptr(), s["pool_after"].data_ptr(), s["numbers"].data_ptr(), s["moves"].data_ptr())
        return {"table": s["table_after"], "shares": s["shares_after"], "numbers": s["numbers"], "moves": s["moves"],
                "free": s["free_after"], "pool": s["pool_after"]}
    if op == "copy":
        h.run(s["moves"].data_ptr(), case["moves"], count=s["count"].data_ptr())
        return s["caches"]
    h.run(s["q"].data_ptr(), s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(),
          s["requests"], s["starts"].data_ptr(), s["shared"].data_ptr(), case["groups"], s["out"].data_ptr(),
          s["lse"].data_ptr())
    return {"out": s["out"], "lse": s["lse"]}


PLAIN = {"select": _plain_select, "fork": _plain_fork, "compact": _plain_compact, "copy": _plain_copy,
         "prefix": _plain_prefix}


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return PLAIN[case["op"]](s, case)


# ------------------------------------------------------------------ in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    return {"select": _exact_select, "fork": _exact_fork, "compact": _exact_compact, "copy": _exact_copy,
            "prefix": _exact_prefix}[case["op"]](s, case)


def _exact_select(s, case):
    batch, beams, vocab, out = case["batch"], case["beams"], case["vocab"], case["out"]
    got = {"scores": torch.full((batch, out), -math.inf, dtype=torch.float64), "tokens": torch.full((batch, out), -1, dtype=torch.int32),
           "parents": torch.full((batch, out), -1, dtype=torch.int32), "ended": torch.zeros(batch, out, dtype=torch.int32)}
    for b in range(batch):
        best = []
        for k in range(beams):
            row, base = b * beams + k, float(s["scores"][b * beams + k])
            if s["ended"] is not None and int(s["ended"][row]):
                best.append((-base, k * vocab + s["end"]))
                continue
            x = s["logits"][row].double()
            top = x.max()
            base -= float(top + torch.log(torch.exp(x - top).sum()))
            # every token that may be among the `out` best of its beam, ties included
            low = torch.topk(x, min(out, vocab)).values[-1]
            at = torch.where((x >= low) & (x > -math.inf))[0]
            best += [(-(base + v), k * vocab + t) for v, t in zip(x[at].tolist(), at.tolist())]
        for j, (v, at) in enumerate(sorted(best)[:out]):
            got["scores"][b, j], got["tokens"][b, j] = -v, at % vocab
            got["parents"][b, j], got["ended"][b, j] = b * beams + at // vocab, int(at % vocab == s["end"])
    return got


def _exact_fork(s, case):
    page, lens, parents = case["page"], s["lens"].tolist(), s["parents"].tolist()
    table, rows, n = s["table"].cpu().numpy(), case["after"], case["before"]
    shares = s["shares"].cpu().numpy().copy()
    head, count = s["pool"].tolist()
    children = set(p for p in parents if 0 <= p < n)
    for q in range(n):
        if q not in children:
            np.subtract.at(shares, table[q, :-(-lens[q] // page)], 1)
    freed = np.where(shares < 0)[0]
    shares[freed] = 0
    pool = np.concatenate([freed, s["free"].cpu().numpy()[head:head + count]]).astype(np.int32)
    after, lens_after = np.full((rows, table.shape[1]), -1, np.int32), np.zeros(rows, np.int32)
    seen, moves, taken, asked, refused = set(), [], 0, 0, 0
    for r, p in enumerate(parents):
        if not 0 <= p < n:
            continue
        full, rest = lens[p] // page, lens[p] % page
        if p in seen:
            if rest:
                asked += 1
                if asked > len(pool):
                    refused += 1
                    continue
                moves.append((table[p, full], pool[taken], rest, 0))
                after[r, full] = pool[taken]
                taken += 1
            shares[table[p, :full]] += 1
            after[r, :full] = table[p, :full]
        else:
            seen.add(p)
            after[r, :full + (rest > 0)] = table[p, :full + (rest > 0)]
        lens_after[r] = lens[p]
    free = np.full(s["pages"], -1, np.int32)
    free[:len(pool) - taken] = pool[taken:]
    four = np.full((rows, 4), -1, np.int32)
    if moves:
        four[:len(moves)] = moves
    return {"table": after, "lens": lens_after, "shares": shares.astype(np.int32), "free": free, "moves": four,
            "pool": np.array([0, len(pool) - taken, len(moves), refused], np.int32)}


def _exact_compact(s, case):
    page, pages, lens = case["page"], s["pages"], s["lens"].tolist()
    head, count = s["pool"].tolist()
    free = np.sort(s["free"].cpu().numpy()[head:head + count])
    used = np.setdiff1d(np.arange(pages), free)
    limit = max(len(used), s["limit"])
    src = used[used >= limit]
    dst = free[:len(src)]
    numbers = np.arange(pages, dtype=np.int32)
    numbers[src] = dst
    shares = np.zeros(pages, np.int32)
    shares[numbers[used]] = s["shares"].cpu().numpy()[used]
    table = s["table"].cpu().numpy().copy()
    for r, row in enumerate(table):
        row[-(-lens[r] // page):] = -1
    table[table >= 0] = numbers[table[table >= 0]]
    left = np.setdiff1d(np.arange(pages), numbers[used])
    listed_free = np.full(pages, -1, np.int32)
    listed_free[:len(left)] = left
    moves = np.full((max(1, pages // 2), 4), -1, np.int32)
    moves[:len(src)] = np.stack([src, dst, np.full(len(src), page), np.zeros(len(src))], 1)
    return {"table": table, "shares": shares, "numbers": numbers, "moves": moves, "free": listed_free,
            "pool": np.array([0, count, len(src), 0], np.int32)}


def _exact_copy(s, case):
    # copies round nothing: the values themselves
    for cache in s["caches"]:
        bits = cache.view(torch.uint8) if cache.element_size() == 1 else cache
        for src, dst, tokens, _ in s["moves"].tolist():
            if case["order"] == "HND":
                bits[dst, :, :tokens] = bits[src, :, :tokens]
            else:
                bits[dst, :tokens] = bits[src, :tokens]
    return s["caches"]


def _exact_prefix(s, case):
    """Request by request over all its tokens, without a thought of what is shared."""
    hq, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["requests"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((s["requests"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        pages = s["table"][r, :-(-n // page)].long()
        kv = []
        for name in ("k", "v"):
            cache = s[name + "_cache"]
            rows = (cache.view(torch.uint8)[pages].view(cache.dtype) if cache.element_size() == 1 else cache[pages]).double()
            rows = rows.transpose(0, 1).flatten(1, 2) if case["order"] == "HND" else rows.flatten(0, 1).transpose(0, 1)
            if s[name + "_scale"] is not None:
                rows = rows * s[name + "_scale"].double()[:, None, None]
            kv.append(rows[:, :n])  # [kv_heads, tokens, dim]
        score = torch.einsum("hgd,hnd->hgn", s["q"][r].double().view(hkv, hq // hkv, d), kv[0]) / math.sqrt(d)
        if case["softcap"]:
            score = case["softcap"] * torch.tanh(score / case["softcap"])
        total = torch.logsumexp(score, 2)
        lse[r] = total.reshape(hq)
        out[r] = torch.einsum("hgn,hnd->hgd", torch.exp(score - total[..., None]), kv[1]).reshape(hq, d)
    return {"out": out, "lse": lse}
