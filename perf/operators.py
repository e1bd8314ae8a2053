"""The paged-cache decode operators: cases, plain forms, 64-bit values and the work each cannot do without.

Four operators that one decoding step runs in this order:

* ``assign``  -- page tables, slots and positions of a step's new tokens, from the requests' lengths;
* ``rope``    -- rotary positions of a [tokens, heads, head_dim] array, forward and gradient;
* ``append``  -- rotary positions of a step's queries and keys, the keys and values written to their cache slots;
* ``attn``    -- attention of one new token per request over the paged cache.

``run`` computes them with elementary torch operations, or, where ``own`` is set, with
manifesto_b200.paged on the same tensors (torch's default stream is the library's default
stream, the legacy one).
"""
import math

import numpy as np
import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
      "e5m2": torch.float8_e5m2}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1, "e5m2": 1}
FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}


def listed():
    return [
        # a small server's decoding step: eight requests, a token each
        {"name": "assign_decode", "op": "assign", "requests": 8, "longest": 700, "page": 16, "new": "one",
         "most_new": 1, "short": False},
        # a large server's mixed step: chunks of prompts beside single tokens, and a pool that runs out
        {"name": "assign_prompts", "op": "assign", "requests": 1500, "longest": 8192, "page": 32, "new": "mixed",
         "most_new": 511, "short": True},
        # training: the queries of 16384 tokens, 32 heads of 128
        {"name": "rope_train", "op": "rope", "tokens": 16384, "heads": 32, "dim": 128, "rot": 128, "layout": "half",
         "dtype": "bf16", "inverse": False, "far": 8192, "scaling": "none"},
        # the gradient of a partial rotation in 32 bits, interleaved, at far positions with interpolated frequencies
        {"name": "rope_grad", "op": "rope", "tokens": 4099, "heads": 20, "dim": 80, "rot": 32,
         "layout": "interleaved", "dtype": "f32", "inverse": True, "far": 500000, "scaling": "linear"},
        # a decoding step of 48 requests, queries, keys and values in one packed projection
        {"name": "append_decode", "op": "append", "tokens": 48, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "layout": "half", "dtype": "bf16", "cache": "bf16", "page": 16, "order": "HND", "far": 8192,
         "scaling": "none"},
        # a long prompt into an 8-bit cache
        {"name": "append_prompt_fp8", "op": "append", "tokens": 32771, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 128, "layout": "half", "dtype": "bf16", "cache": "e4m3", "page": 32, "order": "NHD", "far": 131072,
         "scaling": "bands"},
        # one user, a short chat: latency
        {"name": "attn_one_short", "op": "attn", "requests": 1, "longest": 333, "spread": "equal", "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "order": "HND", "window": 0,
         "softcap": 0.0, "slopes": False},
        # a server's ordinary batch, lengths of all sizes
        {"name": "attn_batch", "op": "attn", "requests": 64, "longest": 4096, "spread": "ragged", "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 16, "order": "HND", "window": 0,
         "softcap": 0.0, "slopes": False},
        # two very long documents: the length has to be split
        {"name": "attn_long", "op": "attn", "requests": 2, "longest": 131071, "spread": "equal", "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "bf16", "page": 64, "order": "HND", "window": 0,
         "softcap": 0.0, "slopes": False},
        # a full server with an 8-bit cache in token order and capped scores
        {"name": "attn_full_fp8", "op": "attn", "requests": 256, "longest": 8192, "spread": "ragged", "heads": 32,
         "kv_heads": 8, "dim": 128, "dtype": "bf16", "cache": "e4m3", "page": 32, "order": "NHD", "window": 0,
         "softcap": 30.0, "slopes": False},
        # a head of keys for each head of queries, a sliding window, a bias by distance, odd pages, empty requests
        {"name": "attn_window_bias", "op": "attn", "requests": 33, "longest": 6001, "spread": "holes", "heads": 16,
         "kv_heads": 16, "dim": 64, "dtype": "f16", "cache": "f16", "page": 20, "order": "HND", "window": 1000,
         "softcap": 0.0, "slopes": True},
        # all queries share one wide head of keys; one request far longer than the others
        {"name": "attn_shared_wide", "op": "attn", "requests": 9, "longest": 30011, "spread": "one_long",
         "heads": 16, "kv_heads": 1, "dim": 256, "dtype": "bf16", "cache": "bf16", "page": 16, "order": "HND",
         "window": 0, "softcap": 0.0, "slopes": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["assign", "rope", "append", "attn", "attn", "attn"])
    if op == "assign":
        new = rng.choice(["one", "mixed"])
        return {"op": op, "requests": _log(rng, 1, 4000), "longest": _log(rng, 1, 8192),
                "page": rng.choice([1, 7, 16, 24, 32, 64, 128]), "new": new,
                "most_new": 1 if new == "one" else _log(rng, 2, 180), "short": rng.random() < 0.3}
    layout, scaling = rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "base", "bands"])
    if op == "rope":
        dim = rng.choice([64, 72, 80, 96, 128, 256])
        heads = _log(rng, 1, 64)
        return {"op": op, "tokens": _log(rng, 1, max(1, 60_000_000 // (heads * dim))), "heads": heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2]), "layout": layout, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "inverse": rng.random() < 0.5, "far": _log(rng, 100, 1_000_000), "scaling": scaling}
    kv_heads, group = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 5, 7, 8, 16])
    dim, dtype = rng.choice([64, 80, 96, 128, 256]), rng.choice(["bf16", "f16"])
    cache = rng.choice([dtype, dtype, "e4m3", "e5m2"])
    both = {"heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cache": cache,
            "page": rng.choice([1, 8, 16, 20, 32, 64, 128]), "order": rng.choice(["HND", "NHD"])}
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 100_000_000 // (kv_heads * (group + 2) * dim)), **both,
                "rot": rng.choice([dim, dim, dim // 2]), "layout": layout, "far": _log(rng, 100, 1_000_000),
                "scaling": scaling}
    requests = _log(rng, 1, 300)
    # no more than a quarter of the largest listed cache, at the longest length for every request
    most = max(1, min(100_000, 500_000_000 // (requests * kv_heads * dim)))
    return {"op": op, "requests": requests, "longest": _log(rng, 1, most),
            "spread": rng.choice(["equal", "ragged", "holes", "one_long"]), **both,
            "window": rng.choice([0, 0, 0, 1, 100, 1024]), "softcap": rng.choice([0.0, 0.0, 50.0]),
            "slopes": rng.random() < 0.25}


# ------------------------------------------------------------------ what a case's numbers mean

def _lengths(case):
    """The requests' lengths, before the seed puts them in another order."""
    n, top = case["requests"], case["longest"]
    spread = case.get("spread", "ragged")
    i = np.arange(n)
    if spread == "equal":
        return np.full(n, top, np.int64)
    if spread == "one_long":
        return np.where(i == 0, top, np.maximum(1, top // 40 - 3 * i))
    got = np.maximum(1, (top * (i + 1)) // n)
    return np.where(i % 5 == 1, 0, got) if spread == "holes" else got


def _new_tokens(case):
    """The new tokens of each request: one each, or chunks of prompts beside single tokens and idle requests."""
    i = np.arange(case["requests"])
    if case["new"] == "one":
        return np.ones(case["requests"], np.int64)
    return np.where(i % 7 == 3, 0, np.where(i % 3 == 1, 1, 1 + (i * 37) % case["most_new"]))


def _table_width(case):
    return max(1, -(-(case["longest"] + case.get("most_new", 0)) // case["page"]))


def _frequencies(case):
    """Frequency of each rotated pair in 64 bits, rounded once to the 32 bits that both sides are given."""
    rot, scaling, factor, base = case["rot"], case["scaling"], 8.0, 10000.0
    if scaling == "base" and rot > 2:
        base *= factor ** (rot / (rot - 2))
    f = base ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if scaling == "linear":
        f /= factor
    if scaling == "bands":  # short waves as they are, long ones interpolated, a ramp between
        turns = 8192 * f / (2 * math.pi)
        ramp = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
        f = (1 - ramp) * f / factor + ramp * f
    return f.astype(np.float32)


def _magnitude(case):
    return 1.0 if case["scaling"] == "none" else 1.125


def work(case):
    op = case["op"]
    if op == "assign":
        n, have, new, page = case["requests"], _lengths(case), _new_tokens(case), case["page"]
        tokens, pages = int(new.sum()), int((-(-(have + new) // page) - -(-have // page)).sum())
        return {"bytes": 16.0 * tokens + 8.0 * pages + 4 * (4 * n + 1), "flops": 2.0 * tokens}
    if op == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2.0 * n * case["dim"] * SIZE[case["dtype"]] + 4 * case["tokens"] + 2 * case["rot"],
                "flops": 3.0 * n * case["rot"]}
    d, hq, hkv, e, c = case["dim"], case["heads"], case["kv_heads"], SIZE[case["dtype"]], SIZE[case["cache"]]
    if op == "append":
        t = case["tokens"]
        return {"bytes": 1.0 * t * ((2 * hq + 2 * hkv) * d * e + 2 * hkv * d * c + 12) + 2 * case["rot"],
                "flops": 3.0 * t * (hq + hkv) * case["rot"]}
    n = _lengths(case)
    n = np.minimum(n, case["window"]) if case["window"] else n
    seen, r = int(n.sum()), case["requests"]
    return {"bytes": 2.0 * seen * hkv * d * c + 2.0 * r * hq * d * e + 4 * r * (hq + 1) + 4.0 * seen / case["page"],
            "flops": 4.0 * seen * hq * d}


# ------------------------------------------------------------------ inputs

def _normal(gen, shape, dtype, std=1.0):
    made = torch.float32 if dtype == torch.float32 or dtype.itemsize == 1 else dtype
    return torch.empty(shape, dtype=made, device="cuda").normal_(0.0, std, generator=gen).to(dtype)


def _shuffled(values, rng):
    return torch.from_numpy(rng.permutation(values).astype(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": case, "keep": {}}
    if case["op"] == "assign":
        page, width, n = case["page"], _table_width(case), case["requests"]
        order = rng.permutation(n)
        have, new = _lengths(case)[order], _new_tokens(case)[order]
        held, after = -(-have // page), -(-(have + new) // page)
        pool = rng.permutation(int(held.sum() + (after - held).sum()) + 5).astype(np.int32)
        table = np.full((n, width), -1, np.int32)
        table[np.arange(width)[None, :] < held[:, None]] = pool[:int(held.sum())]
        free = pool[int(held.sum()):]
        count = int((after - held).sum()) // 2 if case["short"] else len(free)  # half of the pages are there
        tokens = int(new.sum())
        s |= {"lens": torch.from_numpy(have.astype(np.int32)).cuda(), "new": torch.from_numpy(new.astype(np.int32)).cuda(),
              "table": torch.from_numpy(table).cuda(), "free": torch.from_numpy(free).cuda(), "tokens": tokens,
              "pool": torch.tensor([0, count], dtype=torch.int32, device="cuda"),
              "slots": torch.zeros(tokens, dtype=torch.int64, device="cuda"),
              "positions": torch.zeros(tokens, dtype=torch.int32, device="cuda"),
              "owner": torch.zeros(tokens, dtype=torch.int32, device="cuda"),
              "starts": torch.zeros(n + 1, dtype=torch.int32, device="cuda"),
              "lens_after": torch.zeros(n, dtype=torch.int32, device="cuda"),
              "pool_after": torch.zeros(4, dtype=torch.int32, device="cuda")}
        return s
    dtype = DT[case["dtype"]]
    d = case["dim"]
    if case["op"] != "attn":
        t = case["tokens"]
        s["positions"] = torch.from_numpy(rng.integers(0, case["far"], t).astype(np.int32)).cuda()
        s["frequencies"] = torch.from_numpy(_frequencies(case)).cuda()
    if case["op"] == "rope":
        s["x"] = _normal(gen, (t, case["heads"], d), dtype)
        s["y"] = torch.zeros_like(s["x"])
        return s
    hq, hkv, page = case["heads"], case["kv_heads"], case["page"]
    if case["op"] == "append":
        # queries, keys and values side by side, as one projection leaves them
        s["qkv"] = _normal(gen, (t, (hq + 2 * hkv) * d), dtype)
        pages = -(-t // page) + 3
        s["slots"] = torch.from_numpy(rng.permutation(pages * page)[:t].astype(np.int64)).cuda()
        s["q_out"] = torch.zeros(t, hq, d, dtype=dtype, device="cuda")
    else:
        lens = rng.permutation(_lengths(case))
        held = -(-lens // page)
        pages = int(held.sum()) + 3
        table = np.full((len(lens), _table_width(case)), -1, np.int32)
        table[np.arange(table.shape[1])[None, :] < held[:, None]] = rng.permutation(pages)[:int(held.sum())]
        s |= {"lens": torch.from_numpy(lens.astype(np.int32)).cuda(), "table": torch.from_numpy(table).cuda(),
              "q": _normal(gen, (len(lens), hq, d), dtype), "out": torch.zeros(len(lens), hq, d, dtype=dtype, device="cuda"),
              "lse": torch.zeros(len(lens), hq, dtype=torch.float32, device="cuda"), "slopes": None}
        if case["slopes"]:  # a geometric run of slopes over the heads
            s["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) / hq)
    shape = (pages, hkv, page, d) if case["order"] == "HND" else (pages, page, hkv, d)
    scaled = case["cache"] in FP8_MAX
    for name in ("k", "v"):
        if case["op"] == "append":
            s[name + "_cache"] = torch.zeros(shape, dtype=DT[case["cache"]], device="cuda")
        else:
            s[name + "_cache"] = _normal(gen, shape, DT[case["cache"]], 40.0 if scaled else 1.0)
        # what an 8-bit code of each head is multiplied by
        s[name + "_scale"] = (torch.rand(hkv, generator=gen, device="cuda") + 0.5) / 40.0 if scaled else None
    return s


# ------------------------------------------------------------------ the plain forms

def _cos_sin(s, case):
    # The angle is made in 64 bits: a 32-bit product of a far position and a frequency has lost its phase.
    a = s["positions"].double()[:, None] * s["frequencies"].double()
    return (a.cos() * _magnitude(case)).float()[:, None], (a.sin() * _magnitude(case)).float()[:, None]


def _rotate(x, cos, sin, case, inverse=False):
    """The rotated [tokens, heads, dim] in 32 bits; `inverse` turns the other way, which is the gradient."""
    x, rot = x.float(), case["rot"]
    sin = -sin if inverse else sin
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., :rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _split(s, case):
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    q, k, v = s["qkv"].view(-1, hq + 2 * hkv, d).split([hq, hkv, hkv], 1)
    return q, k, v


def _plain_assign(s, case):
    page, tokens = case["page"], s["tokens"]
    have, new = s["lens"].long(), s["new"].long()
    held = (have + page - 1) // page
    need = (have + new + page - 1) // page - held
    before = need.cumsum(0) - need
    fits = (need == 0) | (before + need <= s["pool"][1])
    col = torch.arange(s["table"].shape[1], device="cuda")
    j = col - held[:, None]
    fresh = (j >= 0) & (j < need[:, None]) & fits[:, None]
    at = (s["pool"][0] + before[:, None] + j).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][at], s["table"])
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)])
    owner = torch.repeat_interleave(torch.arange(len(have), device="cuda"), new, output_size=tokens)
    position = have[owner] + torch.arange(tokens, device="cuda") - starts[owner]
    slot = table[owner, position // page].long() * page + position % page
    slot = torch.where(fits[owner], slot, -1)
    taken = torch.where(fits & (need > 0), before + need, 0).amax()
    pool = torch.stack([s["pool"][0] + taken, s["pool"][1] - taken, starts[-1], (~fits).sum()])
    i32 = torch.int32
    return {"table": table, "slots": slot, "positions": position.to(i32), "owner": owner.to(i32), "starts": starts.to(i32),
            "lens": torch.where(fits, have + new, have).to(i32), "pool": pool.to(i32)}


def _encode(x, case, scale):
    """Cache values as they are stored: in the inputs' type, or as the nearest 8-bit code of x over its head's scale."""
    if case["cache"] not in FP8_MAX:
        return x.to(DT[case["cache"]])
    top = FP8_MAX[case["cache"]]
    return (x * (1.0 / scale)[:, None]).clamp(-top, top).to(DT[case["cache"]])


def _plain_append(s, case):
    q, k, v = _split(s, case)
    cos, sin = _cos_sin(s, case)
    page, off = s["slots"] // case["page"], s["slots"] % case["page"]
    for name, x in (("k", _rotate(k, cos, sin, case)), ("v", v.float())):
        at = s[name + "_cache"].permute(0, 2, 1, 3) if case["order"] == "HND" else s[name + "_cache"]
        code = _encode(x, case, s[name + "_scale"])
        if case["cache"] in FP8_MAX:
            at, code = at.view(torch.uint8), code.view(torch.uint8)
        at[page, off] = code
    return {"q": _rotate(q, cos, sin, case).to(q.dtype), "k": s["k_cache"], "v": s["v_cache"]}


def _gathered(cache, table, case, scale):
    """[requests, kv_heads, tokens, dim] of the pages in the table, in 32 bits."""
    wide = cache.view(torch.uint8)[table].view(cache.dtype) if case["cache"] in FP8_MAX else cache[table]
    x = (wide.transpose(1, 2) if case["order"] == "HND" else wide.permute(0, 3, 1, 2, 4)).float()
    x = x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])
    return x if scale is None else x * scale[:, None, None]


def _plain_attn(s, case):
    hq, hkv, d = case["heads"], case["kv_heads"], case["dim"]
    lens, table = s["lens"].long()[:, None], s["table"].long().clamp(min=0)
    q = s["q"].float().view(-1, hkv, hq // hkv, d)
    score = q @ _gathered(s["k_cache"], table, case, s["k_scale"]).transpose(2, 3) * (1.0 / math.sqrt(d))
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    token = torch.arange(score.shape[-1], device="cuda")
    if s["slopes"] is not None:
        score = score + s["slopes"].view(hkv, -1, 1) * (token - (lens - 1))[:, None, None].float()
    seen = token < lens
    if case["window"]:
        seen = seen & (token >= lens - case["window"])
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)  # a request without tokens: zeros, and the logarithm of none
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    out = (p / torch.where(total == 0, 1.0, total)) @ _gathered(s["v_cache"], table, case, s["v_scale"])
    lse = total.log() + top
    return {"out": out.reshape(-1, hq, d).to(s["q"].dtype), "lse": lse.reshape(-1, hq)}


# ------------------------------------------------------------------ the framework's

def _at(t):
    return 0 if t is None else t.data_ptr()


def _handle(s, case):
    """The operator's description, as a program makes it once and keeps it over its steps.  It is made on the first
    pass, since prepare() also runs where the operators are not there."""
    if "handle" in s["keep"]:
        return s["keep"]["handle"]
    from manifesto_b200 import CUDABackend, DType, paged
    kinds = {"bf16": DType.BFLOAT16, "f16": DType.FLOAT16, "f32": DType.FLOAT32, "e4m3": DType.FLOAT8_E4M3,
             "e5m2": DType.FLOAT8_E5M2}
    CUDABackend(0)
    op = case["op"]
    if op == "assign":
        h = paged.PageAssigner(page_size=case["page"], max_pages=_table_width(case))
    else:
        if op != "attn":
            rope = paged.Rope(_at(s["frequencies"]), kinds[case["dtype"]], case["dim"], case["rot"], case["layout"],
                              _magnitude(case))
        if op != "rope":
            layout = paged.CacheLayout(s["k_cache"].shape[0], case["page"], case["kv_heads"], case["dim"],
                                       kinds[case["cache"]], case["order"])
        if op == "rope":
            h = rope
        elif op == "append":
            # compat: codes rounded to nearest and saturated
            h = paged.RopeAppend(rope, layout, case["heads"], k_scale_inv=_at(s["k_scale"]), v_scale_inv=_at(s["v_scale"]),
                                 compat=1, token_stride=s["qkv"].shape[1])
        else:
            h = paged.PagedAttention(layout, case["heads"], kinds[case["dtype"]], max_pages=_table_width(case),
                                     scale=1.0 / math.sqrt(case["dim"]), softcap=case["softcap"], window=case["window"],
                                     slopes=_at(s["slopes"]), k_scale_inv=_at(s["k_scale"]), v_scale_inv=_at(s["v_scale"]))
    s["keep"]["handle"] = h
    return h


def _own(s, case):
    op, h = case["op"], _handle(s, case)
    if op == "assign":
        h.assign(s["lens"].data_ptr(), s["new"].data_ptr(), case["requests"], s["table"].data_ptr(), s["free"].data_ptr(),
                 s["pool"].data_ptr(), s["tokens"], s["slots"].data_ptr(), s["positions"].data_ptr(), s["owner"].data_ptr(),
                 s["starts"].data_ptr(), s["lens_after"].data_ptr(), s["pool_after"].data_ptr())
        return {"table": s["table"], "slots": s["slots"], "positions": s["positions"], "owner": s["owner"],
                "starts": s["starts"], "lens": s["lens_after"], "pool": s["pool_after"]}
    if op == "rope":
        turn = h.backward if case["inverse"] else h.forward
        turn(s["x"].data_ptr(), s["y"].data_ptr(), s["positions"].data_ptr(), case["tokens"], case["heads"])
        return s["y"]
    if op == "append":
        q, k, v = _split(s, case)
        h.run(q.data_ptr(), k.data_ptr(), v.data_ptr(), s["q_out"].data_ptr(), s["k_cache"].data_ptr(),
              s["v_cache"].data_ptr(), s["positions"].data_ptr(), s["slots"].data_ptr(), case["tokens"])
        return {"q": s["q_out"], "k": s["k_cache"], "v": s["v_cache"]}
    h.run(s["q"].data_ptr(), s["k_cache"].data_ptr(), s["v_cache"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(),
          case["requests"], s["out"].data_ptr(), s["lse"].data_ptr())
    return {"out": s["out"], "lse": s["lse"]}


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    op = case["op"]
    if op == "assign":
        return _plain_assign(s, case)
    if op == "rope":
        cos, sin = _cos_sin(s, case)
        return _rotate(s["x"], cos, sin, case, case["inverse"]).to(s["x"].dtype)
    return _plain_append(s, case) if op == "append" else _plain_attn(s, case)


# ------------------------------------------------------------------ in 64 bits, from the definitions

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "assign":
        return _exact_assign(s, case)
    if op == "rope":
        return _exact_turn(s["x"], s, case, -1.0 if case["inverse"] else 1.0)
    if op == "append":
        hq, hkv, d, t = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
        x = s["qkv"].reshape(t, hq + 2 * hkv, d)
        got = {"q": _exact_turn(x[:, :hq], s, case, 1.0)}
        for name, y in (("k", _exact_turn(x[:, hq:hq + hkv], s, case, 1.0)), ("v", x[:, hq + hkv:].double())):
            if s[name + "_scale"] is not None:  # the value that a code stands for, unrounded
                top = FP8_MAX[case["cache"]]
                y = (y / s[name + "_scale"].double().view(1, -1, 1)).clamp(-top, top)
            pages = s[name + "_cache"].shape[0]
            flat = torch.zeros(pages * case["page"], hkv, d, dtype=torch.float64, device="cuda")
            flat[s["slots"]] = y
            flat = flat.view(pages, case["page"], hkv, d)
            got[name] = flat.transpose(1, 2).contiguous() if case["order"] == "HND" else flat
        return got
    return _exact_attn(s, case)


def _exact_turn(x, s, case, sign):
    """Each pair as a complex number, multiplied by m * exp(i * position * frequency)."""
    x, rot = x.double(), case["rot"]
    angle = sign * s["positions"].double()[:, None] * s["frequencies"].double()[None]
    factor = torch.polar(torch.full_like(angle, _magnitude(case)), angle)[:, None]
    if case["layout"] == "half":
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * factor
        turned = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous()) * factor
        turned = torch.view_as_real(z).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _exact_attn(s, case):
    hq, hkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = hq // hkv
    out = torch.zeros(case["requests"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((case["requests"], hq), -math.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n <= first:
            continue
        at = torch.arange(first, n, device="cuda")
        pages = s["table"][r].long()[at // page]
        kv = []
        for name in ("k", "v"):
            cache = s[name + "_cache"]
            bits = cache.view(torch.uint8) if cache.element_size() == 1 else cache
            rows = bits[pages, :, at % page] if case["order"] == "HND" else bits[pages, at % page]
            rows = (rows.view(cache.dtype) if cache.element_size() == 1 else rows).double()
            if s[name + "_scale"] is not None:
                rows = rows * s[name + "_scale"].double()[None, :, None]
            kv.append(rows.repeat_interleave(group, 1))
        score = torch.einsum("hd,nhd->hn", s["q"][r].double(), kv[0]) / math.sqrt(d)
        if case["softcap"]:
            score = case["softcap"] * torch.tanh(score / case["softcap"])
        if s["slopes"] is not None:
            score = score - s["slopes"].double()[:, None] * (n - 1 - at).double()[None]
        lse[r] = torch.logsumexp(score, 1)
        out[r] = torch.einsum("hn,nhd->hd", torch.exp(score - lse[r][:, None]), kv[1])
    return {"out": out, "lse": lse}


def _exact_assign(s, case):
    page, lens, new = case["page"], s["lens"].tolist(), s["new"].tolist()
    table, free = s["table"].cpu().numpy().copy(), s["free"].tolist()
    head, count = s["pool"].tolist()
    slots, positions, owner, starts, after = [], [], [], [0], []
    wanted = taken = refused = 0
    for r, (n, m) in enumerate(zip(lens, new)):
        held, need = -(-n // page), -(-(n + m) // page) - -(-n // page)
        fits = need == 0 or wanted + need <= count
        if fits:
            for j in range(need):
                table[r, held + j] = free[head + wanted + j]
            taken = wanted + need if need else taken
        else:
            refused += 1
        wanted += need
        for p in range(n, n + m):
            positions.append(p)
            owner.append(r)
            slots.append(int(table[r, p // page]) * page + p % page if fits else -1)
        starts.append(starts[-1] + m)
        after.append(n + m if fits else n)
    i32 = np.int32
    return {"table": table, "slots": np.array(slots, np.int64), "positions": np.array(positions, i32),
            "owner": np.array(owner, i32), "starts": np.array(starts, i32), "lens": np.array(after, i32),
            "pool": np.array([head + taken, count - taken, starts[-1], refused], i32)}
