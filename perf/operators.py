"""The paged cache's operators as a serving program calls them, and what they compute in elementary torch operations.

A case is a dict of plain values.  ``op`` names the call:

    slots      blockPagedSlots: pages and slots for the new tokens of every request, from lengths on the GPU
    append     blockPagedAppend: keys and values of new tokens, token-major, into their slots
    attention  blockPagedAttention: one new token per request over its cached keys and values

``requests``/``dist``/``lo``/``hi`` say how long the requests are (drawn from ``sizes``, so a case always has the same
lengths; ``lo`` 0 leaves some empty), ``new`` how many tokens each one adds, ``page`` the tokens of a page, ``kv_heads``,
``group`` (query heads to a key head) and ``d`` the heads, ``dtype`` the type of queries, keys and values, ``layout`` whether
a page holds its tokens head by head (``heads``: pages, heads, page, d) or token by token (``tokens``: pages, page, heads, d,
which the operators get as the transposed view), ``dropped`` how many leading pages of each request are no longer held (a
sliding window), ``lse`` whether the row logarithms are wanted.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def _attention(name, requests, dist, lo, hi, kv_heads, group, d, page, dtype, layout="heads", dropped=0, lse=False, sizes=0):
    return {"name": name, "op": "attention", "requests": requests, "dist": dist, "lo": lo, "hi": hi, "kv_heads": kv_heads,
            "group": group, "d": d, "page": page, "dtype": dtype, "layout": layout, "dropped": dropped, "lse": lse, "sizes": sizes}


def _append(name, requests, dist, lo, hi, new, kv_heads, d, page, dtype, layout="heads", sizes=0):
    return {"name": name, "op": "append", "requests": requests, "dist": dist, "lo": lo, "hi": hi, "new": new, "kv_heads": kv_heads,
            "d": d, "page": page, "dtype": dtype, "layout": layout, "sizes": sizes}


def _slots(name, requests, dist, lo, hi, new, page, sizes=0):
    return {"name": name, "op": "slots", "requests": requests, "dist": dist, "lo": lo, "hi": hi, "new": new, "page": page, "sizes": sizes}


def listed():
    return [
        # one chat: a single request of a thousand tokens, all latency
        _attention("one_request", 1, "fixed", 1000, 1000, 8, 4, 128, 16, "bf16"),
        # a server's ordinary step: a few dozen requests of unlike lengths, token-major pages
        _attention("ordinary_batch", 32, "log", 16, 4096, 8, 4, 128, 16, "bf16", "tokens"),
        # many short answers over molecular graphs: the heads of the fp16 workloads, some requests empty, logarithms kept
        _attention("short_requests", 512, "uniform", 0, 300, 8, 1, 64, 16, "fp16", lse=True),
        # a full server: long documents
        _attention("long_batch", 64, "uniform", 1000, 32000, 8, 8, 128, 64, "bf16"),
        # one very long document, its length no multiple of anything
        _attention("one_long", 1, "fixed", 999983, 999983, 8, 5, 128, 64, "bf16", "tokens"),
        # one key head under many query heads, pages of an odd size, the beginning of every request let go
        _attention("shared_key_head", 12, "log", 700, 20000, 1, 24, 64, 24, "bf16", dropped=3, lse=True),
        # parity runs in 32 bits, head dimension no power of two
        _attention("fp32_batch", 16, "uniform", 1, 2000, 4, 2, 80, 32, "fp32", lse=True),
        # the keys and values of a step's new tokens
        _append("append_step", 64, "uniform", 1, 1000, 1, 8, 128, 16, "bf16"),
        # those of packed prompts, as attention's token-major inputs hold them
        _append("append_prompts", 64, "fixed", 0, 0, 2500, 16, 128, 16, "bf16", "tokens"),
        # 32-bit rows of an odd number of heads behind what is there already
        _append("append_fp32", 40, "uniform", 0, 500, 300, 5, 72, 24, "fp32"),
        # pages and slots of a step
        _slots("slots_step", 64, "uniform", 1, 4000, 1, 16),
        # and of packed prompts
        _slots("slots_prompts", 600, "uniform", 0, 700, 2000, 16),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(("attention",) * 4 + ("append", "append", "slots"))
    page = rng.choice((1, 8, 16, 16, 24, 32, 64, 100, 128, 256))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp16", "fp32"))
    layout = rng.choice(("heads", "tokens"))
    d = rng.choice((64, 64, 128, 128, 128, 32, 72, 80, 96, 192, 256))
    kv_heads = rng.choice((1, 2, 3, 4, 8, 8, 16))
    dist = rng.choice(("uniform", "log", "fixed"))
    sizes = rng.randrange(1 << 20)
    if op == "slots":
        requests = _log(rng, 1, 4096)
        new = _log(rng, 1, max(1, 600000 // requests))
        hi = _log(rng, 1, max(1, min(30000, 4000000 // requests)))
        return _slots("", requests, dist, 0, hi, new, page, sizes)
    if op == "append":
        requests = _log(rng, 1, 1024)
        row = 2 * kv_heads * d * _BYTES[dtype]
        new = _log(rng, 1, max(1, min(8000, (1 << 30) // (row * requests))))
        hi = _log(rng, 1, max(1, min(4000, (1 << 29) // (row * requests))))
        return _append("", requests, dist, 0, hi, new, kv_heads, d, page, dtype, layout, sizes)
    requests = _log(rng, 1, 512)
    group = rng.choice((1, 1, 2, 3, 4, 4, 6, 8, 8, 12, 16, 32))
    row = 2 * kv_heads * d * _BYTES[dtype]
    most = max(1, min(400000, (1 << 31) // (row * requests)))
    hi = _log(rng, min(4, most), most)
    lo = rng.choice((0, 1, 1 + hi // 2)) if dist == "uniform" else 1 if dist == "log" else hi
    return _attention("", requests, dist, min(lo, hi), hi, kv_heads, group, d, page, dtype, layout, rng.choice((0, 0, 0, 2)),
                      rng.choice((False, True)), sizes)


def _lengths(case):
    """Tokens that every request holds, as the host's numbers (the operators read them on the GPU)."""
    rs = np.random.RandomState(case["sizes"])
    n, lo, hi = case["requests"], case["lo"], case["hi"]
    if case["dist"] == "fixed":
        return np.full(n, hi, np.int64)
    if case["dist"] == "log":
        lo = max(lo, 1)
        return np.clip(np.rint(np.exp(rs.uniform(math.log(lo), math.log(max(lo, hi)), n))), lo, hi).astype(np.int64)
    return rs.randint(lo, hi + 1, n).astype(np.int64)


def _new(case):
    """New tokens of every request: one each in a step, up to twice ``new`` less one for prompts."""
    if case["new"] == 1:
        return np.ones(case["requests"], np.int64)
    return np.random.RandomState(case["sizes"] + 1).randint(1, 2 * case["new"], case["requests"]).astype(np.int64)


def _table(case, lengths, columns, g):
    """Pages of every request in an order that many requests coming and going leave behind; the pages in use."""
    held = -(-lengths // case["page"])
    total = int(held.sum())
    spare = 7
    order = torch.randperm(total + spare, generator=g, device="cuda").to(torch.int32)
    first = torch.as_tensor(np.concatenate([[0], np.cumsum(held)[:-1]])).cuda()
    at = torch.arange(columns, device="cuda")[None, :]
    have = at < torch.as_tensor(held).cuda()[:, None]
    table = torch.where(have, order[(first[:, None] + at).clamp(max=total + spare - 1)], -1)
    return table.to(torch.int32).contiguous(), total + spare


def _cache(case, pages, g, filled):
    shape = (pages, case["kv_heads"], case["page"], case["d"])
    if case["layout"] == "tokens":
        shape = (pages, case["page"], case["kv_heads"], case["d"])
    if filled:
        c = torch.randn(shape, generator=g, device="cuda", dtype=_DTYPES[case["dtype"]])
    else:
        c = torch.zeros(shape, device="cuda", dtype=_DTYPES[case["dtype"]])
    return c.transpose(1, 2) if case["layout"] == "tokens" else c


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    lengths, page = _lengths(case), case["page"]
    on_gpu = lambda x: torch.as_tensor(x.astype(np.int32)).cuda()  # noqa: E731
    if case["op"] == "attention":
        columns = max(1, -(-int(lengths.max()) // page))
        table, pages = _table(case, lengths, columns, g)
        table[:, : case["dropped"]] = -1
        q = torch.randn((case["requests"], case["kv_heads"] * case["group"], case["d"]), generator=g, device="cuda")
        return {"case": case, "q": q.to(_DTYPES[case["dtype"]]), "k": _cache(case, pages, g, True), "v": _cache(case, pages, g, True),
                "table": table, "lengths": on_gpu(lengths), "scale": case["d"] ** -0.5}
    new = _new(case)
    columns = -(-int((lengths + new).max()) // page)
    if case["op"] == "slots":
        table, _ = _table(case, lengths, columns, g)
        need = int((-(-(lengths + new) // page) + -lengths // page).sum())
        free = torch.randperm(2 * need + 50, generator=g, device="cuda").to(torch.int32)
        # some pages of the list are gone already, and a batch is padded to a few more tokens than it has
        return {"case": case, "table": table, "free": free, "taken": torch.tensor([5], dtype=torch.int32, device="cuda"),
                "lengths": on_gpu(lengths), "new": on_gpu(new), "tokens": int(new.sum()) + 3}
    table, pages = _table(case, lengths + new, columns, g)
    request = np.repeat(np.arange(len(new)), new)
    place = np.arange(len(request)) - np.repeat(np.cumsum(new) - new, new) + lengths[request]
    place = torch.as_tensor(place).cuda()
    slots = table[torch.as_tensor(request).cuda(), place // page].long() * page + place % page
    slots = torch.cat([slots, torch.full((3,), -1, device="cuda")])  # a padded batch
    shape = (slots.numel(), case["kv_heads"], case["d"])
    k, v = (torch.randn(shape, generator=g, device="cuda", dtype=_DTYPES[case["dtype"]]) for _ in range(2))
    return {"case": case, "new_k": k, "new_v": v, "k": _cache(case, pages, g, False), "v": _cache(case, pages, g, False), "slots": slots}


def run(state):
    case = state["case"]
    if own:
        import blockedattention_b200 as ba
        if case["op"] == "attention":
            return ba.blockPagedAttention(state["q"], state["k"], state["v"], state["table"], state["lengths"], state["scale"],
                                          return_lse=case["lse"])
        if case["op"] == "append":
            ba.blockPagedAppend(state["new_k"], state["new_v"], state["k"], state["v"], state["slots"])
            return state["k"], state["v"]
        slots, lengths, taken = ba.blockPagedSlots(state["lengths"], state["new"], state["table"], state["free"], state["taken"],
                                                   case["page"], state["tokens"])
        return slots, lengths, taken, state["table"]
    return {"attention": _plain_attention, "append": _plain_append, "slots": _plain_slots}[case["op"]](state)


def _plain_attention(s):
    q, table, page = s["q"], s["table"], s["case"]["page"]
    B, heads, d = q.shape
    kv_heads = s["k"].shape[1]
    at = table.clamp(min=0).long()
    k, v = (c[at].transpose(1, 2).reshape(B, kv_heads, -1, d).float() for c in (s["k"], s["v"]))
    there = torch.arange(k.shape[2], device=q.device)[None, :] < s["lengths"][:, None]
    there = (there & (table >= 0).repeat_interleave(page, 1))[:, None, None, :]
    x = torch.matmul(q.float().reshape(B, kv_heads, heads // kv_heads, d), k.transpose(2, 3)) * s["scale"]
    x = x.masked_fill(~there, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top.clamp(min=torch.finfo(torch.float32).min))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total.clamp(min=torch.finfo(torch.float32).tiny)
    out = out.reshape(B, heads, d).to(q.dtype)
    if not s["case"]["lse"]:
        return out
    return out, (top + torch.log(total)).reshape(B, heads)


def _plain_append(s):
    page, slots = s["case"]["page"], s["slots"]
    real = slots >= 0
    some = real.long().argmax()  # what has no slot repeats a row that has one
    slots = torch.where(real, slots, slots[some])
    for x, c in ((s["new_k"], s["k"]), (s["new_v"], s["v"])):
        c[slots // page, :, slots % page] = torch.where(real[:, None, None], x, x[some])
    return s["k"], s["v"]


def _plain_slots(s):
    page, table, free, taken = s["case"]["page"], s["table"], s["free"], s["taken"]
    W, F = table.shape[1], free.numel()
    old, new = s["lengths"].long(), s["new"].long()
    a, b = ((n + page - 1).div(page, rounding_mode="floor").clamp(max=W) for n in (old, old + new))
    first = taken[0] + torch.cumsum(b - a, 0) - (b - a)
    column = torch.arange(W, device=table.device)[None, :]
    number = first[:, None] + column - a[:, None]
    page_of = torch.where(number < F, free[number.clamp(0, F - 1)], -1)
    table.copy_(torch.where((column >= a[:, None]) & (column < b[:, None]), page_of, table))
    ends = torch.cumsum(new, 0)
    t = torch.arange(s["tokens"], device=table.device)
    r = torch.searchsorted(ends, t, right=True)
    inside = r < old.numel()
    r = r.clamp(max=old.numel() - 1)
    place = old[r] + t - (ends - new)[r]
    column = place.div(page, rounding_mode="floor")
    found = torch.where(inside & (column < W), table[r, column.clamp(max=W - 1)].long(), -1)
    slots = torch.where(found >= 0, found * page + place % page, -1)
    return slots, (old + new).int(), (taken + (b - a).sum()).int(), table


def work(case):
    lengths, page = _lengths(case), case["page"]
    if case["op"] == "slots":
        new = _new(case)
        pages = int((-(-(lengths + new) // page) + -lengths // page).sum())
        return {"bytes": 12 * len(new) + 8 * int(new.sum()) + 8 * pages, "flops": 0}
    row = case["kv_heads"] * case["d"] * _BYTES[case["dtype"]]
    if case["op"] == "append":
        tokens = int(_new(case).sum())
        return {"bytes": tokens * (4 * row + 8), "flops": 0}
    gone = np.minimum(lengths, case["dropped"] * page)
    tokens, pages, heads = int((lengths - gone).sum()), int((-(-lengths // page)).sum()), case["kv_heads"] * case["group"]
    rows = case["requests"] * (2 * row * case["group"] + 4 + (4 * heads if case["lse"] else 0))
    return {"bytes": tokens * 2 * row + 4 * pages + rows, "flops": 4 * tokens * heads * case["d"]}


def exact(case, seed):
    """The operators' definitions request by request in 64 bits; nothing for whole numbers, which the plain form has exactly."""
    if case["op"] != "attention":
        return None
    s = prepare(case, seed)
    heads, group, d = case["kv_heads"] * case["group"], case["group"], case["d"]
    outs = torch.zeros((case["requests"], heads, d), dtype=torch.float64, device="cuda")
    logs = torch.full((case["requests"], heads), -math.inf, dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lengths(case).tolist()):
        place = torch.arange(case["dropped"] * case["page"], n, device="cuda") if n > case["dropped"] * case["page"] else None
        if place is None:
            continue
        pages, place = s["table"][r].long()[place // case["page"]], place % case["page"]
        for h in range(case["kv_heads"]):
            mine = slice(h * group, (h + 1) * group)
            x = s["q"][r, mine].double() @ s["k"][pages, h, place].double().T * s["scale"]
            outs[r, mine] = torch.softmax(x, -1) @ s["v"][pages, h, place].double()
            logs[r, mine] = torch.logsumexp(x, -1)
    return (outs, logs) if case["lse"] else outs
