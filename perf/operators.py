"""The operators of the serving step over a paged key-value cache (emmy_ptx.paged), as cases that can be measured.

``assign``  page tables and slot maps of a step, from the requests' lengths
``store``   norm of each query and key head and the position rotation; keys and values go into their pages
``attend``  attention of one new token of each request over its pages

``run`` computes a case in plain torch operations where ``own`` is false and calls the framework's operators where it is
true. Both sides get what ``prepare`` made and return whole outputs: tables, caches and queries among them.
"""

import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f16": 2, "bf16": 2, "e4m3": 1}
EPS = 1e-6


# ---------------------------------------------------------------- cases


def _assign(name, requests, cached, fresh, page, pad=0, short=False):
    """``cached``, ``fresh``: the longest of each; a request's own are drawn up to them (fresh = 1: one token each).
    ``short``: the pool has half of the pages that the step asks for, so the last requests are refused."""
    return dict(name=name, op="assign", requests=requests, cached=cached, fresh=fresh, page=page, pad=pad, short=short)


def _store(name, tokens, heads, kv_heads, dim, rot, dtype, cache, page, interleaved=False, norm=True, pad=0):
    return dict(name=name, op="store", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, dtype=dtype, cache=cache,
                page=page, interleaved=interleaved, norm=norm, pad=pad)


def _attend(name, requests, length, heads, kv_heads, dim, dtype, cache, page, window=0, ragged=True):
    """``length``: every request's, or where ``ragged`` the longest of them (the others are drawn up to it)."""
    return dict(name=name, op="attend", requests=requests, length=length, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                cache=cache, page=page, window=window, ragged=ragged)


def listed():
    return [
        # a few chats, one new token each
        _assign("assign_8_decode", 8, 4096, 1, 16),
        # new prompts only, large pages
        _assign("assign_64_prompts", 64, 0, 2048, 64),
        # a loaded server that takes prompt pieces beside its decodes, rows padded to a fixed count
        _assign("assign_1000_mixed", 1000, 8192, 512, 16, pad=77),
        # the same few chats
        _store("store_8_f16", 8, 32, 8, 128, 128, "f16", "f16", 16),
        # a full decode batch of a captured step: some rows are padding
        _store("store_256_bf16", 256, 32, 8, 128, 128, "bf16", "bf16", 16, pad=13),
        # an odd number of prompt rows, 64-wide heads, half of them rotated in neighbouring pairs, an 8-bit cache
        _store("store_1001_e4m3", 1001, 12, 4, 64, 32, "bf16", "e4m3", 32, interleaved=True),
        # the benchmark's 16384 token rows as one prompt batch
        _store("store_16384_bf16", 16384, 32, 8, 128, 128, "bf16", "bf16", 64),
        # one short chat: latency
        _attend("attend_1x113", 1, 113, 32, 8, 128, "f16", "f16", 16, ragged=False),
        # the benchmark's attention (8 x 32 heads x 4096 x 128), its next token; every head has keys of its own
        _attend("attend_8x4096_mha", 8, 4096, 32, 32, 128, "f16", "f16", 64, ragged=False),
        # a server's ragged batch, four query heads share a key head
        _attend("attend_64_ragged", 64, 8192, 32, 8, 128, "bf16", "bf16", 16),
        # one long document: nothing to spread but the cache's length
        _attend("attend_1x131072", 1, 131072, 32, 8, 128, "bf16", "bf16", 64, ragged=False),
        # 64-wide heads in groups of eight over an 8-bit cache, only the last 2000 tokens seen
        _attend("attend_128_e4m3", 128, 8000, 64, 8, 64, "bf16", "e4m3", 48, window=2000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("assign", "store", "store", "attend", "attend", "attend"))
    page = rng.choice((1, 8, 16, 16, 32, 48, 64, 128))
    if op == "assign":
        c = _assign("", _log(rng, 1, 1000), rng.choice((0, _log(rng, 1, 8192))), rng.choice((1, _log(rng, 2, 512))), max(page, 8), pad=rng.choice((0, rng.randint(1, 100))),
                    short=rng.random() < 0.25)
    else:
        dtype = rng.choice(("f16", "bf16"))
        cache = rng.choice((dtype, dtype, "e4m3"))
        dim = rng.choice((64, 128, 128, 256))
        kv_heads = rng.choice((1, 2, 4, 5, 8, 16))
        group = rng.choice((1, 2, 3, 4, 6, 8, 8, 16, 32))
        if kv_heads * group > 128:
            group = 8
        heads = kv_heads * group
        if op == "store":
            most = max(16, int(4e8 / ((heads + 2 * kv_heads) * dim * 2)))
            rot = rng.choice((0, dim // 2, dim, dim))
            c = _store("", _log(rng, 1, min(16384, most)), heads, kv_heads, dim, rot, dtype, cache, page, rng.random() < 0.4, rng.random() < 0.7, pad=rng.choice((0, 3)))
        else:
            requests = _log(rng, 1, 256)
            most = max(64, int(9e8 / (requests * 2 * kv_heads * dim * SIZE[dtype])))
            length = _log(rng, 1, min(131072, most))
            c = _attend("", requests, length, heads, kv_heads, dim, dtype, cache, page, window=rng.choice((0, 0, 0, rng.randint(1, length))), ragged=rng.random() < 0.7)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs


def _lengths(case):
    """The requests' lengths, from the case alone: what the work is does not change with the seed."""
    g = torch.Generator().manual_seed(case["requests"] * 1000003 + case["page"])
    n = case["requests"]
    if case["op"] == "assign":
        cached = torch.randint(0, case["cached"] + 1, (n,), generator=g)
        fresh = torch.randint(1, case["fresh"] + 1, (n,), generator=g)
        if case["fresh"] > 1 and case["cached"]:  # beside the prompt pieces most requests get one token
            fresh[torch.rand(n, generator=g) < 0.7] = 1
        return cached, fresh
    lengths = torch.randint(1, case["length"] + 1, (n,), generator=g) if case["ragged"] else torch.full((n,), case["length"])
    if case["ragged"]:
        lengths[0] = case["length"]
        if n > 4:
            lengths[-1] = 0  # a padded row of a captured batch
    return lengths, None


def _normal(shape, dtype, gen, scale=1.0):
    x = torch.randn(shape, dtype=torch.float16 if dtype is torch.float8_e4m3fn else dtype, device="cuda", generator=gen)
    return x.mul_(scale).to(dtype) if scale != 1.0 or dtype is torch.float8_e4m3fn else x


def _i32(x):
    return x.to(torch.int32).cuda()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    page = case["page"]
    if case["op"] == "assign":
        cached, fresh = _lengths(case)
        have, want = -(-cached // page), -(-(cached + fresh) // page)
        width = int(want.max()) + 2
        used, taken = int(have.sum()), int((want - have).sum())
        free = 3 + taken // 2 if case["short"] else taken + 64
        pages = torch.randperm(used + free, device="cuda", generator=gen).to(torch.int32)
        table = torch.full((case["requests"], width), -1, dtype=torch.int32, device="cuda")
        filled = torch.arange(width, device="cuda")[None, :] < have.cuda()[:, None]
        table[filled] = pages[:used]
        tokens = int(fresh.sum()) + case["pad"]
        empty = lambda *n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
        s |= dict(cached_lengths=_i32(cached), fresh_lengths=_i32(fresh), table=table, free=pages[used:].contiguous(),
                  head=torch.full((1,), 3, dtype=torch.int32, device="cuda"), tokens=tokens,
                  out=(empty(tokens), empty(tokens), empty(case["requests"] + 1), empty(case["requests"]), empty(1), empty(4)))
        return s
    dtype, cache = TYPES[case["dtype"]], TYPES[case["cache"]]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    s["k_scale"], s["v_scale"] = (0.0625, 0.03125) if case["cache"] == "e4m3" else (1.0, 1.0)
    if case["op"] == "store":
        rows = case["tokens"] + case["pad"]
        count = -(-case["tokens"] // page) + 5  # the last page is nobody's
        qkv = _normal((rows, heads + 2 * kv_heads, dim), dtype, gen, 2.0)  # one projection's output: q, k and v are views of it
        s["q"], s["k"], s["v"] = qkv.split((heads, kv_heads, kv_heads), dim=1)
        s["k_pages"], s["v_pages"] = (_normal((count, page, kv_heads, dim), cache, gen) for _ in range(2))
        slots = torch.randperm((count - 1) * page, device="cuda", generator=gen)[:rows].to(torch.int32)
        positions = torch.randint(0, 8192, (rows,), device="cuda", generator=gen).to(torch.int32)
        if case["pad"]:
            slots[case["tokens"]:] = -1
            positions[case["tokens"]:] = 0
        s["slots"], s["positions"] = slots, positions
        s["rope"] = None
        if case["rot"]:
            angle = torch.arange(8192, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
            s["rope"] = torch.cat((angle.cos(), angle.sin()), 1).float()
        s["q_weight"], s["k_weight"] = ((1 + _normal((dim,), dtype, gen, 0.1) if case["norm"] else None) for _ in range(2))
        return s
    lengths, _ = _lengths(case)
    used = -(-lengths // page)
    width, total = max(1, int(used.max())), int(used.sum())
    s["k_pages"], s["v_pages"] = (_normal((total + 7, page, kv_heads, dim), cache, gen, 16.0 if case["cache"] == "e4m3" else 1.0) for _ in range(2))
    table = torch.full((case["requests"], width), -1, dtype=torch.int32, device="cuda")
    filled = torch.arange(width, device="cuda")[None, :] < used.cuda()[:, None]
    table[filled] = torch.randperm(total + 7, device="cuda", generator=gen)[:total].to(torch.int32)
    s |= dict(q=_normal((case["requests"], heads, dim), dtype, gen, 2.0), table=table, lengths=_i32(lengths), scale=1.0 / math.sqrt(dim))
    return s


# ---------------------------------------------------------------- the framework's operators


def _paged():
    root = str(Path.cwd() / "emmy-ptx-compiler_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from emmy_ptx import paged
    return paged


def _own(s):
    paged = _paged()
    if s["op"] == "assign":
        a = paged.assign(s["cached_lengths"], s["fresh_lengths"], s["table"], s["free"], s["head"], s["page"], s["tokens"], out=s["out"])
        return (s["table"], *a)
    if s["op"] == "store":
        q = paged.store(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"], s["positions"], rope=s["rope"], q_weight=s["q_weight"],
                        k_weight=s["k_weight"], eps=EPS, interleaved=s["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return q, s["k_pages"], s["v_pages"]
    return paged.attend(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], scale=s["scale"], window=s["window"],
                        k_scale=s["k_scale"], v_scale=s["v_scale"])


# ---------------------------------------------------------------- the plain form


def _plain_assign(s):
    cached, fresh, table, page = s["cached_lengths"], s["fresh_lengths"], s["table"], s["page"]
    requests, width = table.shape
    have, want = (cached + page - 1) // page, (cached + fresh + page - 1) // page
    fits = cached + fresh <= width * page
    need = torch.where(fits, want - have, 0)
    upto = need.cumsum(0)
    granted = fits & ((need == 0) | (upto <= s["free"].numel() - s["head"]))
    first = s["head"] + upto - need
    column = torch.arange(width, device=table.device)[None, :]
    at = (first[:, None] + column - have[:, None]).clamp(0, s["free"].numel() - 1)
    mine = granted[:, None] & (column >= have[:, None]) & (column < want[:, None])
    table.copy_(torch.where(mine, s["free"][at], table))
    ends = fresh.cumsum(0)
    starts = torch.cat((torch.zeros_like(ends[:1]), ends)).to(torch.int32)
    row = torch.arange(s["tokens"], device=table.device)
    owner = torch.searchsorted(ends, row, right=True)
    inside = owner < requests
    owner = owner.clamp(max=requests - 1)
    position = cached[owner] + row - starts[owner]
    slot = table[owner, (position // page).clamp(max=width - 1)] * page + position % page
    slots = torch.where(inside & granted[owner], slot, -1).to(torch.int32)
    positions = torch.where(inside, position, 0).to(torch.int32)
    lengths = torch.where(granted, cached + fresh, cached)
    taken = torch.where(granted, need, 0).sum()
    report = torch.stack((taken, (~granted).sum(), (ends[-1] - s["tokens"]).clamp(min=0), ends[-1])).to(torch.int32)
    return table, slots, positions, starts, lengths, (s["head"] + taken).to(torch.int32), report


def _normed(x, weight):
    x = x.float()
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _rotated(x, s):
    if s["rope"] is None:
        return x
    half = s["rot"] // 2
    row = s["rope"][s["positions"]]
    c, d = row[:, None, :half], row[:, None, half:]
    if s["interleaved"]:
        a, b = x[..., 0:s["rot"]:2], x[..., 1:s["rot"]:2]
        turned = torch.stack((a * c - b * d, b * c + a * d), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:s["rot"]]
        turned = torch.cat((a * c - b * d, b * c + a * d), -1)
    return torch.cat((turned, x[..., s["rot"]:]), -1)


def _raw(pages):
    """Pages as rows, one per slot, in a type that indexing takes."""
    rows = pages.view(-1, *pages.shape[2:])
    return rows.view(torch.uint8) if rows.dtype is torch.float8_e4m3fn else rows


def _plain_store(s):
    q = _rotated(_normed(s["q"], s["q_weight"]), s).to(s["q"].dtype)
    keep = (s["slots"] >= 0)[:, None, None]
    spare = s["k_pages"].shape[0] * s["page"] - 1
    at = torch.where(s["slots"] >= 0, s["slots"], spare).long()
    for x, pages, scale in ((_rotated(_normed(s["k"], s["k_weight"]), s), s["k_pages"], s["k_scale"]), (s["v"].float(), s["v_pages"], s["v_scale"])):
        if pages.dtype is torch.float8_e4m3fn:
            code = (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        else:
            code = x.to(pages.dtype)
        rows = _raw(pages)
        rows.index_put_((at,), torch.where(keep, code, rows[-1:]))  # a padded row rewrites the spare slot with what it holds
    return q, s["k_pages"], s["v_pages"]


def _plain_attend(s):
    requests, heads, dim = s["q"].shape
    kv_heads, page = s["kv_heads"], s["page"]
    longest = s["table"].shape[1] * page
    token = torch.arange(longest, device="cuda")
    at = s["table"][:, token // page].clamp(min=0) * page + token % page
    seen = token[None, :] < s["lengths"][:, None]
    if s["window"]:
        seen = seen & (token[None, :] >= s["lengths"][:, None] - s["window"])

    def gathered(pages, scale):
        x = _raw(pages)[at]
        x = x.view(torch.float8_e4m3fn) if x.dtype is torch.uint8 else x
        return (x.float() * scale).masked_fill_(~seen[:, :, None, None], 0.0)  # [requests, token, key head, dim]

    q = s["q"].float().view(requests, kv_heads, heads // kv_heads, dim)
    score = torch.matmul(q, gathered(s["k_pages"], s["k_scale"]).permute(0, 2, 3, 1)) * s["scale"]
    score = score.masked_fill(~seen[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, gathered(s["v_pages"], s["v_scale"]).permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    return out.reshape(requests, heads, dim).to(s["q"].dtype)


def run(state):
    if own:
        return _own(state)
    return {"assign": _plain_assign, "store": _plain_store, "attend": _plain_attend}[state["op"]](state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "assign":
        cached, fresh = _lengths(case)
        page = case["page"]
        taken = int((-(-(cached + fresh) // page) + (-cached // page)).sum())
        tokens = int(fresh.sum()) + case["pad"]
        return {"bytes": 4 * (4 * case["requests"] + 2 * taken + 2 * tokens), "flops": 0}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    elem, held = SIZE[case["dtype"]], SIZE[case["cache"]]
    if case["op"] == "store":
        rows = case["tokens"] + case["pad"]
        table = min(rows, 8192) * case["rot"] * 4
        moved = rows * dim * elem * 2 * heads + case["tokens"] * dim * 2 * kv_heads * (elem + held)
        return {"bytes": moved + table + rows * 8, "flops": rows * (heads + kv_heads) * (4 * dim + 3 * case["rot"])}
    lengths, _ = _lengths(case)
    if case["window"]:
        lengths = lengths.clamp(max=case["window"])
    keys = int(lengths.sum())
    pages = int((-(-lengths // case["page"])).sum())
    return {"bytes": 2 * keys * kv_heads * dim * held + 4 * pages + 4 * case["requests"] + 2 * case["requests"] * heads * dim * elem,
            "flops": 4 * keys * heads * dim}


# ---------------------------------------------------------------- in 64 bits, from the definitions


def exact(case, seed):
    if case["op"] == "assign":
        return None  # whole numbers only
    s = prepare(case, seed)
    if case["op"] == "store":
        return _exact_store(s)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = s["heads"] // s["kv_heads"]
    for b, n in enumerate(s["lengths"].tolist()):
        lo = max(0, n - s["window"]) if s["window"] else 0
        if n == lo:
            continue
        ids = s["table"][b, lo // s["page"]:-(-n // s["page"])].long()
        skip = lo - lo // s["page"] * s["page"]
        k, v = (p.view(torch.uint8)[ids].view(p.dtype).double().flatten(0, 1)[skip:skip + n - lo] * f
                for p, f in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
        for h in range(s["heads"]):
            p = torch.softmax(k[:, h // group] @ s["q"][b, h].double() * s["scale"], 0)
            out[b, h] = p @ v[:, h // group]
    return out


def _exact_store(s):
    def turned(x, weight):
        y = x.double()
        if weight is not None:
            y = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * weight.double()
        if s["rope"] is not None:
            n = s["rot"] // 2
            i = torch.arange(n, device="cuda")
            first, second = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + n)
            z = torch.complex(y[..., first], y[..., second])
            row = s["rope"].double()[s["positions"].long()]
            z = z * torch.complex(row[:, :n], row[:, n:])[:, None, :]
            y = y.clone()
            y[..., first], y[..., second] = z.real, z.imag
        return y

    outs = [turned(s["q"], s["q_weight"])]
    keep = s["slots"] >= 0
    at = s["slots"][keep].long()
    for pages, new, scale in ((s["k_pages"], turned(s["k"], s["k_weight"]), s["k_scale"]), (s["v_pages"], s["v"].double(), s["v_scale"])):
        whole = pages.double()
        whole[at // s["page"], at % s["page"]] = new[keep] / scale
        outs.append(whole)
    return tuple(outs)
