"""The paged-cache operators on a GPU against their definitions in 64 bits.

Tolerances, from the arithmetic. A rounding to a type is off by at most u = eps / 2 of the value (half of the smallest
subnormal below the normal range).
``store``: y is rounded once, after f32 steps that are off by less than 2^-20 of |a c| + |b s| in all.
``attend``: with A = sum_j w_j |v_j| (w: the softmax weights) the rounding of the weights is off by u A at most (and, where a
weight is below f16's normal range, by 2^-25 of the largest weight: sum_j |v_j| 2^-25), the result's own rounding by u |out|.
A score is made of dim / 16 <= 16 tensor-core steps, each of which may cut off 2^-23 of what it adds up, at most
spread = max_j |q| . |k_j| scale: 2^-19 spread. Its scale times log2(e) is two f32 roundings, their product with the sum one
more, the constant and the product that lead back from log2 two more: 5 x 2^-24 spread. Together less than 2^-18 spread, by
which lse may be off besides its own f32 steps (2^-20, and 2^-23 of itself); a weight follows a score in numerator and
denominator: 2^-17 spread A. The f32 sums of n terms and the exponentials add (n 2^-24 + 2^-20) A.
"""

import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def paged():
    from emmy_ptx import paged
    return paged


def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def normal(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


# ---------------------------------------------------------------- assign


def assign_by_hand(cached, fresh, table, free, head, page, tokens):
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    slots, positions, starts, lengths = [-1] * tokens, [0] * tokens, [0], []
    taken = refused = 0
    ended = False
    for b, (c, f) in enumerate(zip(cached, fresh)):
        c, f = max(c, 0), max(f, 0)
        start, end = starts[-1], starts[-1] + f
        starts.append(end)
        have, want = -(-c // page), -(-(c + f) // page)
        ok = f == 0 or (c + f <= width * page and end <= tokens)
        if ok and want > have:
            ended = ended or taken + want - have > len(free) - head
            ok = not ended
            if ok:
                table[b][have:want] = free[head + taken:head + taken + want - have]
                taken += want - have
        refused += not ok
        lengths.append(c + f if ok else c)
        for i in range(start, min(end, tokens)):
            pos = c + i - start
            positions[i] = pos
            if ok and table[b][pos // page] >= 0:
                slots[i] = table[b][pos // page] * page + pos % page
    return table, slots, positions, starts, lengths, head + taken, [taken, refused, max(0, starts[-1] - tokens), starts[-1]]


def check_assign(paged, cached, fresh, width, free, head, page, tokens, seed=0):
    rng = random.Random(seed)
    table = [[rng.randrange(1000) if w * page < max(c, 0) else -1 for w in range(width)] for c in cached]
    want = assign_by_hand(cached, fresh, table, free, head, page, tokens)
    big = torch.full((len(cached), width + 3), -7, dtype=torch.int32, device="cuda")  # rows of a wider table
    on_gpu = big[:, :width]
    if cached:
        on_gpu.copy_(i32(table))
    got = paged.assign(i32(cached), i32(fresh), on_gpu, i32(free), i32([head]), page, tokens)
    assert on_gpu.tolist() == want[0] and bool((big[:, width:] == -7).all())
    for name, mine, his in zip(got._fields, got, want[1:]):
        his = his if isinstance(his, list) else [his]
        assert mine.tolist() == his, name


@pytest.mark.parametrize("page", [1, 3, 16, 64])
@pytest.mark.parametrize("requests, longest, most", [(1, 0, 1), (1, 100, 1), (8, 300, 1), (7, 0, 90), (33, 200, 40), (256, 50, 9), (257, 50, 9), (700, 60, 30)])
def test_assign(paged, page, requests, longest, most):
    rng = random.Random(requests * 100 + page)
    cached = [rng.randint(0, longest) for _ in range(requests)]
    fresh = [rng.choice((0, 1, 1, rng.randint(0, most))) for _ in range(requests)]
    width = max(-(-(c + f) // page) for c, f in zip(cached, fresh)) + 1
    free = rng.sample(range(5000, 5000 + 40 * requests * (most // page + 2)), requests * (most // page + 2) + 5)
    check_assign(paged, cached, fresh, width, free, 2, page, sum(fresh) + rng.choice((0, 5)), seed=page)


def test_assign_refuses_whole_requests(paged):
    """The free pages end in the middle; a table row is too short; the step has too few rows."""
    free = list(range(50, 58))
    check_assign(paged, [0, 30, 5, 0, 64], [40, 1, 33, 1, 0], 4, free, 0, 16, 80)   # 3 + 0 + 3 (ends at 8 with the next 1)
    check_assign(paged, [0, 30, 5, 0, 64], [40, 1, 33, 1, 0], 4, free[:5], 0, 16, 80)
    check_assign(paged, [0, 30, 5, 0, 64], [40, 1, 33, 1, 0], 4, free, 6, 16, 80)
    check_assign(paged, [10, 30, 5], [60, 1, 3], 4, free, 0, 16, 80)                # 70 tokens in a row of 64
    check_assign(paged, [10, 30, 5, 9], [20, 10, 3, 0], 4, free, 0, 16, 31)         # rows end inside the third request
    check_assign(paged, [10, 30], [20, 10], 4, [], 0, 16, 40)                       # no free page at all
    check_assign(paged, [-4, 3], [2, -9], 4, free, 0, 16, 4)                        # negative counts are 0
    check_assign(paged, [], [], 1, free, 0, 16, 3)
    check_assign(paged, [0, 0], [0, 0], 1, free, 0, 16, 0)


def test_assign_many_rows_and_one_long_prompt(paged):
    check_assign(paged, [0, 17], [5000, 1], 320, list(range(9000, 9400)), 0, 16, 5003)
    check_assign(paged, [0] * 1500, [3] * 1500, 2, list(range(3000)), 0, 4, 4500)


def test_assign_clamps_a_wild_free_head(paged):
    for head in (-5, 10 ** 9):
        table = i32([[-1, -1]])
        got = paged.assign(i32([0]), i32([1]), table, i32([4, 5]), i32([head]), 16, 1)
        assert got.slots.tolist() == ([64] if head < 0 else [-1])


# ---------------------------------------------------------------- store


def store_exact(x, weight, rope, positions, interleaved, eps):
    """(values, the sum of |terms| that each was made from) in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    terms = y.abs()
    if rope is not None:
        rot = rope.shape[1]
        half = rot // 2
        j = torch.arange(half, device="cuda")
        p, q = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
        c, s = (t[:, None, :] for t in rope.double()[positions.long()].split(half, 1))
        a, b = y[..., p], y[..., q]
        y, terms = y.clone(), terms.clone()
        y[..., p], y[..., q] = a * c - b * s, b * c + a * s
        terms[..., p], terms[..., q] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, terms


def rounding(y, dtype):
    """What a rounding of y to dtype may be off by."""
    info = torch.finfo(dtype)
    least = 2.0 ** -10 if dtype is E4M3 else info.smallest_normal * info.eps / 2
    return torch.maximum(y.abs() * (2.0 ** -4 if dtype is E4M3 else info.eps / 2), torch.tensor(least, device=y.device, dtype=y.dtype))


def check_rows(got, y, terms, dtype, scale=1.0):
    y, terms = y / scale, terms / scale
    if dtype is E4M3:
        y = y.clamp(-448, 448)
    off = (got.double() - y).abs() - rounding(y, dtype) - terms * 2.0 ** -20
    assert float(off.max()) <= 0, float(off.max())


def make_pages(layout, pages, size, heads, dim, dtype, gen, scale=1.0):
    if layout == "token":
        shape, order = (2, pages, size, heads, dim), (0, 1, 2, 3, 4)
    elif layout == "head":  # head-major pages
        shape, order = (2, pages, heads, size, dim), (0, 1, 3, 2, 4)
    else:                   # keys and values of a page side by side
        shape, order = (pages, 2, size, heads, dim), (1, 0, 2, 3, 4)
    both = normal(shape, torch.float32, gen, scale).to(dtype).permute(order)
    return both[0], both[1]


def raw(t):
    return t.view(torch.uint8) if t.dtype is E4M3 else t


def check_store(paged, tokens, heads, kv_heads, dim, rot, dtype, cache, layout="token", interleaved=False, norm=True, size=16, in_place=False, seed=1):
    gen = generator(seed)
    count = tokens // size + 3
    qkv = normal((tokens, heads + 2 * kv_heads, dim), dtype, gen, 2.0)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    k_pages, v_pages = make_pages(layout, count, size, kv_heads, dim, cache, gen)
    before = [raw(p).clone() for p in (k_pages, v_pages)]
    slots = torch.randperm(count * size, device="cuda", generator=gen)[:tokens].to(torch.int32)
    slots[::5] = -1
    if tokens > 6:
        slots[6] = count * size  # just outside
    positions = torch.randint(0, 500, (tokens,), device="cuda", generator=gen).to(torch.int32)
    rope = None
    if rot:
        angle = torch.arange(500, device="cuda", dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        rope = torch.cat((angle.cos(), angle.sin()), 1).float()
    wq, wk = (normal((dim,), dtype, gen) if norm else None for _ in range(2))
    scales = (0.013, 0.25) if cache is E4M3 else (1.0, 1.0)
    want_q = store_exact(q, wq, rope, positions, interleaved, 1e-5)
    want_k = store_exact(k, wk, rope, positions, interleaved, 1e-5)
    want_v = (v.double(), torch.zeros_like(v.double()))
    out = paged.store(q, k, v, k_pages, v_pages, slots, positions, rope=rope, q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved,
                      k_scale=scales[0], v_scale=scales[1], out=q if in_place else None)
    assert (out.data_ptr() == q.data_ptr()) == in_place
    check_rows(out, *want_q, dtype)
    kept = (slots >= 0) & (slots < count * size)
    at = slots[kept].long()
    untouched = torch.ones(count * size, dtype=torch.bool, device="cuda")
    untouched[at] = False
    for pages, old, (y, terms), scale in zip((k_pages, v_pages), before, (want_k, want_v), scales):
        if at.numel():
            check_rows(raw(pages)[at // size, at % size].view(cache), y[kept], terms[kept], cache, scale)
        flat = untouched.nonzero()[:, 0]
        assert torch.equal(raw(pages)[flat // size, flat % size], old[flat // size, flat % size])


@pytest.mark.parametrize("dtype, cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize("tokens, heads, kv_heads, dim, rot", [(1, 1, 1, 64, 64), (3, 4, 2, 128, 128), (37, 5, 5, 256, 128), (130, 6, 3, 64, 16), (77, 3, 1, 128, 96), (20, 7, 7, 64, 0), (2049, 8, 2, 128, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_store(paged, dtype, cache, tokens, heads, kv_heads, dim, rot, interleaved):
    check_store(paged, tokens, heads, kv_heads, dim, rot, dtype, cache, interleaved=interleaved)


@pytest.mark.parametrize("layout", ["head", "pairs"])
@pytest.mark.parametrize("size", [1, 7, 16])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_store_layouts(paged, layout, size, cache):
    check_store(paged, 45, 4, 2, 128, 64, BF16, cache, layout=layout, size=size)


def test_store_without_norm_and_in_place(paged):
    check_store(paged, 50, 4, 2, 64, 64, BF16, BF16, norm=False)
    check_store(paged, 50, 4, 2, 128, 0, F16, F16, norm=False)
    check_store(paged, 50, 4, 2, 128, 128, BF16, BF16, in_place=True)


def test_store_takes_queries_out_of_a_wider_buffer_and_puts_them_into_one(paged):
    gen = generator(9)
    wide = normal((40, 20, 128), F16, gen)
    q, k, v = wide[:, 2:10], wide[:, 11:13], wide[:, 17:19]
    k_pages, v_pages = make_pages("pairs", 4, 16, 2, 128, F16, gen)
    out = torch.full((40, 11, 128), 3.0, dtype=F16, device="cuda")
    slots = torch.arange(40, device="cuda", dtype=torch.int32)
    weight = normal((128,), F16, gen)
    got = paged.store(q, k, v, k_pages, v_pages, slots, slots, q_weight=weight, out=out[:, 1:9])
    assert got.data_ptr() == out[:, 1:9].data_ptr() and bool((out[:, 0] == 3).all()) and bool((out[:, 9:] == 3).all())
    check_rows(got, *store_exact(q, weight, None, slots, False, 1e-6), F16)
    at = slots.long()
    assert torch.equal(k_pages[at // 16, at % 16], k) and torch.equal(v_pages[at // 16, at % 16], v)


def test_store_extremes(paged):
    """A position outside the table shows as NaN in the rotated dims only; infinities saturate; no rows is no launch."""
    gen = generator(3)
    q, k, v = (normal((4, 2, 64), BF16, gen) for _ in range(3))
    v[1, 0, 5] = math.inf
    v[2, 1, 7] = math.nan
    k_pages, v_pages = (torch.zeros(2, 4, 2, 64, device="cuda").to(E4M3) for _ in range(2))
    rope = torch.ones(10, 32, device="cuda")
    out = paged.store(q, k, v, k_pages, v_pages, i32([0, 1, 2, 3]), i32([0, 9, 10, -1]), rope=rope)
    assert out[2:, :, :32].isnan().all() and not out[2:, :, 32:].isnan().any() and not out[:2].isnan().any()
    held = k_pages.view(8, 2, 64).float()
    assert held[2:4, :, :32].isnan().all() and not held[2:4, :, 32:].isnan().any() and not held[:2].isnan().any()
    held = v_pages.view(8, 2, 64).float()
    assert held[1, 0, 5] == 448 and held[2, 1, 7].isnan() and held.isnan().sum() == 1
    none = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    assert paged.store(none, none, none, k_pages, v_pages, i32([]), i32([]), rope=rope).shape == (0, 2, 64)


# ---------------------------------------------------------------- attend


def attend_exact(q, k_pages, v_pages, table, lengths, scale, window, k_scale, v_scale, w_type):
    """(out, lse, the tolerances of both) in 64 bits."""
    requests, heads, dim = q.shape
    size, kv_heads = k_pages.shape[1:3]
    out = torch.zeros(requests, heads, dim, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((requests, heads), -math.inf, dtype=torch.float64, device="cuda")
    lse_tol = torch.zeros_like(lse)
    u = torch.finfo(w_type).eps / 2
    for b, n in enumerate(lengths.tolist()):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        j = torch.arange(lo, n, device="cuda")
        at = table[b].long()[j // size]
        k, v = (raw(p)[at, j % size].view(p.dtype).double().repeat_interleave(heads // kv_heads, 1) * s for p, s in ((k_pages, k_scale), (v_pages, v_scale)))
        x = q[b].double()
        score = torch.einsum("hd,jhd->hj", x, k) * scale
        spread = torch.einsum("hd,jhd->hj", x.abs(), k.abs()).amax(1) * abs(scale)
        w = score.softmax(1)
        out[b] = torch.einsum("hj,jhd->hd", w, v)
        lse[b] = score.logsumexp(1)
        lse_tol[b] = spread * 2.0 ** -18 + 2.0 ** -20 + lse[b].abs() * 2.0 ** -23
        a = torch.einsum("hj,jhd->hd", w, v.abs())
        tol[b] = (u + (n - lo) * 2.0 ** -24 + 2.0 ** -20 + spread[:, None] * 2.0 ** -17) * a + rounding(out[b], q.dtype)
        if w_type is F16:
            tol[b] += v.abs().sum(0) * 2.0 ** -25 * w.amax(1)[:, None]
    return out, lse, tol, lse_tol


def make_attend(lengths, heads, kv_heads, dim, dtype, cache, size, layout="token", seed=5, spare=3, q_scale=2.0):
    gen = generator(seed)
    used = [-(-n // size) for n in lengths]
    width, total = max(1, max(used)), sum(used)
    k_scale, v_scale = (0.0625, 0.03125) if cache is E4M3 else (1.0, 1.0)
    k_pages, v_pages = make_pages(layout, total + spare, size, kv_heads, dim, cache, gen, 16.0 if cache is E4M3 else 1.0)
    ids = torch.randperm(total + spare, device="cuda", generator=gen)[:total].to(torch.int32)
    table = torch.full((len(lengths), width + 2), -1, dtype=torch.int32, device="cuda")[:, :width]
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    q = normal((len(lengths), heads, dim), dtype, gen, q_scale)
    return dict(q=q, k_pages=k_pages, v_pages=v_pages, table=table, lengths=i32(lengths), k_scale=k_scale, v_scale=v_scale)


def poison(s):
    """NaN into every slot that no request's length covers."""
    size = s["k_pages"].shape[1]
    free = torch.ones(s["k_pages"].shape[0] * size, dtype=torch.bool, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        j = torch.arange(n, device="cuda")
        free[s["table"][b].long()[j // size] * size + j % size] = False
    at = free.nonzero()[:, 0]
    for p in (s["k_pages"], s["v_pages"]):
        raw(p)[at // size, at % size] = 0x7F if p.dtype is E4M3 else math.nan


def check_attend(paged, s, window=0, scale=None, **kw):
    q = s["q"]
    scale_ = q.shape[2] ** -0.5 if scale is None else scale
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    got = paged.attend(**s, window=window, scale=scale, lse=lse, **kw)
    w_type = F16 if s["k_pages"].dtype is E4M3 else q.dtype
    out, want_lse, tol, lse_tol = attend_exact(q, s["k_pages"], s["v_pages"], s["table"], s["lengths"], scale_, window, s["k_scale"], s["v_scale"], w_type)
    off = (got.double() - out).abs()
    assert bool((off <= tol).all()), (float((off / tol.clamp(min=1e-300)).max()), (off > tol).nonzero()[:4].tolist())
    finite = want_lse.isfinite()
    assert torch.equal(finite, lse.isfinite())
    assert bool(((lse.double() - want_lse).abs() <= lse_tol)[finite].all())
    return got


SHAPES = [(1, 1, 64), (4, 4, 128), (8, 2, 128), (8, 1, 64), (14, 2, 128), (32, 2, 64), (33, 1, 128), (96, 2, 128), (6, 3, 256), (40, 1, 256)]


@pytest.mark.parametrize("dtype, cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize("heads, kv_heads, dim", SHAPES)
def test_attend(paged, dtype, cache, heads, kv_heads, dim):
    s = make_attend([1, 0, 15, 16, 17, 64, 65, 200, 0, 513, 129], heads, kv_heads, dim, dtype, cache, 16)
    poison(s)
    got = check_attend(paged, s)
    assert not got[1].any() and not got[8].any()


@pytest.mark.parametrize("size", [1, 3, 16, 48, 200])
@pytest.mark.parametrize("layout", ["token", "head", "pairs"])
@pytest.mark.parametrize("cache", [F16, E4M3])
def test_attend_pages(paged, size, layout, cache):
    s = make_attend([130, 1, 77, 400, 48, 49], 4, 2, 128, F16, cache, size, layout)
    poison(s)
    check_attend(paged, s)


@pytest.mark.parametrize("window", [1, 16, 48, 49, 50, 63, 64, 65, 113, 240, 241, 256, 257, 1000])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_window(paged, window, dim):
    check_attend(paged, make_attend([1, 64, 65, 500, 0, 1200, 2000], 8, 2, dim, BF16, BF16, 16), window=window)


@pytest.mark.parametrize("lengths, heads, kv_heads, dim, cache", [
    ([30000], 8, 2, 128, BF16), ([30000], 8, 8, 64, BF16), ([20000, 3], 4, 1, 128, E4M3), ([1] * 300, 8, 2, 128, BF16), ([9000, 0, 1, 4000, 70] * 9, 8, 4, 128, BF16),
    ([700] * 200, 4, 4, 64, E4M3), ([5000, 6000, 1], 64, 1, 256, BF16), (list(range(0, 1200, 7)), 16, 2, 64, BF16)])
def test_attend_long_many_and_ragged(paged, lengths, heads, kv_heads, dim, cache):
    s = make_attend(lengths, heads, kv_heads, dim, BF16, cache, 16)
    poison(s)
    check_attend(paged, s)


@pytest.mark.parametrize("lengths, heads, kv_heads, dim, dtype, cache", [
    ([6000, 0, 7, 5000] * 20, 4, 4, 64, F16, F16), ([9000, 0, 7, 5000, 8000] * 12, 32, 8, 128, BF16, BF16), ([6000, 100, 5000] * 25, 8, 2, 128, F16, F16),
    ([12000, 1, 9000] * 27, 24, 2, 128, BF16, BF16), ([9000, 0, 17, 12000] * 20, 16, 4, 64, BF16, E4M3), ([7000, 6000, 3] * 20, 4, 4, 128, F16, E4M3),
    ([12000, 3, 9000] * 30, 8, 4, 256, BF16, E4M3), ([5000, 3, 900] * 25, 4, 4, 256, BF16, BF16), ([20000, 11, 20000] * 20, 40, 2, 64, BF16, E4M3)])
@pytest.mark.parametrize("window", [0, 3000])
def test_attend_heads_side_by_side(paged, lengths, heads, kv_heads, dim, dtype, cache, window):
    """Batches that are large enough for a warp to have a head of its own."""
    s = make_attend(lengths, heads, kv_heads, dim, dtype, cache, 16)
    poison(s)
    check_attend(paged, s, window=window)


@pytest.mark.parametrize("size", [24, 7, 64])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attend_many_requests_side_by_side(paged, size, layout, cache):
    """More requests than a CTA has threads, pages of other sizes, head-major pages."""
    s = make_attend([2500, 300, 4000, 0] * 50, 8, 4, 64, BF16, cache, size, layout)
    poison(s)
    check_attend(paged, s)


def test_attend_is_the_same_again(paged):
    """The split and the join have one order: two calls agree bit for bit."""
    s = make_attend([5000, 17, 900, 12000], 8, 2, 128, BF16, BF16, 16)
    assert torch.equal(paged.attend(**s), paged.attend(**s))


def test_attend_scores_far_apart(paged):
    """One key far above the rest (weight 1), all keys equal, and scores of both signs beyond the exponential's range."""
    s = make_attend([300, 300, 300], 4, 2, 128, F16, F16, 16)
    s["q"][0] = s["k_pages"][s["table"][0, 9].long(), 5].repeat_interleave(2, 0) * 3
    s["q"][1] = 0
    check_attend(paged, s)
    check_attend(paged, s, scale=2.0)
    check_attend(paged, s, scale=-0.3)
    check_attend(paged, s, scale=0.0)


def test_attend_values_that_are_not_finite(paged):
    """An infinity or NaN at a key that is seen shows in its request and head and nowhere else."""
    s = make_attend([200, 200], 4, 2, 64, BF16, BF16, 16)
    clean = paged.attend(**s)
    page = s["table"][0, 3].long()
    s["k_pages"][page, 2, 0, 1] = math.nan
    s["v_pages"][page, 2, 1, 7] = math.inf
    got = paged.attend(**s)
    assert got[0, :2].isnan().all() and torch.equal(got[1], clean[1])
    assert got[0, 2:, 7].isinf().all()
    rest = [d for d in range(64) if d != 7]
    assert torch.equal(got[0, 2:][:, rest], clean[0, 2:][:, rest])


def test_attend_bad_pages_and_lengths_show(paged):
    """A table entry outside the cache, and a length beyond the table row, are NaN in their request; a negative length is 0."""
    s = make_attend([200, 200, 200, 200], 4, 2, 64, BF16, BF16, 16)
    clean = paged.attend(**s)
    for bad in (-1, -5, -2 ** 31):
        s["table"][0, 3] = bad
        assert paged.attend(**s)[0].isnan().all()
    s["table"][1, 12] = s["k_pages"].shape[0]
    s["lengths"][2] = 16 * s["table"].shape[1] + 1
    got = paged.attend(**s)
    assert got[:3].isnan().all() and torch.equal(got[3], clean[3])
    s["lengths"][2] = 2 ** 31 - 1
    assert paged.attend(**s)[2].isnan().all()
    s["lengths"][:3] = -1
    got = paged.attend(**s)
    assert not got[:3].any() and torch.equal(got[3], clean[3])
    s["lengths"].fill_(192)
    s["table"][:, 12] = 2 ** 31 - 1  # entries behind the length are not looked at
    s["table"][:2, 3] = 0
    assert paged.attend(**s).isfinite().all()


def test_attend_reads_strided_queries_and_broadcast_pages(paged):
    s = make_attend([100, 33], 4, 2, 128, F16, F16, 16)
    wide = torch.zeros(2, 12, 128, dtype=F16, device="cuda")
    wide[:, 4:8] = s["q"]
    s["q"] = wide[:, 4:8]
    out = torch.full((2, 6, 128), 7.0, dtype=F16, device="cuda")
    got = check_attend(paged, s, out=out[:, 1:5])
    assert got.data_ptr() == out[:, 1:5].data_ptr() and bool((out[:, 0] == 7).all()) and bool((out[:, 5] == 7).all())
    s["k_pages"] = s["k_pages"][:, :, :1].expand(-1, -1, 2, -1)  # both key heads read the same keys
    check_attend(paged, s)


def test_attend_offsets_beyond_32_bits(paged):
    """A page whose first element is more than 2^32 bytes, and more than 2^32 elements, into the buffer."""
    gen = generator(2)
    whole = torch.empty(5, 1 << 30, dtype=F16, device="cuda")
    pages = whole.as_strided((5, 16, 1, 64), (1 << 30, 64, 64, 1))
    k, v = normal((5, 16, 1, 64), F16, gen), normal((5, 16, 1, 64), F16, gen)
    pages.copy_(k)
    table, lengths, q = i32([[4, 0, 3]]), i32([41]), normal((1, 4, 64), F16, gen)
    assert torch.equal(paged.attend(q, pages, v, table, lengths), paged.attend(q, k, v, table, lengths))
    new = normal((3, 1, 64), F16, gen)
    slots = i32([4 * 16 + 15, 3, 64])
    paged.store(normal((3, 2, 64), F16, gen), new, new, pages, v, slots, i32([0, 0, 0]))
    assert torch.equal(pages.reshape(80, 64)[slots.long()], new[:, 0])


# ---------------------------------------------------------------- together


def run_steps(paged, prompts, steps, cache, streams=None, graph=False):
    """Prompts of several requests stored, then single-token steps; returns what the steps attended and all q, k, v."""
    heads, kv_heads, dim, page = 4, 2, 64, 16
    requests = len(prompts)
    gen = generator(11)
    width = -(-(max(prompts) + steps) // page)
    k_pages, v_pages = (torch.zeros(requests * width + 4, page, kv_heads, dim, device="cuda").to(cache) for _ in range(2))
    scale = 0.05 if cache is E4M3 else 1.0
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(requests * width + 4, device="cuda", generator=gen).to(torch.int32)
    angle = torch.arange(max(prompts) + steps, device="cuda")[:, None] * 50.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)
    rope = torch.cat((angle.cos(), angle.sin()), 1).float()
    weight = normal((dim,), BF16, gen)
    lengths, head = i32([0] * requests), i32([0])
    history = []

    def step(qkv, cached, fresh, free_head, out=None):
        a = paged.assign(cached, fresh, table, free, free_head, page, qkv.shape[0], out=out)
        q = paged.store(*qkv.split((heads, kv_heads, kv_heads), 1), k_pages, v_pages, a.slots, a.positions, rope=rope, q_weight=weight,
                        k_weight=weight, k_scale=scale, v_scale=scale)
        return a, q

    qkv = normal((sum(prompts) + 3, heads + 2 * kv_heads, dim), BF16, gen)  # three rows of padding
    a, _ = step(qkv, lengths, i32(prompts), head)
    assert a.report.tolist() == [sum(-(-p // page) for p in prompts), 0, 0, sum(prompts)]
    rows = [qkv[s:e] for s, e in zip(a.starts.tolist(), a.starts.tolist()[1:])]
    lengths, head = a.lengths, a.free_head
    ones = i32([1] * requests)
    for _ in range(steps):
        qkv = normal((requests, heads + 2 * kv_heads, dim), BF16, gen)
        a, q = step(qkv, lengths, ones, head)
        out = paged.attend(q, k_pages, v_pages, table, a.lengths, k_scale=scale, v_scale=scale)
        lengths, head = a.lengths, a.free_head
        rows = [torch.cat((r, qkv[b:b + 1])) for b, r in enumerate(rows)]
        history.append(out)
    return history, rows, rope, weight, scale


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_a_prompt_and_its_steps_are_dense_attention(paged, cache):
    """assign, store and attend as a server calls them, against attention over the whole sequences in 64 bits, with keys and
    queries rounded to their types as the definition says (those of e4m3 by torch's own rounding)."""
    prompts, steps = [37, 1, 16, 90], 20
    history, rows, rope, weight, scale = run_steps(paged, prompts, steps, cache)
    for b, n in enumerate(prompts):
        for t in (0, 1, steps - 1):
            x = rows[b][:n + t + 1]
            pos = torch.arange(n + t + 1, device="cuda")
            q = store_exact(x[-1:, :4], weight, rope, pos[-1:], False, 1e-6)[0]
            k = store_exact(x[:, 4:6], weight, rope, pos, False, 1e-6)[0]
            v = x[:, 6:].double()
            score = torch.einsum("hd,jhd->hj", q[0], k.repeat_interleave(2, 1)) * 64 ** -0.5
            w = score.softmax(1)
            v = v.repeat_interleave(2, 1)
            want = torch.einsum("hj,jhd->hd", w, v)
            # a key rounded by u moves a score by u |q| . |k| scale, and the query's rounding by 2^-8 of it; weights follow by
            # exp of twice that; the value's rounding is another u of A
            u = 2.0 ** -4 if cache is E4M3 else 2.0 ** -8
            spread = torch.einsum("hd,jhd->hj", q[0].abs(), k.abs().repeat_interleave(2, 1)).amax(1) * 64 ** -0.5
            least = (2.0 ** -10 * scale if cache is E4M3 else 0.0)
            shift = (u + 2.0 ** -8) * spread + least * q[0].abs().sum(1) * 64 ** -0.5
            a = torch.einsum("hj,jhd->hd", w, v.abs()) * torch.exp(2 * shift)[:, None]
            tol = a * (torch.expm1(2 * shift)[:, None] + u + 2.0 ** -6) + least
            assert bool(((history[t][b].double() - want).abs() <= tol).all())


def test_steps_on_another_stream(paged):
    plain = run_steps(paged, [20, 3], 6, BF16)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run_steps(paged, [20, 3], 6, BF16)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(plain, other))


def test_two_captured_steps_run_at_once(paged):
    """Two graphs of attend, replayed on two streams over and over, give what eager calls give: they share nothing."""
    cases = [make_attend([4000, 7, 900], 8, 2, 128, BF16, BF16, 16, seed=s) for s in (1, 2)]
    want = [paged.attend(**c) for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for c in cases:
        g = torch.cuda.CUDAGraph()
        out = torch.zeros_like(c["q"])
        with torch.cuda.graph(g):
            paged.attend(**c, out=out)
        graphs.append(g)
        outs.append(out)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_calls_on_two_streams_at_once(paged):
    cases = [make_attend([9000, 7, 900, 3000], 8, 2, 128, BF16, BF16, 16, seed=s) for s in (1, 2, 3, 4)]
    want = [paged.attend(**c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(paged.attend(**c))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_a_graph_of_several_layers_shares_its_memory(paged):
    """Layers of one captured step: a later call's workspace may be an earlier one's, freed within the capture."""
    cases = [make_attend([5000, 33, 1200], 8, 2, 64, F16, F16, 16, seed=s) for s in range(5)]
    want = [paged.attend(**c) for c in cases]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = [paged.attend(**c) for c in cases]
    for _ in range(5):
        for x in got:
            x.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for x, w in zip(got, want))


def test_a_captured_step_follows_its_lengths(paged):
    """One graph of assign, store and attend is replayed while the lengths grow on the device."""
    gen = generator(4)
    heads, kv_heads, dim, page, requests = 4, 2, 64, 4, 3
    k_pages, v_pages = (torch.zeros(40, page, kv_heads, dim, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.full((requests, 12), -1, dtype=torch.int32, device="cuda")
    free, head, lengths, ones = i32(list(range(39, -1, -1))), i32([0]), i32([0, 0, 0]), i32([1, 1, 0])
    qkv = torch.zeros(requests, heads + 2 * kv_heads, dim, dtype=BF16, device="cuda")
    out = torch.zeros(requests, heads, dim, dtype=BF16, device="cuda")
    a = paged.Assigned(i32([0] * requests), i32([0] * requests), i32([0] * (requests + 1)), i32([0] * requests), i32([0]), i32([0] * 4))

    def step():
        paged.assign(lengths, ones, table, free, head, page, requests, out=a)
        q = paged.store(*qkv.split((heads, kv_heads, kv_heads), 1), k_pages, v_pages, a.slots, a.positions)
        paged.attend(q, k_pages, v_pages, table, a.lengths, out=out)
        lengths.copy_(a.lengths)
        head.copy_(a.free_head)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    rows = []
    for t in range(30):
        qkv.copy_(normal(qkv.shape, BF16, gen))
        rows.append(qkv.clone())
        g.replay()
        x = torch.stack(rows, 1)  # [requests, t + 1, heads, dim]
        for b in range(2):
            k, v = (y.double().repeat_interleave(2, 1) for y in (x[b, :, 4:6], x[b, :, 6:]))
            w = (torch.einsum("hd,jhd->hj", x[b, -1, :4].double(), k) * dim ** -0.5).softmax(1)
            tol = torch.einsum("hj,jhd->hd", w, v.abs()) * 2.0 ** -6
            assert bool(((out[b].double() - torch.einsum("hj,jhd->hd", w, v)).abs() <= tol).all()), (t, b)
        assert not out[2].any()
    assert lengths.tolist() == [30, 30, 0] and head.tolist() == [16]


def test_tensors_on_a_device_that_is_not_current(paged):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    s = make_attend([300, 20], 4, 2, 64, BF16, BF16, 16)
    want = paged.attend(**s)
    moved = {k: v.to("cuda:1") if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    got = paged.attend(**moved)
    assert torch.equal(got.cpu(), want.cpu()) and torch.cuda.current_device() == 0
