"""Attention over the pages where scores and weights reach the ends of their types' ranges: what it loses to its 16-bit products.

A weight is at most 2^-32 of the row's largest off below f16's range (what weights refer to lies 7 below the maximum, and half
of f16's smallest step is 2^-25): sum_j |v_j| 2^-32 in all. The f32 sums of one long request are made of less than a thousand
keys in each of the CTAs that it is spread over, and of one part of each of these, at most three on an SM: less than 2048 terms
behind one another, 2^-13. The other terms are those of the general tests of the operators.
"""

import math

import pytest
import torch

from test_gpu_paged import make_attend, raw, rounding

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def paged():
    from emmy_ptx import paged
    return paged


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def one_request(keys, values, page=16):
    """Keys and values [n, kv heads, dim] of one request, in its pages in order."""
    n, kv_heads, dim = keys.shape
    used = -(-n // page)
    pages = []
    for x in (keys, values):
        p = torch.zeros(used * page, kv_heads, dim, dtype=torch.float32, device="cuda")
        p[:n] = x.float()
        pages.append(p.to(x.dtype).view(used, page, kv_heads, dim))
    return pages[0], pages[1], torch.arange(used, dtype=torch.int32, device="cuda")[None], i32([n])


@pytest.mark.parametrize("dtype, cache", [(F16, F16), (F16, E4M3), (BF16, E4M3), (BF16, BF16)])
@pytest.mark.parametrize("n, bits", [(131072, 25.25), (131072, 24.6), (16385, 20.0), (70000, 23.5)])
@pytest.mark.parametrize("heads", [4, 12])
def test_a_long_flat_tail_beside_one_leading_key(paged, dtype, cache, n, bits, heads):
    """The tail's weights are below f16's steps of the leading key's, and together part of the result."""
    dim, lead = 64, n // 3
    keys = torch.zeros(n, 1, dim, device="cuda")
    keys[lead, 0, 0] = 16.0
    values = torch.zeros(n, 1, dim, device="cuda")
    values[:, 0, :32] = 1.0      # a constant stays one
    values[lead, 0, 32:] = 1.0   # the leading key's share
    values[:lead, 0, 48:] = -1.0
    q = torch.zeros(1, heads, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    scale = bits * math.log(2) / 16
    lse = torch.empty(1, heads, device="cuda")
    got = paged.attend(q, *one_request(keys.to(cache), values.to(cache)), scale=scale, lse=lse)[0].double()
    tail = (n - 1) * 2.0 ** -bits
    total = 1.0 + tail
    want = torch.empty(dim, dtype=torch.float64)
    want[:32], want[32:48], want[48:] = 1.0, 1.0 / total, (1.0 - lead * 2.0 ** -bits) / total
    u, w = torch.finfo(dtype).eps / 2, (2.0 ** -11 if cache is E4M3 else torch.finfo(cache).eps / 2)
    spread = 16.0 * scale
    # (of bf16 products a weight keeps its range: only f16 has the step of 2^-32)
    tol = u + w + (0.0 if cache is BF16 else n * 2.0 ** -32) + 2.0 ** -13 + 2.0 ** -20 + spread * 2.0 ** -17
    off = (got.cpu() - want).abs().max()
    assert float(off) <= tol, (float(off), tol)
    assert bool(((lse.double() - math.log(total) - spread).abs() <= spread * 2.0 ** -18 + 2.0 ** -20 + (spread + 1) * 2.0 ** -23 + 2.0 ** -13).all())


@pytest.mark.parametrize("dtype, cache", [(F16, F16), (F16, E4M3), (BF16, E4M3), (BF16, BF16)])
@pytest.mark.parametrize("scale", [3.0e5, 1.0e7, 3.0e9, 1.0e30, -1.0e7])
def test_scores_as_large_as_they_come(paged, dtype, cache, scale):
    """Scores that lie apart by far more than their rounding: the largest one's key alone, and nothing overflows."""
    n, dim = 203, 64
    order = torch.randperm(n, generator=torch.Generator().manual_seed(3)).cuda()
    keys = torch.zeros(n, 1, dim, device="cuda")
    keys[:, 0, 0], keys[:, 0, 1] = (order // 16).float(), (order % 16).float()
    q = torch.zeros(1, 2, dim, dtype=dtype, device="cuda")
    q[:, :, 0], q[:, :, 1] = 16.0, 1.0
    values = torch.randn(n, 1, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(cache)
    got = paged.attend(q, *one_request(keys.to(cache), values), scale=scale)
    best = int(order.argmax() if scale > 0 else order.argmin())
    assert torch.equal(got[0], values[best].to(dtype).expand(2, dim))


@pytest.mark.parametrize("dtype, cache", [(F16, F16), (F16, E4M3), (BF16, BF16)])
def test_a_flat_tail_that_one_warp_sums_up(paged, dtype, cache):
    """As many requests as CTAs, all over the same pages, so that a warp has a head to itself: the tail's weights, 1.46 steps of
    f16 below the leading key's 1, are not rounded to one step."""
    n, dim, heads, bits = 262144, 64, 4, 23.45
    requests = torch.cuda.get_device_properties(0).multi_processor_count * 3
    keys = torch.zeros(n, 1, dim, device="cuda")
    keys[5, 0, 0] = 16.0
    values = torch.zeros(n, 1, dim, device="cuda")
    values[5, 0, :32] = 1.0
    values[6:, 0, 32:] = 1.0
    q = torch.zeros(requests, heads, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    k_pages, v_pages, table, lengths = one_request(keys.to(cache), values.to(cache))
    k_pages, v_pages = (p.expand(-1, -1, heads, -1) for p in (k_pages, v_pages))
    got = paged.attend(q, k_pages, v_pages, table.expand(requests, -1), lengths.expand(requests).contiguous(), scale=bits * math.log(2) / 16).double()
    tail = (n - 1) * 2.0 ** -bits
    u, w = torch.finfo(dtype).eps / 2, (2.0 ** -11 if cache is E4M3 else torch.finfo(cache).eps / 2)
    # a lane adds up an eighth of the weights (2^-24 each), a product sixteen keys (2^-23 each); weights of 2^-24 keep their bits in bf16
    tol = u + w + n / 8 * 2.0 ** -24 + n / 16 * 2.0 ** -23 + 2.0 ** -20 + 16 * 2.0 ** -17
    want = torch.tensor([1.0] * 32 + [(n - 6) * 2.0 ** -bits] * 32, dtype=torch.float64, device="cuda") / (1.0 + tail)
    off = (got - want).abs().amax((0, 1))
    assert float(off.max()) <= tol, (float(off[:32].max()), float(off[32:].max()), tol)


@pytest.mark.parametrize("dtype, cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize("heads, kv_heads, dim", [(4, 2, 64), (8, 8, 128), (12, 1, 128), (24, 2, 64), (16, 1, 256)])
def test_weights_have_more_bits_than_the_result(paged, dtype, cache, heads, kv_heads, dim):
    """A weight is held to 2^-20 of it (f16) or 2^-14 (bf16), over e4m3 codes with a bf16 result to f16's 2^-11: the result is off by
    little more than its own rounding, also where it is far smaller than the values it is made of."""
    s = make_attend([1, 2, 3, 5, 9, 17, 40, 100], heads, kv_heads, dim, dtype, cache, 16, q_scale=0.25)
    got = paged.attend(**s).double()
    held = 2.0 ** -11 if (dtype, cache) == (BF16, E4M3) else 2.0 ** -20 if dtype is F16 else 2.0 ** -14
    for b, n in enumerate(s["lengths"].tolist()):
        j = torch.arange(n, device="cuda")
        at = s["table"][b].long()[j // 16]
        k, v = (raw(p)[at, j % 16].view(cache).double().repeat_interleave(heads // kv_heads, 1) * f
                for p, f in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
        x = s["q"][b].double() * dim ** -0.5
        w = torch.einsum("hd,jhd->hj", x, k).softmax(1)
        want, a = torch.einsum("hj,jhd->hd", w, v), torch.einsum("hj,jhd->hd", w, v.abs())
        spread = torch.einsum("hd,jhd->hj", x.abs(), k.abs()).amax(1)[:, None]
        tol = (held + n * 2.0 ** -24 + 2.0 ** -20 + spread * 2.0 ** -17) * a + rounding(want, dtype)
        if cache is not BF16:
            tol = tol + v.abs().sum(0) * 2.0 ** -32
        off = (got[b] - want).abs()
        assert bool((off <= tol).all()), (n, float((off / tol).max()))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_an_infinite_value_stays_infinite(paged, dtype):
    """Beside weights that a 16-bit number holds exactly (nothing is left of them) and others."""
    s = make_attend([1, 4, 100], 4, 2, 64, dtype, dtype, 16)
    for scale in (0.0, 0.125):
        for b, at in ((0, 0), (1, 3), (2, 50)):
            page, token = int(s["table"][b, at // 16]), at % 16
            s["v_pages"][page, token, 1, 7] = math.inf
            s["v_pages"][page, token, 0, 9] = -math.inf
        got = paged.attend(**s, scale=scale)
        assert (got[:, 2:, 7] == math.inf).all() and (got[:, :2, 9] == -math.inf).all()
        got[:, 2:, 7] = got[:, :2, 9] = 0
        assert got.isfinite().all()


@pytest.mark.parametrize("largest", [2.0 ** 15, 2.0 ** 126, 2.0 ** -90])
@pytest.mark.parametrize("ratio", [2.0 ** -12, 2.0 ** -20, 2.0 ** -27])
@pytest.mark.parametrize("heads, dim", [(2, 64), (2, 128), (12, 128), (3, 256)])
def test_small_elements_beside_a_large_one_in_a_query(paged, largest, ratio, heads, dim):
    """The large element meets keys of 0, so the small ones make the scores: none of their bits is lost over e4m3 codes."""
    n, gen = 40, torch.Generator("cuda").manual_seed(dim)
    k, v = (torch.randn(n, 1, dim, device="cuda", generator=gen).to(E4M3) for _ in range(2))
    k = k.float()
    k[:, 0, 3] = 0
    q = (torch.randn(1, heads, dim, device="cuda", generator=gen).clamp(-4, 4) * (largest * ratio / 4)).bfloat16()
    q[:, :, 3] = largest
    scale = 4 / (largest * ratio) * dim ** -0.5
    got = paged.attend(q, *one_request(k.to(E4M3), v), scale=scale)[0].double()
    x, k, v = q[0].double() * scale, k[:, 0].double(), v[:, 0].double()
    w = (x @ k.T).softmax(1)
    tol = (2.0 ** -11 + n * 2.0 ** -24 + 2.0 ** -20 + (x.abs() @ k.abs().T).amax(1)[:, None] * 2.0 ** -17) * (w @ v.abs()) + v.abs().sum(0) * 2.0 ** -32
    off = (got - w @ v).abs() - rounding(w @ v, BF16) - tol
    assert float(off.max()) <= 0, float(off.max())
