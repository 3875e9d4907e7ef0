"""Attention over the pages where scores and weights reach the ends of their types' ranges."""

import pytest
import torch

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
