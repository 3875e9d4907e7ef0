"""The oracle of a serving step's test can tell: outputs that are wrong in the ways a server's step goes wrong lie outside what it allows."""

import pytest
import torch

from paged_oracle import BF16, E4M3, F16, attended, is_rounded, normed_and_rotated


def rows(n, cache, seed, dtype):
    """A request's queries, keys and values as the operators hold them: normed, rotated, rounded to the cache's type."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 8, 64, generator=gen).to(dtype)
    angle = torch.arange(n)[:, None] * 50.0 ** (-torch.arange(0, 64, 2) / 64)
    rope, weight = torch.cat((angle.cos(), angle.sin()), 1).float(), torch.randn(64, generator=gen).to(dtype)
    scale = 0.05 if cache is E4M3 else 1.0
    q = normed_and_rotated(x[-1:, :4], weight, rope, torch.arange(n)[-1:])[0][0].to(dtype)
    k = normed_and_rotated(x[:, 4:6], weight, rope, torch.arange(n))[0]
    return q, *((y.double() / scale).clamp(-448, 448).to(cache).double() * scale for y in (k, x[:, 6:]))


@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (BF16, E4M3), (F16, F16), (F16, E4M3)])
@pytest.mark.parametrize("n", [2, 17, 21, 38, 57, 91, 110])
def test_wrong_outputs_are_told(dtype, cache, n):
    q, k, v = rows(n, cache, n, dtype)
    out, tol = attended(q, k, v, dtype, cache)
    assert bool(((out.to(dtype).double() - out).abs() <= tol).all())
    last = torch.arange(n) == n - 1
    wrong = {
        "zeros": torch.zeros_like(out), "half": out / 2, "the plain mean": v.mean(0).repeat_interleave(2, 0),
        "the new token dropped": attended(q, k[:-1], v[:-1], dtype, cache)[0],
        "the first token dropped": attended(q, k[1:], v[1:], dtype, cache)[0],
        "the new token's key beside another's values": attended(q, k, torch.where(last[:, None, None], v.roll(1, 0), v), dtype, cache)[0],
        "the new token twice": attended(q, torch.cat((k, k[-1:])), torch.cat((v, v[-1:])), dtype, cache)[0],
        "keys and values of the other head": attended(q, k.flip(1), v.flip(1), dtype, cache)[0],
        "a scale of values that is off by a percent": out * 1.01,
        "a scale of keys that is off by two percent": attended(q, k * 1.02, v, dtype, cache)[0]}
    for name, x in wrong.items():
        assert bool(((x.to(dtype).double() - out).abs() > tol).any()), name


def test_a_row_that_is_not_the_rounded_one_is_told():
    gen = torch.Generator().manual_seed(1)
    x, weight = torch.randn(9, 2, 64, generator=gen).bfloat16(), torch.randn(64, generator=gen).bfloat16()
    angle = torch.arange(20)[:, None] * 50.0 ** (-torch.arange(0, 64, 2) / 64)
    rope = torch.cat((angle.cos(), angle.sin()), 1).float()
    y, terms = normed_and_rotated(x, weight, rope, torch.arange(9))
    for dtype in (BF16, E4M3):
        assert is_rounded(y.to(dtype), y, terms, dtype)
        for other in (normed_and_rotated(x, weight, rope, torch.arange(1, 10))[0], y.roll(1, 0), y * 1.2, torch.zeros_like(y)):
            assert not is_rounded(other.to(dtype), y, terms, dtype)
