"""The serving step over a paged cache in 64 bits, on any device, with what the operators may be off by."""

import torch

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def rounding(y, dtype):
    """What a rounding of y to dtype may be off by: half a step, and below the normal range half of the smallest subnormal."""
    info = torch.finfo(dtype)
    least = 2.0 ** -10 if dtype is E4M3 else info.smallest_normal * info.eps / 2
    return (y.abs() * (2.0 ** -4 if dtype is E4M3 else info.eps / 2)).clamp(min=least)


def normed_and_rotated(x, weight, rope, positions, eps=1e-6):
    """x [rows, heads, dim] -> (values, the sum of |terms| that each was made from); pairs (j, j + half)."""
    y = x.double()
    y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = rope.shape[1] // 2
    c, s = (t[:, None, :] for t in rope.double()[positions].split(half, 1))
    a, b, rest = y[..., :half], y[..., half:2 * half], y[..., 2 * half:]
    values = torch.cat((a * c - b * s, b * c + a * s, rest), -1)
    terms = torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), rest.abs()), -1)
    return values, terms


def is_rounded(got, y, terms, dtype):
    """Whether got is y rounded once to dtype (e4m3: saturating), after f32 steps off by less than 2^-20 of the terms."""
    if dtype is E4M3:
        y = y.clamp(-448, 448)
    return bool(((got.double() - y).abs() <= rounding(y, dtype) + terms * 2.0 ** -20).all())


def attended(q, k, v, dtype, cache):
    """One query [heads, dim] over keys and values [n, kv heads, dim] as they are held, times their scales -> (out, what it may be off by).

    A weight is off by 2^-14 of it (bf16 cache), 2^-20 (f16 queries) or 2^-11 (bf16 queries over e4m3 codes), of f16 products
    also by 2^-32 of the largest; a score by 2^-18 of sum |q k| scale, which a weight follows twice; the f32 sums by 2^-24 a
    term, the exponentials by 2^-20; the result is rounded once."""
    n, kv_heads, dim = k.shape
    q, k, v = q.double() * dim ** -0.5, k.double().repeat_interleave(len(q) // kv_heads, 1), v.double().repeat_interleave(len(q) // kv_heads, 1)
    w = torch.einsum("hd,jhd->hj", q, k).softmax(1)
    out, size = torch.einsum("hj,jhd->hd", w, v), torch.einsum("hj,jhd->hd", w, v.abs())
    spread = torch.einsum("hd,jhd->hj", q.abs(), k.abs()).amax(1)[:, None]
    held = 2.0 ** -20 if dtype is F16 else 2.0 ** -14 if cache is BF16 else 2.0 ** -11
    tol = (held + n * 2.0 ** -24 + 2.0 ** -20 + spread * 2.0 ** -17) * size + rounding(out, dtype)
    return out, tol if cache is BF16 else tol + v.abs().sum(0) * 2.0 ** -32
