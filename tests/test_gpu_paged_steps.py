"""A server's steps, assign, store and attend together: every token of every request, looked up through the table as a reader does, is
the rounded row that the definition gives, and each output is attention over just those rows, as near as one call alone."""

import pytest
import torch

from paged_oracle import BF16, E4M3, F16, attended, is_rounded, normed_and_rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from emmy_ptx import paged
    return paged


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def raw(t):
    return t.view(torch.uint8) if t.dtype is E4M3 else t


@pytest.mark.parametrize("dtype, cache", [(BF16, BF16), (BF16, E4M3), (F16, F16), (F16, E4M3)])
@pytest.mark.parametrize("page", [16, 7])
def test_steps_of_a_server(paged, dtype, cache, page):
    """Prompts in two pieces, then single tokens; one request rests in every third step and one row is padding."""
    heads, kv_heads, dim, steps = 4, 2, 64, 18
    first, second = [37, 1, 16, 60, 0], [0, 0, 5, 30, 9]
    requests, longest = len(first), 90 + steps
    gen = torch.Generator("cuda").manual_seed(page)
    width = -(-longest // page)
    k_scale, v_scale = (0.05, 0.04) if cache is E4M3 else (1.0, 1.0)
    k_pages, v_pages = (torch.full((requests * width + 4, page, kv_heads, dim), 3.0, device="cuda").to(cache) for _ in range(2))
    table = torch.full((requests, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(requests * width + 4, device="cuda", generator=gen).to(torch.int32)
    angle = torch.arange(longest, device="cuda")[:, None] * 50.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)
    rope = torch.cat((angle.cos(), angle.sin()), 1).float()
    wq, wk = (torch.randn(dim, device="cuda", generator=gen).to(dtype) for _ in range(2))
    lengths, head = i32([0] * requests), i32([0])
    seen = [torch.zeros(0, heads + 2 * kv_heads, dim, dtype=dtype, device="cuda") for _ in range(requests)]  # what each request was given
    held = [None] * requests  # and what its rows were in the pages

    def step(fresh, padding):
        nonlocal lengths, head
        rows = sum(fresh) + padding
        qkv = torch.randn(rows, heads + 2 * kv_heads, dim, device="cuda", generator=gen).to(dtype)
        a = paged.assign(lengths, i32(fresh), table, free, head, page, rows)
        q = paged.store(*qkv.split((heads, kv_heads, kv_heads), 1), k_pages, v_pages, a.slots, a.positions, rope=rope, q_weight=wq, k_weight=wk, k_scale=k_scale, v_scale=v_scale)
        assert a.report.tolist()[1:] == [0, 0, sum(fresh)]
        at = 0
        for b, n in enumerate(fresh):
            seen[b] = torch.cat((seen[b], qkv[at:at + n]))
            at += n
        lengths, head = a.lengths, a.free_head
        assert lengths.tolist() == [len(s) for s in seen] and int(head) == sum(-(-len(s) // page) for s in seen)
        return q

    def check_pages():
        pages = []
        for b, x in enumerate(seen):
            j = torch.arange(len(x), device="cuda")
            ids = table[b].long()[j // page]
            pages += ids.unique().tolist()
            k, v = (raw(p)[ids, j % page].view(cache) for p in (k_pages, v_pages))
            want, terms = normed_and_rotated(x[:, heads:heads + kv_heads], wk, rope, j)
            assert is_rounded(k, want / k_scale, terms / k_scale, cache)
            value = x[:, heads + kv_heads:].double() / v_scale
            assert is_rounded(v, value, value.abs(), cache)
            if held[b] is not None:  # what was stored once stays
                assert all(torch.equal(raw(new)[:len(old)], raw(old)) for new, old in zip((k, v), held[b]))
            held[b] = k.clone(), v.clone()
        assert len(pages) == len(set(pages)) == int(head)  # no page is two requests'

    for fresh in (first, second):
        step(fresh, 2)
        check_pages()
    for t in range(steps):
        fresh = [1, 1, 1, 1 if t % 3 else 0, 1]
        q = step(fresh, 0 if t % 2 else 1)
        check_pages()
        of = torch.tensor([b for b in range(requests) if fresh[b]], device="cuda")
        got = paged.attend(q[:len(of)], k_pages, v_pages, table[of], lengths[of], k_scale=k_scale, v_scale=v_scale)
        for i, b in enumerate(of.tolist()):
            n = len(seen[b])
            want, terms = normed_and_rotated(seen[b][-1:, :heads], wq, rope, torch.arange(n - 1, n, device="cuda"))
            assert is_rounded(q[i], want[0], terms[0], dtype)
            out, tol = attended(q[i], held[b][0].double() * k_scale, held[b][1].double() * v_scale, dtype, cache)
            assert bool(((got[i].double() - out).abs() <= tol).all()), (t, b)
