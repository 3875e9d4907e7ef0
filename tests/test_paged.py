"""The paged-cache operators on a machine without a GPU: what they refuse, and the layout of their argument structures."""

import ctypes
import struct
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]

# the structures of include/emmy_b200.h, field by field
CACHE = "QQ 3q 3q iiii i ff i"
ASSIGN = struct.Struct("@QQQQQQQQQQQ q iiii i i".replace(" ", ""))
STORE = struct.Struct(("@QQQQQQQQQ" + CACHE + "2q 2q 2q 2q ii i i i i f i").replace(" ", ""))
ATTEND = struct.Struct(("@QQQQQQ" + CACHE + "2q 2q q q ii i i i f").replace(" ", ""))


@pytest.fixture(scope="module")
def paged():
    import __graft_entry__ as g
    g.build_binding()
    from emmy_ptx import paged
    return paged


def test_the_packed_structures_are_those_of_the_header(tmp_path, paged):
    src = tmp_path / "layout.cpp"
    src.write_text('''
#include <cstddef>
#include <cstdio>
#include "emmy_b200.h"
int main() {
    std::printf("%zu %zu %zu %zu %zu %zu %zu %zu %zu\\n", sizeof(emb_paged_assign_t), sizeof(emb_paged_store_t), sizeof(emb_paged_attend_t),
                offsetof(emb_paged_assign_t, tokens), offsetof(emb_paged_store_t, cache), offsetof(emb_paged_store_t, eps),
                offsetof(emb_paged_attend_t, cache), offsetof(emb_paged_attend_t, table_stride), offsetof(emb_paged_attend_t, scale));
}
''')
    subprocess.run(["g++", "-I", str(ROOT / "include"), "-o", str(tmp_path / "layout"), str(src)], check=True)
    out = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.split()]
    assert out[:3] == [ASSIGN.size, STORE.size, ATTEND.size]
    # a value put into each field of interest is found at the field's offset
    pack = ASSIGN.pack(*range(11), 0, 0, 0, 0, 0, 77, 0)
    assert int.from_bytes(pack[out[3]:out[3] + 4], "little") == 77
    cache = (5, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 1.0, 1.0, 0)
    pack = STORE.pack(*[0] * 9, *cache, *[0] * 8, 0, 0, 0, 0, 0, 0, 0.5, 0)
    assert pack[out[4]] == 5 and pack[out[5]:out[5] + 4] == b"\x00\x00\x00\x3f"
    pack = ATTEND.pack(*[0] * 6, *cache, *[0] * 4, 9, 0, 0, 0, 0, 0, 0, 0.5)
    assert pack[out[6]] == 5 and pack[out[7]] == 9 and pack[out[8]:out[8] + 4] == b"\x00\x00\x00\x3f"


def pages(n=4, size=16, heads=2, dim=64, dtype=torch.float16):
    return torch.zeros(n, size, heads, dim, dtype=dtype), torch.zeros(n, size, heads, dim, dtype=dtype)


def i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def rows(n=3, heads=4, dim=64, dtype=torch.float16):
    return torch.zeros(n, heads, dim, dtype=dtype)


def refused(call, match):
    from emmy_ptx import driver
    with pytest.raises(driver.EmbError, match=match) as err:
        call()
    assert err.value.code == -2


def test_attend_refuses(paged):
    k, v = pages()
    q, table, lengths = rows(), i32(3, 2), i32(3)
    refused(lambda: paged.attend(q[0], k, v, table, lengths), r"q is a tensor \[rows, heads, dim\]")
    refused(lambda: paged.attend(q.float(), k, v, table, lengths), "q is f16 or bf16")
    refused(lambda: paged.attend(q.bfloat16(), k, v, table, lengths), "same 16-bit type")
    refused(lambda: paged.attend(q, k, v[:3], table, lengths), "two tensors")
    refused(lambda: paged.attend(q, k, v, table, lengths, k_scale=2.0), "scales belong")
    refused(lambda: paged.attend(q, *pages(dim=128), table, lengths), "heads of 64, pages of 128")
    refused(lambda: paged.attend(q, k, v, None, lengths), "table is not a tensor")
    refused(lambda: paged.attend(q, k, v, table, lengths, window=1 << 40), "window is beyond 31 bits")
    refused(lambda: paged.attend(q, k, v, table, lengths, scale="a"), "scale is not a number")
    refused(lambda: paged.attend(q, k, v, table.long(), lengths), "table is an int32")
    refused(lambda: paged.attend(q, k, v, table, i32(4)), "lengths is a contiguous int32")
    refused(lambda: paged.attend(q, k, v, i32(2, 3).t(), lengths), "contiguous rows")
    refused(lambda: paged.attend(q, k, v, table, lengths, out=rows(4)), "out is")
    refused(lambda: paged.attend(q, k, v, table, lengths, lse=torch.zeros(3, 5)), "lse is")
    refused(lambda: paged.attend(torch.zeros(3, 64, 4, dtype=torch.float16).transpose(1, 2), k, v, table, lengths), "not contiguous")
    if not torch.cuda.is_available():
        refused(lambda: paged.attend(q, k, v, table, lengths), "GPU only")


def test_store_refuses(paged):
    k_pages, v_pages = pages()
    q, k, v, slots, positions = rows(), rows(heads=2), rows(heads=2), i32(3), i32(3)
    rope = torch.zeros(8, 32)
    refused(lambda: paged.store(q, k[:2], v, k_pages, v_pages, slots, positions), "k is")
    refused(lambda: paged.store(q, k, v.bfloat16(), k_pages, v_pages, slots, positions), "v is")
    refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots.long(), positions), "slots is")
    refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots, positions[:2], rope=rope), "positions is")
    refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots, positions, rope=rope.half()), "rope is")
    refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots, positions, q_weight=torch.zeros(64)), "q_weight is")
    refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots, positions, k_weight=torch.zeros(128).half()), "k_weight is")
    refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots, positions, out=rows(4)), "out is")


def test_tensors_that_require_a_gradient_are_refused(paged):
    k_pages, v_pages = pages()
    q, k, v, slots, weight = rows(), rows(heads=2), rows(heads=2), i32(3), torch.zeros(64, dtype=torch.float16)
    wanted = weight.clone().requires_grad_()
    refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots, slots, q_weight=wanted), "q_weight requires a gradient")
    refused(lambda: paged.store(q, k.clone().requires_grad_(), v, k_pages, v_pages, slots, slots), "k requires a gradient")
    refused(lambda: paged.attend(q.clone().requires_grad_(), k_pages, v_pages, i32(3, 2), slots), "q requires a gradient")
    with torch.no_grad():  # then the next thing is refused
        refused(lambda: paged.store(q, k, v, k_pages, v_pages, slots[:2], slots, q_weight=wanted), "slots is")


def test_assign_refuses(paged):
    cached, fresh, table, free, head = i32(3), i32(3), i32(3, 4), i32(9), i32(1)
    refused(lambda: paged.assign(cached.long(), fresh, table, free, head, 16, 8), "cached is")
    refused(lambda: paged.assign(cached, fresh[:2], table, free, head, 16, 8), "fresh is")
    refused(lambda: paged.assign(cached, fresh, table[:2], free, head, 16, 8), "table is")
    refused(lambda: paged.assign(cached, fresh, table, free, i32(2), 16, 8), "free_head is")
    refused(lambda: paged.assign(cached, fresh, table, free, head, 16, -1), "tokens is negative")
    refused(lambda: paged.assign(cached, fresh, table, free, head, 16, 8, out=(i32(8), i32(8), i32(3), i32(3), i32(1), i32(4))), "out.starts is")


# ---- the C entries' own checks: addresses that no launch ever sees


class Call:
    def __init__(self, paged, name, struct_):
        from emmy_ptx import driver
        self.entry, self.struct = getattr(driver.library(), f"emb_paged_{name}"), struct_
        self.entry.argtypes = [ctypes.c_char_p, ctypes.c_void_p]

    def refused(self, fields, match):
        from emmy_ptx import driver
        assert self.entry(self.struct.pack(*fields), None) == -2
        text = driver.library().emb_last_error().decode()
        assert match in text, text


A = 4096  # an aligned address


def cache_fields(**kw):
    f = dict(k=A, v=A, ks0=2048, ks1=128, ks2=64, vs0=2048, vs1=128, vs2=64, pages=4, size=16, heads=2, dim=64, dtype=1, k_scale=1.0, v_scale=1.0, r=0)
    f.update(kw)
    return list(f.values())


def attend_fields(cache=(), **kw):
    f = dict(q=A, out=A, lse=0, table=A, lengths=A, ws=A, cache=cache_fields(**dict(cache)), q0=256, q1=64, o0=256, o1=64, ts=2, wb=1 << 30, requests=3, heads=4,
             width=2, dtype=1, window=0, scale=0.125)
    f.update(kw)
    return [x for v in f.values() for x in (v if isinstance(v, list) else [v])]


@pytest.mark.parametrize("change, match", [
    (dict(dtype=3), "f16 or bf16"), (dict(dtype=2), "q's type or e4m3"), (dict(cache=dict(dim=96)), "head dim 96"),
    (dict(cache=dict(pages=0)), "at least one"), (dict(cache=dict(pages=1 << 20, size=1 << 11)), "less than 2^31"),
    (dict(cache=dict(heads=0)), "key heads"), (dict(cache=dict(k=A + 8)), "16-byte aligned"), (dict(cache=dict(v=0)), "null"),
    (dict(cache=dict(ks1=100)), "stride of the pages"), (dict(cache=dict(k_scale=0.0)), "positive"), (dict(cache=dict(v_scale=float("nan"))), "positive"),
    (dict(heads=3), "multiple of the key heads"), (dict(requests=-1), "requests"), (dict(width=0), "table row"),
    (dict(width=1 << 28), "table row"), (dict(window=-1), "window"), (dict(scale=float("inf")), "finite"), (dict(lengths=0), "null table or lengths"),
    (dict(q=A + 2), "aligned"), (dict(q0=100), "multiple of 16 bytes"), (dict(o0=0), "overlap"), (dict(o0=64, o1=64), "overlap")])
def test_attend_entry_refuses(paged, change, match):
    Call(paged, "attend", ATTEND).refused(attend_fields(**change), match)


def store_fields(cache=(), **kw):
    f = dict(q=A, k=A, v=A, out=A, slots=A, positions=A, rope=A, qw=A, kw=A, cache=cache_fields(**dict(cache)), q0=256, q1=64, k0=128, k1=64, v0=128,
             v1=64, o0=256, o1=64, tokens=3, heads=4, dtype=1, rot=64, rope_rows=8, interleaved=0, eps=1e-6, r=0)
    f.update(kw)
    return [x for v in f.values() for x in (v if isinstance(v, list) else [v])]


@pytest.mark.parametrize("change, match", [
    (dict(tokens=-1), "rows"), (dict(heads=0), "rows"), (dict(rot=24), "multiple of 16"), (dict(rot=128), "up to the head dim"),
    (dict(rope=0), "without a table"), (dict(rope=A + 4), "16-byte"), (dict(rope_rows=0), "without a table"), (dict(eps=-1.0), "eps"),
    (dict(qw=A + 2), "norm weight"), (dict(slots=0), "null slots"), (dict(positions=0), "positions"), (dict(k=0), "null"), (dict(v0=4), "multiple of 16"),
    (dict(o0=128), "q_out overlap"), (dict(cache=dict(ks0=0)), "cache overlap"), (dict(cache=dict(vs1=64, vs2=64)), "cache overlap")])
def test_store_entry_refuses(paged, change, match):
    Call(paged, "store", STORE).refused(store_fields(**change), match)


def assign_fields(**kw):
    f = dict(cached=A, fresh=2 * A, table=A, free=A, head=A, slots=A, positions=A, starts=A, lengths=3 * A, head_out=2 * A, report=A, ts=4, requests=3,
             width=4, count=9, size=16, tokens=8, r=0)
    f.update(kw)
    return list(f.values())


@pytest.mark.parametrize("change, match", [
    (dict(requests=-1), "negative"), (dict(size=0), "page size below 1"), (dict(width=0), "table width"), (dict(tokens=-1), "negative"),
    (dict(cached=0), "null pointer"), (dict(free=0), "null pointer"), (dict(slots=0), "null pointer"), (dict(ts=3), "overlap"),
    (dict(lengths=A), "may not be"), (dict(head_out=A), "may not be"), (dict(width=1 << 27), "2^31")])
def test_assign_entry_refuses(paged, change, match):
    Call(paged, "assign", ASSIGN).refused(assign_fields(**change), match)


def test_null_arguments_are_refused(paged):
    from emmy_ptx import driver
    for name in ("assign", "store", "attend"):
        assert getattr(driver.library(), f"emb_paged_{name}")(None, None) == -2
        assert b"null arguments" in driver.library().emb_last_error()
