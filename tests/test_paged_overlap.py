"""Memory that an operator of the paged cache would write while it reads it, or write twice: refused by the host.

The calls here carry addresses that no launch may ever see, so they run only where no GPU can: an accepted call ends at the
question for the device's SMs, or at the launch.
"""

import ctypes
import random
import subprocess
from pathlib import Path

import pytest
import torch

from test_paged import ASSIGN, ATTEND, STORE, cache_fields

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are not there")

HARNESS = '''
#include <cstdio>
#include "paged_overlap.h"
using namespace emb::paged;
int main() {
    long long at[2], run[2], n[2], c[2][3], s[2][3];
    for (;;) {
        for (int i = 0; i < 2; ++i) {
            if (std::scanf("%lld %lld %lld", &at[i], &run[i], &n[i]) != 3) return 0;
            for (int k = 0; k < n[i]; ++k) if (std::scanf("%lld %lld", &c[i][k], &s[i][k]) != 2) return 1;
        }
        Area a("a", reinterpret_cast<void*>(at[0]), run[0]), b("b", reinterpret_cast<void*>(at[1]), run[1]);
        for (int k = 0; k < n[0]; ++k) a.by(c[0][k], s[0][k]);
        for (int k = 0; k < n[1]; ++k) b.by(c[1][k], s[1][k]);
        std::printf("%d%d", touch(a, b), touch(b, a));
    }
}
'''


def covered(at, run, dims):
    starts = [at]
    for c, s in dims:
        starts = [x + i * s for x in starts for i in range(c)]
    return {x + i for x in starts for i in range(run)}


def test_areas_touch_where_their_bytes_do(tmp_path):
    (tmp_path / "t.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-O1", "-std=c++17", "-I", str(ROOT / "emmy-ptx-compiler_b200" / "csrc"), "-o", str(tmp_path / "t"), str(tmp_path / "t.cpp")], check=True)
    rng = random.Random(5)
    cases = []
    for _ in range(4000):
        shared = [rng.choice((0, 4, 8, 12, 16, 24, 40, 64, 100, 160)) for _ in range(3)]  # the strides of views of one buffer, or of two
        one = []
        for side in range(2):
            dims = [(rng.choice((0, 1, 2, 3, 5)) if rng.random() < 0.1 else rng.randint(1, 5), s if rng.random() < 0.7 else rng.choice((4, 6, 20, 36, 80))) for s in shared[:rng.randint(0, 3)]]
            one.append((rng.randint(1, 300) if side else 150, rng.choice((1, 2, 4, 8, 16)), dims))
        cases.append(one)
    text = "\n".join(" ".join(f"{at} {run} {len(dims)} " + " ".join(f"{c} {s}" for c, s in dims) for at, run, dims in one) for one in cases)
    got = subprocess.run([str(tmp_path / "t")], input=text, capture_output=True, text=True, check=True).stdout
    want = ["11" if covered(*a) & covered(*b) else "00" for a, b in cases]
    assert [got[2 * i:2 * i + 2] for i in range(len(cases))] == want
    assert 500 < want.count("11") < 3500


class Call:
    def __init__(self, name, struct_):
        import __graft_entry__ as g
        g.build_binding()
        from emmy_ptx import driver
        self.library = driver.library()
        self.entry, self.struct = getattr(self.library, f"emb_paged_{name}"), struct_
        self.entry.argtypes = [ctypes.c_char_p, ctypes.c_void_p]

    def text(self, fields):
        code = self.entry(self.struct.pack(*fields), None)
        assert code != 0
        return self.library.emb_last_error().decode()


def flat(f, changes):
    f.update(changes)
    return [x for v in f.values() for x in (v if isinstance(v, list) else [v])]


# ---- store: 20 tokens of 4 + 2 + 2 heads of 64, 16 bits; a projection's row has 8 heads, 1024 bytes; the pages 4 x 16 x 2 heads

Q, K, V, KP, VP, OUT, SMALL = (x << 20 for x in range(1, 8))


def store_fields(cache=(), **changes):
    cache = dict(dict(k=KP, v=VP), **dict(cache))
    return flat(dict(q=Q, k=K, v=V, out=OUT, slots=SMALL, positions=SMALL + 4096, rope=SMALL + 8192, qw=SMALL + 65536, kw=SMALL + 65792, cache=cache_fields(**cache), q0=256,
                     q1=64, k0=128, k1=64, v0=128, v1=64, o0=256, o1=64, tokens=20, heads=4, dtype=1, rot=64, rope_rows=8, interleaved=0, eps=1e-6, r=0), changes)


QKV = dict(q=Q, k=Q + 512, v=Q + 768, q0=512, k0=512, v0=512)
PAIRS = dict(k=KP, v=KP + 4096, ks0=4096, vs0=4096)  # keys and values of a page behind one another

STORE_APART = [
    dict(), dict(out=Q), QKV, dict(QKV, out=Q, o0=512), dict(QKV, q=Q + 128, k=Q + 640, v=Q + 896, q0=768, k0=768, v0=768, o0=768, out=Q + 1152),
    dict(out=Q + 20 * 512), dict(cache=PAIRS), dict(cache=dict(PAIRS, k=KP, v=KP + 128, ks0=4096, vs0=4096, ks1=256, vs1=256, ks2=128, vs2=128)),
    dict(cache=dict(PAIRS, v=KP + 256, ks0=4096, vs0=4096, ks1=256, vs1=256)), dict(tokens=1, out=Q, q0=0, o0=0), dict(rot=0, rope=OUT, positions=OUT),
    dict(qw=0, kw=0), dict(slots=SMALL, positions=SMALL), dict(q0=0, out=Q + 512), dict(k0=0, v0=0, k=Q, v=Q)]
STORE_TOUCH = [
    (dict(out=Q + 128), "q_out and q"), (dict(out=Q + 256, o0=512), "q_out and q"), (dict(out=Q, o0=512), "q_out and q"), (dict(q0=0, out=Q), "q_out and q"),
    (dict(QKV, out=Q + 128, o0=512), "q_out and q"), (dict(QKV, out=Q + 512, o0=512), "q_out and k"), (dict(QKV, q=Q + 16384 * 4, out=Q + 384, o0=512), "q_out and k"),
    (dict(QKV, q=Q + 128, k=Q + 640, v=Q + 896, q0=768, k0=768, v0=768, o0=768, out=Q + 1024), "q_out and v"),
    (dict(k=OUT + 9728 + 384, k0=128), "q_out and k"), (dict(out=V - 16, o0=256), "q_out and v"), (dict(out=V + 20 * 256 - 16), "q_out and v"),
    (dict(out=KP + 16368), "q_out and the keys' pages"), (dict(out=VP), "q_out and the values' pages"), (dict(cache=dict(v=KP)), "the keys' pages and the values' pages"),
    (dict(cache=dict(v=KP + 2048)), "the keys' pages and the values' pages"), (dict(cache=dict(PAIRS, v=KP + 4096 - 128)), "the keys' pages and the values' pages"),
    (dict(k=KP + 4096), "the keys' pages and k"), (dict(v=KP), "the keys' pages and v"), (dict(q=VP + 128), "the values' pages and q"), (dict(slots=OUT + 512), "q_out and slots"),
    (dict(positions=KP + 64), "the keys' pages and positions"), (dict(rope=VP + 16), "the values' pages and rope"), (dict(qw=OUT), "q_out and q_weight"),
    (dict(kw=KP + 16384 - 16), "the keys' pages and k_weight")]


@pytest.mark.parametrize("changes", STORE_APART)
def test_store_takes_memory_that_is_apart(changes):
    assert "cannot be asked for its SMs" in Call("store", STORE).text(store_fields(**changes))


@pytest.mark.parametrize("changes, match", STORE_TOUCH)
def test_store_refuses_memory_that_it_writes_and_reads(changes, match):
    assert Call("store", STORE).text(store_fields(**changes)) == f"paged_store: {match} share memory"


# ---- attend: 3 requests of 4 heads of 64 over 2 key heads, a table of 2 pages a request

LSE, TABLE, WS = (x << 20 for x in range(8, 11))


def attend_fields(cache=(), **changes):
    cache = dict(dict(k=KP, v=VP), **dict(cache))
    return flat(dict(q=Q, out=OUT, lse=LSE, table=TABLE, lengths=TABLE + 4096, ws=WS, cache=cache_fields(**cache), q0=256, q1=64, o0=256, o1=64, ts=2, wb=1 << 19, requests=3,
                     heads=4, width=2, dtype=1, window=0, scale=0.125), changes)


ATTEND_APART = [
    dict(), dict(out=Q), dict(q0=512, o0=512, out=Q + 512), dict(lse=0), dict(cache=dict(v=KP)), dict(cache=PAIRS), dict(ts=0), dict(out=TABLE + 8192, lse=TABLE + 64),
    dict(out=Q + 3 * 512, lse=Q + 6 * 512), dict(requests=1, q0=0, o0=0, ts=2, out=Q), dict(ts=16, lse=TABLE + 2048), dict(q0=0, out=Q + 512), dict(cache=dict(ks0=4096, ks1=256), out=KP + 2 ** 19)]
ATTEND_TOUCH = [
    (dict(out=Q + 128), "out and q"), (dict(out=Q + 512), "out and q"), (dict(q0=512, o0=512, out=Q + 384), "out and q"), (dict(q0=0, out=Q), "out and q"), (dict(q1=128, q0=512, out=Q), "out and q"),
    (dict(out=KP), "out and the keys' pages"), (dict(out=VP + 16368), "out and the values' pages"), (dict(out=TABLE - 1520), "out and table"), (dict(out=TABLE + 4096), "out and lengths"),
    (dict(lse=OUT + 1532), "out and lse"), (dict(lse=Q), "lse and q"), (dict(lse=KP + 4), "lse and the keys' pages"), (dict(lse=TABLE + 20), "lse and table"), (dict(lse=TABLE + 4096 - 44), "lse and lengths"),
    (dict(ts=4, lse=TABLE + 4), "lse and table")]


@pytest.mark.parametrize("changes", ATTEND_APART)
def test_attend_takes_memory_that_is_apart(changes):
    assert "cannot be asked for its SMs" in Call("attend", ATTEND).text(attend_fields(**changes))


@pytest.mark.parametrize("changes, match", ATTEND_TOUCH)
def test_attend_refuses_memory_that_it_writes_and_reads(changes, match):
    assert Call("attend", ATTEND).text(attend_fields(**changes)) == f"paged_attend: {match} share memory"


# ---- assign: 3 requests, a table of 4 pages a request, 9 free pages, 8 rows


def assign_fields(**changes):
    at = {name: (1 << 20) + 4096 * i for i, name in enumerate(("cached", "fresh", "table", "free", "head", "slots", "positions", "starts", "lengths", "head_out", "report"))}
    return flat(dict(at, ts=4, requests=3, width=4, count=9, size=16, tokens=8, r=0), changes)


def place(name, offset=0):
    names = ("cached", "fresh", "table", "free", "head", "slots", "positions", "starts", "lengths", "head_out", "report")
    return (1 << 20) + 4096 * names.index(name) + offset


ASSIGN_APART = [
    dict(), dict(fresh=place("cached")), dict(head=place("cached", 8)), dict(free=place("fresh")), dict(positions=place("slots", 32)), dict(starts=place("slots", 32), lengths=place("slots", 48)),
    dict(head_out=place("report", 16)), dict(ts=16, slots=place("table", 16), positions=place("table", 80)) | dict(tokens=8), dict(requests=0, cached=0, fresh=0, table=0, lengths=0),
    dict(tokens=0, slots=place("report"), positions=place("report")), dict(count=0, free=place("slots"))]
ASSIGN_TOUCH = [
    (dict(slots=place("positions")), "slots and positions"), (dict(slots=place("positions", 28)), "slots and positions"), (dict(starts=place("lengths", -12)), "starts and lengths"),
    (dict(lengths=place("cached", 4)), "lengths and cached"), (dict(lengths=place("fresh", -8)), "lengths and fresh"), (dict(table=place("free")), "table and free_pages"),
    (dict(table=place("slots", 16)), "table and slots"), (dict(ts=16, slots=place("table", 36)), "table and slots"), (dict(head_out=place("report", 12)), "free_head_out and report"),
    (dict(head_out=place("free", 8)), "free_head_out and free_pages"), (dict(report=place("head", -12)), "report and free_head"), (dict(starts=place("head", -12)), "starts and free_head"),
    (dict(positions=place("fresh", 8)), "positions and fresh"), (dict(slots=place("free", 32)), "slots and free_pages"), (dict(table=place("head")), "table and free_head")]


@pytest.mark.parametrize("changes", ASSIGN_APART)
def test_assign_takes_memory_that_is_apart(changes):
    text = Call("assign", ASSIGN).text(assign_fields(**changes))
    assert text.startswith("launch of paged_assign: "), text  # without a device


@pytest.mark.parametrize("changes, match", ASSIGN_TOUCH)
def test_assign_refuses_memory_that_it_writes_and_reads(changes, match):
    assert Call("assign", ASSIGN).text(assign_fields(**changes)) == f"paged_assign: {match} share memory"
