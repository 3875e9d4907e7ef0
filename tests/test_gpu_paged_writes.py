"""What the paged-cache operators write into, as autograd sees it, and in which memory."""

import pytest
import torch

from test_gpu_paged import generator, make_attend, normal

pytestmark = pytest.mark.gpu

F16 = torch.float16


@pytest.fixture(scope="module")
def paged():
    from emmy_ptx import paged
    return paged


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def assign_arguments():
    return dict(cached=i32([3, 0]), fresh=i32([1, 2]), table=i32([[4, -1], [-1, -1]]), free_pages=i32([1, 2]), free_head=i32([0]), page_size=16, tokens=3,
                out=(i32([0] * 3), i32([0] * 3), i32([0] * 3), i32([0] * 2), i32([0]), i32([0] * 4)))


def store_arguments():
    gen = generator(1)
    return dict(q=normal((3, 4, 64), F16, gen), k=normal((3, 2, 64), F16, gen), v=normal((3, 2, 64), F16, gen), k_pages=normal((2, 4, 2, 64), F16, gen),
                v_pages=normal((2, 4, 2, 64), F16, gen), slots=i32([1, 5, -1]), positions=i32([0, 0, 0]), out=normal((3, 4, 64), F16, gen))


def attend_arguments():
    s = make_attend([40, 3], 4, 2, 64, F16, F16, 16)
    return s | dict(out=torch.empty_like(s["q"]), lse=torch.empty(2, 4, device="cuda"))


def tensors(arguments):
    for name, x in arguments.items():
        for i, t in enumerate(x if isinstance(x, tuple) else (x,)):
            if isinstance(t, torch.Tensor):
                yield (f"{name}[{i}]" if isinstance(x, tuple) else name), t


@pytest.mark.parametrize("name, make, written", [
    ("assign", assign_arguments, {"table"} | {f"out[{i}]" for i in range(6)}), ("store", store_arguments, {"k_pages", "v_pages", "out"}),
    ("attend", attend_arguments, {"out", "lse"})])
def test_written_tensors_count_a_version(paged, name, make, written):
    arguments = make()
    before = {n: t._version for n, t in tensors(arguments)}
    getattr(paged, name)(**arguments)
    assert {n for n, t in tensors(arguments) if t._version != before[n]} == written


def test_a_graph_that_saved_a_written_tensor_says_so(paged):
    s = store_arguments()
    weight = torch.ones(64, dtype=F16, device="cuda", requires_grad=True)
    y = (s["k_pages"] * weight).sum()
    paged.store(**s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_tensors_of_inference_mode_are_taken_in_and_out_of_it(paged):
    with torch.inference_mode():
        s = attend_arguments()
        want = paged.attend(**s).clone()
        paged.store(**store_arguments())
        paged.assign(**assign_arguments())
        other = store_arguments(), assign_arguments()
    assert torch.equal(paged.attend(**s), want)
    paged.store(**other[0])
    paged.assign(**other[1])
    with torch.inference_mode():  # tensors from outside keep their count
        arguments = store_arguments()
    plain = attend_arguments()
    with torch.inference_mode():
        paged.attend(**plain)
    assert plain["out"]._version > 0 and arguments["out"].is_inference()


@pytest.mark.parametrize("lengths, heads, kv_heads, dim, cache", [
    ([5000, 17, 0, 900, 12000], 8, 2, 128, F16), ([9000, 0, 7, 5000, 8000] * 12, 32, 8, 128, F16), ([40, 3, 100], 4, 2, 64, F16), ([9000, 0, 17, 12000] * 20, 16, 4, 64, torch.float8_e4m3fn),
    ([700] * 50, 40, 1, 256, F16)])
def test_attend_puts_its_result_where_the_queries_were(paged, lengths, heads, kv_heads, dim, cache):
    """Heads that are cut, whole, shared by warps and side by side, and groups of more rows than a block has."""
    s = make_attend(lengths, heads, kv_heads, dim, F16, cache, 16)
    want = paged.attend(**s)
    wide = torch.full((len(lengths), heads + 3, dim), 5.0, dtype=F16, device="cuda")
    for queries in (s["q"].clone(), wide[:, 1:heads + 1].copy_(s["q"])):
        got = paged.attend(**(s | dict(q=queries, out=queries)))
        assert got.data_ptr() == queries.data_ptr() and torch.equal(queries, want)
    assert bool((wide[:, 0] == 5).all()) and bool((wide[:, heads + 1:] == 5).all())


def test_attend_refuses_a_workspace_that_something_else_is(paged):
    """Through the C entry: the workspace over out, lse, the queries or the pages, wholly or by its last bytes."""
    from emmy_ptx import driver
    from test_paged import ATTEND
    import ctypes
    library = driver.library()
    library.emb_paged_attend.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    library.emb_paged_attend_workspace.argtypes, library.emb_paged_attend_workspace.restype = [ctypes.c_char_p], ctypes.c_int64
    s = attend_arguments()
    s["table"] = s["table"].contiguous()
    arena = torch.zeros(1 << 22, dtype=torch.uint8, device="cuda")

    def fields(workspace, size, width=1000):
        k, v = s["k_pages"], s["v_pages"]
        return ATTEND.pack(s["q"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(), workspace,
                           k.data_ptr(), v.data_ptr(), *k.stride()[:3], *v.stride()[:3], k.shape[0], 16, 2, 64, 1, 1.0, 1.0, 0, 256, 64, 256, 64, s["table"].shape[1], size, 2, 4,
                           width, 1, 0, 0.125)

    need = library.emb_paged_attend_workspace(fields(0, 0))  # (a table row this wide is never reached by these lengths)
    assert 0 < need < arena.numel()
    s["table"] = torch.zeros(2, 1000, dtype=torch.int32, device="cuda")
    s["out"] = arena[need:].view(F16)[:2 * 4 * 64].view(2, 4, 64)
    s["lse"] = arena[-4096:].view(torch.float32)[:8].view(2, 4)
    for workspace, which in ((arena.data_ptr() + 16, "the workspace and out"), (s["lse"].data_ptr() - need + 16, "the workspace and lse"),
                             (s["q"].data_ptr(), "the workspace and "), (s["k_pages"].data_ptr() - need + 16, "the workspace and ")):
        assert library.emb_paged_attend(fields(workspace, need), None) == -2
        text = library.emb_last_error().decode()
        assert text.startswith("paged_attend: " + which) and text.endswith("share memory"), text
    assert library.emb_paged_attend(fields(arena.data_ptr(), need), torch.cuda.current_stream().cuda_stream) == 0  # it ends where out begins
    torch.cuda.synchronize()
