"""What the paged-cache operators write into, as autograd sees it."""

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
