"""The paged-cache operators have no gradients: what would silently lose one is refused, before anything else is looked at."""

import pytest
import torch


@pytest.fixture(scope="module")
def paged():
    import __graft_entry__ as g
    g.build_binding()
    from emmy_ptx import paged
    return paged


def zeros(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype)


def store_arguments():
    return dict(q=zeros(3, 4, 64), k=zeros(3, 2, 64), v=zeros(3, 2, 64), k_pages=zeros(4, 16, 2, 64), v_pages=zeros(4, 16, 2, 64),
                slots=zeros(3, dtype=torch.int32), positions=zeros(3, dtype=torch.int32), rope=zeros(8, 32, dtype=torch.float32),
                q_weight=zeros(64), k_weight=zeros(64), out=zeros(3, 4, 64))


def attend_arguments():
    return dict(q=zeros(3, 4, 64), k_pages=zeros(4, 16, 2, 64), v_pages=zeros(4, 16, 2, 64), table=zeros(3, 2, dtype=torch.int32),
                lengths=zeros(3, dtype=torch.int32), out=zeros(3, 4, 64), lse=zeros(3, 4, dtype=torch.float32))


FLOATS = [(name, argument) for name, make in (("store", store_arguments), ("attend", attend_arguments)) for argument, t in make().items() if t.is_floating_point()]


def refused(paged, name, arguments, match):
    from emmy_ptx import driver
    with pytest.raises(driver.EmbError, match=match) as err:
        getattr(paged, name)(**arguments)
    assert err.value.code == -2


@pytest.mark.parametrize("name, argument", FLOATS)
def test_each_tensor_that_requires_a_gradient_is_refused(paged, name, argument):
    arguments = store_arguments() if name == "store" else attend_arguments()
    arguments[argument].requires_grad_()
    refused(paged, name, arguments, f"{argument} requires a gradient")
    arguments[argument] = arguments[argument] * 2  # not a leaf
    refused(paged, name, arguments, f"{argument} requires a gradient")
    with torch.no_grad():  # then it is the device that is refused
        refused(paged, name, arguments, "GPU only")


@pytest.mark.parametrize("name, argument", FLOATS)
def test_each_tensor_with_a_tangent_is_refused(paged, name, argument):
    from torch.autograd import forward_ad
    arguments = store_arguments() if name == "store" else attend_arguments()
    plain = arguments[argument]
    with forward_ad.dual_level():
        arguments[argument] = forward_ad.make_dual(plain, torch.ones_like(plain))
        refused(paged, name, arguments, f"{argument} has a tangent")
        with torch.no_grad():
            refused(paged, name, arguments, f"{argument} has a tangent")
        arguments[argument] = plain  # then it is the device that is refused
        refused(paged, name, arguments, "GPU only")
