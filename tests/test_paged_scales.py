"""Scales of an 8-bit cache that the operators could not use, and scales of a cache that has none, are refused by the host."""

import math

import pytest
import torch

from test_paged import ATTEND, STORE
from test_paged_overlap import Call, attend_fields, store_fields

E4M3_CODES = 0  # EMB_U8
SUBNORMAL = (1e-45, 2.9e-39, 1.17e-38)


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are not there")
@pytest.mark.parametrize("name, struct_, fields", [("store", STORE, store_fields), ("attend", ATTEND, attend_fields)])
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_the_entries_refuse_scales(name, struct_, fields, which):
    call = Call(name, struct_)
    for scale in (*SUBNORMAL, 0.0, -1.0, math.inf, math.nan, 3.3e38):
        assert "is not a positive number" in call.text(fields(cache={"dtype": E4M3_CODES, which: scale})), scale
    for scale in (1.18e-38, 1.0, 2.9e38):
        assert "cannot be asked for its SMs" in call.text(fields(cache={"dtype": E4M3_CODES, which: scale})), scale
    for scale in (0.5, 2.0, 1.0000001):
        assert "scales belong to a cache of e4m3 codes" in call.text(fields(cache={"dtype": 1, which: scale})), scale
