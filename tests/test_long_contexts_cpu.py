"""Sinks, shared prefixes and pages: calls that are refused, and host arithmetic, without a GPU."""
import ctypes as C

import pytest
import torch

import parallax_b200 as plx
from parallax_b200 import _cabi
from tests.test_sinks_prefix_cpu import decode_problem, prefix, z

PAGED = dict(page_table=1 << 20, page_size=16, pages_per_seq=80, n_pages=100, cache_len=1280)


@pytest.mark.parametrize("splits", [0, 1, 4])
@pytest.mark.parametrize("scale", [0.088, -0.088])
def test_a_prefix_of_its_own_in_front_of_pages_is_refused(splits, scale):
    """The launch in which every row sweeps the prefix itself knows no page table behind it."""
    one = C.c_void_p(1 << 20)
    call = lambda p: _cabi.lib().plx_decode_prefix(C.byref(p), C.byref(prefix(n_splits=splits)), *[one] * 6, one, 1 << 30, None)    # noqa: E731
    assert call(decode_problem(qk_scale=scale, **PAGED)) == _cabi.PLX_ERR_UNSUPPORTED
