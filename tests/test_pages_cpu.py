"""Pages of a paged cache: what the calls refuse before anything is launched, and the C ABI's own checks."""
import ctypes as C

import pytest
import torch

import parallax_b200 as plx
from parallax_b200 import _cabi

POOL = (8, 16, 2, 64)


def pool(*shape, dtype=torch.bfloat16):
    return torch.zeros(*(shape or POOL), dtype=dtype)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


TABLE, LENS = torch.zeros(2, 4, dtype=torch.int32), ints(5, 20)


@pytest.mark.parametrize("call,error", [
    (lambda: plx.parallax_copy_pages(pool(dtype=torch.float32), pool(dtype=torch.float32), ints(0), ints(1)), TypeError),
    (lambda: plx.parallax_copy_pages(pool(), pool(dtype=torch.float16), ints(0), ints(1)), TypeError),
    (lambda: plx.parallax_copy_pages(pool(), pool(9, 16, 2, 64), ints(0), ints(1)), ValueError),
    (lambda: plx.parallax_copy_pages(pool(8, 12, 2, 64), pool(8, 12, 2, 64), ints(0), ints(1)), ValueError),
    (lambda: plx.parallax_copy_pages(pool(8, 16, 2, 4), pool(8, 16, 2, 4), ints(0), ints(1)), NotImplementedError),
    (lambda: plx.parallax_copy_pages(pool(), pool(), ints(0), ints(1)), RuntimeError),                       # no CPU path
    (lambda: plx.parallax_fork_pages(pool(), pool(), TABLE, LENS, ints(0), ints(1)), RuntimeError),
    (lambda: plx.parallax_compact_pages(pool(), pool(), TABLE, LENS), RuntimeError),
    (lambda: plx.parallax_free_pages(TABLE, LENS, ints(0), 8, 16), RuntimeError),
    (lambda: plx.parallax_free_pages(TABLE.long(), LENS, ints(0), 8, 16), TypeError),
    (lambda: plx.parallax_free_pages(TABLE, LENS.long(), ints(0), 8, 16), TypeError),
    (lambda: plx.parallax_free_pages(TABLE, LENS[:1], ints(0), 8, 16), ValueError),
    (lambda: plx.parallax_free_pages(TABLE[0], LENS, ints(0), 8, 16), ValueError),
    (lambda: plx.parallax_free_pages(TABLE, LENS, TABLE, 8, 16), ValueError),
    (lambda: plx.parallax_free_pages(TABLE, LENS, ints(0), 0, 16), ValueError),
    (lambda: plx.parallax_free_pages(TABLE, LENS, ints(0), 8, 24), ValueError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def c_pool(**kw):
    p = _cabi.PagePool()
    p.k = p.v = 1 << 20
    p.n_pages, p.page_size, p.heads_kv, p.head_dim = POOL
    for s in ("k", "v"):
        for axis, n in zip("pth", (16 * 2 * 64, 2 * 64, 64)):
            setattr(p, f"{s}_stride_{axis}", n)
    for name, x in kw.items():
        setattr(p, name, x)
    return p


@pytest.mark.parametrize("kw", [dict(k=None), dict(page_size=12), dict(n_pages=0), dict(head_dim=60), dict(k_stride_t=100), dict(v=(1 << 20) + 2),
                                dict(k_stride_p=0)])
def test_c_abi_checks_come_before_the_device(kw):
    lib, one = _cabi.lib(), C.c_void_p(1 << 20)
    assert lib.plx_pages_copy(C.byref(c_pool(**kw)), one, one, 1, None) == -1
    assert lib.plx_pages_compact(C.byref(c_pool(**kw)), one, one, 2, 4, one, one, one, 1 << 20, None) == -1


def test_c_abi_workspaces():
    lib, n, one = _cabi.lib(), C.c_size_t(0), C.c_void_p(1 << 20)
    assert lib.plx_pages_workspace_bytes(8, 2, 0, C.byref(n)) == 0 and n.value > 0
    assert lib.plx_pages_compact(C.byref(c_pool()), one, one, 2, 4, one, one, one, n.value - 1, None) == -4
    assert lib.plx_pages_compact(C.byref(c_pool()), one, one, 2, 4, one, one, None, n.value, None) == -4
    assert lib.plx_pages_workspace_bytes(0, 2, 0, C.byref(n)) == -1
    assert lib.plx_pages_fork(C.byref(c_pool()), one, one, 2, 4, one, None, 1, one, one, one, one, 1 << 20, None) == -1
