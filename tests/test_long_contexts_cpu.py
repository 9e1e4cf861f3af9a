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


def test_gathered_pages_outside_the_pool_read_as_zeros():
    """-1 is what forking writes where there was no page, and an entry that no query sees may hold any number."""
    from parallax_b200.decode import _gathered

    pool = torch.randn(5, 2, 3, 8, requires_grad=True)
    pages = torch.tensor([4, -1, 0, 5, 2 ** 31 - 1, -2 ** 31, 3], dtype=torch.int32)
    got = _gathered(pool, pages)
    assert got.shape == (1, 14, 3, 8)
    for i, page in enumerate(pages.tolist()):
        want = pool[page] if 0 <= page < 5 else torch.zeros(2, 3, 8)
        assert torch.equal(got[0, 2 * i:2 * i + 2], want)
    got.sum().backward()
    assert torch.equal(pool.grad, torch.tensor([1., 0., 0., 1., 1.])[:, None, None, None].expand_as(pool))


@pytest.mark.parametrize("call", [
    lambda n: plx.parallax_func(z(1, 2, 8, 64), z(1, 2, 8, 64), z(1, 2, 8, 64), z(1, 2, 8, 64), window_size_left=4, sink_tokens=n),
    lambda n: plx.parallax_varlen_func(z(1, 8, 2, 64), z(1, 8, 2, 64), z(1, 8, 2, 64), z(1, 8, 2, 64), window_size_left=4, sink_tokens=n),
    lambda n: plx.parallax_fwd(z(2, 8, 64), z(2, 8, 64), z(2, 8, 64), z(2, 8, 64), 0.1, sink_tokens=n),
    lambda n: plx.parallax_bwd(*[z(2, 8, 64)] * 6, *[z(2, 8, 1)] * 3, z(2, 8, 64), 0.1, sink_tokens=n),
    lambda n: plx.parallax_decode(z(2, 1, 4, 64), z(2, 1, 4, 64), z(2, 8, 2, 64), z(2, 8, 2, 64), window_size_left=4, sink_tokens=n),
    lambda n: plx.parallax_attn_with_kvcache(z(2, 1, 4, 64), z(2, 1, 4, 64), z(2, 8, 2, 64), z(2, 8, 2, 64), window_size=4, sink_tokens=n),
    lambda n: plx.GraphedDecode(2, 4, 8, 64, window_size=4, sink_tokens=n),
], ids=["func", "varlen", "fwd", "bwd", "decode", "attn", "graphed"])
@pytest.mark.parametrize("sinks", [4.5, 0.5, float("nan"), float("inf"), -1, 2 ** 31])
def test_sinks_that_are_no_number_of_tokens(call, sinks):
    with pytest.raises(ValueError, match="sink_tokens must be a number of tokens"):
        call(sinks)


def plan(*a):                                                              # batch, heads_q, heads_kv, prefix, room for own keys, head_dim, SMs
    x, y = C.c_int32(-1), C.c_int32(-1)
    assert _cabi.lib().plx_decode_prefix_plan(*a, C.byref(x), C.byref(y)) == 0
    return x.value, y.value


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,hq,hkv,p", [(128, 32, 8, 32768), (32, 32, 8, 8192), (16, 8, 1, 16000), (16, 32, 8, 32768), (100, 28, 4, 5000), (64, 16, 2, 16000),
                                        (8, 8, 8, 4000), (12, 16, 16, 6000)])
def test_room_behind_a_prefix_is_not_taken_for_keys(b, hq, hkv, p, d):
    """A page table or a buffer is as wide as the longest row may grow: the prefix stays shared, in about as many parts as without room."""
    tight = plan(b, hq, hkv, p, 512, d, 148)[0]
    assert tight > 0
    for room in (1024, 2048, 8192, 65536, 131072 - p, 2 ** 31 - 1 - p):
        parts, own = plan(b, hq, hkv, p, room, d, 148)
        assert tight / 2 <= parts <= 2 * tight and 1 <= own <= 32, room


@pytest.mark.parametrize("b,hq,hkv,n", [(16, 32, 8, 32768), (4, 8, 8, 32768), (128, 32, 8, 32768), (2, 8, 1, 4096)])
def test_splits_where_there_is_no_shared_kernel(b, hq, hkv, n):
    """Every row sweeps the prefix itself there: its splits are those of a call of all keys, not those of its own ones beside a prefix."""
    room = 512

    def call(x, **kw):
        parts, own = C.c_int32(-1), C.c_int32(-1)
        p = decode_problem(batch=b, heads_q=hq, heads_kv=hkv, kv_stride_t=hkv * 128, **kw)
        assert _cabi.lib().plx_decode_prefix_plan_call(C.byref(p), C.byref(x), 148, C.byref(parts), C.byref(own)) == 0
        return parts.value, own.value

    def paged(page):
        return dict(page_table=1 << 20, page_size=page, pages_per_seq=(n + room) // page, n_pages=100, cache_len=n + room, kv_stride_b=page * hkv * 128)

    every = (0, _cabi.lib().plx_decode_choose_splits_gqa(b, hq, hkv, n + room, 148))
    shared = plan(b, hq, hkv, n, room, 128, 148)
    in_pages, own_tensors = prefix(k=None, v=None, len=n), prefix(len=n, stride_t=hkv * 128)
    for page in (1, 2, 4, 8, 64):
        assert call(in_pages, **paged(page)) == (every if page < 8 else shared)
    dense = dict(cache_len=room, kv_stride_b=room * hkv * 128)
    assert call(own_tensors, **dense) == shared
    for scale in (0.0, -0.1):
        assert call(own_tensors, qk_scale=scale, **dense) == call(in_pages, qk_scale=scale, **paged(64)) == every
    assert call(prefix(len=n, stride_t=0), **dense) == call(prefix(len=n, stride_t=hkv * 128, stride_h=0), **dense) == every


def test_plans_of_calls_that_are_refused():
    x, one = prefix(), C.c_int32(0)
    ask = lambda p, x, sms=148: _cabi.lib().plx_decode_prefix_plan_call(p, x, sms, C.byref(one), C.byref(one))         # noqa: E731
    assert ask(None, C.byref(x)) == ask(C.byref(decode_problem()), None) == ask(C.byref(decode_problem()), C.byref(x), 0) == -1
    assert ask(C.byref(decode_problem(window_left=4)), C.byref(x)) == -1 and ask(C.byref(decode_problem()), C.byref(prefix(len=0))) == -1
    assert ask(C.byref(decode_problem(**PAGED)), C.byref(x)) == ask(C.byref(decode_problem(head_dim=96)), C.byref(x)) == _cabi.PLX_ERR_UNSUPPORTED
    p = decode_problem(batch=65535)
    assert ask(C.byref(p), C.byref(x)) == 0 and one.value >= 1


def test_plans_that_are_kept():
    """A thread keeps its last plans: asked again, in any order and by any thread, each shape has its own."""
    from concurrent.futures import ThreadPoolExecutor

    shapes = [(b, hq, 8, p, room, d, sms) for b in (4, 32, 128) for hq in (8, 32) for p in (500, 8192) for room in (40, 512, 8192) for d in (64, 128) for sms in (74, 148)]
    first = [plan(*x) for x in shapes]
    assert len(set(first)) > 20
    assert [plan(*x) for x in reversed(shapes) for _ in range(2)][::2] == first[::-1]
    with ThreadPoolExecutor(4) as pool:
        for got in pool.map(lambda i: [plan(*x) for x in shapes[i:] + shapes[:i]], range(0, len(shapes), 9)):
            assert sorted(got) == sorted(first)


def test_lists_of_pages_that_are_too_long_for_their_indices():
    """Threads step through pages, entries and lists by the thousand in 32 bits: near 2^31 that would wrap around and read before the list."""
    from tests.test_pages_cpu import c_pool

    lib, one, most, n = _cabi.lib(), C.c_void_p(1 << 20), 1 << 30, C.c_size_t(0)
    refused, ws = _cabi.PLX_ERR_UNSUPPORTED, 1 << 60
    pool, big = C.byref(c_pool()), C.byref(c_pool(n_pages=most + 1))
    assert lib.plx_pages_copy(pool, one, one, most + 1, None) == lib.plx_pages_copy(big, one, one, 1, None) == refused
    for size in (most + 1, 2 ** 31 - 1):
        assert lib.plx_pages_fork(pool, one, one, 2, 4, one, one, size, one, one, one, one, ws, None) == refused
        assert lib.plx_pages_free(one, one, 2, 4, one, size, 8, 16, one, one, one, one, ws, None) == refused          # rows
        assert lib.plx_pages_free(one, one, 2, 4, one, 1, size, 16, one, one, one, one, ws, None) == refused          # pages
        assert lib.plx_pages_free(one, one, 1, size, one, 1, 8, 16, one, one, one, one, ws, None) == refused          # entries
        for sizes in ((size, 2, 0), (8, size, 0), (8, 2, size)):
            assert lib.plx_pages_workspace_bytes(*sizes, C.byref(n)) == refused
    assert lib.plx_pages_fork(big, one, one, 2, 4, one, one, 1, one, one, one, one, ws, None) == refused
    assert lib.plx_pages_compact(big, one, one, 2, 4, one, one, one, ws, None) == refused
    assert lib.plx_pages_workspace_bytes(most, 2, 0, C.byref(n)) == 0 and n.value > 16 * most


def test_what_freeing_needs():
    """A bitmap and ranks where they do not fit in shared memory, not the moves of a compaction."""
    lib, one, n = _cabi.lib(), C.c_void_p(1 << 20), C.c_size_t(1)
    for pages in (1, 8, 524288):
        assert lib.plx_pages_free_workspace_bytes(pages, C.byref(n)) == 0 and n.value == 0
    assert lib.plx_pages_free_workspace_bytes(1700000, C.byref(n)) == 0 and n.value == 2 * 4 * 53125 + 2 * 12       # (16-byte parts)
    free = lambda ws, size: lib.plx_pages_free(one, one, 2, 4, one, 1, 1700000, 16, one, one, one, ws, size, None)     # noqa: E731
    assert free(one, n.value - 1) == free(None, n.value) == free(C.c_void_p((1 << 20) + 4), n.value) == -4
    assert lib.plx_pages_free_workspace_bytes(0, C.byref(n)) == lib.plx_pages_free_workspace_bytes(8, None) == -1
    assert lib.plx_pages_free_workspace_bytes((1 << 30) + 1, C.byref(n)) == _cabi.PLX_ERR_UNSUPPORTED


def test_a_prefix_in_front_of_no_room_is_refused():
    with pytest.raises(ValueError, match="room for a key"):
        plx.parallax_decode_shared_prefix(z(2, 1, 4, 64), z(2, 1, 4, 64), z(16, 2, 64), z(16, 2, 64), z(2, 0, 2, 64), z(2, 0, 2, 64))
