"""Sinks and shared prefixes: what is refused before anything reaches a device, in Python and at the C ABI."""
import ctypes as C

import pytest
import torch

import parallax_b200 as plx
from parallax_b200 import _cabi

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


Q, KV, PRE = (2, 1, 4, 64), (2, 8, 2, 64), (16, 2, 64)


@pytest.mark.parametrize("call", [
    lambda: plx.parallax_func(z(1, 2, 8, 64), z(1, 2, 8, 64), z(1, 2, 8, 64), z(1, 2, 8, 64), window_size_left=4, sink_tokens=-1),
    lambda: plx.parallax_varlen_func(z(1, 8, 2, 64), z(1, 8, 2, 64), z(1, 8, 2, 64), z(1, 8, 2, 64), sink_tokens=-1),
    lambda: plx.parallax_fwd(z(2, 8, 64), z(2, 8, 64), z(2, 8, 64), z(2, 8, 64), 0.1, sink_tokens=-1),
    lambda: plx.parallax_decode(z(*Q), z(*Q), z(*KV), z(*KV), window_size_left=4, sink_tokens=2 ** 31),
    lambda: plx.parallax_attn_with_kvcache(z(*Q), z(*Q), z(*KV), z(*KV), window_size=4, sink_tokens=-2),
    lambda: plx.parallax_attn_with_kvcache(z(*Q), z(*Q), z(*KV), z(*KV), shared_prefix=8),
    lambda: plx.parallax_decode_shared_prefix(z(*Q), z(*Q), z(1, *PRE), z(1, *PRE), z(*KV), z(*KV)),
    lambda: plx.parallax_decode_shared_prefix(z(*Q), z(*Q), z(0, 2, 64), z(0, 2, 64), z(*KV), z(*KV)),
    lambda: plx.parallax_decode_shared_prefix(z(*Q), z(*Q), z(16, 4, 64), z(16, 4, 64), z(*KV), z(*KV)),
    lambda: plx.parallax_decode_shared_prefix(z(2, 2, 4, 64), z(2, 2, 4, 64), z(*PRE), z(*PRE), z(*KV), z(*KV)),
    lambda: plx.parallax_decode_shared_prefix(z(2, 1, 3, 64), z(2, 1, 3, 64), z(*PRE), z(*PRE), z(*KV), z(*KV)),
])
def test_values_refused(call):
    with pytest.raises(ValueError):
        call()


def test_types_and_devices_refused():
    with pytest.raises(TypeError):
        plx.parallax_decode_shared_prefix(z(*Q, dtype=torch.float32), z(*Q), z(*PRE), z(*PRE), z(*KV), z(*KV))
    with pytest.raises(TypeError):
        plx.parallax_decode_shared_prefix(z(*Q), z(*Q), z(*PRE, dtype=torch.float16), z(*PRE), z(*KV), z(*KV))
    with pytest.raises(NotImplementedError):
        plx.parallax_decode_shared_prefix(z(2, 1, 4, 32), z(2, 1, 4, 32), z(16, 2, 32), z(16, 2, 32), z(2, 8, 2, 32), z(2, 8, 2, 32))
    with pytest.raises(RuntimeError):
        plx.parallax_decode_shared_prefix(z(*Q), z(*Q), z(*PRE), z(*PRE), z(*KV), z(*KV))       # no CPU path


def train_problem(**kw):
    p = _cabi.TrainProblem()
    p.dtype, p.batch, p.heads_q, p.heads_kv, p.len_q, p.len_k, p.head_dim = 0, 1, 8, 8, 4096, 4096, 128
    p.window_left, p.qk_scale = 256, 0.088
    p.q_stride_b, p.q_stride_h, p.q_stride_t = 8 * 4096 * 128, 4096 * 128, 128
    p.kv_stride_b, p.kv_stride_h, p.kv_stride_t = 8 * 4096 * 128, 4096 * 128, 128
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def train_bytes(sinks, **kw):
    n = C.c_size_t(0)
    assert _cabi.lib().plx_train_workspace_bytes_sink(C.byref(train_problem(**kw)), sinks, C.byref(n)) == 0
    return n.value


def test_training_workspaces():
    plain = (8 * 4096 + 64) * 12 * 4
    assert train_bytes(0) == train_bytes(4, window_left=-1) == train_bytes(4, window_left=4096) == plain      # nothing is hidden
    part = 2 * 128 * 128 * 4
    assert train_bytes(4) == plain + 8 * 8 * part                          # 8 heads, 8 chunks of 512 rows, one tile of sinks
    assert train_bytes(129) == plain + 8 * 8 * 2 * part
    assert train_bytes(1100) == plain                                      # tiles of sinks enough
    assert train_bytes(4, len_q=512, len_k=512, window_left=64) == (8 * 512 + 64) * 12 * 4      # one chunk: none
    n = C.c_size_t(0)
    assert _cabi.lib().plx_train_workspace_bytes_sink(C.byref(train_problem()), -1, C.byref(n)) == -1
    one = C.c_void_p(1 << 20)
    p = train_problem()
    assert _cabi.lib().plx_train_fwd_sink(C.byref(p), -1, *[one] * 9, None) == -1
    args = [one] * 14
    assert _cabi.lib().plx_train_bwd_sink(C.byref(p), -1, *args, one, 1 << 30, None) == -1
    assert _cabi.lib().plx_train_bwd_sink(C.byref(p), 4, *args, one, plain, None) == -4          # room for the statistics only


def decode_problem(**kw):
    p = _cabi.DecodeProblem()
    p.dtype, p.batch, p.heads_q, p.heads_kv, p.cache_len, p.head_dim, p.window_left, p.n_splits = 0, 2, 8, 2, 64, 128, -1, 2
    p.qk_scale = 0.088
    p.kv_stride_b, p.kv_stride_t, p.kv_stride_h = 64 * 2 * 128, 2 * 128, 128
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def prefix(**kw):
    x = _cabi.Prefix()
    x.k = x.v = 1 << 20
    x.stride_t, x.stride_h, x.len, x.n_splits = 256, 128, 1000, 4
    for k, v in kw.items():
        setattr(x, k, v)
    return x


def test_decode_with_sinks_and_prefixes_at_the_abi():
    lib, one = _cabi.lib(), C.c_void_p(1 << 20)
    p = decode_problem(window_left=16)
    assert lib.plx_decode_sink(C.byref(p), -1, *[one] * 7, one, 1 << 20, None) == -1
    assert lib.plx_decode_step_sink(C.byref(p), -1, *[one] * 9, one, 1 << 20, None) == -1
    assert lib.plx_decode_sink(C.byref(decode_problem(head_dim=96)), 4, *[one] * 7, one, 1 << 20, None) == -2
    assert lib.plx_decode_sink(C.byref(p), 4, None, *[one] * 6, one, 1 << 20, None) == -1
    n = C.c_size_t(0)
    rec = (2 * 128 + 4) * 4
    q = decode_problem()
    base = C.c_size_t(0)
    assert lib.plx_decode_workspace_bytes(C.byref(q), C.byref(base)) == 0
    assert lib.plx_decode_prefix_workspace_bytes(C.byref(q), C.byref(prefix()), C.byref(n)) == 0 and n.value == base.value + 16 * 5 * rec
    assert lib.plx_decode_prefix_workspace_bytes(C.byref(q), C.byref(prefix(n_splits=0)), C.byref(n)) == 0 and n.value == base.value
    assert lib.plx_decode_prefix_workspace_bytes(C.byref(q), C.byref(prefix(n_splits=128)), C.byref(n)) == -1
    call = lambda p, x: lib.plx_decode_prefix(C.byref(p), C.byref(x), *[one] * 6, one, 1 << 20, None)       # noqa: E731
    assert call(decode_problem(dtype=9), prefix()) == -2
    for x in (prefix(len=0), prefix(n_splits=17), prefix(n_splits=-1), prefix(v=None), prefix(k=(1 << 20) + 2), prefix(stride_t=100), prefix(stride_h=-8),
              prefix(k=None, v=None)):                                      # the last: in the pages of a cache that has none
        assert call(decode_problem(), x) == -1
    assert call(decode_problem(window_left=8), prefix()) == -1
    paged = dict(page_table=1 << 20, page_size=16, pages_per_seq=80, n_pages=100, cache_len=1280)
    for x in (prefix(k=None), prefix(k=None, v=None, len=1001), prefix(k=None, v=None, len=1296, n_splits=1)):
        assert call(decode_problem(**paged), x) == -1


def test_how_a_prefix_is_split():
    def plan(*a):                                                          # batch, heads_q, heads_kv, prefix, own keys, head_dim, SMs
        x, y = C.c_int32(-1), C.c_int32(-1)
        assert _cabi.lib().plx_decode_prefix_plan(*a, C.byref(x), C.byref(y)) == 0
        return x.value, y.value

    assert plan(4, 8, 8, 500, 40, 128, 148)[0] == 0 and plan(4, 8, 8, 1000, 40, 128, 148)[0] == 0      # every row by itself, in one launch
    assert plan(1, 32, 8, 4000, 40, 128, 148)[0] == 0
    assert 1 <= plan(16, 8, 8, 500, 40, 128, 148)[0] <= 8                  # at most one part for 64 keys
    wide, own = plan(32, 32, 8, 8192, 512, 128, 148)
    assert 8 <= wide <= 12 and own >= 1                                    # leaves SMs to the rows' own keys
    assert 16 <= plan(32, 32, 8, 32768, 0, 128, 148)[0] <= 18              # where there are some
    assert plan(128, 32, 8, 32768, 512, 128, 148)[0] == 4                  # one round of the SMs
    for b, hq, hkv, n, t in ((1, 1, 1, 1, 0), (300, 64, 8, 100000, 10), (64, 8, 1, 64, 3), (64, 128, 1, 65, 70), (10 ** 4, 32, 8, 10 ** 6, 10 ** 6)):
        parts, own = plan(b, hq, hkv, n, t, 128, 148)
        assert 0 <= parts <= min(127, -(-n // 64)) and 1 <= own <= 256
    one = C.c_int32(0)
    for bad in ((0, 8, 8, 9, 0, 128, 148), (1, 4, 8, 9, 0, 128, 148), (1, 9, 2, 9, 0, 128, 148), (1, 8, 8, 0, 0, 128, 148), (1, 8, 8, 9, -1, 128, 148)):
        assert _cabi.lib().plx_decode_prefix_plan(*bad, C.byref(one), C.byref(one)) == -1
