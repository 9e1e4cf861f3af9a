"""Sliding window with sinks on the GPU, against the definition in 64 bits.

Tolerances (relative 2-norm), in halves of a step of the 16-bit type: one for the rounding of the result, one for that of the
weights which multiply v (or k, q, r, dO), and for gradients one more for o and bar v, which the forward leaves in 16 bits.
"""
import contextlib
import gc

import pytest
import torch

import parallax_b200 as plx

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@contextlib.contextmanager
def no_collection():
    """No garbage collection inside: a graph that it destroys during a capture ends the capture."""
    gc.disable()
    try:
        yield
    finally:
        gc.enable()


def half_steps(dtype, n):
    return n * torch.finfo(dtype).eps / 2


def close(got, want, n, what):
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    off, norm = (got.double() - want).norm().item(), want.norm().item()
    # (where everything cancels, the terms that do are of the order of one each)
    assert off <= half_steps(got.dtype, n) * max(norm, 0.05 * want.numel() ** 0.5), (what, off / max(norm, 1e-30))


def visible(nq, nk, window, sinks, device="cuda"):
    i = torch.arange(nq, device=device)[:, None] + nk - nq
    j = torch.arange(nk, device=device)[None]
    return (j <= i) & ((j > i - window) | (j < sinks)) if window >= 0 else j <= i


def attend(q, r, k, v, ok, scale):
    """(.., n_q, D), (.., n_k, D) in 64 bits -> o; rows that see nothing: 0"""
    s1 = (q @ k.transpose(-1, -2) * scale).masked_fill(~ok, -torch.inf)
    any_key = ok.any(-1, keepdim=True)
    p = torch.softmax(torch.where(any_key, s1, torch.zeros_like(s1)), -1) * any_key
    s2 = r @ k.transpose(-1, -2)
    mean = p @ v
    return mean + (p * s2).sum(-1, keepdim=True) * mean - (p * s2) @ v


def randn(*shape, dtype=BF, scale=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def inputs(b, hq, hkv, nq, nk, d, dtype, seed=1):
    return (randn(b, hq, nq, d, dtype=dtype, seed=seed), randn(b, hq, nq, d, dtype=dtype, scale=0.5, seed=seed + 1),
            randn(b, hkv, nk, d, dtype=dtype, seed=seed + 2), randn(b, hkv, nk, d, dtype=dtype, seed=seed + 3))


def reference(q, r, k, v, go, window, sinks, scale=None, cu=None):
    """o and the four gradients, (B, H, L, D) in 64 bits"""
    rep = q.shape[1] // k.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    leaves = [x.detach().double().requires_grad_() for x in (q, r, k, v)]
    qq, rr, kk, vv = leaves
    kk, vv = kk.repeat_interleave(rep, 1), vv.repeat_interleave(rep, 1)
    nq, nk = q.shape[2], k.shape[2]
    ok = visible(nq, nk, window, sinks)
    if cu is not None:
        ok = torch.zeros(nq, nk, dtype=torch.bool, device=q.device)
        for x, y in zip(cu, cu[1:]):
            ok[x:y, x:y] = visible(y - x, y - x, window, sinks)
    o = attend(qq, rr, kk, vv, ok, scale)
    return [o.detach()] + [g for g in torch.autograd.grad(o, leaves, go.double())]


def run(q, r, k, v, go, fn):
    leaves = [x.detach().requires_grad_() for x in (q, r, k, v)]
    o = fn(*leaves)
    return [o.detach()] + list(torch.autograd.grad(o, leaves, go))


def check(got, want):
    for name, x, y, n in zip(("o", "dq", "dr", "dk", "dv"), got, want, (2, 3, 3, 3, 3)):
        close(x, y, n, name)


# b, hq, hkv, nq, nk, d, dtype, window, sinks
TRAIN = [
    (1, 2, 2, 1, 1, 64, BF, 1, 1),                # one token
    (2, 2, 2, 70, 70, 128, BF, 5, 3),
    (1, 2, 1, 200, 200, 64, FP, 16, 1),           # grouped heads
    (2, 4, 2, 300, 300, 128, FP, 64, 64),         # sinks that end with a tile
    (1, 2, 2, 333, 333, 128, BF, 100, 130),       # sinks in a second tile of keys
    (1, 2, 2, 500, 500, 64, BF, 96, 70),
    (1, 3, 3, 129, 129, 128, BF, 128, 1),         # the window just longer than what it hides
    (1, 2, 2, 256, 256, 64, BF, 1, 4),            # a window of the row itself
    (1, 2, 2, 200, 200, 128, BF, 0, 4),           # nothing but sinks
    (1, 2, 2, 200, 200, 64, FP, 0, 1),
    (1, 2, 2, 150, 150, 64, BF, 40, 400),         # more sinks than tokens
    (1, 2, 2, 150, 150, 64, BF, 400, 4),          # a window that hides nothing
    (1, 2, 2, 64, 300, 128, BF, 50, 10),          # rows at the end of longer keys
    (1, 4, 2, 300, 700, 64, FP, 33, 5),
    (1, 2, 2, 200, 90, 128, BF, 20, 3),           # rows before any key
    (1, 2, 2, 700, 700, 128, BF, 64, 4),          # sinks' gradients in chunks
    (2, 4, 2, 1700, 1700, 64, BF, 100, 4),
    (1, 4, 1, 1537, 1537, 128, FP, 40, 200),      # two tiles of sinks in chunks
    (1, 2, 2, 1300, 2000, 128, BF, 30, 17),
    (1, 1, 1, 2200, 1500, 64, BF, 300, 4),
    (1, 2, 2, 2100, 2100, 128, BF, 1024, 6),
    (9, 16, 16, 700, 700, 64, BF, 350, 4),        # many heads
    (2, 2, 1, 1500, 1500, 64, FP, 20, 1100),      # tiles of sinks enough without chunks
]


@pytest.mark.parametrize("case", TRAIN, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
def test_dense(case):
    b, hq, hkv, nq, nk, d, dtype, window, sinks = case
    q, r, k, v = inputs(b, hq, hkv, nq, nk, d, dtype)
    go = randn(b, hq, nq, d, dtype=dtype, seed=9)
    got = run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, window_size_left=window, sink_tokens=sinks))
    check(got, reference(q, r, k, v, go, window, sinks))
    again = run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, window_size_left=window, sink_tokens=sinks))
    assert all(torch.equal(x, y) for x, y in zip(got, again))


# cu, hq, hkv, d, dtype, window, sinks
PACKED = [
    ([0, 1, 2, 90, 90, 218, 500], 2, 2, 64, BF, 20, 4),
    ([0, 700, 701, 1500, 2300], 4, 2, 128, BF, 64, 4),
    ([0, 513, 1025, 1600, 1601], 2, 1, 64, FP, 30, 140),
    ([0, 0, 0, 2000], 2, 2, 128, FP, 100, 1),
    ([0] + [37 * i for i in range(1, 50)], 2, 2, 128, BF, 8, 2),
]


@pytest.mark.parametrize("case", PACKED, ids=lambda c: f"{len(c[0]) - 1}seqs-{c[0][-1]}-" + "-".join(str(x).replace("torch.", "") for x in c[1:]))
@pytest.mark.parametrize("ints", [torch.int32, torch.int64])
def test_packed(case, ints):
    cu, hq, hkv, d, dtype, window, sinks = case
    n = cu[-1]
    q, r, k, v = (x.transpose(1, 2).contiguous() for x in inputs(1, hq, hkv, n, n, d, dtype))
    go = randn(1, n, hq, d, dtype=dtype, seed=9)
    offsets = torch.tensor(cu, dtype=ints, device="cuda")
    got = run(q, r, k, v, go, lambda *x: plx.parallax_varlen_func(*x, window_size_left=window, cu_seqlens=offsets, sink_tokens=sinks))
    want = reference(*(x.transpose(1, 2) for x in (q, r, k, v, go)), window, sinks, cu=cu)
    check([x.transpose(1, 2) for x in got], want)


def test_without_a_window_or_sinks_it_is_the_call_without():
    q, r, k, v = inputs(1, 4, 2, 600, 600, 128, BF)
    go = randn(1, 4, 600, 128, seed=9)
    plain = run(q, r, k, v, go, lambda *x: plx.parallax_func(*x))
    for window in (-1, 600, 10 ** 9):
        got = run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, window_size_left=window, sink_tokens=7))
        want = plain if window < 0 else run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, window_size_left=window))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("scale", [-0.1, 0.3])
@pytest.mark.parametrize("n,window,sinks", [(150, 20, 3), (700, 64, 4), (200, 0, 2)])
def test_scales(scale, n, window, sinks):
    q, r, k, v = inputs(1, 4, 2, n, n, 64, BF)
    go = randn(1, 4, n, 64, seed=9)
    got = run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, qk_scale=scale, window_size_left=window, sink_tokens=sinks))
    check(got, reference(q, r, k, v, go, window, sinks, scale=scale))


def test_views_and_streams():
    """Heads-last views, a slice of longer keys, and a stream of its own."""
    b, h, n, d, window, sinks = 2, 4, 650, 128, 50, 5
    q, r, go = (randn(b, n, h, d, seed=s).transpose(1, 2) for s in (1, 2, 3))
    k, v = (randn(b, n + 30, h, d, seed=s)[:, :n].transpose(1, 2) for s in (4, 5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, window_size_left=window, sink_tokens=sinks))
    torch.cuda.current_stream().wait_stream(side)
    check(got, reference(q, r, k, v, go, window, sinks))


def test_gradients_against_differences():
    """The directional derivative of <o, dO> in 64 bits by central differences, in all four inputs at once."""
    window, sinks, n = 60, 4, 900
    q, r, k, v = inputs(1, 2, 1, n, n, 64, BF)
    go = randn(1, 2, n, 64, seed=9)
    grads = run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, window_size_left=window, sink_tokens=sinks))[1:]
    ways = [randn(*x.shape, dtype=torch.float64, seed=20 + i) for i, x in enumerate((q, r, k, v))]
    ok, h = visible(n, n, window, sinks), 1e-5

    def loss(step):
        qq, rr, kk, vv = (x.double() + step * w for x, w in zip((q, r, k, v), ways))
        return (attend(qq, rr, kk.repeat_interleave(2, 1), vv.repeat_interleave(2, 1), ok, 64 ** -0.5) * go.double()).sum().item()

    want = (loss(h) - loss(-h)) / (2 * h)
    got = sum((g.double() * w).sum().item() for g, w in zip(grads, ways))
    # the directions are independent of the errors: these add up like a random walk over the elements
    bound = 4 * half_steps(BF, 3) * sum(g.double().norm().item() ** 2 for g in grads) ** 0.5
    assert abs(got - want) <= bound, (got, want, bound)


def test_raw_forward_and_backward():
    """parallax_fwd / parallax_bwd: heads folded into the batch axis."""
    window, sinks, n, d = 70, 4, 700, 64
    q, r, k, v = inputs(1, 4, 2, n, n, d, BF)
    go = randn(1, 4, n, d, seed=9)
    flat = lambda x: x.reshape(-1, n, d)                                                                   # noqa: E731
    saved = plx.parallax_fwd(flat(q), flat(r), flat(k), flat(v), d ** -0.5, 2, window, sinks)
    grads = plx.parallax_bwd(flat(q), flat(r), flat(k), flat(v), *saved, flat(go), d ** -0.5, 2, window, sinks)
    check([saved[0].view_as(q), *(g.view_as(x) for g, x in zip(grads, (q, r, k, v)))], reference(q, r, k, v, go, window, sinks))


def test_captured_training_step():
    window, sinks, n = 40, 4, 800
    q, r, k, v = (x.requires_grad_() for x in inputs(1, 2, 2, n, n, 64, BF))
    go = randn(1, 2, n, 64, seed=9)

    def step():
        o = plx.parallax_func(q, r, k, v, window_size_left=window, sink_tokens=sinks)
        return (o.detach(), *torch.autograd.grad(o, (q, r, k, v), go))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with no_collection(), torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        q.copy_(randn(*q.shape, seed=31))
    graph.replay()
    torch.cuda.synchronize()
    check(out, reference(q, r, k, v, go, window, sinks))


# --------------------------------------------------------------------------- #
# against a cache
# --------------------------------------------------------------------------- #
def decode_reference(q, r, k, v, lens, starts, window, sinks, scale=None):
    out = torch.zeros_like(q, dtype=torch.float64)
    rep = q.shape[2] // k.shape[2]
    for b in range(q.shape[0]):
        n, c = lens[b], starts[b]
        kk, vv = (x[b, c:n].double().transpose(0, 1).repeat_interleave(rep, 0) for x in (k, v))
        ok = visible(q.shape[1], n - c, window, sinks)
        o = attend(q[b].double().transpose(0, 1), r[b].double().transpose(0, 1), kk, vv, ok, q.shape[3] ** -0.5 if scale is None else scale)
        out[b] = o.transpose(0, 1)
    return out


def hide(k, lens, starts, window, sinks, lq=1):
    """NaN in every key that no row may see"""
    k = k.clone()
    for b, (n, c) in enumerate(zip(lens, starts)):
        at = torch.arange(k.shape[1], device=k.device)
        seen = (at >= c) & (at < n) & ((at > n - lq - window) | (at < c + sinks))
        k[b, ~seen] = torch.nan
    return k


def paged(k, v, page, seed=3):
    """The same keys in pages: pools, table"""
    b, t, h, d = k.shape
    m = -(-t // page)
    order = torch.randperm(b * m + 3, generator=torch.Generator().manual_seed(seed))[:b * m].to("cuda")
    pools = []
    for x in (k, v):
        pool = torch.full((b * m + 3, page, h, d), torch.nan, dtype=x.dtype, device="cuda")
        full = torch.full((b, m * page, h, d), torch.nan, dtype=x.dtype, device="cuda")
        full[:, :t] = x
        pool[order] = full.view(b * m, page, h, d)
        pools.append(pool)
    return (*pools, order.view(b, m).to(torch.int32))


# hq, hkv, d, dtype, cache length, window, sinks, lengths
DECODE = [
    (8, 8, 128, BF, 1000, 100, 4, [1000]),                          # splits of a CTA, a cluster
    (8, 8, 64, FP, 4000, 700, 33, [4000, 900, 3333]),
    (4, 4, 128, BF, 300, 20, 3, [1, 2, 23, 24, 25, 300]),           # around the first hidden key
    (1, 1, 64, BF, 500, 64, 16, [500, 80, 81, 79] * 20),
    (2, 2, 128, FP, 2000, 600, 5, [2000, 700] * 40),                # one warp per split
    (12, 12, 64, BF, 1500, 333, 200, [1500, 100, 600] * 12),
    (16, 16, 128, BF, 900, 0, 4, [900, 3, 4, 5, 1]),                # nothing but sinks
    (8, 8, 128, BF, 700, 0, 1, [700] * 9),
    (8, 2, 128, BF, 1000, 100, 4, [1000, 99, 104, 105, 1]),         # grouped heads
    (32, 8, 128, BF, 3000, 1000, 64, [3000, 1064, 1065, 2000]),
    (16, 2, 64, FP, 777, 130, 17, [777, 147, 148, 5, 400]),
    (24, 1, 128, BF, 900, 77, 9, [900, 85, 86, 87, 500]),           # more than 16 heads
    (20, 2, 64, BF, 640, 64, 16, [640, 80, 81, 333]),
    (16, 4, 128, FP, 600, 0, 20, [600, 20, 21, 7]),
    (8, 4, 64, BF, 500, 50, 1000, [500, 60]),                       # more sinks than keys
    (8, 4, 64, BF, 500, 499, 1, [500, 499, 498]),
    (8, 8, 64, BF, 500, 499, 1, [500, 499, 498]),
]


@pytest.mark.parametrize("case", DECODE, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:7]))
@pytest.mark.parametrize("page", [0, 1, 8, 64])
def test_decode(case, page):
    hq, hkv, d, dtype, t, window, sinks, lens = case
    b = len(lens)
    q, r = randn(b, 1, hq, d, dtype=dtype, seed=1), randn(b, 1, hq, d, dtype=dtype, scale=0.5, seed=2)
    k, v = randn(b, t, hkv, d, dtype=dtype, seed=3), randn(b, t, hkv, d, dtype=dtype, seed=4)
    want = decode_reference(q, r, k, v, lens, [0] * b, window, sinks)
    k, v = hide(k, lens, [0] * b, window, sinks), hide(v, lens, [0] * b, window, sinks)
    seqused = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if page:
        kp, vp, table = paged(k, v, page)
        got = plx.parallax_attn_with_kvcache(q, r, kp, vp, page_table=table, seqused_k=seqused, window_size=window, sink_tokens=sinks)
    else:
        got = plx.parallax_decode(q, r, k, v, window_size_left=window, seqused_k=seqused, sink_tokens=sinks)
    close(got, want, 2, "o")


@pytest.mark.parametrize("hq,hkv", [(8, 8), (4, 4), (16, 4), (17, 1)])
@pytest.mark.parametrize("window,sinks", [(50, 4), (0, 7), (120, 16), (300, 2)])
def test_decode_behind_padding(hq, hkv, window, sinks):
    t, d = 400, 128
    starts, lens = [0, 1, 17, 100, 390, 399, 64], [400, 300, 90, 260, 400, 400, 300]
    b = len(lens)
    q, r = randn(b, 1, hq, d, seed=1), randn(b, 1, hq, d, scale=0.5, seed=2)
    k, v = randn(b, t, hkv, d, seed=3), randn(b, t, hkv, d, seed=4)
    want = decode_reference(q, r, k, v, lens, starts, window, sinks)
    k, v = hide(k, lens, starts, window, sinks), hide(v, lens, starts, window, sinks)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")            # noqa: E731
    got = plx.parallax_decode(q, r, k, v, window_size_left=window, seqused_k=ints(lens), cache_start=ints(starts), sink_tokens=sinks)
    close(got, want, 2, "o")


@pytest.mark.parametrize("hq,hkv,d,page,t,lq,window,sinks", [
    (4, 4, 128, 0, 500, 17, 60, 4), (8, 2, 64, 0, 900, 200, 0, 3), (8, 2, 128, 16, 640, 64, 100, 70), (4, 1, 64, 64, 700, 130, 33, 5),
    (2, 2, 64, 128, 1500, 3, 128, 130), (8, 8, 128, 32, 2048, 300, 256, 4)])
def test_extend(hq, hkv, d, page, t, lq, window, sinks):
    lens = [t, max(lq, t // 2 + 1), lq]
    b = len(lens)
    q, r = randn(b, lq, hq, d, seed=1), randn(b, lq, hq, d, scale=0.5, seed=2)
    k, v = randn(b, t, hkv, d, seed=3), randn(b, t, hkv, d, seed=4)
    want = decode_reference(q, r, k, v, lens, [0] * b, window, sinks)
    k, v = hide(k, lens, [0] * b, window, sinks, lq), hide(v, lens, [0] * b, window, sinks, lq)
    seqused = torch.tensor(lens, dtype=torch.int32, device="cuda")
    table = None
    if page:
        k, v, table = paged(k, v, page)
    got = plx.parallax_attn_with_kvcache(q, r, k, v, page_table=table, seqused_k=seqused, window_size=window, sink_tokens=sinks)
    close(got, want, 2, "o")


def test_extend_over_pages_that_are_too_small_for_a_tile():
    """Pages of fewer than 8 keys: gathered row by row, and run as a dense problem of the training forward."""
    t, lq, window, sinks, lens = 300, 9, 20, 2, [300, 151, 9]
    q, r = randn(3, lq, 4, 128, seed=1), randn(3, lq, 4, 128, scale=0.5, seed=2)
    k, v = randn(3, t, 2, 128, seed=3), randn(3, t, 2, 128, seed=4)
    want = decode_reference(q, r, k, v, lens, [0] * 3, window, sinks)
    k, v, table = paged(k, v, 4)
    got = plx.parallax_attn_with_kvcache(q, r, k, v, page_table=table, seqused_k=torch.tensor(lens, dtype=torch.int32, device="cuda"), window_size=window,
                                         sink_tokens=sinks)
    close(got, want, 2, "o")


@pytest.mark.parametrize("lens", [[300, 151, 9], [300, 300, 300]])
@pytest.mark.parametrize("page", [0, 1, 2, 4])
def test_extend_without_its_own_kernel_sees_nothing_hidden(page, lens):
    """Pages of fewer than 8 keys, and dense rows whose channels are not next to one another."""
    t, lq, window, sinks = 300, 9, 20, 2
    q, r = randn(3, lq, 4, 128, seed=1), randn(3, lq, 4, 128, scale=0.5, seed=2)
    k, v = randn(3, t, 2, 128, seed=3), randn(3, t, 2, 128, seed=4)
    want = decode_reference(q, r, k, v, lens, [0] * 3, window, sinks)
    k, v = hide(k, lens, [0] * 3, window, sinks, lq), hide(v, lens, [0] * 3, window, sinks, lq)
    table = None
    if page:
        k, v, table = paged(k, v, page)
    else:
        k, v = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    before = k.clone(), v.clone()
    got = plx.parallax_attn_with_kvcache(q, r, k, v, page_table=table, seqused_k=torch.tensor(lens, dtype=torch.int32, device="cuda"), window_size=window,
                                         sink_tokens=sinks)
    close(got, want, 2, "o")
    assert all(torch.equal(x.view(torch.int16), y.view(torch.int16)) for x, y in zip((k, v), before))      # (bits: there are NaN)


@pytest.mark.parametrize("hq,hkv", [(8, 8), (16, 4)])
def test_graphed_decode(hq, hkv):
    b, t, d, window, sinks = 3, 700, 128, 90, 4
    gd = plx.GraphedDecode(b, hq, t, d, H_kv=hkv, window_size=window, sink_tokens=sinks)
    k, v = randn(b, t, hkv, d, seed=3), randn(b, t, hkv, d, seed=4)
    for step, lens in enumerate(([700, 95, 93], [1, 94, 400], 650)):
        q, r = randn(b, 1, hq, d, seed=10 + step), randn(b, 1, hq, d, scale=0.5, seed=20 + step)
        got = gd(q=q, r=r, k=k if step == 0 else None, v=v if step == 0 else None, cache_seqlens=lens).clone()
        want = decode_reference(q, r, k, v, [lens] * b if isinstance(lens, int) else lens, [0] * b, window, sinks)
        close(got, want, 2, "step")
        close(gd.replay().clone(), want, 2, "replay")


def test_graphs_that_are_garbage_do_not_end_a_capture():
    """A GraphedDecode made while the collector would run at every allocation and find an older one."""
    def litter():
        old = plx.GraphedDecode(1, 4, 64, 64)
        old.itself = old

    gc.collect()
    before = gc.get_threshold()
    litter()
    try:
        gc.set_threshold(1, 1, 1)
        gd = plx.GraphedDecode(1, 8, 300, 64, window_size=50, sink_tokens=2)
    finally:
        gc.set_threshold(*before)
    assert gc.isenabled() and torch.isfinite(gd.replay()).all()


def test_two_captured_calls_do_not_share_a_workspace():
    b, h, t, d, window, sinks = 2, 8, 3000, 128, 1000, 4
    calls, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        q, r = randn(b, 1, h, d, seed=i), randn(b, 1, h, d, scale=0.5, seed=i + 2)
        k, v = randn(b, t, h, d, seed=i + 4), randn(b, t, h, d, seed=i + 6)
        plx.parallax_decode(q, r, k, v, window_size_left=window, sink_tokens=sinks)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with no_collection(), torch.cuda.graph(graph):
            out = plx.parallax_decode(q, r, k, v, window_size_left=window, sink_tokens=sinks)
        calls.append((graph, out, decode_reference(q, r, k, v, [t] * b, [0] * b, window, sinks), (q, r, k, v)))     # (the inputs stay alive)
    torch.cuda.synchronize()
    for _ in range(20):
        for stream, (graph, *_) in zip(streams, calls):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in calls:
        close(out, want, 2, "o")


def test_refusals():
    q, r, k, v = inputs(1, 2, 2, 8, 8, 64, BF)
    x, cache = q.transpose(1, 2)[:, :1].contiguous(), k.transpose(1, 2).contiguous()
    for call in (lambda: plx.parallax_func(q, r, k, v, window_size_left=4, sink_tokens=-1),
                 lambda: plx.parallax_varlen_func(q, r, k, v, window_size_left=4, sink_tokens=-1),
                 lambda: plx.parallax_decode(x, x, cache, cache, window_size_left=4, sink_tokens=-1),
                 lambda: plx.parallax_attn_with_kvcache(x, x, cache, cache, window_size=4, sink_tokens=2 ** 31),
                 lambda: plx.GraphedDecode(1, 2, 8, 64, window_size=4, sink_tokens=-3)):
        with pytest.raises(ValueError):
            call()
