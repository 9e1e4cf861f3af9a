"""Sinks, shared prefixes and pages on the GPU: calls at the edges of what they document, against the definition in 64 bits."""
import pytest
import torch

import parallax_b200 as plx
from parallax_b200 import _cabi, ops
from tests.test_prefix_gpu import make, pages_of, reference
from tests.test_sinks_gpu import check, close, decode_reference, hide, inputs, paged, randn, run
from tests.test_sinks_gpu import reference as train_reference

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("nowhere", [-1, 10 ** 6])
@pytest.mark.parametrize("page,recorded,scale", [(2, False, None), (4, False, None), (16, True, None), (16, False, -0.1), (16, False, None)])
def test_extend_over_a_table_without_its_hidden_pages(page, recorded, scale, nowhere):
    """Pages between the sinks and the first window are somebody else's, and their entries no pages at all: by the gathered way (tiny
    pages, a call that autograd records, scales <= 0) as by the launch for all rows (the last)."""
    t, lq, window, sinks, lens = 300, 9, 20, 2, [300, 151, 9]
    q, r = randn(3, lq, 4, 128, seed=1), randn(3, lq, 4, 128, scale=0.5, seed=2)
    k, v = randn(3, t, 2, 128, seed=3), randn(3, t, 2, 128, seed=4)
    want = decode_reference(q, r, k, v, lens, [0] * 3, window, sinks, scale)
    k, v = hide(k, lens, [0] * 3, window, sinks, lq), hide(v, lens, [0] * 3, window, sinks, lq)
    k, v, table = paged(k, v, page)
    for b, n in enumerate(lens):
        first, last = -(-sinks // page), max(n - lq - window + 1, 0) // page          # wholly hidden pages
        table[b, first:max(first, last)] = nowhere
    got = plx.parallax_attn_with_kvcache(q.requires_grad_(recorded), r, k, v, page_table=table, seqused_k=ints(lens), window_size=window,
                                         sink_tokens=sinks, scale=scale)
    close(got.detach(), want, 2, "o")
    if recorded:
        dq, = torch.autograd.grad(got, q, torch.ones_like(got))
        assert torch.isfinite(dq).all() and dq.abs().max() > 0
    assert _cabi.device_error() == 0


@pytest.mark.parametrize("hq,hkv,d,p,room,page", [(32, 8, 128, 2048, 20000, 0), (32, 8, 128, 2048, 20000, 16), (8, 8, 64, 3000, 9000, 0), (8, 1, 128, 4096, 6000, 64),
                                                  (8, 8, 128, 2048, 3000, 2), (16, 4, 64, 640, 1500, 1)])
def test_a_prefix_in_front_of_rows_with_room(hq, hkv, d, p, room, page):
    """Buffers and tables many times as wide as what the rows hold, of which all but that is NaN or no page."""
    lens = [300, 0, 1, 77, 2, 900, 64, 65]
    b = len(lens)
    q, r, kp, vp, k, v = make(b, hq, hkv, d, BF, p, max(lens))
    want = reference(q, r, [torch.cat((kp, k[i, :n])) for i, n in enumerate(lens)], [torch.cat((vp, v[i, :n])) for i, n in enumerate(lens)])
    if page:
        pools_k, pools_v, table = pages_of(kp, vp, k, v, lens, page)
        table = torch.nn.functional.pad(table, (0, room // page), value=-1)
        call = lambda: plx.parallax_attn_with_kvcache(q, r, pools_k, pools_v, page_table=table, seqused_k=ints([p + n for n in lens]), shared_prefix=p)  # noqa: E731
    else:
        wide = [torch.full((b, room, hkv, d), torch.nan, dtype=BF, device="cuda") for _ in range(2)]
        for x, y in zip(wide, (k, v)):
            for i, n in enumerate(lens):
                x[i, :n] = y[i, :n]
        call = lambda: plx.parallax_decode_shared_prefix(q, r, kp, vp, *wide, seqused_k=ints(lens))        # noqa: E731
    got = call()
    close(got, want, 2, "o")
    assert torch.equal(call(), got) and _cabi.device_error() == 0


@pytest.mark.parametrize("dtype,d", [(BF, 64), (BF, 128), (FP, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 1), (0, 2), (2, 1), (1, 2)])
def test_rows_of_two_keys(window, sinks, dtype, d):
    """Every row but the first sees two keys (or three at most): where the gradients of q and r are differences of two terms, to the
    tolerances of any other window."""
    q, r, k, v = inputs(2, 4, 2, 500, 500, d, dtype)
    go = randn(2, 4, 500, d, dtype=dtype, seed=9)
    step = lambda: run(q, r, k, v, go, lambda *x: plx.parallax_func(*x, window_size_left=window, sink_tokens=sinks))                   # noqa: E731
    got = step()
    check(got, train_reference(q, r, k, v, go, window, sinks))
    assert all(torch.equal(x, y) for x, y in zip(got, step())) and _cabi.device_error() == 0


@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 128), (16, 4, 64)])
def test_a_prefix_cut_out_of_wider_tensors(hq, hkv, d):
    """Prefix and own keys whose tokens lie further apart than a token is long, by the call and by every way to split."""
    p, lens = 700, [60, 0, 17, 1]
    q, r, kp, vp, k, v = make(4, hq, hkv, d, BF, p, 60)
    want = reference(q, r, [torch.cat((kp, k[i, :n])) for i, n in enumerate(lens)], [torch.cat((vp, v[i, :n])) for i, n in enumerate(lens)])
    heads = lambda x: torch.cat((torch.full_like(x, torch.nan), x, torch.full_like(x, torch.nan)), -2)[..., hkv:2 * hkv, :]           # noqa: E731
    channels = lambda x: torch.cat((x, torch.full_like(x, torch.nan)), -1)[..., :d]                                                  # noqa: E731
    for wide in (heads, channels):
        cut = [wide(x) for x in (kp, vp, k, v)]
        assert all(x.stride() != y.stride() and torch.equal(x, y) for x, y in zip(cut, (kp, vp, k, v)))
        assert cut[0].stride(0) > hkv * d
        close(plx.parallax_decode_shared_prefix(q, r, *cut, seqused_k=ints(lens)), want, 2, "o")
        for splits in (0, 1, 7):
            for own in (1, 3):
                out, ws = torch.empty_like(q), torch.zeros(ops.decode_prefix_workspace_bytes(q, cut[2], own, splits, None) // 4, device="cuda")
                ops.decode_prefix(q, r, cut[0], cut[1], p, cut[2], cut[3], out, ws, d ** -0.5, own, splits, ints(lens), None)
                close(out, want, 2, (splits, own))
    assert _cabi.device_error() == 0


def test_prefixes_on_two_streams_at_once():
    """Calls of one shape that overlap on the device have workspaces of their own, and read what their own stream wrote before."""
    p, t, b = 3000, 200, 24
    sets = [make(b, 16, 4, 128, BF, p, t, seed=10 * i + 1) for i in range(2)]
    lens = [[(i * 7 + j) % (t + 1) for i in range(b)] for j in range(2)]
    want = [plx.parallax_decode_shared_prefix(*x, seqused_k=ints(n)) for x, n in zip(sets, lens)]
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    held = [ints(n) for n in lens]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                q = sets[i][0] * 1                                  # made on this stream, right before
                got[i].append(plx.parallax_decode_shared_prefix(q, *sets[i][1:], seqused_k=held[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for xs, y in zip(got, want) for x in xs) and _cabi.device_error() == 0


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_calls(backend):
    """Training with sinks and the page calls inside torch.compile: the same bits as outside."""
    q, r, k, v = inputs(1, 4, 2, 700, 700, 64, BF)
    go = randn(1, 4, 700, 64, seed=9)
    step = lambda *x: plx.parallax_func(*x, window_size_left=64, sink_tokens=4)                     # noqa: E731
    torch._dynamo.reset()
    assert all(torch.equal(x, y) for x, y in zip(run(q, r, k, v, go, torch.compile(step, backend=backend)), run(q, r, k, v, go, step)))

    def pages(k, v, table, lens, rows):
        table, lens, missing = plx.parallax_fork_pages(k, v, table, lens, rows[:1], rows[1:])
        lens, free, n_free = plx.parallax_free_pages(table, lens, rows[:1], 32, 16)
        table, n_live = plx.parallax_compact_pages(k, v, table, lens)
        plx.parallax_copy_pages(k, v, rows[:1], rows[1:] + 20)
        return k, v, table, lens, missing, free, n_free, n_live

    args = (torch.arange(31, 3, -1, dtype=torch.int32, device="cuda").view(2, 14), ints([100, 0]), ints([0, 1]))
    pools = randn(32, 16, 2, 64, seed=1), randn(32, 16, 2, 64, seed=2)
    torch._dynamo.reset()
    got, want = torch.compile(pages, backend=backend)(*(x.clone() for x in pools), *args), pages(*(x.clone() for x in pools), *args)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and _cabi.device_error() == 0


def test_the_layers_of_a_model_under_one_table():
    """Every layer's call takes the table as it was before: all return the same new one, and each layer's rows hold what they held."""
    page, n_pages, lens = 16, 64, [100, 37, 0, 64]
    layers = [(randn(n_pages, page, 2, 64, seed=2 * i), randn(n_pages, page, 2, 64, seed=2 * i + 1)) for i in range(3)]
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(3))[:28].view(4, 7)
    table, used = order.to(torch.int32).cuda(), ints(lens)
    rows = lambda pool, table, lens: [pool[table[b, :-(-n // page)].long()].flatten(0, 1)[:n].clone() for b, n in enumerate(lens.tolist())]   # noqa: E731
    held = [[rows(x, table, used) for x in pair] for pair in layers]

    new = [plx.parallax_fork_pages(*pair, table, used, ints([0, 1]), ints([2, 3])) for pair in layers]
    assert all(torch.equal(x, y) for other in new[1:] for x, y in zip(new[0], other)) and new[0][2].item() == 0
    table, used = new[0][:2]
    want = [[[x[0], x[1], x[0], x[1]] for x in pair] for pair in held]
    used, _, n_free = plx.parallax_free_pages(table, used, ints([0]), n_pages, page)
    new = [plx.parallax_compact_pages(*pair, table, used) for pair in layers]
    assert all(torch.equal(x, y) for other in new[1:] for x, y in zip(new[0], other)) and new[0][1].item() + n_free.item() == n_pages
    for pair, expected in zip(layers, want):
        for pool, x in zip(pair, expected):
            got = rows(pool, new[0][0], used)
            assert got[0].numel() == 0 and all(torch.equal(a, b) for a, b in zip(got[1:], x[1:]))
