"""Sinks, shared prefixes and pages on the GPU: calls at the edges of what they document, against the definition in 64 bits."""
import pytest
import torch

import parallax_b200 as plx
from parallax_b200 import _cabi
from tests.test_prefix_gpu import make, pages_of, reference
from tests.test_sinks_gpu import close, decode_reference, hide, paged, randn

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
