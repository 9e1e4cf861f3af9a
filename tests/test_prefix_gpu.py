"""Decode over a shared prefix on the GPU, against the definition in 64 bits, and the pages, sinks and prefixes of one cache used
together.  Tolerances as in test_sinks_gpu: half a step for the weights that multiply v and half a step for the result."""
import pytest
import torch

import parallax_b200 as plx
from parallax_b200 import _cabi, ops
from tests.test_sinks_gpu import attend, close, no_collection, randn

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def reference(q, r, keys, values, scale=None):
    """keys, values: per row (n, H_kv, D)"""
    out = torch.zeros_like(q, dtype=torch.float64)
    for b, (k, v) in enumerate(zip(keys, values)):
        rep = q.shape[2] // k.shape[1]
        kk, vv = (x.double().transpose(0, 1).repeat_interleave(rep, 0) for x in (k, v))
        ok = torch.ones(1, k.shape[0], dtype=torch.bool, device=q.device)
        out[b] = attend(q[b].double().transpose(0, 1), r[b].double().transpose(0, 1), kk, vv, ok, q.shape[3] ** -0.5 if scale is None else scale).transpose(0, 1)
    return out


def make(b, hq, hkv, d, dtype, p, t, seed=1):
    return (randn(b, 1, hq, d, dtype=dtype, seed=seed), randn(b, 1, hq, d, dtype=dtype, scale=0.5, seed=seed + 1),
            randn(p, hkv, d, dtype=dtype, seed=seed + 2), randn(p, hkv, d, dtype=dtype, seed=seed + 3),
            randn(b, t, hkv, d, dtype=dtype, seed=seed + 4), randn(b, t, hkv, d, dtype=dtype, seed=seed + 5))


# b, hq, hkv, d, dtype, prefix, own keys, lengths of those (None: all)
DENSE = [
    (1, 1, 1, 64, BF, 1, 1, [0]),
    (1, 8, 8, 128, BF, 1, 1, [1]),
    (2, 8, 8, 128, BF, 63, 5, [0, 5]),
    (3, 8, 2, 128, FP, 64, 40, [40, 0, 1]),
    (5, 14, 2, 64, BF, 65, 33, None),                       # 7 heads a kv head: 126 rows a tile
    (40, 32, 8, 128, BF, 1000, 70, [i % 71 for i in range(40)]),
    (33, 4, 4, 64, FP, 2500, 17, [17] * 33),
    (130, 8, 8, 128, BF, 129, 3, [i % 4 for i in range(130)]),   # two tiles of rows, the second of two
    (3, 300, 2, 64, BF, 200, 9, [9, 0, 4]),                 # 150 heads a kv head: more than a tile
    (2, 128, 1, 128, BF, 4097, 1, [1, 0]),
    (300, 16, 2, 128, BF, 700, 4, [i % 5 for i in range(300)]),
    (2, 8, 8, 128, BF, 9000, 1200, [1200, 3]),
]


@pytest.mark.parametrize("case", DENSE, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c[:7]))
def test_dense(case):
    b, hq, hkv, d, dtype, p, t, lens = case
    q, r, kp, vp, k, v = make(b, hq, hkv, d, dtype, p, t)
    n = lens or [t] * b
    want = reference(q, r, [torch.cat((kp, k[i, :n[i]])) for i in range(b)], [torch.cat((vp, v[i, :n[i]])) for i in range(b)])
    for i in range(b):                                      # what is not active may hold anything
        k[i, n[i]:] = v[i, n[i]:] = torch.nan
    got = plx.parallax_decode_shared_prefix(q, r, kp, vp, k, v, seqused_k=None if lens is None else ints(lens))
    close(got, want, 2, "o")
    out = torch.empty_like(q)
    again = plx.parallax_decode_shared_prefix(q, r, kp, vp, k, v, seqused_k=None if lens is None else ints(lens), out=out)
    assert again is out and torch.equal(out, got)           # the Python path, the same kernels
    assert _cabi.device_error() == 0


@pytest.mark.parametrize("splits", [0, 1, 2, 5, 16, 40, 127])
@pytest.mark.parametrize("b,hq,hkv,d,dtype,p,t", [
    (3, 8, 8, 128, BF, 8128, 20), (1, 4, 4, 64, FP, 130, 1), (9, 8, 2, 128, BF, 700, 130), (5, 3, 1, 64, BF, 321, 7), (140, 2, 2, 64, BF, 64, 3),
    (4, 40, 2, 128, FP, 2600, 60), (2, 260, 2, 64, BF, 1000, 5), (33, 16, 4, 128, BF, 1, 40)])
def test_every_way_to_split(b, hq, hkv, d, dtype, p, t, splits):
    """0: every row sweeps the prefix in front of its own keys; else its parts, one for every 64 keys at most."""
    q, r, kp, vp, k, v = make(b, hq, hkv, d, dtype, p, t)
    n = [(i * 7) % (t + 1) for i in range(b)]
    want = reference(q, r, [torch.cat((kp, k[i, :n[i]])) for i in range(b)], [torch.cat((vp, v[i, :n[i]])) for i in range(b)])
    for i in range(b):
        k[i, n[i]:] = v[i, n[i]:] = torch.nan
    out = torch.empty_like(q)
    for own in (1, 3, 8, 40):
        if splits > -(-p // 64):
            with pytest.raises(_cabi.PlxError):
                ops.decode_prefix(q, r, kp, vp, p, k, v, out, torch.zeros(1 << 24, device="cuda"), d ** -0.5, own, splits, ints(n), None)
            continue
        ws = torch.zeros(max(ops.decode_prefix_workspace_bytes(q, k, own, splits, None) // 4, 4), device="cuda")
        for _ in range(2):                                  # (a workspace is left as it was found)
            ops.decode_prefix(q, r, kp, vp, p, k, v, out, ws, d ** -0.5, own, splits, ints(n), None)
            close(out, want, 2, (splits, own))
    assert _cabi.device_error() == 0


@pytest.mark.parametrize("scale", [-0.2, 0.0, 0.4])
def test_scales(scale):
    q, r, kp, vp, k, v = make(3, 8, 2, 64, BF, 300, 20)
    want = reference(q, r, [torch.cat((kp, k[i])) for i in range(3)], [torch.cat((vp, v[i])) for i in range(3)], scale)
    close(plx.parallax_decode_shared_prefix(q, r, kp, vp, k, v, scale), want, 2, "o")
    out, ws = torch.empty_like(q), torch.zeros(1 << 20, device="cuda")
    ops.decode_prefix(q, r, kp, vp, 300, k, v, out, ws, scale, 4, 3, None, None)      # shared where there is a kernel for it
    close(out, want, 2, "o")


def test_layouts():
    """Prefix and own keys as slices of wider buffers, heads first, and q, r that are not contiguous."""
    q, r, kp, vp, k, v = make(4, 8, 4, 128, BF, 500, 60)
    want = plx.parallax_decode_shared_prefix(q, r, kp, vp, k, v)
    wide = lambda x: torch.cat((x, x), 0)[:x.shape[0]]                                             # noqa: E731
    first = lambda x: x.transpose(-3, -2).contiguous().transpose(-3, -2)                           # noqa: E731
    odd = lambda x: torch.stack((x, x), -1)[..., 0]                                                # noqa: E731
    for args in ((q, r, wide(kp), wide(vp), k, v), (q, r, first(kp), first(vp), first(k), first(v)), (q, r, first(kp), vp, k, first(v)),
                 (odd(q), odd(r), odd(kp), kp.new_empty(0) if False else odd(vp), odd(k), odd(v))):
        assert torch.equal(plx.parallax_decode_shared_prefix(*args), want)


def pages_of(kp, vp, k, v, lens, page, seed=5):
    """Prefix (whole pages) and own keys in one pool; unused keys NaN, entries behind the active ones nonsense."""
    p, b, t = kp.shape[0], k.shape[0], k.shape[1]
    m, shared = -(-(p + t) // page), p // page
    n_pages = shared + b * (m - shared) + 2
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    pools = [torch.full((n_pages, page, *kp.shape[1:]), torch.nan, dtype=kp.dtype, device="cuda") for _ in range(2)]
    table = torch.full((b, m), 10 ** 6, dtype=torch.int32)
    for j in range(shared):
        table[:, j] = order[j]
        for pool, x in zip(pools, (kp, vp)):
            pool[order[j]] = x[j * page:(j + 1) * page]
    at = shared
    for i in range(b):
        for j in range(-(-lens[i] // page)):
            table[i, shared + j] = order[at]
            for pool, x in zip(pools, (k, v)):
                part = x[i, j * page:min((j + 1) * page, lens[i])]
                pool[order[at], :part.shape[0]] = part
            at += 1
    return (*pools, table.cuda())


@pytest.mark.parametrize("b,hq,hkv,d,dtype,p,t,page", [
    (3, 8, 8, 128, BF, 64, 20, 16), (5, 16, 4, 64, FP, 96, 70, 32), (4, 8, 2, 128, BF, 1024, 200, 64), (2, 4, 4, 64, BF, 512, 9, 256),
    (20, 32, 8, 128, BF, 40, 33, 8), (3, 8, 4, 128, BF, 12, 5, 4), (6, 20, 1, 128, BF, 2000, 50, 16), (2, 8, 8, 64, BF, 7, 3, 1)])
def test_paged(b, hq, hkv, d, dtype, p, t, page):
    lens = [(t * (i + 1)) // b for i in range(b)]
    lens[0] = 0
    q, r, kp, vp, k, v = make(b, hq, hkv, d, dtype, p, t)
    want = reference(q, r, [torch.cat((kp, k[i, :lens[i]])) for i in range(b)], [torch.cat((vp, v[i, :lens[i]])) for i in range(b)])
    pk, pv, table = pages_of(kp, vp, k, v, lens, page)
    seqused = ints([p + n for n in lens])
    call = lambda **kw: plx.parallax_attn_with_kvcache(q, r, pk, pv, page_table=table, seqused_k=seqused, **kw)      # noqa: E731
    close(call(shared_prefix=p), want, 2, "all of it")
    close(call(shared_prefix=p - 1), want, 2, "its whole pages")
    close(call(), want, 2, "without the word")
    # a window, and several tokens per row: the word changes nothing
    assert torch.equal(call(shared_prefix=p, window_size=50), call(window_size=50))
    with pytest.raises(ValueError):
        plx.parallax_attn_with_kvcache(q, r, pk, pv, page_table=table, seqused_k=ints([p - 1] * b), shared_prefix=p)


def test_captured_and_replayed_on_two_streams():
    calls, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        args = make(6, 16, 4, 128, BF, 1500, 90, seed=10 * i)
        lens = ints([90, 0, 1, 40, 63, 64])
        plx.parallax_decode_shared_prefix(*args, seqused_k=lens)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with no_collection(), torch.cuda.graph(graph):
            out = plx.parallax_decode_shared_prefix(*args, seqused_k=lens)
        calls.append((graph, out, args, lens))
    for round_ in range(3):
        for _, _, _, lens in calls:
            lens.copy_(ints([90 - 7 * round_, 30, 1, 0, 63, 64]))
        torch.cuda.synchronize()
        for _ in range(10):
            for stream, (graph, *_) in zip(streams, calls):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for _, out, (q, r, kp, vp, k, v), lens in calls:
            n = lens.tolist()
            close(out, reference(q, r, [torch.cat((kp, k[i, :n[i]])) for i in range(6)], [torch.cat((vp, v[i, :n[i]])) for i in range(6)]), 2, "o")


@pytest.mark.parametrize("hq,hkv", [(8, 8), (3, 3), (16, 4), (32, 2)])
@pytest.mark.parametrize("p,t,prefix_splits,n_splits", [(30000, 1, 2, 1), (30000, 40, 18, 2), (130, 6000, 1, 1), (4000, 3000, 9, 8)])
def test_whichever_ends_first(hq, hkv, p, t, prefix_splits, n_splits):
    """Own keys are swept beside the prefix: the merge, and what follows it, come behind both, captured too.  Inputs that change between
    the calls show a merge of records of the call before."""
    b, d = 4, 128
    sets = [make(b, hq, hkv, d, BF, p, t, seed=7 * i) for i in range(2)]
    ins = [x.clone() for x in sets[0]]
    q, r, kp, vp, k, v = ins
    out, after = torch.empty_like(q), torch.empty_like(q)
    ws = torch.zeros(ops.decode_prefix_workspace_bytes(q, k, n_splits, prefix_splits, None) // 4, device="cuda")

    def call():
        ops.decode_prefix(q, r, kp, vp, p, k, v, out, ws, d ** -0.5, n_splits, prefix_splits, None, None)
        after.copy_(out)
        out.zero_()

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with no_collection(), torch.cuda.graph(graph):
        call()
    want = [reference(x[0], x[1], [torch.cat((x[2], x[4][i])) for i in range(b)], [torch.cat((x[3], x[5][i])) for i in range(b)]) for x in sets]
    for run in (call, graph.replay):
        for i in range(6):
            for x, y in zip(ins, sets[i % 2]):
                x.copy_(y)
            run()
            close(after, want[i % 2], 2, "o")


def test_two_threads_on_two_streams():
    """Eager calls of one shape at once: a workspace for each stream."""
    import threading
    sets = [make(4, 8, 2, 128, BF, 800, 40, seed=i) for i in (1, 50)]
    want = [plx.parallax_decode_shared_prefix(*x) for x in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(200):
                if not torch.equal(plx.parallax_decode_shared_prefix(*sets[i]), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not bad


def test_refusals():
    q, r, kp, vp, k, v = make(2, 8, 2, 64, BF, 32, 8)
    fn = plx.parallax_decode_shared_prefix
    for call, error in (
            (lambda: fn(q.float(), r, kp, vp, k, v), TypeError), (lambda: fn(q, r, kp.half(), vp, k, v), TypeError),
            (lambda: fn(q, r[:1], kp, vp, k, v), ValueError), (lambda: fn(q, r, kp[None], vp, k, v), ValueError),
            (lambda: fn(q, r, kp[:0], vp[:0], k, v), ValueError), (lambda: fn(q, r, kp, vp[:5], k, v), ValueError),
            (lambda: fn(q, r, kp, vp, k[:1], v[:1]), ValueError), (lambda: fn(q.expand(2, 3, 8, 64), r.expand(2, 3, 8, 64), kp, vp, k, v), ValueError),
            (lambda: fn(q[:, :, :7], r[:, :, :7], kp, vp, k, v), ValueError), (lambda: fn(q, r, kp.cpu(), vp.cpu(), k, v), RuntimeError),
            (lambda: fn(q, r, kp, vp, k, v, seqused_k=ints([9, 1])), ValueError), (lambda: fn(q, r, kp, vp, k, v, seqused_k=ints([-1, 1])), ValueError),
            (lambda: fn(q, r, kp, vp, k, v, seqused_k=ints([1, 1]).long()), TypeError),
            (lambda: fn(q, r, kp, vp, k, v, out=q.half()), ValueError),
            (lambda: plx.parallax_attn_with_kvcache(q, r, k, v, shared_prefix=4), ValueError),
            (lambda: plx.parallax_attn_with_kvcache(q, r, k, v, page_table=ints([[0], [1]]), shared_prefix=9), ValueError),
            (lambda: plx.parallax_attn_with_kvcache(q, r, k, v, page_table=ints([[0], [1]]), shared_prefix=-8), ValueError)):
        with pytest.raises(error):
            call()
    d = torch.randn(2, 1, 8, 32, device="cuda", dtype=BF)
    with pytest.raises(NotImplementedError):
        fn(d, d, d[:, 0, :2], d[:, 0, :2], d[:, :, :2], d[:, :, :2])


def test_the_life_of_a_paged_cache():
    """A prompt in pages, forked into samples that go on by themselves; attention over their shared prefix, with and without a window
    and sinks; one sample freed, another compacted into the room -- each step against dense copies of the rows."""
    torch.manual_seed(0)
    page, hq, hkv, d, rows, m, prompt = 16, 8, 2, 128, 6, 30, 333
    k_pool, v_pool = (torch.full((200, page, hkv, d), torch.nan, dtype=BF, device="cuda") for _ in range(2))
    order = torch.randperm(200)[:m]
    table, lens = torch.zeros(rows, m, dtype=torch.int32, device="cuda"), ints([prompt] + [0] * (rows - 1))
    table[0, :-(-prompt // page)] = order[:-(-prompt // page)].cuda()
    dense = [[randn(m * page, hkv, d, seed=s) for s in (1, 2)] for _ in range(rows)]
    flat = [x.view(-1, hkv, d) for x in (k_pool, v_pool)]

    def write(row, at, k_new, v_new):
        """One key of a row, in a page of its own where the row has come to the end of one."""
        nonlocal table, lens, free
        if at % page == 0:
            table[row, at // page] = free.pop()
        slot = int(table[row, at // page]) * page + at % page
        for pool, x, copy in zip(flat, (k_new, v_new), dense[row]):
            pool[slot] = x
            copy[at] = x

    for j in range(prompt):
        slot = int(table[0, j // page]) * page + j % page
        for pool, x in zip(flat, dense[0]):
            pool[slot] = x[j]
    children = list(range(1, rows))
    table, lens, missing = plx.parallax_fork_pages(k_pool, v_pool, table, lens, ints([0] * len(children)), ints(children))
    assert missing.item() == 0 and lens.tolist() == [prompt] * rows
    for c in children:
        dense[c] = [x.clone() for x in dense[0]]
    shared = prompt // page * page
    assert (table[:, :shared // page] == table[:1, :shared // page]).all() and len(set(table[:, shared // page].tolist())) == rows
    lens, found, n_free = plx.parallax_free_pages(table, lens, ints([]), 200, page)
    free = found[:n_free.item()].tolist()

    def agree(live):
        q, r = randn(len(live), 1, hq, d, seed=7), randn(len(live), 1, hq, d, scale=0.5, seed=8)
        n, t, used = [lens[b].item() for b in live], table[live].contiguous(), lens[live].contiguous()
        want = reference(q, r, [dense[b][0][:x] for b, x in zip(live, n)], [dense[b][1][:x] for b, x in zip(live, n)])
        close(plx.parallax_attn_with_kvcache(q, r, k_pool, v_pool, page_table=t, seqused_k=used, shared_prefix=prompt), want, 2, "shared")
        hidden = [torch.cat([torch.arange(0, 4), torch.arange(x - 40, x)]).cuda() for x in n]
        want = reference(q, r, [dense[b][0][at] for b, at in zip(live, hidden)], [dense[b][1][at] for b, at in zip(live, hidden)])
        close(plx.parallax_attn_with_kvcache(q, r, k_pool, v_pool, page_table=t, seqused_k=used, window_size=40, sink_tokens=4), want, 2, "sinks")

    agree(list(range(rows)))
    for step in range(25):
        for b in range(rows):
            write(b, lens[b].item(), randn(hkv, d, seed=100 * step + b), randn(hkv, d, seed=5000 + 100 * step + b))
            lens[b] += 1
    agree(list(range(rows)))
    lens, found, n_free = plx.parallax_free_pages(table, lens, ints([2, 4]), 200, page)
    live = [0, 1, 3, 5]
    agree(live)
    table, n_live = plx.parallax_compact_pages(k_pool, v_pool, table, lens)
    assert n_live.item() == 200 - n_free.item() and table[live, :lens[0].item() // page].max() < n_live.item()
    k_pool[n_live.item():] = v_pool[n_live.item():] = torch.nan         # nothing behind the live pages is read
    agree(live)


def test_pages_behind_two_to_the_31_elements():
    """Pools of more than 2^31 elements: the last pages of one as a prefix, as sinks and windows, copied, forked and compacted."""
    page, hq, hkv, d, n_pages = 64, 16, 8, 128, 33000
    assert (n_pages - 20) * page * hkv * d > 2 ** 31
    k_pool, v_pool = (torch.empty(n_pages, page, hkv, d, dtype=BF, device="cuda") for _ in range(2))
    b, prefix, own = 2, 4 * page, 50
    order = list(range(n_pages - 1, n_pages - 13, -2))             # pages n - 1, n - 3, ..
    table = ints([order[:4] + [order[4]], order[:4] + [order[5]]])
    for p in order:
        k_pool[p], v_pool[p] = randn(page, hkv, d, seed=p), randn(page, hkv, d, seed=2 * p)
    lens = ints([prefix + own, prefix + 3])
    q, r = randn(b, 1, hq, d, seed=1), randn(b, 1, hq, d, scale=0.5, seed=2)

    def rows():
        return [[pool[table[i].long()].flatten(0, 1)[:lens[i].item()].clone() for i in range(b)] for pool in (k_pool, v_pool)]

    keys, values = rows()
    want = reference(q, r, keys, values)
    ws = torch.zeros(1 << 22, device="cuda")
    for splits in (0, 1, 3):
        out = torch.empty_like(q)
        ops.decode_prefix(q, r, None, None, prefix, k_pool, v_pool, out, ws, d ** -0.5, 2, splits, lens, table)
        close(out, want, 2, splits)
    hidden = [torch.cat([torch.arange(5), torch.arange(n - 90, n)]).cuda() for n in lens.tolist()]
    sinks = reference(q, r, [x[at] for x, at in zip(keys, hidden)], [x[at] for x, at in zip(values, hidden)])
    close(plx.parallax_attn_with_kvcache(q, r, k_pool, v_pool, page_table=table, seqused_k=lens, window_size=90, sink_tokens=5), sinks, 2, "sinks")
    several = plx.parallax_attn_with_kvcache(q.expand(-1, 2, -1, -1).contiguous(), r.expand(-1, 2, -1, -1).contiguous(), k_pool, v_pool, page_table=table,
                                             seqused_k=lens, window_size=90, sink_tokens=5)
    close(several[:, 1:], sinks, 2, "sinks, two tokens")
    plx.parallax_copy_pages(k_pool, v_pool, ints([order[0], order[5]]), ints([7, n_pages - 2]))
    assert torch.equal(k_pool[7], k_pool[order[0]]) and torch.equal(v_pool[n_pages - 2], v_pool[order[5]])
    forked, flens, missing = plx.parallax_fork_pages(k_pool, v_pool, table, lens, ints([0]), ints([1]))
    assert missing.item() == 0 and forked[1].tolist() == order[:4] + [0] and torch.equal(k_pool[0, :own], k_pool[order[4], :own])
    table, n_live = plx.parallax_compact_pages(k_pool, v_pool, table, lens)
    assert n_live.item() == 6 and sorted(set(table.flatten().tolist())) == list(range(6))
    again = rows()
    assert all(torch.equal(x, y) for new, old in zip(again, (keys, values)) for x, y in zip(new, old))


def test_dense_prefix_behind_two_to_the_31_elements():
    """A prefix of more than 2^31 elements, of which all but the last keys weigh nothing."""
    hkv, d, p = 8, 128, 2 ** 21 + 1000
    assert p * hkv * d > 2 ** 31
    kp, vp = (torch.zeros(p, hkv, d, dtype=BF, device="cuda") for _ in range(2))
    q, r = randn(3, 1, 16, d, seed=1), randn(3, 1, 16, d, scale=0.5, seed=2)
    k, v = randn(3, 5, hkv, d, seed=3), randn(3, 5, hkv, d, seed=4)
    kp[-200:], vp[-200:] = randn(200, hkv, d, scale=12.0, seed=5), randn(200, hkv, d, seed=6)      # logits far above those of the zeros
    want = reference(q, r, [torch.cat((kp[-4000:], k[i])) for i in range(3)], [torch.cat((vp[-4000:], v[i])) for i in range(3)])
    close(plx.parallax_decode_shared_prefix(q, r, kp, vp, k, v), want, 2, "shared")
    out, ws = torch.empty_like(q), torch.zeros(1 << 22, device="cuda")
    ops.decode_prefix(q, r, kp, vp, p, k, v, out, ws, d ** -0.5, 16, 0, None, None)
    close(out, want, 2, "every row")
