"""Pages of a paged cache on the GPU, against the definitions written out row by row.  Nothing is computed: everything is equal."""
import random

import pytest
import torch

import parallax_b200 as plx
from tests.test_sinks_gpu import no_collection

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def make_pool(n_pages, page, h, d, dtype=torch.bfloat16, layout="token"):
    def one():
        x = torch.randint(-30000, 30000, (n_pages, page, h, d), dtype=torch.int16, device=DEV).view(dtype)
        if layout == "head":                      # (n_pages, H, page, D) in memory
            return x.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "gap":                       # pages and heads with room between them
            big = torch.zeros(n_pages, 2, page, h + 1, d + 8, dtype=dtype, device=DEV)
            big[:, 1, :, :h, :d] = x
            return big[:, 1, :, :h, :d]
        return x
    torch.manual_seed(n_pages + page)
    return one(), one()


def make_table(rng, rows, m, page, n_pages, share=0):
    """Lengths and a table with garbage behind the active entries; the rows from 1 on begin with `share` pages of row 0."""
    lens = [min(rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, m * page), m * page]), m * page) for _ in range(rows)]
    order = list(range(n_pages))
    rng.shuffle(order)
    table, at = [], 0
    for b, n in enumerate(lens):
        count = -(-n // page)
        entries = []
        for j in range(count):
            if b and j < share and j < -(-lens[0] // page):
                entries.append(table[0][j])
            else:
                entries.append(order[at])
                at += 1
        table.append(entries + [rng.choice([-1, 0, 10 ** 9, -2 ** 31, rng.randrange(n_pages)]) for _ in range(m - count)])
    return table, lens


def live_pages(table, lens, page):
    return {p for row, n in zip(table, lens) for p in row[:-(-n // page)]}


SHAPES = [(64, 16, 2, 64, 5, 6, "token"), (300, 1, 1, 128, 7, 9, "token"), (97, 8, 3, 64, 9, 5, "head"), (120, 64, 2, 128, 4, 11, "gap"),
          (33, 128, 1, 64, 3, 3, "token"), (2000, 4, 5, 8, 60, 20, "token")]


@pytest.mark.parametrize("n_pages,page,h,d,rows,m,layout", SHAPES)
def test_copy(n_pages, page, h, d, rows, m, layout):
    rng = random.Random(1)
    k, v = make_pool(n_pages, page, h, d, layout=layout)
    order = rng.sample(range(n_pages), n_pages)
    n = n_pages // 3
    src, dst = order[:n] + [-1, 0, n_pages, order[0]], order[n:2 * n] + [3, -7, order[-1], 2 ** 30]
    want = [x.clone() for x in (k, v)]
    for x in want:
        x[dst[:n]] = x[src[:n]]
    assert plx.parallax_copy_pages(k, v, ints(src), ints(dst)) is None
    assert torch.equal(k.view(torch.int16), want[0].view(torch.int16)) and torch.equal(v.view(torch.int16), want[1].view(torch.int16))
    plx.parallax_copy_pages(k, v, ints([]), ints([]))


@pytest.mark.parametrize("n_pages,page,h,d,rows,m,layout", SHAPES)
def test_compact(n_pages, page, h, d, rows, m, layout):
    rng = random.Random(2)
    table, lens = make_table(rng, rows, m, page, max(n_pages, 1), share=2) if rows * m <= n_pages else make_table(rng, n_pages // m, m, page, n_pages)
    k, v = make_pool(n_pages, page, h, d, torch.float16, layout)
    old = [x.clone() for x in (k, v)]
    new, n_live = plx.parallax_compact_pages(k, v, torch.tensor(table, dtype=torch.int32, device=DEV), ints(lens))
    live = live_pages(table, lens, page)
    n = len(live)
    moved = dict(zip(sorted(p for p in live if p >= n), sorted(set(range(n)) - live)))
    assert n_live.tolist() == [n] and n_live.dtype == torch.int32
    for row, got, length in zip(table, new.tolist(), lens):
        c = -(-length // page)
        assert got == [moved.get(p, p) for p in row[:c]] + row[c:]
    for x, y in zip((k, v), old):
        want = y.clone()
        for s, t in moved.items():
            want[t] = y[s]
        assert torch.equal(x.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("n_pages,page,h,d,rows,m,layout", SHAPES)
@pytest.mark.parametrize("full", [False, True])
def test_fork(n_pages, page, h, d, rows, m, layout, full):
    rng = random.Random(3)
    rows = min(rows, n_pages // m)
    table, lens = make_table(rng, rows, m, page, n_pages)
    if full:                                       # another row holds what is left but for one page
        left = sorted(set(range(n_pages)) - live_pages(table, lens, page))[1:]
        m = max(m, len(left))
        table = [r + [7] * (m - len(r)) for r in table] + [left + [0] * (m - len(left))]
        lens = lens + [len(left) * page]
        rows += 1
    n = 2 * rows
    parents = [rng.randrange(rows) for _ in range(n)] + [-1, rows, 0]
    children = [rng.randrange(rows) for _ in range(n)] + [0, 1, rows + 5]
    k, v = make_pool(n_pages, page, h, d, layout=layout)
    want = [x.clone() for x in (k, v)]
    new, new_lens, missing = plx.parallax_fork_pages(k, v, torch.tensor(table, dtype=torch.int32, device=DEV), ints(lens), ints(parents), ints(children))
    free = sorted(set(range(n_pages)) - live_pages(table, lens, page))
    want_table, want_lens, short = [list(r) for r in table], list(lens), 0
    for i, (p, c) in enumerate(zip(parents, children)):
        if not (0 <= p < rows and 0 <= c < rows) or c in [y for x, y in zip(parents[i + 1:], children[i + 1:]) if 0 <= x < rows and 0 <= y < rows]:
            continue
        want_table[c], want_lens[c] = list(table[p]), lens[p]
        tail = lens[p] % page
        if tail and p != c:
            slot = lens[p] // page
            if free:
                fresh = free.pop(0)
                for x in want:
                    x[fresh, :tail] = x[table[p][slot], :tail]
                want_table[c][slot] = fresh
            else:
                short += 1
                want_table[c][slot] = -1
                want_lens[c] = lens[p] - tail
    assert missing.tolist() == [short]
    assert new.tolist() == want_table and new_lens.tolist() == want_lens
    assert torch.equal(k.view(torch.int16), want[0].view(torch.int16)) and torch.equal(v.view(torch.int16), want[1].view(torch.int16))


@pytest.mark.parametrize("n_pages,page,rows,m", [(64, 16, 5, 6), (1, 1, 1, 1), (5000, 8, 300, 12), (1700000, 16, 40, 300)])
def test_free(n_pages, page, rows, m):
    rng = random.Random(4)
    table, lens = make_table(rng, rows, m, page, n_pages) if rows * m <= n_pages else ([[0]], [1])
    gone = [b for b in range(0, len(lens), 2)] + [-1, len(lens), 0]
    new_lens, free, n_free = plx.parallax_free_pages(torch.tensor(table, dtype=torch.int32, device=DEV), ints(lens), ints(gone), n_pages, page)
    want_lens = [0 if b in gone else n for b, n in enumerate(lens)]
    left = torch.ones(n_pages, dtype=torch.bool)
    left[list(live_pages(table, want_lens, page))] = False
    found = torch.nonzero(left).flatten()
    assert new_lens.tolist() == want_lens and n_free.tolist() == [found.numel()]
    assert torch.equal(free[:found.numel()].cpu().long(), found) and bool((free[found.numel():] == -1).all())


def test_lengths_and_pages_out_of_range_are_passed_over():
    k, v = make_pool(16, 4, 1, 64)
    old = k.clone()
    table = torch.tensor([[3, 99, -5], [2 ** 31 - 1, 15, 3]], dtype=torch.int32, device=DEV)
    new, n_live = plx.parallax_compact_pages(k, v, table, ints([10 ** 9, 12]))       # longer than the row: the row
    assert n_live.tolist() == [2] and new.tolist() == [[0, 99, -5], [2 ** 31 - 1, 1, 0]]
    assert torch.equal(k[0].view(torch.int16), old[3].view(torch.int16)) and torch.equal(k[1].view(torch.int16), old[15].view(torch.int16))
    new, lens, missing = plx.parallax_fork_pages(k, v, table, ints([-3, 10]), ints([0, 1]), ints([1, 0]))
    assert lens.tolist() == [10, 0] and missing.tolist() == [0] and new[0].tolist() == [2 ** 31 - 1, 15, 0]


@pytest.mark.parametrize("rows,n", [(5000, 4000), (300, 2500), (4096, 1024), (4097, 1025)])
def test_fork_of_many_rows(rows, n):
    """More rows than shared memory has room for, more pairs than a CTA has threads."""
    rng = random.Random(6)
    page, m = 4, 3
    n_pages = rows * m + n
    k, v = make_pool(n_pages, page, 1, 8)
    lens = [rng.randint(0, m * page) for _ in range(rows)]
    order = rng.sample(range(n_pages), rows * m)
    table = torch.tensor(order, dtype=torch.int32).view(rows, m)
    parents, children = [rng.randrange(rows) for _ in range(n)], [rng.randrange(rows) for _ in range(n)]
    want_k, want_table, want_lens = k.clone(), table.clone(), list(lens)
    live = {int(table[b, j]) for b in range(rows) for j in range(-(-lens[b] // page))}
    free = iter(p for p in range(n_pages) if p not in live)
    final = dict(zip(children, range(n)))
    for i, (p, c) in enumerate(zip(parents, children)):
        if final[c] != i:
            continue
        want_table[c], want_lens[c] = table[p], lens[p]
        if lens[p] % page and p != c:
            new, slot = next(free), lens[p] // page
            want_k[new, :lens[p] % page] = k[int(table[p, slot]), :lens[p] % page]
            want_table[c, slot] = new
    got, got_lens, missing = plx.parallax_fork_pages(k, v, table.cuda(), ints(lens), ints(parents), ints(children))
    assert missing.item() == 0 and got_lens.tolist() == want_lens and torch.equal(got.cpu(), want_table)
    assert torch.equal(k.view(torch.int16), want_k.view(torch.int16))


def test_fork_without_a_free_page():
    k, v = make_pool(4, 16, 1, 64)
    table, lens = ints([0, 1, 2, 3]).view(2, 2), ints([20, 30])
    new, new_lens, missing = plx.parallax_fork_pages(k, v, table, lens, ints([0]), ints([1]))       # row 1's own pages are not free yet
    assert missing.tolist() == [1] and new.tolist() == [[0, 1], [0, -1]] and new_lens.tolist() == [20, 16]


def test_captured_calls_follow_the_tables():
    k, v = make_pool(64, 16, 2, 64)
    table, lens = ints(range(40, 46)).view(2, 3), ints([40, 33])
    rows, parents, children = ints([1]), ints([0]), ints([1])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                       # (loads the kernels)
        plx.parallax_fork_pages(k, v, table, lens, parents, children)
        plx.parallax_compact_pages(k, v, table, lens)
        plx.parallax_free_pages(table, lens, rows, 64, 16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with no_collection(), torch.cuda.graph(graph):
        forked, flens, missing = plx.parallax_fork_pages(k, v, table, lens, parents, children)
        packed, n_live = plx.parallax_compact_pages(k, v, forked, flens)
        left, free, n_free = plx.parallax_free_pages(packed, flens, rows, 64, 16)
    for n0 in (40, 48, 17, 0):
        lens.copy_(ints([n0, 33]))
        graph.replay()
        torch.cuda.synchronize()
        shared, own = -(-n0 // 16), 1 if n0 % 16 else 0
        assert flens.tolist() == [n0, n0] and missing.tolist() == [0] and n_live.tolist() == [shared + own]
        assert left.tolist() == [n0, 0] and n_free.tolist() == [64 - shared]
        assert len(set(packed[0, :shared].tolist()) | set(packed[1, :shared].tolist())) == shared + own


def test_another_stream_and_the_current_device_of_the_tensors():
    k, v = make_pool(64, 16, 2, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        src, dst = ints(range(0, 30)), ints(range(30, 60))
        plx.parallax_copy_pages(k, v, src, dst)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(k[:30].view(torch.int16), k[30:60].view(torch.int16))


def test_gpu_refusals():
    k, v = make_pool(8, 16, 2, 64)
    one = ints([1])
    with pytest.raises(ValueError):
        plx.parallax_copy_pages(k[:1].expand(8, -1, -1, -1), v, one, one)
    with pytest.raises(ValueError):
        plx.parallax_copy_pages(k.transpose(2, 3).contiguous().transpose(2, 3), v, one, one)
    with pytest.raises(RuntimeError):
        plx.parallax_copy_pages(k, v, one.cpu(), one)
    with pytest.raises(ValueError):
        plx.parallax_copy_pages(k, v, one, ints([1, 2]))
