"""What the operators of long contexts are measured on: attention with a sliding window whose first tokens stay visible
(sinks), decode of a batch that shares a prefix, and the pages of a paged cache.

A case is a dict of plain values.  `kind` says which call it is:

* ``train``   ``parallax_func(..., window_size_left, sink_tokens)``, forward and the gradients of all four inputs
* ``packed``  ``parallax_varlen_func`` with the same arguments, on sequences of their own lengths
* ``extend``  ``parallax_attn_with_kvcache`` with ``lq`` > 1 new tokens per row, a window and sinks, dense or paged
* ``decode``  the same (paged) or ``parallax_decode`` (dense) for one token per row
* ``prefix``  one token per row behind a shared prefix: ``parallax_decode_shared_prefix`` (``page`` = 0: the prefix is a tensor of
  its own) or ``parallax_attn_with_kvcache(..., shared_prefix)`` (the rows' page tables begin with the same pages)
* ``copy`` / ``fork`` / ``compact`` / ``free``  ``parallax_copy_pages`` and its siblings

With ``own`` false, `run` computes the same in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ATTENTION = ("train", "packed", "extend", "decode", "prefix")


# --------------------------------------------------------------------------- #
# cases
# --------------------------------------------------------------------------- #
def listed():
    return [
        # a unit of a fine-tuning job: one short sequence of an odd length, where launches show
        _named("train_small", _train("train", b=1, hq=4, hkv=4, l=500, d=64, dtype="fp16", window=96, sinks=3)),
        # long-context training: 8192 tokens, each of which sees the last 1024 and the first 4
        _named("train_l8192", _train("train", b=1, hq=16, hkv=16, l=8192, window=1024, sinks=4)),
        # packed documents of 1 to 1500 tokens, grouped-query heads, a short window
        _named("packed_gqa", _train("packed", b=1, hq=16, hkv=4, l=8192, window=256, sinks=16, longest=1500)),
        # chunked prefill: four rows bring 256 tokens each to caches in pages
        _named("extend_paged", _cache("extend", b=4, hq=32, hkv=8, t=4096, lq=256, page=64, window=1024, sinks=64)),
        # one user of a chat whose cache has outgrown the window
        _named("decode_b1", _cache("decode", b=1, hq=8, hkv=8, t=4096, page=0, window=1024, sinks=4)),
        # a serving batch over a paged cache, every row of its own length
        _named("decode_gqa_paged", _cache("decode", b=32, hq=32, hkv=8, t=16384, page=64, window=4096, sinks=64)),
        # a few samples of one question: a short prompt, a few tokens each
        _named("prefix_small", _prefix(b=4, hq=8, hkv=8, p=1000, t=72, page=0)),
        # a system prompt in front of a batch of chats
        _named("prefix_gqa", _prefix(b=32, hq=32, hkv=8, p=8192, t=512, page=0)),
        # a document that many ask about, in pages
        _named("prefix_paged_b128", _prefix(b=128, hq=32, hkv=8, p=32768, t=512, page=64)),
        # copy-on-write of a few pages, the list padded to a fixed size
        _named("copy_small", _pool("copy", pages=256, page=16, hkv=8, moves=8)),
        # a step of parallel sampling: 32 rows go on from 8
        _named("fork_32", _pool("fork", pages=4096, page=64, hkv=8, rows=64, t=3500, moves=32)),
        # a pool that has become scattered
        _named("compact_16384", _pool("compact", pages=16384, page=16, hkv=8, rows=96, t=2000)),
    ]


def draw(rng):
    """One more case of these ranges, at most as costly as the largest listed one of its kind."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("train", "train", "packed", "packed", "extend", "decode", "decode", "decode", "prefix", "prefix", "prefix", "copy", "fork",
                       "compact", "free"))
    d = rng.choice((128, 128, 64))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind in ("train", "packed"):
        hq, hkv = rng.choice(((4, 4), (8, 8), (16, 16), (16, 4), (8, 1)))
        l = log_int(60, 8192)
        window = log_int(16, max(17, min(l, 1024)))
        sinks = rng.choice((1, 4, 4, 16, 70, 130))
        b = 1 if kind == "packed" else log_int(1, max(1, min(8, 2 ** 29 // (l * l * hq))))
        return _train(kind, b=b, hq=hq, hkv=hkv, l=l, d=d, dtype=dtype, window=window, sinks=sinks,
                      longest=log_int(20, max(21, min(l, 3000))) if kind == "packed" else 0)
    if kind in ("extend", "decode"):
        hq, hkv = rng.choice(((32, 8), (16, 4), (16, 2), (8, 8), (12, 12), (24, 2)))
        page = rng.choice((0, 16, 64, 256))
        t = log_int(300, 16384 if kind == "decode" else 4096)
        lq = 1 if kind == "decode" else log_int(2, min(256, t // 4))
        b = log_int(1, 32 if kind == "decode" else 4)
        return _cache(kind, b=b, hq=hq, hkv=hkv, t=-(-t // page) * page if page else t, lq=lq, page=page, d=d, dtype=dtype,
                      window=log_int(32, min(4096, t)), sinks=rng.choice((1, 4, 4, 17, 64, 200)))
    if kind == "prefix":
        hq, hkv = rng.choice(((32, 8), (16, 2), (16, 16), (8, 8), (8, 1), (28, 4)))
        page = rng.choice((0, 0, 16, 64))
        p = log_int(200, 32768)
        return _prefix(b=log_int(2, 128), hq=hq, hkv=hkv, p=-(-p // page) * page if page else p, t=log_int(16, 512), page=page, d=d, dtype=dtype)
    page = rng.choice((16, 64))
    pages = log_int(128, 65536 // page)
    t = log_int(40, 2000)
    if kind == "copy":
        return _pool(kind, pages=pages, page=page, hkv=rng.choice((8, 4, 2)), d=d, dtype=dtype, moves=log_int(2, 64))
    t = min(t, pages * page // 4)
    rows = max(2, min(64, int(0.6 * pages / (t / page + 1))))
    return _pool(kind, pages=pages, page=page, hkv=rng.choice((8, 4, 2)), d=d, dtype=dtype, rows=rows, t=t,
                 moves=max(1, rows // 3) if kind == "fork" else 0)


def _named(name, case):
    return dict(name=name, **case)


def _train(kind, *, b, hq, hkv, l, d=128, dtype="bf16", window, sinks, longest=0):
    return dict(kind=kind, b=b, hq=hq, hkv=hkv, l=l, d=d, dtype=dtype, window=window, sinks=sinks, longest=longest)


def _cache(kind, *, b, hq, hkv, t, lq=1, page, d=128, dtype="bf16", window, sinks):
    return dict(kind=kind, b=b, hq=hq, hkv=hkv, t=t, lq=lq, page=page, d=d, dtype=dtype, window=window, sinks=sinks)


def _prefix(*, b, hq, hkv, p, t, page, d=128, dtype="bf16"):
    return dict(kind="prefix", b=b, hq=hq, hkv=hkv, p=p, t=t, page=page, d=d, dtype=dtype)


def _pool(kind, *, pages, page, hkv, rows=0, t=0, moves=0, d=128, dtype="bf16"):
    return dict(kind=kind, pages=pages, page=page, hkv=hkv, d=d, dtype=dtype, rows=rows, t=t, moves=moves)


def _row_lengths(case):
    """Active keys per row of a cache: spread evenly from the longest row down to a third of it."""
    n, t, least = case.get("b") or case["rows"], case["t"], case.get("lq", 1)
    return [max(least, t - (2 * t * i) // (3 * n)) for i in range(n)]


def _cu_seqlens(case):
    """Sequences of 1 to `longest` tokens, in an irregular order that belongs to the case, until the tokens are dealt out."""
    cu, x = [0], 1
    while cu[-1] < case["l"]:
        x = (x * 1103515245 + 12345) % 2 ** 31
        cu.append(min(case["l"], cu[-1] + 1 + x % case["longest"]))
    return cu


def _pairs(n_q, n_k, window, sinks):
    """Visible (row, key) pairs of one head: row i, at position n_k - n_q + i, sees the last `window` keys and the first `sinks`."""
    total = 0
    for pos in range(n_k - n_q, n_k):
        recent = min(pos + 1, window)
        total += recent + min(sinks, pos + 1 - recent)
    return total


def work(case):
    """Bytes (every input read once, every output written once) and operations of one pass."""
    kind, d = case["kind"], case["d"]
    if kind not in ATTENTION:
        return {"bytes": _moved(case) + _list_bytes(case), "flops": 0}
    hq, hkv = case["hq"], case["hkv"]
    if kind in ("train", "packed"):
        cu = _cu_seqlens(case) if kind == "packed" else [0, case["l"]]
        pairs = case["b"] * sum(_pairs(n, n, case["window"], case["sinks"]) for n in (y - x for x, y in zip(cu, cu[1:])))
        tokens = case["b"] * case["l"]
        # q, r, grad_o in, o, dq, dr out; k, v in, dk, dv out; 12 products over the visible pairs
        return {"bytes": 2 * tokens * d * (6 * hq + 4 * hkv), "flops": 24 * pairs * hq * d}
    if kind == "prefix":
        keys = case["p"] * case["b"] + sum(_row_lengths(case))
        read = case["p"] + sum(_row_lengths(case))
        return {"bytes": 2 * d * (3 * case["b"] * hq + 2 * read * hkv), "flops": 8 * keys * hq * d}
    lens, lq = _row_lengths(case), case["lq"]
    pairs = sum(_pairs(lq, n, case["window"], case["sinks"]) for n in lens)
    seen = sum(min(n, case["window"] + lq - 1 + case["sinks"]) for n in lens)
    return {"bytes": 2 * d * (3 * case["b"] * lq * hq + 2 * seen * hkv), "flops": 8 * pairs * hq * d}


def _list_bytes(case):
    if not case["rows"]:
        return 8 * case["moves"]
    table = case["rows"] * -(-case["t"] // case["page"])
    return 8 * case["moves"] + (4 if case["kind"] == "free" else 8) * table + (4 * case["pages"] if case["kind"] == "free" else 0)


def _moved(case):
    """Bytes of k and v that are read and written."""
    key = 2 * 2 * 2 * case["hkv"] * case["d"]        # k and v, in and out, 16 bits
    if case["kind"] == "copy":
        return _real_moves(case) * case["page"] * key
    if case["kind"] == "fork":
        lens = _row_lengths(case)
        return sum(lens[b] % case["page"] for b in _parents(case)) * key
    if case["kind"] == "compact":
        live = sum(-(-n // case["page"]) for n in _row_lengths(case))
        return int(live * (1 - live / case["pages"])) * case["page"] * key      # live pages lie anywhere in the pool
    return 0


def _real_moves(case):
    return case["moves"] - case["moves"] // 4        # the rest pads the list


def _parents(case):
    return [(5 * i) % (case["rows"] - case["moves"]) for i in range(case["moves"])]


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32) * scale).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)

    def pages_of(lens, page, n_pages, m, shared=0):
        """A table whose rows hold the pages of their lengths, scattered over the pool; the first `shared` entries alike."""
        counts = torch.tensor([max(-(-n // page) - shared, 0) for n in lens], device=DEVICE)
        order = torch.randperm(n_pages, generator=g, device=DEVICE).to(torch.int32)
        table = torch.zeros(len(lens), m, dtype=torch.int32, device=DEVICE)
        table[:, :shared] = order[:shared]
        active = torch.arange(m - shared, device=DEVICE) < counts[:, None]
        rest = table[:, shared:]
        rest[active] = order[shared:shared + int(counts.sum())]
        return table

    kind, d = case["kind"], case["d"]
    s = {"case": case}
    if kind in ("train", "packed"):
        b, l, hq, hkv = case["b"], case["l"], case["hq"], case["hkv"]
        q_shape, kv_shape = ((b, hq, l, d), (b, hkv, l, d)) if kind == "train" else ((1, l, hq, d), (1, l, hkv, d))
        s["leaves"] = [normal(*q_shape).requires_grad_(), normal(*q_shape, scale=0.5).requires_grad_(),
                       normal(*kv_shape).requires_grad_(), normal(*kv_shape).requires_grad_()]
        s["grad_o"] = normal(*q_shape)
        s["cu"] = ints(_cu_seqlens(case)) if kind == "packed" else None
        return s
    if kind in ("extend", "decode", "prefix"):
        b, hq, hkv, page, t = case["b"], case["hq"], case["hkv"], case["page"], case["t"]
        lq, p = case.get("lq", 1), case.get("p", 0)
        lens = _row_lengths(case)
        s["q"], s["r"] = normal(b, lq, hq, d), normal(b, lq, hq, d, scale=0.5)
        if page:
            ceiling = [p + n for n in lens]
            m = -(-max(ceiling) // page)
            n_pages = p // page + sum(-(-n // page) for n in lens) + 5
            s["table"] = pages_of(ceiling, page, n_pages, m, shared=p // page)
            s["k"], s["v"] = normal(n_pages, page, hkv, d), normal(n_pages, page, hkv, d)
            s["lens"] = ints(ceiling)
        else:
            s["table"] = None
            s["k"], s["v"] = normal(b, t, hkv, d), normal(b, t, hkv, d)
            s["lens"] = ints(lens)
            if p:
                s["k_prefix"], s["v_prefix"] = normal(p, hkv, d), normal(p, hkv, d)
        return s
    s["k"] = normal(case["pages"], case["page"], case["hkv"], d)
    s["v"] = normal(case["pages"], case["page"], case["hkv"], d)
    if kind == "copy":
        order = torch.randperm(case["pages"], generator=g, device=DEVICE).to(torch.int32)
        n, real = case["moves"], _real_moves(case)
        s["src"], s["dst"] = order[:n].clone(), order[n:2 * n].clone()
        s["src"][real:] = -1
        s["dst"][real:] = -1
        return s
    lens = _row_lengths(case)
    m = -(-case["t"] // case["page"])
    s["lens"] = ints(lens)
    s["table"] = pages_of(lens, case["page"], case["pages"], m)
    if kind == "fork":
        s["parents"] = ints(_parents(case))
        s["children"] = ints(list(range(case["rows"] - case["moves"], case["rows"])))
    if kind == "free":
        s["rows"] = ints(list(range(0, case["rows"], 3)))
    return s


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import parallax_b200 as plx

    case, kind = s["case"], s["case"]["kind"]
    if kind == "train":
        q, r, k, v = s["leaves"]
        o = plx.parallax_func(q, r, k, v, window_size_left=case["window"], sink_tokens=case["sinks"])
        return (o.detach(), *torch.autograd.grad(o, s["leaves"], s["grad_o"]))
    if kind == "packed":
        q, r, k, v = s["leaves"]
        o = plx.parallax_varlen_func(q, r, k, v, window_size_left=case["window"], cu_seqlens=s["cu"], sink_tokens=case["sinks"])
        return (o.detach(), *torch.autograd.grad(o, s["leaves"], s["grad_o"]))
    if kind == "extend" or (kind == "decode" and s["table"] is not None):
        return plx.parallax_attn_with_kvcache(s["q"], s["r"], s["k"], s["v"], page_table=s["table"], seqused_k=s["lens"],
                                              window_size=case["window"], sink_tokens=case["sinks"])
    if kind == "decode":
        return plx.parallax_decode(s["q"], s["r"], s["k"], s["v"], window_size_left=case["window"], seqused_k=s["lens"],
                                   sink_tokens=case["sinks"])
    if kind == "prefix":
        if s["table"] is not None:
            return plx.parallax_attn_with_kvcache(s["q"], s["r"], s["k"], s["v"], page_table=s["table"], seqused_k=s["lens"],
                                                  shared_prefix=case["p"])
        return plx.parallax_decode_shared_prefix(s["q"], s["r"], s["k_prefix"], s["v_prefix"], s["k"], s["v"], seqused_k=s["lens"])
    if kind == "copy":
        plx.parallax_copy_pages(s["k"], s["v"], s["src"], s["dst"])
        return s["k"], s["v"]
    if kind == "fork":
        table, lens, missing = plx.parallax_fork_pages(s["k"], s["v"], s["table"], s["lens"], s["parents"], s["children"])
        return s["k"], s["v"], table, lens, missing
    if kind == "compact":
        table, live = plx.parallax_compact_pages(s["k"], s["v"], s["table"], s["lens"])
        return s["k"], s["v"], table, live
    return plx.parallax_free_pages(s["table"], s["lens"], s["rows"], case["pages"], case["page"])


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    with torch.no_grad():
        if kind in ("train", "packed"):
            return _plain_train(s)
        if kind in ("extend", "decode"):
            return _plain_cache(s)
        if kind == "prefix":
            return _plain_prefix(s)
        if kind == "copy":
            ok = (s["src"] >= 0) & (s["dst"] >= 0)
            src, dst = s["src"][ok].long(), s["dst"][ok].long()
            s["k"][dst] = s["k"][src]
            s["v"][dst] = s["v"][src]
            return s["k"], s["v"]
        return {"fork": _plain_fork, "compact": _plain_compact, "free": _plain_free}[kind](s, case["page"], case["pages"])


def _visible(pos, key, window, sinks):
    """Row at position `pos` sees key `key`: none after it, the last `window` of those, and the first `sinks`."""
    return (key <= pos) & ((key > pos - window) | (key < sinks))


def _weights(q, r, k, ok, scale):
    """p, and 1 + c - s2, of the rows in 32 bits; p is zero where nothing is visible."""
    s1 = (q @ k.transpose(-1, -2) * scale).masked_fill(~ok, -math.inf)
    s2 = r @ k.transpose(-1, -2)
    m = s1.amax(-1, keepdim=True)
    p = torch.exp(s1 - torch.where(m == -math.inf, torch.zeros_like(m), m))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return p, 1 + (p * s2).sum(-1, keepdim=True) - s2


def _plain_train(s):
    case = s["case"]
    packed = case["kind"] == "packed"
    hq, hkv, l, d = case["hq"], case["hkv"], case["l"], case["d"]
    scale = d ** -0.5
    q, r, k, v, go = (x.detach().float() for x in (*s["leaves"], s["grad_o"]))
    if packed:
        q, r, k, v, go = (x.transpose(1, 2) for x in (q, r, k, v, go))
    b = q.shape[0]
    q, r, go = (x.reshape(b, hkv, hq // hkv, l, d) for x in (q, r, go))
    k, v = k.unsqueeze(2), v.unsqueeze(2)
    at = torch.arange(l, device=q.device)
    ok = _visible(at[:, None], at[None, :], case["window"], case["sinks"])
    if packed:
        seq = torch.searchsorted(s["cu"].long(), at, right=True) - 1
        first = s["cu"].long()[seq]
        ok = _visible(at[:, None] - first[:, None], at[None, :] - first[:, None], case["window"], case["sinks"])
        ok = ok & (seq[:, None] == seq[None, :])
    p, e = _weights(q, r, k, ok, scale)
    w = p * e
    o = w @ v
    a = go @ v.transpose(-1, -2)
    b_row, t_row = (p * a).sum(-1, keepdim=True), (go * o).sum(-1, keepdim=True)
    delta = a - b_row
    gl = w * delta + p * (b_row - t_row)
    gu = -p * delta
    dq = gl @ k * scale
    dr = gu @ k
    dk = (gl.transpose(-1, -2) @ q * scale + gu.transpose(-1, -2) @ r).sum(2)
    dv = (w.transpose(-1, -2) @ go).sum(2)
    out = [x.reshape(b, hq, l, d) for x in (o, dq, dr)] + [dk, dv]
    if packed:
        out = [x.transpose(1, 2) for x in out]
    return tuple(x.to(s["grad_o"].dtype) for x in out)


def _rows_of_cache(s, x, n):
    """The first `n` keys of every row as (B, H_kv, n, D) in 32 bits."""
    if s["table"] is not None:
        x = x[s["table"].long()].flatten(1, 2)
    return x[:, :n].float().transpose(1, 2)


def _grouped(x, hkv):
    """(B, L_q, H_q, D) -> (B, H_kv, n_rep * L_q, D) in 32 bits."""
    b, lq, hq, d = x.shape
    return x.float().transpose(1, 2).reshape(b, hkv, hq // hkv * lq, d)


def _plain_cache(s):
    case = s["case"]
    b, lq, hq, hkv, d = case["b"], case["lq"], case["hq"], case["hkv"], case["d"]
    q, r = _grouped(s["q"], hkv), _grouped(s["r"], hkv)
    k, v = _rows_of_cache(s, s["k"], case["t"]), _rows_of_cache(s, s["v"], case["t"])
    pos = s["lens"].long()[:, None] - lq + torch.arange(lq, device=q.device)
    ok = _visible(pos[:, :, None], torch.arange(k.shape[2], device=q.device), case["window"], case["sinks"])
    p, e = _weights(q, r, k, ok[:, None].repeat(1, 1, hq // hkv, 1), d ** -0.5)
    return ((p * e) @ v).reshape(b, hq, lq, d).transpose(1, 2).to(s["q"].dtype)


def _plain_prefix(s):
    case = s["case"]
    b, hq, hkv, d, p_len, t = case["b"], case["hq"], case["hkv"], case["d"], case["p"], case["t"]
    rep, scale = hq // hkv, d ** -0.5
    q, r = s["q"].float().view(b, hkv, rep, d), s["r"].float().view(b, hkv, rep, d)
    if s["table"] is not None:
        n = p_len // case["page"]
        kp, vp = (x[s["table"][0, :n].long()].flatten(0, 1) for x in (s["k"], s["v"]))
        k, v = (x[s["table"][:, n:].long()].flatten(1, 2) for x in (s["k"], s["v"]))
        own_lens = s["lens"] - p_len
    else:
        kp, vp, k, v, own_lens = s["k_prefix"], s["v_prefix"], s["k"], s["v"], s["lens"]
    kp, vp = kp.float().transpose(0, 1), vp.float().transpose(0, 1)                 # (H_kv, P, D)
    k, v = k.float().transpose(1, 2), v.float().transpose(1, 2)                     # (B, H_kv, T, D)
    rows = lambda x: x.transpose(0, 1).reshape(hkv, b * rep, d)                    # noqa: E731  all rows of a kv head
    back = lambda x: x.view(hkv, b, rep, -1).transpose(0, 1)                       # noqa: E731
    ok = torch.arange(k.shape[2], device=q.device) < own_lens.long()[:, None, None, None]
    s1 = torch.cat((back(rows(q) @ kp.transpose(1, 2)), (q @ k.transpose(2, 3)).masked_fill(~ok, -math.inf)), -1) * scale
    s2 = torch.cat((back(rows(r) @ kp.transpose(1, 2)), r @ k.transpose(2, 3)), -1)
    p = torch.softmax(s1, -1)
    w = p * (1 + (p * s2).sum(-1, keepdim=True) - s2)
    shared = w[..., :p_len].transpose(0, 1).reshape(hkv, b * rep, p_len) @ vp
    return (back(shared) + w[..., p_len:] @ v).reshape(b, 1, hq, d).to(s["q"].dtype)


def _live(table, lens, page, pages):
    """Which pages of the pool some row's active entries name (a truth value each), and those entries (a mask)."""
    active = torch.arange(table.shape[1], device=table.device) * page < lens[:, None]
    live = torch.zeros(pages, dtype=torch.bool, device=table.device)
    live[table[active].long()] = True
    return live, active


def _plain_fork(s, page, pages):
    table, lens, parents, children = s["table"], s["lens"], s["parents"].long(), s["children"].long()
    live, _ = _live(table, lens, page, pages)
    free = torch.nonzero(~live).flatten()
    new_table, new_lens = table.clone(), lens.clone()
    new_table[children] = table[parents]
    new_lens[children] = lens[parents]
    part = lens[parents].long() % page
    needs = part > 0
    taken = free[:int(needs.sum())]
    row, tail = parents[needs], part[needs]
    slot = lens[row].long() // page
    old = table[row, slot].long()
    new_table[children[needs], slot] = taken.to(table.dtype)
    keys = (torch.arange(page, device=table.device) < tail[:, None])[:, :, None, None]
    for x in (s["k"], s["v"]):
        x[taken] = torch.where(keys, x[old], x[taken])
    return s["k"], s["v"], new_table, new_lens, torch.zeros(1, dtype=torch.int32, device=table.device)


def _plain_compact(s, page, pages):
    table, lens = s["table"], s["lens"]
    live, active = _live(table, lens, page, pages)
    n = live.sum()
    at = torch.arange(pages, device=table.device)
    src = torch.nonzero(live & (at >= n)).flatten()
    dst = torch.nonzero(~live & (at < n)).flatten()
    moved = at.clone()
    moved[src] = dst
    new_table = torch.where(active, moved[table.long().clamp(0, pages - 1)].to(table.dtype), table)
    s["k"][dst] = s["k"][src]
    s["v"][dst] = s["v"][src]
    return s["k"], s["v"], new_table, n.to(torch.int32).view(1)


def _plain_free(s, page, pages):
    lens = s["lens"].clone()
    lens[s["rows"].long()] = 0
    live, _ = _live(s["table"], lens, page, pages)
    free = torch.full((pages,), -1, dtype=torch.int32, device=lens.device)
    found = torch.nonzero(~live).flatten().to(torch.int32)
    free[:found.numel()] = found
    return lens, free, torch.tensor([found.numel()], dtype=torch.int32, device=lens.device)


# --------------------------------------------------------------------------- #
# the definition, in 64 bits
# --------------------------------------------------------------------------- #
def exact(case, seed):
    """o = (1 + E[s2]) E[v] - E[s2 v] under the softmax of s1, one head after the other, gradients by autograd.  Pages are only
    moved: there is nothing computed about them."""
    if case["kind"] not in ATTENTION:
        return None
    s = prepare(case, seed)
    if case["kind"] in ("train", "packed"):
        return _exact_train(s, case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    rep, lq, p_len = case["hq"] // case["hkv"], case.get("lq", 1), case.get("p", 0)
    for b, n in enumerate(s["lens"].tolist()):
        if s["table"] is not None:
            k, v = (x[s["table"][b].long()].flatten(0, 1)[:n].double() for x in (s["k"], s["v"]))
        else:
            k, v = (x[b, :n].double() for x in (s["k"], s["v"]))
            if p_len:
                k, v = torch.cat((s["k_prefix"].double(), k)), torch.cat((s["v_prefix"].double(), v))
        i = torch.arange(k.shape[0] - lq, k.shape[0], device=k.device)[:, None]
        j = torch.arange(k.shape[0], device=k.device)[None]
        hidden = j > i
        if "window" in case:
            hidden |= (i - j >= case["window"]) & (j >= case["sinks"])
        for h in range(case["hkv"]):
            q, r = (x[b, :, h * rep:(h + 1) * rep].double().transpose(0, 1) for x in (s["q"], s["r"]))
            out[b, :, h * rep:(h + 1) * rep] = _expectation(q, r, k[:, h], v[:, h], hidden).transpose(0, 1)
    return out


def _expectation(q, r, k, v, hidden):
    logits = torch.einsum("...id,jd->...ij", q, k) / math.sqrt(q.shape[-1])
    prob = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
    tilt = torch.einsum("...id,jd->...ij", r, k)
    mean = torch.einsum("...ij,jd->...id", prob, v)
    return mean + (prob * tilt).sum(-1, keepdim=True) * mean - torch.einsum("...ij,jd->...id", prob * tilt, v)


def _exact_train(s, case):
    packed, rep = case["kind"] == "packed", case["hq"] // case["hkv"]
    tensors = [x.detach().double() for x in (*s["leaves"], s["grad_o"])]
    if packed:
        tensors = [x.transpose(1, 2) for x in tensors]
    q, r, k, v, go = tensors
    outs = [torch.zeros_like(x) for x in (q, q, r, k, v)]
    bounds = _cu_seqlens(case) if packed else [0, case["l"]]
    for b in range(q.shape[0]):
        for lo, hi in zip(bounds, bounds[1:]):
            i = torch.arange(hi - lo, device=q.device)[:, None]
            j = torch.arange(hi - lo, device=q.device)[None]
            hidden = (j > i) | ((i - j >= case["window"]) & (j >= case["sinks"]))
            # all heads at once where they are short, else one by one
            for h0 in range(0, case["hkv"], 1 if hi - lo > 2048 else case["hkv"]):
                h1 = h0 + (1 if hi - lo > 2048 else case["hkv"])
                parts = [x[b, h0 * rep:h1 * rep, lo:hi].unflatten(0, (-1, rep)).clone().requires_grad_() for x in (q, r)]
                parts += [x[b, h0:h1, lo:hi].clone().requires_grad_() for x in (k, v)]
                with torch.enable_grad():
                    qq, rr, kk, vv = parts
                    wide = lambda x: x[:, None].expand(-1, rep, -1, -1)                         # noqa: E731
                    logits = (qq @ wide(kk).transpose(-1, -2) / math.sqrt(case["d"])).masked_fill(hidden, -math.inf)
                    prob, tilt = torch.softmax(logits, -1), rr @ wide(kk).transpose(-1, -2)
                    mean = prob @ wide(vv)
                    o = mean + (prob * tilt).sum(-1, keepdim=True) * mean - (prob * tilt) @ wide(vv)
                grads = torch.autograd.grad(o, parts, go[b, h0 * rep:h1 * rep, lo:hi].unflatten(0, (-1, rep)))
                outs[0][b, h0 * rep:h1 * rep, lo:hi] = o.detach().flatten(0, 1)
                for dst, x in zip(outs[1:3], grads[:2]):
                    dst[b, h0 * rep:h1 * rep, lo:hi] = x.flatten(0, 1)
                for dst, x in zip(outs[3:], grads[2:]):
                    dst[b, h0:h1, lo:hi] = x
    return tuple(x.transpose(1, 2) for x in outs) if packed else tuple(outs)
