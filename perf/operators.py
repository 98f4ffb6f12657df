"""Measured cases of the serving operators: prompt attention over packed sequences, single-token
attention of a batch over a paged cache whose sequences share a prefix, and the page operations
of that cache (fork, free, reserve, write, compact).

`run` computes a case either with elementary torch operations in 32 bits (`own` false) or with
the calls a user makes of this repository's package (`own` true).  `exact` restates each
definition in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------- cases
def listed():
    gqa = dict(heads_q=32, heads_kv=8, head_dim=128, dtype="bf16")
    small = dict(heads_q=14, heads_kv=2, head_dim=64, dtype="bf16")    # the decode layer's heads
    return [
        # A few short chat turns prefilled in one call: latency counts.
        dict(name="packed_short", kind="packed", **small, lse=False,
             lens_q="1,5,23,60,7,131,64,33", lens_k="1,5,23,60,7,131,64,33"),
        # An ordinary prefill batch: prompts of very different lengths, packed.
        dict(name="packed_ragged", kind="packed", **gqa, lse=False,
             lens_q="37,1024,211,2048,640,129,900,77,1500,333,256,1801,18,512,1290,700",
             lens_k="37,1024,211,2048,640,129,900,77,1500,333,256,1801,18,512,1290,700"),
        # One long prompt.
        dict(name="packed_long", kind="packed", **gqa, lse=False, lens_q="8192", lens_k="8192"),
        # A prompt prefilled in chunks: the queries are the last tokens of longer contexts; the
        # log-sum-exp is kept, as for joining with another part of the context.
        dict(name="packed_chunk", kind="packed", **gqa, lse=True, lens_q="512,512,300,1",
             lens_k="4096,1111,300,2049"),
        # Single precision, as the framework's other operators offer it.
        dict(name="packed_f32", kind="packed", heads_q=14, heads_kv=2, head_dim=64, dtype="f32",
             lse=False, lens_q="700,45,1024,3", lens_k="700,45,1024,3"),
        # Four samples of one short prompt, a few tokens in: latency counts.
        dict(name="shared_small", kind="shared", **small, batch=4, page=16, prefix=512,
             own_min=1, own_max=40),
        # A batch of samples of one prompt.
        dict(name="shared_samples", kind="shared", **gqa, batch=32, page=64, prefix=4096,
             own_min=1, own_max=512),
        # A large batch behind one long document.
        dict(name="shared_document", kind="shared", **gqa, batch=128, page=64, prefix=32768,
             own_min=5, own_max=1024),
        # Nothing shared: sequences of all lengths, each with its own pages.
        dict(name="paged_ragged", kind="shared", **gqa, batch=16, page=32, prefix=0, own_min=1,
             own_max=8191),
        # Parallel sampling: every prompt of a batch is continued four times.
        dict(name="fork_samples", kind="fork", heads_kv=4, head_dim=128, dtype="bf16", page=64,
             layers=16, pages=2048, parents=64, children=4, len_min=100, len_max=1500),
        # A cache with half of its pages let go, made dense again.
        dict(name="compact_half", kind="compact", heads_kv=4, head_dim=128, dtype="bf16", page=64,
             layers=16, pages=2048, slots=64, live=1030),
        # A batch of requests leaves and the next one's prompts come in: latency counts.
        dict(name="turnover", kind="turnover", heads_kv=2, head_dim=64, dtype="bf16", page=16,
             layers=2, pages=1500, slots=32, len_min=1, len_max=300),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Seconds that a case cannot do without at nominal rates, and the plain form's score bytes."""
    w = work(case)
    pad = 0
    if case["kind"] == "packed":
        q, k = _lens(case["lens_q"]), _lens(case["lens_k"])
        pad = len(q) * case["heads_q"] * max(q) * max(k) * 4
    if case["kind"] == "shared":
        keys = case["prefix"] + case["own_max"]
        pad = 4 * case["batch"] * (keys * case["heads_q"]
                                   + case["own_max"] * case["heads_kv"] * case["head_dim"])
    rate = 5e13 if case["dtype"] == "f32" else 1e15
    return max(w["bytes"] / 6e12, w["flops"] / rate), pad


def draw(rng):
    """One more case of the listed ones' ranges: kinds, head layouts, lengths over their logarithm."""
    most = max(_cost(c)[0] for c in listed())
    while True:
        kind = rng.choice(["packed", "packed", "shared", "shared", "fork", "compact", "turnover"])
        heads_kv, group = rng.choice([(1, 8), (2, 7), (8, 4), (4, 8), (8, 1), (3, 5), (16, 2)])
        case = dict(kind=kind, heads_kv=heads_kv, head_dim=rng.choice([64, 128]), dtype="bf16")
        if kind == "packed":
            n = _log_int(rng, 1, 24)
            q = [_log_int(rng, 1, 8192 if n < 3 else 2500) for _ in range(n)]
            more = rng.random() < 0.4
            k = [v + (_log_int(rng, 1, 4096) if more else 0) for v in q]
            if rng.random() < 0.2:
                case["dtype"] = "f32"
                q, k = [min(v, 1024) for v in q], [min(v, 1500) for v in k]
            case.update(heads_q=heads_kv * group, lse=rng.random() < 0.5,
                        lens_q=",".join(map(str, q)), lens_k=",".join(map(str, k)))
        elif kind == "shared":
            case.update(heads_q=heads_kv * group, batch=_log_int(rng, 1, 160),
                        page=rng.choice([16, 32, 64, 128]),
                        prefix=rng.choice([0, _log_int(rng, 16, 32768), _log_int(rng, 16, 32768)]),
                        own_min=1, own_max=_log_int(rng, 2, 8192))
        elif kind == "fork":
            case.update(page=rng.choice([16, 32, 64, 128]), layers=_log_int(rng, 1, 16),
                        pages=_log_int(rng, 200, 2048), parents=_log_int(rng, 1, 64),
                        children=_log_int(rng, 1, 6), len_min=1, len_max=_log_int(rng, 4, 1500))
        elif kind == "compact":
            pages = _log_int(rng, 50, 2048)
            slots = _log_int(rng, 2, 64)
            case.update(page=rng.choice([16, 32, 64, 128]), layers=_log_int(rng, 1, 16), pages=pages,
                        slots=slots, live=max(slots, int(pages * rng.uniform(0.1, 0.9))))
        else:
            case.update(page=rng.choice([16, 32, 64, 128]), layers=_log_int(rng, 1, 4),
                        pages=_log_int(rng, 300, 3000), slots=_log_int(rng, 1, 64), len_min=1,
                        len_max=_log_int(rng, 2, 2048))
        if kind in ("fork", "compact", "turnover"):
            if _cache_bytes(case) > 5e9 or _pages_used(case) > case["pages"]:
                continue
        seconds, pad = _cost(case)
        if seconds <= most and pad <= 1.1e10:
            return case


# ---------------------------------------------------------------------- sizes of a case
def _lens(text):
    return [int(v) for v in text.split(",")]


def _spread(n, lo, hi):
    """n lengths over [lo, hi], in a shuffled order that is the same for everybody."""
    step = next(s for s in (7, 11, 13, 17, 19, 23) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((i * step) % n) // max(1, n - 1) for i in range(n)]


def _pages_of(length, page):
    return (length + page - 1) // page


def _pages_used(case):
    if case["kind"] == "fork":
        lens = _spread(case["parents"], case["len_min"], case["len_max"])
        return sum(_pages_of(v, case["page"]) for v in lens) + case["parents"] * case["children"]
    if case["kind"] == "turnover":
        lens = _spread(case["slots"], case["len_min"], case["len_max"])
        return sum(_pages_of(v, case["page"]) for v in lens)
    return case["live"]


def _row_bytes(case):
    return case["heads_kv"] * case["head_dim"] * (4 if case["dtype"] == "f32" else 2)


def _cache_bytes(case):
    return 2 * case["layers"] * case["pages"] * case["page"] * _row_bytes(case)


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "packed":
        q, k = _lens(case["lens_q"]), _lens(case["lens_k"])
        hq, hk, d = case["heads_q"], case["heads_kv"], case["head_dim"]
        pairs = 0
        for a, b in zip(q, k):      # query i sees keys 0 .. i + b - a
            first, last = max(0, b - a + 1), b
            rows = min(a, b)
            pairs += (first + last) * rows // 2 if a <= b else b * (b + 1) // 2
        return {"bytes": size * d * (2 * sum(q) * hq + 2 * sum(k) * hk)
                + (4 * sum(q) * hq if case["lse"] else 0), "flops": 4 * pairs * hq * d}
    if kind == "shared":
        lens = _spread(case["batch"], case["own_min"], case["own_max"])
        hq, hk, d = case["heads_q"], case["heads_kv"], case["head_dim"]
        tables = sum(_pages_of(case["prefix"] + v, case["page"]) for v in lens)
        return {"bytes": size * d * (2 * (case["prefix"] + sum(lens)) * hk + 2 * len(lens) * hq)
                + 4 * tables,
                "flops": 4 * hq * d * sum(case["prefix"] + v for v in lens)}
    row = _row_bytes(case)
    if kind == "fork":
        lens = _spread(case["parents"], case["len_min"], case["len_max"])
        c = case["children"]
        part = sum(v % case["page"] for v in lens)
        entries = sum(_pages_of(v, case["page"]) for v in lens)
        return {"bytes": 2 * case["layers"] * row * part * (1 + c) + 4 * entries * (1 + c)
                + 4 * case["pages"], "flops": 0}
    if kind == "compact":
        moved = sum(1 for p in _live_pages(case) if p >= case["live"])
        return {"bytes": 2 * 2 * case["layers"] * row * case["page"] * moved + 8 * case["pages"],
                "flops": 0}
    tokens = sum(_spread(case["slots"], case["len_min"], case["len_max"]))
    return {"bytes": 2 * 2 * row * tokens + 8 * case["pages"], "flops": 0}


def _live_pages(case):
    """The pages in use before a compaction: a scattered choice that depends on the sizes alone."""
    rs = np.random.RandomState(case["pages"] + 7 * case["live"])
    return rs.permutation(case["pages"])[: case["live"]]


# ---------------------------------------------------------------------------- inputs
def _randn(gen, *shape, dtype):
    return torch.randn(*shape, device="cuda", generator=gen, dtype=dtype)


def _i32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _qkv(gen, tokens_q, tokens_k, case):
    """Q, K, V as slices of one fused projection's rows (heads of q | k | v); keys carry an offset
    for each channel, as trained projections give them."""
    hq, hk, d, dt = case["heads_q"], case["heads_kv"], case["head_dim"], DTYPES[case["dtype"]]
    rows = max(tokens_q, tokens_k)
    fused = _randn(gen, rows, hq + 2 * hk, d, dtype=dt)
    fused[:, hq:hq + hk] += _randn(gen, hk, d, dtype=dt)
    return fused[:tokens_q, :hq], fused[:tokens_k, hq:hq + hk], fused[:tokens_k, hq + hk:]


def _cache(gen, case, layers, pages):
    shape = (layers, pages, case["heads_kv"], case["page"], case["head_dim"])
    dt = DTYPES[case["dtype"]]
    return _randn(gen, *shape, dtype=dt), _randn(gen, *shape, dtype=dt)


def _package():
    """This repository's package, as its documentation says to import it."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "enigma-dsl_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import enigma
    from enigma import kv_cache
    return enigma.cuda_ops, kv_cache


def _page_state(case, seed):
    """The cache and its page map before a page operation, as host arrays and device pages."""
    kind, page = case["kind"], case["page"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 31))
    k, v = _cache(gen, case, case["layers"], case["pages"])
    refs = np.zeros(case["pages"], np.int32)
    if kind == "fork":
        n, c = case["parents"], case["children"]
        slots, lens_of = n * (1 + c), _spread(n, case["len_min"], case["len_max"])
        width = _pages_of(max(lens_of), page) + 1
        order = rs.permutation(case["pages"])
    elif kind == "compact":
        slots = case["slots"]
        sizes = np.random.RandomState(case["live"] + slots)
        cuts = np.sort(sizes.choice(np.arange(1, case["live"]), slots - 1, replace=False))
        counts = np.diff(np.concatenate([[0], cuts, [case["live"]]]))
        lens_of = [int(x) * page - int(rs.randint(0, page)) for x in counts]
        width = int(counts.max())
        order = rs.permutation(_live_pages(case))
    else:
        slots, lens_of = case["slots"], _spread(case["slots"], case["len_min"], case["len_max"])
        width = _pages_of(case["len_max"], page) + 1
        order = rs.permutation(case["pages"])
    table = np.full((slots, width), -1, np.int32)
    lens = np.zeros(slots, np.int32)
    at = 0
    for s, length in enumerate(lens_of):
        m = _pages_of(length, page)
        table[s, :m] = order[at:at + m]
        refs[order[at:at + m]] = 1
        lens[s] = length
        at += m
    return gen, rs, k, v, table, lens, refs


def prepare(case, seed):
    kind = case["kind"]
    if kind == "packed":
        gen = torch.Generator(device="cuda").manual_seed(seed)
        lq, lk = _lens(case["lens_q"]), _lens(case["lens_k"])
        q, k, v = _qkv(gen, sum(lq), sum(lk), case)
        state = dict(case=case, q=q, k=k, v=v, lens_q=lq, lens_k=lk)
        if own:
            ops, _ = _package()
            state["ops"] = ops
            state["plan"] = ops.PackedPlan(lq, lk, heads_q=case["heads_q"], heads_kv=case["heads_kv"])
        else:
            state["index_q"], state["index_k"] = _padded(lq), _padded(lk)
        return state
    if kind == "shared":
        gen = torch.Generator(device="cuda").manual_seed(seed)
        rs = np.random.RandomState(seed % (1 << 31))
        own_lens = _spread(case["batch"], case["own_min"], case["own_max"])
        page, prefix = case["page"], case["prefix"]
        head = prefix // page                       # whole pages of the prefix: shared
        width = _pages_of(prefix + max(own_lens), page)
        tails = [_pages_of(prefix + n, page) - head for n in own_lens]
        pages = head + sum(tails) + 3
        order = rs.permutation(pages)
        table = np.full((case["batch"], width), -1, np.int32)
        table[:, :head] = order[:head]
        at = head
        for b, m in enumerate(tails):
            table[b, head:head + m] = order[at:at + m]
            at += m
        k, v = _cache(gen, case, 1, pages)
        k += _randn(gen, case["heads_kv"], 1, case["head_dim"], dtype=k.dtype)
        if prefix % page:       # the prefix's last, partly filled page was copied by the fork
            first = table[0, head]
            for b in range(1, case["batch"]):
                k[0, table[b, head], :, : prefix % page] = k[0, first, :, : prefix % page]
                v[0, table[b, head], :, : prefix % page] = v[0, first, :, : prefix % page]
        q = _randn(gen, case["batch"], case["heads_q"], case["head_dim"], dtype=k.dtype)
        return dict(case=case, q=q, k=k[0], v=v[0], table=_i32(table), prefix=prefix,
                    lens=_i32([prefix + n for n in own_lens]), own_max=max(own_lens),
                    ops=_package()[0] if own else None)
    gen, rs, k, v, table, lens, refs = _page_state(case, seed)
    state = dict(case=case, k=k, v=v, table=_i32(table), lens=_i32(lens), refs=_i32(refs))
    if kind == "fork":
        n, c = case["parents"], case["children"]
        state["parents"] = _i32(np.repeat(np.arange(n), c))
        state["children"] = _i32(n + rs.permutation(n * c))
    elif kind == "compact":
        state["map"] = [state[x].clone() for x in ("table", "refs")]
    else:
        state["slots"] = _i32(rs.permutation(case["slots"]))
        new = [int(lens[s]) for s in state["slots"].tolist()][::-1]
        state["new_lens"] = _i32(new)
        d, hk = case["head_dim"], case["heads_kv"]
        fused = _randn(gen, sum(new), 3 * hk, d, dtype=k.dtype)     # q | k | v of one layer
        state["new_k"], state["new_v"] = fused[:, hk:2 * hk], fused[:, 2 * hk:]
        state["starts"] = torch.zeros_like(state["new_lens"])
        state["cu"] = _i32(np.concatenate([[0], np.cumsum(new)]))
    if own:
        _, kv_cache = _package()
        state["cache"] = kv_cache.PagedKVCache(k, v, state["table"], state["lens"], state["refs"])
    return state


def _padded(lens):
    """Rows of the packed tensor for [sequence, position], and which of them exist."""
    n, m = len(lens), max(lens)
    starts = np.concatenate([[0], np.cumsum(lens)[:-1]])
    pos = np.arange(m)
    live = pos[None, :] < np.asarray(lens)[:, None]
    rows = np.where(live, starts[:, None] + pos[None, :], 0)
    return (torch.from_numpy(rows).cuda(), torch.from_numpy(live).cuda(),
            torch.tensor(lens, device="cuda"))


# ------------------------------------------------------------------------------ plain forms
def _softmax_parts(s):
    """Weights and log-sum-exp of scores whose masked entries are -inf; an empty row gives zeros."""
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    lse = (m + torch.log(z))[..., 0]
    return p / torch.where(z > 0, z, torch.ones_like(z)), lse


def _plain_packed(st):
    case = st["case"]
    (rows_q, live_q, len_q), (rows_k, live_k, len_k) = st["index_q"], st["index_k"]
    group = case["heads_q"] // case["heads_kv"]
    q = st["q"].float()[rows_q].permute(0, 2, 1, 3)                     # [n, Hq, Mq, D]
    k = st["k"].float()[rows_k].permute(0, 2, 1, 3)
    v = st["v"].float()[rows_k].permute(0, 2, 1, 3)
    n, hk, mk, d = k.shape
    mq = q.shape[2]
    q = q.reshape(n, hk, group * mq, d)
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))     # [n, Hkv, G Mq, Mk]
    s = s.view(n, hk, group, mq, mk)
    i = torch.arange(mq, device=s.device)[None, :, None] + (len_k - len_q)[:, None, None]
    seen = live_k[:, None, :] & (torch.arange(mk, device=s.device)[None, None, :] <= i)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    p, lse = _softmax_parts(s)
    del s
    o = torch.matmul(p.view(n, hk, group * mq, mk), v).view(n, hk * group, mq, d)
    o = o.permute(0, 2, 1, 3)[live_q].to(st["q"].dtype)                 # packed rows again
    if not case["lse"]:
        return o
    return o, lse.view(n, hk * group, mq).permute(0, 2, 1)[live_q]


def _plain_shared(st):
    case = st["case"]
    b, hk, d, page, prefix = (case["batch"], case["heads_kv"], case["head_dim"], case["page"],
                              st["prefix"])
    q = st["q"].float().view(b, hk, -1, d)
    g = q.shape[2]
    pos = torch.arange(prefix, device=q.device)
    at = st["table"][0, pos // page].long()
    kp = st["k"][at, :, pos % page].float().permute(1, 2, 0)            # [Hkv, D, prefix]
    vp = st["v"][at, :, pos % page].float().permute(1, 0, 2)
    sp = torch.matmul(q.permute(1, 0, 2, 3).reshape(hk, b * g, d), kp).view(hk, b, g, prefix)
    pos = prefix + torch.arange(st["own_max"], device=q.device)
    at = st["table"][:, pos // page].long()
    there = pos[None, :] < st["lens"][:, None]
    at = torch.where(there, at, torch.zeros_like(at))
    ks = st["k"][at, :, pos % page].float().permute(0, 2, 3, 1)         # [B, Hkv, D, own]
    vs = st["v"][at, :, pos % page].float().permute(0, 2, 1, 3)
    so = torch.matmul(q, ks).masked_fill(~there[:, None, None], -math.inf)
    s = torch.cat([sp.permute(1, 0, 2, 3), so], -1) * (1.0 / math.sqrt(d))
    p, _ = _softmax_parts(s)
    op = torch.matmul(p[..., :prefix].permute(1, 0, 2, 3).reshape(hk, b * g, prefix), vp)
    o = op.view(hk, b, g, d).permute(1, 0, 2, 3) + torch.matmul(p[..., prefix:], vs)
    return o.reshape(b, hk * g, d).to(st["q"].dtype)


def _add_refs(refs, entries, by):
    e = entries.reshape(-1)
    e = e[e >= 0].long()
    refs.index_add_(0, e, torch.full_like(e, by, dtype=torch.int32))


def _lowest_free(refs, count):
    return torch.nonzero(refs == 0)[:, 0][:count].to(torch.int32)


def _plain_fork(st):
    """Children let go of what they held, then share their parent's full pages; a partly filled
    last page is copied to the lowest free page, in the order of the request."""
    k, v, table, lens, refs = st["k"], st["v"], st["table"], st["lens"], st["refs"]
    page = st["case"]["page"]
    parents, children = st["parents"].long(), st["children"].long()
    _add_refs(refs, table[children], -1)
    length = lens[parents]
    full, fill = length // page, length % page
    rows = table[parents]
    col = torch.arange(table.shape[1], device=table.device)
    rows = torch.where(col[None] < full[:, None], rows, torch.full_like(rows, -1))
    _add_refs(refs, rows, 1)
    part = torch.nonzero(fill > 0)[:, 0]
    dst = _lowest_free(refs, part.numel())
    src = table[parents[part], full[part].long()].long()
    rows[part, full[part].long()] = dst
    refs[dst.long()] = 1
    table[children] = rows
    lens[children] = length
    keep = torch.arange(page, device=k.device)[None, :] < fill[part][:, None]       # [n, page]
    keep = keep[None, :, None, :, None]
    k[:, dst.long()] = torch.where(keep, k[:, src], k[:, dst.long()])
    v[:, dst.long()] = torch.where(keep, v[:, src], v[:, dst.long()])
    return k, v, table, lens, refs


def _plain_compact(st):
    """The n live pages take the page numbers below n: the live pages above go, in order, to the
    holes below."""
    st["table"].copy_(st["map"][0])
    st["refs"].copy_(st["map"][1])
    k, v, table, refs = st["k"], st["v"], st["table"], st["refs"]
    live = refs > 0
    n = live.sum()
    number = torch.arange(refs.numel(), device=refs.device)
    holes = torch.nonzero(~live & (number < n))[:, 0]
    moved = torch.nonzero(live & (number >= n))[:, 0]
    k[:, holes] = k[:, moved]
    v[:, holes] = v[:, moved]
    refs[holes] = refs[moved]
    refs[moved] = 0
    number[moved] = holes
    table.copy_(torch.where(table >= 0, number[table.clamp(min=0).long()].to(torch.int32), table))
    return k, v, table, refs


def _plain_turnover(st):
    k, v, table, lens, refs = st["k"], st["v"], st["table"], st["lens"], st["refs"]
    page, slots = st["case"]["page"], st["slots"].long()
    _add_refs(refs, table[slots], -1)
    table[slots] = -1
    need = (st["new_lens"] + page - 1) // page
    col = torch.arange(table.shape[1], device=table.device)
    wanted = col[None] < need[:, None]
    free = _lowest_free(refs, table.numel())
    rank = torch.cumsum(wanted.reshape(-1).int(), 0).view(wanted.shape) - 1
    rows = torch.where(wanted, free[rank.clamp(min=0, max=free.numel() - 1).long()],
                       torch.full_like(rank, -1, dtype=torch.int32))
    table[slots] = rows
    refs[rows[wanted].long()] = 1
    lens[slots] = st["new_lens"]
    token = torch.arange(st["new_k"].shape[0], device=k.device)
    i = torch.searchsorted(st["cu"], token.int(), right=True) - 1
    pos = token - st["cu"][i] + st["starts"][i]
    at = table[slots[i], pos // page].long()
    k[1 % k.shape[0], at, :, pos % page] = st["new_k"]
    v[1 % k.shape[0], at, :, pos % page] = st["new_v"]
    return k, v, table, lens, refs


# ------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"packed": _plain_packed, "shared": _plain_shared, "fork": _plain_fork,
                "compact": _plain_compact, "turnover": _plain_turnover}[kind](state)
    if kind in ("packed", "shared"):
        ops = state["ops"]
        if kind == "packed":
            return ops.sdpa_packed(state["q"], state["k"], state["v"], state["plan"],
                                   return_lse=case["lse"])
        return ops.sdpa_shared_prefix(state["q"], state["k"], state["v"], state["table"],
                                      state["lens"], prefix_len=state["prefix"])
    cache = state["cache"]
    if kind == "fork":
        cache.fork(state["parents"], state["children"])
        return cache.k, cache.v, cache.table, cache.lens, cache.refs
    if kind == "compact":
        cache.table.copy_(state["map"][0])
        cache.refs.copy_(state["map"][1])
        cache.compact()
        return cache.k, cache.v, cache.table, cache.refs
    cache.free(state["slots"])
    cache.reserve(state["slots"], state["new_lens"])
    cache.write(1 % cache.k.shape[0], state["new_k"], state["new_v"], state["slots"],
                state["starts"], state["cu"])
    return cache.k, cache.v, cache.table, cache.lens, cache.refs


# ----------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, one sequence (or page) after the other."""
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "packed":
        group = case["heads_q"] // case["heads_kv"]
        outs, lses, at_q, at_k = [], [], 0, 0
        for a, b in zip(st["lens_q"], st["lens_k"]):
            o = torch.zeros(a, case["heads_q"], case["head_dim"], dtype=torch.float64, device="cuda")
            e = torch.zeros(a, case["heads_q"], dtype=torch.float64, device="cuda")
            hidden = (torch.arange(b, device="cuda")[None, :]
                      > torch.arange(a, device="cuda")[:, None] + (b - a))
            for h in range(case["heads_q"]):
                qd = st["q"][at_q:at_q + a, h].double()
                kd = st["k"][at_k:at_k + b, h // group].double()
                vd = st["v"][at_k:at_k + b, h // group].double()
                s = (qd @ kd.T) / math.sqrt(case["head_dim"])
                s[hidden] = -math.inf
                e[:, h] = torch.logsumexp(s, -1)
                o[:, h] = torch.exp(s - e[:, h, None]) @ vd
            outs.append(o)
            lses.append(e)
            at_q, at_k = at_q + a, at_k + b
        return (torch.cat(outs), torch.cat(lses)) if case["lse"] else torch.cat(outs)
    if kind == "shared":
        group = case["heads_q"] // case["heads_kv"]
        out = torch.zeros(case["batch"], case["heads_q"], case["head_dim"], dtype=torch.float64,
                          device="cuda")
        for b, length in enumerate(st["lens"].tolist()):
            used = st["table"][b, : _pages_of(length, case["page"])].long()
            kd = st["k"][used].double().transpose(0, 1).reshape(case["heads_kv"], -1, case["head_dim"])
            vd = st["v"][used].double().transpose(0, 1).reshape(case["heads_kv"], -1, case["head_dim"])
            for h in range(case["heads_kv"]):
                rows = slice(h * group, (h + 1) * group)
                s = st["q"][b, rows].double() @ kd[h, :length].T / math.sqrt(case["head_dim"])
                out[b, rows] = torch.softmax(s, -1) @ vd[h, :length]
        return out
    page = case["page"]
    table, lens, refs = (st[x].cpu().numpy().copy() for x in ("table", "lens", "refs"))
    layers = range(case["layers"])
    k64, v64 = st["k"].double(), st["v"].double()

    def lowest():
        p = int(np.flatnonzero(refs == 0)[0])
        refs[p] = 1
        return p

    if kind == "fork":
        parents, children = st["parents"].tolist(), st["children"].tolist()
        for c in children:
            for p in table[c][table[c] >= 0]:
                refs[p] -= 1
            table[c] = -1
        for a, c in zip(parents, children):
            for j in range(lens[a] // page):
                table[c, j] = table[a, j]
                refs[table[a, j]] += 1
        for a, c in zip(parents, children):
            full, fill = divmod(int(lens[a]), page)
            lens[c] = lens[a]
            if fill:
                src, dst = int(table[a, full]), lowest()
                table[c, full] = dst
                k64[:, dst, :, :fill] = k64[:, src, :, :fill]
                v64[:, dst, :, :fill] = v64[:, src, :, :fill]
        return k64, v64, _i32(table), _i32(lens), _i32(refs)
    if kind == "compact":
        used = sorted(np.flatnonzero(refs > 0).tolist())
        holes = [p for p in range(len(used)) if refs[p] == 0]
        for src, dst in zip([p for p in used if p >= len(used)], holes):
            k64[:, dst], v64[:, dst] = k64[:, src], v64[:, src]
            refs[dst], refs[src] = refs[src], 0
            table[table == src] = dst
        return k64, v64, _i32(table), _i32(refs)
    slots, new = st["slots"].tolist(), st["new_lens"].tolist()
    for s in slots:
        for p in table[s][table[s] >= 0]:
            refs[p] -= 1
        table[s] = -1
    layer, at = 1 % case["layers"], 0
    for s, n in zip(slots, new):
        for j in range(_pages_of(n, page)):
            table[s, j] = lowest()
        lens[s] = n
    for s, n in zip(slots, new):
        for j in range(_pages_of(n, page)):
            m = min(page, n - j * page)
            rows = slice(at + j * page, at + j * page + m)
            k64[layer, table[s, j], :, :m] = st["new_k"][rows].double().transpose(0, 1)
            v64[layer, table[s, j], :, :m] = st["new_v"][rows].double().transpose(0, 1)
        at += n
    return k64, v64, _i32(table), _i32(lens), _i32(refs)
