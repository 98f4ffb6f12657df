"""Measured cases of the operators around an 8-bit key/value cache: rotary positions of queries and
keys, a paged cache that is quantised as it is written and read back, and single-token attention
over it.

`run` computes a case either with elementary torch operations in 32 bits (`own` false; angles in
64) or with the calls a user makes of this repository's package (`own` true).  `exact` restates
each definition in 64 bits.

The cache holds 8-bit codes, whole numbers or e4m3 floats, with one scale for each 16 tokens of a
page and head.  A scale is the smallest power of two that brings the largest of the block's values,
or 2^-110 where all are less, into the codes' range; appending to a block keeps the larger of its
scale and the new tokens', and the codes already there are rounded to it.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
BLOCK = 16                                       # tokens of a page that share a scale


# ------------------------------------------------------------------------------- cases
def listed():
    gqa = dict(heads_q=32, heads_kv=8, head_dim=128)
    small = dict(heads_q=14, heads_kv=2, head_dim=64)            # the decode layer's heads
    plain = dict(scaling="none", factor=1.0, theta=1e6)
    return [
        # One decode step of the decode layer's batch: latency counts.
        dict(name="rope_step", kind="rope", **small, rotary=64, layout="half", **plain, dtype="bf16",
             tokens=64, at="step", pos_max=2112),
        # A long prompt's queries and keys, slices of the fused projection.
        dict(name="rope_prompt", kind="rope", **gqa, rotary=128, layout="half", **plain,
             dtype="bf16", tokens=8192, at="prompt", pos_max=8192),
        # Half of each head turned, neighbours paired, far positions of a stretched context, fp32.
        dict(name="rope_stretched", kind="rope", **gqa, rotary=64, layout="interleaved",
             scaling="yarn", factor=32.0, theta=1e4, dtype="f32", tokens=4099, at="step",
             pos_max=1048576),
        # One token appended to every sequence of the decode layer's batch, and its last 64 read
        # back, as a layer with a local window needs them: latency counts.
        dict(name="append_step", kind="write", heads_kv=2, head_dim=64, code="int8", dtype="bf16",
             page=64, slots=64, old_min=100, old_max=2047, new_min=1, new_max=1, window=64),
        # The next chunk of four long prompts goes in; their whole contexts come back for it.
        dict(name="write_chunk", kind="write", heads_kv=8, head_dim=128, code="e4m3", dtype="bf16",
             page=64, slots=4, old_min=1000, old_max=7000, new_min=512, new_max=512, window=0),
        # A batch of prompts of all lengths is written and read back.
        dict(name="write_prompts", kind="write", heads_kv=8, head_dim=128, code="int8", dtype="bf16",
             page=32, slots=16, old_min=0, old_max=0, new_min=18, new_max=2048, window=0),
        # Single precision rows of odd lengths, in the middle of their blocks.
        dict(name="write_f32", kind="write", heads_kv=2, head_dim=64, code="e4m3", dtype="f32",
             page=16, slots=37, old_min=3, old_max=300, new_min=1, new_max=130, window=200),
        # A few short conversations: latency counts.
        dict(name="attend_small", kind="attend", **small, code="int8", dtype="bf16", page=16,
             batch=4, len_min=513, len_max=552),
        # The decode layer's batch and cache.
        dict(name="attend_step", kind="attend", **small, code="e4m3", dtype="bf16", page=64,
             batch=64, len_min=2049, len_max=2049),
        # Sequences of all lengths, an odd page size among the table's widths.
        dict(name="attend_ragged", kind="attend", **gqa, code="int8", dtype="bf16", page=32,
             batch=16, len_min=1, len_max=8191),
        # One very long context, in single precision.
        dict(name="attend_f32", kind="attend", **gqa, code="int8", dtype="f32", page=128,
             batch=1, len_min=131071, len_max=131071),
        # A large batch of long contexts: what the smaller cache is for.
        dict(name="attend_large", kind="attend", **gqa, code="e4m3", dtype="bf16", page=64,
             batch=192, len_min=500, len_max=8000),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Seconds that a case cannot do without at nominal rates, and the plain form's scratch bytes."""
    w = work(case)
    pad = 0
    if case["kind"] == "attend":
        keys = case["batch"] * case["len_max"]
        pad = 4 * keys * (2 * case["heads_kv"] * case["head_dim"] + 2 * case["heads_q"])
    if case["kind"] == "write":
        tokens = sum(map(sum, _old_new(case)))
        pad = 8 * tokens * case["heads_kv"] * case["head_dim"]      # the cache itself, and its values
    return max(w["bytes"] / 6e12, w["flops"] / 1e15), pad


def draw(rng):
    """One more case of the listed ones' ranges: kinds, head layouts, lengths over their logarithm."""
    most = max(_cost(c)[0] for c in listed())
    while True:
        kind = rng.choice(["rope", "write", "attend", "attend"])
        heads_kv, group = rng.choice([(1, 8), (2, 7), (8, 4), (4, 8), (8, 1), (3, 5), (16, 2), (2, 16)])
        case = dict(kind=kind, heads_kv=heads_kv, head_dim=rng.choice([64, 128, 128, 80, 256]),
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
        if kind == "rope":
            d = case["head_dim"]
            case.update(heads_q=heads_kv * group, rotary=rng.choice([d, d, d // 2, d // 4]),
                        layout=rng.choice(["half", "interleaved"]),
                        scaling=rng.choice(["none", "linear", "ntk", "yarn", "bands"]),
                        theta=rng.choice([1e4, 1e6]), tokens=_log_int(rng, 1, 16384),
                        at=rng.choice(["step", "prompt"]), pos_max=_log_int(rng, 20000, 1048576))
            case["factor"] = 1.0 if case["scaling"] == "none" else rng.choice([4.0, 8.0, 32.0])
        elif kind == "write":
            case.update(code=rng.choice(["int8", "e4m3"]), page=rng.choice([16, 32, 64, 128]),
                        slots=_log_int(rng, 1, 128), old_min=0, old_max=_log_int(rng, 1, 8000),
                        new_min=1, new_max=_log_int(rng, 1, 2048), window=rng.choice([0, 50, 200]))
        else:
            case.update(code=rng.choice(["int8", "e4m3"]), heads_q=heads_kv * group,
                        page=rng.choice([16, 32, 64, 128]), batch=_log_int(rng, 1, 256),
                        len_min=rng.choice([0, 1, 100]), len_max=_log_int(rng, 100, 131072))
        for name, some in (("slots", ("old", "new")), ("batch", ("len",))):
            if case.get(name) == 1:          # one sequence has the largest length
                case.update({x + "_min": case[x + "_max"] for x in some})
        seconds, pad = _cost(case)
        if seconds <= most and pad <= 1.1e10:
            return case


# ---------------------------------------------------------------------- sizes of a case
def _spread(n, lo, hi):
    """n lengths over [lo, hi], in a shuffled order that is the same for everybody."""
    step = next(s for s in (7, 11, 13, 17, 19, 23) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((i * step) % n) // max(1, n - 1) for i in range(n)]


def _old_new(case):
    """Tokens that each slot of a write holds before, and that it gets."""
    n = case["slots"]
    return (_spread(n, case["old_min"], case["old_max"]),
            _spread(n, case["new_min"], case["new_max"])[::-1])


def _back(case):
    """First token and number of tokens of each slot that are read back after a write."""
    lens = [a + b for a, b in zip(*_old_new(case))]
    first = [max(0, n - case["window"]) if case["window"] else 0 for n in lens]
    return first, [n - a for n, a in zip(lens, first)]


def _pages_of(length, page):
    return (length + page - 1) // page


def _blocks_of(length):
    return (length + BLOCK - 1) // BLOCK


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    d, hk = case["head_dim"], case["heads_kv"]
    if case["kind"] == "rope":
        heads = case["heads_q"] + hk
        return {"bytes": case["tokens"] * (2 * heads * d * size + 4),
                "flops": 3 * case["tokens"] * heads * case["rotary"]}
    if case["kind"] == "write":
        new, back = sum(_old_new(case)[1]), sum(_back(case)[1])
        blocks = sum(map(_blocks_of, _back(case)[1]))
        return {"bytes": 2 * hk * (d * (new + back) * (size + 1) + 4 * blocks), "flops": 0}
    lens = _spread(case["batch"], case["len_min"], case["len_max"])
    return {"bytes": 2 * hk * sum(d * n + 4 * _blocks_of(n) for n in lens)
            + 2 * size * case["batch"] * case["heads_q"] * d,
            "flops": 4 * case["heads_q"] * d * sum(lens)}


# ---------------------------------------------------------------------------- inputs
def _i32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _package():
    """This repository's package, as its documentation says to import it."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "enigma-dsl_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import enigma
    from enigma import kv_cache
    return enigma.cuda_ops, kv_cache


def _scaling(case):
    """What a model's configuration says about stretched contexts."""
    return {"none": None, "linear": dict(type="linear", factor=case["factor"]),
            "ntk": dict(type="ntk", factor=case["factor"]),
            "yarn": dict(type="yarn", factor=case["factor"], original_len=4096, beta_fast=32.0,
                         beta_slow=1.0),
            "bands": dict(type="bands", factor=case["factor"], original_len=8192, low=1.0,
                          high=4.0)}[case["scaling"]]


def _fused(gen, tokens, case, heads_q):
    """Q, K, V as slices of one fused projection's rows (heads of q | k | v); keys carry an offset
    for each channel, as trained projections give them."""
    hk, d, dt = case["heads_kv"], case["head_dim"], DTYPES[case["dtype"]]
    fused = torch.randn(tokens, heads_q + 2 * hk, d, device="cuda", generator=gen, dtype=dt)
    fused[:, heads_q:heads_q + hk] += torch.randn(hk, d, device="cuda", generator=gen, dtype=dt)
    return fused[:, :heads_q], fused[:, heads_q:heads_q + hk], fused[:, heads_q + hk:]


def _codes(gen, shape, code):
    """Codes of normally distributed values: bell-shaped whole numbers, or the e4m3 floats."""
    x = torch.empty(shape, dtype=CODES[code], device="cuda")
    for part in x.view(-1, shape[-1]).split(1 << 20):
        r = torch.randn(part.shape, device="cuda", generator=gen, dtype=torch.bfloat16)
        part.copy_((r * 30).round().clamp(-127, 127) if code == "int8" else r * 60)
    return x


def _scales(gen, shape, code):
    """Powers of two, as the cache's own writes give them, around what unit variance needs."""
    step = torch.randint(-1, 2, shape, device="cuda", generator=gen).float()
    return torch.exp2(step - (5 if code == "int8" else 6))


def _cache(gen, rs, case, layers, lens):
    """Codes, scales and a table of scattered pages for sequences of these lengths."""
    page = case["page"]
    width = max(1, max(_pages_of(n, page) for n in lens))
    pages = sum(_pages_of(n, page) for n in lens) + 3
    order, at = rs.permutation(pages), 0
    table, refs = np.full((len(lens), width), -1, np.int32), np.zeros(pages, np.int32)
    for s, n in enumerate(lens):
        m = _pages_of(n, page)
        table[s, :m] = order[at:at + m]
        refs[order[at:at + m]] = 1
        at += m
    shape = (layers, pages, case["heads_kv"])
    codes = [_codes(gen, shape + (page, case["head_dim"]), case["code"]) for _ in range(2)]
    scales = [_scales(gen, shape + (page // BLOCK,), case["code"]) for _ in range(2)]
    return dict(k=codes[0], v=codes[1], k_scale=scales[0], v_scale=scales[1], table=_i32(table),
                lens=_i32(lens), refs=_i32(refs))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rs = np.random.RandomState(seed % (1 << 31))
    state = dict(case=case)
    if case["kind"] == "rope":
        n = case["tokens"]
        state["q"], state["k"], _ = _fused(gen, n, case, case["heads_q"])
        if case["at"] == "step":         # tokens of different sequences
            where = rs.randint(0, case["pos_max"], n)
            where[-1] = case["pos_max"] - 1
        else:                            # one sequence's, from somewhere in its context
            where = rs.randint(0, case["pos_max"] - n + 1) + np.arange(n)
        state["positions"] = _i32(where)
        if own:
            ops, _ = _package()
            state["ops"] = ops
            state["table"] = ops.RopeTable(case["head_dim"], rotary_dim=case["rotary"],
                                           theta=case["theta"], layout=case["layout"],
                                           scaling=_scaling(case))
        return state
    if case["kind"] == "write":
        old, new = _old_new(case)
        state.update(_cache(gen, rs, case, 2, [a + b for a, b in zip(old, new)]))
        order = rs.permutation(case["slots"])
        first, back = _back(case)
        _, state["new_k"], state["new_v"] = _fused(gen, sum(new), case, case["heads_kv"])
        state["slots"] = _i32(order)
        state["starts"] = _i32([old[s] for s in order])
        state["cu"] = _i32(np.cumsum([0] + [new[s] for s in order]))
        state["first"] = _i32([first[s] for s in order])
        state["cu_back"] = _i32(np.cumsum([0] + [back[s] for s in order]))
        state["tokens_back"] = sum(back)
        if not own:
            state["blocks"] = _block_list(order, old, new)
    else:
        lens = _spread(case["batch"], case["len_min"], case["len_max"])
        state.update(_cache(gen, rs, case, 1, lens))
        state["len_max"] = max(lens)
        state["q"] = torch.randn(case["batch"], case["heads_q"], case["head_dim"], device="cuda",
                                 generator=gen, dtype=DTYPES[case["dtype"]])
    if own:
        _, kv_cache = _package()
        state["cache"] = kv_cache.QuantizedKVCache(*(state[x] for x in (
            "k", "v", "k_scale", "v_scale", "table", "lens", "refs")))
    return state


def _block_list(order, old, new):
    """The blocks that a write touches: slot, block of the sequence, first and end row in the
    block, and the packed row of the first."""
    out, at = [], 0
    for s in order:
        pos, end = old[s], old[s] + new[s]
        while pos < end:
            stop = min(end, (pos // BLOCK + 1) * BLOCK)
            out.append((s, pos // BLOCK, pos % BLOCK, pos % BLOCK + stop - pos, at))
            at += stop - pos
            pos = stop
    return torch.tensor(out, device="cuda").long().T


# ------------------------------------------------------------------------------ plain forms
def _frequencies(case):
    """Radians per position of each pair, in 64 bits, and the factor on cos and sin."""
    n, theta, f = case["rotary"], case["theta"], case["factor"]
    s = _scaling(case)
    if case["scaling"] == "ntk":
        theta = theta * f ** (n / (n - 2))
    i = torch.arange(0, n, 2, dtype=torch.float64, device="cuda")
    w = torch.exp(i * (-math.log(theta) / n))
    if case["scaling"] == "linear":
        w = w / f
    if case["scaling"] == "yarn":
        def pair(turns):       # the pair that turns this often over the original context
            return n * math.log(s["original_len"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo = max(math.floor(pair(s["beta_fast"])), 0)
        hi = min(math.ceil(pair(s["beta_slow"])), n - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return w * (1 - ramp) + w / f * ramp, 0.1 * math.log(f) + 1
    if case["scaling"] == "bands":
        turns = s["original_len"] * w / (2 * math.pi)
        keep = ((turns - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        w = w * keep + w / f * (1 - keep)
    return w, 1.0


def _plain_rope(st):
    case = st["case"]
    n = case["rotary"]
    w, factor = _frequencies(case)
    angle = st["positions"].double()[:, None] * w[None]
    cos, sin = ((f(angle) * factor).float()[:, None] for f in (torch.cos, torch.sin))
    outs = []
    for x in (st["q"], st["k"]):
        y = x.float()
        if case["layout"] == "half":
            a, b = y[..., :n // 2], y[..., n // 2:n]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., 0:n:2], y[..., 1:n:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        outs.append(torch.cat([turned, y[..., n:]], -1).to(x.dtype))
    return tuple(outs)


def _values(codes, scales):
    """What codes [..., page, D] and scales [..., page / 16] stand for, in fp32."""
    return codes.float() * scales.repeat_interleave(BLOCK, -1)[..., None]


def _to_codes(x, code):
    """Values over their scale, rounded to codes, in fp32."""
    return x.round().clamp(-127, 127) if code == "int8" else x.to(CODES[code]).float()


def _plain_write(st):
    case = st["case"]
    code, page = case["code"], case["page"]
    slot, block, lo, hi, at = st["blocks"]
    row = torch.arange(BLOCK, device=slot.device)
    pg = st["table"][slot, block * BLOCK // page].long()
    sub = block % (page // BLOCK)
    fresh = (row >= lo[:, None]) & (row < hi[:, None])                   # rows that are written
    src = torch.where(fresh, at[:, None] + row - lo[:, None], torch.zeros_like(row))
    layer = 1
    for codes, scales, rows in ((st["k"], st["k_scale"], st["new_k"]),
                                (st["v"], st["v_scale"], st["new_v"])):
        pages = codes[layer].view(torch.uint8).view(codes.shape[1], codes.shape[2], page // BLOCK,
                                                    BLOCK, -1)
        new = rows[src].float().permute(0, 2, 1, 3)                      # [blocks, heads, 16, D]
        new = torch.where(fresh[:, None, :, None], new, torch.zeros_like(new))
        top = new.abs().amax((-1, -2)).clamp(min=2.0 ** -110)
        m, e = torch.frexp(top)                                          # top = m 2^e, m in [1/2, 1)
        limit, shift = (127 / 128, 7) if code == "int8" else (448 / 512, 9)
        scale = torch.ldexp(torch.ones_like(m), e - shift + (m > limit).int())
        before = scales[layer][pg, :, sub]
        held = (lo > 0)[:, None]
        scale = torch.where(held, torch.maximum(scale, before), scale)
        old = pages[pg, :, sub].view(codes.dtype).float()
        grown = (before / scale)[..., None, None]
        kept = torch.where((held & (before < scale))[..., None, None], _to_codes(old * grown, code),
                           old)
        out = torch.where(fresh[:, None, :, None], _to_codes(new / scale[..., None, None], code),
                          kept)
        pages[pg, :, sub] = out.to(codes.dtype).view(torch.uint8)
        scales[layer][pg, :, sub] = scale
    token = torch.arange(st["tokens_back"], device=slot.device)
    i = torch.searchsorted(st["cu_back"], token.int(), right=True) - 1
    pos = token - st["cu_back"][i] + st["first"][i]
    pg = st["table"][st["slots"][i].long(), pos // page].long()
    outs = []
    for codes, scales in ((st["k"], st["k_scale"]), (st["v"], st["v_scale"])):
        x = codes[layer].view(torch.uint8)[pg, :, pos % page].view(codes.dtype).float()
        x = x * scales[layer][pg, :, pos % page // BLOCK][..., None]
        outs.append(x.to(DTYPES[case["dtype"]]))
    return tuple(outs)


def _plain_attend(st):
    case = st["case"]
    b, hk, d, page = case["batch"], case["heads_kv"], case["head_dim"], case["page"]
    q = st["q"].float().view(b, hk, -1, d)
    cols = _pages_of(max(1, st["len_max"]), page)
    at = st["table"][:, :cols].clamp(min=0).long()                       # [B, cols]
    hidden = (torch.arange(cols * page, device=q.device) >= st["lens"][:, None])[:, None, None]

    def dense(codes, scales):                                            # [B, Hkv, keys, D]
        x = codes[0].view(torch.uint8)[at].view(codes.dtype).float()
        x = x.view(b, cols, hk, page // BLOCK, BLOCK, d) * scales[0][at][..., None, None]
        return x.transpose(1, 2).reshape(b, hk, cols * page, d)

    k = dense(st["k"], st["k_scale"])
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    del k
    s.masked_fill_(hidden, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, dense(st["v"], st["v_scale"]))
    o = o / torch.where(z > 0, z, torch.ones_like(z))
    return o.reshape(b, -1, d).to(st["q"].dtype)


# ------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return {"rope": _plain_rope, "write": _plain_write, "attend": _plain_attend}[kind](state)
    if kind == "rope":
        return state["ops"].rope(state["q"], state["k"], state["positions"], state["table"])
    cache = state["cache"]
    if kind == "write":
        cache.write(1, state["new_k"], state["new_v"], state["slots"], state["starts"], state["cu"])
        return cache.read(1, state["slots"], state["first"], state["cu_back"],
                          tokens=state["tokens_back"], dtype=DTYPES[case["dtype"]])
    return cache.attend(0, state["q"])


# ----------------------------------------------------------------------------------- exact
def _exact_angles(case):
    """Radians per position of pair j, one after the other, and the factor."""
    n, f, kind = case["rotary"], case["factor"], case["scaling"]
    s = _scaling(case)
    base = case["theta"] * (f ** (n / (n - 2)) if kind == "ntk" else 1.0)
    out = []
    for j in range(n // 2):
        w = base ** (-2.0 * j / n)
        if kind == "linear":
            w /= f
        elif kind == "yarn":
            ends = [n * math.log(s["original_len"] / (2 * math.pi * t)) / (2 * math.log(base))
                    for t in (s["beta_fast"], s["beta_slow"])]
            a, b = max(0, math.floor(ends[0])), min(n - 1, math.ceil(ends[1]))
            r = min(1.0, max(0.0, (j - a) / ((b - a) or 1e-3)))
            w = (w / f) * r + w * (1 - r)
        elif kind == "bands":
            length = 2 * math.pi / w
            if length > s["original_len"] / s["low"]:
                w /= f
            elif length > s["original_len"] / s["high"]:
                r = (s["original_len"] / length - s["low"]) / (s["high"] - s["low"])
                w = (1 - r) * w / f + r * w
        out.append(w)
    return out, (0.1 * math.log(f) + 1 if kind == "yarn" else 1.0)


def _exact_round(y, code):
    """64-bit values to the nearest code, ties to even."""
    if code == "int8":
        return np.rint(y)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -60))), -6) - 3)
    return np.rint(y / step) * step


def _exact_write(st):
    """Sequence by sequence, block by block, on the host."""
    case = st["case"]
    code, page = case["code"], case["page"]
    table, slots = st["table"].cpu().numpy(), st["slots"].tolist()
    starts, cu = st["starts"].tolist(), st["cu"].tolist()
    first, back = st["first"].tolist(), np.diff(st["cu_back"].cpu().numpy())
    outs = []
    for name in "kv":
        codes = st[name][1].float().cpu().numpy().astype(np.float64)
        scales = st[name + "_scale"][1].cpu().numpy().astype(np.float64)
        rows = st["new_" + name].float().cpu().numpy().astype(np.float64)
        got = []
        for i, s in enumerate(slots):
            t, pos = cu[i], starts[i]
            while t < cu[i + 1]:
                r = pos % BLOCK
                n = min(BLOCK - r, cu[i + 1] - t)
                p, j, o = table[s, pos // page], pos % page // BLOCK, pos % page - r
                x = rows[t:t + n].transpose(1, 0, 2)
                top = np.maximum(np.abs(x).max((1, 2)), 2.0 ** -110)
                scale = 2.0 ** np.ceil(np.log2(top / TOP[code]))
                if r:
                    wide = np.maximum(scale, scales[p, :, j])
                    held = codes[p, :, o:o + r] * (scales[p, :, j] / wide)[:, None, None]
                    codes[p, :, o:o + r] = _exact_round(held, code)
                    scale = wide
                codes[p, :, o + r:o + r + n] = _exact_round(x / scale[:, None, None], code)
                scales[p, :, j] = scale
                t, pos = t + n, pos + n
            where = np.arange(first[i], first[i] + back[i])
            p = table[s, where // page]
            got.append(codes[p, :, where % page] * scales[p, :, where % page // BLOCK][..., None])
        outs.append(torch.from_numpy(np.concatenate(got)).cuda())
    return tuple(outs)


def exact(case, seed):
    """The definitions in 64 bits."""
    st = prepare(case, seed)
    if case["kind"] == "rope":
        n = case["rotary"]
        angles, factor = _exact_angles(case)
        pairs = [(j, j + n // 2) if case["layout"] == "half" else (2 * j, 2 * j + 1)
                 for j in range(n // 2)]
        outs = []
        for x in (st["q"], st["k"]):
            y = x.double()
            for (a, b), w in zip(pairs, angles):
                turn = torch.polar(torch.full_like(st["positions"], 1, dtype=torch.float64) * factor,
                                   st["positions"].double() * w)
                z = torch.complex(y[..., a], y[..., b]) * turn[:, None]
                y[..., a], y[..., b] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    if case["kind"] == "write":
        return _exact_write(st)
    d, hk, page = case["head_dim"], case["heads_kv"], case["page"]
    out = torch.zeros(case["batch"], case["heads_q"], d, dtype=torch.float64, device="cuda")
    for b, n in enumerate(st["lens"].tolist()):
        if n == 0:
            continue
        used = st["table"][b, : _pages_of(n, page)].long()
        k, v = ((st[x][0].view(torch.uint8)[used].view(CODES[case["code"]]).double()
                 * st[x + "_scale"][0][used].double().repeat_interleave(BLOCK, -1)[..., None])
                .transpose(0, 1).reshape(hk, -1, d)[:, :n] for x in "kv")
        q = st["q"][b].double().view(hk, -1, d)
        p = torch.softmax(q @ k.transpose(1, 2) / math.sqrt(d), -1)
        out[b] = (p @ v).view(-1, d)
    return out
