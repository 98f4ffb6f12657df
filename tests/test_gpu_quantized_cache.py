"""GPU parity of the paged cache in 8-bit codes: codes and scales equal to the 64-bit oracle's after
any request (powers of two make every rounding exact), rows read back, requests that are refused;
and attention over it within the bound of oracle.serving.bound."""
import numpy as np
import pytest

from oracle import numerics as orc
from oracle import serving as srv

pytestmark = pytest.mark.gpu

CODES = ["int8", "e4m3"]


def _values(rng, shape, dtype):
    x = rng.standard_normal(shape, dtype=np.float32)
    return orc.bf16_round(x) if dtype == "bf16" else x


def _dev(a, dtype, cuda):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).to(cuda)
    return t.bfloat16() if dtype == "bf16" else t


def _np(t):
    return t.float().cpu().numpy().astype(np.float64)


def _kind(code):
    import torch
    return {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[code]


def _make(cuda, rng, layers, pages, heads, page, d, slots, width, lens, code, scales=None):
    """A cache whose first len(lens) slots hold sequences of random codes on scattered pages."""
    import torch
    from enigma.kv_cache import QuantizedKVCache
    table = np.full((slots, width), -1, np.int32)
    refs, full = np.zeros(pages, np.int32), np.zeros(slots, np.int32)
    order, at = rng.permutation(pages), 0
    for s, n in enumerate(lens):
        m = -(-n // page)
        table[s, :m] = order[at:at + m]
        refs[order[at:at + m]] = 1
        full[s] = n
        at += m
    shape = (layers, pages, heads, page, d)
    if code == "int8":
        codes = [torch.from_numpy(rng.integers(-127, 128, shape).astype(np.int8)) for _ in range(2)]
    else:
        codes = [torch.from_numpy(np.clip(rng.standard_normal(shape) * 90, -448, 448)
                                  .astype(np.float32)).to(_kind(code)) for _ in range(2)]
    if scales is None:
        scales = [np.exp2(rng.integers(-8, -3, shape[:3] + (page // 16,))).astype(np.float32)
                  for _ in range(2)]
    cache = QuantizedKVCache(*(x.to(cuda) for x in codes), *(torch.from_numpy(x).to(cuda) for x in scales),
                             *(torch.from_numpy(x).to(cuda) for x in (table, full, refs)))
    want = srv.QuantizedPages(*(x.float().numpy() for x in codes), *scales, table, full, refs, code)
    return cache, want


def _same(cache, want):
    for name in ("table", "lens", "refs"):
        np.testing.assert_array_equal(getattr(cache, name).cpu().numpy(), getattr(want, name), name)
    for got, ref in ((cache.k_scale, want.scales[0]), (cache.v_scale, want.scales[1]),
                     (cache.k, want.k), (cache.v, want.v)):
        np.testing.assert_array_equal(_np(got), ref)


SHAPES = [(2, 60, 2, 16, 64), (1, 40, 8, 64, 128), (2, 30, 1, 128, 16), (1, 50, 3, 32, 80),
          (1, 40, 2, 64, 256)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layers,pages,heads,page,d", SHAPES)
def test_write(cuda, layers, pages, heads, page, d, dtype, code):
    """Prompts, continued in the middle of blocks and pages, of growing and shrinking magnitude, from
    slices of a fused projection."""
    rng = np.random.default_rng(pages + d)
    cache, want = _make(cuda, rng, layers, pages, heads, page, d, 12, 6, [page + 1, 5], code)
    for size in (1.0, 30.0, 0.01, 1e-4):
        slots = [1, 7, 0, 3]
        lens = [int(want.lens[s]) + n for s, n in zip(slots, (2 * page // 3 + 3, 1, 17, page))]
        if max(lens) > 6 * page:
            break
        starts = [int(want.lens[s]) for s in slots]
        cache.reserve(slots, lens)
        want.reserve(slots, lens)
        cu = np.concatenate([[0], np.cumsum([n - s for n, s in zip(lens, starts)])])
        rows = _values(rng, (int(cu[-1]), 2 * heads + 1, d), dtype) * np.float32(size)
        rows = orc.bf16_round(rows) if dtype == "bf16" else rows
        t = _dev(rows, dtype, cuda)
        cache.write(layers - 1, t[:, 1:1 + heads], t[:, 1 + heads:], slots, starts, cu)
        want.write(layers - 1, rows[:, 1:1 + heads], rows[:, 1 + heads:], slots, starts, cu)
        cache.check()
        _same(cache, want)


@pytest.mark.parametrize("code", CODES)
def test_append(cuda, code):
    """Token by token, of many magnitudes: blocks are rounded again as their scale grows, and stay
    within a step (of the last scale) of what was written."""
    rng = np.random.default_rng(1)
    heads, d, n = 2, 64, 5
    cache, want = _make(cuda, rng, 1, 30, heads, 16, d, n, 5, [], code)
    size = np.exp2(rng.integers(-6, 4, (50, n, heads, 1)))
    rows = [orc.bf16_round((rng.standard_normal((50, n, heads, d)) * size).astype(np.float32))
            for _ in range(2)]
    slots, cu = np.arange(n), np.arange(n + 1)
    for t in range(50):
        cache.reserve(slots, [t + 1] * n)
        want.reserve(slots, [t + 1] * n)
        cache.write(0, *(_dev(x[t], "bf16", cuda) for x in rows), slots, [t] * n, cu)
        want.write(0, *(x[t] for x in rows), slots, [t] * n, cu)
    cache.check()
    _same(cache, want)
    got = cache.read(0, slots, [0] * n, np.arange(n + 1) * 50)
    for x, y, s in zip(got, rows, want.scales):
        back = _np(x).reshape(n, 50, heads, d).transpose(1, 0, 2, 3)
        step = np.stack([[s[0, want.table[i, t // 16], :, 0] for i in range(n)] for t in range(50)])
        unit = step[..., None] * (1.0 if code == "int8" else np.maximum(
            np.exp2(np.floor(np.log2(np.maximum(np.abs(y) / step[..., None], 2.0 ** -6))) - 3), 2.0 ** -9))
        assert (np.abs(back - y) <= unit).all()


def _written(cuda, rng, n, heads, d):
    x = _values(rng, (n, heads, d), "bf16")
    return x, _dev(x, "bf16", cuda)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite(cuda, code, bad):
    """Their block of that head reads as NaN until it is started anew; others do not notice."""
    rng = np.random.default_rng(2)
    cache, want = _make(cuda, rng, 1, 8, 3, 32, 64, 2, 3, [], code)
    cache.reserve([0], [70])
    want.reserve([0], [70])
    x, _ = _written(cuda, rng, 70, 3, 64)
    x[20, 1, 63] = bad
    x[69, 0, 5] = bad
    for req in ((x, [0], [0], [0, 70]), (x[:3], [0], [22], [0, 3]), (x[16:20], [0], [16], [0, 4])):
        cache.write(0, _dev(req[0], "bf16", cuda), _dev(req[0], "bf16", cuda), *req[1:])
        want.write(0, req[0], req[0], *req[1:])
        cache.check()
        _same(cache, want)
    k, _ = cache.read(0, [0], [0], [0, 70])
    nan = np.isnan(_np(k))
    assert nan[64:, 0].all() and nan.sum() == 6 * 64        # the block of 16 .. 31 was started anew


@pytest.mark.parametrize("code", CODES)
def test_small_and_large_values(cuda, code):
    rng = np.random.default_rng(3)
    cache, want = _make(cuda, rng, 1, 8, 4, 16, 64, 1, 4, [], code)
    cache.reserve([0], [33])
    want.reserve([0], [33])
    x = rng.standard_normal((33, 4, 64)).astype(np.float32)
    x[:, 0] *= np.float32(1e-38)
    x[:, 1] = np.clip(x[:, 1], -3, 3) * np.float32(1e38)
    x[:, 2] = 0
    top = np.float32(srv.TOP[code])
    x[:16, 3] = np.clip(x[:16, 3], -1, 1)
    x[3, 3, 7] = np.float32(top * 2.0 ** -9)                # just fits, just does not
    x[16:32, 3] = np.clip(x[16:32, 3], -1, 1)
    x[20, 3, 7] = np.nextafter(np.float32(top * 2.0 ** -8), np.float32(9e9))
    t = _dev(x, "f32", cuda)
    cache.write(0, t, t, [0], [0], [0, 33])
    want.write(0, x, x, [0], [0], [0, 33])
    _same(cache, want)


@pytest.mark.parametrize("code", CODES)
def test_writes_that_are_refused(cuda, code):
    """A token without a place, a shared page, a block named twice: those are left out, the rest is
    written, and check() says so."""
    import torch
    from enigma import EnigmaError
    rng = np.random.default_rng(4)
    cache, want = _make(cuda, rng, 1, 20, 2, 16, 64, 6, 4, [40, 16, 5], code)
    cache.fork([0], [4])                                    # shares two full pages of slot 0
    want.fork([0], [4])
    cache.check()
    x, t = _written(cuda, rng, 8, 2, 64)

    def refuse(match, slots, starts, cu, kept=()):
        cache.write(0, t, t, slots, starts, cu)
        for i in kept:                                      # entries that are met
            want.write(0, x[cu[i]:cu[i + 1]], x[cu[i]:cu[i + 1]], [slots[i]], [starts[i]],
                       [0, cu[i + 1] - cu[i]])
        with pytest.raises(EnigmaError, match=match):
            cache.check()
        cache.check()
        _same(cache, want)

    refuse("share", [0, 2], [3, 5], [0, 4, 8], kept=[1])
    refuse("share", [4], [16], [0, 8])
    refuse("does not exist", [6, 2], [0, 0], [0, 4, 8], kept=[1])
    refuse("does not exist", [-1], [0], [0, 8])
    refuse("does not exist", [3], [0], [0, 8])              # nothing reserved
    refuse("does not exist", [1], [-9], [0, 8])
    refuse("does not exist", [1], [64], [0, 8])             # behind its row
    refuse("does not exist", [1], [2 ** 31 - 4], [0, 8])
    refuse("does not exist", [2], [0], [0, 6], kept=[0])    # rows behind the last entry
    refuse("does not exist", [2], [0], [2, 8], kept=[0])    # and before the first
    refuse("twice", [2, 2], [0, 4], [0, 4, 8])
    refuse("twice", [2, 1, 2], [0, 0, 4], [0, 2, 6, 8], kept=[1])
    cache.reserve([1], [40])
    want.reserve([1], [40])
    cache.write(0, t, t, [1, 1], [16, 32], [0, 4, 8])       # two blocks of one slot are fine
    want.write(0, x, x, [1, 1], [16, 32], [0, 4, 8])
    cache.check()
    _same(cache, want)
    cu = [0, 8]
    cache.write(0, t, t, [1], [28], cu)                     # across a page's end
    want.write(0, x, x, [1], [28], cu)
    cache.check()
    _same(cache, want)
    none = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=cuda)
    cache.write(0, none, none, [], [], [0])
    cache.write(0, none, none, [1, 2], [0, 0], [0, 0, 0])
    cache.write(0, t, t, [2, 2, 1], [0, 3, 16], [0, 0, 0, 8])        # an entry without rows is no second
    want.write(0, x, x, [1], [16], [0, 8])
    cache.check()
    _same(cache, want)


def test_many_entries(cuda):
    """More entries than a search step takes, in any order, some empty; a request as wide as the cache."""
    rng = np.random.default_rng(5)
    n = 3000
    cache, want = _make(cuda, rng, 1, n + 5, 1, 16, 16, n, 1, [], "int8")
    lens = rng.integers(0, 5, n)
    slots = rng.permutation(n)
    cache.reserve(slots, lens)
    want.reserve(slots, lens)
    cu = np.concatenate([[0], np.cumsum(lens)])
    x, t = _written(cuda, rng, int(cu[-1]), 1, 16)
    cache.write(0, t, t, slots, np.zeros(n, int), cu)
    want.write(0, x, x, slots, np.zeros(n, int), cu)
    cache.check()
    _same(cache, want)
    k, v = cache.read(0, slots, np.zeros(n, int), cu)
    ref = np.zeros((2, *x.shape))
    want.read(0, slots, np.zeros(n, int), cu, *ref)
    np.testing.assert_array_equal(_np(k), ref[0])
    np.testing.assert_array_equal(_np(v), ref[1])


@pytest.mark.parametrize("heads,d,dtype,lens", [
    (1, 64, "bf16", [29000, 3]), (2, 16, "bf16", [7, 40000]), (1, 256, "f32", [28999]),
    (1, 256, "bf16", [28500, 500]), (24, 32, "bf16", [600, 31]), (32, 128, "f32", [100, 1, 17])])
def test_long_requests_and_many_heads(cuda, heads, d, dtype, lens):
    """Requests that fill the GPU many times over, and rows of many heads; from the middle of a block."""
    rng = np.random.default_rng(heads + d)
    page, n = 128, len(lens)
    cache, want = _make(cuda, rng, 1, sum(x // page + 2 for x in lens), heads, page, d, n,
                        max(lens) // page + 2, [], "int8")
    slots, starts = list(range(n)), [5] * n
    cache.reserve(slots, [x + 5 for x in lens])
    want.reserve(slots, [x + 5 for x in lens])
    for at, count in (([0] * n, starts), (starts, lens)):
        cu = np.concatenate([[0], np.cumsum(count)])
        x = _values(rng, (int(cu[-1]), heads, d), dtype)
        t = _dev(x, dtype, cuda)
        cache.write(0, t, t, slots, at, cu)
        want.write(0, x, x, slots, at, cu)
    cache.check()
    _same(cache, want)
    got = cache.read(0, slots, starts, cu, dtype=t.dtype)
    ref = np.zeros((2, *x.shape))
    want.read(0, slots, starts, cu, *ref)
    for y, r in zip(got, ref):
        np.testing.assert_array_equal(_np(y), r)


@pytest.mark.parametrize("n,near", [(40, True), (300, True), (2500, False), (9000, True)])
def test_entries_that_clash(cuda, n, near):
    """Among many entries some name a block that another does, next to it or far away, before or behind:
    neither is written.  Slots that differ by a multiple of a power of two, the same slot in another
    block, and entries without rows clash with nobody."""
    from enigma import EnigmaError
    rng = np.random.default_rng(n)
    total = 9000
    cache, want = _make(cuda, rng, 1, total * 2 + 3, 1, 16, 16, total, 2, [20] * total, "int8")
    slots = rng.permutation(total)[:n] if n < total else np.arange(total)
    slots[:8] = [5 + 1024 * i for i in range(8)] if n < total else slots[:8]
    slots[8:] = [s if s not in slots[:8] else 9 for s in slots[8:]] if n < total else slots[8:]
    starts, lens = rng.integers(0, 12, n), rng.integers(0, 4, n)
    lens[:8] = 1
    for _ in range(max(3, n // 50)):
        i = int(rng.integers(0, n))
        j = min(n - 1, i + int(rng.integers(1, 12))) if near else int(rng.integers(0, n))
        slots[j] = slots[i]
        starts[j] = rng.integers(0, 30)                     # the same block, the next, or across their border
    cu = np.concatenate([[0], np.cumsum(lens)])
    x, t = _written(cuda, rng, int(cu[-1]), 1, 16)
    blocks = [[(slots[i], b) for b in range(starts[i] // 16, (starts[i] + lens[i] - 1) // 16 + 1)]
              if lens[i] else [] for i in range(n)]
    count = {}
    for bs in blocks:
        for b in bs:
            count[b] = count.get(b, 0) + 1
    clash = any(c > 1 for c in count.values())
    cache.write(0, t, t, slots, starts, cu)
    for i in range(n):                                      # block by block: the others of an entry are met
        for s, b in blocks[i]:
            if count[s, b] == 1:
                lo, hi = max(starts[i], 16 * b), min(starts[i] + lens[i], 16 * b + 16)
                rows = x[cu[i] + lo - starts[i]:cu[i] + hi - starts[i]]
                want.write(0, rows, rows, [s], [lo], [0, hi - lo])
    if clash:
        with pytest.raises(EnigmaError, match="twice"):
            cache.check()
    cache.check()
    _same(cache, want)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layers,pages,heads,page,d", SHAPES)
@pytest.mark.parametrize("gap", [0, 3])
def test_read(cuda, layers, pages, heads, page, d, dtype, code, gap):
    """Into new tensors and into slices of any alignment; tokens that are not there, rows that no
    entry names."""
    import torch
    rng = np.random.default_rng(pages + 7)
    cache, want = _make(cuda, rng, layers, pages, heads, page, d, 6, 4, [3 * page - 5, 7, 0, page], code)
    slots, starts = [0, 3, 1, 0, -2, 6, 2], [5, 0, 3, page - 3, 0, 0, 0]
    counts = [2 * page, page + 2, 9, 8, 2, 1, 3]            # slots 3 and 1 end before their entries
    cu = np.concatenate([[0], np.cumsum(counts)]) + 4
    tokens = int(cu[-1]) + 3
    kind = torch.bfloat16 if dtype == "bf16" else torch.float32
    ref = np.full((2, tokens, heads, d), 7.0)
    want.read(layers - 1, slots, starts, cu, *ref)
    outs = [torch.full((tokens, heads * d + gap), 7.0, dtype=kind, device=cuda) for _ in range(2)]
    views = [x[:, gap:].unflatten(1, (heads, d)) for x in outs]
    k, v = cache.read(layers - 1, slots, starts, cu, out_k=views[0], out_v=views[1])
    assert k.data_ptr() == views[0].data_ptr()
    np.testing.assert_array_equal(_np(k), ref[0])
    np.testing.assert_array_equal(_np(v), ref[1])
    assert all((x[:, :gap] == 7).all() for x in outs)
    k, v = cache.read(layers - 1, slots, starts, cu, dtype=kind)
    assert k.dtype == kind and k.shape == (cu[-1], heads, d)
    np.testing.assert_array_equal(_np(v)[4:], ref[1][4:cu[-1]])
    k, v = cache.read(layers - 1, [], [], [0])
    assert k.shape == (0, heads, d)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("layers,pages,heads,page,d", SHAPES[:4])
def test_fork_compact_copy(cuda, layers, pages, heads, page, d, code):
    """Pages take their scales along."""
    from enigma import EnigmaError
    rng = np.random.default_rng(pages + 3)
    lens = [page * 3 + 1, 0, page * 2, 1, page * 4 - 1]
    cache, want = _make(cuda, rng, layers, pages, heads, page, d, 14, 5, lens, code)
    for parents, children in (([0, 0, 2, 4], [5, 9, 7, 6]), ([3, 1], [8, 0])):
        cache.fork(parents, children)
        want.fork(parents, children)
    cache.check()
    _same(cache, want)
    for _ in range(2):
        cache.compact()
        want.compact()
        _same(cache, want)
    cache.free([2, 4, 9])
    want.free([2, 4, 9])
    cache.compact()
    want.compact()
    _same(cache, want)
    cache.copy_pages([0, 1, 1], [pages - 1, pages - 2, pages - 3])
    want.copy_pages([0, 1, 1], [pages - 1, pages - 2, pages - 3])
    cache.check()
    _same(cache, want)
    for request in (lambda: cache.fork([0, 0], [1, 1]), lambda: cache.copy_pages([0, pages], [1, 2])):
        request()
        with pytest.raises(EnigmaError):
            cache.check()
        _same(cache, want)
    cache.fork([5] * 3, [10, 11, 12])                      # more than there are pages for: nothing
    if int((want.refs == 0).sum()) < 3 and want.lens[5] % page:
        with pytest.raises(EnigmaError):
            cache.check()
    else:
        want.fork([5] * 3, [10, 11, 12])
    _same(cache, want)


# ------------------------------------------------------------------------------- attention
def _attend(cuda, rng, cache, want, heads_q, dtype, slots=None, scale=None, layer=0, size=1.0, **kw):
    d = want.k.shape[-1]
    b = len(want.table) if slots is None else len(slots)
    q = _values(rng, (b, heads_q, d), dtype) * np.float32(size)
    q = orc.bf16_round(q) if dtype == "bf16" else q
    out = cache.attend(layer, _dev(q, dtype, cuda), slots=slots, scale=scale, **kw)
    k, v = want.values(layer)
    ref = srv.paged(q, k, v, want.table, want.lens, 0, 1 / np.sqrt(d) if scale is None else scale, slots)
    return _np(out), (*ref, _floor(want, dtype, layer))


def _floor(want, dtype, layer=0):
    """What rounding a weight to fp16 may cost a key where the relative bound is less.

    Half the least fp16 is 2^-25.  bf16: a key's weight, in units of one that is at most 2^4 times
    less than the largest weight, times s_v over a v0 that is at most the largest |s_v|, times 2^9, is
    rounded; multiplied back by v0 2^-9 and the key's code, and divided by a sum of weights that is
    1 or more in those units (they are the weight of a key that was seen), that is at most 2^-34
    max|s_v| max|code| for each key.  fp32: the weight over the largest of its chunk, times s_v over
    the chunk's larger one, times 2^15, in two numbers, of which the second is rounded so: 2^-40.  It
    counts for an element to which only keys of small weight contribute, the others' codes being zero."""
    codes = want.v[layer]
    return 2.0 ** (-34 if dtype == "bf16" else -40) * np.abs(want.scales[1][layer]).max() \
        * np.abs(codes).max()


def _hold(got, ref, keys, dtype):
    out, mag, lse, err, *floor = ref
    tol = srv.bound(out, mag, err, keys, dtype == "bf16") + (keys * floor[0] if floor else 0)
    off = np.abs(got - out)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), (off / tol).max()
    assert (got[np.isinf(lse)] == 0).all()


LENS = [[1], [0, 1, 15, 16, 17], [31, 32, 33, 0, 63, 64, 65], [127, 128, 129, 300], [5, 1000, 0, 257]]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x)))
@pytest.mark.parametrize("heads_q,heads_kv,d,page,dtype", [
    (14, 2, 64, 16, "bf16"), (8, 2, 128, 64, "bf16"), (3, 3, 128, 32, "bf16"), (16, 1, 128, 64, "bf16"),
    (40, 2, 64, 128, "bf16"), (4, 2, 80, 16, "bf16"), (8, 1, 256, 64, "bf16"), (6, 2, 16, 32, "bf16"),
    (40, 1, 256, 32, "bf16"), (14, 2, 64, 64, "f32"), (2, 2, 128, 128, "f32"), (16, 1, 128, 16, "f32"),
    (5, 1, 96, 32, "f32"), (12, 1, 256, 16, "f32"), (34, 1, 64, 64, "f32")])
def test_attend(cuda, lens, heads_q, heads_kv, d, page, dtype, code):
    rng = np.random.default_rng(sum(lens) + d + page)
    width = max(-(-max(lens) // page), 1) + 1
    pages = sum(-(-n // page) for n in lens) + 2
    cache, want = _make(cuda, rng, 1, pages, heads_kv, page, d, len(lens), width, lens, code)
    got, ref = _attend(cuda, rng, cache, want, heads_q, dtype)
    _hold(got, ref, max(lens), dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads_q,heads_kv,d,lens", [
    (4, 1, 128, [9000]), (14, 2, 64, [4097, 3, 2000]), (16, 1, 64, [5000, 5001]),
    (8, 8, 128, [700, 2100]), (8, 1, 256, [3500, 40])])
def test_attend_long(cuda, heads_q, heads_kv, d, lens, dtype, code):
    """Long sequences, split over the GPU and joined, in tables wider than they need."""
    rng = np.random.default_rng(sum(lens))
    page = 64
    pages = sum(-(-n // page) for n in lens) + 1
    cache, want = _make(cuda, rng, 1, pages, heads_kv, page, d, len(lens), 300, lens, code)
    got, ref = _attend(cuda, rng, cache, want, heads_q, dtype)
    _hold(got, ref, max(lens), dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads_q,heads_kv,d,lens", [
    (4, 1, 64, [700, 33]), (6, 3, 256, [600, 5, 0]), (1, 1, 80, [1, 900]), (3, 1, 128, [50, 64]),
    (8, 2, 256, [17, 2]), (9, 1, 64, [300]), (12, 1, 128, [1000, 1])])
def test_attend_few_heads(cuda, heads_q, heads_kv, d, lens, code):
    """Groups that fill no tile of heads, in short and wide tables, by themselves and among others."""
    rng = np.random.default_rng(heads_q + d)
    pages = sum(-(-n // 32) for n in lens) + 1
    for dtype in ("bf16", "f32"):
        for width in (-(-max(lens) // 32), 800):
            cache, want = _make(cuda, rng, 1, pages, heads_kv, 32, d, len(lens), width, lens, code)
            got, ref = _attend(cuda, rng, cache, want, heads_q, dtype)
            _hold(got, ref, max(lens), dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads_q,heads_kv", [(32, 2), (14, 2), (8, 2), (3, 3)])
@pytest.mark.parametrize("d", [80, 96, 112])
def test_attend_heads_between(cuda, d, heads_q, heads_kv, code):
    """Heads between 64 and 128 elements: chunks that lie in a page, cross pages, end early."""
    rng = np.random.default_rng(heads_q + d)
    for page, lens in ((16, [1, 31, 32, 33, 100]), (64, [600, 0, 47, 2000]), (128, [9000, 5])):
        pages = sum(-(-n // page) for n in lens) + 1
        for dtype in ("bf16", "f32"):
            cache, want = _make(cuda, rng, 1, pages, heads_kv, page, d, len(lens),
                                -(-max(lens) // page) + 1, lens, code)
            got, ref = _attend(cuda, rng, cache, want, heads_q, dtype)
            _hold(got, ref, max(lens), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads_q,heads_kv,d", [(14, 2, 64), (8, 4, 128), (4, 1, 256)])
def test_attend_little_work(cuda, dtype, heads_q, heads_kv, d):
    """Fewer chunks than the GPU has warps, or hardly more: units that end and begin anywhere in a
    block's share, in tables wide enough for far more."""
    rng = np.random.default_rng(d)
    for n in (1, 2, 5, 17, 60, 149, 400):
        lens = [int(x) for x in rng.integers(0, 200, n) * (rng.random(n) < 0.8)]
        lens[-1] = 1 + n
        cache, want = _make(cuda, rng, 1, sum(-(-x // 16) for x in lens), heads_kv, 16, d, n, 2000, lens,
                            "int8")
        got, ref = _attend(cuda, rng, cache, want, heads_q, dtype)
        _hold(got, ref, max(lens), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_large_batches(cuda, dtype):
    """More sequences than SMs, most of a few keys; and the same slot named many times."""
    rng = np.random.default_rng(11)
    lens = [int(x) for x in rng.integers(0, 40, 400)]
    lens[7] = 900
    cache, want = _make(cuda, rng, 1, sum(-(-n // 16) for n in lens), 2, 16, 64, 400, 60, lens, "int8")
    got, ref = _attend(cuda, rng, cache, want, 4, dtype)
    _hold(got, ref, 900, dtype)
    slots = [int(x) for x in rng.integers(0, 400, 500)] + [7] * 30
    got, ref = _attend(cuda, rng, cache, want, 4, dtype, slots=slots)
    _hold(got, ref, 900, dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype,size", [("bf16", 8.0), ("bf16", 1e-30), ("f32", 8.0), ("f32", 1e-20)])
def test_attend_peaked_and_flat(cuda, code, dtype, size):
    """One key far above the others, in any place; queries too small to tell keys apart."""
    rng = np.random.default_rng(12)
    cache, want = _make(cuda, rng, 1, 30, 2, 32, 128, 2, 20, [500, 77], code)
    got, ref = _attend(cuda, rng, cache, want, 8, dtype, size=size)
    _hold(got, ref, 500, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("code", CODES)
def test_attend_any_scales(cuda, code, dtype):
    """Scales that are no powers of two, negative, zero, of very different sizes."""
    rng = np.random.default_rng(13)
    scales = []
    for lo, hi in ((-7, -5), (-30, 20)):
        x = rng.standard_normal((1, 30, 2, 4)) * np.exp2(rng.integers(lo, hi, (1, 30, 2, 4)))
        x[:, ::7] = 0
        scales.append(x.astype(np.float32))
    cache, want = _make(cuda, rng, 1, 30, 2, 64, 64, 3, 20, [700, 77, 16], code, scales=scales)
    got, ref = _attend(cuda, rng, cache, want, 8, dtype)
    _hold(got, ref, 700, dtype)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [16, 64])
def test_attend_unseen_values_do_not_reach(cuda, code, dtype, page):
    """Codes and scales behind a sequence's last key, in its last block, page and table row, may be
    NaN or anything."""
    import torch
    rng = np.random.default_rng(14)
    lens = [1, 15, 16, 17, 33, 70, 0, 129]
    cache, want = _make(cuda, rng, 1, 40, 2, page, 64, 8, 12, lens, code)
    q = _dev(_values(rng, (8, 8, 64), dtype), dtype, cuda)
    clean = cache.attend(0, q)
    spoil = {"int8": -128, "e4m3": -1}              # e4m3: bits of NaN, as 127 are
    raw = [x.view(torch.int8) for x in (cache.k, cache.v)]
    used = torch.zeros(40, page, dtype=torch.bool)
    for s, n in enumerate(lens):
        for j in range(n):
            used[want.table[s, j // page], j % page] = True
    unseen = ~used.to(cuda)[None, :, None, :, None]
    dead = ~used.view(40, page // 16, 16).any(-1).to(cuda)[None, :, None]
    for x in raw:
        for value in (spoil[code], 127):
            x.copy_(torch.where(unseen, torch.full_like(x, value), x))
            for bad in (np.nan, np.inf, -3e38):
                for s in (cache.k_scale, cache.v_scale):
                    s.copy_(torch.where(dead, torch.full_like(s, bad), s))
                assert (cache.attend(0, q) == clean).all()
    # Numbers of pages behind a sequence's last key.
    for s, n in enumerate(lens):
        cache.table[s, -(-n // page):] = [-7, 1 << 30, 3][s % 3]
    assert (cache.attend(0, q) == clean).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [80, 96, 128, 256])
@pytest.mark.parametrize("heads_q", [6, 32])
def test_attend_unseen_and_nan_other_heads(cuda, d, heads_q, dtype):
    """The same for other head sizes and groups: what is behind the last key reaches nobody, NaN in an
    element of a value that is seen reaches that element of that sequence's kv head alone."""
    import torch
    rng = np.random.default_rng(d)
    lens = [1, 31, 32, 50, 0, 700]
    cache, want = _make(cuda, rng, 1, 60, 2, 32, d, 6, 40, lens, "e4m3")
    q = _dev(_values(rng, (6, heads_q, d), dtype), dtype, cuda)
    clean = cache.attend(0, q)
    used = torch.zeros(60, 32, dtype=torch.bool)
    for s, n in enumerate(lens):
        for j in range(n):
            used[want.table[s, j // 32], j % 32] = True
    unseen = ~used.to(cuda)[None, :, None, :, None]
    for x in (cache.k, cache.v):
        raw = x.view(torch.int8)
        raw.copy_(torch.where(unseen, torch.full_like(raw, 127), raw))   # NaN
    assert (cache.attend(0, q) == clean).all()
    group = heads_q // 2
    for s, j, e in ((3, 49, d - 1), (5, 333, d - 16), (0, 0, 0), (5, 0, 63)):
        p, r = int(want.table[s, j // 32]), j % 32
        raw = cache.v.view(torch.int8)
        was = int(raw[0, p, 1, r, e])
        raw[0, p, 1, r, e] = 127
        nan = torch.isnan(cache.attend(0, q))
        raw[0, p, 1, r, e] = was
        assert nan[s, group:, e].all() and int(nan.sum()) == group
    assert (cache.attend(0, q) == clean).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 33, 1000])
def test_attend_nan_is_not_lost(cuda, dtype, n):
    """NaN in the query, in a key, a value or a scale that is seen gives NaN in that sequence's heads
    of that kv head, and nowhere else."""
    import torch
    rng = np.random.default_rng(15)
    for what in ("q", "k", "v", "k_scale", "v_scale", "all k_scale", "all v_scale"):
        cache, want = _make(cuda, rng, 1, 70, 2, 32, 64, 2, 32, [n, n], "e4m3")
        q = _dev(_values(rng, (2, 8, 64), dtype), dtype, cuda)
        clean = cache.attend(0, q)
        j = n // 2
        p, r = int(want.table[1, j // 32]), j % 32
        mine = torch.from_numpy(want.table[1, : -(-n // 32)]).to(cuda)
        if what == "q":
            q[1, 6, 3] = np.nan
        elif what in ("k", "v"):
            getattr(cache, what).view(torch.int8)[0, p, 1, r, 9] = 0x7f
        elif what.startswith("all"):
            getattr(cache, what[4:])[0, mine, 1] = np.nan
        else:
            getattr(cache, what)[0, p, 1, r // 16] = np.nan
        got = cache.attend(0, q)
        assert (got[0] == clean[0]).all() and (got[1, :4] == clean[1, :4]).all(), what
        nan = torch.isnan(got[1, 4:])
        if what == "q":
            assert nan[2].all() and not nan[[0, 1, 3]].any()
        elif what == "v":
            assert nan[:, 9].all() and int(nan.sum()) == 4
        else:
            assert nan.all(), what


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_missing_pages_and_slots(cuda, code, dtype):
    """A key without a page is a key and a value of zeros; a slot that does not exist has no keys; a
    length past the table's width ends there."""
    rng = np.random.default_rng(16)
    for page in (16, 32, 128):
        cache, want = _make(cuda, rng, 1, 60, 2, page, 64, 5, 4, [3 * page, page + 3, 4 * page, 0, 2], code)
        for s, c, bad in ((0, 1, -1), (1, 0, 60), (2, 3, -5), (4, 0, 1 << 30)):
            cache.table[s, c] = want.table[s, c] = bad
        cache.lens[2] = 1 << 30
        cache.lens[3] = -4
        want.lens[2], want.lens[3] = 4 * page, 0
        got, ref = _attend(cuda, rng, cache, want, 6, dtype)
        _hold(got, ref, 4 * page, dtype)
        got, ref = _attend(cuda, rng, cache, want, 6, dtype, slots=[4, -1, 2, 5, 1 << 30, 0, 0, -1 << 31])
        _hold(got, ref, 4 * page, dtype)


@pytest.mark.parametrize("dtype,gap", [("bf16", 0), ("bf16", 1), ("bf16", 8), ("f32", 0), ("f32", 3)])
@pytest.mark.parametrize("d", [64, 80])
def test_attend_strided(cuda, dtype, gap, d):
    """q a slice of a fused projection, out a slice of any alignment, layers of a larger cache."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(17)
    hq, hk, b = 8, 2, 3
    cache, want = _make(cuda, rng, 3, 40, hk, 16, d, b, 20, [200, 31, 3], "int8")
    wide = _values(rng, (b, (hq + 2 * hk) * d + gap), dtype)
    q = _dev(wide, dtype, cuda)[:, gap:].unflatten(1, (hq + 2 * hk, d))[:, :hq]
    out = torch.full((b, (hq + 1) * d + gap), 7.0, dtype=q.dtype, device=cuda)
    view = out[:, gap:].unflatten(1, (hq + 1, d))[:, 1:]
    assert cache.attend(2, q, out=view, scale=0.2).data_ptr() == view.data_ptr()
    k, v = want.values(2)
    n = wide[:, gap:].reshape(b, hq + 2 * hk, d)[:, :hq]
    _hold(_np(view), (*srv.paged(n, k, v, want.table, want.lens, 0, 0.2), _floor(want, dtype, 2)), 200, dtype)
    assert (out[:, :gap + d] == 7).all()
    # Every second page of a larger pool: a page stride of its own.
    pool = [x[0] for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    doubled = []
    for x in pool:
        y = x.view(torch.int8 if x.dtype == torch.int8 else x.dtype).repeat_interleave(2, 0)
        doubled.append(y[::2])
    got = cuda_ops.sdpa_quantized(q, *doubled, cache.table, cache.lens, scale=0.2)
    k, v = want.values(0)
    _hold(_np(got), (*srv.paged(n, k, v, want.table, want.lens, 0, 0.2), _floor(want, dtype)), 200, dtype)
    one = cuda_ops.sdpa_quantized(q[1:2], *doubled, cache.table[1:2], cache.lens[1:2], scale=0.2)
    assert (one == got[1:2]).all() or np.abs(_np(one) - _np(got[1:2])).max() < 0.1


def test_attend_far_pages(cuda):
    """Offsets past 32 bits: the last pages of a cache of five billion codes."""
    import torch
    from enigma.kv_cache import QuantizedKVCache
    rng = np.random.default_rng(18)
    pages, heads, page, d = 5_000_000_000 // (8 * 64 * 128), 8, 64, 128
    k, v = (torch.zeros(1, pages, heads, page, d, dtype=torch.int8, device=cuda) for _ in range(2))
    scales = [torch.zeros(1, pages, heads, 4, device=cuda) for _ in range(2)]
    table = torch.tensor([[pages - 1, pages - 7], [3, pages - 2]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([100, 128], dtype=torch.int32, device=cuda)
    refs = torch.zeros(pages, dtype=torch.int32, device=cuda)
    refs[table.flatten().long()] = 1
    cache = QuantizedKVCache(k, v, *scales, table, lens, refs)
    x = _values(rng, (228, heads, d), "bf16")
    t = _dev(x, "bf16", cuda)
    cache.write(0, t, t, [0, 1], [0, 0], [0, 100, 228])
    cache.check()
    got = cache.read(0, [0, 1], [0, 0], [0, 100, 228])
    small = QuantizedKVCache.empty(1, 4, page, heads, d, 2, 128, device=cuda)
    small.reserve([0, 1], [100, 128])
    small.write(0, t, t, [0, 1], [0, 0], [0, 100, 228])
    want = small.read(0, [0, 1], [0, 0], [0, 100, 228])
    assert all((a == b).all() for a, b in zip(got, want)) and float(got[0].abs().max()) > 1
    q = _dev(_values(rng, (2, 16, d), "bf16"), "bf16", cuda)
    assert (cache.attend(0, q) == small.attend(0, q)).all()


def test_attend_nothing(cuda):
    import torch
    rng = np.random.default_rng(19)
    cache, _ = _make(cuda, rng, 1, 4, 2, 16, 64, 2, 2, [5], "int8")
    q = torch.empty(0, 4, 64, device=cuda)
    assert cache.attend(0, q, slots=[]).shape == (0, 4, 64)
    cache.lens.zero_()
    assert (cache.attend(0, torch.full((2, 4, 64), float("nan"), device=cuda)) == 0).all()


@pytest.mark.parametrize("lens", [[40, 9], [3000, 2000]])
def test_attend_streams_graphs_workspaces(cuda, lens):
    """Calls side by side on two streams; graphs that share a caller's workspace, replayed in turn over
    lengths that change; every run of a call gives the same bits."""
    import torch
    rng = np.random.default_rng(20)
    cache, want = _make(cuda, rng, 1, 90, 2, 64, 128, 2, 50, lens, "e4m3")
    qs = [_dev(_values(rng, (2, 8, 128), "bf16"), "bf16", cuda) for _ in range(2)]
    plain = [cache.attend(0, q) for q in qs]
    assert all((cache.attend(0, q) == y).all() for _ in range(5) for q, y in zip(qs, plain))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(cache.attend(0, qs[i]))
    torch.cuda.synchronize()
    assert all((y == plain[i]).all() for i in range(2) for y in outs[i])
    ws = torch.empty(64 << 20, dtype=torch.uint8, device=cuda)
    graphs, held = [], []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(cache.attend(0, q, workspace=ws))
        graphs.append(g)
    for cut in (0, 7, 0, lens[1] - 1):
        cache.lens.copy_(torch.tensor(lens, device=cuda) - cut)
        ref = [cache.attend(0, q) for q in qs]
        for i in (0, 1, 1, 0):
            graphs[i].replay()
            assert (held[i] == ref[i]).all()


# --------------------------------------------------------------------------------- together
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads_q,heads_kv,d,layout,rotary", [(14, 2, 64, "half", 64),
                                                             (8, 2, 128, "interleaved", 64)])
def test_together(cuda, code, heads_q, heads_kv, d, layout, rotary):
    """Prompts in two chunks (turned, written, their context read back for the packed attention), forked,
    and continued token by token in a captured step: every result against the 64-bit definition on
    the values that the oracle's cache holds."""
    import torch
    from enigma import cuda_ops
    from enigma.kv_cache import QuantizedKVCache
    rng = np.random.default_rng(21)
    page, hq, hk = 32, heads_q, heads_kv
    table = cuda_ops.RopeTable(d, rotary_dim=rotary, layout=layout)
    cache = QuantizedKVCache.empty(2, 60, page, hk, d, slots=6, max_len=250, dtype=_kind(code),
                                   device=cuda)
    want = srv.QuantizedPages(np.zeros(cache.k.shape), np.zeros(cache.v.shape),
                              np.zeros(cache.k_scale.shape), np.zeros(cache.v_scale.shape),
                              np.full((6, cache.width), -1), np.zeros(6), np.zeros(60), code)
    layer = 1

    def turned(n, at):
        fused = _dev(_values(rng, (n, hq + 2 * hk, d), "bf16"), "bf16", cuda)
        q, k, v = fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:]
        positions = torch.tensor(at, dtype=torch.int32, device=cuda)
        cuda_ops.rope(q, k, positions, table, out_q=q, out_k=k)
        return q, k, v

    done = [0, 0]
    for chunk in ([70, 33], [41, 90]):
        total = [a + b for a, b in zip(done, chunk)]
        q, k, v = turned(sum(chunk), np.concatenate([np.arange(a, b) for a, b in zip(done, total)]))
        cu = np.concatenate([[0], np.cumsum(chunk)])
        for c in (cache, want):
            c.reserve([0, 1], total)
        cache.write(layer, k, v, [0, 1], done, cu)
        want.write(layer, _np(k), _np(v), [0, 1], done, cu)
        _same(cache, want)
        back = np.concatenate([[0], np.cumsum(total)])
        ck, cv = cache.read(layer, [0, 1], [0, 0], back)
        plan = cuda_ops.PackedPlan(chunk, total, heads_q=hq, heads_kv=hk)
        got = cuda_ops.sdpa_packed(q, ck, cv, plan)
        rows = np.zeros((2, sum(total), hk, d))
        want.read(layer, [0, 1], [0, 0], back, *rows)
        ref, mag, _, err = srv.packed(_np(q), *rows, chunk, total, 1 / np.sqrt(d))
        assert (np.abs(_np(got) - ref) <= srv.bound(ref, mag, err, max(total), True)).all()
        done = total
    for c in (cache, want):
        c.fork([0, 1, 0], [3, 4, 5])
    _same(cache, want)
    slots = torch.tensor([3, 4, 5], dtype=torch.int32, device=cuda)
    cu = torch.arange(4, dtype=torch.int32, device=cuda)
    q, k, v = (torch.zeros(3, h, d, dtype=torch.bfloat16, device=cuda) for h in (hq, hk, hk))
    starts = cache.lens[slots.long()].clone()

    def step():
        cuda_ops.rope(q, k, starts, table, out_q=q, out_k=k)
        cache.reserve(slots, starts + 1)
        cache.write(layer, k, v, slots, starts, cu)
        return cache.attend(layer, q, slots=slots)

    graph = None
    for t in range(20):
        fresh = [_values(rng, x.shape, "bf16") for x in (q, k, v)]
        for x, y in zip((q, k, v), fresh):
            x.copy_(_dev(y, "bf16", cuda))
        at = [int(want.lens[s]) for s in (3, 4, 5)]
        starts.copy_(torch.tensor(at, device=cuda))
        if t == 1:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        if graph is None:
            out = step()
        else:
            graph.replay()
        want.reserve([3, 4, 5], [a + 1 for a in at])
        want.write(layer, _np(k), _np(v), [3, 4, 5], at, [0, 1, 2, 3])
        for x, y, heads in ((q, fresh[0], hq), (k, fresh[1], hk)):
            ref, mag = srv.rope(y, at, table.frequencies, 1.0, layout)
            tol = 12 * srv.U32 * mag + srv.UBF * (np.abs(ref) + mag * 1e-5)
            assert (np.abs(_np(x) - ref) <= tol).all()
        _same(cache, want)
        ref = srv.paged(_np(q), *want.values(layer), want.table, want.lens, 0, 1 / np.sqrt(d), [3, 4, 5])
        _hold(_np(out), (*ref, _floor(want, "bf16", layer)), max(at) + 1, "bf16")
    cache.check()
