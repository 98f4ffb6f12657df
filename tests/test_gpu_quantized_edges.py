"""GPU parity of the 8-bit cache where its other tests do not look: blocks of caches made elsewhere, rows of
any alignment, heads of 48 and of 144 to 240 elements.  Codes and scales are equal to the 64-bit
oracle's, attention is within the bound of oracle.serving.bound."""
import numpy as np
import pytest

from oracle import numerics as orc
from oracle import serving as srv
from test_gpu_quantized_cache import CODES, _attend, _dev, _hold, _make, _np, _same, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_behind_negative_scales(cuda, code, dtype):
    """A block's scale may be negative where the cache was made elsewhere.  The one of larger magnitude
    stays, with its sign: negative and large enough, negative and too small, zero."""
    rng = np.random.default_rng(31)
    scales = [np.where(rng.random((1, 12, 2, 1)) < 0.7, -1, 1) * np.exp2(rng.integers(-12, 6, (1, 12, 2, 1)))
              for _ in range(2)]
    for x in scales:
        x[0, ::5] = 0
    cache, want = _make(cuda, rng, 1, 12, 2, 16, 64, 6, 2, [5, 1, 15, 16, 9, 30], code,
                        scales=[x.astype(np.float32) for x in scales])
    slots, starts, cu = [0, 1, 2, 4, 5], [5, 1, 15, 9, 30], [0, 3, 4, 5, 12, 14]
    x = _values(rng, (14, 2, 64), dtype)
    cache.write(0, _dev(x, dtype, cuda), _dev(x, dtype, cuda), slots, starts, cu)
    want.write(0, x, x, slots, starts, cu)
    cache.check()
    _same(cache, want)
    assert (want.scales[0] < 0).any()


@pytest.mark.parametrize("code", CODES)
def test_append_behind_any_scale(cuda, code):
    """Scales that are no powers of two: quotients are products with a rounded reciprocal, off by two
    roundings (2^-23) of at most the largest code before they are rounded to a code: half a step, and
    2^-23 of the value."""
    rng = np.random.default_rng(32)
    heads, d = 2, 64
    scales = [(rng.standard_normal((1, 12, heads, 1)) * np.exp2(rng.integers(-4, 6, (1, 12, heads, 1)))
               ).astype(np.float32) for _ in range(2)]
    cache, want = _make(cuda, rng, 1, 12, heads, 16, d, 6, 2, [5, 1, 15, 16, 9, 2], code, scales=scales)
    slots, starts, cu = [0, 1, 2, 4, 5], [5, 1, 15, 9, 2], [0, 3, 4, 5, 12, 16]
    cache.reserve(slots, [8, 2, 16, 16, 6])
    want.reserve(slots, [8, 2, 16, 16, 6])
    x = _values(rng, (16, heads, d), "f32")
    old = [want.values(0)[i].copy() for i in range(2)]
    cache.write(0, _dev(x, "f32", cuda), _dev(x, "f32", cuda), slots, starts, cu)
    want.write(0, x, x, slots, starts, cu)
    cache.check()
    for name, ref, was in (("k", want.scales[0], old[0]), ("v", want.scales[1], old[1])):
        got = getattr(cache, name + "_scale").cpu().numpy()
        np.testing.assert_array_equal(got, ref)
        values = _np(getattr(cache, name))[0] * got[0][..., None]           # pages of one block
        for i, s in enumerate(slots):
            p = want.table[s, 0]
            lens = starts[i] + cu[i + 1] - cu[i]
            true = np.concatenate([was[p][:, :starts[i]], x[cu[i]:cu[i + 1]].transpose(1, 0, 2)], 1)
            y = np.abs(true / got[0, p][..., None])
            step = 1.0 if code == "int8" else np.exp2(np.maximum(np.floor(np.log2(np.maximum(y, 2.0 ** -60))),
                                                                 -6) - 3)
            off = np.abs(values[p][:, :lens] - true)
            assert (off <= np.abs(got[0, p][..., None]) * (step / 2 + y * 2.0 ** -22)).all()


# ------------------------------------------------------------------------- rows of any alignment
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype,gap", [("bf16", 1), ("bf16", 3), ("bf16", 4), ("f32", 1), ("f32", 3)])
@pytest.mark.parametrize("heads,page,d", [(2, 16, 64), (3, 64, 128), (1, 32, 16), (2, 128, 80), (2, 64, 96),
                                          (1, 16, 144), (2, 32, 160), (1, 64, 256)])
def test_write_rows_off_16_bytes(cuda, heads, page, d, dtype, gap, code):
    """Rows that start and lie anywhere: single tokens, short parts, whole blocks, each alone in a request
    (so that a block has them in one, two or more vectors a lane) and together."""
    rng = np.random.default_rng(heads + d + gap)
    cache, want = _make(cuda, rng, 1, 40, heads, page, d, 6, 4 * 128 // page, [5, 17, 0, 2 * page], code)
    for counts in ([1, 1, 1, 1], [2, 3, 5, 1], [page + 9, 0, 33, 16], [1, 20, 3, 40]):
        slots = [3, 0, 1, 2]
        starts = [int(want.lens[s]) for s in slots]
        lens = [a + b for a, b in zip(starts, counts)]
        if max(lens) > want.table.shape[1] * page:
            break
        cache.reserve(slots, lens)
        want.reserve(slots, lens)
        cu = np.concatenate([[0], np.cumsum(counts)])
        wide = _values(rng, (int(cu[-1]), 2 * heads * d + gap), dtype)
        t = _dev(wide, dtype, cuda)[:, gap:].unflatten(1, (2 * heads, d))
        rows = wide[:, gap:].reshape(-1, 2 * heads, d)
        cache.write(0, t[:, :heads], t[:, heads:], slots, starts, cu)
        want.write(0, rows[:, :heads], rows[:, heads:], slots, starts, cu)
        cache.check()
        _same(cache, want)


# ------------------------------------------------------------------- heads of 48, and of 144 to 240
WIDE = [48, 144, 160, 176, 208, 240]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("d", WIDE)
def test_write_and_read_other_heads(cuda, d, page, dtype, code):
    import torch
    rng = np.random.default_rng(d + page)
    heads = 2
    cache, want = _make(cuda, rng, 1, 30, heads, page, d, 4, 128 // page + 2, [5, 33], code)
    for counts in ([1, 1, 70], [2, 3, 1], [30, 17, 16]):
        slots = [0, 1, 3]
        starts = [int(want.lens[s]) for s in slots]
        lens = [a + b for a, b in zip(starts, counts)]
        cache.reserve(slots, lens)
        want.reserve(slots, lens)
        cu = np.concatenate([[0], np.cumsum(counts)])
        x = _values(rng, (int(cu[-1]), heads, d), dtype)
        cache.write(0, _dev(x, dtype, cuda), _dev(x, dtype, cuda), slots, starts, cu)
        want.write(0, x, x, slots, starts, cu)
        cache.check()
        _same(cache, want)
    cu = np.concatenate([[0], np.cumsum([int(want.lens[s]) + 2 for s in slots])])
    ref = np.zeros((2, int(cu[-1]), heads, d))
    want.read(0, slots, [0, 0, 0], cu, *ref)
    kind = torch.bfloat16 if dtype == "bf16" else torch.float32
    for y, r in zip(cache.read(0, slots, [0, 0, 0], cu, dtype=kind), ref):
        np.testing.assert_array_equal(_np(y), r)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads_q,heads_kv", [(8, 2), (14, 2), (20, 1), (3, 3)])
@pytest.mark.parametrize("d", WIDE)
def test_attend_other_heads(cuda, d, heads_q, heads_kv, code):
    """Pages of one block and of several, short and long contexts, tables as wide as the contexts need and
    wider."""
    rng = np.random.default_rng(heads_q + d)
    for page, lens, more in ((16, [1, 15, 16, 17, 33, 100], 0), (64, [700, 0, 47], 1), (128, [2500, 5], 300)):
        pages = sum(-(-n // page) for n in lens) + 2
        for dtype in ("bf16", "f32"):
            cache, want = _make(cuda, rng, 1, pages, heads_kv, page, d, len(lens),
                                -(-max(lens) // page) + more, lens, code)
            got, ref = _attend(cuda, rng, cache, want, heads_q, dtype)
            _hold(got, ref, max(lens), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [48, 144, 240])
def test_attend_unseen_and_nan_other_widths(cuda, d, dtype):
    """What is behind the last key reaches nobody; NaN in an element of a value that is seen reaches that
    element of that sequence's kv head alone; results between other columns leave those as they were."""
    import torch
    rng = np.random.default_rng(d + 1)
    lens, heads_q = [1, 31, 50, 0, 700], 6
    cache, want = _make(cuda, rng, 1, 60, 2, 32, d, 5, 40, lens, "e4m3")
    q = _dev(_values(rng, (5, heads_q, d), dtype), dtype, cuda)
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
    for s, j, e in ((2, 49, d - 1), (4, 333, d - 16), (0, 0, 0)):
        p, r = int(want.table[s, j // 32]), j % 32
        raw = cache.v.view(torch.int8)
        was = int(raw[0, p, 1, r, e])
        raw[0, p, 1, r, e] = 127
        nan = torch.isnan(cache.attend(0, q))
        raw[0, p, 1, r, e] = was
        assert nan[s, heads_q // 2:, e].all() and int(nan.sum()) == heads_q // 2
    wide = torch.full((5, heads_q, d + 3), 7.0, dtype=q.dtype, device=cuda)
    cache.attend(0, q, out=wide[..., 1:1 + d])
    assert (wide[..., 1:1 + d] == clean).all() and (wide[..., 0] == 7).all() and (wide[..., 1 + d:] == 7).all()


# --------------------------------------------------------------------------- far rows, replayed maps
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_past_32_bits(cuda, dtype):
    """Rows of rope, write, read and attention that lie more than 2^31 elements apart."""
    import torch
    from enigma import cuda_ops
    from enigma.kv_cache import QuantizedKVCache
    rng = np.random.default_rng(41)
    kind = torch.bfloat16 if dtype == "bf16" else torch.float32
    n, heads, d, far = 3, 4, 64, 1_100_000_000              # the last row begins past 2^31 elements
    pool = torch.empty(2 * far + heads * d, dtype=kind, device=cuda)
    rows = pool.as_strided((n, heads, d), (far, d, 1))
    x = _values(rng, (n, heads, d), dtype)
    near = _dev(x, dtype, cuda)
    rows.copy_(near)
    table = cuda_ops.RopeTable(d)
    at = torch.tensor([5, 1, 900], dtype=torch.int32, device=cuda)
    want = cuda_ops.rope(near, None, at, table)
    assert (cuda_ops.rope(rows, None, at, table) == want).all()
    assert (cuda_ops.rope(rows, None, at, table, out_q=rows) == want).all()
    caches = [QuantizedKVCache.empty(1, 2, 16, heads, d, 1, 32, device=cuda) for _ in range(2)]
    for cache, t in zip(caches, (rows, want)):
        cache.reserve([0], [n])
        cache.write(0, t, t, [0], [0], [0, n])
        cache.check()
    for name in ("k", "v", "k_scale", "v_scale"):
        assert (getattr(caches[0], name) == getattr(caches[1], name)).all()
    plain = caches[1].attend(0, want, slots=[0] * n)
    assert (caches[0].attend(0, rows, slots=[0] * n) == plain).all()
    got = caches[0].attend(0, want, slots=[0] * n, out=rows)
    assert got.data_ptr() == rows.data_ptr() and (rows == plain).all()
    other = torch.empty_like(want)
    caches[0].read(0, [0], [0], [0, n], out_k=rows, out_v=other)
    k, _ = caches[1].read(0, [0], [0], [0, n], dtype=kind)
    assert (rows == k).all() and (other == k).all()


@pytest.mark.parametrize("code", CODES)
def test_maps_replayed(cuda, code):
    """Forks, a write behind them and a compaction as one captured graph, replayed: pages and scales as the
    same requests give them one by one."""
    import torch
    rng = np.random.default_rng(42)
    cache, want = _make(cuda, rng, 2, 40, 3, 32, 64, 6, 4, [70, 33, 96], code)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    parents, children, gone = ints(0, 1, 0), ints(3, 4, 5), ints(4)
    slots, starts, cu = ints(3, 5), ints(70, 70), ints(0, 2, 7)
    lens = ints(72, 75)
    x = _values(rng, (7, 3, 64), "bf16")
    t = _dev(x, "bf16", cuda)

    def requests(c, a, b, s, n, r, begin, packed, g):
        c.fork(a, b)
        c.reserve(s, n)
        c.write(1, r, r, s, begin, packed)
        c.free(g)
        c.compact()

    def plain():
        requests(want, [0, 1, 0], [3, 4, 5], [3, 5], [72, 75], x, [70, 70], [0, 2, 7], [4])

    requests(cache, parents, children, slots, lens, t, starts, cu, gone)
    plain()
    cache.check()
    _same(cache, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        requests(cache, parents, children, slots, lens, t, starts, cu, gone)
    for i in range(3):
        t.mul_(2.0)
        x = x * np.float32(2)
        graph.replay()
        plain()
        cache.check()
        _same(cache, want)
