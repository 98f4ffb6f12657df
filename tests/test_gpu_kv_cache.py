"""GPU parity of the paged cache's operations: the page map and every page, bit for bit, against
the oracle's cache; requests that cannot be met change nothing."""
import numpy as np
import pytest

from oracle import serving as srv

pytestmark = pytest.mark.gpu


def _make(cuda, rng, layers, pages, heads, page, d, slots, width, lens, dtype="bf16"):
    """A cache whose first len(lens) slots hold sequences on scattered pages, and its oracle."""
    import torch
    from enigma.kv_cache import PagedKVCache
    table = np.full((slots, width), -1, np.int32)
    refs, full = np.zeros(pages, np.int32), np.zeros(slots, np.int32)
    order, at = rng.permutation(pages), 0
    for s, n in enumerate(lens):
        m = -(-n // page)
        table[s, :m] = order[at:at + m]
        refs[order[at:at + m]] = 1
        full[s] = n
        at += m
    k, v = (rng.integers(0, 30000, (layers, pages, heads, page, d)).astype(np.int16)
            for _ in range(2))       # bit patterns; compared as such

    def dev(x):
        t = torch.from_numpy(x).to(cuda)
        return t.view(torch.bfloat16) if dtype == "bf16" else t.to(torch.float32)

    cache = PagedKVCache(dev(k), dev(v), *(torch.from_numpy(x).to(cuda)
                                           for x in (table, full, refs)))
    return cache, srv.Pages(k, v, table, full, refs)


def _bits(t):
    import torch
    return (t.view(torch.int16) if t.dtype == torch.bfloat16 else t.to(torch.int16)).cpu().numpy()


def _same(cache, want):
    for name in ("table", "lens", "refs"):
        np.testing.assert_array_equal(getattr(cache, name).cpu().numpy(), getattr(want, name), name)
    np.testing.assert_array_equal(_bits(cache.k), want.k)
    np.testing.assert_array_equal(_bits(cache.v), want.v)


SHAPES = [(2, 60, 2, 16, 64, "bf16"), (1, 300, 3, 4, 5, "bf16"), (3, 50, 1, 128, 8, "f32"),
          (1, 9000, 1, 16, 2, "f32")]


@pytest.mark.parametrize("layers,pages,heads,page,d,dtype", SHAPES)
def test_fork(cuda, layers, pages, heads, page, d, dtype):
    rng = np.random.default_rng(pages)
    lens = [page * 3 + 1, 0, page * 2, 1, page * 4 - 1]
    cache, want = _make(cuda, rng, layers, pages, heads, page, d, 16, 5, lens, dtype)
    for parents, children in (([0, 0, 0, 2, 4], [5, 9, 7, 15, 6]), ([3, 1], [8, 0]),
                              ([5, 9], [7, 15]), ([2], [4])):
        cache.fork(parents, children)
        want.fork(parents, children)
        cache.check()
        _same(cache, want)


@pytest.mark.parametrize("layers,pages,heads,page,d,dtype", SHAPES)
def test_reserve_write_free(cuda, layers, pages, heads, page, d, dtype):
    import torch
    rng = np.random.default_rng(pages + 1)
    cache, want = _make(cuda, rng, layers, pages, heads, page, d, 12, 6, [page + 1, 5], dtype)
    slots, lens = [1, 7, 0, 3], [2 * page + 3, 1, page + 1, 3 * page]
    starts = [int(want.lens[s]) for s in slots]
    cache.reserve(slots, lens)
    want.reserve(slots, lens)
    _same(cache, want)
    cu = np.concatenate([[0], np.cumsum([n - s for n, s in zip(lens, starts)])])
    rows = rng.integers(0, 30000, (2, int(cu[-1]), heads + 2, d)).astype(np.int16)
    t = torch.from_numpy(rows).to(cuda)
    t = t.view(torch.bfloat16) if dtype == "bf16" else t.to(torch.float32)
    cache.write(layers - 1, t[0][:, 1:1 + heads], t[1][:, 2:2 + heads], slots, starts, cu)
    want.write(layers - 1, rows[0][:, 1:1 + heads], rows[1][:, 2:2 + heads], slots, starts, cu)
    cache.check()
    _same(cache, want)
    cache.fork([1, 0], [10, 11])
    want.fork([1, 0], [10, 11])
    for gone in ([1, 3, 2], [10, 0]):
        cache.free(gone)
        want.free(gone)
        cache.check()
        _same(cache, want)


@pytest.mark.parametrize("layers,pages,heads,page,d,dtype", SHAPES)
def test_compact(cuda, layers, pages, heads, page, d, dtype):
    rng = np.random.default_rng(pages + 2)
    lens = [page * (1 + i % 3) - i % 2 for i in range(9)]
    cache, want = _make(cuda, rng, layers, pages, heads, page, d, 14, 4, lens, dtype)
    cache.fork([0, 3], [10, 11])
    want.fork([0, 3], [10, 11])
    for _ in range(2):                  # the second time nothing moves
        cache.compact()
        want.compact()
        cache.check()
        _same(cache, want)
    live = int((want.refs > 0).sum())
    assert (want.refs[:live] > 0).all()
    cache.free(list(range(12)))
    want.free(list(range(12)))
    cache.compact()                     # nothing is in use
    _same(cache, want)


def test_copy_pages(cuda):
    rng = np.random.default_rng(5)
    cache, want = _make(cuda, rng, 3, 40, 2, 16, 24, 4, 4, [30, 2])
    cache.copy_pages([0, 7, 7, 39], [1, 2, 3, 38])
    want.copy_pages([0, 7, 7, 39], [1, 2, 3, 38])
    cache.check()
    _same(cache, want)


def test_requests_that_cannot_be_met_change_nothing(cuda):
    from enigma import EnigmaError
    rng = np.random.default_rng(6)
    page = 16
    cache, want = _make(cuda, rng, 2, 8, 2, page, 8, 6, 4, [page + 2, 3 * page, 5])   # 6 pages used
    bad = [lambda: cache.fork([0, 1], [3, 3]), lambda: cache.fork([0, 1], [1, 3]),
           lambda: cache.fork([6], [3]), lambda: cache.fork([0], [-1]), lambda: cache.free([0, 0]),
           lambda: cache.free([9]), lambda: cache.reserve([0], [page]),
           lambda: cache.reserve([0], [4 * page + 1]), lambda: cache.reserve([2, 2], [9, 9]),
           lambda: cache.copy_pages([0, 8], [8, 0]), lambda: cache.copy_pages([-1], [0])]
    for request in bad:
        request()
        with pytest.raises(EnigmaError, match="does not exist"):
            cache.check()
        cache.check()                   # said once
        _same(cache, want)
    for request in (lambda: cache.reserve([3], [3 * page]), lambda: cache.fork([0, 2, 0], [3, 4, 5])):
        request()
        with pytest.raises(EnigmaError, match="free pages"):
            cache.check()
        _same(cache, want)
    cache.fork([0, 2], [3, 4])          # what fits still does
    want.fork([0, 2], [3, 4])
    cache.check()
    _same(cache, want)


def test_write_without_a_page_is_left_out(cuda):
    import torch
    from enigma import EnigmaError
    rng = np.random.default_rng(7)
    cache, want = _make(cuda, rng, 1, 6, 1, 16, 8, 2, 2, [10])
    rows = torch.zeros(3, 1, 8, dtype=torch.bfloat16, device=cuda)
    for slots, starts in (([0], [16]), ([1], [0]), ([5], [0]), ([0], [40]), ([0], [-9])):
        cache.write(0, rows, rows, slots, starts, [0, 3])
        with pytest.raises(EnigmaError):
            cache.check()
        _same(cache, want)


def test_graph_capture(cuda):
    """A turnover captured once and replayed: the same map as the calls one by one."""
    import torch
    rng = np.random.default_rng(8)
    cache, want = _make(cuda, rng, 1, 64, 2, 16, 16, 8, 6, [40, 3, 64])
    slots = torch.tensor([0, 2, 5], dtype=torch.int32, device=cuda)
    lens = torch.tensor([17, 90, 33], dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.free(slots)
        cache.reserve(slots, lens)
    for _ in range(3):
        graph.replay()
        want.free([0, 2, 5])
        want.reserve([0, 2, 5], [17, 90, 33])
        cache.check()
        _same(cache, want)


def test_refusals(cuda):
    import torch
    from enigma import _native
    from enigma.kv_cache import PagedKVCache
    cache = PagedKVCache.empty(2, 8, 16, 2, 64, slots=4, max_len=100)
    assert cache.width == 7 and cache.k.shape == (2, 8, 2, 16, 64)
    rows = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="layer"):
        cache.write(2, rows, rows, [0], [0], [0, 3])
    with pytest.raises(ValueError, match="expected rows"):
        cache.write(0, rows[:, :1], rows[:, :1], [0], [0], [0, 3])
    with pytest.raises(TypeError, match="share a dtype"):
        cache.write(0, rows.float(), rows.float(), [0], [0], [0, 3])
    with pytest.raises(ValueError, match="cu holds"):
        cache.write(0, rows, rows, [0], [0], [0, 1, 3])
    with pytest.raises(ValueError, match="differ in length"):
        cache.fork([0, 1], [2])
    with pytest.raises(_native.EnigmaCudaError, match="at most once"):
        cache.free([0, 1, 2, 3, 0])
    with pytest.raises(ValueError, match="int32"):
        PagedKVCache(cache.k, cache.v, cache.table.long(), cache.lens, cache.refs)
    with pytest.raises(ValueError, match="expected table"):
        PagedKVCache(cache.k, cache.v, cache.table, cache.lens, cache.refs[:4].contiguous())
    with pytest.raises(TypeError, match="unsupported dtype"):
        PagedKVCache(cache.k.half(), cache.v.half(), cache.table, cache.lens, cache.refs)


def test_many_pages_and_requests(cuda):
    """More pages than threads, requests of hundreds of entries, long rows."""
    rng = np.random.default_rng(9)
    lens = [int(x) for x in rng.integers(0, 300, 700)]
    cache, want = _make(cuda, rng, 1, 60000, 1, 4, 2, 2300, 80, lens, "f32")
    parents = [int(x) for x in rng.integers(0, 700, 1400)]
    children = [int(x) for x in 700 + rng.permutation(1600)[:1400]]
    cache.fork(parents, children)
    want.fork(parents, children)
    cache.check()
    _same(cache, want)
    slots = [int(x) for x in rng.permutation(2300)[:1100]]
    grown = [int(min(320, want.lens[s] + x)) for s, x in zip(slots, rng.integers(0, 90, 1100))]
    cache.reserve(slots, grown)
    want.reserve(slots, grown)
    cache.free(slots[::2])
    want.free(slots[::2])
    cache.compact()
    want.compact()
    cache.check()
    _same(cache, want)


def test_more_pages_asked_for_than_an_int_holds(cuda):
    """The sum of what a request needs does not wrap into something that fits."""
    import torch
    from enigma import EnigmaError
    from enigma.kv_cache import PagedKVCache
    n, width = 4096, 1 << 20
    k = torch.zeros(1, 8, 1, 1, 2, device=cuda)
    cache = PagedKVCache(k, k.clone(), torch.full((n, width), -1, dtype=torch.int32, device=cuda),
                         torch.zeros(n, dtype=torch.int32, device=cuda),
                         torch.zeros(8, dtype=torch.int32, device=cuda))
    cache.reserve(list(range(n)), [width] * n)              # 2^32 pages
    with pytest.raises(EnigmaError, match="free pages"):
        cache.check()
    assert int(cache.refs.sum()) == 0 and int(cache.lens.sum()) == 0
