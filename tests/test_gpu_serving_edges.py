"""Edge values of the serving operators on all their kernels: padded slots, tables with holes, NaN and
what lies behind a length.  The same meaning whatever the type and the head size, against the 64-bit
oracle under its derived bound (oracle.serving.bound)."""
import numpy as np
import pytest

from oracle import numerics as orc
from oracle import serving as srv

pytestmark = pytest.mark.gpu

# Heads of 64 and 128 in bf16 run on the tensor cores, the others on CUDA cores.
KINDS = [("f32", 64), ("bf16", 96), ("bf16", 64), ("bf16", 128)]


def _values(rng, shape, dtype):
    x = rng.standard_normal(shape, dtype=np.float32)
    return orc.bf16_round(x) if dtype == "bf16" else x


def _dev(a, dtype, cuda):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    return t.bfloat16() if dtype == "bf16" else t


def _ints(x, cuda):
    import torch
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def _paged(cuda, dtype, q, k, v, table, lens, **args):
    from enigma import cuda_ops
    slots = args.pop("slots", None)
    out = cuda_ops.sdpa_shared_prefix(
        *(_dev(x, dtype, cuda) for x in (q, k, v)), _ints(table, cuda), _ints(lens, cuda),
        slots=None if slots is None else _ints(slots, cuda), **args)
    return out.float().cpu().numpy().astype(np.float64)


def _hold(got, ref, mag, err, keys, dtype):
    tol = srv.bound(ref, mag, err, keys, dtype == "bf16")
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= tol).all(), (np.abs(got - ref) / tol).max()


# Table widths in pages of 16: one launch reads the rows, or the prefix and own keys are apart.
@pytest.mark.parametrize("width", [4, 120])
@pytest.mark.parametrize("dtype,d", KINDS)
def test_a_slot_that_does_not_exist_is_alone(cuda, dtype, d, width):
    """A padded batch: only the padded rows are empty, in first place too."""
    rng = np.random.default_rng(d + width)
    k, v = (_values(rng, (9, 2, 16, d), dtype) for _ in range(2))
    table = np.full((4, width), -1, np.int32)
    table[:3, :3] = rng.permutation(9).reshape(3, 3)
    lens = np.array([40, 17, 33, 0], np.int32)
    q = _values(rng, (4, 8, d), dtype)
    for slots in ([-1, 0, 2, 1], [4, 1, -7, 2], [0, -1, 1 << 30, 2]):
        got = _paged(cuda, dtype, q, k, v, table, lens, slots=slots)
        ref, mag, _, err = srv.paged(q, k, v, table, lens, 0, d ** -0.5, slots)
        _hold(got, ref, mag, err, 40, dtype)
        assert [bool((row == 0).all()) for row in got] == [not 0 <= s < 3 for s in slots]


@pytest.mark.parametrize("width", [4, 120])
@pytest.mark.parametrize("dtype,d", KINDS)
def test_a_key_without_a_page_reads_as_zeros(cuda, dtype, d, width):
    """Holes in a table, page numbers outside the cache, a prefix behind a slot that does not exist:
    keys and values of zeros, with a weight of their own."""
    rng = np.random.default_rng(d + width + 1)
    k, v = (_values(rng, (9, 2, 16, d), dtype) for _ in range(2))
    table = np.full((3, width), -1, np.int32)
    table[:, :3] = [[0, -1, 4], [5, 1 << 30, 2], [-1, 8, 9]]
    lens = np.array([40, 33, 20], np.int32)
    q = _values(rng, (3, 8, d), dtype)
    for prefix, slots in ((0, None), (20, None), (20, [1, 0, 2]), (7, [-1, 2, 0]), (39, [9, 1, 0])):
        got = _paged(cuda, dtype, q, k, v, table, lens, prefix_len=prefix, slots=slots)
        ref, mag, _, err = srv.paged(q, k, v, table, lens, prefix, d ** -0.5, slots)
        _hold(got, ref, mag, err, 40, dtype)


@pytest.mark.parametrize("width", [4, 120])
@pytest.mark.parametrize("dtype,d", KINDS)
def test_nan_reaches_the_rows_that_see_it_paged(cuda, dtype, d, width):
    """A NaN query, or a NaN in a key that is seen: NaN, not the softmax of the other keys.  The other
    sequences' results are the same bits as without it."""
    rng = np.random.default_rng(d + width + 2)
    k, v = (_values(rng, (9, 2, 16, d), dtype) for _ in range(2))
    table = np.full((3, width), -1, np.int32)
    table[:, :3] = rng.permutation(9).reshape(3, 3)
    q = _values(rng, (3, 8, d), dtype)
    for lens in ([40, 17, 33], [5, 1, 48]):
        for prefix in (0, 20):
            clean = _paged(cuda, dtype, q, k, v, table, lens, prefix_len=prefix)
            bad = q.copy()
            bad[1, 2] = np.nan
            got = _paged(cuda, dtype, bad, k, v, table, lens, prefix_len=prefix)
            assert np.isnan(got[1, 2]).all()
            others = np.ones((3, 8), bool)
            others[1, 2] = False
            assert (got[others] == clean[others]).all()
        # Key 4 of sequence 0, kv head 1; with a prefix everybody who has that many keys sees it.
        bad = k.copy()
        bad[table[0, 0], 1, 4, 3] = np.nan
        for prefix in (0, 20):
            clean = _paged(cuda, dtype, q, k, v, table, lens, prefix_len=prefix)
            got = _paged(cuda, dtype, q, bad, v, table, lens, prefix_len=prefix)
            for b in range(3):
                hit = b == 0 or (prefix > 0 and lens[b] > 4)
                assert np.isnan(got[b, 4:]).all() if hit else (got[b] == clean[b]).all()
                assert (got[b, :4] == clean[b, :4]).all()


# Rows whose keys the plan splits, that are split inside one launch (CUDA cores), and that are not.
@pytest.mark.parametrize("lens_q,lens_k", [([700, 45, 1024, 3], [700, 45, 1024, 3]),
                                           ([5, 30], [7, 2000]), ([150], [150])])
@pytest.mark.parametrize("dtype,d", KINDS)
def test_nan_reaches_the_rows_that_see_it_packed(cuda, dtype, d, lens_q, lens_k):
    """A NaN query or a NaN in a key that is seen gives NaN in the result and the log-sum-exp; the
    rows that do not see it keep their bits."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(d + sum(lens_k))
    tq, tk = sum(lens_q), sum(lens_k)
    q, k, v = (_values(rng, (t, h, d), dtype) for t, h in ((tq, 14), (tk, 2), (tk, 2)))
    plan = cuda_ops.PackedPlan(lens_q, lens_k, heads_q=14, heads_kv=2)

    def run(*arrays):
        return cuda_ops.sdpa_packed(*(_dev(x, dtype, cuda) for x in arrays), plan, return_lse=True)

    clean, clean_lse = run(q, k, v)
    at_q, at_k = np.cumsum([0] + lens_q), np.cumsum([0] + lens_k)
    s = int(np.argmax(lens_k))                     # the longest sequence
    for where in ("middle query", "last query", "first key", "late key"):
        hit = torch.zeros(tq, 14, dtype=torch.bool, device=cuda)
        bad_q, bad_k = q.copy(), k.copy()
        if where.endswith("query"):
            row = at_q[s] + (lens_q[s] - 1 if where.startswith("last") else lens_q[s] // 2)
            bad_q[row, 3] = np.nan
            hit[row, 3] = True
        else:
            j = 0 if where == "first key" else lens_k[s] * 3 // 4
            bad_k[at_k[s] + j, 1, d // 2] = np.nan
            first = max(0, j - (lens_k[s] - lens_q[s]))        # the first token that sees key j
            hit[at_q[s] + first:at_q[s + 1], 7:] = True
        out, lse = run(bad_q, bad_k, v)
        assert out[hit].isnan().all() and lse[hit].isnan().all()
        assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])


@pytest.mark.parametrize("width,prefix", [(4, 60), (120, 60), (120, 700), (120, 1920)])
@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("lens", [[40] * 5, [40, 0, 7, 33, 12], [0, 0, 50, 0, 1], [1] * 70 + [0, 690],
                                  [300] * 40 + [5] * 40 + [129, 64], [128, 128], [0, 0]],
                         ids=lambda x: f"{len(x)}-{max(x)}")
def test_what_no_sequence_sees_of_the_prefix(cuda, dtype, d, width, prefix, lens):
    """Sequences that end before the prefix does: what their pages hold behind that (unwritten rows,
    NaN here) reaches nobody."""
    lens = [min(n, width * 16) for n in lens]
    rng = np.random.default_rng(d + width + prefix + len(lens))
    most, held = max(lens), -(-max(max(lens), min(prefix, 800)) // 16)      # keys seen; pages held
    k, v = (_values(rng, (held, 2, 16, d), dtype) for _ in range(2))
    order = rng.permutation(held)
    for x in (k, v):                               # in the order of the keys: NaN from key `most` on
        y = np.empty((2, held * 16, d), np.float32)
        y[:] = x.transpose(1, 0, 2, 3).reshape(2, held * 16, d)
        y[:, most:] = np.nan
        x[order] = y.reshape(2, held, 16, d).transpose(1, 0, 2, 3)
    table = np.full((len(lens), width), -1, np.int32)
    table[:, :min(width, held)] = order[:width]
    q = _values(rng, (len(lens), 8, d), dtype)
    slots = rng.permutation(len(lens))
    for s in (None, slots):
        got = _paged(cuda, dtype, q, k, v, table, lens, prefix_len=prefix, slots=s)
        ref, mag, _, err = srv.paged(q, k, v, table, lens, prefix, d ** -0.5, s)
        _hold(got, ref, mag, err, max(1, most), dtype)


def test_waits_that_give_up(cuda):
    """With a timeout already reported, waits may give up early: calls made then have no result, but
    end in order, the report arrives, and the next calls are right."""
    import torch
    from enigma import _native, cuda_ops
    rng = np.random.default_rng(31)
    lens = [2000, 37, 900]
    q, k, v = (_dev(_values(rng, (sum(lens), h, 128), "bf16"), "bf16", cuda) for h in (8, 2, 2))
    plan = cuda_ops.PackedPlan(lens, heads_q=8, heads_kv=2)
    pages = [_dev(_values(rng, (300, 2, 64, 128), "bf16"), "bf16", cuda) for _ in range(2)]
    table = _ints([list(range(50)) + list(range(60 + 10 * b, 90 + 10 * b)) for b in range(20)], cuda)
    rows = _ints([3200 + 90 * b for b in range(20)], cuda)

    def calls():
        return [cuda_ops.sdpa_packed(q, k, v, plan)] + [
            cuda_ops.sdpa_shared_prefix(q[:20], *pages, table, n, prefix_len=p)
            for n, p in ((rows, 3200), (rows, 0), (rows // 4, 0))]

    want = calls()
    torch.cuda.synchronize()
    lib = _native.lib()
    for _ in range(3):
        _native.check(lib.enigma_check_timeout_path(10, None), "timeout probe")
        calls()
        with pytest.raises(_native.EnigmaCudaError, match="exceeded its limit"):
            cuda_ops.synchronize(0)
        got = calls()
        cuda_ops.synchronize(0)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype,d", KINDS)
def test_more_queries_than_table_rows(cuda, dtype, d):
    """Slots may name a row more than once, and padding needs no row of its own."""
    rng = np.random.default_rng(d + 3)
    k, v = (_values(rng, (5, 2, 16, d), dtype) for _ in range(2))
    table, lens, slots = [[3, 1], [3, 4]], [30, 18], [1, 0, 1, 1, -1, 0]
    q = _values(rng, (6, 8, d), dtype)
    for prefix in (0, 16):
        got = _paged(cuda, dtype, q, k, v, np.array(table), lens, prefix_len=prefix, slots=slots)
        ref, mag, _, err = srv.paged(q, k, v, np.array(table), lens, prefix, d ** -0.5, slots)
        _hold(got, ref, mag, err, 30, dtype)


def _cache(cuda, rng, pages=8):
    import torch
    from enigma.kv_cache import PagedKVCache
    cache = PagedKVCache.empty(2, pages, 16, 2, 8, slots=4, max_len=64, dtype=torch.float32,
                               device=cuda)
    for x in (cache.k, cache.v):
        x.copy_(torch.from_numpy(rng.standard_normal(x.shape, dtype=np.float32)))
    return cache


def test_copy_pages_is_whole_or_not_at_all(cuda):
    """One page that does not exist among others that do: nothing is copied."""
    import torch
    from enigma import EnigmaError
    cache = _cache(cuda, np.random.default_rng(41))
    k, v = cache.k.clone(), cache.v.clone()
    for src, dst in (([0, 99], [1, 2]), ([0, 1], [2, -1]), ([0, -1, 3], [4, 5, 6]),
                     ([0, 1, 2, 3], [4, 5, 6, 8])):
        cache.copy_pages(src, dst)
        with pytest.raises(EnigmaError, match="does not exist"):
            cache.check()
        assert torch.equal(cache.k, k) and torch.equal(cache.v, v)
    cache.copy_pages([0, 3], [7, 5])
    cache.check()
    k[:, 7], k[:, 5], v[:, 7], v[:, 5] = k[:, 0], k[:, 3], v[:, 0], v[:, 3]
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)


def test_requests_are_whole_numbers_of_any_width(cuda):
    """A slot that an int32 does not hold is not another slot; fractions and masks are no slots."""
    import torch
    from enigma import EnigmaError
    cache = _cache(cuda, np.random.default_rng(42))
    cache.reserve([0, 1], [20, 5])
    for bad in (1 << 32, (1 << 32) + 1, -(1 << 33), 1 << 31):
        cache.free(torch.tensor([bad], device=cuda))
        with pytest.raises(EnigmaError, match="does not exist"):
            cache.check()
        for host in (torch.tensor([bad]), [bad], np.array([bad])):
            with pytest.raises(ValueError, match="int32"):
                cache.free(host)
    cache.reserve([2], torch.tensor([(1 << 32) + 3], device=cuda))
    with pytest.raises(EnigmaError, match="does not fit"):
        cache.check()
    for bad in ([0.7], torch.tensor([0.0], device=cuda), torch.tensor([True]), np.array([1.0])):
        with pytest.raises(TypeError, match="whole numbers"):
            cache.free(bad)
    assert cache.lens.tolist() == [20, 5, 0, 0]
    for good in ([1], torch.tensor([1]), np.array([1], np.uint8), torch.tensor([1], device=cuda),
                 torch.tensor([1, 0], dtype=torch.int16, device=cuda)[:1], []):
        cache.free(good)
        cache.check()
        assert cache.lens.tolist() == [20, 0 if len(good) else cache.lens[1].item(), 0, 0]
        cache.reserve([1], [5])


def test_check_waits_for_every_stream(cuda):
    """A request on another stream that cannot be met is raised, though this stream is idle."""
    import torch
    from enigma import EnigmaError
    cache = _cache(cuda, np.random.default_rng(43))
    twice = _ints([1, 1], cuda)
    side = torch.cuda.Stream()
    for wait in (1000, 200_000_000):               # the first time loads what runs
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(wait)
            cache.free(twice)
        with pytest.raises(EnigmaError, match="a slot twice"):
            cache.check()
        cache.check()


def test_rows_without_a_slot_are_refused(cuda):
    import torch
    from enigma import _native
    cache = _cache(cuda, np.random.default_rng(44))
    rows = torch.zeros(3, 2, 8, device=cuda)
    with pytest.raises(_native.EnigmaCudaError, match="without a slot"):
        cache.write(0, rows, rows, [], [], [0])
    cache.write(0, rows[:0], rows[:0], [], [], [0])          # nothing to write
    cache.write(0, rows[:0], rows[:0], [1], [0], [0, 0])
    cache.check()


@pytest.mark.parametrize("dtype,d", KINDS)
def test_axes_of_length_one_have_any_stride(cuda, dtype, d):
    """One row of a wider table, one length of several, one kv head seen through a transpose, one
    page: contiguous whatever the stride of an axis that holds one element."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(d + 4)
    k, v = (_dev(_values(rng, (4, 16, 1, d), dtype), dtype, cuda).transpose(1, 2) for _ in range(2))
    q = _dev(_values(rng, (1, 4, d), dtype), dtype, cuda)
    table, lens, slots = _ints([[2, 0, 3], [1, 2, 3]], cuda), _ints([30, 7], cuda), _ints([0, 5], cuda)
    want = cuda_ops.sdpa_shared_prefix(q, k.contiguous(), v.contiguous(),
                                       table[:1, :2].contiguous().clone(), lens[:1].clone())
    ref, mag, _, err = srv.paged(q.float().cpu().numpy(), k.float().cpu().numpy(),
                                 v.float().cpu().numpy(), [[2, 0]], [30], 0, d ** -0.5)
    _hold(want.float().cpu().numpy().astype(np.float64), ref, mag, err, 30, dtype)
    got = cuda_ops.sdpa_shared_prefix(q, k, v, table[:1, :2], lens[::2], slots=slots[::2])
    assert torch.equal(got, want)
    one = [x[2:3].as_strided((1, 1, 16, d), (7, 3, d, 1)) for x in (k, v)]
    assert torch.equal(cuda_ops.sdpa_shared_prefix(q, *one, _ints([[0]], cuda), _ints([16], cuda)),
                       cuda_ops.sdpa_shared_prefix(q, k, v, table[:1, :1], _ints([16], cuda)))
    with pytest.raises(ValueError, match="int32"):
        cuda_ops.sdpa_shared_prefix(q, k, v, table[:, :2], lens)


@pytest.mark.parametrize("dtype,d", KINDS)
def test_an_empty_batch(cuda, dtype, d):
    """No sequences, with or without table rows: an empty result."""
    import torch
    from enigma import cuda_ops
    k = torch.zeros(4, 2, 16, d, device=cuda, dtype=torch.float32 if dtype == "f32" else torch.bfloat16)
    q, table, lens = k.new_zeros(0, 8, d), _ints([[0, 1], [2, 3]], cuda), _ints([5, 20], cuda)
    for rows in (2, 0):
        for prefix in (0, 20):
            out = cuda_ops.sdpa_shared_prefix(q, k, k, table[:rows], lens[:rows], prefix_len=prefix)
            assert out.shape == (0, 8, d) and out.dtype == k.dtype
    out = cuda_ops.sdpa_shared_prefix(q, k, k, table, lens, slots=lens[:0])
    assert out.shape == (0, 8, d)


@pytest.mark.parametrize("lens_q,lens_k", [([70, 5, 300], [70, 5, 300]), ([3, 20], [4000, 700])])
@pytest.mark.parametrize("dtype,d", KINDS)
def test_a_plan_for_more_heads_writes_no_others(cuda, dtype, d, lens_q, lens_k):
    """The C entry is given a plan that was made for more kv heads than the tensors have: the heads
    they have are computed, and nothing is written beside them."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(d + 5)
    tq, tk = sum(lens_q), sum(lens_k)
    q, k, v = (_dev(_values(rng, (t, 2, d), dtype), dtype, cuda) for t in (tq, tk, tk))
    want = cuda_ops.sdpa_packed(q, k, v, cuda_ops.PackedPlan(lens_q, lens_k, heads_q=2, heads_kv=2))
    plan = cuda_ops.PackedPlan(lens_q, lens_k, heads_q=8, heads_kv=8)
    plan.heads_q = plan.heads_kv = 2
    wide = torch.full((tq, 9, d), 5.0, dtype=q.dtype, device=cuda)       # room for 8 heads and more
    got = cuda_ops.sdpa_packed(q, k, v, plan, out=wide[:, :2])
    assert (wide[:, 2:] == 5).all()
    tol = srv.bound(np.zeros(()), 4.0, np.zeros(1), max(lens_k), dtype == "bf16")
    assert float((got.float() - want.float()).abs().max()) <= 2 * float(tol.max())
