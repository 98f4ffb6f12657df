"""GPU parity of packed prompt attention and of paged attention with a shared prefix against the
64-bit oracle, at the sizes, masks, strides and values where they can go wrong.  The bound is
oracle.serving.bound: derived from the roundings of fp32 sums and of bf16 weights and results."""
import numpy as np
import pytest

from oracle import numerics as orc
from oracle import serving as srv

pytestmark = pytest.mark.gpu


def _values(rng, shape, dtype):
    x = rng.standard_normal(shape, dtype=np.float32)
    return orc.bf16_round(x) if dtype == "bf16" else x


def _dev(a, dtype, cuda):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a)).to(cuda)
    return t.bfloat16() if dtype == "bf16" else t


def _np(t):
    return t.float().cpu().numpy().astype(np.float64)


def _hold(got, ref, mag, err, keys, dtype):
    tol = srv.bound(ref, mag, err, keys, dtype == "bf16")
    off = np.abs(got - ref)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), (off / tol).max()


# ------------------------------------------------------------------ packed prompts
LENS = [
    ([1], [1]),
    ([5, 1, 131], [5, 1, 131]),
    ([127, 128, 129], [127, 128, 129]),
    ([0, 257, 0, 33], [0, 257, 0, 33]),
    ([3, 64, 1], [300, 64, 515]),           # the last tokens of longer contexts
    ([70, 9], [40, 0]),                     # more queries than keys: rows that see nothing
    ([300], [700]),
]


@pytest.mark.parametrize("lens", LENS, ids=lambda p: "-".join(map(str, p[0])))
@pytest.mark.parametrize("heads_q,heads_kv,d,dtype", [
    (14, 2, 64, "bf16"), (8, 2, 128, "bf16"), (3, 3, 128, "bf16"), (8, 1, 64, "bf16"),
    (40, 2, 64, "bf16"), (4, 2, 96, "bf16"), (14, 2, 64, "f32"), (2, 2, 128, "f32"),
    (4, 1, 80, "f32"), (3, 1, 7, "f32")])
def test_packed(cuda, lens, heads_q, heads_kv, d, dtype):
    from enigma import cuda_ops
    lq, lk = lens
    rng = np.random.default_rng(len(lq) * 1000 + sum(lq) + d)
    q = _values(rng, (sum(lq), heads_q, d), dtype)
    k = _values(rng, (sum(lk), heads_kv, d), dtype)
    v = _values(rng, (sum(lk), heads_kv, d), dtype)
    plan = cuda_ops.PackedPlan(lq, lk, heads_q=heads_q, heads_kv=heads_kv)
    out, lse = cuda_ops.sdpa_packed(_dev(q, dtype, cuda), _dev(k, dtype, cuda),
                                    _dev(v, dtype, cuda), plan, return_lse=True)
    ref, mag, rlse, err = srv.packed(q, k, v, lq, lk, 1 / np.sqrt(d))
    _hold(_np(out), ref, mag, err, max(lk), dtype)
    got = _np(lse)
    empty = np.isinf(rlse)
    assert (got[empty] == -np.inf).all() and (_np(out)[empty] == 0).all()
    tol = 4 * (err + (max(lk) + 16) * srv.U32) + 8 * srv.U32 * np.abs(np.where(empty, 0, rlse))
    assert (np.abs(got[~empty] - rlse[~empty]) <= tol[~empty]).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_packed_not_causal(cuda, dtype, d):
    from enigma import cuda_ops
    rng = np.random.default_rng(3)
    lq, lk = [130, 17], [5, 300]
    q, k, v = (_values(rng, (sum(n), h, d), dtype) for n, h in ((lq, 6), (lk, 2), (lk, 2)))
    plan = cuda_ops.PackedPlan(lq, lk, heads_q=6, heads_kv=2, causal=False)
    out = cuda_ops.sdpa_packed(*(_dev(x, dtype, cuda) for x in (q, k, v)), plan, scale=0.3)
    ref, mag, _, err = srv.packed(q, k, v, lq, lk, 0.3, causal=False)
    _hold(_np(out), ref, mag, err, max(lk), dtype)


@pytest.mark.parametrize("dtype,gap", [("bf16", 0), ("bf16", 8), ("bf16", 1), ("f32", 0), ("f32", 3)])
def test_packed_strided(cuda, dtype, gap):
    """Slices of a fused projection; a gap that breaks the 16-byte alignment; out as a slice."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(4)
    lens, hq, hk, d = [150, 31, 260], 8, 2, 64
    t = sum(lens)
    wide = _values(rng, (t, (hq + 2 * hk) * d + gap), dtype)
    x = _dev(wide, dtype, cuda)
    body = x[:, gap:].unflatten(1, (hq + 2 * hk, d))
    q, k, v = body[:, :hq], body[:, hq:hq + hk], body[:, hq + hk:]
    out = torch.full((t, hq + 3, d), 7.0, dtype=x.dtype, device=cuda)
    plan = cuda_ops.PackedPlan(lens, heads_q=hq, heads_kv=hk)
    assert cuda_ops.sdpa_packed(q, k, v, plan, out=out[:, 2:2 + hq]).data_ptr() \
        == out[:, 2:].data_ptr()
    n = wide[:, gap:].reshape(t, hq + 2 * hk, d)
    ref, mag, _, err = srv.packed(n[:, :hq], n[:, hq:hq + hk], n[:, hq + hk:], lens, lens,
                                  1 / np.sqrt(d))
    _hold(_np(out[:, 2:2 + hq]), ref, mag, err, max(lens), dtype)
    assert (out[:, :2] == 7).all() and (out[:, 2 + hq:] == 7).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 32)])
@pytest.mark.parametrize("poison", [np.nan, np.inf, -3e38])
def test_packed_neighbours_do_not_reach(cuda, dtype, d, poison):
    """Whatever other sequences hold, a sequence's result is the same bits."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(5)
    lens = [100, 37, 200, 5]
    at = np.concatenate([[0], np.cumsum(lens)])
    q, k, v = (_dev(_values(rng, (sum(lens), h, d), dtype), dtype, cuda) for h in (4, 2, 2))
    plan = cuda_ops.PackedPlan(lens, heads_q=4, heads_kv=2)
    clean = cuda_ops.sdpa_packed(q, k, v, plan)
    for s in range(len(lens)):
        if s % 2 == 0:
            for x in (q, k, v):
                x[at[s]:at[s + 1]] = poison
    got = cuda_ops.sdpa_packed(q, k, v, plan)
    for s in (1, 3):
        assert torch.equal(got[at[s]:at[s + 1]], clean[at[s]:at[s + 1]])


@pytest.mark.parametrize("gain", [8.0, 60.0])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_peaked(cuda, gain, d):
    """A softmax that is nearly one key's: the running maximum moves often and far."""
    from enigma import cuda_ops
    rng = np.random.default_rng(6)
    lens = [400, 129]
    q, k, v = (_values(rng, (sum(lens), h, d), "bf16") for h in (4, 2, 2))
    q = orc.bf16_round(q * np.float32(gain))
    plan = cuda_ops.PackedPlan(lens, heads_q=4, heads_kv=2)
    out = cuda_ops.sdpa_packed(*(_dev(x, "bf16", cuda) for x in (q, k, v)), plan)
    ref, mag, _, err = srv.packed(q, k, v, lens, lens, 1 / np.sqrt(d))
    _hold(_np(out), ref, mag, err, max(lens), "bf16")


def test_packed_same_bits_twice(cuda):
    import torch
    from enigma import cuda_ops
    g = torch.Generator(device=cuda).manual_seed(1)
    lens = [700, 31, 1200, 5, 400]
    q, k, v = (torch.randn(sum(lens), h, 128, device=cuda, generator=g).bfloat16()
               for h in (16, 4, 4))
    plan = cuda_ops.PackedPlan(lens, heads_q=16, heads_kv=4)
    first = cuda_ops.sdpa_packed(q, k, v, plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [cuda_ops.sdpa_packed(q, k, v, plan) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_packed_long(cuda):
    """A long prompt against fp32 torch attention on the same inputs (rows sampled)."""
    import torch
    from enigma import cuda_ops
    g = torch.Generator(device=cuda).manual_seed(2)
    n, hq, hk, d = 9001, 8, 2, 128
    q, k, v = (torch.randn(n, h, d, device=cuda, generator=g).bfloat16() for h in (hq, hk, hk))
    plan = cuda_ops.PackedPlan([n], heads_q=hq, heads_kv=hk)
    out = cuda_ops.sdpa_packed(q, k, v, plan)
    for i in (0, 1, 4095, 4096, 8999, 9000):
        for h in (0, hq - 1):
            kd, vd = (x[:i + 1, h // 4].double() for x in (k, v))
            w = torch.softmax(kd @ q[i, h].double() / d ** 0.5, 0)
            ref, mag = w @ vd, w @ vd.abs()
            tol = srv.UBF * 1.01 * (mag + ref.abs()) + 1e-4 * mag
            assert ((out[i, h].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("f32", 8)])
def test_packed_many_sequences(cuda, dtype, d):
    """More items than a grid's second axis holds; each of one token, whose result is its value."""
    import torch
    from enigma import cuda_ops
    n = 9000
    g = torch.Generator(device=cuda).manual_seed(3)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    q, k, v = (torch.randn(n, h, d, device=cuda, generator=g).to(dt) for h in (16, 8, 8))
    plan = cuda_ops.PackedPlan([1] * n, heads_q=16, heads_kv=8)
    out = cuda_ops.sdpa_packed(q, k, v, plan)
    assert torch.equal(out, v.repeat_interleave(2, 1))


def test_packed_empty(cuda):
    import torch
    from enigma import cuda_ops
    plan = cuda_ops.PackedPlan([], heads_q=4, heads_kv=2)
    e = torch.empty(0, 4, 64, device=cuda)
    assert cuda_ops.sdpa_packed(e, e[:, :2], e[:, :2], plan).shape == (0, 4, 64)


def test_packed_refusals(cuda):
    import torch
    from enigma import _native, cuda_ops
    plan = cuda_ops.PackedPlan([4, 3], heads_q=4, heads_kv=2)
    q, k = torch.zeros(7, 4, 64, device=cuda), torch.zeros(7, 2, 64, device=cuda)
    with pytest.raises(ValueError, match="plan's lengths"):
        cuda_ops.sdpa_packed(q[:6], k, k, plan)
    with pytest.raises(ValueError, match="other heads"):
        cuda_ops.sdpa_packed(q, q, q, plan)
    with pytest.raises(ValueError, match="last axis"):
        cuda_ops.sdpa_packed(q, k, torch.zeros(7, 2, 128, device=cuda)[..., ::2], plan)
    with pytest.raises(TypeError, match="share a dtype"):
        cuda_ops.sdpa_packed(q, k.bfloat16(), k, plan)
    with pytest.raises(TypeError, match="unsupported dtype"):
        cuda_ops.sdpa_packed(q.half(), k.half(), k.half(), plan)
    with pytest.raises(ValueError, match="no CPU fallback"):
        cuda_ops.sdpa_packed(q.cpu(), k.cpu(), k.cpu(), plan)
    with pytest.raises(ValueError, match="shapes"):
        cuda_ops.sdpa_packed(q, k, k[:6], plan)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(_native.EnigmaCudaError, match="scale"):
            cuda_ops.sdpa_packed(q, k, k, plan, scale=scale)
    wide = torch.zeros(7, 2, 257, device=cuda)
    with pytest.raises(_native.EnigmaCudaError, match="head_dim"):
        cuda_ops.sdpa_packed(torch.zeros(7, 4, 257, device=cuda), wide, wide, plan)


# ------------------------------------------------------------------ paged, shared prefix
def _paged_case(rng, batch, prefix, own, page, hk, d, dtype, spare=2):
    """Pages in a shuffled order; what no sequence uses holds NaN."""
    lens = [prefix + n for n in own]
    head = prefix // page
    width = max(1, -(-max(lens + [1]) // page))
    tails = [max(0, -(-n // page) - head) for n in lens]
    total = head + sum(tails) + spare
    order = rng.permutation(total)
    table = np.full((batch, width), -1, np.int32)
    table[:, :head] = order[:head]
    at = head
    for b, m in enumerate(tails):
        table[b, head:head + m] = order[at:at + m]
        at += m
    shape = (total, hk, page, d)
    k, v = (np.full(shape, np.nan, np.float32) for _ in range(2))
    for p in order[:head]:
        k[p], v[p] = _values(rng, shape[1:], dtype), _values(rng, shape[1:], dtype)
    part_k, part_v = _values(rng, shape[1:], dtype), _values(rng, shape[1:], dtype)
    for b, n in enumerate(lens):
        for c in range(head, -(-n // page)):
            p, rows = table[b, c], min(page, n - c * page)
            k[p, :, :rows] = _values(rng, (hk, rows, d), dtype)
            v[p, :, :rows] = _values(rng, (hk, rows, d), dtype)
        if prefix % page and n > prefix - prefix % page:     # the copied part of the prefix
            m = min(prefix % page, n - head * page)
            k[table[b, head], :, :m], v[table[b, head], :, :m] = part_k[:, :m], part_v[:, :m]
    return k, v, table, np.array(lens, np.int32)


@pytest.mark.parametrize("batch,prefix,own,page", [
    (1, 0, [1], 16), (3, 0, [1, 0, 40], 16), (2, 16, [1, 3], 16), (4, 37, [1, 90, 5, 33], 32),
    (5, 128, [1, 64, 65, 200, 7], 64), (3, 515, [1, 130, 12], 128), (33, 256, [3] * 33, 16),
    (4, 1000, [25, 1, 7, 300], 16), (2, 0, [700, 1300], 64), (40, 130, list(range(1, 41)), 64)])
@pytest.mark.parametrize("heads_q,heads_kv,d,dtype", [
    (14, 2, 64, "bf16"), (8, 2, 128, "bf16"), (2, 2, 128, "bf16"), (20, 1, 64, "bf16"),
    (4, 2, 96, "bf16"), (6, 2, 64, "f32")])
def test_shared_prefix(cuda, batch, prefix, own, page, heads_q, heads_kv, d, dtype):
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(batch + prefix + d)
    k, v, table, lens = _paged_case(rng, batch, prefix, own, page, heads_kv, d, dtype)
    q = _values(rng, (batch, heads_q, d), dtype)
    out = cuda_ops.sdpa_shared_prefix(
        _dev(q, dtype, cuda), _dev(k, dtype, cuda), _dev(v, dtype, cuda),
        torch.from_numpy(table).to(cuda), torch.from_numpy(lens).to(cuda), prefix_len=prefix)
    ref, mag, _, err = srv.paged(q, k, v, table, lens, prefix, 1 / np.sqrt(d))
    _hold(_np(out), ref, mag, err, int(lens.max()), dtype)
    assert (_np(out)[lens == 0] == 0).all()


@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_shared_prefix_slots_and_strides(cuda, dtype, d):
    """Rows named by slots, sequences shorter than the prefix or empty, one layer of a larger
    cache, q and out as slices of wider tensors."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(9)
    page, hk, hq, prefix = 32, 2, 8, 100
    k, v, table, lens = _paged_case(rng, 6, prefix, [1, 60, 2, 200, 9, 31], page, hk, d, dtype)
    lens[4], lens[2] = 0, 50                       # nothing; less than the prefix
    slots = np.array([3, 4, 2, 0], np.int32)
    pages = [_dev(np.stack([np.full_like(x, np.nan), x]), dtype, cuda) for x in (k, v)]
    wide = _values(rng, (4, hq + 4, d), dtype)
    got = torch.full((4, hq + 1, d), 3.0, dtype=pages[0].dtype, device=cuda)
    cuda_ops.sdpa_shared_prefix(_dev(wide, dtype, cuda)[:, 2:2 + hq], pages[0][1], pages[1][1],
                                torch.from_numpy(table).to(cuda), torch.from_numpy(lens).to(cuda),
                                prefix_len=prefix, slots=torch.from_numpy(slots).to(cuda),
                                scale=0.2, out=got[:, :hq])
    ref, mag, _, err = srv.paged(wide[:, 2:2 + hq], k, v, table, lens, prefix, 0.2, slots)
    _hold(_np(got[:, :hq]), ref, mag, err, int(lens.max()), dtype)
    assert (got[:, hq:] == 3).all() and (got[1, :hq] == 0).all()


@pytest.mark.parametrize("d,heads", [(64, (14, 2)), (128, (16, 4))])
def test_shared_prefix_large(cuda, d, heads):
    """A long prefix and a wide batch against 64-bit torch attention (sequences sampled), the
    same bits twice, and the same result as without sharing."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(12)
    hq, hk = heads
    batch, prefix, page = 70, 5000, 64
    own = [1 + (b * 37) % 500 for b in range(batch)]
    k, v, table, lens = _paged_case(rng, batch, prefix, own, page, hk, d, "bf16")
    kd, vd = _dev(k, "bf16", cuda), _dev(v, "bf16", cuda)
    td, ld = torch.from_numpy(table).to(cuda), torch.from_numpy(lens).to(cuda)
    q = _dev(_values(rng, (batch, hq, d), "bf16"), "bf16", cuda)
    out = cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=prefix)
    again = cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=prefix)
    alone = cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=0)
    assert torch.equal(out, again)
    for b in (0, 1, 33, 69):
        n, rows = int(lens[b]), td[b].long()
        used = rows[: -(-n // page)].clone()
        used[: prefix // page] = td[0, : prefix // page].long()
        for h in (0, hq - 1):
            kk = kd[used, h // (hq // hk)].reshape(-1, d)[:n].double()
            vv = vd[used, h // (hq // hk)].reshape(-1, d)[:n].double()
            w = torch.softmax(kk @ q[b, h].double() / d ** 0.5, 0)
            ref, mag = w @ vv, w @ vv.abs()
            tol = srv.UBF * 1.01 * (mag + ref.abs()) + 1e-4 * mag
            assert ((out[b, h].double() - ref).abs() <= tol).all()
            assert ((alone[b, h].double() - ref).abs() <= tol).all()


def test_shared_prefix_graph(cuda):
    """Captured once, replayed as the lengths on the device move on."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(13)
    k, v, table, lens = _paged_case(rng, 5, 70, [90, 1, 30, 64, 7], 32, 2, 64, "bf16")
    kd, vd = _dev(k, "bf16", cuda), _dev(v, "bf16", cuda)
    td, ld = torch.from_numpy(table).to(cuda), torch.from_numpy(lens).to(cuda)
    q = _values(rng, (5, 14, 64), "bf16")
    qd, out = _dev(q, "bf16", cuda), torch.empty(5, 14, 64, dtype=torch.bfloat16, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cuda_ops.sdpa_shared_prefix(qd, kd, vd, td, ld, prefix_len=70, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda_ops.sdpa_shared_prefix(qd, kd, vd, td, ld, prefix_len=70, out=out)
    for step in ([0, 0, 0, 0, 0], [-40, 0, -10, -1, -7], [-90, -1, -30, -64, -7]):
        now = lens + np.array(step, np.int32)
        ld.copy_(torch.from_numpy(now))
        graph.replay()
        ref, mag, _, err = srv.paged(q, k, v, table, now, 70, 1 / 8)
        _hold(_np(out), ref, mag, err, int(now.max()), "bf16")


def test_shared_prefix_invalid_pages_are_no_fault(cuda):
    """Lengths past the table and page numbers outside the cache read nothing outside it."""
    import torch
    from enigma import cuda_ops
    for dtype, d in ((torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)):
        k = torch.randn(4, 2, 16, d, device=cuda).to(dtype)
        table = torch.tensor([[0, -1, 9], [1, 2, 1 << 30]], dtype=torch.int32, device=cuda)
        lens = torch.tensor([1 << 30, -5], dtype=torch.int32, device=cuda)
        q = torch.randn(2, 8, d, device=cuda).to(dtype)
        for prefix in (0, 20, 48):
            out = cuda_ops.sdpa_shared_prefix(q, k, k, table, lens, prefix_len=prefix)
            assert (out[1] == 0).all() and torch.isfinite(out.float()).all()
        slots = torch.tensor([7, -1], dtype=torch.int32, device=cuda)
        out = cuda_ops.sdpa_shared_prefix(q, k, k, table, lens, prefix_len=20, slots=slots)
        assert (out == 0).all()
    torch.cuda.synchronize()


def test_shared_prefix_refusals(cuda):
    import torch
    from enigma import _native, cuda_ops
    k = torch.zeros(4, 2, 16, 64, device=cuda, dtype=torch.bfloat16)
    q = torch.zeros(2, 8, 64, device=cuda, dtype=torch.bfloat16)
    table = torch.zeros(2, 3, dtype=torch.int32, device=cuda)
    lens = torch.zeros(2, dtype=torch.int32, device=cuda)
    run = cuda_ops.sdpa_shared_prefix
    with pytest.raises(ValueError, match="int32"):
        run(q, k, k, table.long(), lens)
    with pytest.raises(ValueError, match="lens"):
        run(q, k, k, table, lens[:1])
    with pytest.raises(ValueError, match="a page must be contiguous"):
        run(q, k.transpose(1, 2).contiguous().transpose(1, 2), k, table, lens)
    with pytest.raises(TypeError, match="share a dtype"):
        run(q, k.float(), k.float(), table, lens)
    with pytest.raises(_native.EnigmaCudaError, match="prefix_len"):
        run(q, k, k, table, lens, prefix_len=49)
    with pytest.raises(_native.EnigmaCudaError, match="page must be"):
        run(q, k[:, :, :8].contiguous(), k[:, :, :8].contiguous(), table, lens)
    with pytest.raises(_native.EnigmaCudaError, match="multiple"):
        run(q[:, :3], k, k, table, lens)
    with pytest.raises(_native.EnigmaCudaError, match="more sequences"):
        run(q.repeat(2, 1, 1), k, k, table, lens)
    with pytest.raises(ValueError, match="slots"):
        run(q, k, k, table, lens, slots=lens[:1])


def test_shared_prefix_side_by_side_in_a_graph_and_on_streams(cuda):
    """Large enough for the prefix and the own keys to run on two streams: captured, replayed with
    other lengths, and called on several streams at once."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(21)
    k, v, table, lens = _paged_case(rng, 40, 3000, [1 + 11 * b for b in range(40)], 64, 4, 128, "bf16")
    kd, vd = _dev(k, "bf16", cuda), _dev(v, "bf16", cuda)
    td, ld = torch.from_numpy(table).to(cuda), torch.from_numpy(lens).to(cuda)
    q = _dev(_values(rng, (40, 16, 128), "bf16"), "bf16", cuda)
    want = cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=3000)
    short = cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld - 20, prefix_len=3000)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=3000, out=out)
    graph.replay()
    assert torch.equal(out, want)
    ld -= 20
    graph.replay()
    assert torch.equal(out, short)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams * 2:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=3000))
    torch.cuda.synchronize()
    assert all(torch.equal(g, short) for g in got)


def test_shared_prefix_side_by_side_while_another_stream_captures(cuda):
    """Two streams per call: a call that is not captured, made between two that are, stays out of the
    graph, and the graph is whole."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(22)
    k, v, table, lens = _paged_case(rng, 40, 3000, [1 + 11 * b for b in range(40)], 64, 4, 128, "bf16")
    kd, vd = _dev(k, "bf16", cuda), _dev(v, "bf16", cuda)
    td, ld = torch.from_numpy(table).to(cuda), torch.from_numpy(lens).to(cuda)
    q = _dev(_values(rng, (40, 16, 128), "bf16"), "bf16", cuda)
    want = cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=3000)
    workspaces = [torch.empty(64 << 20, dtype=torch.uint8, device=cuda) for _ in range(2)]
    outs = [torch.zeros_like(want) for _ in range(3)]
    other = torch.cuda.Stream()
    torch.cuda.synchronize()

    def call(out, workspace):
        cuda_ops.sdpa_shared_prefix(q, kd, vd, td, ld, prefix_len=3000, out=out, workspace=workspace)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="relaxed"):
        call(outs[0], workspaces[0])
        with torch.cuda.stream(other):
            call(outs[1], workspaces[1])
        call(outs[2], workspaces[0])
    torch.cuda.synchronize()
    assert torch.equal(outs[1], want) and not outs[0].any() and not outs[2].any()
    outs[1].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[2], want) and not outs[1].any()


@pytest.mark.parametrize("batch,prefix,own,page,heads,d", [
    (1, 0, [22251], 16, (15, 3), 64),
    (3, 0, [0, 1, 30000], 16, (8, 1), 128),
    (2, 20000, [5, 300], 64, (8, 1), 128),
    (4, 9000, [0, 1, 2, 130], 64, (16, 2), 64),
    (2, 0, [9001, 64], 32, (40, 2), 128),
])
def test_shared_prefix_few_rows_of_many_parts(cuda, batch, prefix, own, page, heads, d):
    """Few sequences with long caches: every SM has a part of each row."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(23)
    hq, hk = heads
    k, v, table, lens = _paged_case(rng, batch, prefix, own, page, hk, d, "bf16")
    q = _values(rng, (batch, hq, d), "bf16")
    td, ld = torch.from_numpy(table).to(cuda), torch.from_numpy(lens).to(cuda)
    args = (_dev(q, "bf16", cuda), _dev(k, "bf16", cuda), _dev(v, "bf16", cuda), td, ld)
    out = cuda_ops.sdpa_shared_prefix(*args, prefix_len=prefix)
    assert torch.equal(out, cuda_ops.sdpa_shared_prefix(*args, prefix_len=prefix))
    ref, mag, _, err = srv.paged(q, k, v, table, lens, prefix, d ** -0.5)
    _hold(_np(out), ref, mag, err, int(lens.max()), "bf16")


@pytest.mark.parametrize("lq,lk", [
    ([30], [2000]), ([1, 1, 1], [500, 3000, 20]), ([5, 0, 9], [1025, 700, 3]), ([40], [4000]),
    ([64, 3], [257, 1])])
@pytest.mark.parametrize("heads,d,dtype", [
    ((8, 2), 64, "f32"), ((4, 4), 128, "f32"), ((3, 1), 200, "f32"), ((8, 2), 80, "bf16"),
    ((2, 1), 33, "f32")])
def test_packed_few_rows_of_many_keys(cuda, lq, lk, heads, d, dtype):
    """Too few rows to fill the SMs: their keys are split inside one launch."""
    import torch
    from enigma import cuda_ops
    hq, hk = heads
    rng = np.random.default_rng(sum(lk) + d)
    q = _values(rng, (sum(lq), hq, d), dtype)
    k = _values(rng, (sum(lk), hk, d), dtype)
    v = _values(rng, (sum(lk), hk, d), dtype)
    plan = cuda_ops.PackedPlan(lq, lk, heads_q=hq, heads_kv=hk)
    args = (_dev(q, dtype, cuda), _dev(k, dtype, cuda), _dev(v, dtype, cuda), plan)
    out, lse = cuda_ops.sdpa_packed(*args, return_lse=True)
    again, _ = cuda_ops.sdpa_packed(*args, return_lse=True)
    assert torch.equal(out, again)
    ref, mag, rlse, err = srv.packed(q, k, v, lq, lk, d ** -0.5)
    _hold(_np(out), ref, mag, err, max(lk), dtype)
    got, empty = _np(lse), np.isinf(rlse)
    assert (got[empty] == -np.inf).all() and (_np(out)[empty] == 0).all()
    tol = 4 * (err + (max(lk) + 16) * srv.U32) + 8 * srv.U32 * np.abs(np.where(empty, 0, rlse))
    assert (np.abs(got[~empty] - rlse[~empty]) <= tol[~empty]).all()
