"""GPU parity of rotary positions against the 64-bit oracle: layouts, parts of a head, scaled
frequencies, far and negative positions, strides, in place, back again, and as a gradient.

The bound: an angle in [-pi, pi] is rounded once (pi 2^-24), sin and cos are off by two units in the
last place at most (2^-22) and multiplied by the factor (2^-24); two products and a sum (3 2^-24): less
than 12 2^-24 (|a| + |b|).  The oracle's own 64-bit product of a far position, and the frequency in
turns, are off by 2^-51 of the angle.  bf16 results are rounded once more."""
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


def _hold(got, x, positions, table, dtype, inverse=False):
    ref, mag = srv.rope(x, positions, table.frequencies, table.factor, table.layout, inverse)
    far = np.abs(np.asarray(positions, np.float64)) * max([abs(w) for w in table.frequencies] + [0])
    tol = mag * (12 * srv.U32 + far[:, None, None] * 2.0 ** -51)
    if dtype == "bf16":
        tol = tol + np.where(mag > 0, srv.UBF * (np.abs(ref) + tol), 0)
    off = np.abs(got - ref)
    assert np.isfinite(got).all() and (off <= tol).all(), (off - tol).max()


SCALINGS = [None, dict(type="linear", factor=8.0), dict(type="ntk", factor=4.0),
            dict(type="yarn", factor=16.0, original_len=4096),
            dict(type="bands", factor=8.0, original_len=8192, low=1.0, high=4.0)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens,heads_q,heads_k,d,rotary", [
    (1, 14, 2, 64, 64), (130, 14, 2, 64, 64), (67, 32, 8, 128, 128), (40, 32, 8, 128, 64),
    (33, 5, 5, 128, 32), (9, 8, 1, 256, 256), (21, 4, 2, 80, 80), (21, 4, 2, 80, 40),
    (5, 3, 1, 96, 48), (3, 1, 1, 2, 2), (17, 3, 2, 10, 6), (6, 2, 2, 16, 0), (700, 3, 1, 7, 4),
    (2500, 9, 3, 64, 16)])
def test_rope(cuda, layout, dtype, tokens, heads_q, heads_k, d, rotary):
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(tokens + d)
    q, k = _values(rng, (tokens, heads_q, d), dtype), _values(rng, (tokens, heads_k, d), dtype)
    at = rng.integers(0, 40000, tokens)
    for i, scaling in enumerate(SCALINGS if rotary == 64 else [SCALINGS[tokens % 5]]):
        table = cuda_ops.RopeTable(d, rotary_dim=rotary, theta=(1e6, 1e4)[i % 2], layout=layout,
                                   scaling=scaling)
        positions = torch.from_numpy(at).to(cuda, torch.int32 if i % 2 == 0 else torch.int64)
        got_q, got_k = cuda_ops.rope(_dev(q, dtype, cuda), _dev(k, dtype, cuda), positions, table)
        _hold(_np(got_q), q, at, table, dtype)
        _hold(_np(got_k), k, at, table, dtype)
        assert (_np(got_q)[..., rotary:] == q[..., rotary:]).all()


@pytest.mark.parametrize("wide", [False, True])
def test_far_and_negative_positions(cuda, wide):
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(1)
    at = np.array([0, 1, -1, 131071, 1048575, -70000, 2 ** 31 - 1, -2 ** 31]
                  + ([2 ** 33 + 5, -2 ** 35 - 1] if wide else []), np.int64)
    q = _values(rng, (len(at), 4, 64), "f32")
    table = cuda_ops.RopeTable(64, theta=1e4)
    positions = torch.from_numpy(at).to(cuda, torch.int64 if wide else torch.int32)
    got = cuda_ops.rope(_dev(q, "f32", cuda), None, positions, table)
    assert (_np(got)[0] == q[0]).all()                    # position 0 changes nothing
    _hold(_np(got), q, at, table, "f32")


@pytest.mark.parametrize("dtype,gap", [("bf16", 0), ("bf16", 8), ("bf16", 1), ("bf16", 4), ("f32", 0),
                                       ("f32", 2), ("f32", 1)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rotary", [64, 32, 36])
def test_strided_and_in_place(cuda, dtype, gap, layout, rotary):
    """Slices of a fused projection, whatever their alignment, into other slices and onto themselves;
    what lies between stays."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(gap + rotary)
    t, hq, hk, d = 45, 6, 2, 64
    wide = _values(rng, (t, (hq + 2 * hk) * d + gap), dtype)
    x = _dev(wide, dtype, cuda)
    body = lambda y: y[:, gap:].unflatten(1, (hq + 2 * hk, d))  # noqa: E731
    at = rng.integers(0, 5000, t)
    positions = torch.from_numpy(at).to(cuda, torch.int32)
    table = cuda_ops.RopeTable(d, rotary_dim=rotary, layout=layout)
    out = torch.full_like(x, 7.0)
    q, k = body(x)[:, :hq], body(x)[:, hq:hq + hk]
    res = cuda_ops.rope(q, k, positions, table, out_q=body(out)[:, :hq], out_k=body(out)[:, hq:hq + hk])
    n = wide[:, gap:].reshape(t, hq + 2 * hk, d)
    _hold(_np(res[0]), n[:, :hq], at, table, dtype)
    _hold(_np(body(out)[:, hq:hq + hk]), n[:, hq:hq + hk], at, table, dtype)
    assert (out[:, :gap] == 7).all() and (body(out)[:, hq + hk:] == 7).all()
    cuda_ops.rope(q, k, positions, table, out_q=q, out_k=k)
    assert (body(x)[:, :hq + hk] == body(out)[:, :hq + hk]).all()
    assert (_np(body(x)[:, hq + hk:]) == n[:, hq + hk:]).all() and (_np(x[:, :gap]) == wide[:, :gap]).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_heads_in_front(cuda, layout):
    """[heads, tokens, head_dim] storage, read and written through a transposed view."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(3)
    q = _values(rng, (6, 50, 128), "bf16")
    at = np.arange(50) + 1000
    table = cuda_ops.RopeTable(128, layout=layout)
    x = _dev(q, "bf16", cuda)
    cuda_ops.rope(x.transpose(0, 1), None, torch.from_numpy(at).to(cuda), table, out_q=x.transpose(0, 1))
    _hold(_np(x.transpose(0, 1)), q.transpose(1, 0, 2), at, table, "bf16")


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rotary", [(64, 64), (96, 32)])
def test_inverse_is_the_gradient(cuda, layout, d, rotary):
    """inverse=True turns back (factor 1), and takes a result's gradient to its input's: against the
    formula differentiated by torch in 64 bits, and against differences."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(5)
    t, hq, hk = 19, 4, 2
    at = rng.integers(0, 100000, t)
    positions = torch.from_numpy(at).to(cuda)
    table = cuda_ops.RopeTable(d, rotary_dim=rotary, layout=layout)
    q, k = (_values(rng, (t, h, d), "f32") for h in (hq, hk))
    y = cuda_ops.rope(_dev(q, "f32", cuda), _dev(k, "f32", cuda), positions, table)
    back = cuda_ops.rope(*y, positions, table, inverse=True)
    for a, b in zip(back, (q, k)):
        mag = srv.rope(b, at, table.frequencies, 1.0, layout)[1]
        twice = srv.rope(mag, at, table.frequencies, 1.0, layout)[1] + np.abs(b)
        assert (np.abs(_np(a) - b) <= 24 * srv.U32 * twice).all()
    table = cuda_ops.RopeTable(d, rotary_dim=rotary, layout=layout,
                               scaling=dict(type="yarn", factor=4.0, original_len=1024))
    gq, gk = (_values(rng, (t, h, d), "f32") for h in (hq, hk))
    got = cuda_ops.rope(_dev(gq, "f32", cuda), _dev(gk, "f32", cuda), positions, table, inverse=True)
    w = torch.tensor(table.frequencies, dtype=torch.float64)
    angle = torch.from_numpy(at).double()[:, None] * w
    c, s = (table.factor * f(angle)[:, None] for f in (torch.cos, torch.sin))
    n = rotary
    for x, g, grad in ((q, gq, got[0]), (k, gk, got[1])):
        x = torch.from_numpy(x).double().requires_grad_()
        a, b = (x[..., :n // 2], x[..., n // 2:n]) if layout == "half" else (x[..., 0:n:2], x[..., 1:n:2])
        u, v = a * c - b * s, b * c + a * s
        g = torch.from_numpy(g).double()
        gu, gv = (g[..., :n // 2], g[..., n // 2:n]) if layout == "half" else (g[..., 0:n:2], g[..., 1:n:2])
        loss = (u * gu).sum() + (v * gv).sum() + (x[..., n:] * g[..., n:]).sum()
        loss.backward()
        mag = srv.rope(g.numpy(), at, table.frequencies, table.factor, layout, True)[1]
        far = (at.max() * 2.0 ** -51)
        assert (np.abs(_np(grad) - x.grad.numpy()) <= mag * (12 * srv.U32 + far)).all()
    # Differences: the map is linear, so a step of any size gives <gradient, step>.
    step = _values(rng, q.shape, "f32")
    lo, hi = (cuda_ops.rope(_dev(q + e * step, "f32", cuda), None, positions, table) for e in (0, 1))
    lhs = ((_np(hi) - _np(lo)) * gq).sum()
    moved = (q + step).astype(np.float32).astype(np.float64) - q
    rhs = (_np(got[0]) * moved).sum()
    size = np.abs(gq).sum() * (np.abs(q) + np.abs(step)).max() * 4 * table.factor
    assert abs(lhs - rhs) <= 40 * srv.U32 * size


def test_nothing_to_do(cuda):
    import torch
    from enigma import cuda_ops
    table = cuda_ops.RopeTable(64)
    q, k = (torch.empty(0, h, 64, device=cuda) for h in (4, 2))
    a, b = cuda_ops.rope(q, k, torch.empty(0, dtype=torch.int32, device=cuda), table)
    assert a.shape == q.shape and b.shape == k.shape


def test_what_does_not_turn_is_copied(cuda):
    """Bits of elements behind the part that turns, NaN and infinities among them."""
    import torch
    from enigma import cuda_ops
    x = torch.randint(-2 ** 15, 2 ** 15, (30, 3, 128), dtype=torch.int16, device=cuda).view(torch.bfloat16)
    table = cuda_ops.RopeTable(128, rotary_dim=32)
    y = cuda_ops.rope(x, None, torch.arange(30, device=cuda), table)
    assert (y[..., 32:].view(torch.int16) == x[..., 32:].view(torch.int16)).all()


def test_streams_and_graphs(cuda):
    """Another stream than the tensors'; a captured call that reads new positions at replay."""
    import torch
    from enigma import cuda_ops
    rng = np.random.default_rng(8)
    q, k = _values(rng, (64, 14, 64), "bf16"), _values(rng, (64, 2, 64), "bf16")
    x, y = _dev(q, "bf16", cuda), _dev(k, "bf16", cuda)
    at = torch.arange(64, dtype=torch.int32, device=cuda)
    table = cuda_ops.RopeTable(64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, b = cuda_ops.rope(x, y, at, table)
    torch.cuda.current_stream().wait_stream(side)
    _hold(_np(a), q, np.arange(64), table, "bf16")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = cuda_ops.rope(x, y, at, table)
    for shift in (0, 1000):
        at.copy_(torch.arange(64, device=cuda) + shift)
        graph.replay()
        _hold(_np(b), k, np.arange(64) + shift, table, "bf16")
