"""Host side of rotary positions and of the cache in 8-bit codes: frequencies and their binary
fractions, what calls refuse (in Python and at the C entries, before any launch), and which device
they run on."""
import ctypes
import math

import numpy as np
import pytest
import torch

from test_current_device import OnOne, _check, _on_one, calls  # noqa: F401


# ---------------------------------------------------------------------------- frequencies
def test_frequencies():
    from enigma.cuda_ops import rope_frequencies
    w, f = rope_frequencies(64, 1e6)
    np.testing.assert_allclose(w, 1e6 ** (-np.arange(32) / 32.0), rtol=1e-14)
    assert f == 1.0 and rope_frequencies(0)[0] == []
    np.testing.assert_allclose(rope_frequencies(64, 1e6, {"type": "linear", "factor": 4})[0],
                               np.array(w) / 4, rtol=1e-14)
    # ntk: the fastest pair stays, the slowest is stretched by the factor.
    n, _ = rope_frequencies(64, 1e4, {"type": "ntk", "factor": 8})
    base = rope_frequencies(64, 1e4)[0]
    assert n[0] == 1.0
    np.testing.assert_allclose(n[-1], base[-1] / 8, rtol=1e-12)


def test_yarn_and_bands_frequencies():
    from enigma.cuda_ops import rope_frequencies
    base = np.array(rope_frequencies(128, 1e4)[0])
    length, s = 4096, 16.0
    w, f = rope_frequencies(128, 1e4, dict(type="yarn", factor=s, original_len=length))
    turns = length * base / (2 * math.pi)
    w = np.array(w)
    assert f == pytest.approx(0.1 * math.log(s) + 1)
    assert (w[turns > 33 * 1.2] == base[turns > 33 * 1.2]).all()       # ends are rounded outwards
    np.testing.assert_allclose(w[turns < 0.85], base[turns < 0.85] / s, rtol=1e-14)
    assert (np.diff(w / base) <= 1e-15).all()
    assert rope_frequencies(128, 1e4, dict(type="yarn", factor=s, original_len=length,
                                           attention_factor=1.5))[1] == 1.5
    w = np.array(rope_frequencies(128, 1e4, dict(type="bands", factor=s, original_len=length, low=1,
                                                 high=4))[0])
    assert (w[turns >= 4] == base[turns >= 4]).all()
    np.testing.assert_allclose(w[turns <= 1], base[turns <= 1] / s, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    r = (turns[mid] - 1) / 3
    np.testing.assert_allclose(w[mid], base[mid] * r + base[mid] / s * (1 - r), rtol=1e-12)


@pytest.mark.parametrize("scaling", [
    {"type": "other"}, {"type": "linear", "factor": 0}, {"type": "linear", "factor": math.nan},
    {"type": "yarn", "factor": 2}, {"type": "yarn", "factor": 2, "original_len": -1},
    {"type": "bands", "factor": 2, "original_len": 10, "low": 4, "high": 4},
    {"type": "linear", "factor": 2, "original_len": 3}, {"factor": 2}])
def test_scalings_refused(scaling):
    from enigma.cuda_ops import rope_frequencies
    with pytest.raises(ValueError):
        rope_frequencies(64, 1e4, scaling)


def test_table():
    """turns[i] is the frequency in full turns, to 53 bits, as a 64-bit fraction."""
    from fractions import Fraction
    from enigma.cuda_ops import RopeTable
    t = RopeTable(80, rotary_dim=40, theta=1e4, device="cpu")
    assert t.turns.shape == (20,) and t.turns.dtype == torch.int64
    for w, turns in zip(t.frequencies, t.turns.tolist()):
        want = Fraction(w) / Fraction(2 * math.pi) * 2 ** 64
        assert abs(int(turns) % 2 ** 64 - want) <= want * 2.0 ** -52 + 1
    # A quarter turn over whole ones (three of them take two of the 53 bits), one back, none.
    got = RopeTable(8, frequencies=[2 * math.pi * 3.25, -math.pi / 2, 0, 1], device="cpu").turns
    assert abs(got[0].item() - (1 << 62)) <= 3.25 * 2 ** 12
    assert got.tolist()[1:3] == [-(1 << 62), 0]
    for bad in (dict(head_dim=0), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=3),
                dict(head_dim=64, layout="other"), dict(head_dim=64, theta=1.0),
                dict(head_dim=64, frequencies=[1.0]), dict(head_dim=4, frequencies=[1, math.inf]),
                dict(head_dim=4, frequencies=[1, 1], scaling={"type": "linear", "factor": 2}),
                dict(head_dim=8192)):
        with pytest.raises(ValueError):
            RopeTable(device="cpu", **bad)


# ------------------------------------------------------------------------- calls, devices
def _table(**kw):
    from enigma.cuda_ops import RopeTable
    t = RopeTable(64, device="cpu", **kw)
    t.turns = t.turns.as_subclass(OnOne)
    return t


def _ints(*shape, dtype=torch.int32):
    return _on_one(*shape, dtype=dtype)


def _cache(code=torch.int8, d=64, page=16, pages=4, slots=2, width=3):
    from enigma.kv_cache import QuantizedKVCache
    codes = [_on_one(1, pages, 2, page, d, dtype=torch.int8).view(code).as_subclass(OnOne)
             for _ in range(2)]
    scales = [_on_one(1, pages, 2, page // 16, dtype=torch.float32) for _ in range(2)]
    return QuantizedKVCache(*codes, *scales, _ints(slots, width), _ints(slots), _ints(pages))


def test_calls_run_on_their_tensors_device(calls):  # noqa: F811
    from enigma import cuda_ops
    q, k, at = _on_one(5, 4, 64), _on_one(5, 2, 64), _ints(5)
    for _ in range(2):
        cuda_ops.rope(q, k, at, _table())
        assert all(device == 1 for name, device in calls.calls if name != "enigma_init")
    assert calls.device == 0
    cache = _cache()
    calls.calls.clear()
    one = _ints(1)
    cuda_ops._quantized_head.cache_clear()
    cache.reserve(one, one)
    cache.write(0, _on_one(1, 2, 64), _on_one(1, 2, 64), one, one, _ints(2))
    cache.read(0, one, one, _ints(2), out_k=_on_one(1, 2, 64), out_v=_on_one(1, 2, 64))
    cache.fork(one, one)
    cache.free(one)
    cache.compact()
    cache.copy_pages(one, one)
    cache.attend(0, _on_one(2, 4, 64))
    _check(calls, "enigma_kv_cache_reserve", *("enigma_kv_cache_q8_" + x for x in (
        "write", "read", "fork")), "enigma_kv_cache_free", "enigma_kv_cache_q8_compact",
        "enigma_kv_cache_q8_copy_pages", "enigma_sdpa_quantized_workspace_bytes",
        "enigma_sdpa_quantized")
    cuda_ops._quantized_head.cache_clear()


def test_rope_refuses(calls):  # noqa: F811
    from enigma import cuda_ops
    q, k, at, t = _on_one(5, 4, 64), _on_one(5, 2, 64), _ints(5), _table()
    wide = _on_one(5, 4, 128)
    for error, call in (
            (ValueError, lambda: cuda_ops.rope(q[..., :32], k, at, t)),
            (ValueError, lambda: cuda_ops.rope(q, k[:4], at, t)),
            (ValueError, lambda: cuda_ops.rope(q[0], k, at, t)),
            (ValueError, lambda: cuda_ops.rope(q, k, at[:4], t)),
            (ValueError, lambda: cuda_ops.rope(q, k, _ints(10)[::2], t)),
            (TypeError, lambda: cuda_ops.rope(q, k, at.float(), t)),
            (TypeError, lambda: cuda_ops.rope(q, k.float(), at, t)),
            (TypeError, lambda: cuda_ops.rope(q.half(), k.half(), at, t)),
            (ValueError, lambda: cuda_ops.rope(wide[..., ::2], k, at, t)),
            (ValueError, lambda: cuda_ops.rope(q, k, at, t, out_q=k)),
            (ValueError, lambda: cuda_ops.rope(q, None, at, t, out_k=k)),
            (ValueError, lambda: cuda_ops.rope(q, k, at, t, out_q=q[:1].expand(5, 4, 64))),
            (ValueError, lambda: cuda_ops.rope(q, k, at, t, out_q=_on_one(900).as_strided(
                (5, 4, 64), (100, 64, 1)))),
            (ValueError, lambda: cuda_ops.rope(torch.zeros(5, 4, 64).bfloat16(), k, at, t)),
            (ValueError, lambda: cuda_ops.rope(q, torch.zeros(5, 2, 64).bfloat16(), at, t))):
        with pytest.raises(error):
            call()
    assert not any(name == "enigma_rope" for name, _ in calls.calls)
    cuda_ops.rope(q, None, at.long(), t, out_q=q)          # in place, wide positions, queries alone
    cuda_ops.rope(wide[..., :64], k, at, t, inverse=True)
    assert sum(name == "enigma_rope" for name, _ in calls.calls) == 2


def test_cache_refuses(calls):  # noqa: F811
    from enigma.kv_cache import QuantizedKVCache
    for kw in (dict(d=72), dict(d=272), dict(page=48), dict(page=256)):
        with pytest.raises(ValueError):
            _cache(**kw)
    ok = _cache(torch.float8_e4m3fn)
    parts = (ok.k, ok.v, ok.k_scale, ok.v_scale, ok.table, ok.lens, ok.refs)
    for i, x in ((0, ok.k.float()), (1, _cache().v), (2, ok.k_scale[..., :0]), (3, ok.k_scale.double()),
                 (4, ok.table.long()), (5, ok.lens[:1]), (6, ok.refs[:1])):
        with pytest.raises((ValueError, TypeError)):
            QuantizedKVCache(*parts[:i], x, *parts[i + 1:])
    moved = _on_one(1 * 4 * 2 * 16 * 64 + 16, dtype=torch.int8)
    with pytest.raises(ValueError, match="aligned"):
        k = moved[1:1 + 8192].view(1, 4, 2, 16, 64).as_subclass(OnOne)
        QuantizedKVCache(k, _cache().v, *parts[2:])
    cache, rows, one = _cache(), _on_one(3, 2, 64), _ints(1)
    for error, call in (
            (ValueError, lambda: cache.write(1, rows, rows, [0], [0], [0, 3])),
            (ValueError, lambda: cache.write(0, rows[:, :1], rows[:, :1], [0], [0], [0, 3])),
            (ValueError, lambda: cache.write(0, rows, rows[:2], one, one, _ints(2))),
            (TypeError, lambda: cache.write(0, rows, rows.float(), one, one, _ints(2))),
            (TypeError, lambda: cache.write(0, rows.half(), rows.half(), one, one, _ints(2))),
            (ValueError, lambda: cache.write(0, rows, rows, one, one, _ints(3))),
            (ValueError, lambda: cache.write(0, rows, rows, one, _ints(2), _ints(2))),
            (ValueError, lambda: cache.read(0, one, one, _ints(2))),               # how many rows?
            (ValueError, lambda: cache.read(0, one, one, _ints(2), out_k=rows)),
            (ValueError, lambda: cache.read(0, one, one, _ints(2), tokens=2, out_k=rows, out_v=rows)),
            (ValueError, lambda: cache.read(0, one, one, _ints(2), dtype=torch.float32, out_k=rows,
                                            out_v=rows)),
            (ValueError, lambda: cache.read(0, one, one, _ints(2), out_k=rows[:1].expand(3, 2, 64),
                                            out_v=rows)),
            (ValueError, lambda: cache.attend(0, _on_one(3, 4, 64))),              # more than rows
            (ValueError, lambda: cache.attend(0, _on_one(2, 4, 32))),
            (ValueError, lambda: cache.attend(1, _on_one(2, 4, 64))),
            (ValueError, lambda: cache.attend(-1, _on_one(2, 4, 64))),
            (ValueError, lambda: cache.attend(0, _on_one(2, 3, 64))),
            (TypeError, lambda: cache.attend(0, _on_one(2, 4, 64, dtype=torch.float16))),
            (ValueError, lambda: cache.attend(0, _on_one(2, 4, 64), out=_on_one(2, 4, 32))),
            (ValueError, lambda: cache.attend(0, _on_one(2, 4, 64), out=_on_one(1, 4, 64).expand(
                2, 4, 64))),
            (ValueError, lambda: cache.attend(0, _on_one(2, 4, 64), slots=_ints(3)))):
        calls.calls.clear()
        with pytest.raises((error, RuntimeError)):
            call()
        assert not {"enigma_kv_cache_q8_write", "enigma_kv_cache_q8_read"} & {n for n, _ in calls.calls}


# ------------------------------------------------------------------------------ C entries
class _Rope(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in (
        "tokens", "heads_q", "heads_k", "head_dim", "rotary_dim", "q_token", "q_head", "k_token",
        "k_head", "oq_token", "oq_head", "ok_token", "ok_head")] + [("factor", ctypes.c_float)] + \
        [(n, ctypes.c_int32) for n in ("dtype", "layout", "inverse", "position_bytes", "reserved")] + \
        [(n, ctypes.c_void_p) for n in ("positions", "turns", "q", "k", "out_q", "out_k")]


def test_c_rope_refuses():
    from enigma import _native
    good = dict(tokens=0, heads_q=2, heads_k=1, head_dim=64, rotary_dim=64, q_token=128, q_head=64,
                k_token=64, k_head=64, oq_token=128, oq_head=64, ok_token=64, ok_head=64, factor=1.0,
                dtype=1, layout=0, position_bytes=4, positions=64, turns=64, q=64, k=64, out_q=64,
                out_k=64)
    lib = _native.lib()
    assert lib.enigma_rope(ctypes.byref(_Rope(**good)), None) == 0        # no tokens: no launch
    assert lib.enigma_rope(None, None) == _native.ERR_BADARG
    for key, values in dict(tokens=[-1, 1 << 31], heads_q=[0, 65536], heads_k=[-1], head_dim=[0, 5000],
                            rotary_dim=[-2, 66, 3], dtype=[2], layout=[2], position_bytes=[2],
                            q_token=[-1], ok_head=[-1], positions=[0, 2], turns=[0, 4], q=[0, 1],
                            k=[0], out_q=[0, 65], out_k=[0]).items():
        for x in values:
            d = _Rope(**{**good, "tokens": 1, key: x})
            assert lib.enigma_rope(ctypes.byref(d), None) == _native.ERR_BADARG, (key, x)


class _Rows(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in ("layer", "n", "tokens", "k_token", "k_head", "v_token",
                                              "v_head")] + \
        [(n, ctypes.c_int32) for n in ("dtype", "reserved")] + \
        [(n, ctypes.c_void_p) for n in ("k", "v", "slots", "starts", "cu")]


def test_c_cache_refuses():
    from enigma import _native
    from enigma.kv_cache import _CacheDesc, _QuantizedDesc
    lib = _native.lib()
    base = dict(layers=1, pages=4, heads_kv=2, page=16, head_dim=64, elem_bytes=1, slots=2,
                table_width=3, k=64, v=64, table=64, lens=64, refs=64, status=64, workspace=64,
                workspace_bytes=1 << 20)
    bad = _native.ERR_BADARG

    def desc(scale=64, code=0, **kw):
        return ctypes.byref(_QuantizedDesc(_CacheDesc(**{**base, **kw}), scale, scale, code, 0))

    # The map's own entries take a cache of codes, the copies of plain caches do not.
    c = _CacheDesc(**base)
    assert lib.enigma_kv_cache_free(ctypes.byref(c), 64, 0, None) == 0
    assert lib.enigma_kv_cache_reserve(ctypes.byref(c), 64, 64, 0, None) == 0
    assert lib.enigma_kv_cache_fork(ctypes.byref(c), 64, 64, 0, None) == bad
    assert lib.enigma_kv_cache_compact(ctypes.byref(c), None) == bad
    assert lib.enigma_kv_cache_copy_pages(ctypes.byref(c), 64, 64, 0, None) == bad
    for d in (None, desc(scale=0), desc(scale=66), desc(code=2), desc(elem_bytes=2), desc(page=48), desc(heads_kv=65536),
              desc(head_dim=24), desc(head_dim=512), desc(k=72), desc(v=0), desc(workspace_bytes=8)):
        assert lib.enigma_kv_cache_q8_compact(d, None) == bad
        assert lib.enigma_kv_cache_q8_fork(d, 64, 64, 0, None) == bad
        assert lib.enigma_kv_cache_q8_copy_pages(d, 64, 64, 0, None) == bad
    good = dict(layer=0, n=1, tokens=1, k_token=128, k_head=64, v_token=128, v_head=64, dtype=1, k=64, v=64,
                slots=64, starts=64, cu=64)
    for fn in (lib.enigma_kv_cache_q8_write, lib.enigma_kv_cache_q8_read):
        assert fn(desc(), ctypes.byref(_Rows(**{**good, "tokens": 0})), None) == 0
        assert fn(desc(), None, None) == bad and fn(None, ctypes.byref(_Rows(**good)), None) == bad
        for key, values in dict(layer=[-1, 1], n=[0, -1, 1 << 31], tokens=[-1, 1 << 31], k_token=[-1],
                                k_head=[-1], v_token=[-1], v_head=[-1], dtype=[2], k=[0, 65], v=[0, 65],
                                slots=[0, 66], starts=[0, 66], cu=[0, 66]).items():
            for x in values:
                assert fn(desc(), ctypes.byref(_Rows(**{**good, key: x})), None) == bad, (key, x)
    for n in (-1, 5):
        assert lib.enigma_kv_cache_q8_copy_pages(desc(), 64, 64, n, None) == bad
    assert lib.enigma_kv_cache_q8_fork(desc(), 64, 64, 3, None) == bad


class _Attend(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in (
        "batch", "heads_q", "heads_kv", "head_dim", "page", "pages", "table_width", "n_slots",
        "q_batch", "q_head", "o_batch", "o_head", "k_page", "v_page", "ks_page", "vs_page")] + \
        [("scale", ctypes.c_float)] + [(n, ctypes.c_int32) for n in ("dtype", "code", "reserved")] + \
        [(n, ctypes.c_void_p) for n in ("table", "lens", "slots", "q", "k_pages", "v_pages", "k_scale",
                                        "v_scale", "out", "workspace")] + \
        [("workspace_bytes", ctypes.c_size_t)]


def test_c_attend_refuses():
    from enigma import _native
    lib, bad = _native.lib(), _native.ERR_BADARG
    good = dict(batch=1, heads_q=4, heads_kv=2, head_dim=64, page=16, pages=4, table_width=3, n_slots=2,
                q_batch=256, q_head=64, o_batch=256, o_head=64, k_page=2048, v_page=2048, ks_page=2,
                vs_page=2, scale=0.1, dtype=1, code=0, table=64, lens=64, slots=64, q=64, k_pages=64,
                v_pages=64, k_scale=64, v_scale=64, out=64, workspace=256, workspace_bytes=1 << 30)
    none = _Attend(**{**good, "batch": 0})
    assert lib.enigma_sdpa_quantized(ctypes.byref(none), None) == 0
    need = ctypes.c_size_t()
    assert lib.enigma_sdpa_quantized_workspace_bytes(ctypes.byref(none), ctypes.byref(need)) == 0
    assert lib.enigma_sdpa_quantized_workspace_bytes(ctypes.byref(none), None) == bad
    assert lib.enigma_sdpa_quantized(None, None) == bad
    for key, values in dict(batch=[-1, 4097], heads_q=[0, 3], heads_kv=[0, 3], head_dim=[0, 24, 272],
                            page=[0, 8, 48, 256], pages=[0, 1 << 40], table_width=[0, 1 << 31],
                            n_slots=[0, 1 << 31], q_batch=[-1], o_head=[-1], k_page=[-16, 8],
                            v_page=[8], ks_page=[-1], scale=[0.0, -1.0, math.inf, math.nan], dtype=[2],
                            code=[2], table=[0, 2], lens=[0], slots=[2], q=[0, 1], k_pages=[0, 72],
                            v_pages=[0, 72], k_scale=[0, 2], v_scale=[0], out=[0, 1]).items():
        for x in values:
            d = _Attend(**{**good, key: x})
            assert lib.enigma_sdpa_quantized(ctypes.byref(d), None) == bad, (key, x)
    many = dict(batch=4096, n_slots=1 << 20)                             # chunks past 32 bits
    for kw in (dict(many, table_width=1 << 25), dict(many, table_width=1 << 18, heads_q=60000, heads_kv=60000,
                                                     pages=1, page=16)):
        d = _Attend(**{**good, **kw})
        assert lib.enigma_sdpa_quantized(ctypes.byref(d), None) == bad, kw
    d = _Attend(**{**good, "slots": 0, "batch": 3})                      # more sequences than rows
    assert lib.enigma_sdpa_quantized(ctypes.byref(d), None) == bad


# --------------------------------------------------------------------------------- oracle
def test_oracle_codes():
    """The oracle's e4m3 rounding is torch's; scales are the least that fit."""
    from oracle import serving as srv
    x = np.random.default_rng(0).standard_normal(4096) * np.exp2(np.linspace(-14, 8, 4096))
    x = np.clip(x, -448, 448).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(srv.to_code(x, "e4m3"), want)
    for code, top in srv.TOP.items():
        t = np.array([top, np.nextafter(top, 1e9), 1.0, 0.0, 1e-40, 3e38])
        s = srv.scale_of(t, code)
        assert (np.log2(s) % 1 == 0).all() and s[0] == 1 and s[1] == 2
        big = np.maximum(t, 2.0 ** -110)
        assert (big <= top * s).all() and (big > top * s / 2).all()
