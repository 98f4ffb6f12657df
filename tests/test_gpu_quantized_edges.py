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
