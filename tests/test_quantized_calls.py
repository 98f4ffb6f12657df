"""Calls around the 8-bit cache and rotary positions that have to be refused, or whose defaults have to
be the definition's: found by reading the calls that other tests do not make (host logic)."""
import pytest
import torch

from test_current_device import _on_one, calls  # noqa: F401
from test_quantized_host import _cache, _ints


def test_attend_takes_no_prefix_by_position(calls):  # noqa: F811
    """What follows `slots` in PagedKVCache.attend is a prefix's length, here the softmax's scale: a call
    that gives it by position means one of the two, and must not get the other."""
    cache, q, slots = _cache(), _on_one(2, 4, 64), _ints(2)
    with pytest.raises(TypeError):
        cache.attend(0, q, slots, 48)
    with pytest.raises(TypeError):
        cache.attend(0, q, None, 0)
    with pytest.raises(TypeError):
        cache.attend(0, q, slots, prefix_len=48)
    assert not any(name.startswith("enigma_sdpa") for name, _ in calls.calls)
    cache.attend(0, q, slots, scale=0.1, out=torch.zeros_like(q))
    assert calls.calls[-1][0] == "enigma_sdpa_quantized"


def test_yarn_factor_of_no_stretch():
    """The default factor on cos and sin is 0.1 ln f + 1 where a context is stretched, and 1 where it is
    not (f up to 1); a factor that is given stands."""
    import math
    from enigma.cuda_ops import RopeTable, rope_frequencies
    for f, want in ((0.5, 1.0), (0.999, 1.0), (1.0, 1.0), (1.5, 0.1 * math.log(1.5) + 1),
                    (32.0, 0.1 * math.log(32.0) + 1)):
        scaling = dict(type="yarn", factor=f, original_len=4096)
        assert rope_frequencies(64, 1e4, scaling)[1] == pytest.approx(want, rel=1e-15)
        assert RopeTable(64, theta=1e4, scaling=scaling, device="cpu").factor == pytest.approx(want, rel=1e-15)
        assert rope_frequencies(64, 1e4, dict(scaling, attention_factor=0.75))[1] == 0.75


def test_a_factor_that_nothing_would_use_is_refused():
    from enigma.cuda_ops import rope_frequencies
    with pytest.raises(ValueError, match="factor"):
        rope_frequencies(64, 1e4, {"type": "none", "factor": 8})
    assert rope_frequencies(64, 1e4, {"type": "none", "factor": 1}) == rope_frequencies(64, 1e4)


def test_yarn_borders_in_the_wrong_order_are_refused():
    """Pairs that turn more than beta_fast times stay, those below beta_slow are stretched: with beta_fast
    below beta_slow some pairs would be both."""
    from enigma.cuda_ops import rope_frequencies
    scaling = dict(type="yarn", factor=4.0, original_len=4096)
    with pytest.raises(ValueError, match="beta"):
        rope_frequencies(64, 1e4, dict(scaling, beta_fast=1.0, beta_slow=32.0))
    rope_frequencies(64, 1e4, dict(scaling, beta_fast=4.0, beta_slow=4.0))


def test_queries_without_heads_are_refused(calls):  # noqa: F811
    """A wrong number of axes is a ValueError whether keys come along or not."""
    from enigma import cuda_ops
    from test_quantized_host import _table
    for q in (_on_one(64), _on_one(64)[0], _on_one(5, 64)):
        for k in (None, _on_one(5, 2, 64)):
            with pytest.raises(ValueError):
                cuda_ops.rope(q, k, _ints(5), _table())
    assert not any(name == "enigma_rope" for name, _ in calls.calls)


def test_turns_are_rounded_to_nearest():
    """A frequency's share of a full turn as a 64-bit fraction is off by half a unit, and by the rounding of
    its 64-bit float (2^-52 of it): also where it is so small that the unit counts."""
    import math
    from fractions import Fraction
    from enigma.cuda_ops import RopeTable
    w = [x * 10.0 ** -e for e in range(6, 20) for x in (1.0, -1.7, 2.3, 7.9)]
    t = RopeTable(2 * len(w), frequencies=w, device="cpu")
    for x, got in zip(w, t.turns.tolist()):
        want = Fraction(x) / Fraction(2 * math.pi) * 2 ** 64
        assert abs(got - want) <= abs(want) * Fraction(1, 2 ** 52) + Fraction(1, 2), x


def test_example_keeps_no_tables_of_angles():
    """The sampling example turns by its RopeTable; cos and sin of the whole context are made only where a
    plain decoder asks for them, and are the same turns."""
    import importlib.util
    import math
    import sys
    from pathlib import Path
    path = Path(__file__).resolve().parents[1] / "examples" / "parallel_sampling.py"
    spec = importlib.util.spec_from_file_location("parallel_sampling_host", path)
    ex = sys.modules[spec.name] = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    cfg = ex.Config(layers=1, hidden=64, heads_q=2, heads_kv=1, head_dim=32, intermediate=64, vocab=16,
                    max_len=100)
    model = ex.Decoder(cfg, device="cpu")
    held = [n for n, x in vars(model).items() if isinstance(x, torch.Tensor) and cfg.max_len in x.shape]
    assert held == []
    w = torch.tensor(model.rope.frequencies, dtype=torch.float64)
    angle = torch.arange(100.0, dtype=torch.float64)[:, None] * w
    assert (model.cos - angle.cos()).abs().max() <= 2 ** -24 and (model.sin - angle.sin()).abs().max() <= 2 ** -24
    turns = (model.rope.turns.double() * 2.0 ** -63 * math.pi)               # radians a position, to 2^-52
    assert torch.allclose(turns.cos(), model.cos[1].double(), rtol=0, atol=2 ** -22)
