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
