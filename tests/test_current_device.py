"""Calls reach the library with their tensors' device current, and the caller's device is current again
afterwards (host logic: a stand-in for torch's device state and for the library's launches)."""
import contextlib
import types

import pytest
import torch


class OnOne(torch.Tensor):
    """A host tensor that says it is on cuda:1."""

    def get_device(self):
        return 1

    is_cuda = True


def _on_one(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnOne)


@pytest.fixture
def calls(monkeypatch):
    """(entry, current device) of every call into the library; device 0 is the caller's."""
    from enigma import _native, cuda_ops
    real = _native.lib()
    state = types.SimpleNamespace(device=0, calls=[])

    @contextlib.contextmanager
    def device(index):
        before, state.device = state.device, index
        try:
            yield
        finally:
            state.device = before

    class Torch:
        _C = types.SimpleNamespace(_cuda_getDevice=lambda: state.device,
                                   _cuda_getCurrentRawStream=lambda index: 0)
        cuda = types.SimpleNamespace(
            device=device, synchronize=lambda device=None: None,
            current_stream=lambda device=None: types.SimpleNamespace(cuda_stream=0))

        def __getattr__(self, name):
            return getattr(torch, name)

    class Library:
        def __getattr__(self, name):
            def call(*args):
                state.calls.append((name, state.device))
                if name == "enigma_init":
                    state.device = args[0]            # as cudaSetDevice does
                    return 0
                host = name.endswith("_bytes") or name.endswith("_plan")
                return getattr(real, name)(*args) if host else 0
            return call

    monkeypatch.setattr(cuda_ops, "_torch_module", Torch())
    monkeypatch.setattr(cuda_ops, "_initialised", set())
    monkeypatch.setattr(_native, "_lib", Library())
    cuda_ops._shared_head.cache_clear()
    yield state
    cuda_ops._shared_head.cache_clear()


def _check(state, *entries):
    """These entries were called, all but the first use of the device with device 1 current."""
    assert [name for name, _ in state.calls if name != "enigma_init"] == list(entries)
    assert all(device == 1 for name, device in state.calls if name != "enigma_init")
    assert state.device == 0
    state.calls.clear()


def test_serving_operators(calls):
    from enigma import cuda_ops
    for _ in range(2):                                # the first use of the device, and a later one
        plan = cuda_ops.PackedPlan([5], heads_q=4, heads_kv=2, device="cpu")
        plan.ints = plan.ints.as_subclass(OnOne)
        calls.calls.clear()
        q, k = _on_one(5, 4, 64), _on_one(5, 2, 64)
        cuda_ops.sdpa_packed(q, k, k, plan)
        assert all(x == 1 for name, x in calls.calls if name == "enigma_sdpa_packed")
        assert calls.device == 0
        calls.calls.clear()
        pages, ints = _on_one(3, 2, 16, 64), _on_one(5, 2, dtype=torch.int32)
        cuda_ops._shared_head.cache_clear()
        cuda_ops.sdpa_shared_prefix(q, pages, pages, ints, _on_one(5, dtype=torch.int32))
        _check(calls, "enigma_sdpa_shared_prefix_workspace_bytes", "enigma_sdpa_shared_prefix")


def test_cache(calls):
    from enigma.kv_cache import PagedKVCache
    ints = lambda *shape: _on_one(*shape, dtype=torch.int32)  # noqa: E731
    cache = PagedKVCache(_on_one(1, 4, 2, 16, 8), _on_one(1, 4, 2, 16, 8), ints(2, 3), ints(2),
                         ints(4))
    assert calls.device == 0
    calls.calls.clear()
    one = ints(1)
    cache.reserve(one, one)
    cache.write(0, _on_one(1, 2, 8), _on_one(1, 2, 8), one, one, ints(2))
    cache.fork(one, one)
    cache.free(one)
    cache.compact()
    cache.copy_pages(one, one)
    _check(calls, *("enigma_kv_cache_" + x for x in ("reserve", "write", "fork", "free", "compact",
                                                     "copy_pages")))


def test_dense_operators(calls):
    from enigma import cuda_ops
    x, w = _on_one(2, 8), _on_one(8)
    cuda_ops.rmsnorm(x, w)
    cuda_ops.gemm(_on_one(8, 8), _on_one(8, 8), out=_on_one(8, 8))
    cuda_ops.sdpa(*(_on_one(1, 2, 4, 8) for _ in range(3)))
    cuda_ops.synchronize(1)
    _check(calls, "enigma_rmsnorm", "enigma_gemm_bf16", "enigma_sdpa_bf16", "enigma_synchronize")


def test_plan_of_another_device(calls):
    """A plan is dealt out over the SMs of the device that it is for."""
    from enigma import cuda_ops
    with contextlib.suppress(RuntimeError, AssertionError):      # no such device here
        cuda_ops.PackedPlan([5], heads_q=4, heads_kv=2, device="cuda:1")
    _check(calls, "enigma_sdpa_packed_plan", "enigma_sdpa_packed_plan")
