"""The packed attention's work list (host): every row of every sequence exactly once, the keys it
needs, heaviest first; and the oracle of the serving operators against a direct computation."""
import ctypes

import numpy as np
import pytest

from oracle import serving as srv


def _parts(plan):
    """header, (n_ctas + 1) offsets, items, groups of a plan."""
    ints = plan.ints.tolist()
    n, ctas, slots, n_groups, items_at, groups_at, total, _ = ints[:8]
    assert total == len(ints) and list(plan.header) == ints[:8]
    assert items_at % 4 == 0 and items_at >= 9 + ctas
    items = [ints[items_at + 12 * i:items_at + 12 * i + 12] for i in range(n)]
    groups = [ints[groups_at + 8 * i:groups_at + 8 * i + 8] for i in range(n_groups)]
    return ints[8:9 + ctas], items, groups, slots


@pytest.mark.parametrize("heads_q,heads_kv", [(14, 2), (8, 8), (32, 8), (200, 1), (128, 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [([300, 0, 1, 257, 64], [300, 5, 700, 100, 64]), ([1], [9000]),
                                  ([40, 1], [5000, 20000]), ([5000], [5000]), ([3, 0], [0, 0])])
def test_plan_covers_every_pair_of_row_and_key_once(heads_q, heads_kv, causal, lens):
    from enigma import cuda_ops
    lens_q, lens_k = lens
    plan = cuda_ops.PackedPlan(lens_q, lens_k, heads_q=heads_q, heads_kv=heads_kv, causal=causal,
                               device="cpu")
    offsets, items, groups, slots = _parts(plan)
    assert plan.tokens_q == sum(lens_q) and plan.tokens_k == sum(lens_k)
    assert offsets[0] == 0 and offsets[-1] == len(items) and offsets == sorted(offsets)
    group = heads_q // heads_kv
    starts_q, starts_k = np.cumsum([0] + lens_q), np.cumsum([0] + lens_k)
    seen, used = {}, set()
    for q0, lq, k0, lk, t0, tokens, j0, j1, kvh, slot, _, _ in items:
        assert tokens == max(1, 128 // group) and 0 <= kvh < heads_kv and 0 <= t0 < lq
        assert any((starts_q[i], lens_q[i], starts_k[i], lens_k[i]) == (q0, lq, k0, lk)
                   for i in range(len(lens_q)))
        seen.setdefault((q0 + t0, kvh), []).append((j0, j1, slot))
        if slot >= 0:
            assert 0 <= slot < slots and slot % 2 == 0 and slot not in used
            used.add(slot)
    want = {(int(starts_q[i]) + t0, h) for i in range(len(lens_q))
            for t0 in range(0, lens_q[i], 2 * max(1, 128 // group)) for h in range(heads_kv)}
    assert set(seen) == want and len(used) * 2 == slots
    by_group = {(g[0], g[3]): g for g in groups}
    for (tok, kvh), parts in seen.items():
        parts.sort()
        i = max(x for x in range(len(lens_q)) if starts_q[x] <= tok and lens_q[x])
        t0, tokens = tok - starts_q[i], max(1, 128 // group)
        last = min(t0 + 2 * tokens, lens_q[i]) - 1
        keys = min(lens_k[i], last + lens_k[i] - lens_q[i] + 1) if causal else lens_k[i]
        assert parts[0][0] == 0 and parts[-1][1] == max(0, -(-keys // 128))
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        if parts[0][2] >= 0:
            g = by_group[tok, kvh]
            assert g[1] == starts_q[i] + lens_q[i] and g[2] == tokens and g[5] == len(parts)
            assert [p[2] for p in parts] == list(range(g[4], g[4] + 2 * len(parts), 2))
            assert group <= 128
        else:
            assert len(parts) == 1 and (tok, kvh) not in by_group


def test_plan_is_even():
    """No thread block has much more than its share of the key tiles."""
    from enigma import cuda_ops
    for lens, heads in (([8192], (32, 8)), ([37, 1024, 211, 2048, 640, 129, 900], (32, 8)),
                        ([1] * 5, (14, 2)), ([20000], (14, 2))):
        offsets, items, _, _ = _parts(cuda_ops.PackedPlan(lens, heads_q=heads[0],
                                                          heads_kv=heads[1], device="cpu"))
        cost = [i[7] - i[6] + 2 for i in items]
        load = [sum(cost[a:b]) for a, b in zip(offsets, offsets[1:])]
        assert max(load) <= sum(cost) / len(load) + 1.5 * max(cost)


def test_plan_refusals():
    from enigma import _native, cuda_ops
    with pytest.raises(ValueError, match="differ in number"):
        cuda_ops.PackedPlan([1, 2], [1], heads_q=4, heads_kv=2, device="cpu")
    with pytest.raises(_native.EnigmaCudaError, match="multiple"):
        cuda_ops.PackedPlan([1], heads_q=5, heads_kv=2, device="cpu")
    with pytest.raises(_native.EnigmaCudaError, match="negative"):
        cuda_ops.PackedPlan([-1], heads_q=4, heads_kv=2, device="cpu")
    with pytest.raises(_native.EnigmaCudaError, match="int32"):
        cuda_ops.PackedPlan([1 << 30, 1 << 30], heads_q=4, heads_kv=2, device="cpu")


def test_abi_refuses_before_launch():
    """NULL descriptors and buffers are refused on any host, without a GPU."""
    from enigma import _native
    lib = _native.lib()
    n = ctypes.c_int64()
    size = ctypes.c_size_t()
    for rc in (lib.enigma_sdpa_packed(None, None), lib.enigma_sdpa_shared_prefix(None, None),
               lib.enigma_sdpa_shared_prefix_workspace_bytes(None, ctypes.byref(size)),
               lib.enigma_kv_cache_workspace_bytes(None, ctypes.byref(size)),
               lib.enigma_kv_cache_compact(None, None),
               lib.enigma_kv_cache_fork(None, None, None, 1, None),
               lib.enigma_sdpa_packed_plan(None, None, 1, 4, 2, 1, None, 0, ctypes.byref(n)),
               lib.enigma_sdpa_packed_plan(None, None, 0, 4, 2, 1, None, 0, None)):
        assert rc == _native.ERR_BADARG


def test_oracle_attend_is_softmax():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal(s) for s in ((2, 8), (9, 8), (9, 8)))
    out, mag, lse, err = srv.attend(q, k, v, 0.5, [9, 0])
    w = np.exp(0.5 * k @ q[0])
    np.testing.assert_allclose(out[0], w @ v / w.sum(), rtol=1e-12)
    np.testing.assert_allclose(lse[0], np.log(w.sum()), rtol=1e-12)
    assert (out[1] == 0).all() and lse[1] == -np.inf and (mag[0] >= np.abs(out[0])).all()


def test_a_plan_that_is_too_large_is_refused_before_it_is_made():
    """In a process that has no room for it: as an argument that is refused, not by running out."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import ctypes, resource
resource.setrlimit(resource.RLIMIT_AS, (2 << 30, 2 << 30))
from enigma import _native
for heads, tokens in ((65535, (1 << 31) - 300), (65535, 1 << 20)):
    length, n = (ctypes.c_int64 * 1)(tokens), ctypes.c_int64()
    rc = _native.lib().enigma_sdpa_packed_plan(length, length, 1, heads, heads, 1, None, 0,
                                               ctypes.byref(n))
    print(rc, _native.last_error())
"""
    root = Path(__file__).resolve().parents[1] / "enigma-dsl_b200"
    out = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True,
                         timeout=120)
    lines = out.stdout.splitlines()
    assert out.returncode == 0 and len(lines) == 2, out.stderr
    assert all(x.startswith("-4 ") and "too much work" in x for x in lines), lines
