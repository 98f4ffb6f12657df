"""The sampling example over a cache in 8-bit codes."""
import importlib.util
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "parallel_sampling.py"
    spec = importlib.util.spec_from_file_location("parallel_sampling_codes", path)
    mod = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = mod
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("code", ["int8", "float8_e4m3fn"])
def test_prompts_and_samples(cuda, code):
    """Prompts do not read the cache: the same logits as without codes.  A sample's pages hold what its
    prompt's do, and go back at the end."""
    import torch
    ex = _example()
    cfg = ex.Config(layers=2, hidden=256, heads_q=8, heads_kv=2, head_dim=64, intermediate=512,
                    vocab=128, max_len=256, page=16)
    model = ex.Decoder(cfg, seed=3)
    prompts = [torch.arange(n, device="cuda") % cfg.vocab for n in (37, 1, 96)]
    plain = ex.Sampler(model, prompts, samples=3, new_tokens=20)
    run = ex.Sampler(model, prompts, samples=3, new_tokens=20, codes=getattr(torch, code))
    logits = run.prefill()
    assert (logits == plain.prefill()).all()
    for layer in range(cfg.layers):
        for p, n in enumerate((37, 1, 96)):
            mine = [run.cache.read(layer, [s], [0], [0, n]) for s in (p, 3 + 3 * p, 5 + 3 * p)]
            for k, v in mine[1:]:
                assert (k == mine[0][0]).all() and (v == mine[0][1]).all()
    logits = logits.repeat_interleave(3, dim=0)
    for _ in range(20):
        logits = run.step(logits.argmax(1))
        assert logits.shape == (9, cfg.vocab) and bool(torch.isfinite(logits).all())
    run.cache.check()
    assert run.cache.lens[3:].tolist() == [57] * 3 + [21] * 3 + [116] * 3
    assert run.finish() == 3 + 1 + 6
    assert int(run.cache.lens[3:].abs().sum()) == 0


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_the_command_runs(cuda, capsys, code):
    ex = _example()
    tokens = ex.main(["--prompts", "2", "--samples", "4", "--tokens", "3", "--codes", code])
    assert tuple(tokens.shape) == (8, 3)
    assert "tokens/s" in capsys.readouterr().out
