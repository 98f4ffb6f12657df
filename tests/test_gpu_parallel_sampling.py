"""The sampling example: packed prompts, forked samples and paged decoding against a plain fp32
decoder that sees each sample's whole sequence."""
import importlib.util
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "parallel_sampling.py"
    spec = importlib.util.spec_from_file_location("parallel_sampling", path)
    mod = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = mod
    spec.loader.exec_module(mod)
    return mod


def _plain(model, tokens):
    """Logits of every position of one sequence, in fp32 torch operations."""
    import torch
    cfg = model.cfg

    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.eps)

    def rotate(x):
        half = cfg.head_dim // 2
        cos, sin = model.cos[:len(x), None], model.sin[:len(x), None]
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)

    x = model.embed[tokens].float()
    n = len(x)
    mask = torch.ones(n, n, dtype=torch.bool, device=x.device).tril()
    for w in model.layers:
        qkv = (norm(x) @ w["qkv"].float()).view(n, -1, cfg.head_dim)
        q, k, v = qkv.split([cfg.heads_q, cfg.heads_kv, cfg.heads_kv], dim=1)
        group = cfg.heads_q // cfg.heads_kv
        q, k, v = rotate(q), rotate(k).repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = torch.einsum("ihd,jhd->hij", q, k) / cfg.head_dim ** 0.5
        s = s.masked_fill(~mask, float("-inf")).softmax(-1)
        x = x + torch.einsum("hij,jhd->ihd", s, v).reshape(n, -1) @ w["o"].float()
        gate, up = (norm(x) @ w["gate_up"].float()).chunk(2, dim=1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].float()
    return norm(x) @ model.head.float()


def test_samples_match_a_plain_decoder(cuda):
    """Each layer rounds its activations to bf16 (2^-8 relative at most) nine times on the way to the
    residual stream, the head twice: 2 layers, 20 roundings, 20 * 2^-8 = 0.08 if all added up."""
    import torch
    ex = _example()
    torch.backends.cuda.matmul.allow_tf32 = False
    cfg = ex.Config(layers=2, hidden=256, heads_q=8, heads_kv=2, head_dim=64, intermediate=512,
                    vocab=128, max_len=256, page=16)
    model = ex.Decoder(cfg, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(5)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen, device="cuda") for n in (37, 1, 96)]
    run = ex.Sampler(model, prompts, samples=3, new_tokens=20)
    logits = run.prefill().repeat_interleave(3, dim=0)
    seen = [logits]
    chosen = []
    for _ in range(20):
        chosen.append(torch.multinomial(logits.softmax(1), 1, generator=gen)[:, 0])
        logits = run.step(chosen[-1])
        seen.append(logits)
    run.cache.check()
    chosen = torch.stack(chosen, dim=1)
    for row in range(9):
        prompt = prompts[row // 3]
        want = _plain(model, torch.cat([prompt, chosen[row]]))[len(prompt) - 1:]
        got = torch.stack([x[row] for x in seen])
        error = (got - want).norm() / want.norm()
        assert float(error) <= 0.08
    assert run.finish() == sum(-(-len(p) // cfg.page) for p in prompts)
    assert int(run.cache.lens[3:].abs().sum()) == 0


def test_the_command_runs(cuda, capsys):
    ex = _example()
    tokens = ex.main(["--prompts", "2", "--samples", "4", "--tokens", "3"])
    assert tuple(tokens.shape) == (8, 3)
    assert "tokens/s" in capsys.readouterr().out
