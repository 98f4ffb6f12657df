"""Several samples of several prompts from one small decoder, on the serving operators.

The prompts, of different lengths, run packed through every layer once (`sdpa_packed`); their
keys and values go into a paged cache (`PagedKVCache.reserve`, `write`). Each prompt is forked into
its samples, which share its pages; every new token is one row per sample, and a prompt's samples
read the prompt's keys once for all (`attend`). At the end the samples are freed and the pages
that prompts still hold move together (`free`, `compact`).

    python examples/parallel_sampling.py --prompts 3 --samples 8 --tokens 32
"""
from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "enigma-dsl_b200"))

from enigma import cuda_ops  # noqa: E402
from enigma.kv_cache import PagedKVCache  # noqa: E402


@dataclass
class Config:
    """Heads as in the framework's decode layer; random weights."""
    layers: int = 4
    hidden: int = 896
    heads_q: int = 14
    heads_kv: int = 2
    head_dim: int = 64
    intermediate: int = 4864
    vocab: int = 1024
    max_len: int = 4096
    page: int = 64
    eps: float = 1e-6
    rope_theta: float = 1e6


class Decoder:
    """A pre-norm decoder with grouped heads, rotary positions and a SwiGLU MLP, in bf16."""

    def __init__(self, cfg: Config, seed: int = 0, device="cuda"):
        import torch
        self.cfg, self.device = cfg, torch.device(device)
        gen = torch.Generator(device=self.device).manual_seed(seed)

        def weight(rows, cols):
            w = torch.randn(rows, cols, generator=gen, device=self.device)
            return (w / rows ** 0.5).bfloat16()

        qkv = (cfg.heads_q + 2 * cfg.heads_kv) * cfg.head_dim
        self.layers = [dict(norm=torch.ones(cfg.hidden, device=self.device).bfloat16(),
                            qkv=weight(cfg.hidden, qkv),
                            o=weight(cfg.heads_q * cfg.head_dim, cfg.hidden),
                            post=torch.ones(cfg.hidden, device=self.device).bfloat16(),
                            gate_up=weight(cfg.hidden, 2 * cfg.intermediate),
                            down=weight(cfg.intermediate, cfg.hidden))
                       for _ in range(cfg.layers)]
        self.embed = torch.randn(cfg.vocab, cfg.hidden, generator=gen, device=self.device).bfloat16()
        self.head = weight(cfg.hidden, cfg.vocab)
        half = cfg.head_dim // 2
        inv = cfg.rope_theta ** (-torch.arange(half, device=self.device, dtype=torch.float64)
                                 * 2.0 / cfg.head_dim)
        angle = torch.arange(cfg.max_len, device=self.device, dtype=torch.float64)[:, None] * inv
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def rotate(self, x, positions):
        """Rotary positions on [tokens, heads, head_dim], in place (a view of the projection)."""
        half = self.cfg.head_dim // 2
        cos, sin = self.cos[positions][:, None], self.sin[positions][:, None]
        a, b = x[..., :half].float(), x[..., half:].float()
        x[..., :half] = (a * cos - b * sin).to(x.dtype)
        x[..., half:] = (b * cos + a * sin).to(x.dtype)
        return x

    def forward(self, tokens, positions, attention, last=None):
        """Logits (fp32) of the rows `last`, or of all; attention(layer, q, k, v) -> o."""
        import torch
        cfg = self.cfg
        x = self.embed[tokens]
        for i, w in enumerate(self.layers):
            qkv = cuda_ops.gemm(cuda_ops.rmsnorm(x, w["norm"], cfg.eps), w["qkv"])
            q, k, v = qkv.view(len(x), -1, cfg.head_dim).split(
                [cfg.heads_q, cfg.heads_kv, cfg.heads_kv], dim=1)
            o = attention(i, self.rotate(q, positions), self.rotate(k, positions), v)
            x = x + cuda_ops.gemm(o.reshape(len(x), -1), w["o"])
            up = cuda_ops.gemm(cuda_ops.rmsnorm(x, w["post"], cfg.eps), w["gate_up"])
            gate, up = up.chunk(2, dim=1)
            x = x + cuda_ops.gemm((torch.nn.functional.silu(gate.float()) * up).bfloat16(),
                                  w["down"])
        if last is not None:
            x = x[last]
        ones = torch.ones(cfg.hidden, device=self.device).bfloat16()
        return cuda_ops.gemm(cuda_ops.rmsnorm(x.contiguous(), ones, cfg.eps), self.head).float()


class Sampler:
    """Prompts and their samples over one cache: slot p is prompt p, then prompt by prompt its
    samples."""

    def __init__(self, model: Decoder, prompts, samples: int, new_tokens: int):
        import torch
        cfg = model.cfg
        self.model, self.samples = model, samples
        self.lens = [len(p) for p in prompts]
        n = len(prompts)
        longest = max(self.lens) + new_tokens
        # A sample's own pages: a copy of the prompt's last, and room for its new tokens.
        pages = sum(-(-x // cfg.page) for x in self.lens) + n * samples * (-(-new_tokens // cfg.page) + 1)
        self.cache = PagedKVCache.empty(cfg.layers, pages, cfg.page, cfg.heads_kv, cfg.head_dim,
                                        slots=n * (1 + samples), max_len=longest,
                                        device=model.device)
        self.tokens = torch.cat([torch.as_tensor(p, device=model.device) for p in prompts])
        self.sample_slots = torch.arange(n, n * (1 + samples), dtype=torch.int32,
                                         device=model.device)

    def prefill(self):
        """Every prompt's keys and values into the cache; logits after each prompt's last token."""
        import torch
        cfg, cache, dev = self.model.cfg, self.cache, self.model.device
        n = len(self.lens)
        lens = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        cu = torch.zeros(n + 1, dtype=torch.int32, device=dev)
        cu[1:] = lens.cumsum(0)
        slots = torch.arange(n, dtype=torch.int32, device=dev)
        starts = torch.zeros(n, dtype=torch.int32, device=dev)
        positions = torch.cat([torch.arange(x, device=dev) for x in self.lens])
        plan = cuda_ops.PackedPlan(self.lens, heads_q=cfg.heads_q, heads_kv=cfg.heads_kv, device=dev)
        scratch = torch.empty(plan.workspace_bytes(cfg.head_dim), dtype=torch.uint8, device=dev)
        cache.reserve(slots, lens)

        def attention(layer, q, k, v):
            cache.write(layer, k, v, slots, starts, cu)
            return cuda_ops.sdpa_packed(q, k, v, plan, workspace=scratch if len(scratch) else None)

        logits = self.model.forward(self.tokens, positions, attention, last=cu[1:].long() - 1)
        cache.fork(slots.repeat_interleave(self.samples), self.sample_slots)
        return logits

    def step(self, tokens):
        """One token per sample (in slot order); logits for the next ones."""
        import torch
        cache, slots = self.cache, self.sample_slots
        starts = cache.lens[slots.long()]
        cu = torch.arange(len(slots) + 1, dtype=torch.int32, device=slots.device)
        cache.reserve(slots, starts + 1)

        def attention(layer, q, k, v):
            cache.write(layer, k, v, slots, starts, cu)
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            for p, prompt_len in enumerate(self.lens):
                mine = slice(p * self.samples, (p + 1) * self.samples)
                cache.attend(layer, q[mine], slots=slots[mine], prefix_len=prompt_len,
                             out=out[mine])
            return out

        return self.model.forward(tokens, starts.long(), attention)

    def finish(self):
        """The samples' pages go back; the prompts' move to the front.  Pages still in use."""
        self.cache.free(self.sample_slots)
        self.cache.compact()
        self.cache.check()
        return int((self.cache.refs > 0).sum())


def main(argv=None):
    import torch
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompts", type=int, default=3)
    ap.add_argument("--samples", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=32, help="new tokens per sample")
    ap.add_argument("--temperature", type=float, default=1.0)
    args = ap.parse_args(argv)
    cfg = Config()
    model = Decoder(cfg)
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab, (300 + 611 * p,), generator=gen, device="cuda")
               for p in range(args.prompts)]
    run = Sampler(model, prompts, args.samples, args.tokens)
    logits = run.prefill().repeat_interleave(args.samples, dim=0)
    out = []
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(args.tokens):
        weights = (logits / args.temperature).softmax(dim=1)
        out.append(torch.multinomial(weights, 1, generator=gen)[:, 0])
        logits = run.step(out[-1])
    run.cache.check()
    seconds = time.perf_counter() - start
    pages = int((run.cache.refs > 0).sum())
    kept = run.finish()
    tokens = torch.stack(out, dim=1)
    print(f"{args.prompts} prompts of {run.lens} tokens, {args.samples} samples each, "
          f"{args.tokens} tokens per sample: {tokens.numel() / seconds:.0f} tokens/s, "
          f"{pages} pages in use, {kept} after the samples were freed")
    return tokens


if __name__ == "__main__":
    main()
