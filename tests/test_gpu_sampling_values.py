"""The sampling example's steps over an 8-bit cache against a plain decoder: each sample's logits are
recomputed in fp32 from its own token, its position and the keys and values that `read` gives for its
slot, so a slot, a position or a prompt that belongs to another sample shows."""
import pytest

from test_gpu_sampling_codes import _example

pytestmark = pytest.mark.gpu


def _step(model, token, position, held):
    """Logits of one token at `position`; held(layer) -> k, v [position + 1, heads_kv, head_dim] fp32."""
    import torch
    cfg = model.cfg
    half = cfg.head_dim // 2
    inv = cfg.rope_theta ** (-torch.arange(half, device="cuda", dtype=torch.float64) * 2.0 / cfg.head_dim)
    cos, sin = ((position * inv).cos().float(), (position * inv).sin().float())

    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + cfg.eps)

    x = model.embed[token].float()[None]
    for i, w in enumerate(model.layers):
        q = (norm(x) @ w["qkv"].float()).view(-1, cfg.head_dim)[:cfg.heads_q]
        a, b = q[:, :half], q[:, half:]
        q = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        k, v = (y.repeat_interleave(cfg.heads_q // cfg.heads_kv, 1) for y in held(i))
        s = (torch.einsum("hd,jhd->hj", q, k) / cfg.head_dim ** 0.5).softmax(-1)
        x = x + torch.einsum("hj,jhd->hd", s, v).reshape(1, -1) @ w["o"].float()
        gate, up = (norm(x) @ w["gate_up"].float()).chunk(2, dim=1)
        x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].float()
    return (norm(x) @ model.head.float())[0]


@pytest.mark.parametrize("code", ["int8", "float8_e4m3fn"])
def test_steps_match_a_plain_decoder(cuda, code):
    """The bound of the bf16 cache's example: each layer rounds its activations to bf16 (2^-8 relative at
    most) nine times on the way to the residual stream, the head twice: 2 layers, 20 roundings, 20 * 2^-8
    = 0.08 if all added up.  Keys and values are what `read` gives, the token's own among them, so their
    codes' rounding is on both sides.  (The weights' rounding to fp16 in attention, 2^-11, is among the
    roundings of its result.)"""
    import torch
    ex = _example()
    torch.backends.cuda.matmul.allow_tf32 = False
    cfg = ex.Config(layers=2, hidden=256, heads_q=8, heads_kv=2, head_dim=64, intermediate=512,
                    vocab=128, max_len=256, page=16)
    model = ex.Decoder(cfg, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(5)
    lens = (37, 1, 96)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=gen, device="cuda") for n in lens]
    run = ex.Sampler(model, prompts, samples=3, new_tokens=20, codes=getattr(torch, code))
    logits = run.prefill().repeat_interleave(3, dim=0)
    for t in range(20):
        tokens = torch.multinomial(logits.softmax(1), 1, generator=gen)[:, 0]
        logits = run.step(tokens)
        for row in range(9):
            at, slot = lens[row // 3] + t, 3 + row

            def held(layer):
                return run.cache.read(layer, [slot], [0], [0, at + 1], dtype=torch.float32)

            want = _step(model, tokens[row], at, held)
            error = (logits[row] - want).norm() / want.norm()
            assert float(error) <= 0.08, (t, row, float(error))
    run.cache.check()
