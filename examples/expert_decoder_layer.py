"""A decoder layer with experts served from 4-bit weights and the 4-bit KV cache.

    python examples/expert_decoder_layer.py [--agents 8] [--prefill 200] [--steps 16]

Several agents share one layer: their prompts go through it as a chunk, then one token each a
step.  The projections, the shared MLP and the experts are Q4 weights (quantized here from
random matrices with the cache's own kernel), the keys and values live in the paged Q4 pool.
The same tokens also run through dense matrices in float32 (the weights dequantized, the
experts one by one), and the relative difference is printed with the time of a decode step.
(Both round to bfloat16 on the way, so now and then a token near a tie goes to another expert.)
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from __graft_entry__ import load_package  # noqa: E402

am = load_package()

WIDTH, HEADS, KV_HEADS, HEAD_DIM = 2048, 16, 4, 128
EXPERTS, TOP_K, INNER = 64, 6, 1408


def rms_norm(x: torch.Tensor) -> torch.Tensor:
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class ExpertDecoderLayer:
    """Attention and a layer of experts (with a shared MLP beside them) over 4-bit weights."""

    def __init__(self, device: torch.device, dtype: torch.dtype = torch.bfloat16, seed: int = 0):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.device, self.dtype, self._plain = device, dtype, {}

        def matrix(name, *shape):
            w = torch.randn(*shape, generator=gen, device=device) * shape[-1] ** -0.5
            parts = am.quantize(w.to(dtype))
            self._plain[name] = parts
            return am.Q4Weight(*parts)

        self.wq = matrix("wq", HEADS * HEAD_DIM, WIDTH)
        self.wk = matrix("wk", KV_HEADS * HEAD_DIM, WIDTH)
        self.wv = matrix("wv", KV_HEADS * HEAD_DIM, WIDTH)
        self.wo = matrix("wo", WIDTH, HEADS * HEAD_DIM)
        self.shared = [matrix(n, INNER, WIDTH) for n in ("shared_gate", "shared_up")]
        self.shared_down = matrix("shared_down", WIDTH, INNER)
        self.experts = [matrix(n, EXPERTS, INNER, WIDTH) for n in ("gate", "up")]
        self.experts_down = matrix("down", EXPERTS, WIDTH, INNER)
        self.router = torch.randn(EXPERTS, WIDTH, generator=gen, device=device) * WIDTH ** -0.5

    def attend(self, h: torch.Tensor, cache, project) -> torch.Tensor:
        """h [agents, L, WIDTH] through the projections and the cache's attention."""
        agents, length = h.shape[:2]
        q, k, v = (project(h, name).view(agents, length, -1, HEAD_DIM).transpose(1, 2).contiguous()
                   for name in ("wq", "wk", "wv"))
        cache.append(k, v)
        a = cache.attention(q, HEAD_DIM ** -0.5)
        return project(a.transpose(1, 2).reshape(agents, length, -1), "wo")

    def forward(self, x: torch.Tensor, cache) -> torch.Tensor:
        """x [agents, L, WIDTH]: the agents' next L tokens -> the layer's output."""
        x = x + self.attend(rms_norm(x), cache, lambda h, n: am.quantized_matmul(h, getattr(self, n)))
        tokens = x.reshape(-1, WIDTH)
        h = rms_norm(tokens)
        r = am.route_experts(h.float() @ self.router.T, TOP_K)
        y = am.expert_matmul(am.expert_swiglu(h, *self.experts, r), self.experts_down, r)
        shared = am.quantized_matmul(am.quantized_swiglu(h, *self.shared), self.shared_down)
        return am.combine_experts(y, r.weights, r.positions, residual=tokens + shared).view_as(x)

    def forward_plain(self, x: torch.Tensor, cache) -> torch.Tensor:
        """The same with dense float32 products (the attention stays the cache's)."""
        dense = lambda name: am.dequantize(*self._plain[name], dtype=torch.float32)  # noqa: E731
        mlp = lambda h, g, u, d: (torch.nn.functional.silu(h @ g.T) * (h @ u.T)) @ d.T  # noqa: E731
        x = x + self.attend(rms_norm(x), cache, lambda h, n: (h.float() @ dense(n).T).to(self.dtype))
        tokens = x.reshape(-1, WIDTH)
        h = rms_norm(tokens).float()
        out = tokens.float() + mlp(h, *map(dense, ("shared_gate", "shared_up", "shared_down")))
        top, chosen = (h @ self.router.T).topk(TOP_K, dim=-1)
        weights = torch.softmax(top, -1)
        gate, up, down = map(dense, ("gate", "up", "down"))
        for e in range(EXPERTS):
            token, slot = (chosen == e).nonzero(as_tuple=True)
            if token.numel():
                out[token] += weights[token, slot, None] * mlp(h[token], gate[e], up[e], down[e])
        return out.to(self.dtype).view_as(x)


def make_cache(agents: int, tokens: int, dtype: torch.dtype, device: torch.device):
    spec = am.ModelCacheSpec(n_layers=1, n_kv_heads=KV_HEADS, head_dim=HEAD_DIM, block_tokens=256,
                             layer_types=["global"])
    blocks = agents * (-(-tokens // 256))
    pool = am.PagedQ4Pool.for_spec(spec, blocks, dtype, device)
    return am.PagedLayerCache(pool, am.shuffled_allocator(spec, blocks, seed=1), 0,
                              [f"agent{i}" for i in range(agents)], tokens)


@torch.no_grad()
def run(agents: int = 8, prefill: int = 200, steps: int = 16, device: str = "cuda:0") -> dict:
    """-> {"error": the largest relative difference of a step, "step_us" and "prefill_us": times}."""
    dev, dtype = torch.device(device), torch.bfloat16
    torch.backends.cuda.matmul.allow_tf32 = False
    layer = ExpertDecoderLayer(dev, dtype)
    caches = [make_cache(agents, prefill + steps, dtype, dev) for _ in range(2)]
    gen = torch.Generator(device=dev).manual_seed(1)
    inputs = [torch.randn(agents, n, WIDTH, generator=gen, device=dev).to(dtype)
              for n in [prefill] + [1] * steps]
    for x in inputs[:2]:  # (the first calls load the kernels)
        layer.forward(x, make_cache(agents, prefill, dtype, dev))
    error, times = 0.0, []
    for x in inputs:
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        got = layer.forward(x, caches[0])
        end.record()
        want = layer.forward_plain(x, caches[1]).float()
        error = max(error, float((got.float() - want).norm() / want.norm()))
        times.append(start.elapsed_time(end) * 1e3)
    return {"error": error, "step_us": sorted(times[1:])[len(times[1:]) // 2] if steps else float("nan"),
            "prefill_us": times[0]}


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--agents", type=int, default=8)
    p.add_argument("--prefill", type=int, default=200)
    p.add_argument("--steps", type=int, default=16)
    a = p.parse_args()
    r = run(a.agents, a.prefill, a.steps)
    print(f"{a.agents} agents: chunk of {a.prefill} tokens each {r['prefill_us']:.0f} us, "
          f"decode step {r['step_us']:.0f} us, relative difference {r['error']:.2e}")
