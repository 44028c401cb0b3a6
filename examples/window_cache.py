"""One attention layer through its life: a training step under the window, a prompt, then
tokens over the paged cache with eviction by attention weight.

    python examples/window_cache.py

Run on a B200 with the library built (``python -m ascendc_kernel_b200.build``).
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ascendc_kernel_b200.paged_cache import PagedKVCache  # noqa: E402
from ascendc_kernel_b200.window_attn import WindowAttention  # noqa: E402


class Layer(torch.nn.Module):
    """Projections around the windowed attention; the kv head serves as keys and values."""

    def __init__(self, dim: int, n_heads: int, head_dim: int, window: int, n_first: int):
        super().__init__()
        self.n_heads, self.head_dim = n_heads, head_dim
        self.wq = torch.nn.Linear(dim, n_heads * head_dim, bias=False)
        self.wkv = torch.nn.Linear(dim, head_dim, bias=False)
        self.wo = torch.nn.Linear(n_heads * head_dim, dim, bias=False)
        self.attn = WindowAttention(n_heads, head_dim, window, n_first)

    def heads(self, x: torch.Tensor):
        b, t, _ = x.shape
        return (self.wq(x).view(b, t, self.n_heads, self.head_dim),
                self.wkv(x).view(b, t, 1, self.head_dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        q, kv = self.heads(x)
        return self.wo(self.attn(q, kv).flatten(2))

    @torch.no_grad()
    def prompt(self, x: torch.Tensor, cache: PagedKVCache) -> torch.Tensor:
        q, kv = self.heads(x)
        cache.append(kv)
        return self.wo(self.attn(q, kv).flatten(2))

    @torch.no_grad()
    def token(self, x: torch.Tensor, cache: PagedKVCache) -> torch.Tensor:
        """x [b, 1, dim]. The cache holds what eviction left, so every row of it is read."""
        q, kv = self.heads(x)
        cache.append(kv)
        out = cache.attend(q[:, 0], self.attn.attn_sink)
        return self.wo(out.flatten(1)).unsqueeze(1)


def main(batch: int = 2, prompt: int = 300, tokens: int = 64, budget: int = 128, dim: int = 256,
         device="cuda") -> dict:
    torch.manual_seed(0)
    layer = Layer(dim, n_heads=16, head_dim=128, window=128, n_first=4).to(device, torch.bfloat16)
    layer.attn.attn_sink.data = layer.attn.attn_sink.data.float()
    x = torch.randn(batch, prompt, dim, device=device, dtype=torch.bfloat16)

    # a training step
    opt = torch.optim.SGD(layer.parameters(), lr=1e-2)
    before = (layer(x).float() - x.float()).square().mean()
    before.backward()
    opt.step()
    after = (layer(x).float() - x.float()).square().mean()

    # serving
    cache = PagedKVCache(batch, num_pages=64, page_size=16, max_len=512, n_kv_heads=1,
                         head_dim=128, shared=True, track_weights=True, device=device)
    y = layer.prompt(x, cache)[:, -1:]
    lengths = []
    for _ in range(tokens):
        y = layer.token(y, cache)
        if cache.host_lens[0] > 2 * budget:
            cache.evict(budget, n_first=4, n_recent=32)
        lengths.append(cache.host_lens[0])
    torch.cuda.synchronize()
    return {"loss_before": before.item(), "loss_after": after.item(), "lengths": lengths,
            "last": y, "cache": cache, "layer": layer}


if __name__ == "__main__":
    r = main()
    print(f"loss {r['loss_before']:.4f} -> {r['loss_after']:.4f}; "
          f"cache lengths {min(r['lengths'])} .. {max(r['lengths'])}")
