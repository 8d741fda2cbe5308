"""A continuous batch over the paged cache, then its requests as compressed tiers.

A small random decoder (no checkpoint needed) serves prompts of text and an
image grid, whose tokens have positions on three axes (time, height, width):

1. prompts enter in chunks of any size, new and running requests mixed in one
   step: ``PagedKVCache.plan`` (pages, slots), ``append`` (rotary positions, K
   and V to their pages) and ``attend`` (chunk attention) per layer;
2. decode steps are the same calls with one token per request;
3. a finished request gives its pages back (``release``) to the next one;
4. ``gather`` hands K/V on to ``TieredDecoder``, which keeps decoding from
   FADE's INT4 tiers.

    python examples/paged_serving.py
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch
from torch import Tensor

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from fade_b200 import PagedKVCache, TieredDecoder  # noqa: E402
from fade_b200.rope import MRope  # noqa: E402


class TinyDecoder:
    """Attention layers with random weights: hidden = hidden + out(attention(qkv(hidden)))."""

    def __init__(self, n_layers=2, n_q_heads=8, n_kv_heads=2, head_dim=64, vocab=1000, dtype=torch.bfloat16, seed=0,
                 device="cuda"):
        g = torch.Generator().manual_seed(seed)
        self.L, self.Hq, self.Hkv, self.D, self.dtype = n_layers, n_q_heads, n_kv_heads, head_dim, dtype
        width = n_q_heads * head_dim

        def weight(*shape):
            return (torch.randn(*shape, generator=g) / shape[0] ** 0.5).to(dtype).to(device)

        self.embed = torch.randn(vocab, width, generator=g).to(dtype).to(device)
        self.qkv = [weight(width, (n_q_heads + 2 * n_kv_heads) * head_dim) for _ in range(n_layers)]
        self.out = [weight(width, width) for _ in range(n_layers)]
        self.rope = MRope(theta=10000.0, head_dim=head_dim, mrope_section=[8, 12, 12])
        self.inv_freq = self.rope.axes_inv_freq(torch.device(device))

    def step(self, cache: PagedKVCache, tokens: Tensor, positions: Tensor, new_lens: Tensor, queries=None) -> Tensor:
        """One step: tokens [T] of the requests one after the other (new_lens
        each, the rest padding), positions [3, T].  Returns hidden [T, width];
        ``queries`` collects each layer's rotated queries."""
        T = tokens.shape[0]
        plan = cache.plan(new_lens, T)
        hidden = self.embed[tokens]
        for i in range(self.L):
            heads = (hidden @ self.qkv[i]).view(T, -1, self.D)
            q, k, v = heads.split([self.Hq, self.Hkv, self.Hkv], dim=1)
            q = cache.append(i, plan, q, k, v, self.inv_freq, self.rope.mrope_section, positions)
            if queries is not None:
                queries.append(q)
            o = cache.attend(i, plan, q)                 # zeros for padding tokens
            hidden = hidden + o.reshape(T, -1) @ self.out[i]
        return hidden


def image_prompt_positions(before: int, grid: tuple[int, int], after: int) -> Tensor:
    """[3, tokens] for text, an image grid and text: text counts on all axes,
    the image's tokens share a time and count rows and columns from there."""
    h, w = grid
    text = torch.arange(before).expand(3, -1)
    rows = before + torch.arange(h).repeat_interleave(w)
    cols = before + torch.arange(w).repeat(h)
    image = torch.stack([torch.full((h * w,), before), rows, cols])
    rest = before + max(h, w) + torch.arange(after)
    return torch.cat([text, image, rest.expand(3, -1)], 1)


def serve(model: TinyDecoder, prompts: list[tuple[Tensor, Tensor]], chunk: int, decode_steps: int, page_size: int = 16,
          pages: int = 64) -> tuple[PagedKVCache, list[Tensor], list[Tensor]]:
    """Prefill `prompts` ((tokens [n], positions [3, n]) each) `chunk` tokens per
    request and step, then decode greedily.  Returns the cache, each
    request's last hidden state of its prompt, and its decoded tokens."""
    dev = model.embed.device
    R = len(prompts)
    longest = max(len(t) for t, _ in prompts) + decode_steps
    cache = PagedKVCache(model.L, model.Hkv, model.D, pages, R, longest, page_size, model.dtype, dev)
    done = [0] * R
    last = [None] * R
    while any(done[r] < len(prompts[r][0]) for r in range(R)):
        new = [min(chunk, len(prompts[r][0]) - done[r]) for r in range(R)]
        tokens = torch.cat([prompts[r][0][done[r]:done[r] + new[r]] for r in range(R)]).to(dev)
        positions = torch.cat([prompts[r][1][:, done[r]:done[r] + new[r]] for r in range(R)], 1).to(dev)
        hidden = model.step(cache, tokens, positions, torch.tensor(new, dtype=torch.int32, device=dev))
        at = 0
        for r in range(R):
            done[r] += new[r]
            at += new[r]
            if new[r] and done[r] == len(prompts[r][0]):
                last[r] = hidden[at - 1].clone()
    one = torch.ones(R, dtype=torch.int32, device=dev)
    where = torch.stack([p[:, -1] for _, p in prompts], 1).to(dev)
    token = (torch.stack(last) @ model.embed.t()).argmax(-1)
    decoded = [token]
    for _ in range(decode_steps - 1):
        where = where + 1
        token = (model.step(cache, token, where, one) @ model.embed.t()).argmax(-1)
        decoded.append(token)
    return cache, last, list(torch.stack(decoded, 1))


def main() -> None:
    model = TinyDecoder()
    g = torch.Generator().manual_seed(1)
    prompts = []
    for before, grid, after in ((5, (6, 8), 20), (40, (4, 4), 3), (1, (9, 10), 11)):
        positions = image_prompt_positions(before, grid, after)
        prompts.append((torch.randint(0, 1000, (positions.shape[1],), generator=g), positions))
    cache, last, decoded = serve(model, prompts, chunk=32, decode_steps=6)
    cache.check()
    print("decoded:", [d.tolist() for d in decoded])
    for chunk in (1, 7, 200):
        _, other, tokens = serve(model, prompts, chunk, decode_steps=6)
        far = max(float((a - b).abs().max()) for a, b in zip(last, other))
        print(f"prompts in chunks of {chunk}: largest difference of the hidden states {far:.4f}, tokens equal:",
              all(torch.equal(a, b) for a, b in zip(decoded, tokens)))

    # a request's pages go back to the pool
    free = int(cache.n_free)
    cache.release(torch.tensor([False, True, False], device="cuda"))
    cache.check()
    print(f"pages free: {free}, after releasing request 1: {int(cache.n_free)}")

    # request 0 moves on to INT4 tiers: the same next step, from the pages and from the tiers
    n = int(cache.kv_lens[0])
    tiers = TieredDecoder(model.L, 1, model.Hq, model.Hkv, model.D, model.dtype, n_sink=4, recent_window=16,
                          mid_capacity=256)
    for layer in range(model.L):
        tiers.load_prompt(layer, *cache.gather(layer, [0], n))
    queries: list[Tensor] = []
    new_lens = torch.tensor([1, 0, 0], dtype=torch.int32, device="cuda")
    positions = torch.full((3, 1), int(prompts[0][1][0, -1]) + 6, device="cuda")
    model.step(cache, decoded[0][-1:], positions, new_lens, queries)
    k_new, v_new = (torch.stack([cache.gather(layer, [0], n + 1)[i][:, :, -1] for layer in range(model.L)])
                    for i in (0, 1))
    out = tiers.step(torch.stack(queries).unsqueeze(3), k_new, v_new)
    for layer in range(model.L):
        pages = cache.attend(layer, _one_token_plan(cache), queries[layer])
        err = (out[layer, 0, :, 0].float() - pages[0].float()).norm() / pages.float().norm()
        print(f"layer {layer}: attention from INT4 tiers against pages, relative difference {float(err):.3f}")


def _one_token_plan(cache: PagedKVCache):
    """The plan of a step whose last token of request 0 is in the cache already."""
    from fade_b200.paged import StepPlan

    plan = StepPlan.empty(cache.max_requests, 1)
    plan.cu_q.fill_(1)
    plan.cu_q[0] = 0
    plan.kv_lens.copy_(cache.kv_lens)
    return plan


if __name__ == "__main__":
    main()
