"""Serves a small random decoder with the serving operators: prompts of different lengths are
prefilled in chunks, then all sequences decode greedily, one token a step.

    python examples/serve_decoder.py [--layers 4] [--new-tokens 16]

Every projection runs as an i8 product with a scale per token and channel, keys are rotated
on their way into a paged cache, and one attention call serves chunks and single tokens alike.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from rustgears_b200 import serving  # noqa: E402


class Decoder:
    """Pre-norm decoder layers of the transformer configuration's widths: attention, then SwiGLU."""

    def __init__(self, layers, d=1024, heads=16, kv_heads=4, hidden=2816, vocab=32000, positions=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(n, k):
            return torch.randn((n, k), device="cuda", generator=g) * k ** -0.5

        dim = d // heads
        table = serving.rope_table(positions, dim)
        self.embedding = torch.randn((vocab, d), device="cuda", generator=g).bfloat16()
        self.attention = [serving.DecoderAttention(normal((heads + 2 * kv_heads) * dim, d), normal(d, d), heads, kv_heads,
                                                   table) for _ in range(layers)]
        self.mlp = [(serving.quantize_weight_i8(normal(hidden, d)), serving.quantize_weight_i8(normal(hidden, d)),
                     serving.quantize_weight_i8(normal(d, hidden))) for _ in range(layers)]
        self.head = serving.quantize_weight_i8(self.embedding.float())
        self.cache_shape = (layers, kv_heads, dim)

    @staticmethod
    def norm(x):
        y = x.float()
        return (y * (y.square().mean(-1, keepdim=True) + 1e-5).rsqrt()).to(x.dtype)

    def __call__(self, ids, cache, step):
        """The logits of each sequence's last new token."""
        x = self.embedding[ids]
        for i, (attention, (gate, up, down)) in enumerate(zip(self.attention, self.mlp)):
            x = x + attention(self.norm(x), cache.k[i], cache.v[i], step)
            y = self.norm(x)
            x = x + serving.linear_i8_token(serving.linear_i8_token(y, *gate, act="silu") *
                                            serving.linear_i8_token(y, *up), *down)
        last = step.cu_q[1:].long() - 1
        return serving.linear_i8_token(self.norm(x[last]), *self.head, out_dtype=torch.float32)


def generate(model, prompts, new_tokens, chunk=256, page_size=16):
    """Greedy continuation of every prompt (lists of token ids), and the logits of each step."""
    layers, kv_heads, dim = model.cache_shape
    pages = sum(-(-(len(p) + new_tokens) // page_size) for p in prompts)
    cache = serving.PagedKvCache(layers, pages, page_size, kv_heads, dim)
    done, logits = [0] * len(prompts), {}
    while any(n < len(p) for n, p in zip(done, prompts)):       # chunks of all unfinished prompts together
        take = {s: min(chunk, len(p) - done[s]) for s, p in enumerate(prompts) if done[s] < len(p)}
        ids = torch.tensor([t for s, n in take.items() for t in prompts[s][done[s]:done[s] + n]], device="cuda")
        out = model(ids, cache, cache.extend(take))
        for row, (s, n) in enumerate(take.items()):
            done[s] += n
            logits[s] = out[row]
    steps = [torch.stack([logits[s] for s in range(len(prompts))])]
    tokens = [steps[0].argmax(-1)]
    for _ in range(new_tokens - 1):
        steps.append(model(tokens[-1], cache, cache.extend({s: 1 for s in range(len(prompts))})))
        tokens.append(steps[-1].argmax(-1))
    serving.check()
    return torch.stack(tokens, 1), torch.stack(steps, 1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--new-tokens", type=int, default=16)
    a = ap.parse_args()
    model = Decoder(a.layers)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 32000, (n,), generator=g).tolist() for n in (7, 300, 64, 1000)]
    tokens, _ = generate(model, prompts, a.new_tokens)
    for p, t in zip(prompts, tokens.tolist()):
        print(f"prompt of {len(p)} tokens -> {t}")


if __name__ == "__main__":
    main()
