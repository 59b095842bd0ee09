"""Greedy decoding with 4-bit weights and a 4-bit key/value cache: what a serving loop calls, in order.

    python examples/decode_4bit.py            # a small random model, a ragged batch of prompts

A layer's step: RMS norm (`row_reduce`), the W4A16 product for queries, keys and values, `kv4_append` (rotates queries and
keys, quantises keys and values into the paged cache), `kv4_attention` over the pages, and the W4A16 products of the output
and the MLP. Tokens come in through `gather_rows` (the embedding) and leave through `row_max_argmax` (the head's logits).
Prompts and single tokens take the same calls: only the batch's token count differs.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from unpopped_b200 import ops  # noqa: E402

GROUP = 128  # of the weights' scales


class Linear:
    """int4 [out, in] weights, two per byte, with an f16 scale a group of 128."""

    def __init__(self, n, k, gen):
        self.w = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        self.scale = torch.full((n, k // GROUP), 0.25 / k ** 0.5, device="cuda").half()

    def __call__(self, x):
        return torch.cat([ops.w4a16(self.w, self.scale, r.contiguous(), GROUP) for r in x.split(16)])  # 16 rows a product


class Model:
    def __init__(self, layers=2, hidden=256, heads=4, kv_heads=2, dim=64, mlp=512, vocab=1024, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.hidden = heads, kv_heads, dim, hidden
        self.embedding = torch.randn(vocab, hidden, generator=gen, device="cuda").bfloat16()
        self.layers = [dict(qkv=Linear((heads + 2 * kv_heads) * dim, hidden, gen), o=Linear(hidden, heads * dim, gen),
                            up=Linear(2 * mlp, hidden, gen), down=Linear(hidden, mlp, gen)) for _ in range(layers)]
        self.head = Linear(vocab, hidden, gen)
        self.rotation = ops.rope_table(4096, dim, scaling=("wavelength", 8.0, 1.0, 4.0, 512))


class Sequences:
    """The cache's pages and what each sequence holds of them; one cache a layer, the same pages in each."""

    def __init__(self, model, batch, pages=64, page=16):
        self.page = page
        self.caches = [ops.kv4_cache(pages, model.kv_heads, model.dim, page) for _ in model.layers]
        self.free = list(range(pages))
        self.pages = [[] for _ in range(batch)]
        self.lens = [0] * batch

    def extend(self, counts):
        """Room for counts[b] more tokens of sequence b: their slots and positions, and where each sequence's begin."""
        slots, positions, starts = [], [], [0]
        for b, n in enumerate(counts):
            while len(self.pages[b]) * self.page < self.lens[b] + n:
                self.pages[b].append(self.free.pop())
            for t in range(self.lens[b], self.lens[b] + n):
                slots.append(self.pages[b][t // self.page] * self.page + t % self.page)
                positions.append(t)
            self.lens[b] += n
            starts.append(starts[-1] + n)
        width = max(len(p) for p in self.pages)
        table = [p + [0] * (width - len(p)) for p in self.pages]
        on = dict(device="cuda", dtype=torch.int32)
        return (torch.tensor(slots, **on), torch.tensor(positions, **on), torch.tensor(starts, **on),
                torch.tensor(table, **on), torch.tensor(self.lens, **on))


def norm(x):
    return ops.row_reduce(x.float(), "rms_norm", eps=1e-5).bfloat16()


def step(model, sequences, tokens):
    """Feeds tokens[b] (a list) to each sequence b; the logits after each sequence's last one."""
    counts = [len(t) for t in tokens]
    slots, positions, starts, table, lens = sequences.extend(counts)
    ids = torch.tensor([t for s in tokens for t in s], device="cuda", dtype=torch.int32)
    x = ops.gather_rows(model.embedding, ids, "zero_fill")
    h, kv, d = model.heads, model.kv_heads, model.dim
    for layer, cache in zip(model.layers, sequences.caches):
        qkv = layer["qkv"](norm(x)).view(-1, h + 2 * kv, d)
        q = ops.kv4_append(qkv[:, h:h + kv], qkv[:, h + kv:], cache, slots, positions, model.rotation, q=qkv[:, :h])
        a = ops.kv4_attention(q, cache, table, lens, cu_q=starts)
        x = x + layer["o"](a.flatten(1))
        gate, up = layer["up"](norm(x)).chunk(2, dim=1)
        x = x + layer["down"]((torch.nn.functional.silu(gate) * up).contiguous())
    last = starts[1:].long() - 1
    return model.head(norm(x[last]))


def generate(model, prompts, steps):
    """Greedy continuations of the prompts, `steps` tokens each."""
    sequences = Sequences(model, len(prompts))
    feed, out = prompts, [[] for _ in prompts]
    for _ in range(steps):
        best = ops.row_max_argmax(step(model, sequences, feed), want_max=False)[1].tolist()
        feed = [[t] for t in best]
        for o, t in zip(out, best):
            o.append(t)
    return out


def main():
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 1024, (n,), generator=gen).tolist() for n in (1, 7, 40, 19)]
    for prompt, tokens in zip(prompts, generate(Model(), prompts, 12)):
        print(f"{len(prompt):3d} prompt tokens -> {tokens}")
    ops.check_workspace("kv4", torch.device("cuda", torch.cuda.current_device()))


if __name__ == "__main__":
    main()
