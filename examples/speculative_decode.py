"""Train a small decoder, then generate with it from draft trees.

The model (two layers, grouped key heads, normed and rotated queries and keys) learns a
fixed successor of every token.  Training runs `qk_norm_rope` and its gradient; generation
runs `qkv_to_cache`, `tree_attention`, `verify_drafts` and `KVCache.keep_path`: each pass
takes a tree of guesses of a table that only knows the last token, and keeps the longest
path that the model agrees with.

    python examples/speculative_decode.py [--format int8] [--temperature 0.0]
"""
from __future__ import annotations

import argparse
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "ojasx-open-source-cuda-_b200"))
from torchcl import serving  # noqa: E402

VOCAB, WIDTH, LAYERS, Q_HEADS, KV_HEADS, DIM = 256, 256, 2, 8, 2, 64
PAGE, LONGEST = 16, 512
# Draft tree: three guesses after the last token, two after each of those, one after each of these.
PARENTS = [-1, 0, 0, 0, 1, 1, 2, 2, 3, 3, 4, 5, 6, 7, 8, 9]


class Decoder(torch.nn.Module):
    def __init__(self, seed: int = 0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        new = lambda *shape: torch.nn.Parameter(torch.randn(*shape, generator=g) * shape[0] ** -0.5)  # noqa: E731
        self.embed, self.head = torch.nn.Parameter(torch.randn(VOCAB, WIDTH, generator=g)), new(WIDTH, VOCAB)
        self.qkv = torch.nn.ParameterList(new(WIDTH, (Q_HEADS + 2 * KV_HEADS) * DIM) for _ in range(LAYERS))
        self.out = torch.nn.ParameterList(new(Q_HEADS * DIM, WIDTH) for _ in range(LAYERS))
        self.q_norm = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(DIM)) for _ in range(LAYERS))
        self.k_norm = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(DIM)) for _ in range(LAYERS))
        self.register_buffer("table", serving.rope_table(LONGEST, DIM))

    def project(self, x, layer: int):
        """Query, key and value heads of [tokens, WIDTH] rows."""
        qkv = (x @ self.qkv[layer]).view(x.shape[0], -1, DIM)
        return qkv.split([Q_HEADS, KV_HEADS, KV_HEADS], dim=1)

    def forward(self, tokens):
        """Logits of whole sequences [batch, length], for training."""
        batch, length = tokens.shape
        positions = torch.arange(length, dtype=torch.int32, device=tokens.device).repeat(batch)
        x = self.embed[tokens.reshape(-1)]
        for layer in range(LAYERS):
            q, k, v = self.project(x, layer)
            q, k = serving.qk_norm_rope(q, k, self.q_norm[layer], self.k_norm[layer], self.table, positions)
            heads = [t.view(batch, length, -1, DIM).transpose(1, 2) for t in (q, k, v)]
            y = torch.nn.functional.scaled_dot_product_attention(*heads, is_causal=True, enable_gqa=True)
            x = x + y.transpose(1, 2).reshape(batch * length, -1) @ self.out[layer]
        return (x @ self.head).view(batch, length, VOCAB)


def train(model: Decoder, successor, steps: int = 60, batch: int = 16, length: int = 64, seed: int = 1):
    """Losses of `steps` steps on chains of successors."""
    g = torch.Generator().manual_seed(seed)
    device = model.embed.device
    optimiser = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        chain = [torch.randint(VOCAB, (batch,), generator=g).to(device)]
        for _ in range(length):
            chain.append(successor[chain[-1]])
        tokens = torch.stack(chain, dim=1)
        loss = torch.nn.functional.cross_entropy(model(tokens[:, :-1]).reshape(-1, VOCAB), tokens[:, 1:].reshape(-1))
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(loss.item())
    return losses


class Generator:
    """Sequences that grow together over one paged cache per layer."""

    def __init__(self, model: Decoder, batch: int, format: str = "float16"):
        self.model, self.batch, device = model, batch, model.embed.device
        pages = LONGEST // PAGE
        self.caches = [serving.KVCache(batch * pages, PAGE, KV_HEADS, DIM, format) for _ in range(LAYERS)]
        # any order of pages will do
        order = torch.randperm(batch * pages, generator=torch.Generator().manual_seed(2), dtype=torch.int32)
        self.pages = order.view(batch, pages).to(device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.fused = torch.float16

    def logits(self, tokens, depths, mask=None):
        """Logits [batch, nodes, VOCAB] of new tokens, whose keys and values go behind the context."""
        model, nodes = self.model, tokens.shape[1]
        place = (self.lens[:, None] + torch.arange(nodes, device=tokens.device)).long()
        slots = (self.pages.gather(1, place // PAGE) * PAGE + place % PAGE).int().reshape(-1)
        positions = (self.lens[:, None] + depths).int().reshape(-1)
        x = model.embed[tokens.reshape(-1)]
        for layer, cache in enumerate(self.caches):
            q, k, v = (t.to(self.fused) for t in model.project(x, layer))
            q = serving.qkv_to_cache(q, k, v, model.q_norm[layer], model.k_norm[layer], model.table, positions, cache, slots)
            y = serving.tree_attention(q.view(self.batch, nodes, Q_HEADS, DIM), cache, self.pages, self.lens, mask)
            x = x + y.reshape(self.batch * nodes, -1).float() @ model.out[layer]
        return (x @ model.head).view(self.batch, nodes, VOCAB)

    @torch.no_grad()
    def generate(self, prompts, new_tokens: int, temperature: float = 0.0, drafts: bool = True, seed: int = 3):
        """(tokens per sequence after its prompt, passes over the model)."""
        device = prompts.device
        parents = PARENTS if drafts else PARENTS[:1]
        depths = [0] * len(parents)
        for i, p in enumerate(parents):
            depths[i] = depths[p] + 1 if p >= 0 else 0
        depth = torch.tensor(depths, device=device)
        mask = serving.tree_mask(torch.tensor(parents)).to(device)
        parent = torch.tensor(parents, dtype=torch.int32, device=device).repeat(self.batch, 1)
        guesses = (self.model.embed @ self.model.head).topk(3).indices  # of the last token alone
        g = torch.Generator().manual_seed(seed)

        self.logits(prompts[:, :-1], torch.arange(prompts.shape[1] - 1, device=device))
        self.lens += prompts.shape[1] - 1
        root, out, passes = prompts[:, -1], [[] for _ in range(self.batch)], 0
        while min(map(len, out)) < new_tokens:
            columns, taken = [root], [0] * len(parents)
            for p in parents[1:]:
                columns.append(guesses[columns[p], taken[p]])
                taken[p] += 1
            tokens = torch.stack(columns, dim=1)
            logits = self.logits(tokens, depth, mask)
            if temperature == 0.0:
                probs = torch.zeros_like(logits).scatter_(2, logits.argmax(2, keepdim=True), 1.0)
            else:
                probs = (logits / temperature).softmax(2)
            uniforms = torch.rand(self.batch, len(parents), generator=g).to(device)
            path, count, following = serving.verify_drafts(probs, tokens.int(), parent, uniforms)
            for cache in self.caches:
                cache.keep_path(self.pages, self.lens, path, count)
            self.lens += 1 + count
            root = following.long()
            passes += 1
            for b, (nodes, n, last) in enumerate(zip(path.tolist(), count.tolist(), following.tolist())):
                out[b] += [int(tokens[b, i]) for i in nodes[1:n + 1]] + [last]
        return [o[:new_tokens] for o in out], passes


def main(format: str = "float16", temperature: float = 0.0, new_tokens: int = 64, batch: int = 4) -> dict:
    successor = torch.randperm(VOCAB, generator=torch.Generator().manual_seed(4)).cuda()
    model = Decoder().cuda()
    losses = train(model, successor)
    prompts = torch.randint(VOCAB, (batch, 21), generator=torch.Generator().manual_seed(5)).cuda()
    out, passes = Generator(model, batch, format).generate(prompts, new_tokens, temperature)
    plain, plain_passes = Generator(model, batch, format).generate(prompts, new_tokens, temperature, drafts=False)
    torch.cuda.synchronize()
    return {"model": model, "losses": losses, "prompts": prompts, "tokens": out, "passes": passes,
            "plain": plain, "plain_passes": plain_passes}


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--format", default="float16", choices=["float16", "int8", "float8"])
    parser.add_argument("--temperature", type=float, default=0.0)
    args = parser.parse_args()
    r = main(args.format, args.temperature)
    print(f"loss {r['losses'][0]:.3f} -> {r['losses'][-1]:.3f}; 64 tokens of 4 sequences in {r['passes']} passes with draft "
          f"trees, {r['plain_passes']} without")
