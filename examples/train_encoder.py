"""Trains a small text encoder, encodes a corpus with it and searches the corpus: the encoder's operators
and the index together.

A passage is a bag of token ids drawn from its topic's words and common ones; a query is a few tokens of
one passage.  Both become vectors by the same path,

    embedding (scaled rows, padded batches)  ->  layer norm  ->  mean over the tokens  ->  projection

(with ``--layers N``, N transformer layers before that layer norm: attention over each passage's tokens,
turned by their positions, and a gated feed-forward block), which is trained so that a query is nearest to its passage within the batch: the table's gradient is
summed by ordered tokens, the table's optimizer keeps its moments in 8 bits, the small tensors' in 32.
The corpus is then encoded with the projection in 8-bit floating point, indexed (TridentV4Index) and
searched exactly, as are single queries.

    python examples/train_encoder.py [--steps 200] [--passages 20000] ...
"""
import argparse
import math
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from trident_amd import SharedClusterStorage, TridentV4Index, choose_tile, encoder, train_clustering  # noqa: E402

PAD = -1  # an empty slot of a padded batch


def make_corpus(passages, vocab, length, g, device):
    """Token ids [passages, length], -1 past each passage's end: three quarters of a passage's words are
    of its topic (64 of them), the others any, frequent ones first."""
    topics = max(8, passages // 64)
    words = torch.randint(0, vocab, (topics, 64), generator=g, device=device)
    topic = torch.randint(0, topics, (passages, 1), generator=g, device=device)
    own = words[topic, torch.randint(0, 64, (passages, length), generator=g, device=device)]
    u = torch.rand((passages, length), generator=g, device=device)
    common = (torch.exp(u * math.log(vocab + 1)).long() - 1).clamp(0, vocab - 1)
    ids = torch.where(torch.rand((passages, length), generator=g, device=device) < 0.75, own, common)
    lengths = torch.randint(length // 2, length + 1, (passages, 1), generator=g, device=device)
    ids[torch.arange(length, device=device)[None, :] >= lengths] = PAD
    return ids, lengths[:, 0]


def make_queries(ids, lengths, rows, tokens, g):
    """A few tokens of each of the passages `rows`."""
    at = (torch.rand((rows.numel(), tokens), generator=g, device=ids.device) * lengths[rows][:, None]).long()
    return ids[rows][torch.arange(rows.numel(), device=ids.device)[:, None], at]


class Layer:
    """Attention and a gated feed-forward block, each on the layer norm of what it adds to."""

    def __init__(self, dim, heads, g, device):
        rand = lambda *s: (torch.randn(s, generator=g, device=device) / math.sqrt(s[-1])).requires_grad_()  # noqa: E731
        self.heads, self.head_dim = heads, dim // heads
        self.norms = [torch.ones(dim, device=device).requires_grad_() for _ in range(2)]
        self.qkv, self.mix = rand(3 * dim, dim), rand(dim, dim)
        self.gate, self.up, self.down = rand(2 * dim, dim), rand(2 * dim, dim), rand(dim, 2 * dim)
        self.frequencies = encoder.rotary_frequencies(self.head_dim, device=device)

    def parameters(self):
        return [*self.norms, self.qkv, self.mix, self.gate, self.up, self.down]

    def __call__(self, x, lengths):
        B, L, dim = x.shape
        qkv = (encoder.layer_norm(x, self.norms[0]) @ self.qkv.t()).view(B, L, 3 * self.heads, self.head_dim)
        turned = encoder.rotary(qkv[:, :, :2 * self.heads], self.frequencies)  # queries and keys
        q, k, v = turned[:, :, :self.heads], turned[:, :, self.heads:], qkv[:, :, 2 * self.heads:]
        x = x + encoder.attention(q, k, v, lengths=lengths).reshape(B, L, dim) @ self.mix.t()
        return x + encoder.gated_linear(encoder.layer_norm(x, self.norms[1]), self.gate, self.up) @ self.down.t()


class TextEncoder:
    def __init__(self, vocab, dim, out, g, device, layers=0, heads=4):
        rand = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
        self.scale = math.sqrt(dim)
        self.table = (rand(vocab, dim) / self.scale).requires_grad_()
        self.gamma = torch.ones(dim, device=device).requires_grad_()
        self.beta = torch.zeros(dim, device=device).requires_grad_()
        self.weight = (rand(out, dim) / self.scale).requires_grad_()
        self.bias = torch.zeros(out, device=device).requires_grad_()
        self.layers = [Layer(dim, heads, g, device) for _ in range(layers)]
        self.optimizers = [encoder.AdamW([self.table], lr=3e-3, weight_decay=0.0, state_bits=8),
                           encoder.AdamW([self.gamma, self.beta, self.weight, self.bias], lr=3e-3)]
        if layers:
            self.optimizers.append(encoder.AdamW([p for layer in self.layers for p in layer.parameters()], lr=1e-3))

    def pooled(self, ids):
        x = encoder.embedding(ids, self.table, scale=self.scale)
        lengths = (ids >= 0).sum(1) if self.layers else None
        for layer in self.layers:
            x = layer(x, lengths)
        x = encoder.layer_norm(x, self.gamma, self.beta)
        live = (ids >= 0).unsqueeze(-1).float()
        return (x * live).sum(1) / live.sum(1).clamp(min=1.0)

    def train_step(self, queries, passages, temperature=0.05):
        """One step on a batch of (query, passage) pairs; the other passages of the batch are the wrong ones."""
        q, p = (torch.nn.functional.normalize(self.pooled(i) @ self.weight.t() + self.bias, dim=1)
                for i in (queries, passages))
        loss = torch.nn.functional.cross_entropy(q @ p.t() / temperature, torch.arange(len(q), device=q.device))
        loss.backward()
        for opt in self.optimizers:
            opt.step()
            opt.zero_grad()
        return loss.detach()

    def freeze(self):
        """The projection for serving: 8-bit floating point."""
        self.weight8 = encoder.quantize_fp8(self.weight.detach())

    @torch.no_grad()
    def encode(self, ids):
        z = encoder.fp8_linear(self.pooled(ids), self.weight8, self.bias)
        return torch.nn.functional.normalize(z, dim=1)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--vocab", type=int, default=32768)
    ap.add_argument("--dim", type=int, default=256, help="columns of the table")
    ap.add_argument("--out", type=int, default=128, help="dimensions of the vectors")
    ap.add_argument("--layers", type=int, default=0, help="transformer layers between the table and the mean")
    ap.add_argument("--heads", type=int, default=4, help="attention heads of a layer: dim / heads a multiple of 8 up to 128")
    ap.add_argument("--passages", type=int, default=20000)
    ap.add_argument("--length", type=int, default=64, help="tokens of a passage at most")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--batch", type=int, default=512)
    ap.add_argument("--nlist", type=int, default=128)
    ap.add_argument("--nprobe", type=int, default=16)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    device = torch.device("cuda:0")
    g = torch.Generator(device=device).manual_seed(a.seed)
    ids, lengths = make_corpus(a.passages, a.vocab, a.length, g, device)
    model = TextEncoder(a.vocab, a.dim, a.out, g, device, a.layers, a.heads)

    losses, began = [], time.perf_counter()
    for step in range(a.steps):
        rows = torch.randint(0, a.passages, (a.batch,), generator=g, device=device)
        losses.append(model.train_step(make_queries(ids, lengths, rows, 8, g), ids[rows]))
    losses = torch.stack(losses).cpu()
    print(f"{a.steps} steps of {a.batch} pairs in {time.perf_counter() - began:.2f} s: "
          f"loss {losses[:10].mean():.3f} -> {losses[-10:].mean():.3f}")

    model.freeze()
    vectors = torch.cat([model.encode(ids[s:s + 4096]) for s in range(0, a.passages, 4096)])
    centroids, list_ids, r, mean64, R64, _ = train_clustering(vectors.cpu(), a.nlist, seed=a.seed, niter=6)
    storage = SharedClusterStorage(vectors.cpu().numpy(), list_ids, r, a.nlist, device=device)
    index = TridentV4Index(storage, centroids, mean64, R64, tile_size=choose_tile(a.out), device=device,
                           max_batch=1024, max_nprobe=a.nprobe, k=10)

    rows = torch.randint(0, a.passages, (1000,), generator=g, device=device)
    q = model.encode(make_queries(ids, lengths, rows, 8, g))
    found = index.search(q, a.nprobe)[1].clone()
    hits = (found == rows[:, None]).any(1).float().mean().item()
    exact = torch.cdist(q, vectors).topk(10, largest=False).indices
    recall = np.mean([len(set(x) & set(y)) / 10 for x, y in zip(found.tolist(), exact.tolist())])
    one = model.encode(make_queries(ids, lengths, rows[:1], 8, g))  # a single query: the same path
    print(f"1000 queries over {a.passages} passages: the right one among the first ten for {100 * hits:.1f}%; "
          f"{100 * recall:.1f}% of the exhaustive first ten at nprobe {a.nprobe}; "
          f"one query's nearest: {index.search(one, a.nprobe)[1][0, 0].item()} (drawn from {rows[0].item()})")
    return dict(first=float(losses[:10].mean()), last=float(losses[-10:].mean()), hits=hits, recall=float(recall))


if __name__ == "__main__":
    main()
