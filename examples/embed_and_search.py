"""Passages and queries as token ids -> vectors -> neighbours, on one GPU.

A small text encoder (random weights: there is nothing to download) built from beam_search_collab_amd.embed
turns packed sequences of token ids into one float32 vector each, the last token's row after the last norm,
projected and normalised.  The passages' vectors become a Vamana graph; the queries' vectors go from the
projection to the search on the same stream, without leaving the GPU.  At the end the last norm is tuned for a
few steps with layer_norm_backward, so that each query moves closer to its passage.

    python examples/embed_and_search.py [--passages 4000] [--queries 64] [--dim 128]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from beam_search_collab_amd import GPUBaseSearchCfg, GPUGraph, embed  # noqa: E402
from beam_search_collab_amd.search import build_vamana_device  # noqa: E402


class Encoder:
    """`layers` blocks of causal attention (grouped heads) and a gelu product; bf16 weights"""

    def __init__(self, vocabulary=1000, width=256, heads=8, kv_heads=2, layers=2, dim=128, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols):
            return (torch.randn(rows, cols, generator=g, device="cuda") * cols ** -0.5).bfloat16()

        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, width // heads
        self.tokens = torch.randn(vocabulary, width, generator=g, device="cuda").bfloat16()
        both = (heads + 2 * kv_heads) * self.head_dim
        self.blocks = [dict(qkv=weight(both, width), mix=weight(width, width), up=weight(4 * width, width),
                            down=weight(width, 4 * width), n1=torch.ones(width, device="cuda"), n2=torch.ones(width, device="cuda"))
                       for _ in range(layers)]
        self.norm, self.shift = torch.ones(width, device="cuda"), torch.zeros(width, device="cuda")
        self.project = weight(dim, width)

    def last_rows(self, ids, offsets, longest):
        """the residual stream of every sequence's last token"""
        x = self.tokens[ids]
        h, kv, d = self.heads, self.kv_heads, self.head_dim
        for b in self.blocks:
            qkv = embed.linear(embed.layer_norm(x, b["n1"]), b["qkv"]).unflatten(1, (h + 2 * kv, d))
            o = embed.attention(qkv[:, :h], qkv[:, h:h + kv], qkv[:, h + kv:], offsets, longest_q=longest, longest_k=longest)
            x = embed.linear(o.flatten(1), b["mix"], residual=x)
            y = embed.linear(embed.layer_norm(x, b["n2"]), b["up"], activation="gelu")
            x = embed.linear(y, b["down"], residual=x)
        return x[offsets[1:].long() - 1]

    def vectors(self, rows):
        """float32, of length 1: what the index holds"""
        z = embed.linear(embed.layer_norm(rows, self.norm, self.shift), self.project, out_dtype=torch.float32)
        return torch.nn.functional.normalize(z, dim=1)


def pack(sequences):
    offsets = np.concatenate([[0], np.cumsum([len(s) for s in sequences])])
    ids = torch.from_numpy(np.concatenate(sequences)).cuda()
    return ids, torch.from_numpy(offsets.astype(np.int32)).cuda(), max(len(s) for s in sequences)


def search(graph, queries, entry, k):
    """queries: float32 on the GPU.  The search runs on the stream that makes them."""
    ids = torch.empty(queries.shape[0], k, dtype=torch.int32, device="cuda")
    graph.search_device(queries.data_ptr(), queries.shape[0], ids.data_ptr(), k, "base", GPUBaseSearchCfg(64, 1024, entry, 1024, 16),
                        stream=torch.cuda.current_stream().cuda_stream)
    return ids


def tune(encoder, rows, targets, steps=20, rate=0.5):
    """Moves the last norm's weight and bias so that the rows' vectors approach `targets`; mean cosine before and after"""
    rows, first = rows.contiguous(), None
    for _ in range(steps):
        y, mean, rstd = embed.layer_norm(rows, encoder.norm, encoder.shift, stats=True)
        z = embed.linear(y, encoder.project, out_dtype=torch.float32)
        length = z.norm(dim=1, keepdim=True)
        unit = z / length
        cosine = (unit * targets).sum(1, keepdim=True)
        first = cosine.mean().item() if first is None else first
        dz = (cosine * unit - targets) / length / len(rows)  # of the mean of 1 - cosine
        dy = embed.linear(dz.bfloat16(), encoder.project.t().contiguous())
        _, dw, db = embed.layer_norm_backward(dy, rows, mean, rstd, encoder.norm)
        encoder.norm -= rate * rows.shape[1] ** 0.5 * dw
        encoder.shift -= rate * rows.shape[1] ** 0.5 * db
    unit = encoder.vectors(rows)
    return first, (unit * targets).sum(1).mean().item()


def main(argv=None):
    a = argparse.ArgumentParser()
    a.add_argument("--passages", type=int, default=4000)
    a.add_argument("--queries", type=int, default=64)
    a.add_argument("--dim", type=int, default=128)
    a = a.parse_args(argv)
    rng = np.random.default_rng(0)
    encoder = Encoder(dim=a.dim)
    passages = [rng.integers(0, 1000, rng.integers(16, 120)) for _ in range(a.passages)]
    picked = rng.choice(a.passages, a.queries, replace=False)
    # a query is the end of its passage with a few tokens changed
    queries = []
    for p in picked:
        q = passages[p][len(passages[p]) // 3:].copy()
        q[rng.integers(0, max(1, len(q) - 4), 2)] = rng.integers(0, 1000, 2)
        queries.append(q)

    vectors = encoder.vectors(encoder.last_rows(*pack(passages)))
    base = vectors.cpu().numpy()
    graph = GPUGraph(base, build_vamana_device(base, degree=32, beam_width=64, alpha=1.2))
    entry = graph.entry_point()
    rows = encoder.last_rows(*pack(queries))
    found = search(graph, encoder.vectors(rows), entry, 10)
    want = torch.from_numpy(graph.groundtruth(encoder.vectors(rows).cpu().numpy(), 10)).cuda()
    recall = (found[:, :, None] == want[:, None, :]).any(2).float().mean().item()
    own = (found == torch.from_numpy(picked).cuda()[:, None]).any(1).float().mean().item()
    before, after = tune(encoder, rows, vectors[torch.from_numpy(picked).cuda()])
    print(f"{a.passages} passages, {a.queries} queries: recall@10 of the search {recall:.3f}, own passage among 10 {own:.3f}, "
          f"cosine to it {before:.3f} -> {after:.3f} after tuning the last norm")
    return recall, own, before, after


if __name__ == "__main__":
    main()
