"""From a search to a reader's decoding steps, all of it in 4 bits.

A MaxSim search finds passages for a batch of queries; one attention layer of a
reader takes the passages' tokens into its key/value cache and decodes a few
tokens over them: projections by ``Int4Linear``, keys and values into
``Int4KVCache``, attention over it.  Synthetic corpus, random weights; the passages'
token embeddings stand for the hidden states that a reader's lower layers would make
of their text.

    python examples/answer_step.py
"""
from __future__ import annotations

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import maxsim_amd as maxsim  # noqa: E402
from maxsim_amd import synthetic  # noqa: E402

WIDTH, HEADS, KV_HEADS, HEAD_DIM = 128, 8, 2, 64


class ReaderLayer:
    """An attention layer with 4-bit projections and a 4-bit cache."""

    def __init__(self, tokens: int, batch: int, page_size: int = 16, seed: int = 0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)

        def matrix(out, width):
            return torch.randn((out, width), generator=g, device="cuda") / width**0.5

        self.weights = {"q": matrix(HEADS * HEAD_DIM, WIDTH), "k": matrix(KV_HEADS * HEAD_DIM, WIDTH),
                        "v": matrix(KV_HEADS * HEAD_DIM, WIDTH), "o": matrix(WIDTH, HEADS * HEAD_DIM)}
        self.linear = {name: maxsim.Int4Linear.from_float(w, group_size=32) for name, w in self.weights.items()}
        pages = -(-tokens // page_size)  # of a sequence, at most
        self.cache = maxsim.Int4KVCache(batch * pages, KV_HEADS, HEAD_DIM, page_size=page_size)
        self.table = torch.arange(batch * pages, dtype=torch.int32, device="cuda").view(batch, pages)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def __call__(self, x, offsets=None):
        """New tokens x [rows, WIDTH] of every sequence (offsets; without: one each)
        attend to what the cache holds and to themselves."""
        self.lengths += 1 if offsets is None else offsets[1:] - offsets[:-1]
        q = self.linear["q"](x).view(-1, HEADS, HEAD_DIM)
        k = self.linear["k"](x).view(-1, KV_HEADS, HEAD_DIM)
        v = self.linear["v"](x).view(-1, KV_HEADS, HEAD_DIM)
        self.cache.append(k, v, self.table, self.lengths, offsets)
        out = self.cache.attend(q, self.table, self.lengths, offsets)
        return self.linear["o"](out.view(-1, HEADS * HEAD_DIM))


def plain_layer(weights, sequence):
    """The same layer on one whole sequence [tokens, WIDTH], unquantised."""
    q, k, v = (sequence @ weights[name].t() for name in "qkv")
    q = q.view(-1, HEADS, HEAD_DIM).transpose(0, 1)
    k, v = (t.view(-1, KV_HEADS, HEAD_DIM).transpose(0, 1).repeat_interleave(HEADS // KV_HEADS, 0) for t in (k, v))
    s = q @ k.transpose(1, 2).contiguous() / HEAD_DIM**0.5
    s = s.masked_fill(torch.ones(s.shape[1:], dtype=torch.bool, device=s.device).triu(1), -torch.inf)
    out = torch.softmax(s, -1) @ v
    return out.transpose(0, 1).reshape(-1, HEADS * HEAD_DIM) @ weights["o"].t()


def main(num_docs: int = 512, batch: int = 4, k: int = 3, steps: int = 8):
    """Cosine similarity of the 4-bit layer's outputs to the unquantised layer's,
    over the passages and the decoded tokens."""
    corpus = synthetic.make_corpus(num_docs, 32, 64, dim=WIDTH)
    queries = synthetic.make_queries(corpus, batch)
    index = maxsim.Index.from_embeddings([f"doc{i}" for i in range(num_docs)], corpus.embeddings, corpus.offsets)
    found = maxsim.Reranker(index).search(queries, k=k)

    # The passages of each query, one after the other.
    rows = [np.concatenate([np.arange(*corpus.offsets[d:d + 2]) for d in (int(hit.doc_id[3:]) for hit in hits)])
            for hits in found]
    sequences = [torch.from_numpy(corpus.embeddings[r]).cuda() * WIDTH**0.5 for r in rows]
    offsets = torch.tensor(np.cumsum([0] + [len(r) for r in rows]), dtype=torch.int32, device="cuda")
    layer = ReaderLayer(max(len(r) for r in rows) + steps, batch)
    outputs = [list(part) for part in layer(torch.cat(sequences), offsets).split([len(r) for r in rows])]

    # Decoding: each sequence's next token is made of its last output.
    for _ in range(steps):
        x = torch.stack([out[-1] for out in outputs])
        x = x / x.norm(dim=-1, keepdim=True) * WIDTH**0.5
        y = layer(x)
        for b in range(batch):
            sequences[b] = torch.cat((sequences[b], x[b:b + 1]))
            outputs[b].append(y[b])
    got = torch.cat([torch.stack(out) for out in outputs])
    plain = torch.cat([plain_layer(layer.weights, s) for s in sequences])
    similarity = torch.nn.functional.cosine_similarity(got, plain, dim=-1)
    print(f"{got.shape[0]} tokens of {batch} sequences: cosine to the unquantised layer "
          f"mean {similarity.mean():.4f}, least {similarity.min():.4f}")
    return similarity


if __name__ == "__main__":
    main()
