"""A small decoder in 8 bits on the GPU: prompts, then token by token.

    python examples/decode_i8.py [--layers 4] [--prompt 200] [--tokens 64] [--sequences 3]

Attention-only layers with random weights: norm to int8 rows, one int8 product
for queries, keys and values, the keys and values written into a paged int8
cache, attention to it, an int8 product back into the residual stream; after
the last layer a norm and the product with the vocabulary.  Every call goes
through spinnv2_amd.decoder on DeviceArrays; torch is not needed.  The prompts
run as one batch of all their tokens, then each step runs one token a sequence,
chosen as the largest logit.
"""

from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from spinnv2_amd import decoder  # noqa: E402
from spinnv2_amd.decoder import DeviceArray, KvCache  # noqa: E402


@dataclass
class Sizes:
    layers: int = 4
    heads: int = 8
    kv_heads: int = 2
    dim: int = 64
    vocabulary: int = 1000
    page: int = 16

    @property
    def width(self) -> int:
        return self.heads * self.dim


class Weights:
    """An int8 matrix [out, in] with a scale for each output channel."""

    def __init__(self, rng, out: int, width: int) -> None:
        w = (rng.standard_normal((out, width)) / np.sqrt(width)).astype(np.float32)
        self.codes, self.scale = DeviceArray((out, width), "int8"), DeviceArray((out,), "float32")
        decoder.quantize_i8(DeviceArray.of(w), self.codes, self.scale)


class Decoder:
    """The model, its caches, and the page tables of a fixed number of sequences."""

    def __init__(self, sizes: Sizes, sequences: int, longest: int, seed: int = 0) -> None:
        s, rng = sizes, np.random.default_rng(seed)
        self.sizes, self.sequences, self.longest = s, sequences, longest
        qkv = (s.heads + 2 * s.kv_heads) * s.dim
        self.embedding = rng.standard_normal((s.vocabulary, s.width)).astype(np.float32)
        self.norms = [DeviceArray.of((1 + 0.1 * rng.standard_normal(s.width)).astype(np.float32), "bfloat16") for _ in range(s.layers + 1)]
        self.inward = [Weights(rng, qkv, s.width) for _ in range(s.layers)]
        self.outward = [Weights(rng, s.width, s.width) for _ in range(s.layers)]
        self.head = Weights(rng, s.vocabulary, s.width)
        pages = -(-longest // s.page)
        self.caches = [KvCache.empty(sequences * pages, s.kv_heads, s.page, s.dim) for _ in range(s.layers)]
        # any order of pages will do
        self.table = rng.permutation(sequences * pages).astype(np.int32).reshape(sequences, pages)
        self.device_table = DeviceArray.of(self.table)
        self.lengths = np.zeros(sequences, np.int32)

    def forward(self, tokens: list) -> np.ndarray:
        """Logits after the last of each sequence's new tokens (one array of ids for each sequence, none of them empty)."""
        s = self.sizes
        counts = np.array([len(t) for t in tokens], np.int32)
        if (self.lengths + counts).max() > self.longest:
            raise ValueError("a sequence is longer than its pages")
        place = [np.arange(n, n + c) for n, c in zip(self.lengths, counts)]
        self.lengths = self.lengths + counts
        slots = np.concatenate([self.table[i, p // s.page].astype(np.int64) * s.page + p % s.page for i, p in enumerate(place)])
        offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        total, widest, bound = int(offsets[-1]), int(counts.max()), int(self.lengths.max())
        slots, lengths, device_offsets = DeviceArray.of(slots), DeviceArray.of(self.lengths), DeviceArray.of(offsets)

        stream = DeviceArray.of(self.embedding[np.concatenate(tokens)], "bfloat16")  # the residual stream
        codes, scale = DeviceArray((total, s.width), "int8"), DeviceArray((total,), "float32")
        wide = (s.heads + 2 * s.kv_heads) * s.dim
        qkv = DeviceArray((total, wide), "bfloat16")
        q, k, v = (DeviceArray((total, n, s.dim), "bfloat16", buffer=qkv.buffer, at=at * s.dim, strides=(wide, s.dim, 1))
                   for n, at in ((s.heads, 0), (s.kv_heads, s.heads), (s.kv_heads, s.heads + s.kv_heads)))
        mixed = DeviceArray((total, s.heads, s.dim), "bfloat16")
        rows = DeviceArray((total, s.width), "bfloat16", buffer=mixed.buffer)
        update = DeviceArray((total, s.width), "bfloat16")
        size = decoder.attention_workspace(self.sequences, total, s.heads, self.caches[0], max_queries=widest, max_length=bound)
        workspace = DeviceArray((size,), "int8") if size else None

        for layer, cache in enumerate(self.caches):
            # the layer before's update joins the stream in the norm's pass
            decoder.rmsnorm_i8(stream, self.norms[layer], codes, scale, residual=update if layer else None,
                               residual_out=stream if layer else None)
            w = self.inward[layer]
            decoder.matmul_i8(codes, scale, w.codes, w.scale, qkv)
            cache.write(k, v, slots)
            decoder.attention(q, cache, self.device_table, lengths, device_offsets, mixed, max_queries=widest, max_length=bound,
                              workspace=workspace)
            decoder.quantize_i8(rows, codes, scale)
            w = self.outward[layer]
            decoder.matmul_i8(codes, scale, w.codes, w.scale, update)
        decoder.rmsnorm_i8(stream, self.norms[-1], codes, scale, residual=update, residual_out=stream)
        logits = DeviceArray((total, s.vocabulary), "float32")
        decoder.matmul_i8(codes, scale, self.head.codes, self.head.scale, logits)
        return logits.download()[offsets[1:] - 1]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--sequences", type=int, default=3)
    a = ap.parse_args()
    sizes = Sizes(layers=a.layers)
    model = Decoder(sizes, a.sequences, a.prompt + a.tokens)
    rng = np.random.default_rng(1)
    tokens = [rng.integers(0, sizes.vocabulary, a.prompt - i) for i in range(a.sequences)]  # prompts of different lengths
    began = time.perf_counter()
    logits = model.forward(tokens)
    print(f"{sum(map(len, tokens))} prompt tokens in {(time.perf_counter() - began) * 1e3:.1f} ms")
    text = [[] for _ in range(a.sequences)]
    began = time.perf_counter()
    for _ in range(a.tokens):
        chosen = logits.argmax(1)
        for t, c in zip(text, chosen):
            t.append(int(c))
        logits = model.forward([np.array([c]) for c in chosen])
    print(f"{a.tokens} steps of {a.sequences} sequences in {(time.perf_counter() - began) * 1e3:.1f} ms, transfers and the host's part included")
    for t in text:
        print(*t[:16])


if __name__ == "__main__":
    main()
