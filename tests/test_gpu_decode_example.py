"""The example decoder: a prompt read at once and token by token gives the
same logits, and both those of the layers computed in 64 bits from the same
codes."""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

pytestmark = pytest.mark.gpu


def _reference(model, tokens):
    """The model in 64 bits with its weights' codes, without rounding activations to 8 bits."""
    s = model.sizes
    x = model.embedding[tokens].astype(np.float64)

    def norm(x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * w.download().astype(np.float64)

    def product(x, w):
        return x @ (w.codes.download().astype(np.float64) * w.scale.download()[:, None]).T

    n = len(tokens)
    mask = np.tril(np.ones((n, n), bool))
    for layer in range(s.layers):
        y = product(norm(x, model.norms[layer]), model.inward[layer]).reshape(n, -1, s.dim)
        q, k, v = y[:, :s.heads], y[:, s.heads:s.heads + s.kv_heads], y[:, s.heads + s.kv_heads:]
        out = np.zeros((n, s.heads, s.dim))
        for h in range(s.heads):
            j = h // (s.heads // s.kv_heads)
            p = np.where(mask, q[:, h] @ k[:, j].T * s.dim ** -0.5, -np.inf)
            p = np.exp(p - p.max(1, keepdims=True))
            out[:, h] = p @ v[:, j] / p.sum(1, keepdims=True)
        x = x + product(out.reshape(n, -1), model.outward[layer])
    return product(norm(x, model.norms[-1]), model.head)


def test_prompt_and_single_tokens_agree(gpu):
    from decode_i8 import Decoder, Sizes

    sizes = Sizes(layers=2)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, sizes.vocabulary, n) for n in (37, 5, 90)]
    whole, step = Decoder(sizes, 3, 100), Decoder(sizes, 3, 100)
    at_once = whole.forward(prompts)
    step.forward([p[:3] for p in prompts])
    for i in range(3, 90):
        # sequences that have ended go on with any token: only the longest is compared to its end
        single = step.forward([np.array([p[i] if i < len(p) else 0]) for p in prompts])
        for j, p in enumerate(prompts):
            if i == len(p) - 1:
                want = _reference(whole, p)[-1]
                size = np.abs(want).max()
                # 8-bit rows: a product's inputs are off by up to 1 / 254 of their row's largest value, about
                # 3 / 254 of their root mean square, at random; five such roundings lie between tokens and logits
                for got in (at_once[j], single[j]):
                    rms = np.sqrt(np.mean((got - want) ** 2) / np.mean(want ** 2))
                    assert rms < 5 * 3 / 254, (j, rms)
                assert np.abs(at_once[j] - single[j]).max() < 0.1 * size


def test_example_refuses_more_tokens_than_pages(gpu):
    from decode_i8 import Decoder, Sizes

    model = Decoder(Sizes(layers=1), 1, 16)
    with pytest.raises(ValueError):
        model.forward([np.zeros(17, np.int64)])
