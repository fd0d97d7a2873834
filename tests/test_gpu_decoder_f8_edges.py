"""Edges of the decoder layer's positions, 8-bit floats and experts, against their
formulas in 64 bits; tolerances as in test_gpu_decoder_f8."""

from __future__ import annotations

import numpy as np
import pytest

from spinnv2_amd import decoder
from spinnv2_amd.decoder import DeviceArray as Array

from .test_gpu_decoder import rounded
from .test_gpu_decoder_f8 import F8, coded

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ 8-bit floats

def _gate(x, dtype):
    """(codes' values, scales) of gate_f8 for x [rows, 2 cols], and the values in 64 bits."""
    rows, cols = x.shape[0], x.shape[1] // 2
    q, s = Array((rows, cols), F8), Array((rows, -(-cols // 128)), "float32")
    decoder.gate_f8(Array.of(x, dtype), q, s)
    with np.errstate(over="ignore", invalid="ignore"):
        v = x[:, :cols] / (1 + np.exp(-x[:, :cols])) * x[:, cols:]
    return q.download(), s.download(), v


@pytest.mark.parametrize("dtype,least", [("float32", 2.0 ** -149), ("bfloat16", 2.0 ** -133)])
@pytest.mark.parametrize("factor", [2.0 ** 66, 2.0 ** 100, 2.0 ** 123])
def test_gates_below_fp32s_normal_values(gpu, factor, dtype, least):
    """Gates whose half is subnormal, with factors that make it a block's largest, alone and beside ordinary gates."""
    rng = np.random.default_rng(41)
    t = rng.integers(1, 60, (8, 256)) * least
    t[2:4] = rng.uniform(0.5, 8.0, (2, 256)) * 2.0 ** -126  # around the smallest normal value
    u = rng.uniform(1.0, 2.0, t.shape) * factor
    some = rng.random((4, 256)) < 0.5
    u[4:] = np.where(some, rng.uniform(1.0, 8.0, (4, 256)), u[4:])
    t[4:] = np.where(some, rng.uniform(1.0, 8.0, (4, 256)) * least * factor, t[4:])
    t[6, :128] = 0.0
    x = rounded(np.concatenate([t * rng.choice([-1.0, 1.0], t.shape), u * rng.choice([-1.0, 1.0], t.shape)], 1), dtype)
    got, scale, v = _gate(x, dtype)
    want, want_scale = coded(v)
    np.testing.assert_array_equal(got, want)
    np.testing.assert_allclose(scale, want_scale, rtol=2.0 ** -20.5, atol=2.0 ** -149)
