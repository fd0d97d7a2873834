"""Edges of the decoder layer's positions, 8-bit floats and experts that need no
GPU: what is refused at the last size that a launch cannot take."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

from .test_decoder import UNSUPPORTED, _refused
from .test_decoder_f8 import _rows


@pytest.mark.parametrize("kind", [0, 2])
@pytest.mark.parametrize("rows,cols", [((1 << 28) - 1, 1), ((1 << 28) - 15, 128), ((1 << 27) - 7, 129)])
def test_blocks_are_refused_from_2_to_the_32_threads_on(kind, rows, cols):
    """Sixteen blocks are a workgroup of 256 threads, so 2^28 - 15 of them are 2^24 workgroups, 2^32 threads along one axis."""
    blocks = -(-cols // 128)
    _refused("rows", _rows(kind=kind, rows=rows, cols=cols, x_stride=2 * cols, q_stride=cols, scale_stride=blocks), UNSUPPORTED)


def test_inline_assembly_names_the_registers_that_it_writes():
    """m0, which the compiler has uses of its own for, and which no operand stands for."""
    kernels = Path(__file__).resolve().parent.parent / "spinnv2_amd" / "csrc" / "kernels"
    statements = [s for f in sorted(kernels.glob("*.h*")) for s in re.findall(r"asm volatile\((.*?)\);", f.read_text(), re.S)]
    writers = [s for s in statements if "s_mov_b32 m0" in s]
    assert writers and all('"m0"' in s.rsplit(":", 1)[1] for s in writers)
