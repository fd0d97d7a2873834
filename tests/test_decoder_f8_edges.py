"""Edges of the decoder layer's positions, 8-bit floats and experts that need no
GPU: what is refused at the last size that a launch cannot take."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

from spinnv2_amd import build, decoder

from .test_decoder import UNSUPPORTED, Fake, _cache, _refused
from .test_decoder import test_cache_refuses_what_does_not_fit as cache_refusals
from .test_decoder_f8 import F8, _rows
from .test_decoder_f8 import Fake as FakeF8


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


@pytest.fixture
def no_calls(monkeypatch, tmp_path):
    """An interpreter that the native calls were not built for."""
    monkeypatch.setattr(build, "CALLS", tmp_path / "calls.so")
    monkeypatch.setattr(decoder, "_calls", None)


def test_the_cache_needs_the_library_alone(no_calls):
    cache, x, none = _cache(), Fake((0, 2, 64), "bfloat16"), Fake((0,), "int64")
    cache.write(x, x, none)
    cache.read(Fake((3, 5), "int32"), None, Fake((4,), "int32"), x, x)
    cache.read(Fake((3, 5), "int32"), Fake((3,), "int32"), Fake((4,), "int32"), x, x)
    cache_refusals()
    assert decoder._calls is None
    with pytest.raises(RuntimeError):  # the calls that came with the module
        decoder.quantize_f8(Fake((0, 300), "float32"), FakeF8((0, 300), F8), Fake((0, 3), "float32"))


def test_builds_without_a_host_compiler_of_its_own(no_calls, monkeypatch):
    monkeypatch.delenv("CXX", raising=False)
    monkeypatch.setattr(build.shutil, "which", lambda name: None)
    assert build.build_calls() == build.CALLS and build.CALLS.exists()
    x = Fake((0, 2, 64), "bfloat16")
    _cache().write(x, x, Fake((0,), "int64"))
    assert decoder._calls is not None


def test_builds_without_the_interpreters_headers(no_calls, monkeypatch, tmp_path, capsys):
    monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    build.CALLS.write_bytes(b"of another header")
    assert build.build_calls() is None and not build.CALLS.exists()
    assert "Python.h" in capsys.readouterr().err
