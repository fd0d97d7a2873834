"""Edges of the decoder layer's positions, 8-bit floats and experts that need no
GPU: what is refused at the last size that a launch cannot take."""

from __future__ import annotations

import functools
import re
from pathlib import Path

import pytest

from spinnv2_amd import build, decoder

from .test_decoder import UNSUPPORTED, Fake, _cache, _refused
from .test_decoder import test_cache_refuses_what_does_not_fit as cache_refusals
from .test_decoder_f8 import F8, FORMS, _rows, kernel_of
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


# ------------------------------------------------ sizes that take a kernel over several steps of k

#: blocks of k -> k of whole runs of 16 bytes, k of none; the last block is never whole
STEPS = {5: (528, 517), 9: (1040, 1030), 22: (2704, 2701), 70: (8848, 8837)}


@functools.lru_cache(maxsize=None)
def sizes_of_steps(dtype, by_expert):
    """(kernel, blocks of k) -> (m, n, k, experts): the smallest sizes found, none of them a multiple of a tile."""
    found = {}
    for blocks, ks in STEPS.items():
        for k in ks:
            for m in (1, 3, 9, 18, 33, 70, 100, 130, 200, 400, 520, 700, 1030, 1500, 2100, 3000, 4100):
                for n in (17, 33, 65, 100, 130, 190, 260, 390, 515, 770, 1029, 1540, 2050, 3000, 4100, 6200):
                    for experts in ((1, 3, 7, 40) if by_expert else (0,)):
                        if m * n * k > 1.2e10 or max(1, experts) * n * k > 4e7:
                            continue
                        key, size = (kernel_of(dtype, m, n, k, experts, m), blocks), m * n * k + experts * n * k * 20
                        if key not in found or size < found[key][0]:
                            found[key] = (size, m, n, k, experts)
    return {key: v[1:] for key, v in found.items()}


def _groups(form):
    return int(re.search(r"groups=(\d)", form).group(1)) if "groups" in form else 8


@pytest.mark.parametrize("by_expert", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_sizes_take_every_kernel_over_several_steps(dtype, by_expert):
    sizes = sizes_of_steps(dtype, by_expert)
    for form in FORMS:
        if not (dtype == "float32" and "x256" in form):
            steps = {-(-blocks // _groups(form)) for kernel, blocks in sizes if kernel == "matmul_" + form}
            assert max(steps) >= 3, (form, steps)
    assert any(blocks == 70 for _, blocks in sizes)
