"""Sizes and addresses at the edges of what the beam-drafting and 8-bit entry points take.  CPU only."""

from __future__ import annotations

import ctypes
import os
import subprocess
import sys
from pathlib import Path

import pytest


@pytest.fixture(scope="module")
def lib():
    from dels_b200 import _lib, build

    build.build()
    _lib.load()
    return _lib


def test_workspace_query_of_refused_shapes(lib):
    """A shape that the selection refuses needs the header only; no shape ends the process."""
    most = 2**31 - 1
    shapes = [(2**30, 64, 4, 1000), (2**26, 64, 4, 1000), (most, 64, 64, most), (most, most, most, most), (2**20 + 1, 1, 1, 9),
              (1, 65, 1, 100), (1, 1, 65, 100), (1, 1, 1, 524289), (1, 4, 8, 7), (-1, 4, 4, 100), (1, 0, 1, 100)]
    code = ("from dels_b200 import _lib\n"
            f"print([_lib.query('dels_beam_select_workspace_bytes', *s) for s in {shapes}])\n")
    env = dict(os.environ, PYTHONPATH=str(Path(lib.__file__).resolve().parent.parent))
    run = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr
    assert run.stdout.strip() == str([lib.DELS_WS_HEADER_BYTES] * len(shapes))
    # the largest ones that it takes: maxima of every 128 logits of 2^20 rows
    assert lib.query("dels_beam_select_workspace_bytes", 2**20, 1, 1, 524288) >= 2**20 * 1024 * 16
    assert lib.query("dels_beam_select_workspace_bytes", 2**14, 64, 64, 524288) >= 2**20 * 1024 * 16


@pytest.fixture(scope="module")
def buf():
    b = ctypes.create_string_buffer(1 << 16)
    return (ctypes.addressof(b) + 255) // 256 * 256, b


def misaligned(lib, name, args, numbers):
    """Every argument of `numbers` one byte off is refused."""
    for i in numbers:
        bad = list(args)
        bad[i] += 1
        with pytest.raises(lib.DelsError) as e:
            lib.call(name, *bad)
        assert e.value.status == lib.DELS_ERR_ALIGNMENT, i


def test_every_array_is_aligned_to_its_elements(lib, buf):
    """An address that a kernel could not load from is refused before any device work."""
    p = buf[0]
    #                             logits    ld  base  ld prior beta cum finished pad, sizes, parents tokens scores
    misaligned(lib, "dels_beam_select", (p, 0, 100, p, 100, p, p, p, p, 0, 1, 2, 2, 100, p, p, p, p, 1 << 15, None),
               (0, 3, 5, 6, 7, 14, 15, 16, 17))
    misaligned(lib, "dels_quantize_rows_i8", (p, 1, 64, 2, 64, p, 64, p, None), (0, 5, 7))
    misaligned(lib, "dels_linear_i8", (p, 64, p, p, 64, p, p, 2, 64, 8, p, 1, 8, p, 256, None), (0, 2, 3, 5, 6, 10, 13))
    for rows in (1, 3):  # the form for a few rows and the tiles
        misaligned(lib, "dels_linear_w8a8", (p, 1, 64, p, 64, p, p, rows, 64, 8, p, 1, 8, p, 1 << 15, None),
                   (0, 3, 5, 6, 10, 13))
    state = (ctypes.c_int64 * 8)(p, p + 4096, 16, 16, 0, 0, 1, 16)
    misaligned(lib, "dels_beam_reorder", (state, 1, p, 2, 2, 2, p, None), (2, 6))
