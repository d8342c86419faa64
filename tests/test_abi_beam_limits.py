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
