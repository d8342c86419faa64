"""The beam-drafting entry points report bad arguments before any device work.  CPU only."""

from __future__ import annotations

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from dels_b200 import _lib, build

    build.build()
    _lib.load()
    return _lib


@pytest.fixture(scope="module")
def buf():
    b = ctypes.create_string_buffer(1 << 16)
    return (ctypes.addressof(b) + 255) // 256 * 256, b


def refused(lib, name, *args, status=None, match=None):
    with pytest.raises(lib.DelsError, match=match) as e:
        lib.call(name, *args)
    if status is not None:
        assert e.value.status == status


def select(lib, p, **kw):
    a = dict(logits=p, dtype=lib.DELS_DTYPE_BF16, ld=100, base=None, ld_base=0, prior=None, beta=None, cum=p,
             finished=None, pad=0, n_seq=1, beams=2, select=2, V=100, parents=p, tokens=p, scores=p, ws=p,
             ws_bytes=1 << 15, stream=None)
    a.update(kw)
    return ("dels_beam_select", *a.values())


def test_select_arguments(lib, buf):
    p = buf[0]
    bad = lib.DELS_ERR_INVALID_ARG
    for kw in (dict(n_seq=-1), dict(beams=0), dict(beams=65), dict(select=65), dict(select=101, V=100), dict(V=1 << 20),
               dict(dtype=2), dict(cum=None), dict(tokens=None), dict(ld=99), dict(base=p, ld_base=99), dict(prior=p),
               dict(finished=p, pad=100), dict(finished=p, pad=-1), dict(n_seq=1 << 20, beams=2)):
        refused(lib, *select(lib, p, **kw), status=bad)
    refused(lib, *select(lib, p, logits=p + 1), status=lib.DELS_ERR_ALIGNMENT)
    refused(lib, *select(lib, p, ws_bytes=256), status=lib.DELS_ERR_WORKSPACE)
    refused(lib, *select(lib, p, ws=p + 8), status=lib.DELS_ERR_ALIGNMENT)
    # a workspace for one sequence holds its group maxima and parts; none needs the header only
    q = lib.query
    assert q("dels_beam_select_workspace_bytes", 0, 4, 4, 100) == lib.DELS_WS_HEADER_BYTES
    assert q("dels_beam_select_workspace_bytes", 1, 4, 4, 151936) >= 4 * 297 * 16
    assert q("dels_beam_select_workspace_bytes", 64, 8, 8, 151936) >= 512 * 297 * 16


def test_reorder_arguments(lib, buf):
    p = buf[0]
    bad = lib.DELS_ERR_INVALID_ARG

    def state(src, dst, row_s, row_d, so=0, do=0, outer=1, inner=16):
        return (ctypes.c_int64 * 8)(src, dst, row_s, row_d, so, do, outer, inner)

    def call(st, n_seq=2, beams=2, sel=2, n=1):
        return ("dels_beam_reorder", st, n, p, n_seq, beams, sel, None, None)

    far = p + 4096
    refused(lib, *call(state(p, far, 16, 16), n_seq=-1), status=bad)
    refused(lib, *call(state(p, far, 16, 16), beams=65), status=bad)
    refused(lib, *call(state(p, far, 16, 16), sel=0), status=bad)
    refused(lib, *call(state(p, far, -16, 16)), status=bad, match="negative")
    refused(lib, *call(state(p, far, 16, 15)), status=bad, match="rows of dst overlap")
    refused(lib, *call(state(p, far, 64, 64, 8, 8, outer=2)), status=bad, match="rows of dst overlap")
    refused(lib, *call(state(p, p + 16, 16, 16)), status=bad, match="overlap without being the same")
    refused(lib, *call(state(p, p, 16, 32)), status=bad, match="overlap without being the same")
    refused(lib, *call(state(p, p, 16, 16), sel=3), status=bad, match="overlap without being the same")
    refused(lib, *call(state(0, far, 16, 16)), status=bad, match="NULL")
    refused(lib, *call(state(p, far, 16, 16, inner=-1)), status=bad)
    refused(lib, "dels_beam_reorder", None, 1, p, 2, 2, 2, None, None, status=bad)


def test_i8_arguments(lib, buf):
    p = buf[0]
    bad, align = lib.DELS_ERR_INVALID_ARG, lib.DELS_ERR_ALIGNMENT
    quant = lambda x=p, dt=0, ld=64, rows=2, K=64, q=p, ldq=64, s=p: ("dels_quantize_rows_i8", x, dt, ld, rows, K, q, ldq, s, None)  # noqa: E731
    for args in (quant(rows=-1), quant(K=0), quant(dt=3), quant(x=None), quant(s=None), quant(ld=63), quant(q=None)):
        refused(lib, *args, status=bad)
    refused(lib, *quant(x=p + 1), status=align)
    refused(lib, *quant(q=p + 8), status=align)
    refused(lib, *quant(ldq=72), status=align)

    def product(x=p, ldx=64, sx=p, w=p, ldw=64, sw=p, b=None, rows=2, K=64, N=8, out=p, dt=0, ldo=8, ws=p, n=256):
        return ("dels_linear_i8", x, ldx, sx, w, ldw, sw, b, rows, K, N, out, dt, ldo, ws, n, None)

    for args in (product(rows=-1), product(K=0), product(N=0), product(sx=None), product(sw=None), product(out=None),
                 product(dt=5), product(ldo=7), product(w=None)):
        refused(lib, *args, status=bad)
    for args in (product(ldx=72), product(ldw=56), product(w=p + 4), product(out=p + 1), product(b=p + 1)):
        refused(lib, *args, status=align)
    refused(lib, *product(K=131072, ldx=131072, ldw=131072), status=lib.DELS_ERR_UNSUPPORTED, match="32 bits")
    refused(lib, *product(n=0), status=lib.DELS_ERR_WORKSPACE)
    w8 = lambda **kw: ("dels_linear_w8a8", *{**dict(x=p, dt=0, ldx=64, w=p, ldw=64, sw=p, b=None, rows=2, K=64, N=8,  # noqa: E731
                                                    out=p, od=0, ldo=8, ws=p, n=1 << 15, st=None), **kw}.values())
    refused(lib, *w8(n=256), status=lib.DELS_ERR_WORKSPACE)
    refused(lib, *w8(sw=None), status=bad)
    refused(lib, *w8(ldw=40), status=align)
    assert lib.query("dels_linear_w8a8_workspace_bytes", 0, 64) == lib.DELS_WS_HEADER_BYTES
    assert lib.query("dels_linear_w8a8_workspace_bytes", 3, 65) >= lib.DELS_WS_HEADER_BYTES + 3 * 4 + 3 * 80
