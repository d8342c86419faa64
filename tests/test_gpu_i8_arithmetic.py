"""The 8-bit product's roundings, one by one: which integers fp32 rows become, whichever kernel
quantises them."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def near_halves(seed, rows, K):
    """fp32 rows whose values lie within two units in the last place of a quantisation step's half,
    where the rounding of 127 / a decides the integer."""
    rng = np.random.default_rng(seed)
    top = (0.5 + rng.random((rows, 1)) * 4).astype(np.float32)
    half = rng.integers(-126, 126, (rows, K)) + 0.5
    x = (half * top.astype(np.float64) / 127).astype(np.float32)
    for _ in range(2):
        step = rng.integers(-1, 2, (rows, K)).astype(np.float32)
        x = np.where(step == 0, x, np.nextafter(x, np.inf * np.where(step == 0, 1, step))).astype(np.float32)
    x[:, :1] = top  # the row's largest value
    return x


def expected(x):
    """Every operation of rint(x * (127 * (1 / a))) rounded to fp32 by itself."""
    top = np.abs(x).max(axis=1, keepdims=True)
    inv = (np.float32(1) / top) * np.float32(127)
    return np.clip(np.rint(x * inv), -127, 127).astype(np.int8)


@pytest.mark.parametrize("rows,K", [(1, 515), (2, 4096), (3, 77), (64, 1000)])
def test_fp32_rows_quantise_as_tensor_operations_do(cuda_device, rows, K):
    """The integers of fp32 rows are those of the same formula in elementary tensor operations
    (x * (127 / a) of tensors multiplies by the reciprocal), in the row kernel and in the product of
    a few rows, which quantises for itself."""
    from dels_b200 import ops

    dev = cuda_device
    x = near_halves(rows + K, rows, K)
    want = expected(x)
    once = np.float32(127) / np.abs(x).max(axis=1, keepdims=True)  # 127 / a rounded once
    if rows >= 2 and K >= 500:  # (a single row's two forms of 127 / a may be equal)
        assert (np.clip(np.rint(x * once), -127, 127) != want).any()  # the rows tell the two apart
    dx = torch.from_numpy(x).to(dev)
    q, scale = ops.quantize_rows_i8(dx)
    np.testing.assert_array_equal(q.cpu().numpy(), want)
    plain = (dx * (127 / dx.abs().amax(1, keepdim=True))).round().clamp(-127, 127)
    assert torch.equal(q.float(), plain)
    # a product with the identity gives the integers back, times the scale
    pad = -(-K // 16) * 16
    eye = torch.eye(K, pad, dtype=torch.int8, device=dev)[:, :K]
    y = ops.linear_w8a8(dx, eye, torch.ones(K, device=dev))
    assert torch.equal(y, q.float() * scale[:, None])
    strided = torch.zeros(rows, K + 3, device=dev)
    strided[:, 3:] = dx
    assert torch.equal(ops.quantize_rows_i8(strided[:, 3:])[0], q)


def test_fp32_rows_of_extreme_magnitude(cuda_device):
    """Rows whose reciprocal leaves the normal range keep all their bits: powers of two change no
    integer."""
    from dels_b200 import ops

    dev = cuda_device
    x = near_halves(5, 4, 900)
    want = expected(x)
    for e in (-110, -100, 60, 105, 124):  # (the smallest values stay normal numbers)
        dx = torch.from_numpy(np.ldexp(x, e).astype(np.float32)).to(dev)
        np.testing.assert_array_equal(ops.quantize_rows_i8(dx)[0].cpu().numpy(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("biased", [True, False])
def test_a_row_gives_the_same_bits_in_any_call(cuda_device, dtype, biased):
    """A row's products do not depend on how many rows come with it: one and two rows, a tile of them,
    pairs of tiles; scales of both signs and a channel of zeros with a negative one among the weights."""
    from dels_b200 import ops

    dev = cuda_device
    K, N = 300, 30011
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn(300, K, generator=g, device=dev).to(dtype)
    wq, sw = ops.quantize_rows_i8(torch.randn(N, K, generator=g, device=dev))
    wq[6] = 0
    sw[::3] *= -1
    bias = torch.randn(N, generator=g, device=dev).to(dtype) if biased else None
    whole = ops.linear_w8a8(x, wq, sw, bias)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    for rows in (1, 2, 3, 40, 129):
        part = ops.linear_w8a8(x[:rows], wq, sw, bias)
        assert torch.equal(part.view(bits), whole[:rows].view(bits)), rows
        # and from rows that were quantised before
        q, s = ops.quantize_rows_i8(x[:rows])
        assert torch.equal(ops.linear_i8(q, s, wq, sw, bias, out_dtype=dtype).view(bits), part.view(bits)), rows
