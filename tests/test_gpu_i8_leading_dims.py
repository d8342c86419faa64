"""linear_w8a8 takes F.linear's shapes: any number of leading dimensions."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_leading_dimensions(cuda_device, dtype):
    from dels_b200 import ops

    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(1)
    K, N = 72, 203
    wq, sw = ops.quantize_rows_i8(torch.randn(N, K, generator=g, device=dev))
    bias = torch.randn(N, generator=g, device=dev).to(dtype)
    x = torch.randn(3, 5, K, generator=g, device=dev).to(dtype)
    want = ops.linear_w8a8(x.view(15, K), wq, sw, bias)
    for shape in ((3, 5), (15, 1), (1, 15), (1, 3, 5), (5, 3, 1, 1)):
        y = ops.linear_w8a8(x.view(*shape, K), wq, sw, bias)
        assert y.shape == (*shape, N) and y.dtype == dtype
        assert torch.equal(y.view(15, N), want)
    assert torch.equal(ops.linear_w8a8(x[0, 0], wq, sw, bias), want[0])
    # hiddens [:, 1:4] of a draft block, and a transposed batch
    assert torch.equal(ops.linear_w8a8(x[:, 1:4], wq, sw, bias), want.view(3, 5, N)[:, 1:4])
    assert torch.equal(ops.linear_w8a8(x.transpose(0, 1), wq, sw, bias), want.view(3, 5, N).transpose(0, 1))
    for shape in ((0, 5), (3, 0)):
        assert ops.linear_w8a8(x[: shape[0], : shape[1]], wq, sw, bias).shape == (*shape, N)
    # outputs: whole, and every other row of a wider one
    out = torch.full((3, 5, N + 5), 7.0, dtype=dtype, device=dev)
    inner = out[:, :, 2 : 2 + N]
    assert ops.linear_w8a8(x, wq, sw, bias, out=inner) is inner
    assert torch.equal(inner, want.view(3, 5, N)) and (out[:, :, :2] == 7).all() and (out[:, :, 2 + N :] == 7).all()
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
    assert ops.linear_w8a8(x, wq, sw, out_dtype=other).dtype == other


def test_leading_dimension_refusals(cuda_device):
    from dels_b200 import ops

    dev = cuda_device
    wq, sw = ops.quantize_rows_i8(torch.randn(8, 32, device=dev))
    x = torch.randn(2, 3, 32, device=dev)
    for bad in (dict(out=torch.zeros(6, 8, device=dev)), dict(out=torch.zeros(3, 2, 8, device=dev)),
                dict(out=torch.zeros(2, 3, 9, device=dev)), dict(out=torch.zeros(2, 4, 8, device=dev)[:, :3]),
                dict(out=torch.zeros(2, 3, 8, device=dev).half()), dict(x=x.cpu()), dict(x=x.half()),
                dict(x=x[..., :31]), dict(x=x[0, 0, 0])):
        args = {"x": x, **bad}
        with pytest.raises(ValueError):
            ops.linear_w8a8(args.pop("x"), wq, sw, **args)
