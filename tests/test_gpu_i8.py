"""Row quantisation and the 8-bit integer product on the B200 kernels against their
definitions (float64 / exact integers, numpy)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def ref_quantize(x):
    """fp32 arithmetic of the definition, operation by operation."""
    x = x.astype(np.float32)
    top = np.abs(x).max(axis=1)
    with np.errstate(divide="ignore"):
        inv = np.where(top > 0, np.float32(127) / top, np.float32(0)).astype(np.float32)
    inv = np.minimum(inv, np.finfo(np.float32).max)
    q = np.clip(np.rint(x * inv[:, None]), -127, 127).astype(np.int8)
    return q, (top / np.float32(127)).astype(np.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (2, 8), (5, 100), (1, 4096), (33, 2561), (700, 264), (2, 20000)])
def test_quantize_matches_definition(cuda_device, dtype, rows, K):
    from dels_b200 import ops

    dev = cuda_device
    rng = np.random.default_rng(rows * K)
    x = torch.from_numpy((rng.standard_normal((rows, K)) * 10.0 ** rng.integers(-3, 4, (rows, 1))).astype(np.float32))
    x = x.to(dtype)
    if rows > 2:
        x[1] = 0  # a row of zeros
    q, scale = ops.quantize_rows_i8(x.to(dev))
    want_q, want_scale = ref_quantize(x.float().numpy())
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
    assert q.stride(0) % 16 == 0 or rows == 1
    # x ~ q * scale to half a step (and the roundings of x * inv, 127 values of 2^-24 each)
    err = np.abs(x.float().numpy() - want_q.astype(np.float64) * want_scale[:, None].astype(np.float64))
    assert (err <= want_scale[:, None] * (0.5 + 2e-5)).all()


def test_quantize_extremes(cuda_device):
    """Ties to even, denormal and lowest-value rows, NaN and infinities; a strided view."""
    from dels_b200 import ops

    dev = cuda_device
    x = torch.zeros(7, 40, device=dev)
    x[0, :6] = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -3.5])
    x[1, :3] = torch.tensor([1e-40, -5e-41, 0.0])
    x[2, :3] = torch.tensor([torch.finfo(torch.float32).max, torch.finfo(torch.float32).min, 1.0])
    x[3, 5] = float("nan")
    x[4, 9] = float("-inf")
    x[5] = -1.0
    q, scale = ops.quantize_rows_i8(x)
    assert q[0, :6].tolist() == [127, 0, 2, 2, 0, -4] and float(scale[0]) == 1.0
    assert 0 < q[1, 0].item() <= 127 and q[1, 2].item() == 0
    assert q[2, :3].tolist() == [127, -127, 0]
    assert torch.isnan(scale[3]) and q[3].abs().max() == 0
    assert torch.isinf(scale[4]) and q[4].abs().max() == 0
    assert (q[5] == -127).all() and float(scale[6]) == 0.0 and q[6].abs().max() == 0
    wide = torch.randn(4, 101, device=dev)
    a, sa = ops.quantize_rows_i8(wide[:, 1:98])
    b, sb = ops.quantize_rows_i8(wide[:, 1:98].contiguous())
    assert torch.equal(a, b) and torch.equal(sa, sb)


def make(seed, rows, K, N, dev, low=-127):
    rng = np.random.default_rng(seed)

    def padded(a):
        t = torch.zeros(a.shape[0], -(-K // 16) * 16, dtype=torch.int8)
        t[:, :K] = torch.from_numpy(a)
        return t.to(dev)[:, :K]

    xq = rng.integers(low, 128, (rows, K)).astype(np.int8)
    wq = rng.integers(low, 128, (N, K)).astype(np.int8)
    sx = (0.5 + rng.random(rows)).astype(np.float32) * np.float32(0.01)
    sw = (0.5 + rng.random(N)).astype(np.float32) * np.float32(0.001)
    bias = rng.standard_normal(N).astype(np.float32)
    return xq, wq, sx, sw, bias, padded(xq), padded(wq)


def check_product(got, xq, wq, sx, sw, bias):
    acc = xq.astype(np.float64) @ wq.astype(np.float64).T  # exact: below 2^53
    prod = acc * sx[:, None].astype(np.float64) * sw[None, :].astype(np.float64)
    ref = prod + (0 if bias is None else bias.astype(np.float64))
    # roundings: acc to fp32, two products, the bias addition, each half an ulp (2^-24) of
    # the product or the result; then the result's own type (bf16: 8 significant bits, half an ulp up to 2^-8)
    tol = 2.0**-24 * (3 * np.abs(prod) + np.abs(ref)) * 1.01
    if got.dtype == torch.bfloat16:
        tol = tol + (np.abs(ref) + tol) * 2.0**-8 * 1.01
    err = np.abs(got.float().cpu().numpy().astype(np.float64) - ref)
    assert (err <= tol + 1e-30).all(), float((err - tol).max())


@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,N", [
    (1, 1, 1), (1, 16, 8), (2, 127, 7), (5, 128, 129), (16, 129, 64), (17, 100, 1003), (32, 512, 2000), (33, 2561, 77),
    (64, 256, 5001), (65, 4096, 256), (128, 384, 640), (129, 1000, 333), (256, 130, 1300), (513, 640, 1026),
    (1, 4096, 20011), (300, 3000, 2),
    # enough tiles for CTA pairs: tiles of 160, 192 and 256 rows, a last wave split along the rows
    (129, 200, 38001), (300, 256, 30000), (513, 130, 19001), (512, 384, 20480),
])
def test_product_is_exact(cuda_device, out_dtype, rows, K, N):
    from dels_b200 import ops

    dev = cuda_device
    xq, wq, sx, sw, bias, dxq, dwq = make(rows + K + N, rows, K, N, dev)
    dsx, dsw = torch.from_numpy(sx).to(dev), torch.from_numpy(sw).to(dev)
    check_product(ops.linear_i8(dxq, dsx, dwq, dsw, out_dtype=out_dtype), xq, wq, sx, sw, None)
    b = torch.from_numpy(bias).to(dev).to(out_dtype)
    check_product(ops.linear_i8(dxq, dsx, dwq, dsw, b, out_dtype=out_dtype), xq, wq, sx, sw,
                  b.float().cpu().numpy())


@pytest.mark.parametrize("source", [torch.int8, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,N", [
    (1, 768, 30001), (2, 1000, 20003), (1, 1500, 9001), (2, 2047, 7777), (1, 130, 14211), (2, 15, 15000), (1, 1024, 7103),
])
def test_product_of_few_rows_and_many_channels(cuda_device, source, rows, K, N):
    """One or two rows take several channels at a time; the last channel's row of the weights
    ends with its last value."""
    from dels_b200 import ops

    dev = cuda_device
    xq, wq, sx, sw, _, dxq, dwq = make(rows + K + N, rows, K, N, dev)
    ld = -(-K // 16) * 16
    tight = torch.empty((N - 1) * ld + K, dtype=torch.int8, device=dev)
    w = tight.as_strided((N, K), (ld, 1))
    w.copy_(dwq)
    dsx, dsw = torch.from_numpy(sx).to(dev), torch.from_numpy(sw).to(dev)
    if source == torch.int8:
        check_product(ops.linear_i8(dxq, dsx, w, dsw, out_dtype=torch.float32), xq, wq, sx, sw, None)
        return
    x = (dxq.float() * dsx[:, None]).to(source)
    q, scale = ops.quantize_rows_i8(x)
    check_product(ops.linear_w8a8(x, w, dsw, out_dtype=torch.float32), q.cpu().numpy(), wq, scale.cpu().numpy(), sw, None)


@pytest.mark.parametrize("rows,K,N", [
    # less than a wave of whole tiles; a second one of whole tiles, of halves, of quarters
    (200, 130, 12001), (777, 256, 4099), (1024, 129, 5000), (512, 200, 32000), (513, 128, 6501),
])
def test_product_in_large_tiles(cuda_device, rows, K, N):
    from dels_b200 import ops

    dev = cuda_device
    xq, wq, sx, sw, _, dxq, dwq = make(rows + K + N, rows, K, N, dev)
    dsx, dsw = torch.from_numpy(sx).to(dev), torch.from_numpy(sw).to(dev)
    check_product(ops.linear_i8(dxq, dsx, dwq, dsw, out_dtype=torch.float32), xq, wq, sx, sw, None)


def test_product_keeps_the_largest_sums(cuda_device):
    """K at its bound with every value at -128: the sum is 2^31 - 2^14, still exact."""
    from dels_b200 import _lib, ops

    dev = cuda_device
    K = _lib.DELS_I8_MAX_K
    x = torch.full((2, 131072), -128, dtype=torch.int8, device=dev)[:, :K]
    w = torch.full((3, 131072), -128, dtype=torch.int8, device=dev)[:, :K]
    one = torch.ones(3, device=dev)
    y = ops.linear_i8(x, one[:2], w, one, out_dtype=torch.float32)
    assert (y == float(np.float32(K * 16384))).all()


def test_product_strides_and_untouched_padding(cuda_device):
    """Outputs of odd and even row strides, column slices of a larger buffer: nothing
    outside the result is written; operands with rows further apart than K."""
    from dels_b200 import ops

    dev = cuda_device
    for out_dtype in (torch.bfloat16, torch.float32):
        for N, pad, at in ((64, 3, 1), (63, 0, 0), (62, 2, 2), (65, 1, 1)):
            xq, wq, sx, sw, _, dxq, dwq = make(N + pad, 40, 72, N, dev)
            wide = torch.full((40, N + pad), 7.0, dtype=out_dtype, device=dev)
            xs = torch.zeros(40, 112, dtype=torch.int8, device=dev)
            xs[:, 16:88] = dxq
            ops.linear_i8(xs[:, 16:88], torch.from_numpy(sx).to(dev), dwq, torch.from_numpy(sw).to(dev),
                          out=wide[:, at : at + N])
            check_product(wide[:, at : at + N], xq, wq, sx, sw, None)
            outside = torch.ones(N + pad, dtype=torch.bool, device=dev)
            outside[at : at + N] = False
            assert (wide[:, outside] == 7.0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K,N", [(1, 4096, 256), (3, 77, 1003), (48, 520, 130), (200, 2561, 515)])
def test_w8a8_equals_its_two_parts(cuda_device, dtype, rows, K, N):
    """The fused call gives the bits of the two calls, also when the weights were quantised
    by the call right before it, and again on a workspace another call has used."""
    from dels_b200 import ops

    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(K)
    x = torch.randn(rows, K, generator=g, device=dev).to(dtype)
    w = (torch.randn(N, K, generator=g, device=dev) * 0.02).to(dtype)
    bias = torch.randn(N, generator=g, device=dev).to(dtype)
    wq, sw = ops.quantize_rows_i8(w)
    fused = ops.linear_w8a8(x, wq, sw, bias)
    xq, sx = ops.quantize_rows_i8(x)
    parts = ops.linear_i8(xq, sx, wq, sw, bias, out_dtype=dtype)
    again = ops.linear_w8a8(x, wq, sw, bias)
    assert torch.equal(fused, parts) and torch.equal(fused, again)
    # and it is the product of the quantised operands, near F.linear of the originals
    check_product(fused, xq.cpu().numpy(), wq.cpu().numpy(), sx.cpu().numpy(), sw.cpu().numpy(),
                  bias.float().cpu().numpy())
    ref = x.double() @ w.double().t() + bias.double()
    # a quantised operand is off by an error uniform in half a step of (4.x deviations / 127):
    # about 1% of its deviation, each; the bias adds none
    assert (fused.double() - ref).norm() / ref.norm() < 0.03


def test_w8a8_non_finite_rows_stay_in_their_row(cuda_device):
    from dels_b200 import ops

    dev = cuda_device
    x = torch.randn(5, 64, device=dev)
    wq, sw = ops.quantize_rows_i8(torch.randn(40, 64, device=dev))
    good = ops.linear_w8a8(x, wq, sw)
    x[1, 3] = float("nan")
    x[3, 63] = float("inf")
    y = ops.linear_w8a8(x, wq, sw)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all()
    for r in (0, 2, 4):
        assert torch.equal(y[r], good[r])


def test_w8a8_other_stream_and_graph(cuda_device):
    """On a side stream and replayed from a CUDA graph with new inputs."""
    from dels_b200 import ops

    dev = cuda_device
    x = torch.randn(24, 300, device=dev).bfloat16()
    wq, sw = ops.quantize_rows_i8(torch.randn(500, 300, device=dev))
    want = ops.linear_w8a8(x, wq, sw)
    ws = ops.Workspace(ops.linear_w8a8_workspace_bytes(24, 300), dev)
    out = torch.empty_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear_w8a8(x, wq, sw, out=out, ws=ws)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_w8a8(x, wq, sw, out=out, ws=ws)
    for seed in range(3):
        x.copy_(torch.randn(24, 300, generator=torch.Generator(device=dev).manual_seed(seed), device=dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.linear_w8a8(x, wq, sw))
    assert ws.status() == 0


def test_empty_and_refusals(cuda_device):
    from dels_b200 import _lib, ops

    dev = cuda_device
    x = torch.randn(4, 32, device=dev)
    wq, sw = ops.quantize_rows_i8(torch.randn(8, 32, device=dev))
    xq, sx = ops.quantize_rows_i8(x)
    assert ops.linear_w8a8(x[:0], wq, sw).shape == (0, 8)
    assert ops.linear_i8(xq[:0], sx[:0], wq, sw).shape == (0, 8)
    assert ops.quantize_rows_i8(x[:0])[0].shape == (0, 32)
    with pytest.raises(_lib.DelsArgumentError, match="multiple of 16"):
        ops.linear_i8(torch.zeros(4, 33, dtype=torch.int8, device=dev), sx, torch.zeros(8, 48, dtype=torch.int8,
                                                                                        device=dev)[:, :33], sw)
    with pytest.raises(_lib.DelsArgumentError, match="16-byte aligned"):
        wide = torch.zeros(8, 64, dtype=torch.int8, device=dev)
        ops.linear_i8(xq, sx, wide[:, 8:40], sw)
    with pytest.raises(_lib.DelsArgumentError, match="multiple of 16"):
        ops.quantize_rows_i8(x, q=torch.zeros(4, 40, dtype=torch.int8, device=dev)[:, :32])
    with pytest.raises(_lib.DelsError, match="leave 32 bits"):
        big = torch.zeros(1, 131072, dtype=torch.int8, device=dev)
        ops.linear_i8(big, sx[:1], big, sw[:1])
    with pytest.raises(ValueError):
        ops.quantize_rows_i8(x.half())
    with pytest.raises(ValueError):
        ops.quantize_rows_i8(x.t())
    for bad in (dict(w_scale=sw[:7]), dict(w_scale=sw.double()), dict(wq=wq[:, :16]), dict(wq=wq.cpu()),
                dict(bias=torch.zeros(8, dtype=torch.bfloat16, device=dev)), dict(bias=torch.zeros(7, device=dev)),
                dict(out=torch.zeros(4, 9, device=dev)), dict(out=torch.zeros(4, 8, device=dev).half()),
                dict(out=torch.zeros(8, 4, device=dev).t()), dict(x=x.cpu()), dict(x=x.int()),
                dict(out_dtype=torch.float16)):
        args = {"x": x, "wq": wq, "w_scale": sw, **bad}
        with pytest.raises(ValueError):
            ops.linear_w8a8(args.pop("x"), args.pop("wq"), args.pop("w_scale"), **args)
