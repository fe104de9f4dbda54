"""The root-mean-square norm against its formula in 64 bits, and its packed form against `quantize` of its 16-bit one.

The plain form keeps the operator's own roundings (the sum to 16 bits, the factor, the two products and the result) and takes the
mean in 64 bits. A factor is the correctly rounded one but for a few rows in 2^28, so outputs are compared bit for bit.
"""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(x, weight, eps, residual=None):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    factor = (h.double().square().mean(-1, keepdim=True) + eps).rsqrt().float()
    return (h.float() * factor * weight.float()).to(x.dtype), h


def tensors(rows, cols, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + rows + 31 * cols)
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x[:, ::53] *= 20
    return x.to(dtype), (torch.randn(rows, cols, generator=g, device=DEV) * 2).to(dtype), (1 + 0.1 * torch.randn(cols, generator=g, device=DEV))


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


SHAPES = [(1, 1), (1, 8), (3, 7), (1, 1024), (5, 1032), (16, 8192), (2, 4096), (7, 4104), (333, 2880), (4, 8200), (3, 32768), (2, 32776), (2, 40000),
          (300, 64), (1000, 136), (2, 5001)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("weight_type", ["same", "float32"])
def test_sixteen_bits(rows, cols, dtype, with_residual, weight_type):
    x, r, w = tensors(rows, cols, dtype)
    w = w.to(dtype) if weight_type == "same" else w
    want, h = plain(x, w, 1e-5, r if with_residual else None)
    got = fos.rms_norm(x, w, eps=1e-5, residual=r if with_residual else None)
    if with_residual:
        got, total = got
        assert same(total, h)
    assert same(got, want)
    exact = h.double() / (h.double().square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    # half a step of the output, and three binary32 roundings before it
    bound = (torch.finfo(dtype).eps / 2 + 4 * 2.0 ** -24) * exact.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((got.double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("rows,cols", [(1, 64), (16, 8192), (16, 100), (333, 2880), (130, 1000), (700, 512), (2, 40000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("fmt,rule", [("nvfp4", "mse"), ("nvfp4", "static_6"), ("nvfp4", "static_4"), ("nvfp4", "mae"), ("nvfp4", "abs_max"),
                                      ("if4", "mse"), ("mxfp4", "static_6"), ("mxfp4", "static_4")])
def test_packed(rows, cols, dtype, with_residual, fmt, rule):
    x, r, w = tensors(rows, cols, dtype, seed=1)
    w = w.to(dtype)
    config = fos.QuantizationConfig(dtype=fmt, scale_rule=rule)
    y, h = plain(x, w, 1e-6, r if with_residual else None)
    want = fos.quantize(y, config)
    got = fos.rms_norm(x, w, residual=r if with_residual else None, config=config)
    if with_residual:
        got, total = got
        assert same(total, h)
    assert torch.equal(got.amax, want.amax)
    assert torch.equal(got.values, want.values)
    assert torch.equal(got.scale_factors.view(torch.uint8), want.scale_factors.view(torch.uint8))
    assert (got.dtype, got.original_shape, got.padded_shape, got.scale_rule) == (want.dtype, want.original_shape, want.padded_shape, want.scale_rule)


@pytest.mark.parametrize("rows,cols", [(1, 8), (1, 24), (5, 72), (256, 64), (512, 504), (513, 512), (2, 8192), (17, 8192), (32, 8184), (33, 8192), (16, 8200),
                                       (3, 16384), (17, 16384), (2, 16392), (64, 2880), (65, 2880), (128, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("weight_type", ["same", "float32"])
@pytest.mark.parametrize("fmt", ["nvfp4", "if4"])
def test_packed_on_both_sides_of_one_launch(rows, cols, dtype, with_residual, weight_type, fmt):
    x, r, w = tensors(rows, cols, dtype, seed=11)
    w = w.to(dtype) if weight_type == "same" else w
    config = fos.QuantizationConfig(dtype=fmt)
    y, h = plain(x, w, 1e-6, r if with_residual else None)
    want = fos.quantize(y, config)
    got = fos.rms_norm(x, w, residual=r if with_residual else None, config=config)
    if with_residual:
        got, total = got
        assert same(total, h)
    assert torch.equal(got.amax, want.amax)
    assert torch.equal(got.values, want.values)
    assert torch.equal(got.scale_factors.view(torch.uint8), want.scale_factors.view(torch.uint8))


@pytest.mark.parametrize("rows", [5, 700])
def test_packed_rows_beside_infinities_and_nan(rows):
    """Where a row holds infinities or NaN the packed rows are those of the 16-bit result."""
    x, _, w = tensors(rows, 512, torch.float16, seed=12)
    x[1, 3], x[3, 7] = float("inf"), float("nan")
    config = fos.QuantizationConfig()
    want, got = fos.quantize(fos.rms_norm(x, w), config), fos.rms_norm(x, w, config=config)
    others = [i for i in range(rows) if i not in (1, 3)]
    assert torch.equal(got.amax, want.amax) and torch.isfinite(got.amax).all()
    assert torch.equal(got.values[others], want.values[others])


@pytest.mark.parametrize("config", [dict(block_scale_2d=True), dict(transpose=True), dict(rht=True), dict(round_style="stochastic")])
def test_other_ways_to_pack(config):
    x, r, w = tensors(96, 512, torch.bfloat16, seed=2)
    config = fos.QuantizationConfig(**config)
    y, _ = plain(x, w, 1e-6, r)
    torch.manual_seed(5)
    want = fos.quantize(y, config)
    torch.manual_seed(5)
    got, _ = fos.rms_norm(x, w, residual=r, config=config)
    assert torch.equal(got.values, want.values) and torch.equal(got.amax, want.amax)
    assert torch.equal(got.scale_factors.view(torch.uint8), want.scale_factors.view(torch.uint8))


@pytest.mark.parametrize("cols", [64, 1000, 4096])
@pytest.mark.parametrize("fmt", [None, "nvfp4"])
def test_zero_rows_and_far_magnitudes(cols, fmt):
    x, r, w = tensors(6, cols, torch.bfloat16, seed=3)
    x[0] = 0
    r[0] = 0
    x[1] *= 2.0 ** 100
    x[2] *= 2.0 ** -100
    r[2] = 0
    w = w.bfloat16()
    want, h = plain(x, w, 1e-6, r)
    if fmt is None:
        got, total = fos.rms_norm(x, w, residual=r)
        assert same(got, want) and same(total, h)
        assert (got[0] == 0).all()
    else:
        config = fos.QuantizationConfig(dtype=fmt)
        got, total = fos.rms_norm(x, w, residual=r, config=config)
        q = fos.quantize(want, config)
        assert torch.equal(got.values, q.values) and torch.equal(got.amax, q.amax)
    zero, _ = fos.rms_norm(torch.zeros_like(x), w, residual=torch.zeros_like(x), config=fos.QuantizationConfig())
    assert zero.amax.item() == 0 and (fos.dequantize(zero) == 0).all()


@pytest.mark.parametrize("cols", [64, 1001, 8192])
def test_infinities_and_nan_stay_in_their_rows(cols):
    x, _, w = tensors(5, cols, torch.float16, seed=4)
    x[1, 3], x[3, 7] = float("inf"), float("nan")
    got, want = fos.rms_norm(x, w), plain(x, w, 1e-6)[0]
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert same(got[[0, 2, 4]], want[[0, 2, 4]])
    assert torch.equal(got[1][~torch.isnan(got[1])], want[1][~torch.isnan(want[1])])


def test_shapes_and_strides():
    x, r, w = tensors(24, 264, torch.bfloat16, seed=6)
    want, h = plain(x, w, 1e-6, r)
    got, total = fos.rms_norm(x.reshape(2, 3, 4, 264), w, residual=r.reshape(2, 3, 4, 264))
    assert got.shape == total.shape == (2, 3, 4, 264)
    assert same(got.reshape(24, 264), want) and same(total.reshape(24, 264), h)
    for cut in (slice(8, 208), slice(3, 203)):
        want, h = plain(x[:, cut], w[cut], 1e-6, r[:, cut])
        got, total = fos.rms_norm(x[:, cut], w[cut], residual=r[:, cut])
        assert same(got, want) and same(total, h)
    want, _ = plain(x.T, w[:24].bfloat16(), 1e-6)
    assert same(fos.rms_norm(x.T, w[:24].bfloat16()), want)
    broadcast = x[:1].expand(9, 264)
    assert same(fos.rms_norm(broadcast, w), plain(broadcast, w, 1e-6)[0])
    assert fos.rms_norm(x[:0], w).shape == (0, 264)
    assert fos.rms_norm(x[0], w).shape == (264,)


@pytest.mark.parametrize("rows", [1, 16, 600])
def test_graphs_streams_and_repeats(rows):
    x, r, w = tensors(rows, 2048, torch.bfloat16, seed=8)
    config = fos.QuantizationConfig()
    held, held_r = x.clone(), r.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        fos.rms_norm(held, w, residual=held_r, config=config)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, total = fos.rms_norm(held, w, residual=held_r, config=config)
    for scale in (1.0, 0.25, 4.0):                           # a smaller largest value follows a larger one
        held.copy_(x * scale)
        graph.replay()
        y, h = plain(x * scale, w, 1e-6, r)
        want = fos.quantize(y, config)
        assert same(total, h)
        assert torch.equal(q.amax, want.amax) and torch.equal(q.values, want.values)
        assert torch.equal(q.scale_factors.view(torch.uint8), want.scale_factors.view(torch.uint8))


@pytest.mark.parametrize("rows", [16, 300])
@pytest.mark.parametrize("fmt", [None, "nvfp4", "mxfp4"])
def test_the_sum_in_place_of_the_residual(rows, fmt):
    """The C entries may write the sum over the residual (a residual stream that stays where it is)."""
    from fouroversix_b200 import _native

    cols = 4096
    x, r, w = tensors(rows, cols, torch.bfloat16, seed=41)
    w = w.bfloat16()
    want, h = plain(x, w, 1e-6, r)
    lib, stream = _native.lib(), _native.stream_ptr(x.device)
    head = (x.data_ptr(), _native.FOS_BF16, rows, cols, cols, r.data_ptr(), cols, w.data_ptr(), _native.FOS_BF16, 1e-6, r.data_ptr(), cols)
    if fmt is None:
        y = torch.empty_like(x)
        _native.check(lib.fos_rms_norm(*head, y.data_ptr(), cols, 0, stream), "fos_rms_norm")
        assert same(y, want)
    else:
        q = fos.quantize(want, fos.QuantizationConfig(dtype=fmt, scale_rule="static_6"))
        values, scales, amax = torch.empty_like(q.values), torch.empty_like(q.scale_factors), torch.empty_like(q.amax)
        need = lib.fos_rms_norm_quantize_workspace_bytes(rows, cols)
        work = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
        _native.check(lib.fos_rms_norm_quantize(*head, {"nvfp4": 0, "mxfp4": 2}[fmt], 0, _native.FOS_SF_TILED, values.data_ptr(), scales.data_ptr(), amax.data_ptr(),
                                                work.data_ptr(), need, stream), "fos_rms_norm_quantize")
        assert torch.equal(values, q.values) and torch.equal(amax, q.amax)
        assert torch.equal(scales.view(torch.uint8), q.scale_factors.view(torch.uint8))
    assert same(r, h)
