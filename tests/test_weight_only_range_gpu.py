"""The ends of the range of numbers that the products of 16-bit activations with packed weights multiply in fp16."""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos
from fouroversix_b200.matmul import GroupLayout, StackedQuantizedTensor, grouped_weight_only_matmul
from fouroversix_b200.quantize import to_blocked
from tests.test_weight_only_gpu import check, unpacked

pytestmark = pytest.mark.gpu
DEV = "cuda"


def every_scale():
    """An MXFP4 weight [256, 128] whose row f has the scale byte f in every block (255 is NaN, which no tensor of numbers has: 127 instead) and
    all sixteen codes."""
    code = torch.arange(128, device=DEV) % 16
    values = (code[0::2] | (code[1::2] << 4)).to(torch.uint8).expand(256, 64).contiguous()
    byte = torch.arange(256, device=DEV).masked_fill(torch.arange(256, device=DEV) == 255, 127).to(torch.uint8)
    scales = to_blocked(byte[:, None].expand(256, 4).contiguous())
    return fos.QuantizedTensor(values, scales.view(torch.float8_e8m0fnu), torch.ones(1, device=DEV), "mxfp4", (256, 128), "static_6", "nearest", (256, 128))


@pytest.mark.parametrize("rows", [1, 8, 12, 40, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("grouped", [False, True])
def test_mxfp4_scales_at_both_ends(rows, dtype, grouped):
    """Every scale there is, against the numbers themselves where they are exact and against `dequantize` outside. A row of x has one 1, so an
    output is one of the weight's numbers."""
    q = every_scale()
    x = torch.zeros(rows, 128, dtype=dtype, device=DEV)
    pick = torch.arange(rows, device=DEV) * 7 % 128
    x[torch.arange(rows, device=DEV), pick] = 1
    if grouped:
        layout = GroupLayout.compact(torch.tensor([rows], device=DEV), rows)
        got = grouped_weight_only_matmul(x, StackedQuantizedTensor.stack([q]), layout, out_dtype=torch.float32)
    else:
        got = fos.weight_only_matmul(x, q, out_dtype=torch.float32)
    exact = unpacked(q)[:, pick].T
    whole = slice(127 - 23, 127 + 13 + 1)
    assert torch.equal(got[:, whole].double(), exact[:, whole])
    # outside: the scale in fp16 times the code's number in fp16, which is what `dequantize` gives
    scale = torch.exp2(torch.arange(255, device=DEV).double() - 127).half()
    half = scale[:, None] * (unpacked(q)[127].half())                               # (row 127 has the scale 1: the codes' numbers)
    finite = torch.isfinite(half).all(1)                                             # (in the others an infinity times 0 is NaN)
    assert finite.tolist() == [f <= 127 + 13 for f in range(255)]
    assert torch.equal(got[:, :255][:, finite], half[finite][:, pick].T.float())
    assert torch.equal(fos.dequantize(q, torch.float16)[:255][finite], half[finite])
    assert not torch.isfinite(got[:, 127 + 14:255]).any()
    # what the documentation names for such weights
    wide = fos.dequantize(q, torch.float32, intermediate_dtype=torch.float32)[:, pick].T
    near = slice(127 - 120, 127 + 120)                                               # (clear of binary32's own ends)
    assert torch.equal(wide[:, near].double(), exact[:, near])


@pytest.mark.parametrize("rows", [1, 8, 12, 40, 300])
@pytest.mark.parametrize("fmt,rule", [("nvfp4", "mse"), ("if4", "mse"), ("mxfp4", "static_6")])
@pytest.mark.parametrize("below", [20, 29, 34, 39, 45])
def test_bf16_rows_that_span_many_binades(rows, fmt, rule, below):
    """One large value that meets weights of zero, the others 2^below smaller: exact to 2^-29 of the largest, off by 2^-39 of it at most."""
    n, k = 200, 256
    g = torch.Generator(device=DEV).manual_seed(rows)
    w = torch.randn(n, k, generator=g, device=DEV) * 0.02
    w[:, 0] = 0
    q = fos.quantize(w.bfloat16(), fos.QuantizationConfig(dtype=fmt, scale_rule=rule))
    w64 = unpacked(q)
    assert (w64[:, 0] == 0).all()
    x = (1 + torch.rand(rows, k, generator=g, device=DEV)).bfloat16() * 2.0 ** -below
    x[:, 0] = 1
    got = fos.weight_only_matmul(x, q, out_dtype=torch.float32)
    want, mass = x.double() @ w64.T, (x.double().abs() @ w64.abs().T)
    off = (got.double() - want).abs()
    # fp32's own rounding and its sums, and what the values lose: nothing down to 2^-29
    bound = 2.0 ** -23 * want.abs() + (k + 64) * 2.0 ** -23 * mass
    if below > 29:
        bound = bound + 2.0 ** -39 * w64.abs().sum(-1)
    assert (off <= bound).all()
    if below <= 29:
        check(fos.weight_only_matmul(x, q), x, w64)
