"""Every kernel of the products of 16-bit activations with packed weights against the product in 64 bits (the bounds are those of
test_weight_only_gpu), on shapes that tests/test_weight_only_choice_cpu.py holds to the kernel they are meant for."""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos
from fouroversix_b200 import _native
from fouroversix_b200.matmul import GroupLayout, StackedQuantizedTensor, grouped_weight_only_matmul
from tests.test_weight_only_choice_cpu import FORWARD, GRADIENT, GROUPED
from tests.test_weight_only_gpu import check, tensors, unpacked

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = [("nvfp4", "mse"), ("if4", "mse"), ("mxfp4", "static_6")]
TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("case", FORWARD)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt,rule", FORMATS)
def test_forward(case, dtype, fmt, rule):
    rows, n, k = case[2:]
    x, w, bias = tensors(rows, n, k, dtype, seed=41)
    q, bias = fos.quantize(w, fos.QuantizationConfig(dtype=fmt, scale_rule=rule)), bias.to(dtype)
    got = fos.weight_only_matmul(x, q, bias=bias)
    check(got, x, unpacked(q), bias)
    for _ in range(2):
        assert torch.equal(fos.weight_only_matmul(x, q, bias=bias), got)
    aligned = torch.zeros(rows, -(-k // 8) * 8, dtype=dtype, device=DEV)        # (fp16 rows that the copy engine takes as they are)
    aligned[:, :k] = x
    assert torch.equal(fos.weight_only_matmul(aligned[:, :k], q, bias=bias), got)
    assert _native.wait_failure_site() == 0


@pytest.mark.parametrize("case", GRADIENT)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt,rule", FORMATS)
def test_gradient(case, dtype, fmt, rule):
    rows, n, k = case[2:]
    x, w, _ = tensors(rows, n, k, dtype, seed=43)
    q = fos.quantize(w, fos.QuantizationConfig(dtype=fmt, scale_rule=rule))
    x.requires_grad_()
    y = fos.weight_only_matmul(x, q)
    dy = (torch.randn(rows, n, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV) * 1e-3).to(dtype)
    dx, = torch.autograd.grad(y, x, dy, retain_graph=True)
    check(dx, dy, unpacked(q).T)
    for _ in range(2):
        assert torch.equal(torch.autograd.grad(y, x, dy, retain_graph=True)[0], dx)
    assert _native.wait_failure_site() == 0


@pytest.mark.parametrize("case", GROUPED)
@pytest.mark.parametrize("spread", ["even", "ragged", "one"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("fmt,rule", FORMATS)
def test_grouped(case, spread, dtype, fmt, rule):
    """Rows fetched by index, groups in descending order."""
    rows, n, k, groups = case[1:]
    g = torch.Generator(device=DEV).manual_seed(rows + k)
    config = fos.QuantizationConfig(dtype=fmt, scale_rule=rule)
    weights = [fos.quantize((torch.randn(n, k, generator=g, device=DEV) * (0.02 + 0.001 * e)).to(dtype), config) for e in range(groups)]
    if spread == "one":
        counts = [0] * (groups - 1) + [rows]
    elif spread == "even":
        counts = [rows // groups + (e < rows % groups) for e in range(groups)]
    else:
        cuts = sorted(torch.randint(0, rows + 1, (groups - 1,), generator=torch.Generator().manual_seed(rows)).tolist())
        counts = [b - a for a, b in zip([0, *cuts], [*cuts, rows])]
    start = [sum(counts[e + 1:]) for e in range(groups)]
    x = torch.randn(rows + 7, k, generator=g, device=DEV).to(dtype)
    index = torch.randint(0, rows + 7, (rows,), generator=g, device=DEV, dtype=torch.int32)
    layout = GroupLayout(torch.tensor([*start, rows], dtype=torch.int32, device=DEV), torch.tensor(counts, dtype=torch.int32, device=DEV), rows, groups)
    stacked = StackedQuantizedTensor.stack(weights)
    got = grouped_weight_only_matmul(x, stacked, layout, row_index=index)
    for e, c in enumerate(counts):
        if c:
            mine = slice(start[e], start[e] + c)
            check(got[mine], x[index[mine].long()], unpacked(weights[e]))
    assert torch.equal(grouped_weight_only_matmul(x, stacked, layout, row_index=index), got)
    assert _native.wait_failure_site() == 0


@pytest.mark.parametrize("case", FORWARD)
def test_rows_of_infinities_stay_alone(case):
    rows, n, k = case[2:]
    x, w, _ = tensors(rows, n, k, torch.bfloat16, seed=33)
    q = fos.quantize(w)
    want = fos.weight_only_matmul(x, q)
    x[1, 5], x[2, 7] = float("inf"), float("nan")
    got = fos.weight_only_matmul(x, q)
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[1]).any()
    keep = [i for i in range(rows) if i not in (1, 2)]
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("case", [c for c in FORWARD if c[1] == 1 or c[0] in (128, 256)])
def test_in_a_graph(case):
    rows, n, k = case[2:]
    x, w, _ = tensors(rows, n, k, torch.bfloat16, seed=47)
    q = fos.quantize(w)
    held = x.clone()
    fos.weight_only_matmul(held, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fos.weight_only_matmul(held, q)
    for scale in (1, 2):
        held.copy_(x * scale)
        graph.replay()
        assert torch.equal(out, fos.weight_only_matmul(x * scale, q))
