"""Refusals of the 16-bit-activation operators, on the host: Python's checks and those of the C entries, all of which come before anything
touches a device."""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos
from fouroversix_b200 import _native
from fouroversix_b200.matmul import GroupLayout, StackedQuantizedTensor, grouped_weight_only_matmul

INVALID, UNSUPPORTED, MISALIGNED, TOO_LARGE = -1, -2, -3, -7
A = 1 << 20           # an address that is aligned and never followed


def packed(n=128, k=64):
    return fos.QuantizedTensor(torch.zeros(n, k // 2, dtype=torch.uint8), torch.zeros(n * k // 16, dtype=torch.float8_e4m3fn), torch.ones(1),
                               "nvfp4", (n, k), "mse", "nearest", (n, k))


def test_python_refusals():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), packed()
    with pytest.raises(ValueError, match="CUDA"):
        fos.weight_only_matmul(x, w)
    with pytest.raises(ValueError, match="QuantizedTensor"):
        fos.weight_only_matmul(x, torch.zeros(128, 64))
    w.dtype = fos.DataType.nvfp6_e2m3 if hasattr(fos.DataType, "nvfp6_e2m3") else fos.DataType.mxfp6_e2m3
    with pytest.raises(ValueError, match="not implemented"):
        fos.weight_only_matmul(x, w)
    layout = GroupLayout.compact(torch.tensor([4]), 4)
    with pytest.raises(ValueError, match="Stacked"):
        grouped_weight_only_matmul(x, packed(), layout)
    stacked = StackedQuantizedTensor.stack([packed()])
    with pytest.raises(ValueError, match="CUDA"):
        grouped_weight_only_matmul(x, stacked, layout)
    with pytest.raises(ValueError, match="CUDA"):
        fos.rms_norm(x, torch.ones(64, dtype=torch.bfloat16))


def test_compact_layout():
    layout = GroupLayout.compact(torch.tensor([3, 0, 5]), 9)
    assert layout.group_start.tolist() == [0, 3, 3, 8] and layout.group_rows.tolist() == [3, 0, 5]
    assert layout.capacity == 9 and layout.num_groups == 3
    assert layout.group_start.dtype == layout.group_rows.dtype == torch.int32
    with pytest.raises(ValueError, match="groups"):
        GroupLayout.compact(torch.zeros(257, dtype=torch.int64), 0)
    with pytest.raises(ValueError, match="groups"):
        GroupLayout.compact(torch.zeros(0, dtype=torch.int64), 0)


def product(**change):
    a = dict(x=A, x_dtype=0, rows=4, k=64, ld_x=64, codes=A, sf=A, amax=A, format=0, rule=3, unbiased=0, layout=1, n=128, n_p=128, k_p=64, bias=0,
             out=A, out_dtype=0, ld_out=128, workspace=0, bytes=0, status=0, stream=0)
    a.update(change)
    return _native.lib().fos_weight_only_matmul(*a.values())


@pytest.mark.parametrize("change,status", [
    (dict(x=0), INVALID), (dict(codes=0), INVALID), (dict(sf=0), INVALID), (dict(amax=0), INVALID), (dict(out=0), INVALID),
    (dict(x_dtype=2), INVALID), (dict(out_dtype=3), INVALID), (dict(format=3), INVALID), (dict(rule=5), INVALID), (dict(layout=2), INVALID),
    (dict(rows=0), INVALID), (dict(k=0), INVALID), (dict(n=0), INVALID), (dict(ld_x=63), INVALID), (dict(ld_out=127), INVALID),
    (dict(n_p=127), INVALID), (dict(n=129), INVALID), (dict(k_p=32), INVALID), (dict(k=65, ld_x=65), INVALID), (dict(format=2), INVALID),
    (dict(rows=1 << 31), TOO_LARGE), (dict(n_p=1 << 30), TOO_LARGE), (dict(k_p=1 << 30), TOO_LARGE),
    (dict(x=A + 1), MISALIGNED), (dict(codes=A + 8), MISALIGNED), (dict(sf=A + 2), MISALIGNED), (dict(out=A + 1), MISALIGNED),
    (dict(out=A + 2, out_dtype=2), MISALIGNED), (dict(bias=A + 1), MISALIGNED), (dict(bias=A + 2, out_dtype=2), MISALIGNED),
])
def test_product_entry(change, status):
    assert product(**change) == status


def grouped(**change):
    a = dict(x=A, x_dtype=0, x_rows=4, k=64, ld_x=64, row_index=0, codes=A, sf=A, amax=A, format=0, rule=3, layout=1, start=A, group_rows=A, groups=4,
             rows=4, n=128, n_p=128, k_p=64, out=A, out_dtype=0, ld_out=128, workspace=0, bytes=0, status=0, stream=0)
    a.update(change)
    return _native.lib().fos_weight_only_matmul_grouped(*a.values())


@pytest.mark.parametrize("change,status", [
    (dict(start=0), INVALID), (dict(group_rows=0), INVALID), (dict(groups=0), INVALID), (dict(groups=257), INVALID), (dict(x_rows=0), INVALID),
    (dict(rows=0), INVALID), (dict(groups=256, n_p=1 << 24), TOO_LARGE), (dict(codes=A + 4), MISALIGNED), (dict(ld_out=100), INVALID),
])
def test_grouped_entry(change, status):
    assert grouped(**change) == status


def gradient(**change):
    a = dict(dy=A, dtype=0, rows=4, n=128, ld_dy=128, codes=A, sf=A, amax=A, format=0, rule=3, unbiased=0, layout=1, k=64, n_p=128, k_p=64, dx=A,
             out_dtype=0, ld_dx=64, workspace=0, bytes=0, status=0, stream=0)
    a.update(change)
    return _native.lib().fos_weight_only_matmul_dgrad(*a.values())


@pytest.mark.parametrize("change,status", [(dict(dy=0), INVALID), (dict(ld_dy=127), INVALID), (dict(ld_dx=63), INVALID), (dict(dx=0), INVALID),
                                           (dict(dx=A + 1), MISALIGNED), (dict(k_p=32), INVALID)])
def test_gradient_entry(change, status):
    assert gradient(**change) == status


def test_workspace_sizes():
    lib = _native.lib()
    assert lib.fos_weight_only_workspace_bytes(100, 128, 256, 0, 1) == 100 * 128 * 2 + 512
    assert lib.fos_weight_only_workspace_bytes(100, 128, 256, 0, 0) >= 100 * 256 * 2 + 512
    assert lib.fos_weight_only_workspace_bytes(3, 128, 64, 0, 1) == 768 + 256
    assert lib.fos_weight_only_workspace_bytes(3, 128, 64, 0, 0) == 0
    assert lib.fos_weight_only_workspace_bytes(0, 128, 64, 0, 0) == 0
    assert lib.fos_rms_norm_quantize_workspace_bytes(1000, 64) == 4096 + 128000
    assert lib.fos_rms_norm_quantize_workspace_bytes(3, 64) == 0          # (one launch, y never in memory)
    assert lib.fos_rms_norm_quantize_workspace_bytes(0, 64) == 0


def norm(entry="fos_rms_norm", **change):
    a = dict(x=A, dtype=0, rows=4, cols=64, ld_x=64, residual=A, ld_residual=64, weight=A, weight_dtype=0, eps=1e-6, sum=A, ld_sum=64)
    a |= dict(y=A, ld_y=64, amax=0, stream=0) if entry == "fos_rms_norm" else dict(
        format=0, rule=3, layout=1, codes=A, sf=A, amax=A, workspace=A, bytes=1 << 20, stream=0)
    a.update(change)
    return getattr(_native.lib(), entry)(*a.values())


@pytest.mark.parametrize("change,status", [
    (dict(x=0), INVALID), (dict(weight=0), INVALID), (dict(sum=0), INVALID), (dict(dtype=2), INVALID), (dict(weight_dtype=1), INVALID), (dict(rows=0), INVALID),
    (dict(cols=0), INVALID), (dict(ld_x=63), INVALID), (dict(ld_residual=63), INVALID), (dict(ld_sum=63), INVALID), (dict(eps=0.0), INVALID),
    (dict(eps=-1.0), INVALID), (dict(eps=float("nan")), INVALID), (dict(x=A + 1), MISALIGNED), (dict(weight=A + 2, weight_dtype=2), MISALIGNED),
])
@pytest.mark.parametrize("entry", ["fos_rms_norm", "fos_rms_norm_quantize"])
def test_norm_entries(entry, change, status):
    assert norm(entry, **change) == status


@pytest.mark.parametrize("change,status", [
    (dict(codes=0), INVALID), (dict(sf=0), INVALID), (dict(amax=0), INVALID), (dict(format=3), INVALID), (dict(rule=7), INVALID), (dict(layout=2), INVALID),
    (dict(format=1, rule=0), UNSUPPORTED), (dict(format=2, rule=3), UNSUPPORTED), (dict(codes=A + 4), MISALIGNED), (dict(x=A + 2), UNSUPPORTED),
    (dict(cols=60), UNSUPPORTED), (dict(ld_x=68), UNSUPPORTED), (dict(cols=40000, ld_x=40000, ld_residual=40000, ld_sum=40000), UNSUPPORTED),
    (dict(rows=1000, workspace=0), INVALID), (dict(rows=1000, bytes=100), INVALID), (dict(rows=1000, workspace=A + 64), MISALIGNED),
])
def test_norm_quantize_entry(change, status):
    assert norm("fos_rms_norm_quantize", **change) == status


def test_compact_routing_entry():
    def call(**change):
        a = dict(routing=A, index_bytes=8, tokens=4, top_k=2, experts=8, capacity=8, start=A, rows=A, row_token=A, row_expert=A, pair_row=A, pair_expert=A,
                 workspace=A, stream=0)
        a.update(change)
        return _native.lib().fos_experts_route_compact(*a.values())

    assert call(capacity=7) == INVALID
    assert call(routing=0) == INVALID
    assert call(experts=257) == UNSUPPORTED
