"""Where a stack of packed weights says its scale factors lie."""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos
from fouroversix_b200.matmul import StackedQuantizedTensor
from fouroversix_b200.matmul.grouped import GroupedQuantizedTensor, GroupLayout, grouped_quantized_matmul


def packed(fmt, tiled):
    block = fos.DataType(fmt).block_size
    scales = torch.arange(128 * 256 // block).to(torch.uint8)
    rule = "static_6" if fmt == "mxfp4" else "mse"
    return fos.QuantizedTensor(torch.zeros(128, 128, dtype=torch.uint8), scales, torch.ones(1), fmt, (100, 250), rule, "nearest", (128, 256),
                               scale_factors_are_in_blackwell_layout=tiled)


@pytest.mark.parametrize("fmt", ["nvfp4", "if4", "mxfp4"])
@pytest.mark.parametrize("tiled", [True, False])
def test_a_stack_keeps_its_members_layout(fmt, tiled):
    stacked = StackedQuantizedTensor.stack([packed(fmt, tiled)] * 3)
    assert stacked.scale_factors_are_in_blackwell_layout is tiled
    member = stacked[1]
    assert member.scale_factors_are_in_blackwell_layout is tiled and member.dtype == fos.DataType(fmt)
    assert torch.equal(member.scale_factors, packed(fmt, tiled).scale_factors)


@pytest.mark.parametrize("fmt,tiled", [("nvfp4", True), ("mxfp4", True), ("if4", False)])
def test_a_stack_by_its_constructor_lies_as_quantize_lays_out(fmt, tiled):
    q = packed(fmt, tiled)
    stacked = StackedQuantizedTensor(q.values[None], q.scale_factors[None], q.amax, q.dtype, q.scale_rule, q.original_shape, q.padded_shape)
    assert stacked.scale_factors_are_in_blackwell_layout is tiled and stacked[0].scale_factors_are_in_blackwell_layout is tiled


def test_refusals():
    with pytest.raises(ValueError, match="layout"):
        StackedQuantizedTensor.stack([packed("if4", True), packed("if4", False)])
    q = packed("nvfp4", True)
    q.round_style = fos.RoundStyle.stochastic_unbiased
    with pytest.raises(ValueError, match="rounding"):
        StackedQuantizedTensor.stack([q])
    rows = GroupedQuantizedTensor(torch.zeros(256, 128, dtype=torch.uint8), torch.zeros(4096, dtype=torch.uint8), torch.ones(1),
                                  GroupLayout.from_counts(torch.tensor([100]), 100), fos.DataType.nvfp4, fos.ScaleRule.mse, 256)
    with pytest.raises(ValueError, match="tiles"):
        grouped_quantized_matmul(rows, StackedQuantizedTensor.stack([packed("nvfp4", False)]))


def test_copies_and_what_was_saved_before_there_was_a_layout():
    import copy
    import pickle

    for fmt, tiled in (("nvfp4", True), ("nvfp4", False), ("if4", True), ("if4", False)):
        stacked = StackedQuantizedTensor.stack([packed(fmt, tiled)])
        assert copy.deepcopy(stacked).scale_factors_are_in_blackwell_layout is tiled
        assert pickle.loads(pickle.dumps(stacked)).scale_factors_are_in_blackwell_layout is tiled
        del stacked.__dict__["scale_factors_are_in_blackwell_layout"]
        assert pickle.loads(pickle.dumps(stacked)).scale_factors_are_in_blackwell_layout is (fmt != "if4")
