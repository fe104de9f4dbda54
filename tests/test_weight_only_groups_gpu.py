"""Grouped products of 16-bit activations with packed weights where the groups lie in the output in any order: each group's rows against
the product in 64 bits (the bounds are those of test_weight_only_gpu), rows of nobody zero, nothing written around the output."""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos
from fouroversix_b200 import _native
from fouroversix_b200.matmul import GroupLayout, StackedQuantizedTensor, grouped_weight_only_matmul
from fouroversix_b200.quantize import from_blocked, to_blocked
from tests.test_weight_only_gpu import check, unpacked

pytestmark = pytest.mark.gpu
DEV = "cuda"


def placed(counts: list[int], order: str, gap: int, empty: str) -> tuple[list[int], int]:
    """Where each group starts when the groups are laid out in another order than their numbers', `gap` rows of nobody before each that has
    rows and one behind the last; and the rows in all. Groups without rows start where they come, at 0, or in the middle of another's."""
    places = list(range(len(counts)))
    if order == "descending":
        places.reverse()
    elif order == "shuffled":
        places = torch.randperm(len(counts), generator=torch.Generator().manual_seed(len(counts) + sum(counts))).tolist()
    start, at = [0] * len(counts), 0
    for g in places:
        at += gap * (counts[g] > 0)
        start[g] = at
        at += counts[g]
    largest = max(range(len(counts)), key=counts.__getitem__)
    for g, c in enumerate(counts):
        if c == 0 and empty != "in place":
            start[g] = 0 if empty == "zero" else start[largest] + counts[largest] // 2
    return start, at + 1


def test_an_output_in_the_inputs_memory_is_refused():
    """CTAs that read a row of x may run behind others that have written there."""
    n = k = 128
    stacked = StackedQuantizedTensor.stack([fos.quantize((torch.randn(n, k, device=DEV) * 0.02).bfloat16())] * 2)
    both = torch.randn(40, k, device=DEV).bfloat16()
    layout = GroupLayout.compact(torch.tensor([9, 11], device=DEV), 20)
    want = grouped_weight_only_matmul(both[:20], stacked, layout)
    for out in (both[:20], both[19:39], both.reshape(20, 2 * k)[:, :n]):
        with pytest.raises(ValueError, match="memory"):
            grouped_weight_only_matmul(both[:20], stacked, layout, out=out)
    assert torch.equal(grouped_weight_only_matmul(both[:20], stacked, layout, out=both[20:]), want)
    wide = torch.randn(20, 3 * k, device=DEV).bfloat16()     # columns of one tensor share none
    x = wide[:, k:2 * k].clone()
    want = grouped_weight_only_matmul(x, stacked, layout)
    for at in (0, 2 * k):
        assert torch.equal(grouped_weight_only_matmul(wide[:, k:2 * k], stacked, layout, out=wide[:, at:at + n]), want)
    assert torch.equal(wide[:, k:2 * k], x)
    for at in (1, k, 2 * k - 1):
        with pytest.raises(ValueError, match="memory"):
            grouped_weight_only_matmul(wide[:, k:2 * k], stacked, layout, out=wide[:, at:at + n])
    # an input that is copied first is not read in place
    turned = both[:20].T.contiguous().T
    assert torch.equal(grouped_weight_only_matmul(turned, stacked, layout, out=both[20:]), grouped_weight_only_matmul(both[:20], stacked, layout))


SOME = [3, 5, 0, 2, 6, 1, 0, 4]
LAYOUTS = {
    "two": [5, 6],
    "few": SOME,
    "sixteen": [7, 12, 0, 3, 10, 1, 0, 9],
    "tile": [40, 61, 0, 1, 130, 9, 0, 33],                  # tensor cores
    "more groups than rows": [0] * 9 + [4] + [0] * 7 + [1, 0, 2] + [0] * 5 + [3],
    "one of many": [0] * 30 + [9] + [0] * 9,
    "nobody": [0] * 12,
}


@pytest.mark.parametrize("name", list(LAYOUTS))
@pytest.mark.parametrize("order", ["ascending", "descending", "shuffled"])
@pytest.mark.parametrize("gap", [0, 2])
@pytest.mark.parametrize("empty", ["in place", "zero", "inside"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_groups_in_any_order(name, order, gap, empty, dtype):
    counts, k, n = LAYOUTS[name], 264, 200
    if empty == "inside" and not any(counts):
        pytest.skip("no group has rows")
    start, capacity = placed(counts, order, gap, empty)
    g = torch.Generator(device=DEV).manual_seed(len(counts))
    pair = [fos.quantize((torch.randn(n, k, generator=g, device=DEV) * s).to(dtype)) for s in (0.02, 0.03)]
    weights = [pair[e % 2] for e in range(len(counts))]
    stacked = StackedQuantizedTensor.stack(weights)
    needs_workspace = _native.lib().fos_weight_only_workspace_bytes(capacity, *stacked.padded_shape, len(counts), 0) > 0
    assert needs_workspace == (name == "tile")              # both kinds of kernel are asked
    x = torch.randn(capacity, k, generator=g, device=DEV).to(dtype)
    layout = GroupLayout(torch.tensor(start + [capacity], dtype=torch.int32, device=DEV), torch.tensor(counts, dtype=torch.int32, device=DEV),
                         capacity, len(counts))
    buffer = torch.full((capacity + 2, n + 8), 7.0, dtype=dtype, device=DEV)
    got = grouped_weight_only_matmul(x, stacked, layout, out=buffer[1:-1, :n])
    assert (buffer[0] == 7).all() and (buffer[-1] == 7).all() and (buffer[:, n:] == 7).all()
    free = torch.ones(capacity, dtype=torch.bool, device=DEV)
    for e, c in enumerate(counts):
        if c:
            free[start[e]:start[e] + c] = False
            check(got[start[e]:start[e] + c], x[start[e]:start[e] + c], unpacked(weights[e]))
    assert (got[free] == 0).all()
    for _ in range(3):
        assert torch.equal(grouped_weight_only_matmul(x, stacked, layout), got)


@pytest.mark.parametrize("rows", [9, 60, 127])
@pytest.mark.parametrize("k,n", [(8192, 200), (2048, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_passes_over_a_split_sum(rows, k, n, dtype):
    """All rows in one of many groups: the kernel for few rows takes them a handful at a time, K shared by a cluster whose CTAs write
    their sums into each other's memory pass after pass. The same bits from every repeat."""
    groups, at = 32, 5
    g = torch.Generator(device=DEV).manual_seed(rows + k)
    weight = fos.quantize((torch.randn(n, k, generator=g, device=DEV) * 0.02).to(dtype))
    stacked = StackedQuantizedTensor.stack([weight] * groups)
    assert _native.lib().fos_weight_only_workspace_bytes(rows, *stacked.padded_shape, groups, 0) == 0
    x = torch.randn(rows, k, generator=g, device=DEV).to(dtype)
    layout = GroupLayout.compact(torch.tensor([rows * (e == at) for e in range(groups)], device=DEV), rows)
    got = grouped_weight_only_matmul(x, stacked, layout)
    check(got, x, unpacked(weight))
    for _ in range(30):
        assert torch.equal(grouped_weight_only_matmul(x, stacked, layout), got)


def in_the_other_layout(q: fos.QuantizedTensor) -> fos.QuantizedTensor:
    """The same tensor with its scale factors row by row instead of in tiles, or the other way round."""
    shape = (q.padded_shape[0], q.padded_shape[1] // q.dtype.block_size)
    tiled = q.scale_factors_are_in_blackwell_layout
    scales = from_blocked(q.scale_factors, shape).reshape(-1) if tiled else to_blocked(q.scale_factors.reshape(shape))
    return fos.QuantizedTensor(q.values, scales, q.amax, q.dtype, q.original_shape, q.scale_rule, q.round_style, q.padded_shape,
                               scale_factors_are_in_blackwell_layout=not tiled)


@pytest.mark.parametrize("other", [False, True])
@pytest.mark.parametrize("rows", [12, 100, 600])
@pytest.mark.parametrize("fmt,rule", [("nvfp4", "mse"), ("if4", "mse"), ("mxfp4", "static_6")])
def test_stacks_of_either_scale_layout(fmt, rule, rows, other):
    """Stacked from tensors as `quantize` returns them and in the other layout: the grouped product, the product with one member and what a
    member dequantizes to are those of the tensors that were stacked."""
    n, k, counts = 391, 520, [rows // 3, 0, rows - rows // 3]
    g = torch.Generator(device=DEV).manual_seed(rows)
    weights = [fos.quantize((torch.randn(n, k, generator=g, device=DEV) * s).bfloat16(), fos.QuantizationConfig(dtype=fmt, scale_rule=rule))
               for s in (0.02, 0.03, 0.04)]
    stacked = StackedQuantizedTensor.stack([in_the_other_layout(w) for w in weights] if other else weights)
    x = torch.randn(rows, k, generator=g, device=DEV).bfloat16()
    got = grouped_weight_only_matmul(x, stacked, GroupLayout.compact(torch.tensor(counts, device=DEV), rows))
    at = 0
    for e, c in enumerate(counts):
        assert torch.equal(unpacked(stacked[e]), unpacked(weights[e]))
        assert torch.equal(fos.dequantize(stacked[e]), fos.dequantize(weights[e]))
        if c:
            check(got[at:at + c], x[at:at + c], unpacked(weights[e]))
            assert torch.equal(fos.weight_only_matmul(x[at:at + c], stacked[e]), fos.weight_only_matmul(x[at:at + c], weights[e]))
        at += c
