"""The operators that read their inputs' memory refuse what is more than memory: forward-mode duals and tensors that a function transform
has wrapped. The refusal comes before the one of CPU tensors, so no GPU is asked for."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import fouroversix_b200 as fos
from fouroversix_b200.matmul import GroupLayout, StackedQuantizedTensor, grouped_weight_only_matmul

X = torch.ones(4, 64, dtype=torch.bfloat16)
ONES = torch.ones(64, dtype=torch.bfloat16)
BIAS = torch.ones(128, dtype=torch.bfloat16)


def packed():
    return fos.QuantizedTensor(torch.zeros(128, 32, dtype=torch.uint8), torch.zeros(128 * 4, dtype=torch.float8_e4m3fn), torch.ones(1), "nvfp4", (128, 64),
                               "mse", "nearest", (128, 64))


CALLS = {
    "product": (lambda t: fos.weight_only_matmul(t, packed()), X),
    "product's bias": (lambda t: fos.weight_only_matmul(X, packed(), bias=t), BIAS),
    "grouped": (lambda t: grouped_weight_only_matmul(t, StackedQuantizedTensor.stack([packed()]), GroupLayout.compact(torch.tensor([4]), 4)), X),
    "norm": (lambda t: fos.rms_norm(t, ONES), X),
    "norm's weight": (lambda t: fos.rms_norm(X, t), ONES),
    "norm's residual": (lambda t: fos.rms_norm(X, ONES, residual=t), X),
}


@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(name, grad):
    call, t = CALLS[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
        with pytest.raises(ValueError, match="forward-mode"):
            call(dual)
        with pytest.raises(ValueError, match="CUDA"):          # (a tensor without a tangent is none of this)
            call(t)


@pytest.mark.parametrize("name", list(CALLS))
def test_transforms_are_refused(name):
    call, t = CALLS[name]

    def loss(v):
        out = call(v)
        return out.float().sum()

    for transformed in (lambda: torch.func.grad(loss)(t), lambda: torch.vmap(loss)(t.expand(2, *t.shape)), lambda: torch.func.jvp(loss, (t,), (t,))):
        with pytest.raises(ValueError, match="transforms"):
            transformed()


def test_the_one_call_linear_layer_refuses_its_input():
    """(Its bias may be more than memory: it is then added by torch.)"""
    module = fos.FourOverSixLinear(torch.nn.Linear(64, 24, bias=True, dtype=torch.bfloat16), fos.ModuleQuantizationConfig())
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        module._forward_one_call(forward_ad.make_dual(X, torch.ones_like(X)), packed())
    with pytest.raises(ValueError, match="transforms"):
        torch.vmap(lambda t: module._forward_one_call(t, packed()))(X.expand(2, 4, 64))
