"""A layer under forward mode: the tangent of its bias is kept, the one of its input refused, never dropped."""

from __future__ import annotations

import pytest
import torch
from torch import nn
from torch.autograd import forward_ad

import fouroversix_b200 as fos
from fouroversix_b200.model import FourOverSixLinear

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layer(activations):
    torch.manual_seed(0)
    linear = nn.Linear(128, 64, bias=True, device=DEV, dtype=torch.bfloat16)
    return FourOverSixLinear(linear, fos.ModuleQuantizationConfig(activation_dtype=activations, output_dtype="bfloat16")).quantize_weight_()


@pytest.mark.parametrize("activations", ["bfloat16", "nvfp4"])
@pytest.mark.parametrize("grad", [False, True])
def test_linear(activations, grad):
    module = layer(activations)
    x = torch.randn(5, 128, device=DEV).bfloat16()
    tangent = torch.randn(64, device=DEV).bfloat16()
    with torch.set_grad_enabled(grad):
        with forward_ad.dual_level():
            want = module(x)                                  # (under a level the bias is added by torch: a rounding more than in the kernel)
            with pytest.raises((ValueError, RuntimeError), match="forward-mode|forward mode|jvp"):
                module(forward_ad.make_dual(x, torch.ones_like(x)))
            bias = module.bias
            del module._parameters["bias"]
            module.bias = forward_ad.make_dual(bias.detach(), tangent)
            y = module(x)
            got, moved = forward_ad.unpack_dual(y)
            assert torch.equal(got, want) and torch.equal(moved, tangent.expand(5, 64))
