"""The 16-bit-activation operators as layers use them: the linear layer and the experts layer with a 16-bit `activation_dtype`, and a
run of norm, products and norm again as a model makes it."""

from __future__ import annotations

import pytest
import torch
from torch import nn

import fouroversix_b200 as fos
from fouroversix_b200.model import FourOverSixExperts, FourOverSixLinear
from tests.test_weight_only_gpu import check, unpacked

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layer(n, k, bias, kind, **config):
    torch.manual_seed(n + k)
    linear = nn.Linear(k, n, bias=bias, device=DEV, dtype=kind)
    name = {torch.bfloat16: "bfloat16", torch.float16: "float16"}[kind]
    return FourOverSixLinear(linear, fos.ModuleQuantizationConfig(activation_dtype=name, output_dtype=name, **config)).quantize_weight_()


@pytest.mark.parametrize("rows", [1, 16, 70])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("config", [dict(), dict(dtype="if4"), dict(dtype="mxfp4", scale_rule="static_6"), dict(weight_scale_2d=True)])
def test_linear(rows, bias, dtype, config):
    module = layer(300, 512, bias, dtype, **config)
    x = torch.randn(2, rows, 512, device=DEV).to(dtype)
    with torch.no_grad():
        y = module(x)
    assert y.shape == (2, rows, 300) and y.dtype == dtype
    check(y.reshape(-1, 300), x.reshape(-1, 512), unpacked(module.quantized_weight()), module.bias if bias else None)


def test_linear_is_differentiable_in_its_input():
    module = layer(256, 320, True, torch.bfloat16)
    x = torch.randn(40, 320, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = module(x)
    dy = torch.randn_like(y)
    y.backward(dy)
    check(x.grad, dy, unpacked(module.quantized_weight()).T)
    assert torch.equal(module.bias.grad, dy.sum(0))
    # a frozen layer between trainable ones, twice through the same leaves
    adapter = nn.Linear(320, 320, bias=False, device=DEV, dtype=torch.bfloat16)
    for _ in range(2):
        module(adapter(x.detach())).float().square().sum().backward()
    assert torch.isfinite(adapter.weight.grad).all() and adapter.weight.grad.abs().sum() > 0


def test_linear_refusals():
    module = layer(128, 128, False, torch.bfloat16)
    with pytest.raises(ValueError, match="activation_dtype"):
        module(torch.randn(4, 128, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError, match="columns"):
        module(torch.randn(4, 64, device=DEV, dtype=torch.bfloat16))
    kept = FourOverSixLinear(nn.Linear(128, 128, device=DEV, dtype=torch.bfloat16),
                             fos.ModuleQuantizationConfig(activation_dtype="bfloat16", keep_master_weights=True))
    with pytest.raises(ValueError, match="bfloat16"):
        kept(torch.randn(4, 128, device=DEV, dtype=torch.bfloat16))


def test_quantize_model():
    torch.manual_seed(0)
    model = nn.Sequential(nn.Linear(128, 256, device=DEV, dtype=torch.bfloat16), nn.GELU(), nn.Linear(256, 128, device=DEV, dtype=torch.bfloat16))
    fos.quantize_model(model, fos.ModelQuantizationConfig(activation_dtype="bfloat16"))
    for module in model:
        if isinstance(module, FourOverSixLinear):
            module.quantize_weight_()
    x = torch.randn(9, 128, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        hidden = model[1](model[0](x))
        check(model(x), hidden, unpacked(model[2].quantized_weight()), model[2].bias)


def experts(e, hidden, inner, dtype, **more):
    g = torch.Generator(device=DEV).manual_seed(e + hidden)

    def rand(*shape, scale):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    name = {torch.bfloat16: "bfloat16", torch.float16: "float16"}[dtype]
    return FourOverSixExperts(rand(e, 2 * inner, hidden, scale=hidden ** -0.5), rand(e, 2 * inner, scale=0.1), rand(e, hidden, inner, scale=inner ** -0.5),
                              rand(e, hidden, scale=0.1), fos.ModuleQuantizationConfig(activation_dtype=name, output_dtype=name), **more)


def plain_experts(module, x, indices, weights):
    """The layer in 64 bits on the unpacked weights."""
    down, gate_up = module.quantized_weights()
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(module.num_experts):
        token, slot = torch.where(indices == e)
        if not token.numel():
            continue
        gu = x[token].double() @ unpacked(gate_up[e]).T + module.gate_up_proj_bias[e].double()
        gate, up = gu[:, ::2].clamp(max=module.limit), gu[:, 1::2].clamp(-module.limit, module.limit)
        y = ((up + 1) * gate * torch.sigmoid(gate * module.alpha)) @ unpacked(down[e]).T + module.down_proj_bias[e].double()
        out.index_add_(0, token, y * weights[token, slot].double()[:, None])
    return out


@pytest.mark.parametrize("tokens,e,top", [(1, 8, 2), (16, 32, 4), (130, 8, 2), (600, 4, 4)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_experts(tokens, e, top, dtype, native, index):
    if not native and index == torch.int32:
        pytest.skip("the tensor operations index with int64")
    module = experts(e, 192, 128, dtype, native_elementwise=native)
    g = torch.Generator(device=DEV).manual_seed(tokens)
    x = torch.randn(tokens, 192, generator=g, device=DEV).to(dtype)
    scores, indices = torch.randn(tokens, e, generator=g, device=DEV).topk(top)
    weights = scores.softmax(-1).to(dtype)
    with torch.no_grad():
        got = module(x.reshape(1, tokens, 192), indices.to(index), weights)
    assert got.shape == (1, tokens, 192) and got.dtype == dtype
    want = plain_experts(module, x, indices, weights)
    # seven 16-bit roundings up to the hidden product's operand (its own, the bias's, +1, the gate's product with alpha, the sigmoid, two
    # products) and four behind it (its own, the bias's, the weight's, and one per expert of the sum): half a step each, of terms that the
    # clamped SwiGLU amplifies by at most 1 + alpha * limit / 4 < 4 and the sums average: 32 half steps over the norm
    eps = torch.finfo(dtype).eps / 2
    assert ((got[0].double() - want).norm() / want.norm()).item() <= 32 * eps
    assert (got[0].double() - want).abs().max().item() <= 64 * eps * want.abs().max().item()


def test_experts_nobody_goes_to():
    """An index outside the experts gives its pair nothing; a token whose experts are all outside gets zeros."""
    module = experts(4, 64, 64, torch.bfloat16)
    x = torch.randn(6, 64, device=DEV, dtype=torch.bfloat16)
    indices = torch.tensor([[0, 1], [2, 9], [-1, 3], [7, 7], [1, 0], [3, 2]], device=DEV)
    weights = torch.full((6, 2), 0.5, dtype=torch.bfloat16, device=DEV)
    got = module(x, indices, weights)
    want = plain_experts(module, x, indices, weights)
    assert (got[3] == 0).all()
    assert ((got.double() - want).norm() / want.norm()).item() <= 32 * 2.0 ** -8


def test_experts_in_a_graph():
    module = experts(8, 128, 64, torch.bfloat16)
    x = torch.randn(12, 128, device=DEV, dtype=torch.bfloat16)
    indices = torch.randint(0, 8, (12, 2), device=DEV)
    weights = torch.full((12, 2), 0.5, dtype=torch.bfloat16, device=DEV)
    module(x, indices, weights)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = module(x, indices, weights)
    for seed in range(3):
        indices.copy_(torch.randint(0, 8, (12, 2), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)))
        graph.replay()
        assert torch.equal(out, module(x, indices, weights))


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_a_block_as_a_model_runs_it(tokens):
    """Norm in 16 bits -> weight-only projection -> residual -> norm packed to NVFP4 -> block-scaled projection, against the same steps in
    64 bits on what each step was given."""
    k, n = 512, 256
    up = layer(n, k, False, torch.bfloat16)
    back = layer(k, n, False, torch.bfloat16)
    head = fos.quantize((torch.randn(384, k, device=DEV) * 0.02).bfloat16())
    x = torch.randn(tokens, k, device=DEV, dtype=torch.bfloat16)
    stream = torch.randn(tokens, k, device=DEV, dtype=torch.bfloat16)
    gain = (1 + 0.1 * torch.randn(k, device=DEV)).bfloat16()
    with torch.no_grad():
        y, stream2 = fos.rms_norm(x, gain, residual=stream)
        hidden = up(y)
        delta = back(hidden)
        packed, stream3 = fos.rms_norm(delta, gain, residual=stream2, config=fos.QuantizationConfig())
        logits = fos.quantized_matmul(packed, head)
    assert torch.equal(stream2, x + stream) and torch.equal(stream3, delta + stream2)
    check(hidden, y, unpacked(up.quantized_weight()))
    check(delta, hidden, unpacked(back.quantized_weight()))
    exact = unpacked(packed) @ unpacked(head).T
    assert ((logits.double() - exact).norm() / exact.norm()).item() <= 2.0 ** -8
