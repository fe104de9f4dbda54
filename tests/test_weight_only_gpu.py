"""Products of 16-bit activations with packed 4-bit weights against the same products in 64 bits.

The oracle takes the packed bytes apart itself (codes, scale bytes in either layout, amax) and multiplies in float64. What may
differ from it, per output: the rounding to the output's type (half a step, `eps / 2` of the value), the product with alpha and
the division that forms it (2^-23 of the value), and the fp32 sums: every addition is off by at most 2^-23 of the running sum
(tensor cores truncate), so k + 64 of them by (k + 64) * 2^-23 of the sum of the terms' magnitudes. bf16 activations that
become fp16 by a power of two are off by at most 2^-39 of the row's largest value.
"""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos
from fouroversix_b200 import _native
from fouroversix_b200.matmul import GroupLayout, StackedQuantizedTensor, grouped_weight_only_matmul
from fouroversix_b200.quantize import from_blocked

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMATS = [("nvfp4", "mse"), ("nvfp4", "static_4"), ("if4", "mse"), ("mxfp4", "static_6")]
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def unpacked(q: fos.QuantizedTensor) -> torch.Tensor:
    """What a packed tensor stands for, in 64 bits, cropped."""
    n_p, k_p = q.padded_shape
    block = q.dtype.block_size
    nb = k_p // block
    v = q.values.reshape(n_p, k_p // 2).long()
    code = torch.stack([v % 16, v // 16], -1).reshape(n_p, nb, block)
    number = torch.tensor(E2M1 + [-x for x in E2M1], dtype=torch.float64, device=v.device)[code]
    flat = q.scale_factors.reshape(-1).view(torch.uint8)
    byte = (from_blocked(flat, (n_p, nb)) if q.scale_factors_are_in_blackwell_layout else flat.reshape(n_p, nb)).long()
    if q.dtype == fos.DataType.mxfp4:
        scale = torch.where(byte == 0, 0.0, torch.exp2(byte.double() - 127))
    else:
        scale = (byte % 128).to(torch.uint8).view(torch.float8_e4m3fn).double()
        if q.dtype == fos.DataType.if4:
            ints = (code - 16 * (code // 8)).double() * (6 / 7)
            number = torch.where((byte >= 128).unsqueeze(-1), ints, number)
        ceiling = {"static_6": 2688, "static_4": 1792}.get(q.scale_rule.value, 1536) if q.dtype == fos.DataType.nvfp4 else 2688
        if q.round_style == fos.RoundStyle.stochastic_unbiased:
            ceiling *= 16 / 17
        scale = scale * (q.amax.double() / ceiling)
    return (number * scale.unsqueeze(-1)).reshape(n_p, k_p)[:q.original_shape[0], :q.original_shape[1]]


def check(got: torch.Tensor, x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None = None) -> None:
    x = x.double()
    want, mass = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        want = want + bias.double()
        mass = mass + bias.double().abs()
    k = x.shape[1]
    eps = torch.finfo(got.dtype).eps
    smallest = torch.finfo(got.dtype).smallest_normal * eps
    largest = x.abs().amax(-1, keepdim=True) * w.abs().sum(-1) * 2.0 ** -39
    bound = (eps / 2 + 2.0 ** -23) * want.abs() + (k + 64) * 2.0 ** -23 * mass + largest + smallest
    off = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"worst {(off / bound).max().item():.2f} times the bound"
    # the sums' errors have either sign: over all outputs they stay far below the worst case
    norm = (off.norm() / want.norm().clamp_min(1e-300)).item()
    assert norm <= eps / 2 + 1e-5, f"relative error {norm:.2e}"


def tensors(rows: int, n: int, k: int, dtype: torch.dtype, seed: int = 0):
    g = torch.Generator(device=DEV).manual_seed(seed + 1000 * rows + n + 7 * k)
    x = torch.randn(rows, k, generator=g, device=DEV)
    x[:, ::97] *= 20
    w = torch.randn(n, k, generator=g, device=DEV) * 0.02
    return x.to(dtype), w.to(dtype), (torch.randn(n, generator=g, device=DEV) * 0.1)


@pytest.mark.parametrize("rows,n,k", [
    (1, 1, 1), (1, 128, 64), (1, 4096, 4096), (2, 130, 200), (3, 257, 1000), (4, 64, 8192), (5, 1000, 136), (7, 384, 14336),
    (8, 640, 2048), (9, 513, 2047), (15, 128, 129), (16, 5000, 2880), (17, 200, 65), (31, 256, 1024), (32, 4096, 512), (33, 300, 777),
    (64, 512, 512), (65, 1153, 320), (100, 128, 4096), (128, 256, 256), (129, 130, 1100), (300, 1000, 2880), (513, 640, 96),
    (40, 40, 40), (20, 8, 8), (700, 16, 56), (600, 700, 24),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,rule", FORMATS)
def test_product(rows, n, k, dtype, fmt, rule):
    x, w, _ = tensors(rows, n, k, dtype)
    q = fos.quantize(w, fos.QuantizationConfig(dtype=fmt, scale_rule=rule))
    got = fos.weight_only_matmul(x, q)
    assert got.dtype == dtype and got.shape == (rows, n)
    check(got, x, unpacked(q))


@pytest.mark.parametrize("rows", [1, 12, 40, 300])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bias_and_output_types(rows, out, dtype):
    x, w, bias = tensors(rows, 391, 520, dtype)
    q, bias = fos.quantize(w), bias.to(out)
    got = fos.weight_only_matmul(x, q, bias=bias, out_dtype=out)
    assert got.dtype == out
    x64 = x.double()
    want = x64 @ unpacked(q).T + bias.double()
    mass = x64.abs() @ unpacked(q).abs().T + bias.double().abs()
    bound = torch.finfo(out).eps / 2 * want.abs() + (520 + 64) * 2.0 ** -23 * mass + 1e-9
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("rows", [1, 5, 16, 50, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strides_and_alignment(rows, dtype):
    """Inputs that are columns of a wider tensor, start off 16 bytes, are transposed, broadcast or have more dimensions."""
    k, n = 328, 200
    _, w, _ = tensors(rows, n, k, dtype)
    q = fos.quantize(w)
    w64 = unpacked(q)
    g = torch.Generator(device=DEV).manual_seed(rows)
    wide = torch.randn(rows, k + 40, generator=g, device=DEV).to(dtype)
    for view in (wide[:, 8:8 + k], wide[:, 3:3 + k], torch.randn(k, rows, generator=g, device=DEV).to(dtype).T,
                 wide[:1, :k].expand(rows, k), wide[:, :k].flip(0)):
        check(fos.weight_only_matmul(view, q), view, w64)
    three = wide[:, :k].reshape(rows, 1, k).expand(rows, 2, k)
    got = fos.weight_only_matmul(three, q)
    assert got.shape == (rows, 2, n)
    check(got.reshape(-1, n), three.reshape(-1, k), w64)
    assert fos.weight_only_matmul(wide[0, :k], q).shape == (n,)
    assert fos.weight_only_matmul(wide[:0, :k], q).shape == (0, n)


@pytest.mark.parametrize("rows", [1, 16, 40, 300])
@pytest.mark.parametrize("fmt,rule", FORMATS)
def test_far_apart_magnitudes(rows, fmt, rule):
    """Rows of bf16 whose largest values lie near both ends of the type's range, rows of zeros, subnormals."""
    k, n = 512, 256
    x, w, _ = tensors(rows, n, k, torch.bfloat16, seed=3)
    q = fos.quantize(w, fos.QuantizationConfig(dtype=fmt, scale_rule=rule))
    w64 = unpacked(q)
    for exponent in (-110, -60, 60, 100):
        big = (x.double() * 2.0 ** exponent).bfloat16()
        got = fos.weight_only_matmul(big, q, out_dtype=torch.float32)
        want, mass = big.double() @ w64.T, big.double().abs() @ w64.abs().T
        assert ((got.double() - want).abs() <= (k + 64) * 2.0 ** -23 * mass + 2.0 ** -149 + 2.0 ** -126 * (exponent < 0)).all()
    zero = torch.zeros_like(x)
    assert (fos.weight_only_matmul(zero, q) == 0).all()
    mixed = x.clone()
    mixed[:, 0] = 3e4                                       # one outlier; the others keep their digits
    check(fos.weight_only_matmul(mixed, q), mixed, w64)


@pytest.mark.parametrize("rows", [1, 9, 40, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_infinities_and_nan_stay_in_their_rows(rows, dtype):
    k, n = 256, 192
    x, w, _ = tensors(rows + 3, n, k, dtype, seed=5)
    w = w.abs() + 0.01                                      # no weight is zero
    q = fos.quantize(w)
    w64 = unpacked(q)
    assert (w64 != 0).all()
    x[0, 5], x[rows // 2 + 1, 100], x[rows + 2, 255] = float("inf"), float("nan"), float("-inf")
    got = fos.weight_only_matmul(x, q)
    assert (got[0] == float("inf")).all() and (got[rows + 2] == float("-inf")).all()
    assert torch.isnan(got[rows // 2 + 1]).all()
    keep = [r for r in range(rows + 3) if r not in (0, rows // 2 + 1, rows + 2)]
    if keep:
        check(got[keep], x[keep], w64)


@pytest.mark.parametrize("rows", [4, 64, 256])
def test_other_ways_to_pack(rows):
    """2-D blocks, a transposed source, stochastic rounding with and without the 16/17, IF4 in either layout, every rule."""
    k, n = 320, 256
    x, w, _ = tensors(rows, n, k, torch.bfloat16, seed=9)
    for config in (dict(block_scale_2d=True), dict(transpose=True), dict(round_style="stochastic"), dict(round_style="stochastic_unbiased"),
                   dict(scale_rule="mae"), dict(scale_rule="abs_max"), dict(dtype="if4", block_scale_2d=True),
                   dict(dtype="mxfp4", scale_rule="static_4")):
        q = fos.quantize(w.T.contiguous() if config.get("transpose") else w, fos.QuantizationConfig(**config))
        check(fos.weight_only_matmul(x, q), x, unpacked(q))
    q = fos.quantize(w, fos.QuantizationConfig(dtype="if4"))
    from fouroversix_b200.quantize import to_blocked

    n_p, k_p = q.padded_shape
    tiled = fos.QuantizedTensor(q.values, to_blocked(q.scale_factors.reshape(n_p, k_p // 16)), q.amax, q.dtype, q.original_shape,
                                q.scale_rule, q.round_style, q.padded_shape, scale_factors_are_in_blackwell_layout=True)
    assert torch.equal(fos.weight_only_matmul(x, tiled), fos.weight_only_matmul(x, q))


@pytest.mark.parametrize("rows,n,k", [(1, 128, 64), (5, 200, 328), (40, 391, 520), (64, 1000, 136), (129, 640, 1100), (300, 1000, 2880), (513, 96, 640),
                                      (33, 4096, 192), (256, 256, 257), (40, 40, 40), (20, 8, 8), (700, 56, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,rule", FORMATS)
def test_gradient(rows, n, k, dtype, fmt, rule):
    """The gradient of the input against the formula, dx = dy W, and of the bias."""
    x, w, bias = tensors(rows, n, k, dtype, seed=13)
    q = fos.quantize(w, fos.QuantizationConfig(dtype=fmt, scale_rule=rule))
    x.requires_grad_()
    bias = bias.to(dtype).requires_grad_()
    y = fos.weight_only_matmul(x, q, bias=bias)
    dy = (torch.randn(rows, n, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV) * 1e-3).to(dtype)
    dx, db = torch.autograd.grad(y, (x, bias), dy)
    assert dx.dtype == dtype and dx.shape == x.shape
    check(dx, dy, unpacked(q).T)
    assert torch.equal(db, dy.sum(0))
    # another type out than in, and a gradient that is not contiguous
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    y = fos.weight_only_matmul(x, q, out_dtype=other)
    wide = torch.zeros(n, rows, dtype=other, device=DEV)
    wide.copy_(dy.T)
    dx, = torch.autograd.grad(y, x, wide.T)
    exact = wide.T.double() @ unpacked(q)
    mass = wide.T.double().abs() @ unpacked(q).abs()
    bound = (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * exact.abs() + (n + 64) * 2.0 ** -23 * mass + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((dx.double() - exact).abs() <= bound).all()


def test_gradient_against_differences():
    """(f(x + h v) - f(x - h v)) / 2h is exact for a linear f but for the outputs' rounding: fp32 outputs, a step that fp16 holds."""
    rows, n, k = 24, 96, 128
    x, w, _ = tensors(rows, n, k, torch.float16, seed=17)
    q = fos.quantize(w)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = (x * 8).round() / 8
    v = torch.randint(-2, 3, (rows, k), generator=g, device=DEV).half()
    dy = torch.randn(rows, n, generator=g, device=DEV).half()
    step = 0.5
    up, down = (fos.weight_only_matmul(x + s * v, q, out_dtype=torch.float32).double() for s in (step, -step))
    slope = ((up - down) / (2 * step) * dy.double()).sum()
    leaf = x.clone().requires_grad_()
    dx, = torch.autograd.grad(fos.weight_only_matmul(leaf, q), leaf, dy)
    mass = ((dy.double().abs() @ unpacked(q).abs()) * v.double().abs()).sum() + (x.double().abs() @ unpacked(q).abs().T * dy.double().abs()).sum()
    # fp16 rounding of dx (2^-11 of it) and the sums in fp32 ((n + k + 128) * 2^-23)
    assert (slope - (dx.double() * v.double()).sum()).abs() <= (2.0 ** -11 + (n + k + 128) * 2.0 ** -23) * mass


COUNTS = {
    "ragged": [5, 0, 30, 128, 1, 0, 77, 257],
    "tokens": [0, 0, 1, 0, 1, 0, 0, 2],
    "one": [33],
    "many": [((7 * i) % 23) * ((i % 3) != 0) for i in range(48)],
    "large": [700, 3, 1200, 90],
}


@pytest.mark.parametrize("name", list(COUNTS))
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,rule", [("nvfp4", "mse"), ("if4", "mse"), ("mxfp4", "static_6")])
def test_grouped(name, padded, dtype, fmt, rule):
    """Groups with and without padding, rows fetched by index (some of them outside x) or lying in order."""
    counts, k, n, tokens = COUNTS[name], 328, 200, 61
    g = torch.Generator(device=DEV).manual_seed(len(counts))
    x = (torch.randn(tokens, k, generator=g, device=DEV)).to(dtype)
    config = fos.QuantizationConfig(dtype=fmt, scale_rule=rule)
    weights = [fos.quantize((torch.randn(n, k, generator=g, device=DEV) * (0.02 + 0.01 * e)).to(dtype), config) for e in range(len(counts))]
    first = weights[0]
    stacked = StackedQuantizedTensor(torch.stack([w.values for w in weights]), torch.stack([w.scale_factors.reshape(-1).view(torch.uint8) for w in weights]).view(
        first.scale_factors.dtype), torch.cat([w.amax for w in weights]), first.dtype, first.scale_rule, first.original_shape, first.padded_shape)
    table = torch.tensor(counts, device=DEV)
    layout = GroupLayout.from_counts(table, sum(counts)) if padded else GroupLayout.compact(table, sum(counts) + 3)
    index = torch.randint(0, tokens, (layout.capacity,), generator=g, device=DEV, dtype=torch.int32)
    index[::11] = -1
    index[5::13] = tokens
    rows = torch.where(((index >= 0) & (index < tokens)).unsqueeze(1), x[index.clamp(0, tokens - 1).long()], torch.zeros((), dtype=dtype, device=DEV))
    got = grouped_weight_only_matmul(x, stacked, layout, row_index=index)
    again = grouped_weight_only_matmul(rows, stacked, layout)
    assert torch.equal(got, again)
    start = layout.group_start.tolist()
    free = torch.ones(layout.capacity, dtype=torch.bool, device=DEV)
    for e, c in enumerate(counts):
        mine = slice(start[e], start[e] + c)
        free[mine] = False
        if c:
            check(got[mine], rows[mine], unpacked(weights[e]))
    assert (got[free] == 0).all()
    # a given buffer: all of it written, nothing around it
    buffer = torch.full((layout.capacity + 2, n + 8), 7.0, dtype=dtype, device=DEV)
    grouped_weight_only_matmul(x, stacked, layout, row_index=index, out=buffer[1:-1, :n])
    assert torch.equal(buffer[1:-1, :n], got)
    assert (buffer[0] == 7).all() and (buffer[-1] == 7).all() and (buffer[:, n:] == 7).all()


def test_tables_that_point_anywhere_stay_inside():
    """Group tables a caller got wrong: rows beyond the buffer, negative counts. Nothing outside the output is written."""
    k, n, cap = 64, 128, 40
    x, w, _ = tensors(cap, n, k, torch.bfloat16)
    q = fos.quantize(w)
    stacked = StackedQuantizedTensor.stack([q, q, q])
    start = torch.tensor([-5, 30, 200, 1 << 30], dtype=torch.int32, device=DEV)
    rows = torch.tensor([12, 50, 9], dtype=torch.int32, device=DEV)
    buffer = torch.full((cap + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
    grouped_weight_only_matmul(x, stacked, GroupLayout(start, rows, cap, 3), out=buffer[1:-1])
    torch.cuda.synchronize()
    assert (buffer[0] == 7).all() and (buffer[-1] == 7).all()


@pytest.mark.parametrize("rows", [1, 16, 64, 300])
def test_streams_graphs_and_repeats(rows):
    """The same bits from another stream, from a replayed graph and from every repeat."""
    x, w, _ = tensors(rows, 640, 1024, torch.bfloat16, seed=11)
    q = fos.quantize(w)
    want = fos.weight_only_matmul(x, q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = fos.weight_only_matmul(x, q)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(other, want)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fos.weight_only_matmul(held, q)
    for scale in (1, 2):
        held.copy_(x * scale)
        graph.replay()
        assert torch.equal(out, fos.weight_only_matmul(x * scale, q))
    for _ in range(3):
        assert torch.equal(fos.weight_only_matmul(x, q), want)
    assert _native.wait_failure_site() == 0


def streams(rows, n_p, k_p, groups=0):
    """Whether a product's stages are dealt out evenly to the CTAs: its workspace then has room for two parts of a tile for each of 148."""
    from fouroversix_b200 import _native

    return _native.lib().fos_weight_only_workspace_bytes(rows, n_p, k_p, groups, 0) >= 2 * 148 * 128 * 128 * 4


@pytest.mark.parametrize("rows,n,k", [(12, 16640, 4160), (16, 10240, 8192), (20, 9590, 2810), (40, 9700, 3584), (300, 6528, 4220), (600, 3840, 4288),
                                      (1000, 2500, 4800)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt,rule", FORMATS)
def test_stages_dealt_out_evenly(rows, n, k, dtype, fmt, rule):
    """Tiles that begin and end within a CTA's share: a sum is made of up to four parts."""
    x, w, bias = tensors(rows, n, k, dtype, seed=21)
    q = fos.quantize(w, fos.QuantizationConfig(dtype=fmt, scale_rule=rule))
    assert streams(rows, *q.padded_shape)
    check(fos.weight_only_matmul(x, q), x, unpacked(q))
    bias = bias.to(dtype)
    got = fos.weight_only_matmul(x[:, :], q, bias=bias)
    check(got, x, unpacked(q), bias)
    for _ in range(3):
        assert torch.equal(fos.weight_only_matmul(x, q, bias=bias), got)
    far = torch.empty(rows, k + 9, dtype=dtype, device=DEV)
    far[:, 1:k + 1] = x                                      # rows that no 16-byte load can take
    assert torch.equal(fos.weight_only_matmul(far[:, 1:k + 1], q, bias=bias), got)


@pytest.mark.parametrize("counts", [[400, 0, 1, 599], [250, 250, 250, 250], [0, 0, 0, 1000], [1000, 0, 0, 0]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_grouped_stages_dealt_out_evenly(counts, dtype):
    k, n, tokens = 4088, 4096, 333
    assert streams(1007, n, 4096, len(counts))
    g = torch.Generator(device=DEV).manual_seed(sum(counts) + counts[0])
    x = torch.randn(tokens, k, generator=g, device=DEV).to(dtype)
    weights = [fos.quantize((torch.randn(n, k, generator=g, device=DEV) * 0.02).to(dtype)) for _ in counts]
    layout = GroupLayout.compact(torch.tensor(counts, device=DEV), 1007)
    index = torch.randint(-3, tokens + 3, (1007,), generator=g, device=DEV, dtype=torch.int32)
    got = grouped_weight_only_matmul(x, StackedQuantizedTensor.stack(weights), layout, row_index=index)
    rows = torch.where(((index >= 0) & (index < tokens)).unsqueeze(1), x[index.clamp(0, tokens - 1).long()], torch.zeros((), dtype=dtype, device=DEV))
    at = 0
    for w, c in zip(weights, counts):
        if c:
            check(got[at:at + c], rows[at:at + c], unpacked(w))
        at += c
    assert (got[at:] == 0).all()
    assert torch.equal(grouped_weight_only_matmul(rows, StackedQuantizedTensor.stack(weights), layout), got)


def test_parts_of_two_graphs_and_streams_stay_apart():
    """Two captured products and an eager one, on three streams at once: each has counters and parts of its own."""
    x, w, _ = tensors(16, 10240, 8192, torch.bfloat16, seed=22)
    q = fos.quantize(w)
    assert streams(16, *q.padded_shape)
    xs = [x, x * 2, x * 4]
    wants = [fos.weight_only_matmul(v, q) for v in xs]
    graphs, outs = [], []
    for v in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fos.weight_only_matmul(v, q))
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
        with torch.cuda.stream(sides[2]):
            eager = fos.weight_only_matmul(xs[2], q)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1]) and torch.equal(eager, wants[2])


@pytest.mark.parametrize("rows", [1, 16])
def test_few_rows_that_are_long(rows):
    """More values of K than shared memory holds of 16 rows."""
    x, w, _ = tensors(rows, 100, 60000, torch.bfloat16, seed=23)
    q = fos.quantize(w)
    check(fos.weight_only_matmul(x, q), x, unpacked(q))


@pytest.mark.parametrize("rows", [4, 40, 500])
def test_forward_and_backward_in_a_graph(rows):
    """Captured after an eager pass on a side stream whose graph is gone (autograd ties a leaf to the stream of the graph that it lives in);
    replayed with other values in the leaf."""
    x, w, bias = tensors(rows, 640, 1024, torch.bfloat16, seed=31)
    q, bias = fos.quantize(w), bias.bfloat16()
    leaf, dy = x.clone().requires_grad_(), torch.randn(rows, 640, device=DEV).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(fos.weight_only_matmul(leaf, q, bias=bias), leaf, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fos.weight_only_matmul(leaf, q, bias=bias)
        dx, = torch.autograd.grad(y, leaf, dy)
    for scale in (1.0, 0.5):
        with torch.no_grad():
            leaf.copy_(x * scale)
        graph.replay()
        again = fos.weight_only_matmul(leaf, q, bias=bias)
        assert torch.equal(y, again) and torch.equal(dx, torch.autograd.grad(again, leaf, dy)[0])


def test_overlapping_groups_stay_inside_where_stages_are_dealt_out():
    """Groups that each claim all rows: more tiles than the workspace has counters for. Nothing outside the output is written."""
    k, n, cap, groups = 4096, 4096, 1007, 4
    assert streams(cap, n, k, groups)
    x = torch.randn(cap, k, device=DEV).bfloat16()
    q = fos.quantize((torch.randn(n, k, device=DEV) * 0.02).bfloat16())
    stacked = StackedQuantizedTensor.stack([q] * groups)
    start = torch.zeros(groups + 1, dtype=torch.int32, device=DEV)
    rows = torch.full((groups,), 1 << 20, dtype=torch.int32, device=DEV)
    buffer = torch.full((cap + 2, n), 7.0, dtype=torch.bfloat16, device=DEV)
    grouped_weight_only_matmul(x, stacked, GroupLayout(start, rows, cap, groups), out=buffer[1:-1])
    torch.cuda.synchronize()
    assert (buffer[0] == 7).all() and (buffer[-1] == 7).all()


def test_rows_of_infinities_stay_alone():
    """A row with an infinity or NaN leaves the others what they are, on every kernel."""
    for rows, n, k in ((3, 640, 1024), (16, 10240, 8192), (40, 640, 1024), (333, 1000, 2880), (2048, 2560, 4096)):
        x, w, _ = tensors(rows, n, k, torch.bfloat16, seed=33)
        q = fos.quantize(w)
        want = fos.weight_only_matmul(x, q)
        x[1, 5], x[2, 7] = float("inf"), float("nan")
        got = fos.weight_only_matmul(x, q)
        assert torch.isnan(got[2]).all() and not torch.isfinite(got[1]).any()
        keep = [i for i in range(rows) if i not in (1, 2)]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("counts", [[0] * 40 + [1] + [0] * 9, [0, 0, 3] + [0] * 20 + [2, 0, 1], [0] * 30, [5] + [0] * 250, [0] * 255 + [4]])
@pytest.mark.parametrize("gap", [0, 2])
def test_more_groups_than_rows(counts, gap):
    """A few rows among many groups, with rows of nobody in front of every group."""
    k, n = 264, 200
    g = torch.Generator(device=DEV).manual_seed(len(counts))
    weight = fos.quantize((torch.randn(n, k, generator=g, device=DEV) * 0.02).bfloat16())
    other = fos.quantize((torch.randn(n, k, generator=g, device=DEV) * 0.03).bfloat16())
    stacked = StackedQuantizedTensor.stack([weight, other] * (len(counts) // 2) + [weight] * (len(counts) % 2))
    rows = torch.tensor(counts, dtype=torch.int32, device=DEV)
    first = (rows > 0).cumsum(0) * gap + rows.cumsum(0) - rows
    capacity = sum(counts) + gap * sum(c > 0 for c in counts) + 1
    start = torch.cat([first, torch.tensor([capacity - 1], device=DEV)]).int()
    layout = GroupLayout(start, rows, capacity, len(counts))
    x = torch.randn(capacity, k, generator=g, device=DEV).bfloat16()
    got = grouped_weight_only_matmul(x, stacked, layout)
    free = torch.ones(capacity, dtype=torch.bool, device=DEV)
    for e, c in enumerate(counts):
        if c:
            at = int(start[e])
            free[at:at + c] = False
            check(got[at:at + c], x[at:at + c], unpacked(other if e % 2 and e < len(counts) - len(counts) % 2 else weight))
    assert (got[free] == 0).all()
