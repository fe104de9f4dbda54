"""The operators around 4-bit weights whose speed is followed, with their plain forms.

`do` names the operator of a case:
  product   16-bit activations times a packed 4-bit weight (`weight_only_matmul`), with the input's gradient where `grad`
  experts   the same for rows grouped by expert, ragged, fetched by index (`grouped_weight_only_matmul`)
  norm      root-mean-square norm of the input plus the residual stream, as it is or packed to 4 bits (`rms_norm`)

Weights are N(0, 0.02^2), activations N(0, 1) with one channel in a hundred times 20, gradients N(0, 1e-3^2), residuals
N(0, 2^2). Everything is made from the seed on the GPU.
"""

from __future__ import annotations

import math

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "fp16": torch.float16}
OUT = {"bf16": "bfloat16", "fp16": "float16"}
BLOCK = {"nvfp4": 16, "if4": 16, "mxfp4": 32}
BYTES = {"nvfp4": 0.5 + 1 / 16, "if4": 0.5 + 1 / 16, "mxfp4": 0.5 + 1 / 32}     # of a packed value with its scale
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-5

LARGEST_FLOPS = 2.0 * 4096 * 8192 * 10240
LARGEST_VALUES = 8192 * 8192


def listed():
    return [
        # one token through a small projection: nothing but latency
        {"name": "product_token", "do": "product", "tokens": 1, "k": 4096, "n": 4096, "type": "bf16", "format": "nvfp4", "bias": False, "grad": False},
        # one decoding step of 16 sequences through the grouped-query projection of an 8192-wide model
        {"name": "product_decode", "do": "product", "tokens": 16, "k": 8192, "n": 10240, "type": "bf16", "format": "nvfp4", "bias": False, "grad": False},
        # one decoding step of 32 sequences through an MLP down projection kept in MXFP4
        {"name": "product_decode_mx", "do": "product", "tokens": 32, "k": 14336, "n": 4096, "type": "bf16", "format": "mxfp4", "bias": False, "grad": False},
        # a short prompt of an odd length, fp16, IF4, with a bias, sizes off the tile grid
        {"name": "product_ragged", "do": "product", "tokens": 333, "k": 2880, "n": 5000, "type": "fp16", "format": "if4", "bias": True, "grad": False},
        # an ordinary prompt
        {"name": "product_prompt", "do": "product", "tokens": 4096, "k": 8192, "n": 10240, "type": "bf16", "format": "nvfp4", "bias": False, "grad": False},
        # training adapters around a frozen 4-bit weight: the output and the input's gradient
        {"name": "product_frozen", "do": "product", "tokens": 2048, "k": 4096, "n": 14336, "type": "bf16", "format": "nvfp4", "bias": False, "grad": True},
        # a mixture-of-experts layer's first projection: a decoding step of 16 sequences, and a prompt
        {"name": "experts_decode", "do": "experts", "tokens": 16, "top": 4, "experts": 32, "k": 2880, "n": 5760, "type": "bf16", "format": "nvfp4"},
        {"name": "experts_prompt", "do": "experts", "tokens": 2048, "top": 4, "experts": 32, "k": 2880, "n": 5760, "type": "bf16", "format": "nvfp4"},
        # the norm before a projection in 4 bits: a decoding step, and a batch of prompts
        {"name": "norm_decode", "do": "norm", "rows": 16, "cols": 8192, "type": "bf16", "format": "nvfp4", "rule": "mse", "residual": True},
        {"name": "norm_prompt", "do": "norm", "rows": 8192, "cols": 8192, "type": "bf16", "format": "nvfp4", "rule": "mse", "residual": True},
        # the first norm of a model (no residual yet), fp16, MXFP4, an odd number of rows
        {"name": "norm_mx_ragged", "do": "norm", "rows": 333, "cols": 2880, "type": "fp16", "format": "mxfp4", "rule": "static_6", "residual": False},
        # the norm before a product with a 4-bit weight: 16 bits out
        {"name": "norm_plain", "do": "norm", "rows": 4096, "cols": 4096, "type": "bf16", "format": "none", "rule": "none", "residual": True},
    ]


def _log(rng, low, high, unit=1):
    """A multiple of `unit` between low and high, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(unit, min(high // unit, round(v / unit)) * unit)


def draw(rng):
    do = rng.choice(["product", "product", "product", "experts", "norm", "norm"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if do == "product":
        grad = rng.random() < 0.2
        k, n = _log(rng, 1024, 14336, rng.choice([1, 8, 64])), _log(rng, 1024, 14336, rng.choice([1, 8, 8]))
        tokens = _log(rng, 1, 4096)
        while 2.0 * (1 + grad) * tokens * k * n > LARGEST_FLOPS:
            tokens //= 2
        return {"do": do, "tokens": tokens, "k": k, "n": n, "type": kind, "format": rng.choice(["nvfp4", "nvfp4", "if4", "mxfp4"]),
                "bias": rng.random() < 0.25, "grad": grad}
    if do == "experts":
        return {"do": do, "tokens": _log(rng, 1, 2048), "top": rng.choice([1, 2, 4]), "experts": rng.choice([8, 16, 32]),
                "k": _log(rng, 512, 2880, 8), "n": _log(rng, 512, 5760, 8), "type": kind, "format": rng.choice(["nvfp4", "nvfp4", "if4", "mxfp4"])}
    rows, cols = _log(rng, 1, 8192), _log(rng, 512, 8192, rng.choice([1, 8, 64]))
    form, rule = rng.choice([("nvfp4", "mse"), ("nvfp4", "mse"), ("nvfp4", "static_6"), ("mxfp4", "static_6"), ("none", "none")])
    return {"do": do, "rows": rows, "cols": cols, "type": kind, "format": form, "rule": rule, "residual": rng.random() < 0.7}


# ---------------------------------------------------------------------------------------------------------- inputs

def _up(v, unit):
    return -(-v // unit) * unit


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _activations(g, rows, cols, case):
    x = _randn(g, rows, cols)
    x[:, torch.randperm(cols, generator=g, device="cuda")[: max(1, cols // 100)]] *= 20
    return x.to(TORCH[case["type"]])


def _tiles(scales):
    """Scales [rows, blocks of a row], a multiple of 128 by one of 4, in the order of 128 x 4 tiles."""
    rows, cols = scales.shape
    return scales.reshape(rows // 128, 4, 32, cols // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1).contiguous()


def _packed_weight(g, n, k, case):
    """What a checkpoint in 4 bits holds: codes [n padded to 128, k padded to 4 blocks / 2], scales and the largest magnitude."""
    form, block = case["format"], BLOCK[case["format"]]
    n_p, k_p = _up(n, 128), _up(k, 4 * block)
    w = torch.zeros(n_p, k_p, device="cuda")
    w[:n, :k] = _randn(g, n, k) * 0.02
    amax = w.abs().amax().reshape(1)
    blocks = w.reshape(n_p, k_p // block, block)
    top = blocks.abs().amax(-1)
    if form == "mxfp4":
        exponent = torch.where(top > 0, torch.ceil(torch.log2((top / 6).clamp_min(1e-30))), -127.0)
        scales, step = (exponent + 127).to(torch.uint8), torch.exp2(exponent)
    else:
        stored = (top * (448.0 / amax)).to(torch.float8_e4m3fn)
        scales, step = stored.view(torch.uint8), stored.float() * (amax / 2688.0)
    units = blocks / torch.where(step > 0, step, torch.inf).unsqueeze(-1)
    grid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    codes = torch.bucketize(units.abs(), grid).to(torch.uint8) | ((units < 0).to(torch.uint8) << 3)
    if form == "if4":                                       # every other block, at random, on the integer grid
        whole = torch.rand(n_p, k_p // block, generator=g, device="cuda") < 0.5
        ints = (units * (7.0 / 6.0)).round().clamp(-7, 7).to(torch.int8).view(torch.uint8) & 15
        codes = torch.where(whole.unsqueeze(-1), ints, codes)
        scales = torch.where(whole, scales | 128, scales)
    codes = codes.reshape(n_p, k_p // 2, 2)
    values = codes[..., 0] | (codes[..., 1] << 4)
    flat = scales.reshape(-1) if form == "if4" else _tiles(scales)
    flat = flat.view(torch.float8_e8m0fnu if form == "mxfp4" else torch.float8_e4m3fn)
    return values, flat, torch.ones_like(amax) if form == "mxfp4" else amax


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, do = TORCH[case["type"]], case["do"]
    state = {"case": case}
    if do == "norm":
        rows, cols = case["rows"], case["cols"]
        state["x"] = _activations(g, rows, cols, case)
        state["residual"] = (_randn(g, rows, cols) * 2).to(kind) if case["residual"] else None
        state["weight"] = (1 + 0.1 * _randn(g, cols)).to(kind)
        return state
    n, k, tokens = case["n"], case["k"], case["tokens"]
    state["x"] = _activations(g, tokens, k, case)
    if do == "product":
        state["weight"] = _packed_weight(g, n, k, case)
        state["bias"] = (_randn(g, n) * 0.1).to(kind) if case["bias"] else None
        if case["grad"]:
            state["x"].requires_grad_()
            state["dy"] = (_randn(g, tokens, n) * 1e-3).to(kind)
        return state
    experts, top = case["experts"], case["top"]
    packed = [_packed_weight(g, n, k, case) for _ in range(experts)]
    state["weight"] = (torch.stack([p[0] for p in packed]), torch.stack([p[1].view(torch.uint8) for p in packed]).view(packed[0][1].dtype),
                       torch.cat([p[2] for p in packed]))
    # some experts are asked for more often than others; a token goes to `top` different ones
    scores = _randn(g, tokens, experts) + 0.5 * _randn(g, 1, experts)
    expert = scores.topk(top).indices.reshape(-1)
    order = torch.argsort(expert, stable=True)
    counts = torch.bincount(expert, minlength=experts)
    state["row_index"] = (order // top).to(torch.int32)
    state["group_rows"] = counts.to(torch.int32)
    state["group_start"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    state["most"] = int(counts.max())
    return state


# ------------------------------------------------------------------------------------------------------ plain forms

def _plain_weight(weight, case):
    """The numbers that packed weights [..., n padded, k padded] stand for, without the tensor's own factor, in 32 bits."""
    values, scales, _ = weight
    block = BLOCK[case["format"]]
    *lead, n_p, half = values.shape
    nb = 2 * half // block
    code = torch.stack([values & 15, values >> 4], -1).reshape(*lead, n_p, nb, block)
    number = torch.tensor(E2M1 + tuple(-v for v in E2M1), device="cuda")[code.int()]
    if case["format"] == "if4":
        byte = scales.view(torch.uint8).reshape(*lead, n_p, nb)
        signed = torch.tensor([*range(8), *range(-8, 0)], device="cuda", dtype=torch.float32) * 6
        # seven times the values, which 32 bits hold exactly
        number = torch.where((byte >= 128).unsqueeze(-1), signed[code.int()], number * 7)
        step = (byte & 127).view(torch.float8_e4m3fn).float()
    else:
        tiles = scales.view(torch.uint8).reshape(*lead, n_p // 128, nb // 4, 32, 4, 4)
        byte = tiles.transpose(-4, -2).reshape(*lead, n_p, nb)
        step = (byte.int() << 23).view(torch.float32) if case["format"] == "mxfp4" else byte.view(torch.float8_e4m3fn).float()
    return (number * step.unsqueeze(-1)).reshape(*lead, n_p, 2 * half)


def _factor(weight, case):
    """What the tensor's largest magnitude makes of those numbers."""
    return {"nvfp4": 1 / 2688, "if4": 1 / (2688 * 7), "mxfp4": 1.0}[case["format"]] * weight[2]


def _plain_quantized(y, case):
    """The values that 4-bit packing leaves of y [rows, cols] (16-bit numbers held in 32 bits), and the largest magnitude."""
    rows, cols = y.shape
    block = BLOCK[case["format"]]
    width = _up(cols, block)
    b = torch.nn.functional.pad(y, (0, width - cols)).reshape(rows, width // block, block)
    top = b.abs().amax(-1, keepdim=True)
    if case["format"] == "mxfp4":
        bits = (top / 6.0).view(torch.int32)
        step = torch.where(bits & 0x7FFFFF != 0, (bits >> 23) + 1, bits >> 23).bitwise_left_shift(23).view(torch.float32)
        out = _to_e2m1(torch.where(step > 0, b / step, 0.0)) * step
        return out.reshape(rows, width)[:, :cols], torch.ones(1, device=y.device)
    amax = y.abs().amax().reshape(1)
    adaptive = case["rule"] == "mse"
    ceiling = 1536.0 if adaptive else 2688.0
    encode = torch.where(amax > 0, ceiling / amax, 0.0)
    decode = 1.0 / (ceiling / amax)

    def candidate(stretch):
        s = (top / 6.0 * encode * stretch).to(torch.float8_e4m3fn).float()
        q = _to_e2m1(torch.where(s > 0, b * (1.0 / (decode * s)), 0.0))
        return q * s * amax / ceiling

    out = candidate(1.0)
    if adaptive:
        other = candidate(1.5)
        out = torch.where(_error(other, b) < _error(out, b), other, out)
    return out.reshape(rows, width)[:, :cols], amax


def _to_e2m1(v):
    a = v.abs()
    r = torch.where(a < 2, (2 * a).round() / 2, torch.where(a < 4, a.round(), 2 * (a / 2).round()))
    return torch.copysign(r, v)


def _error(have, want):
    """The sum of a block's 16 squared differences, added in the order that decides between two scales."""
    e = (have - want).square()
    p = e[..., :8] + e[..., 8:]
    return (p[..., :1] + p[..., 1:2] + p[..., 2:3] + p[..., 3:4] + p[..., 4:5] + p[..., 5:6] + p[..., 6:7] + p[..., 7:])


def _plain_norm(state, case):
    x, kind = state["x"].float(), TORCH[case["type"]]
    if state["residual"] is not None:
        x = (x + state["residual"].float()).to(kind).float()
    # the mean in 64 bits: the factor decides values that lie next to a border of the 4-bit grid
    factor = (x.double().square().mean(-1, keepdim=True) + EPS).rsqrt().float()
    y = (x * factor * state["weight"].float()).to(kind)
    return y, x.to(kind)


# ------------------------------------------------------------------------------------------------------- one pass

def _own_weight(fos, weight, case, cls, n, k):
    form = fos.DataType(case["format"])
    rule = fos.ScaleRule.mse if case["format"] == "if4" else fos.ScaleRule.static_6
    padded = (weight[0].shape[-2], 2 * weight[0].shape[-1])
    if cls is fos.QuantizedTensor:
        return cls(*weight, form, (n, k), rule, fos.RoundStyle.nearest, padded,
                   scale_factors_are_in_blackwell_layout=case["format"] != "if4")
    return cls(*weight, form, rule, (n, k), padded)


def run(state):
    case = state["case"]
    do, kind, x = case["do"], TORCH[case["type"]], state["x"]
    if do == "norm":
        if own:
            import fouroversix_b200 as fos

            config = None if case["format"] == "none" else fos.QuantizationConfig(dtype=case["format"], scale_rule=case["rule"])
            out = fos.rms_norm(x, state["weight"], eps=EPS, residual=state["residual"], config=config)
            y, residual = out if state["residual"] is not None else (out, None)
            got = {"y": y} if config is None else {"y": fos.dequantize(y, kind), "amax": y.amax}
            return got if residual is None else {**got, "residual": residual}
        y, residual = _plain_norm(state, case)
        got = {"y": y}
        if case["format"] != "none":
            values, amax = _plain_quantized(y.float(), case)
            got = {"y": values.to(kind), "amax": amax}
        return got if state["residual"] is None else {**got, "residual": residual}

    weight, n, k = state["weight"], case["n"], case["k"]
    if do == "product":
        if own:
            import fouroversix_b200 as fos

            w = _own_weight(fos, weight, case, fos.QuantizedTensor, n, k)
            y = fos.weight_only_matmul(x, w, bias=state["bias"])
            return {"y": y.detach(), "dx": torch.autograd.grad(y, x, state["dy"])[0]} if case["grad"] else y
        w = _plain_weight(weight, case)[:n, :k]
        with torch.no_grad():
            y = x.float() @ w.T * _factor(weight, case)
            y = (y if state["bias"] is None else y + state["bias"].float()).to(kind)
            return {"y": y, "dx": (state["dy"].float() @ w * _factor(weight, case)).to(kind)} if case["grad"] else y

    rows, experts = case["tokens"] * case["top"], case["experts"]
    if own:
        import fouroversix_b200 as fos
        from fouroversix_b200.matmul import GroupLayout, StackedQuantizedTensor, grouped_weight_only_matmul

        layout = GroupLayout(state["group_start"], state["group_rows"], rows, experts)
        return grouped_weight_only_matmul(x, _own_weight(fos, weight, case, StackedQuantizedTensor, n, k), layout, row_index=state["row_index"])
    # every expert's rows in a buffer as long as the longest
    start = state["group_start"][:-1]
    expert = torch.repeat_interleave(torch.arange(experts, device=x.device), state["group_rows"], output_size=rows)
    place = torch.arange(rows, device=x.device) - start[expert]
    padded = torch.zeros(experts, state["most"], k, device=x.device)
    padded[expert, place] = x.float()[state["row_index"]]
    y = torch.bmm(padded, _plain_weight(weight, case)[:, :n, :k].mT) * _factor(weight, case).reshape(-1, 1, 1)
    return y[expert, place].to(kind)


def work(case):
    if case["do"] == "norm":
        values = case["rows"] * case["cols"]
        # in: x and the residual; out: the sum, and y in 16 bits, packed on the way where there is a format
        packed = 0 if case["format"] == "none" else 2 * BYTES[case["format"]]
        return {"bytes": values * (2 + 2 + 4 * case["residual"] + packed), "flops": 4 * values}
    k, n, t = case["k"], case["n"], case["tokens"]
    if case["do"] == "product":
        times = 1 + case["grad"]
        return {"bytes": times * (BYTES[case["format"]] * n * k + 2 * t * k + 2 * t * n), "flops": times * 2 * t * n * k}
    pairs = t * case["top"]
    hit = case["experts"] * (1 - (1 - case["top"] / case["experts"]) ** t)       # experts that some token goes to
    return {"bytes": hit * BYTES[case["format"]] * n * k + 2 * t * k + 2 * pairs * n, "flops": 2 * pairs * n * k}


# ---------------------------------------------------------------------------------------------------------- 64 bits

def _exact_weight(values, scales, amax, case):
    """One packed matrix as numbers in 64 bits, from the definition of its format."""
    form, block = case["format"], BLOCK[case["format"]]
    n_p, k_p = values.shape[0], values.shape[1] * 2
    code = torch.empty(n_p, k_p, dtype=torch.long, device="cuda")
    code[:, 0::2], code[:, 1::2] = (values % 16).long(), (values // 16).long()
    e, m = code // 2 % 4, code % 2
    grid = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1)) * (1 - 2.0 * (code // 8))
    r = torch.arange(n_p, device="cuda")[:, None]
    c = torch.arange(k_p // block, device="cuda")[None, :]
    nb = k_p // block
    at = r * nb + c if form == "if4" else (r // 128 * (nb // 4) + c // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4
    byte = scales.view(torch.uint8)[at].long()
    if form == "mxfp4":
        step = torch.where(byte == 0, 0.0, torch.exp2(byte.double() - 127))
    else:
        e8, m8 = byte // 8 % 16, byte % 8
        step = torch.where(e8 == 0, m8 * 2.0 ** -9, (1 + m8 / 8.0) * torch.exp2(e8.double() - 7)) * (amax.double() / 2688)
    if form == "if4":
        whole = (byte >= 128).repeat_interleave(block, 1)
        grid = torch.where(whole, (code - 16 * (code // 8)).double() * 6 / 7, grid)
    return grid * step.repeat_interleave(block, 1)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["do"] == "norm":
            x = s["x"].double()
            if s["residual"] is not None:
                x = (x + s["residual"].double()).to(TORCH[case["type"]]).double()      # the stream is kept in 16 bits
            y = x / (x.pow(2).sum(-1, keepdim=True) / case["cols"] + EPS).sqrt() * s["weight"].double()
            got = {"y": y}
            if case["format"] != "none":
                got = _exact_packed(y.to(TORCH[case["type"]]).double(), case)
            return got if s["residual"] is None else {**got, "residual": x}
        n, k = case["n"], case["k"]
        if case["do"] == "product":
            w = _exact_weight(*s["weight"], case)[:n, :k]
            y = s["x"].double() @ w.T
            y = y if s["bias"] is None else y + s["bias"].double()
            return {"y": y, "dx": s["dy"].double() @ w} if case["grad"] else y
        values, scales, amax = s["weight"]
        y = torch.zeros(case["tokens"] * case["top"], n, dtype=torch.float64, device="cuda")
        for e, (start, rows) in enumerate(zip(s["group_start"].tolist(), s["group_rows"].tolist())):
            w = _exact_weight(values[e], scales[e], amax[e], case)[:n, :k]
            y[start:start + rows] = s["x"].double()[s["row_index"][start:start + rows].long()] @ w.T
        return y


def _exact_packed(y, case):
    """y [rows, cols] through the 4-bit grid in 64 bits."""
    form, block = case["format"], BLOCK[case["format"]]
    rows, cols = y.shape
    b = torch.zeros(rows, _up(cols, block), dtype=torch.float64, device="cuda")
    b[:, :cols] = y
    b = b.reshape(rows, -1, block)
    top = b.abs().amax(-1, keepdim=True)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device="cuda")
    grid = torch.tensor(E2M1, dtype=torch.float64, device="cuda")

    def rounded(v):
        a = v.abs()
        low, high = torch.bucketize(a, borders), torch.bucketize(a, borders, right=True)     # differ on a border:
        return torch.sign(v) * grid[torch.where(low % 2 == 0, low, high)]                    # the even code then

    if form == "mxfp4":
        step = torch.exp2(torch.ceil(torch.log2((top / 6).clamp_min(2.0 ** -126))))
        return {"y": (rounded(b / step) * step).reshape(rows, -1)[:, :cols], "amax": torch.ones(1, dtype=torch.float64, device="cuda")}
    amax = y.abs().amax().reshape(1)
    ceiling = 256 if case["rule"] == "mse" else 448
    unit = amax / (6 * ceiling)
    best = None
    for stretch in (1.0, 1.5) if case["rule"] == "mse" else (1.0,):
        step = (top / 6 / unit.clamp_min(1e-300) * stretch).float().to(torch.float8_e4m3fn).double() * unit
        v = rounded(torch.where(step > 0, b / step.clamp_min(1e-300), 0.0)) * step
        error = (v - b).pow(2).sum(-1, keepdim=True)
        best = (v, error) if best is None else (torch.where(error < best[1], v, best[0]), None)
    return {"y": best[0].reshape(rows, -1)[:, :cols], "amax": amax}
