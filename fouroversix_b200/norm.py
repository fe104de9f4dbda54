"""Root-mean-square norm with the residual's addition, in 16 bits or packed for the next product."""

from __future__ import annotations

import torch

from fouroversix_b200 import _native
from fouroversix_b200.quantize import B200QuantizeBackend, QuantizationConfig, QuantizedTensor
from fouroversix_b200.utils import DataType, QuantizeBackend


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    t = t.reshape(-1, cols)
    return t if (t.stride(1) == 1 or cols == 1) and (t.stride(0) >= cols or t.shape[0] == 1) else t.contiguous()


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor | None = None,
             config: QuantizationConfig | None = None):
    """`y = h / sqrt(mean(h^2) + eps) * weight` over the last dimension of `h = x + residual` (`h = x` without one), for bf16 or
    fp16 `x`; `weight` has x's type or float32. h is rounded to x's type, the mean is exact, y is formed in float32 and rounded
    once to x's type. With `config`, y is not returned but `quantize(y, config)` of its rows: the operand of `quantized_matmul`.
    Returns y, or (y, h) with a residual: h is the residual stream of the layers behind. Inference only: no gradient."""
    if x.device.type != "cuda":
        raise ValueError("rms_norm: input must be a CUDA tensor (there is no CPU path)")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("rms_norm: input must be bfloat16 or float16")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("rms_norm: the last dimension is the one that is normalised and cannot be empty")
    cols, dev = x.shape[-1], x.device
    if weight.shape != (cols,) or weight.dtype not in (x.dtype, torch.float32) or weight.device != dev:
        raise ValueError("rms_norm: weight must be one number per column, of the input's type or float32, on its device")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != dev):
        raise ValueError("rms_norm: residual must have the input's shape, type and device")
    if not eps >= 1e-30:
        raise ValueError("rms_norm: eps must be positive (1e-30 at least)")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("rms_norm: no gradient is implemented (detach the inputs, or run under torch.no_grad)")
    x2, w = _rows(x, cols), weight.contiguous()
    rows = x2.shape[0]
    if config is not None:
        if config.pseudo_quantize or config.backend not in (None, QuantizeBackend.cuda):
            raise ValueError("rms_norm: the output is packed by the B200 kernels or not at all")
        reason = B200QuantizeBackend.unsupported_reason(x2, config)
        if reason is None and rows == 0:
            reason = "no rows to pack"
        if reason is not None:
            raise ValueError(f"rms_norm: {reason}")
    r2 = None if residual is None else _rows(residual, cols)
    total = None if residual is None else torch.empty(rows, cols, dtype=x.dtype, device=dev)
    y = torch.empty(rows, cols, dtype=x.dtype, device=dev)
    if rows:
        scaled = config is not None and config.dtype != DataType.mxfp4 and not config.rht
        amax = torch.empty(1, dtype=torch.float32, device=dev) if scaled else None
        with _native.on_device(dev):
            _native.check(_native.lib().fos_rms_norm(
                x2.data_ptr(), _native.elem_code(x.dtype), rows, cols, max(x2.stride(0), cols), 0 if r2 is None else r2.data_ptr(),
                0 if r2 is None else max(r2.stride(0), cols), w.data_ptr(), _native.elem_code(w.dtype), float(eps),
                0 if total is None else total.data_ptr(), cols, y.data_ptr(), cols, 0 if amax is None else amax.data_ptr(),
                _native.stream_ptr(dev)), "fos_rms_norm")
        if config is not None:
            y = B200QuantizeBackend._quantize(y, config, amax)
    if config is None:
        y = y.reshape(x.shape)
    return y if total is None else (y, total.reshape(x.shape))
