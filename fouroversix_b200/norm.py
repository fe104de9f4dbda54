"""Root-mean-square norm with the residual's addition, in 16 bits or packed for the next product."""

from __future__ import annotations

import torch

from fouroversix_b200 import _native
from fouroversix_b200.quantize import B200QuantizeBackend, QuantizationConfig, QuantizedTensor
from fouroversix_b200.quantize.backend import _FORMATS, _is_tiled
from fouroversix_b200.quantize.quantized_tensor import padded_shape_for
from fouroversix_b200.utils import DataType, QuantizeBackend, RoundStyle


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """`t` [..., cols] as rows that the kernels can step through: unit column stride, rows that do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    return t if (t.stride(1) == 1 or cols == 1) and (t.stride(0) >= cols or t.shape[0] == 1) else t.contiguous()


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: torch.Tensor | None = None,
             config: QuantizationConfig | None = None):
    """`y = h / sqrt(mean(h^2) + eps) * weight` over the last dimension of `h = x + residual` (`h = x` without one), for bf16 or
    fp16 `x`; `weight` has x's type or float32. h is rounded to x's type, the mean is exact, y is formed in float32 and rounded
    once to x's type. With `config`, y is not returned but `quantize(y, config)` of its rows: the operand of `quantized_matmul`.
    Returns y, or (y, h) with a residual: h is the residual stream of the layers behind. Inference only: no gradient."""
    dev, dtype = x.device, x.dtype
    if dev.type != "cuda":
        raise ValueError("rms_norm: input must be a CUDA tensor (there is no CPU path)")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError("rms_norm: input must be bfloat16 or float16")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("rms_norm: the last dimension is the one that is normalised and cannot be empty")
    cols = x.shape[-1]
    if weight.shape != (cols,) or (weight.dtype is not dtype and weight.dtype is not torch.float32) or weight.device != dev:
        raise ValueError("rms_norm: weight must be one number per column, of the input's type or float32, on its device")
    if residual is not None and (residual.shape != x.shape or residual.dtype is not dtype or residual.device != dev):
        raise ValueError("rms_norm: residual must have the input's shape, type and device")
    if not eps >= 1e-30:
        raise ValueError("rms_norm: eps must be positive (1e-30 at least)")
    if (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)) and torch.is_grad_enabled():
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
    if residual is None:
        total, r_ptr, r_ld, total_ptr = None, 0, 0, 0
    else:
        r2 = _rows(residual, cols)
        total = torch.empty(rows, cols, dtype=dtype, device=dev)
        r_ptr, r_ld, total_ptr = r2.data_ptr(), max(r2.stride(0), cols), total.data_ptr()
    lib = _native.lib()
    head = (x2.data_ptr(), _native.elem_code(dtype), rows, cols, max(x2.stride(0), cols), r_ptr, r_ld, w.data_ptr(),
            _native.elem_code(w.dtype), float(eps), total_ptr, cols)
    y = None if config is None else _packed(lib, head, config, dev)
    if y is None:
        y = torch.empty(rows, cols, dtype=dtype, device=dev)
        scaled = config is not None and config.dtype != DataType.mxfp4 and not config.rht
        amax = torch.empty(1, dtype=torch.float32, device=dev) if scaled else None
        if rows:
            with _native.on_device(dev):
                _native.check(lib.fos_rms_norm(*head, y.data_ptr(), cols, 0 if amax is None else amax.data_ptr(),
                                               _native.stream_ptr(dev)), "fos_rms_norm")
        y = y.reshape(x.shape) if config is None else B200QuantizeBackend._quantize(y, config, amax)
    if total is None:
        return y
    return y, total if x.dim() == 2 else total.reshape(x.shape)


def _packed(lib, head: tuple, config: QuantizationConfig, dev: torch.device) -> QuantizedTensor | None:
    """The norm with its rows packed by one host call (fos_rms_norm_quantize), or None for what that does not take."""
    if config.block_scale_2d or config.transpose or config.rht or config.round_style is not RoundStyle.nearest:
        return None
    rows, cols = head[2], head[3]
    form = config.dtype
    rows_p, cols_p = padded_shape_for((rows, cols), form)
    values = torch.empty(rows_p, cols_p // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(rows_p * cols_p // form.block_size, dtype=form.scale_type.torch_dtype, device=dev)
    amax = torch.empty(1, dtype=torch.float32, device=dev)
    need, workspace = 0, None
    if form is not DataType.mxfp4:
        need = lib.fos_rms_norm_quantize_workspace_bytes(rows, cols)
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    tiled = _is_tiled(form)
    with _native.on_device(dev):
        status = lib.fos_rms_norm_quantize(*head, _FORMATS[form], config.scale_rule.cuda_id, _native.FOS_SF_TILED if tiled else _native.FOS_SF_ROWMAJOR,
                                           values.data_ptr(), scales.data_ptr(), amax.data_ptr(), workspace.data_ptr() if need else 0, need,
                                           _native.stream_ptr(dev))
    if status == -2:
        return None
    _native.check(status, "fos_rms_norm_quantize")
    return QuantizedTensor(values, scales, amax, form, (rows, cols), config.scale_rule, config.round_style, (rows_p, cols_p),
                           scale_factors_are_in_blackwell_layout=tiled)
