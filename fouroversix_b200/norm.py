"""Root-mean-square norm with the residual's addition, in 16 bits or packed for the next product."""

from __future__ import annotations

import torch

from fouroversix_b200 import _native
from fouroversix_b200.quantize import B200QuantizeBackend, QuantizationConfig, QuantizedTensor
from fouroversix_b200.quantize.backend import _FORMATS, _is_tiled
from fouroversix_b200.utils import DataType, QuantizeBackend, RoundStyle

_BF16, _FP16, _FP32 = torch.bfloat16, torch.float16, torch.float32


def _form(dtype: DataType) -> tuple:
    """What packing in a format needs to know: its native number, block size, scale type and scale layout."""
    return (_FORMATS[dtype], dtype.block_size, dtype.scale_type.torch_dtype, _native.FOS_SF_TILED if _is_tiled(dtype) else _native.FOS_SF_ROWMAJOR)


# (asked for by identity below: a decoding step is bound by the host)
_NVFP4, _IF4, _MXFP4 = DataType.nvfp4, DataType.if4, DataType.mxfp4
_NVFP4_FORM, _IF4_FORM, _MXFP4_FORM = _form(_NVFP4), _form(_IF4), _form(_MXFP4)


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
    Returns y, or (y, h) with a residual: h is the residual stream of the layers behind. Inference only: no gradient,
    no forward mode."""
    _native.refuse_transforms("rms_norm", x, weight, residual)
    dev, dtype, shape = x.device, x.dtype, x.shape
    if not x.is_cuda:
        raise ValueError("rms_norm: input must be a CUDA tensor (there is no CPU path)")
    if dtype is not _BF16 and dtype is not _FP16:
        raise ValueError("rms_norm: input must be bfloat16 or float16")
    if not shape or shape[-1] == 0:
        raise ValueError("rms_norm: the last dimension is the one that is normalised and cannot be empty")
    cols = shape[-1]
    if weight.shape != (cols,) or (weight.dtype is not dtype and weight.dtype is not _FP32) or weight.device != dev:
        raise ValueError("rms_norm: weight must be one number per column, of the input's type or float32, on its device")
    if residual is not None and (residual.shape != shape or residual.dtype is not dtype or residual.device != dev):
        raise ValueError("rms_norm: residual must have the input's shape, type and device")
    if not eps >= 1e-30:
        raise ValueError("rms_norm: eps must be positive (1e-30 at least)")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
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
        total = torch.empty((rows, cols), dtype=dtype, device=dev)
        r_ptr, r_ld, total_ptr = r2.data_ptr(), max(r2.stride(0), cols), total.data_ptr()
    lib = _native.lib()
    code = _native.FOS_BF16 if dtype is _BF16 else _native.FOS_FP16
    head = (x2.data_ptr(), code, rows, cols, max(x2.stride(0), cols), r_ptr, r_ld, w.data_ptr(),
            _native.FOS_FP32 if w.dtype is _FP32 else code, eps, total_ptr, cols)
    y = None if config is None else _packed(lib, head, config, dev)
    if y is None:
        y = torch.empty((rows, cols), dtype=dtype, device=dev)
        scaled = config is not None and config.dtype is not _MXFP4 and not config.rht
        amax = torch.empty(1, dtype=_FP32, device=dev) if scaled else None
        if rows:
            with _native.on_device(dev):
                _native.check(lib.fos_rms_norm(*head, y.data_ptr(), cols, 0 if amax is None else amax.data_ptr(),
                                               _native.stream_ptr(dev)), "fos_rms_norm")
        if config is not None:
            y = B200QuantizeBackend._quantize(y, config, amax)
        elif len(shape) != 2:
            y = y.reshape(shape)
    if total is None:
        return y
    return y, total if len(shape) == 2 else total.reshape(shape)


def _packed(lib, head: tuple, config: QuantizationConfig, dev: torch.device) -> QuantizedTensor | None:
    """The norm with its rows packed by one host call (fos_rms_norm_quantize), or None for what that does not take."""
    if config.block_scale_2d or config.transpose or config.rht or config.round_style is not RoundStyle.nearest:
        return None
    rows, cols, form = head[2], head[3], config.dtype
    number, block, scale_type, layout = _NVFP4_FORM if form is _NVFP4 else _MXFP4_FORM if form is _MXFP4 else _IF4_FORM
    rows_p, cols_p = -(-rows // 128) * 128, -(-cols // (4 * block)) * (4 * block)
    values = torch.empty((rows_p, cols_p // 2), dtype=torch.uint8, device=dev)
    scales = torch.empty(rows_p * cols_p // block, dtype=scale_type, device=dev)
    amax = torch.empty(1, dtype=_FP32, device=dev)
    need = 0 if form is _MXFP4 else lib.fos_rms_norm_quantize_workspace_bytes(rows, cols)
    workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _native.on_device(dev):
        status = lib.fos_rms_norm_quantize(*head, number, config.scale_rule.cuda_id, layout, values.data_ptr(), scales.data_ptr(),
                                           amax.data_ptr(), workspace.data_ptr() if need else 0, need, _native.stream_ptr(dev))
    if status == -2:
        return None
    _native.check(status, "fos_rms_norm_quantize")
    return QuantizedTensor(values, scales, amax, form, (rows, cols), config.scale_rule, config.round_style, (rows_p, cols_p),
                           scale_factors_are_in_blackwell_layout=layout == _native.FOS_SF_TILED)
