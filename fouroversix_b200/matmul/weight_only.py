"""Products of 16-bit activations with packed 4-bit weights: only the weight is quantized.

`quantized_matmul` quantizes both operands, which is what the FP4 tensor cores want. With few tokens the product is bound by
the weight's bytes alone, and 4-bit activations buy nothing there but their error: these functions leave the activations in
bf16 or fp16 and unpack the weight on its way into the product (`fos_weight_only_matmul`). The sums are in fp32 and the result is
rounded once.

The numbers are multiplied in fp16. Those of NVFP4 and IF4 weights are exactly the ones the packed weight stands for, and so are MXFP4's where a
block's scale is between 2^-23 and 2^13. Outside they are what `dequantize` makes of them by default: smaller scales become zero (2^-24 stays, but not
exact with every code), larger ones make infinities. (`quantized_matmul` multiplies such weights as they are, and so does a product with
`dequantize(weight, intermediate_dtype=torch.float32)`.) A row of bf16 activations is multiplied by one power of two, which is taken back from the sums:
that is exact for values down to 2^-29 of the row's largest, smaller ones are off by at most 2^-39 of it.
"""

from __future__ import annotations

import torch

from fouroversix_b200 import _native
from fouroversix_b200.quantize import QuantizedTensor
from fouroversix_b200.utils import DataType, RoundStyle

from .grouped import MAX_GROUPS, GroupLayout, StackedQuantizedTensor

_OUT = {DataType.bfloat16: torch.bfloat16, DataType.float16: torch.float16, DataType.float32: torch.float32}
_NVFP4, _IF4, _MXFP4 = DataType.nvfp4, DataType.if4, DataType.mxfp4
_BF16, _FP16 = torch.bfloat16, torch.float16


def _format(dtype: DataType) -> tuple[int, int]:
    """The native number of a format and its block size (asked for by identity: a decoding step is bound by the host)."""
    if dtype is _NVFP4:
        return _native.FOS_NVFP4, 16
    if dtype is _MXFP4:
        return _native.FOS_MXFP4, 32
    if dtype is _IF4:
        return _native.FOS_IF4, 16
    raise ValueError(f"weight-only matmul: dtype {dtype.value} is not implemented (nvfp4, if4 and mxfp4 are)")


def _torch_out(out_dtype: DataType | torch.dtype | None, input: torch.Tensor) -> torch.dtype:
    if out_dtype is None:
        return input.dtype
    if isinstance(out_dtype, torch.dtype):
        if out_dtype in _OUT.values():
            return out_dtype
    elif DataType(out_dtype) in _OUT:
        return _OUT[DataType(out_dtype)]
    raise ValueError(f"weight-only matmul: output type {out_dtype} is not supported")


def _check_input(x: torch.Tensor, k: int, device: torch.device) -> None:
    if x.device != device or device.type != "cuda":
        if x.device.type != "cuda":
            raise ValueError("weight-only matmul: input must be a CUDA tensor (there is no CPU path)")
        raise ValueError("weight-only matmul: input and weight must live on the same CUDA device")
    if x.dtype is not _BF16 and x.dtype is not _FP16:
        raise ValueError("weight-only matmul: input must be bfloat16 or float16")
    if x.dim() == 0 or x.shape[-1] != k:
        raise ValueError(f"weight-only matmul: the input's last dimension must be the weight's {k} columns, got {tuple(x.shape)}")


def _check_packed(weight: QuantizedTensor | StackedQuantizedTensor, groups: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """The packed buffers as the kernels read them, or ValueError for what they would read past."""
    n, k = weight.original_shape
    n_p, k_p = weight.padded_shape
    block = _format(weight.dtype)[1]
    values, scales, amax = weight.values, weight.scale_factors, weight.amax
    if n <= 0 or k <= 0 or n_p < n or k_p < k or n_p % 128 or k_p % (4 * block):
        raise ValueError(f"weight-only matmul: a weight of shape {(n, k)} cannot be padded to {(n_p, k_p)}")
    size = groups * n_p * k_p
    if values.dtype.itemsize != 1 or values.numel() != size // 2:
        raise ValueError("weight-only matmul: the weight's values do not have the size of its padded shape")
    if scales.dtype.itemsize != 1 or scales.numel() != size // block:
        raise ValueError("weight-only matmul: the weight's scale factors do not have the size of its padded shape")
    dev = values.device
    if scales.device != dev:
        raise ValueError("weight-only matmul: the weight's values and scale factors must live on the same device")
    if weight.dtype is _MXFP4:
        return values.contiguous(), scales.contiguous(), None
    if amax is None or amax.numel() != groups or amax.dtype is not torch.float32 or amax.device != dev:
        raise ValueError("weight-only matmul: amax must be a float32 tensor beside the weight's values, one number per weight")
    return values.contiguous(), scales.contiguous(), amax.contiguous()


def _layout(w: QuantizedTensor | StackedQuantizedTensor) -> int:
    return _native.FOS_SF_TILED if w.scale_factors_are_in_blackwell_layout else _native.FOS_SF_ROWMAJOR


def _rows(x: torch.Tensor) -> torch.Tensor:
    """`x` [..., k] as rows that the kernels can step through: unit column stride, rows that do not overlap."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if (x.stride(1) == 1 or x.shape[1] == 1) and (x.stride(0) >= x.shape[1] or x.shape[0] == 1) else x.contiguous()


def _ld(x: torch.Tensor) -> int:
    return max(x.stride(0), x.shape[1])


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of rows (unit column stride, rows that do not overlap) have bytes in common. Rows of one stride side by side, as columns
    of a wider tensor are, have none; where the strides differ, so much as a meeting of the memory they span counts."""
    def place(t: torch.Tensor) -> tuple[int, int, int]:
        width, step = t.shape[1] * t.element_size(), _ld(t) * t.element_size()
        return t.data_ptr(), width, step
    (a0, a_width, a_step), (b0, b_width, b_step) = place(a), place(b)
    if a0 >= b0 + (b.shape[0] - 1) * b_step + b_width or b0 >= a0 + (a.shape[0] - 1) * a_step + a_width:
        return False
    between = (b0 - a0) % a_step
    return a_step != b_step or between < a_width or between + b_width > a_step


def _workspace(lib, device: torch.device, *sizes: int) -> tuple[torch.Tensor | None, int]:
    """Scratch of a call (the sizes are those of fos_weight_only_workspace_bytes) and its bytes; few rows need none."""
    need = lib.fos_weight_only_workspace_bytes(*sizes)
    return (torch.empty(need, dtype=torch.uint8, device=device) if need else None), need


def _product(x: torch.Tensor, w: QuantizedTensor, bias: torch.Tensor | None, torch_out: torch.dtype) -> torch.Tensor:
    n, k = w.original_shape
    n_p, k_p = w.padded_shape
    x2 = _rows(x)
    dev, rows = x.device, x2.shape[0]
    out = torch.empty(rows, n, dtype=torch_out, device=dev)
    if rows == 0:
        return out.reshape(*x.shape[:-1], n)
    values, scales, amax = _check_packed(w, 1)
    lib = _native.lib()
    workspace, need = _workspace(lib, dev, rows, n_p, k_p, 0, 0)
    with _native.on_device(dev):
        _native.check(lib.fos_weight_only_matmul(
            x2.data_ptr(), _native.elem_code(x2.dtype), rows, k, _ld(x2), values.data_ptr(), scales.data_ptr(),
            0 if amax is None else amax.data_ptr(), _format(w.dtype)[0], w.scale_rule.cuda_id,
            int(w.round_style is RoundStyle.stochastic_unbiased), _layout(w), n, n_p, k_p, 0 if bias is None else bias.data_ptr(),
            out.data_ptr(), _native.elem_code(torch_out), n, workspace.data_ptr() if need else 0, need, 0, _native.stream_ptr(dev)),
            "fos_weight_only_matmul")
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], n)


def _input_gradient(dy: torch.Tensor, w: QuantizedTensor, dtype: torch.dtype) -> torch.Tensor:
    """`dy @ weight` (fos_weight_only_matmul_dgrad) in `dtype`."""
    n, k = w.original_shape
    n_p, k_p = w.padded_shape
    dy2 = _rows(dy)
    dev, rows = dy.device, dy2.shape[0]
    dx = torch.empty(rows, k, dtype=dtype, device=dev)
    if rows:
        values, scales, amax = _check_packed(w, 1)
        lib = _native.lib()
        workspace, need = _workspace(lib, dev, rows, n_p, k_p, 0, 1)
        with _native.on_device(dev):
            _native.check(lib.fos_weight_only_matmul_dgrad(
                dy2.data_ptr(), _native.elem_code(dy2.dtype), rows, n, _ld(dy2), values.data_ptr(), scales.data_ptr(),
                0 if amax is None else amax.data_ptr(), _format(w.dtype)[0], w.scale_rule.cuda_id,
                int(w.round_style is RoundStyle.stochastic_unbiased), _layout(w), k, n_p, k_p, dx.data_ptr(), _native.elem_code(dtype), k,
                workspace.data_ptr(), need, 0, _native.stream_ptr(dev)), "fos_weight_only_matmul_dgrad")
    return dx.reshape(*dy.shape[:-1], k)


class _WeightOnlyMatmul(torch.autograd.Function):
    """The product with a frozen packed weight, differentiable in its input and bias."""

    @staticmethod
    def forward(ctx, input, weight, bias, torch_out):
        ctx.weight, ctx.input_dtype = weight, input.dtype
        return _product(input, weight, bias, torch_out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dx = _input_gradient(dy, ctx.weight, ctx.input_dtype) if ctx.needs_input_grad[0] else None
        db = dy.reshape(-1, dy.shape[-1]).sum(0) if ctx.needs_input_grad[2] else None
        return dx, None, db, None


def weight_only_matmul(input: torch.Tensor, weight: QuantizedTensor, *, bias: torch.Tensor | None = None,
                       out_dtype: DataType | torch.dtype | None = None) -> torch.Tensor:
    """`input @ weight.T (+ bias)` with `input` [..., k] in bf16 or fp16 and `weight` packed (nvfp4, if4 or mxfp4, any scale
    rule and rounding; the module says what range of numbers is exact). Sums in fp32, one rounding to `out_dtype` (default: the input's type), whose type `bias` [n] has.
    Differentiable in `input` and `bias` (16-bit outputs), once and in reverse mode; the weight is frozen. Forward and backward can be captured in a CUDA graph
    as long as no eager graph of the same leaves is alive (autograd would wait for that one's stream, which a capture does not allow)."""
    if not isinstance(weight, QuantizedTensor):
        raise ValueError("weight-only matmul: the weight must be a QuantizedTensor (quantize it first)")
    _format(weight.dtype)
    _native.refuse_transforms("weight-only matmul", input, bias)
    _check_input(input, weight.original_shape[1], weight.values.device)
    torch_out = _torch_out(out_dtype, input)
    if bias is not None:
        if bias.shape != (weight.original_shape[0],) or bias.dtype != torch_out or bias.device != input.device:
            raise ValueError("weight-only matmul: bias must be one number of the output's type per output feature, on the input's device")
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (input.requires_grad or (bias is not None and bias.requires_grad)):
        if torch_out == torch.float32:
            raise ValueError("weight-only matmul: the gradient takes an output in bfloat16 or float16")
        return _WeightOnlyMatmul.apply(input, weight, bias, torch_out)
    return _product(input, weight, bias, torch_out)


def grouped_weight_only_matmul(x: torch.Tensor, weight: StackedQuantizedTensor, layout: GroupLayout, *,
                               row_index: torch.Tensor | None = None, out_dtype: DataType | torch.dtype | None = None,
                               out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r] = x[row_index[r]] @ weight[g].T for the rows r of every group g of `layout`, in one launch; without `row_index`
    (int32 [layout.capacity]) row r of the groups is row r of `x`. Rows whose index is outside `x` are taken as zeros. Groups
    need no padding (`GroupLayout.compact`) but may have it, and lie in any order. `out` may not share memory with `x`. Returns
    [layout.capacity, n]; rows that belong to no group are zero."""
    if not isinstance(weight, StackedQuantizedTensor):
        raise ValueError("grouped weight-only matmul: the weights must be a StackedQuantizedTensor")
    n, k = weight.original_shape
    n_p, k_p = weight.padded_shape
    _format(weight.dtype)
    _native.refuse_transforms("grouped weight-only matmul", x, out)
    _check_input(x, k, weight.values.device)
    groups, cap, dev = layout.num_groups, layout.capacity, x.device
    if x.dim() != 2:
        raise ValueError("grouped weight-only matmul: x must be [rows, k]")
    if not 0 < groups <= MAX_GROUPS or weight.values.shape[0] != groups:
        raise ValueError("grouped weight-only matmul: operands disagree on the number of groups")
    if row_index is None:
        if x.shape[0] != cap:
            raise ValueError("grouped weight-only matmul: x must have the layout's rows")
    elif row_index.dtype != torch.int32 or row_index.shape != (cap,) or row_index.device != dev:
        raise ValueError("grouped weight-only matmul: row_index must be one int32 per row of the layout, on x's device")
    for t, count in ((layout.group_start, groups + 1), (layout.group_rows, groups)):
        if t.dtype != torch.int32 or t.numel() < count or not t.is_contiguous() or t.device != dev:
            raise ValueError("grouped weight-only matmul: the layout's tables must be contiguous int32 on x's device")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("grouped weight-only matmul: no gradient is implemented (detach the input, or run under torch.no_grad)")
    torch_out = _torch_out(out_dtype, x)
    given = out is not None
    if not given:
        out = torch.empty(cap, n, dtype=torch_out, device=dev)
    elif out.shape != (cap, n) or out.dtype != torch_out or out.stride(1) != 1 or out.stride(0) < n or out.device != dev:
        raise ValueError("grouped weight-only matmul: `out` has the wrong shape, dtype, device or layout")
    if cap == 0:
        return out
    if x.shape[0] == 0:
        return out.zero_()
    values, scales, amax = _check_packed(weight, groups)
    x = _rows(x)
    if given and _share_memory(out, x):
        raise ValueError("grouped weight-only matmul: `out` must not lie in the memory of x, whose rows are read while others are written")
    index = None if row_index is None else row_index.contiguous()
    lib = _native.lib()
    workspace, need = _workspace(lib, dev, cap, n_p, k_p, groups, 0)
    with _native.on_device(dev):
        _native.check(lib.fos_weight_only_matmul_grouped(
            x.data_ptr(), _native.elem_code(x.dtype), x.shape[0], k, _ld(x), 0 if index is None else index.data_ptr(),
            values.data_ptr(), scales.data_ptr(), 0 if amax is None else amax.data_ptr(), _format(weight.dtype)[0],
            weight.scale_rule.cuda_id, _layout(weight),
            layout.group_start.data_ptr(), layout.group_rows.data_ptr(), groups, cap, n, n_p, k_p, out.data_ptr(),
            _native.elem_code(torch_out), out.stride(0), workspace.data_ptr() if need else 0, need, 0, _native.stream_ptr(dev)),
            "fos_weight_only_matmul_grouped")
    return out
