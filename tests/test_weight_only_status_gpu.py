"""The status word of the 16-bit-activation products through the C entries: 0 after every call, whatever the caller left in it."""

from __future__ import annotations

import pytest
import torch

import fouroversix_b200 as fos
from fouroversix_b200 import _native

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("entry", ["product", "gradient", "grouped"])
@pytest.mark.parametrize("rows", [1, 12, 60, 400])
def test_status_is_written(entry, rows):
    n, k, groups = 256, 512, 4
    lib, stream = _native.lib(), _native.stream_ptr(torch.device(DEV, 0))
    q = fos.quantize((torch.randn(groups * n, k, device=DEV) * 0.02).bfloat16())
    x = torch.randn(rows, k if entry != "gradient" else n, device=DEV).bfloat16()
    out = torch.empty(rows, n if entry != "gradient" else k, device=DEV, dtype=torch.bfloat16)
    status = torch.full((1,), 77, dtype=torch.int32, device=DEV)
    need = lib.fos_weight_only_workspace_bytes(rows, n, k, groups if entry == "grouped" else 0, int(entry == "gradient"))
    workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
    weight = (q.values.data_ptr(), q.scale_factors.data_ptr(), q.amax.data_ptr(), _native.FOS_NVFP4, q.scale_rule.cuda_id)
    tail = (workspace.data_ptr(), need, status.data_ptr(), stream)
    if entry == "product":
        code = lib.fos_weight_only_matmul(x.data_ptr(), 0, rows, k, k, *weight, 0, 1, n, n, k, 0, out.data_ptr(), 0, n, *tail)
    elif entry == "gradient":
        code = lib.fos_weight_only_matmul_dgrad(x.data_ptr(), 0, rows, n, n, *weight, 0, 1, k, n, k, out.data_ptr(), 0, k, *tail)
    else:
        start = torch.tensor([0, rows, rows, rows, rows], dtype=torch.int32, device=DEV)
        counts = torch.tensor([rows, 0, 0, 0], dtype=torch.int32, device=DEV)
        amax = q.amax.expand(groups).contiguous()
        code = lib.fos_weight_only_matmul_grouped(x.data_ptr(), 0, rows, k, k, 0, *weight[:2], amax.data_ptr(), *weight[3:], 1, start.data_ptr(),
                                                  counts.data_ptr(), groups, rows, n, n, k, out.data_ptr(), 0, n, *tail)
    assert code == 0 and status.item() == 0
