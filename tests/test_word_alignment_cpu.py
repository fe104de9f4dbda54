"""32-bit words that do not lie on 4 bytes are refused by the C entries on the host: a kernel that reads or writes one would fault."""

from __future__ import annotations

import pytest

from tests.test_weight_only_cpu import A, MISALIGNED, gradient, grouped, norm, product


@pytest.mark.parametrize("entry,word", [(product, "amax"), (product, "status"), (gradient, "amax"), (gradient, "status"), (grouped, "amax"),
                                        (grouped, "status"), (grouped, "row_index"), (grouped, "start"), (grouped, "group_rows")])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_products(entry, word, off):
    assert entry(**{word: A + off}) == MISALIGNED


@pytest.mark.parametrize("rows", [4, 1000])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_norms(rows, off):
    assert norm("fos_rms_norm", rows=rows, amax=A + off) == MISALIGNED
    assert norm("fos_rms_norm_quantize", rows=rows, amax=A + off) == MISALIGNED
    assert norm("fos_rms_norm_quantize", rows=rows, amax=A + off, format=2, rule=0) == MISALIGNED
