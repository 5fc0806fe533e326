"""Sizes past what the plain product's arguments hold are refused."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_rows_than_an_int_holds():
    """2^32 + 5 rows are not taken for 5."""
    from vllm_moe_offload_amd import native

    w = native.quantize_mx4(torch.randn((16, 32), device="cuda"))
    for rows in ((1 << 31) + 5, (1 << 32) + 5):
        with pytest.raises(ValueError, match="more than an int"):
            native.mx4_linear(native.Mx4Rows.allocate(rows, 32, "cuda"), w)
        torch.cuda.empty_cache()
