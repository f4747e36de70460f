"""Sizes and pitches that the block-scaled e4m3 entry points take and refuse,
as far as a machine without a GPU shows them."""

import pytest
import torch

from test_fp8_cpu import gemm


@pytest.mark.parametrize("out,pitch", [(0, 4), (1, 8), (2, 8), (3, 16)])
def test_output_rows_start_on_16_byte_borders(out, pitch):
    """Any such pitch is taken, whatever the type; no other is."""
    if torch.cuda.is_available():
        pytest.skip("the made-up addresses are for machines without a GPU")
    for n in range(1, 17):
        assert gemm(n=256, ldc=256 + n, out=out) == (3 if n % pitch else 8), n
