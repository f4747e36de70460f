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


def test_outputs_that_overlap_an_operand():
    """Found from addresses and pitches; columns of one buffer side by side are apart."""
    from tjkernels.kernels import _need_apart

    def apart(out, *inputs):
        try:
            _need_apart("out", out, *inputs)
            return True
        except ValueError:
            return False

    buf = torch.zeros(40, 96)
    other = torch.zeros(40, 96)
    assert apart(buf, other) and apart(buf, None) and apart(buf, other, None, other[3:])
    assert not apart(buf, buf) and not apart(buf, other, buf)
    assert apart(buf[:10], buf[10:]) and apart(buf[10:], buf[:10])
    assert not apart(buf[:10], buf[9:]) and not apart(buf[9:], buf[:10])
    assert apart(buf[:, :32], buf[:, 32:]) and apart(buf[:, 64:], buf[:, :64])
    assert apart(buf[5:, :32], buf[:20, 32:])
    assert not apart(buf[:, :32], buf[:, 31:]) and not apart(buf[:, 32:], buf[:, :33])
    wrapped = buf.as_strided((39, 40), (96, 1), 64)  # its rows end in the next ones
    assert not apart(buf[1:, :8], wrapped) and apart(buf[1:, 8:64], wrapped)
    # Another pitch over the same memory.
    assert not apart(buf.view(-1)[:960].view(20, 48), buf[:, 64:])
    assert not apart(buf, buf.view(torch.float16))
    assert apart(buf[:0], buf) and apart(buf, buf[:0])
    assert not apart(buf[:1], buf[:1, 95:]) and apart(buf[:1, :32], buf[:1, 32:])
