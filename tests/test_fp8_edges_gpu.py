"""Block-scaled e4m3 operators where a call can go wrong without a sign: outputs
that a call has to write, values at the ends of the number range, sizes at the
ends of the index range.  Against 64-bit formulas, as in test_fp8_gpu.py."""

import pytest
import torch

from test_fp8_gpu import DEV, NORM_REL, K, check_out, gen, rand, rms_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


# ----------------------------------------------- a norm without a delta

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d,offset", [(37, 256, 0), (5, 1000, 0), (9, 1004, 0), (3, 8192, 0),
                                           (37, 256, 4)])
def test_residual_is_written_without_a_delta(rows, d, offset, dtype):
    """x = res: the buffer for the sum gets the residual, whatever its type,
    width and alignment; a masked row too."""
    from tjkernels import _lib
    from tjkernels.kernels import _code, _launch
    g = gen(rows, d, offset, 21)
    res = rand(g, rows * d + 16).to(dtype)[offset:offset + rows * d].view(rows, d)
    mask = torch.ones(rows, dtype=torch.uint8, device=DEV)
    mask[rows // 2] = 0
    w = rand(g, d)
    _, ref = rms_ref(res, None, w, 1e-5)
    ref = ref * mask.double()[:, None]
    res_out = torch.full((rows, d), 7.0, dtype=dtype, device=DEV)
    out = torch.empty(rows, d, device=DEV)
    _launch("tjb_add_rmsnorm", res.device, res.data_ptr(), None, res_out.data_ptr(),
            out.data_ptr(), None, w.data_ptr(), rows, d, 1e-5, _code(dtype), _lib.TJB_F32,
            _lib.TJB_F32, mask.data_ptr(), None)
    assert torch.equal(res_out, res)
    check_out(out, ref, NORM_REL * ref.abs())
    res_out.fill_(7.0)
    new, out = K().fused_add_rmsnorm(res, None, w, 1e-5, out_dtype=torch.float32, row_mask=mask,
                                     residual_out=res_out)
    assert new is res_out and torch.equal(res_out, res)
    check_out(out, ref, NORM_REL * ref.abs())
    keep = res.clone()
    new, _ = K().fused_add_rmsnorm(res, None, w, 1e-5, residual_out=res)
    assert new is res and torch.equal(res, keep)
    res_out.fill_(7.0)
    new, _ = K().fused_add_rmsnorm(res, None, w, 1e-5, residual_out=res_out,
                                   write_residual=False)
    assert new is res and (res_out == 7).all()


def test_residual_out_without_a_delta_is_checked():
    x, w = torch.zeros(4, 32, device=DEV), torch.ones(32, device=DEV)
    for bad in (x.half(), x[:2], torch.zeros(32, 4, device=DEV).t()):
        with pytest.raises(ValueError):
            K().fused_add_rmsnorm(x, None, w, 1e-5, residual_out=bad)
