"""Host-side checks of the block-scaled e4m3 entry points that need no GPU:
what they refuse before any device work, and that the facade has no CPU path."""

import pytest
import torch

FAKE = 1 << 20  # a 16-byte aligned address that is never read


def lib():
    from tjkernels import _lib
    return _lib.lib()


def quantize(x=FAKE, ldx=256, dtype=0, q=FAKE, s=FAKE, rows=4, k=256, fn="tjb_quantize_blocks"):
    more = (None, None) if fn == "tjb_quantize_blocks" else (None,)
    return getattr(lib(), fn)(x, ldx, dtype, q, s, rows, k, *more)


@pytest.mark.parametrize("fn", ["tjb_quantize_blocks", "tjb_quantize_weight_blocks"])
def test_quantize_refusals(fn):
    assert quantize(fn=fn, x=None) == 1
    assert quantize(fn=fn, q=None) == 1
    assert quantize(fn=fn, s=None) == 1
    assert quantize(fn=fn, rows=-1) == 1
    assert quantize(fn=fn, k=0) == 1
    assert quantize(fn=fn, dtype=3) == 4
    assert quantize(fn=fn, k=24) == 2
    assert quantize(fn=fn, ldx=128) == 2
    assert quantize(fn=fn, rows=2 ** 31) == 2
    assert quantize(fn=fn, k=2 ** 31 - 16, ldx=2 ** 31 - 16) == 2
    assert quantize(fn=fn, ldx=258) == 3
    assert quantize(fn=fn, x=FAKE + 8) == 3
    assert quantize(fn=fn, x=FAKE + 4, dtype=1) == 3
    assert quantize(fn=fn, q=FAKE + 4) == 3


def norm(res=FAKE, delta=FAKE, res_out=FAKE, out=FAKE, scales=FAKE, w=FAKE, rows=4, d=256,
         res_dtype=0, delta_dtype=1, out_dtype=3):
    return lib().tjb_add_rmsnorm(res, delta, res_out, out, scales, w, rows, d, 1e-5, res_dtype,
                                 delta_dtype, out_dtype, None, None, None)


def test_add_rmsnorm_refusals():
    assert norm(res=None) == 1
    assert norm(out=None) == 1
    assert norm(w=None) == 1
    assert norm(scales=None) == 1            # 8-bit output without room for its scales
    assert norm(rows=-1) == 1
    assert norm(d=24) == 2                   # 8-bit rows are whole 16-byte pieces
    assert norm(d=6, out_dtype=1) == 2
    assert norm(d=16400) == 2
    assert norm(rows=2 ** 31) == 2
    assert norm(res_dtype=3) == 4
    assert norm(delta_dtype=3) == 4
    assert norm(out_dtype=4) == 4
    assert norm(res=FAKE + 8) == 3
    assert norm(delta=FAKE + 4) == 3
    assert norm(res_out=FAKE + 8) == 3
    assert norm(out=FAKE + 8) == 3
    assert norm(w=FAKE + 4) == 3


def gemm(a=FAKE, sa=FAKE, w=FAKE, sw=FAKE, bias=None, c=FAKE, sc=FAKE, m=4, n=256, k=256,
         lda=None, ldw=None, ldc=None, out=3, act=0, row=2, blk=1):
    return lib().tjb_gemm_fp8(a, sa, row, blk, w, sw, bias, c, sc, m, n, k,
                              k if lda is None else lda, k if ldw is None else ldw,
                              n if ldc is None else ldc, out, act, None, None)


def test_gemm_fp8_refusals():
    for name in ("a", "sa", "w", "sw", "c", "sc"):
        assert gemm(**{name: None}) == 1, name
    assert gemm(m=-1) == 1
    assert gemm(n=0) == 1
    assert gemm(act=2) == 1
    assert gemm(row=-1) == 1
    assert gemm(out=4) == 4
    assert gemm(k=264) == 2
    assert gemm(n=264) == 2                  # 8-bit output: whole 16-byte pieces
    assert gemm(n=260, out=1) == 2
    assert gemm(lda=128) == 2
    assert gemm(ldw=128) == 2
    assert gemm(ldc=128) == 2
    assert gemm(k=2 ** 31 - 16) == 2         # rounded up, these would pass 2^31
    assert gemm(n=2 ** 31 - 16) == 2
    assert gemm(m=2 ** 31 - 1) == 2
    assert gemm(lda=264) == 3
    assert gemm(ldw=264) == 3
    assert gemm(ldc=260, out=1) == 3
    assert gemm(a=FAKE + 8) == 3
    assert gemm(w=FAKE + 8) == 3
    assert gemm(c=FAKE + 8) == 3
    assert gemm(bias=FAKE + 8) == 3
    assert gemm(sa=FAKE + 2) == 3


def test_valid_calls_reach_the_device_check():
    """Without a B200 a valid call answers "no device" and launches nothing."""
    if torch.cuda.is_available():
        pytest.skip("the made-up addresses are for machines without a GPU")
    assert quantize() == 8
    assert quantize(fn="tjb_quantize_weight_blocks") == 8
    assert norm() == 8
    assert gemm() == 8
    assert gemm(out=0, n=264, sc=None, ldc=272) == 8


def test_facade_has_no_cpu_path():
    import tjkernels.kernels as K
    x = torch.zeros(4, 256)
    with pytest.raises(RuntimeError):
        K.quantize_blocks(x)
    with pytest.raises(RuntimeError):
        K.quantize_weight_blocks(x)
    with pytest.raises(RuntimeError):
        K.rmsnorm(x, torch.ones(256), 1e-5)
    q = x.to(torch.float8_e4m3fn)
    with pytest.raises(RuntimeError):
        K.gemm_fp8(q, torch.ones(4, 2), q, torch.ones(1, 2))
