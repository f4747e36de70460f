"""Block-scaled e4m3 operators where a call can go wrong without a sign: outputs
that a call has to write, values at the ends of the number range, sizes at the
ends of the index range.  Against 64-bit formulas, as in test_fp8_gpu.py."""

import math

import pytest
import torch

from test_fp8_gpu import (DEV, F8, NORM_REL, U32, K, check_out, check_quantised, gen, operands,
                          per_block, product_ref, rand, rms_ref)

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


# ------------------------------------------------------------------------ GELU

# One size of each form of the product: 16, 32 and 64 tokens, wide tiles whose
# k-blocks are split, whole, in pairs, and with rows left over.
GELU_ROWS = [1, 20, 40, 100, 700, 5000, 11000]


def gelu_of(x, m, dtype):
    """The product's GELU of exactly x: zero operands, so that the sums are the bias."""
    n = x.numel()
    a, sa = K().quantize_blocks(torch.zeros(m, 1024, device=DEV))
    w, sw = K().quantize_weight_blocks(torch.ones(n, 1024, device=DEV))
    return K().gemm_fp8(a, sa, w, sw, x, act=K().ACT_GELU, out_dtype=dtype)


def between(points, a):
    """The exponential of the straight line between the points' logarithms, at a."""
    at, val = (torch.tensor(v, dtype=torch.float64, device=a.device) for v in zip(*points))
    i = torch.bucketize(a, at).clamp(1, len(points) - 1)
    f = ((a - at[i - 1]) / (at[i] - at[i - 1])).clamp(0, 1)
    return torch.exp(val[i - 1].log() * (1 - f) + val[i].log() * f)


def gelu_ref(x, fit):
    """GELU(x) in 64 bits and the bound of its error.

    GELU(x) = max(x, 0) - t with t = a Phi(-a), a = |x|, and Phi(-a) = 2^q with
    a polynomial q.  `fit` bounds what the polynomial, with its fp32
    coefficients, is off, relative to Phi.  Horner's scheme rounds the partial
    sum p_k, which is still to be multiplied by a^k, by at most U32 |p_k|: in q
    that is U32 HORNER(a), in Phi ln 2 times as much.  2^q is off by 2^-22 at
    most, the last product and the sum by a rounding each.  Beyond 12.9, where
    t is below 4e-37, it may be dropped."""
    x = x.double()
    a = x.abs()
    t = a * 0.5 * torch.erfc(a / math.sqrt(2.0))
    rel = between(fit, a) + U32 * (4 + 1 + math.log(2.0) * between(HORNER, a))
    ref = x.clamp_min(0) - t
    return ref, t * rel + U32 * ref.abs() + torch.where(a > 12.9, 4e-37, 0.0)


# sum_k |p_k| a^k: 1, 4.87, 12.6, 25, 58.7, 147, 704, 3890, 19100 and 49200 at
# these points for degree 13, less for degree 7; a straight line between their
# logarithms falls below it by 14 % at most.
HORNER = [(0, 1.2), (1, 5.7), (2, 14.5), (3, 29), (4.5, 68), (6, 170), (8, 815), (10, 4500),
          (12, 22100), (13.3, 57000)]
# Largest difference between the neighbouring points.
FIT32 = [(0, 1.8e-8), (0.5, 1.8e-8), (1, 2.9e-8), (1.5, 2.9e-8), (2, 1.9e-7), (2.5, 3.2e-7),
         (3, 1.6e-6), (3.5, 1.7e-6), (4, 2e-5), (5, 3.2e-5), (6, 6.3e-5), (8, 1.3e-4),
         (10, 2.9e-4), (13.3, 2.9e-4)]
FIT16 = [(0, 8.7e-7), (0.25, 1.9e-6), (0.5, 1.9e-6), (1, 2.5e-6), (1.5, 3e-6), (2, 1.4e-5),
         (2.5, 1.5e-5), (3, 1.4e-4), (3.5, 3.9e-4), (4, 8.2e-4), (5, 8.2e-4), (6, 0.011),
         (8, 0.012), (10, 0.1), (13.3, 0.1)]


def gelu_inputs(g, n):
    """Values over the whole range: tiny, ordinary, in the tail and beyond it."""
    x = torch.exp(torch.empty(n, device=DEV).uniform_(math.log(1e-6), math.log(20.0), generator=g))
    x[n // 2:] = torch.empty(n - n // 2, device=DEV).uniform_(0, 14, generator=g)
    x = x * torch.where(torch.rand(n, device=DEV, generator=g) < 0.7, -1.0, 1.0)
    x[:6] = torch.tensor([0.0, -100.0, 100.0, -1e30, 1e30, -13.0], device=DEV)
    return x


@pytest.mark.parametrize("m", GELU_ROWS)
def test_gelu_fp32(m):
    """To a few roundings of the result near zero, and right in the tail."""
    x = gelu_inputs(gen(m, 31), 4096)
    ref, tol = gelu_ref(x, FIT32)
    near = (x.abs() <= 1) & (x != 0)
    assert (tol[near] <= 14 * U32 * ref[near].abs()).all()  # what the bound above comes to
    out = gelu_of(x, m, torch.float32).double()
    bad = (out - ref).abs() > tol
    assert not bad.any(), x.expand_as(out)[bad][:8]


@pytest.mark.parametrize("m", GELU_ROWS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gelu_16_bit(m, dtype):
    x = gelu_inputs(gen(m, 32), 4096).clamp(-60000, 60000)
    ref, tol = gelu_ref(x, FIT16)
    check_out(gelu_of(x, m, dtype), ref.expand(m, -1), tol)


@pytest.mark.parametrize("m", GELU_ROWS)
def test_gelu_blocks_of_the_tail(m):
    """Blocks of small results only: their 8-bit values keep the results' ratios."""
    g = gen(m, 33)
    lo = torch.tensor([-1e-4, -2.0, -5.0, -7.0, -9.0, -12.0, -40.0], device=DEV)
    x = (lo[:, None] * (1 + 0.1 * torch.rand(7, 128, device=DEV, generator=g))).flatten()
    ref, tol = gelu_ref(x, FIT16)
    q, s = gelu_of(x, m, F8)
    check_quantised(q, s, ref.expand(m, -1).contiguous(), tol)
    assert (q[:, -128:].float() == 0).all()


@pytest.mark.parametrize("m", GELU_ROWS)
def test_gelu_of_large_sums(m):
    """Up to the largest numbers: themselves, or zero."""
    x = torch.exp(torch.linspace(math.log(14.0), 88.7, 256, device=DEV))
    x[-1] = torch.finfo(torch.float32).max
    x = torch.cat([x, -x])
    ref = x.clamp_min(0).double().expand(m, -1)
    for dtype in (torch.float32, torch.bfloat16):
        out = gelu_of(x, m, dtype)
        assert torch.equal(out, ref.to(torch.float32).to(dtype))
    q, s = gelu_of(x, m, F8)
    check_quantised(q, s, ref.contiguous(), 0.0)


@pytest.mark.parametrize("m", GELU_ROWS)
def test_gelu_of_infinities(m):
    """As 0.5 x (1 + erf(x / sqrt 2)): NaN at minus infinity, infinity at infinity."""
    x = rand(gen(m, 34), 512)
    x[5], x[200], x[300] = -math.inf, math.inf, math.nan
    for dtype in DTYPES:
        out = gelu_of(x, m, dtype)
        assert out[:, 5].isnan().all() and (out[:, 200] == math.inf).all()
        assert out[:, 300].isnan().all()
        rest = torch.ones(512, dtype=torch.bool, device=DEV)
        rest[[5, 200, 300]] = False
        assert out[:, rest].isfinite().all()
    q, s = gelu_of(x, m, F8)
    held = q.double() * per_block(s, m, 512)
    assert held[:, :384].isnan().all() and held[:, 384:].isfinite().all()


@pytest.mark.parametrize("m", [5, 90, 600, 9000])
def test_infinite_scale_under_gelu(m):
    """A row whose scale is infinite ends with no finite value."""
    g = gen(m, 35)
    a, sa, w, sw = operands(g, m, 768, 528)
    sa[m - 1, 2] = math.inf
    for dtype in DTYPES:
        out = K().gemm_fp8(a, sa, w, sw, act=K().ACT_GELU, out_dtype=dtype)
        assert not out[m - 1].isfinite().any() and out[:m - 1].isfinite().all()


# ------------------------------------------------------------- infinite blocks

def e4m3_of(y, s):
    """e4m3(y / s), with what inf / inf and finite / inf are."""
    return (y.double() / s).float().to(F8)


def test_bytes_of_infinite_blocks():
    """q = e4m3(y / s) also where s is infinite or NaN: zeros beside the NaN of
    an infinite element, NaN throughout a block with a NaN."""
    x = rand(gen(36), 8, 512) * 3
    x[0, 3], x[1, 130], x[2, 200] = math.inf, -math.inf, math.nan
    x[3, 300], x[3, 301] = math.inf, math.nan
    x[4] = math.inf
    want_s = x.abs().view(8, 4, 128).amax(dim=2)
    for dtype in DTYPES:
        y = x.to(dtype)
        q, s = K().quantize_blocks(y)
        odd = per_block(want_s, 8, 512).isfinite().logical_not()
        want = e4m3_of(y, per_block(want_s, 8, 512))
        got, want = q.float()[odd], want.float()[odd]
        assert torch.equal(got.isnan(), want.isnan()) and (got[~got.isnan()] == 0).all()
        assert got.isnan().any() and (~got.isnan()).any()
        qw, sw = K().quantize_weight_blocks(y[:1])
        assert sw[0, 0].isinf() and qw[0, 3].isnan() and (qw[0, :3].float() == 0).all()
    # As an output of the norm (an infinite weight) and of the product (a bias).
    w = torch.ones(512, device=DEV)
    w[7] = math.inf
    q, s = K().rmsnorm(x[5:7], w, 1e-5, out_dtype=F8)
    assert s[:, 0].isinf().all() and q[:, 7].isnan().all() and (q[:, 8:128].float() == 0).all()
    for m in (3, 100, 9000):
        a, sa, wq, ws = operands(gen(m, 37), m, 512, 256)
        bias = torch.zeros(512, device=DEV)
        bias[7] = math.inf
        q, s = K().gemm_fp8(a, sa, wq, ws, bias, out_dtype=F8)
        assert s[:, 0].isinf().all() and q[:, 7].isnan().all() and (q[:, 8:128].float() == 0).all()


# ------------------------------------------------------------------ the output

@pytest.mark.parametrize("m", [5, 40, 100, 700, 11000])
def test_fp32_rows_at_any_16_byte_pitch(m):
    g = gen(m, 38)
    n, k = 520, 656
    a, sa, w, sw = operands(g, m, n, k)
    out = torch.full((m, n + 12), 7.0, device=DEV)
    got = K().gemm_fp8(a, sa, w, sw, out_dtype=torch.float32, out=out[:, :n])
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(out[:, :n], K().gemm_fp8(a, sa, w, sw, out_dtype=torch.float32))
    assert (out[:, n:] == 7).all()
    from tjkernels._lib import KernelError
    if m > 1:
        with pytest.raises(KernelError):
            K().gemm_fp8(a, sa, w, sw, out_dtype=torch.float16,
                         out=torch.zeros(m, n + 4, device=DEV, dtype=torch.float16)[:, :n])


def test_as_many_rows_as_an_int_counts():
    """The most tokens of a call: counts of them, rounded up to tiles of 256."""
    m, n, k = 2 ** 31 - 129, 8, 16
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 90e9:
        pytest.skip("needs 70 GB of device memory")
    g = gen(39)
    tail, sa, w, sw = operands(g, 500, n, k)
    a = torch.zeros(m, k, dtype=torch.uint8, device=DEV)
    a[-500:] = tail.view(torch.uint8)
    out = torch.full((m, n), 7.0, dtype=torch.float16, device=DEV)
    K().gemm_fp8(a.view(F8), sa[:1].expand(m, 1), w, sw, out_dtype=torch.float16, out=out)
    ref, tol = product_ref(tail, sa[:1].expand(500, 1), w, sw)
    check_out(out[-500:], ref, tol)
    assert (out[:4096] == 0).all() and (out[:-500:65537] == 0).all()
    del a, out
    torch.cuda.empty_cache()


def test_outputs_over_an_operand_are_refused():
    """While a call writes its output other blocks of it still read the operands."""
    g = gen(40)
    a, sa, w, sw = operands(g, 300, 256, 256)
    for out in (a, a[:200], w):
        with pytest.raises(ValueError):
            K().gemm_fp8(a[:out.shape[0]], sa[:out.shape[0]], w, sw, out_dtype=F8, out=out)
    both = torch.zeros(300, 512, device=DEV).to(F8)
    both[:, :256] = a
    want, scales = K().gemm_fp8(a, sa, w, sw, out_dtype=F8)
    got, s = K().gemm_fp8(both[:, :256], sa, w, sw, out_dtype=F8, out=both[:, 256:])
    assert torch.equal(got.float(), want.float()) and torch.equal(s, scales)
    assert torch.equal(both[:, :256].float(), a.float())
    nw = torch.ones(256, device=DEV)
    buf = rand(g, 101, 256).half()
    with pytest.raises(ValueError):
        K().fused_add_rmsnorm(buf[1:], rand(g, 100, 256), nw, 1e-5, residual_out=buf[:-1])
    with pytest.raises(ValueError):
        K().fused_add_rmsnorm(rand(g, 100, 256).half(), buf[1:], nw, 1e-5, residual_out=buf[:-1])
    with pytest.raises(ValueError):  # the same address, another type
        K().fused_add_rmsnorm(buf[:100], buf.view(torch.bfloat16)[:100], nw, 1e-5,
                              residual_out=buf[:100])
    res, delta = rand(g, 100, 256).half(), rand(g, 100, 256).half()
    want, out = K().fused_add_rmsnorm(res, delta, nw, 1e-5)
    got, out2 = K().fused_add_rmsnorm(res, delta, nw, 1e-5, residual_out=delta)
    assert got is delta and torch.equal(delta, want) and torch.equal(out2, out)
