"""The block-scaled e4m3 operators (RMS norm, quantisation, product) against
64-bit formulas.  Calls go through the C ABI via the tjkernels.kernels facade.

Tolerances count roundings: half a step of the output type, plus the fp32
error of what is computed before it (derived beside each bound)."""

import math
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U32 = 2.0 ** -24  # half a step of fp32, relative
F8 = torch.float8_e4m3fn


@pytest.fixture(autouse=True, scope="module")
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a CUDA device")
    yield


def K():
    import tjkernels.kernels as kernels
    return kernels


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(hash(key) % (1 << 31))


def rand(g, *shape, scale=1.0):
    return torch.randn(*shape, device=DEV, generator=g) * scale


def acts(g, rows, k):
    """Activations with a few large channels."""
    return rand(g, rows, k) * torch.exp(0.7 * rand(g, k))


def per_block(scales, rows, k, block_rows=1):
    s = scales.double()
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, dim=0)[:rows]
    return s.repeat_interleave(128, dim=1)[:, :k]


def block_amax(y, block_rows=1):
    rows, k = y.shape
    rb, kb = -(-rows // block_rows), -(-k // 128)
    t = torch.zeros(rb * block_rows, kb * 128, dtype=torch.float64, device=y.device)
    t[:rows, :k] = y.abs()
    return t.view(rb, block_rows, kb, 128).amax(dim=(1, 3))


def check_quantised(q, scales, y, tol, block_rows=1):
    """(q, scales) stands for y (fp64) that was computed to within tol (an
    absolute bound, a tensor of y's shape or a number)."""
    rows, k = y.shape
    assert q.dtype == F8 and q.shape == y.shape
    amax = block_amax(y, block_rows)
    assert scales.dtype == torch.float32 and scales.shape == amax.shape
    tol = torch.as_tensor(tol, dtype=torch.float64, device=y.device).expand_as(y)
    want = (amax / 448).clamp_min(2.0 ** -126)
    # The amax is off by at most its element's tol, the division by half a step.
    off = block_amax(tol.contiguous(), block_rows) / 448 + U32 * want
    assert ((scales.double() - want).abs() <= off).all()
    s = per_block(scales, rows, k, block_rows)
    r = y / s
    slack = tol / s + 2 * U32 * r.abs()
    _, e = torch.frexp(r.abs() + slack)
    half = torch.exp2((e - 1).clamp(-6, 8).double() - 4)
    bad = (q.double() - r).abs() > half + slack
    assert not bad.any(), (int(bad.sum()), (q.double() - r).abs().max().item())


# -------------------------------------------------------------- quantisation

QUANT_SHAPES = [(1, 16), (1, 4096), (3, 128), (7, 144), (129, 1040), (1000, 512), (33, 2064),
                (4, 16384)]


@pytest.mark.parametrize("rows,k", QUANT_SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_quantize_blocks(rows, k, dtype):
    x = acts(gen(rows, k), rows, k).to(dtype)
    q, s = K().quantize_blocks(x)
    check_quantised(q, s, x.double(), 0.0)


@pytest.mark.parametrize("n,k", [(8, 16), (128, 128), (136, 144), (1000, 1040), (2, 4096),
                                 (2048, 512)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_quantize_weight_blocks(n, k, dtype):
    w = rand(gen(n, k), n, k, scale=k ** -0.5).to(dtype)
    q, s = K().quantize_weight_blocks(w)
    check_quantised(q, s, w.double(), 0.0, block_rows=128)


def test_quantize_extremes():
    """Zero blocks, subnormals, the largest finite values, NaN and infinity."""
    x = torch.zeros(6, 256, device=DEV)
    x[1, :128] = 1e-42           # subnormal: the scale stops at 2^-126
    x[2] = 3.0e38
    x[3, 5] = float("nan")
    x[3, 6] = 2.0
    x[4, 200] = float("inf")
    x[5] = -448.0
    q, s = K().quantize_blocks(x)
    held = q.double() * per_block(s, 6, 256)
    assert (s[0] == 2.0 ** -126).all() and (held[0] == 0).all()
    assert s[1, 0] == 2.0 ** -126 and (held[1] == 0).all()
    assert ((held[2] - 3.0e38).abs() <= 3.0e38 * 2.0 ** -4).all()
    assert held[3, :128].isnan().all() and (held[3, 128:] == 0).all()
    assert held[4, 128:].isnan().all() and (held[4, :128] == 0).all()
    assert (held[5] == -448).all() and (s[5] == 1).all()
    qw, sw = K().quantize_weight_blocks(x)
    assert sw.isnan()[0, 0] and sw.isinf()[0, 1]
    assert (qw.double() * per_block(sw, 6, 256, 128)).isnan().all()


def test_quantize_strided_rows():
    g = gen(5)
    wide = acts(g, 40, 1024).half()
    for x in (wide[:, 128:400], wide[::3, :528], wide.t()[:64, :32], wide[:1, 3:19],
              wide[:, 1:17], wide[0].expand(5, 1024)):
        q, s = K().quantize_blocks(x)
        check_quantised(q, s, x.double(), 0.0)
        qw, sw = K().quantize_weight_blocks(x)
        check_quantised(qw, sw, x.double(), 0.0, block_rows=128)


def test_quantize_empty():
    q, s = K().quantize_blocks(torch.empty(0, 256, device=DEV))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    q, s = K().quantize_weight_blocks(torch.empty(0, 256, device=DEV))
    assert q.shape == (0, 256) and s.shape == (0, 2)


# ------------------------------------------------------------------ RMS norm

def rms_ref(res, delta, w, eps):
    x = res.double() + (0 if delta is None else delta.double())
    return x, x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + eps) * w.double()


# fp32 error of the norm, relative to the result: the sum of squares goes
# through at most 53 additions (32 a thread, 5 in the warp and 16 across warps;
# or 16, 5 and 32) after one rounding of each x (twice in its square) and of each square, so its
# relative error is below 56 u and the root's half of that; x, 1/sqrt, the two
# products and the mean's division and sum with eps add at most 6 u.
NORM_REL = 40 * U32


def check_out(out, ref, tol):
    if out.dtype == torch.float32:
        half, tiny = U32, 2.0 ** -150
    else:
        half = torch.finfo(out.dtype).eps / 2
        tiny = torch.finfo(out.dtype).smallest_normal * half  # subnormal half step
    bad = (out.double() - ref).abs() > tol + half * (ref.abs() + tol) + tiny
    assert not bad.any(), (int(bad.sum()), (out.double() - ref).abs().max().item())


NORM_SHAPES = [(1, 16), (1, 1024), (37, 80), (130, 768), (5, 1040), (64, 2064), (257, 4096),
               (9, 8192), (3, 8208), (2, 16384), (3000, 512)]


@pytest.mark.parametrize("rows,d", NORM_SHAPES)
@pytest.mark.parametrize("res_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("delta_dtype", [None, torch.float32, torch.float16, torch.bfloat16])
def test_add_rmsnorm(rows, d, res_dtype, delta_dtype):
    g = gen(rows, d)
    res = acts(g, rows, d).to(res_dtype)
    delta = None if delta_dtype is None else acts(g, rows, d).to(delta_dtype)
    w = 1 + 0.2 * rand(g, d)
    _, ref = rms_ref(res, delta, w, 1e-5)
    # The sum x is rounded to fp32 once; where res and delta cancel that is
    # still relative to x, so NORM_REL covers it.
    tol = NORM_REL * ref.abs()
    for out_dtype in (torch.float32, torch.float16, torch.bfloat16):
        new, out = K().fused_add_rmsnorm(res, delta, w, 1e-5, out_dtype=out_dtype)
        check_out(out, ref, tol)
        if delta is None:
            assert new is res
        else:
            assert torch.equal(new, (res.float() + delta.float()).to(res_dtype))
    same, (q, s) = K().fused_add_rmsnorm(res, delta, w, 1e-5, out_dtype=F8, write_residual=False)
    assert same is res
    check_quantised(q, s, ref, tol)
    if delta is None:
        q2, s2 = K().rmsnorm(res, w, 1e-5, out_dtype=F8)
        assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


@pytest.mark.parametrize("d", [4, 20, 132, 1004])
def test_add_rmsnorm_odd_width(d):
    g = gen(d)
    res, delta, w = rand(g, 11, d), rand(g, 11, d).bfloat16(), rand(g, d)
    _, ref = rms_ref(res, delta, w, 1e-6)
    _, out = K().fused_add_rmsnorm(res, delta, w, 1e-6, out_dtype=torch.float16)
    check_out(out, ref, NORM_REL * ref.abs())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,offset", [(4, 0), (1000, 0), (1004, 0), (1024, 4), (256, 12)])
def test_add_rmsnorm_16_bit_odd_rows(d, offset, dtype):
    """Widths that are no multiple of 16 columns, and rows that start between
    16-byte borders."""
    g = gen(d, offset)

    def shifted():
        return rand(g, 23 * d + 16).to(dtype)[offset:offset + 23 * d].view(23, d)

    for res, delta in ((shifted(), shifted()), (shifted(), rand(g, 23, d).to(dtype)),
                       (rand(g, 23, d).to(dtype), shifted()), (shifted(), None)):
        w = rand(g, d)
        _, ref = rms_ref(res, delta, w, 1e-5)
        new, out = K().fused_add_rmsnorm(res, delta, w, 1e-5, out_dtype=dtype)
        check_out(out, ref, NORM_REL * ref.abs())
        if delta is not None:
            assert torch.equal(new, (res.float() + delta.float()).to(dtype))


@pytest.mark.parametrize("rows,d", [(300, 1024), (7000, 256), (130, 4096)])
@pytest.mark.parametrize("delta_dtype", [torch.float16, torch.bfloat16])
def test_add_rmsnorm_masked_rows_in_place(rows, d, delta_dtype):
    g = gen(rows, d, 1)
    res, delta, w = rand(g, rows, d).bfloat16(), rand(g, rows, d).to(delta_dtype), rand(g, d)
    mask = torch.rand(rows, device=DEV, generator=g) > 0.4
    _, ref = rms_ref(res, delta, w, 1e-5)
    want = (res.float() + delta.float()).bfloat16()
    got, (q, s) = K().fused_add_rmsnorm(res, delta, w, 1e-5, out_dtype=F8, row_mask=mask,
                                        residual_out=res)
    assert got.data_ptr() == res.data_ptr() and torch.equal(res, want)
    assert (q[~mask].float() == 0).all() and (s[~mask] == 2.0 ** -126).all()
    ref = ref * mask[:, None]
    check_quantised(q, s, ref, NORM_REL * ref.abs())


def test_add_rmsnorm_zero_and_nan_rows():
    g = gen(8)
    res, w = rand(g, 5, 512), rand(g, 512)
    res[1] = 0
    res[2, 100] = float("nan")
    res[3, 100] = float("inf")
    _, ref = rms_ref(res, None, w, 1e-5)
    out = K().rmsnorm(res, w, 1e-5)
    assert (out[1] == 0).all() and out[2].isnan().all() and out[3, 100].isnan()
    keep = torch.tensor([0, 1, 4], device=DEV)
    check_out(out[keep], ref[keep], NORM_REL * ref[keep].abs())
    q, s = K().rmsnorm(res, w, 1e-5, out_dtype=F8)
    check_quantised(q[keep], s[keep], ref[keep], NORM_REL * ref[keep].abs())
    assert (q[2].float() * per_block(s, 5, 512)[2].float()).isnan().all()


# ------------------------------------------------------------------- product

def operands(g, m, n, k):
    a, sa = K().quantize_blocks(acts(g, m, k))
    w, sw = K().quantize_weight_blocks(rand(g, n, k, scale=k ** -0.5))
    return a, sa, w, sw


def product_ref(a, sa, w, sw):
    """The product in 64 bits and the bound of its fp32 error.

    One 128-column block is summed by the tensor core: 128 exact products,
    each addition rounded or cut to fp32 (2 u); the block's scale takes 2 u,
    and each block's addition one: (256 + 2 + blocks) u of the sum of
    magnitudes, and up to 8 more for joining split sums."""
    m, k = a.shape
    n = w.shape[0]
    da = a.double() * per_block(sa, m, k)
    dw = w.double() * per_block(sw, n, k, 128)
    mag = da.abs() @ dw.abs().t()
    return da @ dw.t(), (256 + 2 + sa.shape[1] + 8) * U32 * mag


def finish(ref, tol, bias, act):
    if bias is not None:
        ref = ref + bias.double()
        tol = tol + U32 * (ref.abs() + tol)
    if act:
        # GELU's slope is at most 1.13; its own error 5e-7 and 2 u relative.
        tol = 1.13 * tol + 5e-7 + 4 * U32 * ref.abs()
        ref = 0.5 * ref * torch.erfc(-ref / math.sqrt(2.0))
    return ref, tol


GEMM_SHAPES = [(1, 64, 16), (1, 4096, 4096), (2, 136, 128), (15, 384, 1040), (16, 16, 4096),
               (17, 1024, 48), (32, 128, 512), (33, 264, 2064), (64, 640, 256), (65, 1160, 144),
               (127, 256, 1024), (128, 128, 128), (129, 120, 640), (300, 1000, 1040),
               (513, 2048, 272), (1000, 768, 768), (2000, 1160, 4096), (2500, 4096, 1024),
               (5000, 1024, 1040),
               # On 148 SMs: wide tiles whose k-blocks are split over clusters
               # of two, four and eight; rounds of wide tiles with the rows left
               # over in 64-token tiles, and with the tiles left over split.
               (1900, 1024, 4096), (1000, 1016, 8192), (500, 1024, 16384), (5000, 1024, 4096),
               (640, 8192, 8192),
               # Pairs: even and odd counts of 128-row tiles, one and several
               # chunks of scales, a last tile of 8 columns.
               (9400, 1032, 656), (9500, 2048, 1168), (4700, 4096, 2064), (11000, 528, 128),
               # Many columns and one tile of rows: single CTAs.
               (128, 40000, 256)]


@pytest.mark.parametrize("m,n,k", GEMM_SHAPES)
@pytest.mark.parametrize("bias,act", [(False, 0), (True, 0), (True, 1)])
def test_gemm_fp8(m, n, k, bias, act):
    g = gen(m, n, k)
    a, sa, w, sw = operands(g, m, n, k)
    b = rand(g, n) if bias else None
    ref, tol = finish(*product_ref(a, sa, w, sw), b, act)
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        out = K().gemm_fp8(a, sa, w, sw, b, act=act, out_dtype=dtype)
        check_out(out, ref, tol)
    if n % 16 == 0:
        q, s = K().gemm_fp8(a, sa, w, sw, b, act=act, out_dtype=F8)
        check_quantised(q, s, ref, tol)


@pytest.mark.parametrize("m", [1, 20, 40, 100, 700, 11000])
def test_gemm_fp8_strides(m):
    """Scales in either order, rows at a pitch, a pitched output whose gaps
    stay as they were."""
    g = gen(m)
    n, k = 520, 656
    a, sa, w, sw = operands(g, m, n, k)
    ref, tol = product_ref(a, sa, w, sw)
    wide_a = torch.zeros(m, k + 48, device=DEV).to(F8)
    wide_a[:, :k] = a
    wide_w = torch.zeros(n, k + 16, device=DEV).to(F8)
    wide_w[:, :k] = w
    out = torch.full((m, n + 24), 7.0, device=DEV, dtype=torch.float16)
    got = K().gemm_fp8(wide_a[:, :k], sa.t().contiguous().t(), wide_w[:, :k],
                       sw.t().contiguous().t(), out_dtype=torch.float16, out=out[:, :n])
    assert got.data_ptr() == out.data_ptr()
    check_out(out[:, :n], ref, tol)
    assert (out[:, n:] == 7).all()
    whole = K().gemm_fp8(a, sa, w, sw, out_dtype=torch.float16)
    assert torch.equal(whole, out[:, :n])


@pytest.mark.parametrize("m", [5, 90, 600, 9000])
def test_gemm_fp8_bad_values_stay_in_their_rows(m):
    """A NaN or an infinity in one token's operand or scale reaches that
    token's outputs only."""
    g = gen(m, 3)
    n, k = 768, 528
    a, sa, w, sw = operands(g, m, n, k)
    clean = K().gemm_fp8(a, sa, w, sw)
    r1, r2 = m // 2, m - 1
    a[r1, 17] = float("nan")
    sa[r2, 4] = float("inf")
    out = K().gemm_fp8(a, sa, w, sw)
    assert out[r1].isnan().all() and not out[r2].isfinite().any()
    keep = torch.ones(m, dtype=torch.bool, device=DEV)
    keep[[r1, r2]] = False
    assert torch.equal(out[keep], clean[keep])
    q, s = K().gemm_fp8(a, sa, w, sw, out_dtype=F8)
    assert (q[r1].float() * per_block(s, m, n)[r1].float()).isnan().all()


def test_gemm_fp8_same_bits_again():
    """A call's result depends on its operands alone: not on the stream, on
    what runs beside it or on being replayed."""
    g = gen(77)
    cases = [operands(g, m, 1024, 2048) for m in (1, 24, 200, 1500, 5000)]
    want = [K().gemm_fp8(*c, out_dtype=torch.float32) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for st, c in zip(streams, cases):
            with torch.cuda.stream(st):
                got.append(K().gemm_fp8(*c, out_dtype=torch.float32))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


# ------------------------------------------------------------- padded batches

@pytest.mark.parametrize("seq", [200, 1024, 8192])
@pytest.mark.parametrize("res_dtype", [torch.float32, torch.float16])
def test_live_tiles(seq, res_dtype):
    """With a live-tile list, rows of unlisted tiles are left as they were and
    the listed ones come out as without it."""
    g = gen(seq)
    b, d, n = 4, 272, 528
    lengths = torch.tensor([seq, 0, seq // 3, 1], dtype=torch.int32, device=DEV)
    tiles = K().row_tiles(lengths, None, b, seq, torch.device(DEV, 0))
    rows = b * seq
    listed = tiles[1:1 + int(tiles[0])].tolist()
    live = torch.zeros(rows, dtype=torch.bool, device=DEV)
    for t in listed:
        live[t * 128:(t + 1) * 128] = True
    assert live.any() and not live.all()
    res, delta, w = rand(g, rows, d).to(res_dtype), rand(g, rows, d).half(), rand(g, d)
    full_res, (fq, fs) = K().fused_add_rmsnorm(res, delta, w, 1e-5, out_dtype=F8)
    keep = res.clone()
    new, (q, s) = K().fused_add_rmsnorm(res, delta, w, 1e-5, out_dtype=F8, residual_out=res,
                                        m_tiles=tiles)
    assert torch.equal(new[live], full_res[live]) and torch.equal(new[~live], keep[~live])
    assert torch.equal(q.view(torch.uint8)[live], fq.view(torch.uint8)[live])
    assert torch.equal(s[live], fs[live])
    x = rand(g, rows, d).bfloat16()
    q2, s2 = K().quantize_blocks(x, m_tiles=tiles)
    fq2, fs2 = K().quantize_blocks(x)
    assert torch.equal(q2.view(torch.uint8)[live], fq2.view(torch.uint8)[live])
    assert torch.equal(s2[live], fs2[live])
    wq, ws = K().quantize_weight_blocks(rand(g, n, d, scale=d ** -0.5))
    full = K().gemm_fp8(fq, fs, wq, ws, out_dtype=torch.float16)
    out = torch.full((rows, n), 3.0, dtype=torch.float16, device=DEV)
    # Operands of unlisted rows may hold anything.
    q.view(torch.uint8)[~live] = 0x7f
    s[~live] = float("nan")
    K().gemm_fp8(q, s, wq, ws, out_dtype=torch.float16, out=out, m_tiles=tiles)
    assert torch.equal(out[live], full[live]) and (out[~live] == 3).all()


@pytest.mark.parametrize("rows", [1, 100, 700, 70000])
def test_no_live_tiles(rows):
    g = gen(rows, 9)
    tiles = torch.zeros(1 + (rows + 127) // 128, dtype=torch.int32, device=DEV)
    a, sa, w, sw = operands(g, rows, 256, 256)
    out = torch.full((rows, 256), 3.0, device=DEV)
    K().gemm_fp8(a, sa, w, sw, out_dtype=torch.float32, out=out, m_tiles=tiles)
    assert (out == 3).all()
    res, delta = rand(g, rows, 256), rand(g, rows, 256)
    keep = res.clone()
    K().fused_add_rmsnorm(res, delta, torch.ones(256, device=DEV), 1e-5, residual_out=res,
                          m_tiles=tiles)
    assert torch.equal(res, keep)


# ------------------------------------------------------------------- together

def ffn_block(res, delta, norm_w, w1, s1, b1, w2, s2, b2):
    """norm -> FFN-in with GELU, hidden in 8 bits -> FFN-out, as a block runs them."""
    res, (h, hs) = K().fused_add_rmsnorm(res, delta, norm_w, 1e-5, out_dtype=F8)
    hid, hids = K().gemm_fp8(h, hs, w1, s1, b1, act=K().ACT_GELU, out_dtype=F8)
    out = K().gemm_fp8(hid, hids, w2, s2, b2, out_dtype=torch.float16)
    return res, h, hs, hid, hids, out


def ffn_operands(g, rows, d, f):
    w1, s1 = K().quantize_weight_blocks(rand(g, f, d, scale=d ** -0.5))
    w2, s2 = K().quantize_weight_blocks(rand(g, d, f, scale=f ** -0.5))
    return (rand(g, rows, d), rand(g, rows, d).half(), 1 + 0.1 * rand(g, d), w1, s1,
            rand(g, f, scale=0.1), w2, s2, rand(g, d, scale=0.1))


@pytest.mark.parametrize("rows,d,f", [(1, 512, 2048), (77, 768, 1536), (1100, 1024, 4096)])
def test_ffn_block(rows, d, f):
    g = gen(rows, d, f)
    ops = ffn_operands(g, rows, d, f)
    res, delta, nw, w1, s1, b1, w2, s2, b2 = ops
    new, h, hs, hid, hids, out = ffn_block(*ops)
    assert torch.equal(new, res + delta.float())
    _, y = rms_ref(res, delta, nw, 1e-5)
    check_quantised(h, hs, y, NORM_REL * y.abs())
    y, tol = finish(*product_ref(h, hs, w1, s1), b1, 1)
    check_quantised(hid, hids, y, tol)
    y, tol = finish(*product_ref(hid, hids, w2, s2), b2, 0)
    check_out(out, y, tol)


@pytest.mark.parametrize("rows", [1, 300])
def test_ffn_block_captured(rows):
    """Captured on a side stream, replayed with new inputs, beside an eager run."""
    g = gen(rows, 6)
    ops = ffn_operands(g, rows, 512, 1024)
    ffn_block(*ops)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ffn_block(*ops)
        with torch.cuda.graph(graph, stream=side):
            captured = ffn_block(*ops)
    torch.cuda.current_stream().wait_stream(side)
    for seed in range(3):
        g2 = gen(rows, 7, seed)
        ops[0].copy_(rand(g2, rows, 512))
        ops[1].copy_(rand(g2, rows, 512).half())
        graph.replay()
        want = ffn_block(*ops)
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_large_offsets():
    """Element offsets past 2^31 in every operand that can have them."""
    rows, d = (1 << 31) // 1024 + 300, 1024
    res = torch.zeros(rows, d, device=DEV, dtype=torch.float16)
    g = gen(1)
    tail = rand(g, 300, d).half()
    res[-300:] = tail
    w = torch.ones(d, device=DEV)
    _, ref = rms_ref(tail, None, w, 1e-5)
    q, s = K().rmsnorm(res, w, 1e-5, out_dtype=F8)
    check_quantised(q[-300:], s[-300:], ref, NORM_REL * ref.abs())
    del q, s
    q, s = K().quantize_blocks(res)
    check_quantised(q[-300:], s[-300:], tail.double(), 0.0)
    del res
    wq, ws = K().quantize_weight_blocks(rand(g, 1024, d, scale=d ** -0.5))
    out = K().gemm_fp8(q, s, wq, ws, out_dtype=torch.float16)
    ref, tol = product_ref(q[-300:], s[-300:], wq, ws)
    check_out(out[-300:], ref, tol)
    assert (out[:1000] == 0).all()


def test_row_pitch_past_32_bits():
    """Rows of an operand 2^32 + 256 elements apart."""
    g = gen(2)
    pitch = (1 << 32) + 256
    a, sa, w, sw = operands(g, 2, 64, 16)
    raw = torch.zeros(pitch + 512, dtype=torch.uint8, device=DEV)
    far = raw.as_strided((2, 16), (pitch, 1)).view(F8)
    far.view(torch.uint8).copy_(a.view(torch.uint8))
    raw[256:272] = 0x38
    assert far.stride(0) == pitch
    assert torch.equal(K().gemm_fp8(far, sa, w, sw), K().gemm_fp8(a, sa, w, sw))
    out = raw.view(torch.bfloat16).as_strided((2, 64), (1 << 31, 1))
    with pytest.raises(ValueError):
        K().gemm_fp8(a, sa, w, sw, out=out)
    half = raw.view(torch.float16)
    assert half.numel() > 1 << 31
    with pytest.raises(ValueError):
        K().quantize_blocks(half[:1 << 31].view(1, -1))
    with pytest.raises(ValueError):
        K().quantize_weight_blocks(half[:1 << 31].view(1, -1))
    many = (1 << 32) + 5
    with pytest.raises(ValueError):
        K().gemm_fp8(a[:1].expand(many, 16), sa[:1].expand(many, 1), w, sw)


def test_two_streams():
    """Calls of every form in flight on two streams at once give what each
    gives alone."""
    g = gen(12)
    n, k = 1024, 2048
    wq, ws = K().quantize_weight_blocks(rand(g, n, k, scale=k ** -0.5))
    sets = [operands(g, m, 16, k)[:2] for m in (5, 30, 60, 300, 3000)]
    x = acts(g, 700, k)
    nw = torch.ones(k, device=DEV)

    def work():
        outs = [K().gemm_fp8(a, s, wq, ws) for a, s in sets]
        return outs + [*K().rmsnorm(x, nw, 1e-5, out_dtype=F8), *K().quantize_weight_blocks(x)]

    want = work()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        for s, kept in zip(streams, got):
            with torch.cuda.stream(s):
                kept.append(work())
    torch.cuda.synchronize()
    for outs in got[0] + got[1]:
        for a, b in zip(outs, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


FIRST_CAPTURED = """
import torch
import tjkernels.kernels as K
torch.manual_seed(0)
x = torch.randn({rows}, 512, device="cuda")
w = torch.randn(256, 512, device="cuda")
nw = torch.ones(512, device="cuda")
graph = torch.cuda.CUDAGraph()

def work():
    wq, ws = K.quantize_weight_blocks(w)
    h, hs = K.rmsnorm(x, nw, 1e-5, out_dtype=torch.float8_e4m3fn)
    return K.gemm_fp8(h, hs, wq, ws), K.gemm_fp8(*K.quantize_blocks(x), wq, ws)

with torch.cuda.graph(graph):
    got = work()
graph.replay()
for a, b in zip(got, work()):
    assert a.isfinite().all() and torch.equal(a, b)
"""


@pytest.mark.parametrize("rows", [3, 2000])
def test_first_calls_of_a_process_captured(rows):
    """Nothing has to be called once before it can be captured."""
    import tjkernels
    path = os.path.dirname(os.path.dirname(tjkernels.__file__))
    subprocess.run([sys.executable, "-c", FIRST_CAPTURED.format(rows=rows)], check=True,
                   timeout=120, env={**os.environ, "PYTHONPATH": path})


# ------------------------------------------------------------------ refusals

def test_refusals():
    from tjkernels._lib import KernelError
    g = gen(4)
    a, sa, w, sw = operands(g, 8, 128, 256)
    with pytest.raises(TypeError):
        K().gemm_fp8(a.half(), sa, w, sw)
    with pytest.raises(TypeError):
        K().gemm_fp8(a, sa.half(), w, sw)
    with pytest.raises(ValueError):
        K().gemm_fp8(a, sa[:, :1], w, sw)
    with pytest.raises(ValueError):
        K().gemm_fp8(a, sa, w, sw[:, :1])
    with pytest.raises(ValueError):
        K().gemm_fp8(a[:, :128], sa, w, sw)
    with pytest.raises(ValueError):
        K().gemm_fp8(a, sa, w, sw, bias=torch.zeros(64, device=DEV))
    with pytest.raises(ValueError):
        K().gemm_fp8(a, sa, w, sw, out=torch.zeros(8, 120, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        K().gemm_fp8(a, sa, w, sw, m_tiles=torch.zeros(1, dtype=torch.int32, device=DEV))
    with pytest.raises(TypeError):
        K().gemm_fp8(a, sa, w, sw, out_dtype=torch.float64)
    with pytest.raises(KernelError):
        K().gemm_fp8(a, sa, w, sw, act=2)
    with pytest.raises(KernelError):  # K not a multiple of 16
        K().gemm_fp8(a[:, :24].contiguous(), sa[:, :1], w[:, :24].contiguous(),
                     sw[:, :1])
    with pytest.raises(KernelError):
        K().quantize_blocks(torch.zeros(4, 24, device=DEV))
    with pytest.raises(KernelError):
        K().quantize_weight_blocks(torch.zeros(4, 24, device=DEV))
    with pytest.raises(TypeError):
        K().quantize_blocks(torch.zeros(4, 32, device=DEV, dtype=torch.float64))
    w32 = torch.ones(32, device=DEV)
    x = torch.zeros(4, 32, device=DEV)
    with pytest.raises(ValueError):
        K().fused_add_rmsnorm(x, x[:2], w32, 1e-5)
    with pytest.raises(ValueError):
        K().fused_add_rmsnorm(x, None, w32[:16], 1e-5)
    with pytest.raises(ValueError):
        K().fused_add_rmsnorm(x, x, w32, 1e-5, residual_out=x.half())
    with pytest.raises(ValueError):
        K().fused_add_rmsnorm(x.t(), None, torch.ones(4, device=DEV), 1e-5)
    with pytest.raises(KernelError):
        K().rmsnorm(torch.zeros(4, 16400, device=DEV), torch.ones(16400, device=DEV), 1e-5)
    with pytest.raises(KernelError):
        K().rmsnorm(torch.zeros(4, 20, device=DEV), torch.ones(20, device=DEV), 1e-5,
                    out_dtype=F8)
    with pytest.raises(RuntimeError):
        K().gemm_fp8(a, sa.cpu(), w, sw)
