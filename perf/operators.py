"""The block-scaled 8-bit operators: their plain forms, the sizes they are measured at, and what each pass costs at least.

Four operators that make up the linear layers of a block with 8-bit (e4m3) operands:

* ``norm``      residual addition and root-mean-square norm, output in 32, 16 or 8 bits
* ``quantize``  activations to e4m3 with one scale for each row and 128 columns
* ``weights``   weights to e4m3 with one scale for each 128 x 128 block
* ``gemm``      product of two such matrices, with bias, GELU and an output in 32, 16 or 8 bits

A block of values y gets the scale s = max(amax|y| / 448, 2^-126) and is held as e4m3(y / s).
"""

import functools
import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
EPS = 1e-5
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
          "e4m3": torch.float8_e4m3fn}


@functools.cache
def _kernels():
    pkg = str(Path.cwd() / "tiktok-techjam-2026_b200")
    sys.path.insert(0, pkg)
    import tjkernels.kernels as K
    return K


# ---------------------------------------------------------------------- cases

def listed():
    return [
        # One token through the norm in front of a product (d_model 1024).
        dict(name="norm_token", op="norm", rows=1, d=1024, res="f32", delta="f16", out="e4m3"),
        # A ragged batch, 16-bit residual stream, a width that ends inside a block of 128.
        dict(name="norm_ragged", op="norm", rows=4999, d=1040, res="bf16", delta="bf16",
             out="bf16"),
        # A large-model batch (d_model 4096, 32 sequences of 2048 tokens), fp32 residual stream.
        dict(name="norm_large", op="norm", rows=65536, d=4096, res="f32", delta="f16",
             out="e4m3"),
        # The attention output of a few decoded tokens, before the out-projection.
        dict(name="quantize_tokens", op="quantize", rows=5, k=4096, src="f16"),
        # The attention output of a large-model batch on one GPU (8 sequences of 2048).
        dict(name="quantize_context", op="quantize", rows=16384, k=4096, src="f16"),
        # The FFN-in weights of the large model, once when they are loaded.
        dict(name="weights_ffn", op="weights", n=16384, k=4096, src="f32"),
        # One token through a projection of the large model: the weights' bytes count.
        dict(name="gemm_token", op="gemm", m=1, n=4096, k=4096, out="f16", act="none", bias=True),
        # A small batch of tokens through the FFN-in, hidden activations kept in 8 bits.
        dict(name="gemm_small_batch", op="gemm", m=48, n=16384, k=4096, out="e4m3", act="gelu",
             bias=True),
        # Sizes that end inside a tile in every direction, fp32 output.
        dict(name="gemm_ragged", op="gemm", m=1357, n=1160, k=1040, out="f32", act="none",
             bias=False),
        # The live tokens of a half-padded 8 x 1024 batch through the FFN-out (d_model 1024).
        dict(name="gemm_ffn_out", op="gemm", m=5000, n=1024, k=4096, out="bf16", act="none",
             bias=True),
        # 4 sequences of 4096 tokens through the FFN-in, GELU, 8-bit hidden activations.
        dict(name="gemm_ffn_in", op="gemm", m=16384, n=4096, k=1024, out="e4m3", act="gelu",
             bias=True),
        # The large model's FFN-out on one GPU.
        dict(name="gemm_large", op="gemm", m=16384, n=4096, k=16384, out="f16", act="none",
             bias=True),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(step, int(round(v / step)) * step)


def draw(rng):
    op = rng.choice(["norm", "quantize", "weights", "gemm", "gemm", "gemm"])
    if op == "norm":
        out = rng.choice(["e4m3", "e4m3", "bf16", "f16", "f32"])
        d = _log(rng, 64, 8192, 16 if out == "e4m3" else 4)
        rows = _log(rng, 1, min(65536, (1 << 28) // d))
        return dict(op=op, rows=rows, d=d, res=rng.choice(["f32", "f16", "bf16"]),
                    delta=rng.choice(["none", "f32", "f16", "bf16"]), out=out)
    if op == "quantize":
        k = _log(rng, 64, 16384, 16)
        return dict(op=op, rows=_log(rng, 1, min(65536, (1 << 26) // k)), k=k,
                    src=rng.choice(["f32", "f16", "bf16"]))
    if op == "weights":
        return dict(op=op, n=_log(rng, 8, 16384, 8), k=_log(rng, 64, 4096, 16),
                    src=rng.choice(["f32", "f16", "bf16"]))
    out = rng.choice(["e4m3", "bf16", "f16", "f32"])
    return dict(op=op, m=_log(rng, 1, 16384), n=_log(rng, 64, 8192, 16 if out == "e4m3" else 8),
                k=_log(rng, 64, 8192, 16), out=out, act=rng.choice(["none", "gelu"]),
                bias=rng.random() < 0.7)


# --------------------------------------------------------------------- inputs

def _channels(n, g, dev, spread):
    """Per-channel magnitudes: most alike, a few large ones, as activations have."""
    return torch.exp(spread * torch.randn(n, device=dev, generator=g))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    op = case["op"]
    if op == "norm":
        rows, d = case["rows"], case["d"]
        ch = _channels(d, g, dev, 0.7)
        res = (randn(rows, d) * ch).to(DTYPES[case["res"]])
        delta = None
        if case["delta"] != "none":
            delta = (randn(rows, d) * (0.3 * ch)).to(DTYPES[case["delta"]])
        return dict(case=case, res=res, delta=delta, weight=1.0 + 0.1 * randn(d))
    if op == "quantize":
        x = randn(case["rows"], case["k"]) * _channels(case["k"], g, dev, 0.7)
        return dict(case=case, x=x.to(DTYPES[case["src"]]))
    if op == "weights":
        w = randn(case["n"], case["k"]) * case["k"] ** -0.5
        return dict(case=case, x=w.to(DTYPES[case["src"]]))
    m, n, k = case["m"], case["n"], case["k"]
    a, a_scales = _plain_rows(randn(m, k) * _channels(k, g, dev, 0.7))
    w, w_scales = _plain_tiles(randn(n, k) * k ** -0.5)
    bias = randn(n) * 0.1 if case["bias"] else None
    return dict(case=case, a=a, a_scales=a_scales, w=w, w_scales=w_scales, bias=bias)


# ----------------------------------------------------------------- plain forms

def _plain_rows(y):
    """fp32 [R, K] -> e4m3 [R, K] and one scale for each row and 128 columns."""
    rows, k = y.shape
    kb = -(-k // BLOCK)
    t = torch.nn.functional.pad(y, (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
    s = (t.abs().amax(dim=2) / E4M3_MAX).clamp_min(SCALE_MIN)
    q = (t / s[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(rows, kb * BLOCK)[:, :k].contiguous(), s


def _plain_tiles(w):
    """fp32 [N, K] -> e4m3 [N, K] and one scale for each 128 x 128 block."""
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    t = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    t = t.view(nb, BLOCK, kb, BLOCK)
    s = (t.abs().amax(dim=(1, 3)) / E4M3_MAX).clamp_min(SCALE_MIN)
    q = (t / s[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous(), s


def _plain_out(y, out):
    if out == "e4m3":
        return _plain_rows(y)
    return y.to(DTYPES[out])


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        K = _kernels()
        if op == "norm":
            return K.fused_add_rmsnorm(state["res"], state["delta"], state["weight"], EPS,
                                       out_dtype=DTYPES[case["out"]])
        if op == "quantize":
            return K.quantize_blocks(state["x"])
        if op == "weights":
            return K.quantize_weight_blocks(state["x"])
        return K.gemm_fp8(state["a"], state["a_scales"], state["w"], state["w_scales"],
                          state["bias"],
                          act=K.ACT_GELU if case["act"] == "gelu" else K.ACT_NONE,
                          out_dtype=DTYPES[case["out"]])
    if op == "norm":
        x = state["res"].float()
        if state["delta"] is not None:
            x = x + state["delta"].float()
        y = x * torch.rsqrt(x.square().mean(dim=1, keepdim=True) + EPS) * state["weight"]
        return x.to(state["res"].dtype), _plain_out(y, case["out"])
    if op == "quantize":
        return _plain_rows(state["x"].float())
    if op == "weights":
        return _plain_tiles(state["x"].float())
    m, n, k = case["m"], case["n"], case["k"]
    a = state["a"].float() * state["a_scales"].repeat_interleave(BLOCK, dim=1)[:, :k]
    w = state["w"].float() * state["w_scales"].repeat_interleave(BLOCK, dim=0)[:n] \
        .repeat_interleave(BLOCK, dim=1)[:, :k]
    y = a @ w.t()
    if state["bias"] is not None:
        y = y + state["bias"]
    if case["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    return _plain_out(y, case["out"])


# ------------------------------------------------------------------------ cost

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "none": 0}
    op = case["op"]
    if op == "norm":
        rows, d = case["rows"], case["d"]
        # residual read, delta read, sum written (with a delta), output written
        a = size[case["res"]] * (2 if case["delta"] != "none" else 1)
        b = rows * d * (a + size[case["delta"]] + size[case["out"]]) + 4 * d
        if case["out"] == "e4m3":
            b += 4 * rows * -(-d // BLOCK)
        return {"bytes": b, "flops": 6 * rows * d}
    if op == "quantize":
        rows, k = case["rows"], case["k"]
        return {"bytes": rows * k * (size[case["src"]] + 1) + 4 * rows * -(-k // BLOCK),
                "flops": 3 * rows * k}
    if op == "weights":
        n, k = case["n"], case["k"]
        return {"bytes": n * k * (size[case["src"]] + 1) + 4 * -(-n // BLOCK) * -(-k // BLOCK),
                "flops": 3 * n * k}
    m, n, k = case["m"], case["n"], case["k"]
    kb, nb = -(-k // BLOCK), -(-n // BLOCK)
    b = m * k + n * k + 4 * (m + nb) * kb + m * n * size[case["out"]]
    if case["bias"]:
        b += 4 * n
    if case["out"] == "e4m3":
        b += 4 * m * nb
    return {"bytes": b, "flops": 2 * m * n * k}


# ------------------------------------------------------------ 64-bit reference

def _e4m3(v):
    """The e4m3 value nearest to v (ties to even), saturating; v in 64 bits."""
    mag = v.abs()
    _, e = torch.frexp(mag)                       # mag = f 2^e, f in [1/2, 1)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3.0)
    return torch.copysign((torch.round(mag / step) * step).clamp_max(E4M3_MAX), v)


def _exact_blocks(y, rows_per_block):
    """(values, scales) of y's blocks of rows_per_block x 128, from the definition."""
    r, k = y.shape
    scales = []
    out = torch.empty_like(y)
    for c in range(0, k, BLOCK):
        col = y[:, c:c + BLOCK]
        top = col.abs().amax(dim=1)
        if rows_per_block > 1:
            pieces = [p.amax() for p in top.split(rows_per_block)]
            s = torch.stack(pieces).div(E4M3_MAX).clamp_min(SCALE_MIN)
            per_row = s[torch.arange(r, device=y.device) // rows_per_block]
        else:
            per_row = s = top.div(E4M3_MAX).clamp_min(SCALE_MIN)
        out[:, c:c + BLOCK] = _e4m3(col / per_row[:, None])
        scales.append(s)
    return out, torch.stack(scales, dim=1)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_blocks(st["x"].double(), 1)
    if op == "weights":
        return _exact_blocks(st["x"].double(), BLOCK)
    if op == "norm":
        x = st["res"].double()
        if st["delta"] is not None:
            x += st["delta"].double()
        y = x / (x.pow(2).sum(dim=1, keepdim=True) / case["d"] + EPS).sqrt()
        y *= st["weight"].double()
        return x, (_exact_blocks(y, 1) if case["out"] == "e4m3" else y)
    a, w = st["a"].double(), st["w"].double()
    rows = torch.arange(case["n"], device=w.device) // BLOCK
    for b in range(-(-case["k"] // BLOCK)):
        cols = slice(b * BLOCK, (b + 1) * BLOCK)
        a[:, cols] *= st["a_scales"][:, b:b + 1].double()
        w[:, cols] *= st["w_scales"][rows, b].double()[:, None]
    y = torch.mm(a, w.T)
    if st["bias"] is not None:
        y += st["bias"].double()
    if case["act"] == "gelu":
        y = 0.5 * y * torch.erfc(-y / math.sqrt(2.0))
    return _exact_blocks(y, 1) if case["out"] == "e4m3" else y
