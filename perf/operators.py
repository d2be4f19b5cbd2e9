"""The operators around a projection in 8-bit floating point, in their plain form and as the library's calls.

A program that runs an attention layer's projections in 8 bits quantises its rows (and once its
weights) to e4m3 with a power-of-two scale for each block of 128, multiplies the two, and rotates the
queries and keys that come out by their positions.  `own` chooses between elementary torch operations
and the library's kernels (quant_fp8, gemm_fp8 and rope of awa_hip.Context).

Inputs come from the seed alone and are made on the GPU: activations N(0, 1) with one value in a
thousand eight times as large, weights N(0, 0.02), biases N(0, 0.02).
"""
import math
import os
import sys

import torch

own = False

DIM, QKV, MLP, HEADS, HEAD_D = 2560, 7680, 6912, 20, 128  # the model's widths
BLOCK = 128    # values per scale
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases

def _quant(name, rows, cols, dtype, blocks=False, ld=0):
    return {"name": name, "kind": "quant", "rows": rows, "cols": cols, "ld": ld or cols, "dtype": dtype,
            "blocks": blocks}


def _gemm(name, rows, n, k, dtype, bias=False):
    return {"name": name, "kind": "gemm", "rows": rows, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _rope(name, tokens, heads, head_d, axes, pairs, layout, dtype, ld=0, far=1 << 15, factor=1.0, inverse=False):
    """pairs: rotated channel pairs of each axis; ld: elements from token to token; factor: context stretch."""
    return {"name": name, "kind": "rope", "tokens": tokens, "heads": heads, "head_d": head_d, "axes": axes,
            "pairs": pairs, "layout": layout, "dtype": dtype, "ld": ld or heads * head_d, "far": far,
            "factor": factor, "inverse": inverse}


def listed():
    return [
        # the text rows of one layer: the smallest call of the quantiser, bounded by its launch
        _quant("quant_text", 58, DIM, "bf16"),
        # a clip of five latent frames of 1080p and its text, the projections' input
        _quant("quant_clip", 5 * 5440 + 58, DIM, "bf16"),
        # fp32 rows of no round size inside a wider buffer
        _quant("quant_odd_f32", 1237, 2693, "f32", ld=2701),
        # a weight laid out once: the fused SwiGLU matrix
        _quant("quant_weight", 2 * MLP, DIM, "bf16", blocks=True),
        # one row through the qkv projection (a timestep's vector, a single token): bound by the weight
        _gemm("gemm_one_row", 1, QKV, DIM, "bf16"),
        # a prompt's text rows through the qkv projection
        _gemm("gemm_text", 58, QKV, DIM, "bf16"),
        # 360p, the MLP's second product, added to an fp32 residual by the caller
        _gemm("gemm_360p_mlp_out_f32", 621 + 58, DIM, MLP, "f32", bias=True),
        # 1080p, the MLP's first product: the largest of a layer
        _gemm("gemm_1080p_mlp_in", 5440 + 58, 2 * MLP, DIM, "bf16"),
        # sizes that no tile divides
        _gemm("gemm_odd", 1237, 1999, 2693, "bf16", bias=True),
        # one token's queries and keys
        _rope("rope_one_token", 1, 2 * HEADS, HEAD_D, 3, 21, "interleaved", "bf16"),
        # 1080p: queries and keys inside the qkv rows, three axes of 21 pairs, two channels left alone
        _rope("rope_1080p_qkv", 5440, 2 * HEADS, HEAD_D, 3, 21, "interleaved", "bf16", ld=QKV, far=80),
        # a long text, stretched to 32 times its trained length, the gradient's direction
        _rope("rope_long_half_f32", 20000, 12, 96, 1, 32, "half", "f32", far=1 << 20, factor=32.0, inverse=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(("quant", "gemm", "rope"))
    if kind == "quant":
        cols = _log(rng, 96, 8192)
        rows = _log(rng, 1, min(27000, 41_000_000 // cols))
        ld = cols + rng.choice((0, 0, 8, 13))
        return _quant("", rows, cols, rng.choice(("bf16", "f32")), rng.random() < 0.3, ld)
    if kind == "gemm":
        rows, n, k = _log(rng, 1, 6000), _log(rng, 64, 14000), _log(rng, 100, 8192)
        while rows * n * k > 5498 * 2 * MLP * DIM:
            rows = (rows + 1) // 2
        if rng.random() < 0.5:  # a width that a model has
            n, k = max(64, n // 64 * 64), max(128, k // 128 * 128)
        return _gemm("", rows, n, k, rng.choice(("bf16", "f32")), rng.random() < 0.5)
    heads, head_d = rng.choice((1, 2, 5, 8, 16, 40)), rng.choice((64, 80, 96, 128, 256))
    axes = rng.choice((1, 1, 2, 3))
    tokens = _log(rng, 1, min(60000, 22_000_000 // (heads * head_d)))
    pairs = head_d // 2 // axes // rng.choice((1, 1, 2))
    return _rope("", tokens, heads, head_d, axes, pairs, rng.choice(("interleaved", "half")),
                 rng.choice(("bf16", "f32")), heads * head_d + rng.choice((0, 0, 256, 3)),
                 rng.choice((64, 4096, 1 << 20)), rng.choice((1.0, 1.0, 8.0)), rng.random() < 0.3)


# ------------------------------------------------------------------ inputs

def _padded(k):
    return (k + BLOCK - 1) // BLOCK * BLOCK


def _groups(k):
    """Words of four blocks' scales in a row."""
    return (k + 4 * BLOCK - 1) // (4 * BLOCK)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, cols, g):
    x = torch.randn((rows, cols), generator=g, device="cuda")
    return torch.where(torch.rand((rows, cols), generator=g, device="cuda") < 1e-3, 8 * x, x)


def _frequencies(case):
    """Radians per position of each pair, axis after axis, base 10000; a stretched context keeps the pairs
    that turn often over the trained length and slows the others."""
    n, lo, hi, trained = case["pairs"], 1.0, 32.0, 4096.0
    f = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    t = ((trained * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
    f = f * (t + (1 - t) / case["factor"])
    return f.repeat(case["axes"]).numpy()


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": dict(case), "dtype": dtype}
    if case["kind"] == "quant":
        x = _activations(case["rows"], case["ld"], g)
        s["x"] = (x * 0.02 if case["blocks"] else x).to(dtype)[:, : case["cols"]]
    elif case["kind"] == "gemm":
        s["a"], s["as"] = _plain_quant(_activations(case["rows"], case["k"], g), False)
        s["w"], s["ws"] = _plain_quant(torch.randn((case["n"], case["k"]), generator=g, device="cuda") * 0.02, True)
        s["bias"] = torch.randn(case["n"], generator=g, device="cuda") * 0.02 if case["bias"] else None
    else:
        t, h, d = case["tokens"], case["heads"], case["head_d"]
        buf = torch.randn((t, case["ld"]), generator=g, device="cuda").to(dtype)
        s["x"] = buf[:, : h * d].unflatten(1, (h, d))
        s["pos"] = torch.randint(0, case["far"], (t, case["axes"]), generator=g, device="cuda", dtype=torch.int32)
        s["freqs"] = _frequencies(case)
        s["freqs_dev"] = torch.from_numpy(s["freqs"]).cuda()
        s["scale"] = 0.1 * math.log(case["factor"]) + 1.0
    return s


# ------------------------------------------------------------------ the plain forms

def _plain_quant(x, blocks):
    """(e4m3 rows, padded with zeros to whole blocks; e8m0 scales [groups of four blocks][rows][4])."""
    rows, cols = x.shape
    kp, per = _padded(cols), BLOCK if blocks else 1
    x = torch.nn.functional.pad(x.float(), (0, kp - cols, 0, -rows % per))
    x = x.unflatten(0, (-1, per)).unflatten(2, (-1, BLOCK))  # row groups, rows, blocks, values
    top = x.abs().amax((1, 3), keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(top > 0, e - torch.where(m <= 0.875, 9, 8), -127).clamp(min=-127)
    q = torch.ldexp(x, -e).to(torch.float8_e4m3fn).flatten(2).flatten(0, 1)[:rows]
    b = (e[:, 0, :, 0] + 127).to(torch.uint8)
    b = torch.nn.functional.pad(b, (0, 4 * _groups(cols) - b.shape[1]))
    return q.contiguous(), b.unflatten(1, (-1, 4)).transpose(0, 1).contiguous().view(torch.float8_e8m0fnu)


def _scales(s, kp):
    """[rows][blocks] fp32 of the words' layout; the exponent bytes put into place (a power of two is exact)."""
    b = s.view(torch.uint8).transpose(0, 1).flatten(1)[:, : kp // BLOCK]
    return torch.ldexp(torch.ones_like(b, dtype=torch.float32), b.int() - 127)


def _plain_gemm(s):
    kp, n = s["a"].shape[1], s["w"].shape[0]
    a = s["a"].float().unflatten(1, (-1, BLOCK)) * _scales(s["as"], kp)[:, :, None]
    w = s["w"].float().unflatten(1, (-1, BLOCK)) * _scales(s["ws"], kp).repeat_interleave(BLOCK, 0)[:n, :, None]
    c = a.flatten(1) @ w.flatten(1).T
    if s["bias"] is not None:
        c = c + s["bias"]
    return c.to(s["dtype"])


def _plain_rope(s):
    case, x = s["case"], s["x"].float()
    turn = s["pos"].double().repeat_interleave(case["pairs"], 1) * s["freqs_dev"]  # angles of far positions
    cos, sin = (s["scale"] * turn.cos()).float()[:, None], (s["scale"] * turn.sin()).float()[:, None]
    if case["inverse"]:
        sin = -sin
    p = cos.shape[-1]
    if case["layout"] == "half":
        a, b = x[..., :p], x[..., p:2 * p]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos, x[..., 2 * p:]), -1)
    else:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        y = torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), x[..., 2 * p:]), -1)
    return y.to(s["dtype"])


# ------------------------------------------------------------------ one pass

_held = []


def _context():
    """The library's handle, which a program makes once."""
    if not _held:
        sys.path.insert(0, os.path.join(os.getcwd(), "seedvr2-2b-ncnn_amd"))
        import awa_hip
        _held.append(awa_hip.Context(0))
    return _held[0]


def run(state):
    s, case = state, state["case"]
    if case["kind"] == "quant":
        if own:
            return _context().quant_fp8(s["x"], blocks=case["blocks"])
        return _plain_quant(s["x"], case["blocks"])
    if case["kind"] == "gemm":
        if own:
            return _context().gemm_fp8(s["a"], s["as"], s["w"], s["ws"], bias=s["bias"], dtype=s["dtype"])
        return _plain_gemm(s)
    if own:
        return _context().rope(s["x"], s["pos"], s["freqs"], pairs=(case["pairs"],) * case["axes"],
                               layout=case["layout"], scale=s["scale"], inverse=case["inverse"])
    return _plain_rope(s)


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "quant":
        rows, cols = case["rows"], case["cols"]
        words = _groups(cols) * (-(-rows // BLOCK) if case["blocks"] else rows)
        return {"bytes": rows * (cols * size + _padded(cols)) + 4 * words, "flops": 3 * rows * cols}
    if case["kind"] == "gemm":
        m, n, k = case["rows"], case["n"], _padded(case["k"])
        words = _groups(k) * (m + -(-n // BLOCK))
        return {"bytes": m * k + n * k + 4 * words + m * n * size + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    values = case["tokens"] * case["heads"] * case["head_d"]
    turned = case["tokens"] * case["heads"] * 2 * case["pairs"] * case["axes"]
    return {"bytes": 2 * values * size + 4 * case["tokens"] * case["axes"], "flops": 3 * turned}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_quant(x, blocks):
    rows, cols = x.shape
    nb, per = _padded(cols) // BLOCK, BLOCK if blocks else 1
    nr = -(-rows // per)
    v = torch.zeros((nr * per, nb * BLOCK), dtype=torch.float64, device=x.device)
    v[:rows, :cols] = x.double()
    v = v.reshape(nr, per, nb, BLOCK)
    top = v.abs().amax((1, 3))
    e = torch.ceil(torch.log2(top / E4M3_MAX)).clamp(min=-127.0)  # of zero: -inf, then -127
    v = v / torch.exp2(e)[:, None, :, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs())).clamp(min=-6.0) - 3)  # e4m3: three bits after the first
    q = (torch.round(v / step) * step).reshape(nr * per, nb * BLOCK)[:rows]
    scales = torch.full((nr, 4 * _groups(cols)), 2.0 ** -127, dtype=torch.float64, device=x.device)
    scales[:, :nb] = torch.exp2(e)
    return q, scales.reshape(nr, -1, 4).permute(1, 0, 2).contiguous()


def _exact_gemm(s):
    def values(q, scale, per):
        rows, kp = q.shape
        sc = scale.double().permute(1, 0, 2).reshape(scale.shape[1], -1)[:, : kp // BLOCK]
        row = torch.arange(rows, device=q.device) // per
        col = torch.arange(kp, device=q.device) // BLOCK
        return q.double() * sc[row][:, col]

    c = values(s["a"], s["as"], 1) @ values(s["w"], s["ws"], BLOCK).T
    return c if s["bias"] is None else c + s["bias"].double()


def _exact_rope(s):
    case = s["case"]
    y = s["x"].double().clone()
    p = case["pairs"] * case["axes"]
    axis = torch.arange(p, device=y.device) // case["pairs"]
    angle = s["pos"].double()[:, axis] * torch.from_numpy(s["freqs"]).to(y.device)
    z = torch.polar(torch.full_like(angle, s["scale"]), -angle if case["inverse"] else angle)[:, None]
    i = torch.arange(p, device=y.device)
    first, second = (i, i + p) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        return _exact_quant(s["x"], case["blocks"])
    return _exact_gemm(s) if case["kind"] == "gemm" else _exact_rope(s)
