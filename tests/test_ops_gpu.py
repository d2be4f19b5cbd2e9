"""GPU tests of the operators of dit_ops.h against plain forms in 64 bits.

Quantising is exact arithmetic up to one rounding that both sides make alike: bytes are compared for
equality.  The product's inputs are its 8-bit values, so its reference has no rounding; an fp32 sum of
products p_i is off by at most half a step (2^-24) of a partial sum per addition.  A partial sum is at most
S = sum |p_i|; a block of 128 is four bf16 instructions, and the parts of a split K are added at the end (at
most 16): bar (4 K / 128 + 16) 2^-24 S, and half a step of C's type.  For bf16 C the 8-bit instructions may sum:
they align the products of eight consecutive columns to the exponent e of the largest of them and drop what lies
below 2^(e - 13) (2^3 stays beside a product of 2^16, 2^2 does not), so each of the seven others loses less than
2^-13 of the largest, which is at most the product of the two rows' largest magnitudes in those columns: 7 2^-13
sum over the groups of those products in addition.  Rotation: a sine or cosine is off by at most 2^-22
(rounding the reduced angle, its product with pi / 2, the polynomial, the factor: under 2^-24 each) and by the
angle's own 2^-51 of itself in fp64; products and sum are fp32: bar (|a| + |b|) scale (2^-21 + |angle| 2^-51)
and half a step of the type.
"""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BF16, F32 = "bfloat16", "float32"


def dt(name):
    import torch
    return getattr(torch, name)


def half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


def within(out, ref, bar):
    """out within bar of ref everywhere; NaN where ref is, and only there."""
    import torch
    out = out.double()
    assert torch.equal(out.isnan(), ref.isnan())
    d = torch.nan_to_num((out - ref).abs() - bar, nan=-1.0)
    assert float(d.max() if d.numel() else -1) <= 0, f"over the bar by {float(d.max())}"


# ------------------------------------------------------------------ quantising

def plain_quant(x, per):
    """(e4m3 values as fp64, scale exponents [row blocks][blocks]) of the definition, for finite and other values."""
    import torch
    rows, cols = x.shape
    kp, rp = -(-cols // 128) * 128, -(-max(rows, 1) // per) * per
    v = torch.zeros((rp, kp), dtype=torch.float64, device=x.device)
    v[:rows, :cols] = x.double()
    fin = torch.where(v.isfinite(), v.abs(), 0.0).reshape(rp // per, per, kp // 128, 128).amax((1, 3))
    e = torch.ceil(torch.log2(fin / 448.0)).clamp(min=-127.0)
    y = v / torch.exp2(e).repeat_interleave(per, 0).repeat_interleave(128, 1)
    step = torch.exp2(torch.floor(torch.log2(y.abs())).clamp(min=-6.0) - 3)
    q = torch.where(y.isfinite(), torch.round(y / step) * step, math.nan)
    q = torch.where(y == 0, 0.0, q)
    return q[:rows], e.int()


def check_quant(q, scale, x, per):
    import torch
    ref, e = plain_quant(x, per)
    assert q.shape == ref.shape
    got = q.view(torch.float8_e4m3fn).double()
    assert torch.equal(got.isnan(), ref.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0), ref.nan_to_num(nan=0.0))
    b = scale.view(torch.uint8).transpose(0, 1).flatten(1).int()
    want = torch.zeros_like(b)
    want[:, :e.shape[1]] = e + 127
    assert torch.equal(b, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols,ld", [(1, 1, 1), (1, 128, 128), (3, 129, 129), (5, 511, 517), (4, 512, 520),
                                          (33, 513, 513), (58, 2560, 2560), (300, 130, 131), (2000, 2693, 2701),
                                          (1700, 2560, 7680)])
@pytest.mark.parametrize("blocks", [False, True])
def test_quant(ctx, dtype, rows, cols, ld, blocks):
    import torch
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = torch.randn((rows, ld), generator=g, device="cuda")
    x = (x * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=g, device="cuda").float())).to(dt(dtype))
    x = x[:, ld - cols:]  # begins at any element
    q, s = ctx.quant_fp8(x, blocks=blocks)
    check_quant(q, s, x, 128 if blocks else 1)


# rows times groups of 512 columns from 16384 on: two rows a wave, eight a workgroup, here with 1 to 7 left over
@pytest.mark.parametrize("rows,cols,ld", [(16387, 130, 131), (5499, 1537, 1540), (27259, 200, 200), (16385, 1, 1),
                                          (8198, 600, 611), (4100, 2048, 2048), (3282, 2560, 2561)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quant_two_rows_a_wave(ctx, awa, dtype, rows, cols, ld):
    """Against the definition, and with guard rows and words after the last row."""
    import torch
    groups, kp = -(-cols // 512), -(-cols // 128) * 128
    assert rows * groups >= 16384 and rows % 8
    test_quant(ctx, dtype, rows, cols, ld, False)
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, cols), generator=g, device="cuda").to(dt(dtype))
    q = torch.full((rows + 9, kp), 99, dtype=torch.uint8, device="cuda")
    s = torch.full((groups + 1, rows + 9), 77, dtype=torch.int32, device="cuda")
    ctx.check(awa.lib().dit_quant_fp8(ctx.ptr, awa.AWA_F32 if dtype == F32 else awa.AWA_BF16, x.data_ptr(), cols, rows,
                                      cols, 1, q.data_ptr(), s.data_ptr(), rows + 9,
                                      torch.cuda.current_stream().cuda_stream), "dit_quant_fp8")
    check_quant(q[:rows], s[:-1, :rows].contiguous().view(torch.uint8).reshape(groups, rows, 4), x, 1)
    assert bool((q[rows:] == 99).all()) and bool((s[-1] == 77).all()) and bool((s[:, rows:] == 77).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quant_two_rows_a_wave_special_values(ctx, dtype):
    """Zeros, infinities, NaN, subnormals and the type's largest value in either row of a wave."""
    import torch
    t = dt(dtype)
    x = torch.randn((16391, 256), device="cuda").to(t)
    for r, v in enumerate((0.0, math.inf, -math.inf, math.nan, torch.finfo(t).max, torch.finfo(t).tiny,
                           torch.finfo(t).smallest_normal * 2.0 ** -7, 448.0, 449.0, 452.0)):
        for at in (r, 8000 + 11 * r, 16390 - r):
            x[at, 128:] = v
            x[at, r] = v
    q, s = ctx.quant_fp8(x)
    check_quant(q, s, x, 1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("blocks", [False, True])
def test_quant_special_values(ctx, dtype, blocks):
    """Zeros, values of 448 2^e and just over, ties, the ends of the type's range, subnormals, infinities, NaN."""
    import torch
    t = dt(dtype)
    x = torch.zeros((256, 640), dtype=t, device="cuda")
    x[1, :128] = torch.linspace(-448, 448, 128)
    x[2, :128] = torch.linspace(-449, 449, 128)
    x[2, 5] = 452.0  # over 448 in either type
    x[3, :128] = (torch.arange(128) + 0.5) * 2.0 ** -9  # ties of e4m3's subnormals and small values
    x[3, 0] = 448.0
    x[4, :128] = torch.finfo(t).max
    x[5, :128] = torch.finfo(t).tiny
    x[6, :128] = torch.finfo(t).smallest_normal * 2.0 ** -7  # subnormal
    x[6, 1] = 0.0
    x[7, :256] = 1.0
    x[7, 3], x[7, 130] = math.inf, -math.inf
    x[8, 128:256] = 3.0
    x[8, 131] = math.nan
    x[9, :128] = math.nan
    x[10, :128] = math.inf
    x[130:, 512:] = 2.0 ** -100
    x[200, 513] = -(2.0 ** -90)
    q, s = ctx.quant_fp8(x, blocks=blocks)
    check_quant(q, s, x, 128 if blocks else 1)


def test_quant_leaves_what_is_not_its_own(ctx, awa):
    """Rows and words past the last one, at a wider scale stride."""
    import torch
    x = torch.randn((5, 700), device="cuda")
    q = torch.full((7, 768), 99, dtype=torch.uint8, device="cuda")
    s = torch.full((3, 9), 77, dtype=torch.int32, device="cuda")
    ctx.check(awa.lib().dit_quant_fp8(ctx.ptr, awa.AWA_F32, x.data_ptr(), 700, 5, 700, 1, q.data_ptr(), s.data_ptr(), 9,
                                      torch.cuda.current_stream().cuda_stream), "dit_quant_fp8")
    check_quant(q[:5], s[:2, :5].contiguous().view(torch.uint8).reshape(2, 5, 4), x, 1)
    assert bool((q[5:] == 99).all()) and bool((s[2] == 77).all()) and bool((s[:, 5:] == 77).all())
    assert ctx.quant_fp8(x[:0])[0].shape == (0, 768)


# ------------------------------------------------------------------ the product

def fp8_matrix(awa, ctx, rows, k, blocks, g, spread=0):
    """Rows quantised by the plain form above: (q, scale, values in fp64)."""
    import torch
    x = torch.randn((rows, k), generator=g, device="cuda")
    if spread:
        x = x * torch.exp2(torch.randint(-spread, spread, (rows, k // 128), generator=g, device="cuda")
                           .float()).repeat_interleave(128, 1)
    per = 128 if blocks else 1
    ref, e = plain_quant(x, per)
    b = torch.zeros((e.shape[0], -(-k // 512) * 4), dtype=torch.uint8, device="cuda")
    b[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    s = b.reshape(e.shape[0], -1, 4).transpose(0, 1).contiguous().view(torch.float8_e8m0fnu)
    v = ref * torch.exp2(e.double()).repeat_interleave(per, 0)[:rows].repeat_interleave(128, 1)
    return ref.float().to(torch.float8_e4m3fn), s, v


def gemm_bar(va, vw, ref, dtype, k):
    import torch
    e = (4 * k / 128 + 16) * 2.0 ** -24 * (va.abs() @ vw.abs().T)
    if dtype == torch.bfloat16:
        e = e + 7 * 2.0 ** -13 * (va.abs().unflatten(1, (-1, 8)).amax(2) @ vw.abs().unflatten(1, (-1, 8)).amax(2).T)
    return e + half_step(dtype) * (ref.abs() + e)


SIZES = [(1, 1, 128), (1, 7680, 2560), (2, 130, 640), (15, 257, 384), (16, 16, 512), (17, 2560, 1664), (31, 100, 128),
         (33, 129, 512), (58, 7680, 2560), (64, 256, 6912), (65, 384, 1024), (127, 511, 256), (129, 1000, 640),
         (257, 513, 896), (300, 2560, 512), (679, 2560, 6912), (1000, 1536, 2560), (1237, 1999, 2816),
         (2100, 5120, 384), (4440, 2560, 256), (671, 7601, 640), (700, 3000, 256), (2500, 7681, 256), (6000, 4104, 384),
         (1300, 20001, 128)]
# 256 x 256 tiles, more of them than CUs, of even and odd numbers of blocks over several scale words
LARGE = [(6000, 4104, 256), (4300, 6600, 512), (5890, 4601, 1152), (6100, 4101, 1792), (4000, 4001, 1280)]
# 64 x 64 tiles in groups of waves: more than a workgroup of 32 x 64 per CU
WIDE = [(58, 15360, 640), (120, 9001, 896), (40, 16001, 128), (250, 2600, 1152)]
# up to 16 rows: the widest share of features a workgroup, whole and cut
FEW = [(16, 13824, 640), (9, 13801, 384), (1, 16000, 1152), (5, 4099, 1408)]


@pytest.mark.parametrize("m,n,k", SIZES + LARGE + WIDE + FEW)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gemm(awa, ctx, m, n, k, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, sa, va = fp8_matrix(awa, ctx, m, k, False, g, spread=6)
    w, sw, vw = fp8_matrix(awa, ctx, n, k, True, g, spread=3)
    bias = torch.randn(n, generator=g, device="cuda") * 100
    ref = va @ vw.T
    # rows inside a wider buffer whose other values stay: an odd stride when n is odd
    buf = torch.full((m + 2, n + (n & 1) * 2 + 8), 7.0, dtype=dt(dtype), device="cuda")
    out = buf[1:-1, :n]
    ctx.gemm_fp8(a, sa, w, sw, out=out)
    bar = gemm_bar(va, vw, ref, dt(dtype), k)
    within(out, ref, bar)
    assert bool((buf[0] == 7).all()) and bool((buf[-1] == 7).all()) and bool((buf[:, n:] == 7).all())
    again = ctx.gemm_fp8(a, sa, w, sw, dtype=dt(dtype))
    assert torch.equal(again, out)  # the same sums, whatever the output's strides
    ref = ref + bias.double()
    within(ctx.gemm_fp8(a, sa, w, sw, bias=bias, dtype=dt(dtype)), ref,
           bar + (2.0 ** -24 + half_step(dt(dtype))) * (ref.abs() + bias.abs()))


@pytest.mark.parametrize("m", [17, 32, 300, 1500, 6000])
@pytest.mark.parametrize("times", [1, 16, 256, 2048])
@pytest.mark.parametrize("k", [640, 2560])
def test_gemm_loses_no_more_than_stated(awa, ctx, m, times, k):
    """What the 8-bit sums of bf16 C drop, before C's rounding: rows alike and a bias of minus the exact result (in
    fp32, the difference kept) leave the error itself.  A product loses less than s = 2^(e - 13), e the exponent of its
    group's largest, and nothing if it is a multiple of s.  Bars: for each result the sum of s over the products that
    are none (and what an fp32 sum may lose, as in gemm_bar); over all of them, since the losses have their products'
    signs, which are independent here, the root of the mean sum of s^2 (and K / 8 + 1 random additions of half a step
    of sums no larger than the last, in the root mean square)."""
    import torch
    n = 2048
    g = torch.Generator(device="cuda").manual_seed(m + k + times)
    x = torch.randn((1, k), generator=g, device="cuda")
    x[:, ::8] *= times
    a, w = ctx.quant_fp8(x), ctx.quant_fp8(torch.randn((n, k), generator=g, device="cuda") * 0.02, blocks=True)
    va, vw = awa.fp8_values(*a).double(), awa.fp8_values(*w).double()
    p = (va * vw).abs().unflatten(1, (-1, 8))
    exact = (va * vw).sum(1)
    bias = -exact.float()
    out = ctx.gemm_fp8(a[0].view(torch.uint8).expand(m, -1).contiguous(), a[1].view(torch.uint8).expand(-1, m, -1).contiguous(),
                       *w, bias=bias)
    assert bool((out == out[0]).all())
    e = out[0].double() - (exact + bias.double())
    s = torch.exp2(torch.floor(torch.log2(p.amax(2, keepdim=True))) - 13)
    s = torch.where(torch.remainder(p, s) != 0, s, 0.0)
    most = s.sum((1, 2)) + (4 * k / 128 + 16) * 2.0 ** -24 * p.sum((1, 2)) + 2.0 ** -24 * exact.abs()
    within(e, torch.zeros_like(e), most * (1 + 2.0 ** -8))
    rms = math.sqrt(float((s ** 2).sum((1, 2)).mean())) + math.sqrt(k / 8 + 1) * 2.0 ** -24 * math.sqrt(float((exact ** 2).mean()))
    assert math.sqrt(float((e ** 2).mean())) <= rms * (1 + 2.0 ** -8)


# tiles of 256 rows or features, more of them than CUs, over two to six scale words of odd strides: for fp32 C (1793 x
# 8244 and 2093 x 7582) 256 x 128, 495 and 510 of them, (2305 x 6673) 256 x 192, 351, (3501 x 7000) 256 x 256, 392; for
# bf16 C 256 x 192 and (3501 x 7000) 256 x 256
WALKS = [(1793, 8244, 640), (2305, 6673, 640), (3501, 7000, 1664), (2093, 7582, 2688)]


@pytest.mark.parametrize("m,n,k", WALKS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gemm_walks(awa, ctx, m, n, k, dtype):
    test_gemm(awa, ctx, m, n, k, dtype)


@pytest.mark.parametrize("m", [16, 17, 65, 300, 2000, 20000])
@pytest.mark.parametrize("n", [1, 2, 3, 5, 31, 33])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gemm_few_features(awa, ctx, m, n, dtype):
    test_gemm(awa, ctx, m, n, 384, dtype)


def test_gemm_most_rows(awa, ctx):
    """2^24 rows and, the other way round, 2^20 features: every row a multiple of one of 64, times exact values."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(5)

    def some(rows):
        return torch.randint(-1, 2, (rows, 128), generator=g, device="cuda").float()

    def scales(rows):
        return torch.full((1, rows, 4), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)

    few, w = some(64), some(130)
    m = 1 << 24
    a = few.to(torch.float8_e4m3fn).view(torch.uint8).repeat(m // 64, 1)
    for n in (3, 130):  # sums of at most 128 products of 1: exact in every form and type
        for t in (BF16, F32):
            out = ctx.gemm_fp8(a, scales(m), w[:n].to(torch.float8_e4m3fn), scales(-(-n // 128)), dtype=dt(t))
            want = (few @ w[:n].T).to(dt(t))
            assert bool((out.view(-1, 64, n) == want).all())
            del out
    del a
    n = 1 << 20
    wide = few.to(torch.float8_e4m3fn).view(torch.uint8).repeat(n // 64, 1)
    for rows in (3, 130):
        for t in (BF16, F32):
            out = ctx.gemm_fp8(w[:rows].to(torch.float8_e4m3fn), scales(rows), wide, scales(n // 128), dtype=dt(t))
            want = (w[:rows] @ few.T).to(dt(t))
            assert bool((out.view(rows, -1, 64) == want[:, None]).all())


@pytest.mark.parametrize("m,n", [(5, 300), (20, 300), (300, 520), (700, 2600), (1300, 3301), (2304, 4096)])
def test_gemm_most_columns(awa, ctx, m, n):
    """2^20 columns, 1024 of them repeated: sums of at most 2^20, exact in every form; the quantiser on as many."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m)
    small = [torch.randint(-1, 2, (rows, 1024), generator=g, device="cuda").float() for rows in (m, n)]
    a, w = (t.to(torch.float8_e4m3fn).view(torch.uint8).repeat(1, 1024) for t in small)

    def scales(rows):
        return torch.full((2048, rows, 4), 127, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)

    want = small[0] @ small[1].T * 1024.0
    for t in (BF16, F32):
        out = ctx.gemm_fp8(a, scales(m), w, scales(-(-n // 128)), dtype=dt(t))
        assert torch.equal(out, want.to(dt(t)))
    if m <= 300:  # quantised, a block's largest value 1 becomes 256 and its scale 2^-8
        for blocks in (False, True):
            q, s = ctx.quant_fp8(small[0].bfloat16().repeat(1, 1024), blocks=blocks)
            assert torch.equal(q.float(), 256 * small[0].repeat(1, 1024)) and bool((s.view(torch.uint8) == 119).all())


@pytest.mark.parametrize("m,n", [(40, 600), (250, 2600), (500, 2600), (700, 3300), (671, 8001), (2400, 7000), (3501, 7000)])
@pytest.mark.parametrize("ld", [0, 1, 2, 3])
def test_gemm_scales_at_any_word(awa, ctx, m, n, ld):
    """Scale words that begin 4, 8 and 12 bytes off 16, at strides of any remainder, in every form: rows cut at 1, 2 and
    3 give the bits of their copies."""
    import torch
    k = 1664  # four words a row
    g = torch.Generator(device="cuda").manual_seed(m + ld)
    a, sa, _ = fp8_matrix(awa, ctx, m + 4 + ld, k, False, g, spread=6)
    w, sw, _ = fp8_matrix(awa, ctx, n + 128 * ld, k, True, g, spread=3)
    for r in (1, 2, 3):
        ca, csa = a[r:r + m], sa[:, r:r + m]
        cw, csw = w[128 * (r % (ld + 1)):][:n], sw[:, r % (ld + 1):][:, :-(-n // 128)]
        for t in (BF16, F32):
            want = ctx.gemm_fp8(ca.clone(), csa.contiguous(), cw.clone(), csw.contiguous(), dtype=dt(t))
            assert torch.equal(ctx.gemm_fp8(ca, csa, cw, csw, dtype=dt(t)), want)


@pytest.mark.parametrize("m,n", [(1, 300), (16, 300), (20, 300), (250, 2600), (700, 2560), (700, 7601), (2500, 7681), (6000, 4104)])
@pytest.mark.parametrize("side", ["rows", "weights"])
def test_gemm_least_scale(awa, ctx, m, n, side):
    """Scale byte 0 is 2^-127 like any other: values of 2 to 448 times it, against scales of 2^60."""
    import torch
    k = 768
    g = torch.Generator(device="cuda").manual_seed(m + n)

    def matrix(rows, blocks, byte):
        v = torch.rand((rows, k), generator=g, device="cuda") * 446 + 2
        q = torch.where(torch.rand((rows, k), generator=g, device="cuda") < 0.5, v, -v).to(torch.float8_e4m3fn)
        s = torch.full((2, -(-rows // 128) if blocks else rows, 4), byte, dtype=torch.uint8, device="cuda")
        return q, s.view(torch.float8_e8m0fnu), q.double() * 2.0 ** (byte - 127)

    a, sa, va = matrix(m, False, 0 if side == "rows" else 187)
    w, sw, vw = matrix(n, True, 187 if side == "rows" else 0)
    ref = va @ vw.T
    for t in (BF16, F32):
        within(ctx.gemm_fp8(a, sa, w, sw, dtype=dt(t)), ref, gemm_bar(va, vw, ref, dt(t), k))
    for q, s, v, per in ((a, sa, va, 1), (w, sw, vw, 128)):
        assert torch.equal(awa.fp8_values(q, s).double(), v)


# each form of whole products, some walking over several tiles (the last three), with and without whole chunks
@pytest.mark.parametrize("m,n,k", [(5, 300, 384), (17, 2560, 384), (300, 2560, 512), (120, 9001, 896), (700, 3000, 256),
                                   (671, 7601, 640), (1793, 8244, 640), (2305, 6673, 640), (3467, 6679, 640)])
def test_gemm_whole(awa, ctx, m, n, k):
    """bf16 C with whole products: the bits of the fp32 C, rounded; rows wider than C keep their other values."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, sa, _ = fp8_matrix(awa, ctx, m, k, False, g, spread=6)
    w, sw, _ = fp8_matrix(awa, ctx, n, k, True, g, spread=3)
    for bias in (None, torch.randn(n, generator=g, device="cuda") * 100):
        want = ctx.gemm_fp8(a, sa, w, sw, bias=bias, dtype=torch.float32)
        assert torch.equal(ctx.gemm_fp8(a, sa, w, sw, bias=bias, dtype=torch.float32, whole=True), want)
        assert torch.equal(ctx.gemm_fp8(a, sa, w, sw, bias=bias, whole=True), want.bfloat16())
        buf = torch.full((m + 2, n + 9), 7.0, dtype=torch.bfloat16, device="cuda")
        ctx.gemm_fp8(a, sa, w, sw, bias=bias, out=buf[1:-1, :n], whole=True)
        assert torch.equal(buf[1:-1, :n], want.bfloat16())
        assert bool((buf[0] == 7).all()) and bool((buf[-1] == 7).all()) and bool((buf[:, n:] == 7).all())


@pytest.mark.parametrize("m", [16, 17, 700, 6000])
def test_gemm_whole_cancels(awa, ctx, m):
    """Sums that cancel keep their bits with whole products, whatever the number of rows: the difference to a bias of
    minus the exact result is within what an fp32 sum may lose (gemm_bar's first part and the addition's 2^-24), where
    one column in eight is 2048 times the others."""
    import torch
    k, n = 1280, 1000
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn((1, k), generator=g, device="cuda")
    x[:, ::8] *= 2048
    a, w = ctx.quant_fp8(x), ctx.quant_fp8(torch.randn((n, k), generator=g, device="cuda"), blocks=True)
    va, vw = awa.fp8_values(*a).double(), awa.fp8_values(*w).double()
    exact = (va @ vw.T)[0]
    bias = -exact.float()
    out = ctx.gemm_fp8(a[0].view(torch.uint8).expand(m, -1).contiguous(), a[1].view(torch.uint8).expand(-1, m, -1).contiguous(),
                       *w, bias=bias, whole=True)
    e = exact + bias.double()
    bar = (4 * k / 128 + 16) * 2.0 ** -24 * (va.abs() @ vw.abs().T)[0] + 2.0 ** -24 * exact.abs()
    within(out, e.expand(m, -1), (bar + 2.0 ** -8 * (e.abs() + bar)).expand(m, -1))


def test_gemm_misaligned_output(awa, ctx):
    """An output that begins at an odd element: no 16-byte stores."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    a, sa, va = fp8_matrix(awa, ctx, 300, 512, False, g)
    w, sw, vw = fp8_matrix(awa, ctx, 520, 512, True, g)
    for t in (BF16, F32):
        buf = torch.full((300 * 520 + 2,), 7.0, dtype=dt(t), device="cuda")
        out = buf[1:-1].view(300, 520)
        ctx.gemm_fp8(a, sa, w, sw, out=out)
        ref = va @ vw.T
        within(out, ref, gemm_bar(va, vw, ref, dt(t), 512))
        assert float(buf[0]) == 7 and float(buf[-1]) == 7


@pytest.mark.parametrize("m", [3, 40, 200, 700])
def test_gemm_rows_apart(awa, ctx, m):
    """A row with NaN, a row of zeros and one with scales at the ends of their range stay their own."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m)
    a, sa, va = fp8_matrix(awa, ctx, m, 1024, False, g)
    w, sw, vw = fp8_matrix(awa, ctx, 300, 1024, True, g)
    a[0, 700] = math.nan
    a[1] = 0
    va[0], va[1] = math.nan, 0
    sa.view(torch.uint8)[:, 1] = 0
    sa.view(torch.uint8)[1, 2] = 0  # blocks 4 .. 7 of row 2: 2^-127, nothing beside the others
    va[2, 512:] = a[2, 512:].double() * 2.0 ** -127
    ref = va @ vw.T
    out = ctx.gemm_fp8(a, sa, w, sw, dtype=torch.float32)
    within(out, ref, gemm_bar(va.nan_to_num(nan=0.0), vw, ref.nan_to_num(nan=0.0), torch.float32, 1024))
    assert bool((out[1] == 0).all()) and bool(out[0].isnan().all())


@pytest.mark.parametrize("m,n", [(20, 300), (200, 1000), (700, 2560), (700, 7601), (2500, 7681), (6000, 4104)])
@pytest.mark.parametrize("k", [768, 896])
def test_gemm_rows_apart_in_8_bits(awa, ctx, m, n, k):
    """The same for bf16 C of more rows, in every form of tile, and at each row's place of a tile."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(m + k)
    a, sa, va = fp8_matrix(awa, ctx, m, k, False, g)
    w, sw, vw = fp8_matrix(awa, ctx, n, k, True, g)
    nans, zeros, lows = (slice(i, None, 37) for i in (0, 1, 2))
    a[nans, 300] = math.nan
    a[zeros] = 0
    va[nans], va[zeros] = 0, 0
    sa.view(torch.uint8)[:, zeros] = 0
    sa.view(torch.uint8)[1, lows] = 0  # blocks from the fifth on: 2^-127
    va[lows, 512:] = a[lows, 512:].double() * 2.0 ** -127
    ref = va @ vw.T
    out = ctx.gemm_fp8(a, sa, w, sw)
    assert bool(out[nans].isnan().all()) and bool((out[zeros] == 0).all())
    out[nans] = 0
    within(out, ref, gemm_bar(va, vw, ref, torch.bfloat16, k))


@pytest.mark.parametrize("m", [4, 40, 700])
def test_gemm_ends_of_the_range(awa, ctx, m):
    """Rows that quantise to 2^128: infinite where products enter whole, values like others in 8 bits."""
    import torch
    x = torch.zeros((m, 128), device="cuda")
    x[:, 0] = 3.4e38
    x[1, 0] = -247.0 * 2.0 ** 120  # to 240 2^120
    x[2, 0] = 2.0 ** -120
    wt = torch.zeros((300, 128), device="cuda")
    wt[:, 0] = 2.0 ** -10
    a, w = ctx.quant_fp8(x), ctx.quant_fp8(wt, blocks=True)
    for t in (F32, BF16):
        out = ctx.gemm_fp8(*a, *w, dtype=dt(t)).double()
        whole = t == F32 or m <= 16
        assert bool((out[0] == (math.inf if whole else 2.0 ** 118)).all())
        assert bool((out[1] == -240.0 * 2.0 ** 110).all())
        assert bool((out[2] == 2.0 ** -130).all()) or bool((out[2] == 0).all())
        assert bool((out[3:] == out[0]).all())


def test_gemm_slices(awa, ctx):
    """Rows cut from a larger quantised matrix (the scale stride of the whole), through the C entry."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(2)
    a, sa, va = fp8_matrix(awa, ctx, 100, 640, False, g)
    w, sw, vw = fp8_matrix(awa, ctx, 600, 640, True, g)
    out = torch.empty((31, 300), device="cuda")
    ctx.check(awa.lib().dit_gemm_fp8(ctx.ptr, a[13:].data_ptr(), sa.data_ptr() + 13 * 4, 100, w[256:].data_ptr(),
                                     sw.data_ptr() + 2 * 4, 5, None, awa.AWA_F32, out.data_ptr(), 300, 31, 300, 640,
                                     torch.cuda.current_stream().cuda_stream), "dit_gemm_fp8")
    ref = va[13:44] @ vw[256:556].T
    within(out, ref, gemm_bar(va[13:44], vw[256:556], ref, torch.float32, 640))
    assert torch.equal(ctx.gemm_fp8(a[13:44], sa[:, 13:44], w[256:556], sw[:, 2:], dtype=torch.float32), out)
    one = ctx.gemm_fp8(a[20:21], sa[:, 20:21], w[256:300], sw[:, 2:3])
    within(one, ref[7:8, :44], gemm_bar(va[20:21], vw[256:300], ref[7:8, :44], torch.bfloat16, 640))
    assert ctx.gemm_fp8(a[:0], sa[:, :0], w, sw).shape == (0, 600)
    with pytest.raises(ValueError):
        ctx.gemm_fp8(a[::2], sa[:, ::2], w, sw)


# ------------------------------------------------------------------ rotary positions

def plain_rope(x, pos, freqs, pairs, layout, scale, inverse):
    """(the rotation in fp64, its bar without the type's half step)."""
    import torch
    y, bar = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    p = sum(pairs)
    axis = torch.tensor([i for i, n in enumerate(pairs) for _ in range(n)], dtype=torch.long, device=x.device)
    f = torch.as_tensor(np.asarray(freqs), device=x.device)
    ang = pos.reshape(pos.shape[0], -1)[:, axis].double() * f
    c, s = scale * ang.cos()[:, None], scale * ang.sin()[:, None] * (-1 if inverse else 1)
    i = torch.arange(p, device=x.device)
    first, second = (i, i + p) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., first].double(), x[..., second].double()
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    e = (a.abs() + b.abs()) * abs(scale) * (2.0 ** -21 + ang.abs()[:, None] * 2.0 ** -51)
    bar[..., first], bar[..., second] = e, e
    return y, bar


ROPES = [  # tokens, heads, head_d, pairs per axis, layout, extra elements between tokens
    (1, 40, 128, (21, 21, 21), "interleaved", 0), (1, 1, 2, (1,), "half", 0), (7, 3, 64, (32,), "half", 0),
    (300, 40, 128, (21, 21, 21), "interleaved", 2560), (65, 5, 96, (32,), "half", 3), (65, 5, 96, (32,), "interleaved", 3),
    (129, 1, 256, (64, 64), "half", 256), (33, 2, 77, (11, 7), "half", 0), (33, 2, 77, (11, 7), "interleaved", 0),
    (50, 9, 80, (40,), "interleaved", 16), (50, 9, 80, (20,), "half", 16), (11, 4, 128, (16, 0, 8, 24), "half", 8),
    (3000, 2, 64, (16,), "interleaved", 0), (5, 70, 8, (4,), "half", 0), (9, 2, 32, (0,), "half", 0),
]


@pytest.mark.parametrize("tokens,heads,head_d,pairs,layout,extra", ROPES)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope(awa, ctx, tokens, heads, head_d, pairs, layout, extra, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(tokens * heads + head_d)
    buf = torch.randn((tokens, heads * head_d + extra), generator=g, device="cuda").to(dt(dtype))
    x = buf[:, :heads * head_d].unflatten(1, (heads, head_d))
    pos = torch.randint(-100, 5000, (tokens, len(pairs)), generator=g, device="cuda", dtype=torch.int32)
    freqs = np.concatenate([awa.rope_freqs(n) for n in pairs if n] or [np.zeros(0)])
    args = dict(pairs=pairs, layout=layout)
    for scale, inverse in ((1.0, False), (1.25, True)):
        ref, bar = plain_rope(x, pos, freqs, pairs, layout, scale, inverse)
        out = ctx.rope(x, pos, freqs, scale=scale, inverse=inverse, **args)
        within(out, ref, bar + half_step(dt(dtype)) * ref.abs())
        turned = torch.zeros(head_d, dtype=torch.bool)
        turned[:2 * sum(pairs)] = True
        assert torch.equal(out[..., ~turned], x[..., ~turned])
    # in place, inside the buffer, whose other values stay
    rest = buf[:, heads * head_d:].clone()
    out = ctx.rope(x, pos, freqs, **args)
    assert ctx.rope(x, pos, freqs, out=x, **args) is x
    assert torch.equal(x, out) and torch.equal(buf[:, heads * head_d:], rest)


def rope_heads_a_thread(tokens, heads, head_d, pairs, layout, size, copy):
    """(threads per token and piece, heads of the first of them, heads in flight) by the launcher's rule: 8 workgroups of
    256 per CU, pieces of up to 16 bytes that the pairs and the head are whole numbers of."""
    half, v = layout == "half", 16 // size // (1 if layout == "half" else 2)
    while v > 1 and (pairs % v or head_d % v if half else head_d % (2 * v)):
        v //= 2
    w, turning = v if half else 2 * v, -(-pairs // v)
    passing = max(0, head_d - (2 * pairs if half else w * turning))
    units = turning + (-(-passing // w) if copy else 0)
    lanes = min(heads, -(-2048 * 256 // (tokens * units)))
    return lanes, -(-heads // lanes), 2 if half and v == 8 else 4


# several heads a thread, whole numbers of those in flight and not, with channels that pass and without
ROPES_LONG = [
    (5440, 40, 128, (21, 21, 21), "interleaved", 2560), (5440, 40, 128, (21, 21, 21), "half", 2560),
    (5440, 40, 128, (64,), "half", 2560), (20000, 12, 96, (32,), "half", 0), (20000, 12, 96, (32,), "interleaved", 0),
    (9000, 37, 80, (20,), "half", 3), (9000, 37, 80, (20,), "interleaved", 3), (30000, 8, 80, (40,), "half", 16),
    (30011, 7, 96, (8, 24), "half", 1), (70001, 9, 64, (30,), "interleaved", 0), (300000, 2, 64, (32,), "half", 0),
    (150001, 5, 16, (8,), "interleaved", 8), (100003, 3, 33, (13,), "half", 0),
]


@pytest.mark.parametrize("tokens,heads,head_d,pairs,layout,extra", ROPES_LONG)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_heads_in_turn(awa, ctx, tokens, heads, head_d, pairs, layout, extra, dtype):
    size = 2 if dtype == BF16 else 4
    lanes, most, _ = rope_heads_a_thread(tokens, heads, head_d, sum(pairs), layout, size, True)
    assert lanes < heads and most > 1
    test_rope(awa, ctx, tokens, heads, head_d, pairs, layout, extra, dtype)


def test_rope_heads_in_turn_reach_every_remainder():
    """ROPES_LONG has threads whose heads fit those in flight once, and more than once with and without a remainder."""
    for flight in (2, 4):
        seen = set()
        for tokens, heads, head_d, pairs, layout, _ in ROPES_LONG:
            for size in (2, 4):
                for copy in (False, True):
                    lanes, most, r = rope_heads_a_thread(tokens, heads, head_d, sum(pairs), layout, size, copy)
                    if r == flight:
                        seen |= {(most > r, (-(-(heads - i) // lanes)) % r != 0) for i in range(lanes)}
        assert seen >= {(False, False), (True, False), (True, True)}, (flight, seen)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_heads_of_two_tensors(awa, ctx, layout, dtype):
    """Queries and keys of different numbers of heads, several a thread, in place inside qkv rows."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(9)
    tok, hq, hk, d = 20001, 14, 3, 64
    buf = torch.randn((tok, (hq + 2 * hk) * d), generator=g, device="cuda").to(dt(dtype))
    was = buf.clone()
    q, k = buf[:, :hq * d].unflatten(1, (hq, d)), buf[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    pos = torch.arange(tok, dtype=torch.int32, device="cuda")
    f = awa.rope_freqs(32)
    want = [plain_rope(t, pos, f, (32,), layout, 1.0, False) for t in (q, k)]
    ctx.rope((q, k), pos, f, layout=layout, out=(q, k))
    for t, (ref, bar) in zip((q, k), want):
        within(t, ref, bar + half_step(dt(dtype)) * ref.abs())
    assert torch.equal(buf[:, (hq + hk) * d:], was[:, (hq + hk) * d:])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_far_positions(awa, ctx, layout):
    import torch
    pos = torch.tensor([0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, -12345679], dtype=torch.int32, device="cuda")
    freqs = awa.rope_freqs(32, kind="bands", factor=8.0, trained=4096.0)
    x = torch.randn((7, 3, 64), device="cuda")
    ref, bar = plain_rope(x, pos, freqs, (32,), layout, 1.0, False)
    within(ctx.rope(x, pos, freqs, layout=layout), ref, bar + 2.0 ** -24 * ref.abs())


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("scale", [1.0, 1.3465735902799727])
def test_rope_sines_are_rounded_once(awa, ctx, layout, scale):
    """Pairs (1, 0) turn to scale (cos, sin) alone: half a step, what the series leaves out (under 2^-28) and rounds
    (the terms from x^4 / 24 <= 2^-5.9 on in fp32, at most four half steps of 2^-24 of them: under 2^-27.9), and the
    angle's own error."""
    import torch
    tokens, pairs = 20000, 32
    g = torch.Generator(device="cuda").manual_seed(12)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    pos[:4000] = torch.arange(4000)
    freqs = np.concatenate([awa.rope_freqs(pairs - 2), [2 * np.pi / 4000, -0.5 * np.pi / 4000]])
    x = torch.zeros((tokens, 1, 2 * pairs), device="cuda")
    first = slice(0, pairs) if layout == "half" else slice(0, None, 2)
    second = slice(pairs, None) if layout == "half" else slice(1, None, 2)
    x[..., first] = 1.0
    out = ctx.rope(x, pos, freqs, layout=layout, scale=scale)
    angle = pos.double()[:, None, None] * torch.from_numpy(freqs).cuda()
    for part, ref in ((first, scale * angle.cos()), (second, scale * angle.sin())):
        within(out[..., part], ref, 2.0 ** -24 * ref.abs() + scale * (2.0 ** -28 + 2.0 ** -27.9 + angle.abs() * 2.0 ** -51))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_quarter_turns(awa, ctx, layout):
    """Angles at and around the borders of the reduction: multiples of a sixteenth turn."""
    import torch
    pos = torch.arange(-40, 41, dtype=torch.int32, device="cuda")
    freqs = np.array([2 * np.pi / 16, -2 * np.pi / 16 * (1 + 2.0 ** -40), 0.0, 2 * np.pi])
    x = torch.randn((81, 2, 8), device="cuda")
    ref, bar = plain_rope(x, pos, freqs, (4,), layout, 1.0, False)
    within(ctx.rope(x, pos, freqs, layout=layout), ref, bar + 2.0 ** -24 * ref.abs())


def test_rope_not_finite_stays_in_its_pair(awa, ctx):
    import torch
    for t in (BF16, F32):
        for layout, other in (("interleaved", 5), ("half", 36)):
            x = torch.randn((2, 1, 72), device="cuda").to(dt(t))
            x[0, 0, 4], x[1, 0, 70] = math.nan, math.inf
            out = ctx.rope(x, torch.tensor([3, 4], dtype=torch.int32, device="cuda"), awa.rope_freqs(32), layout=layout)
            bad = ~out.isfinite().cpu()
            want = torch.zeros((2, 72), dtype=torch.bool)
            want[0, 4] = want[0, other] = want[1, 70] = True
            assert torch.equal(bad[:, 0], want)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_passes_every_bit(awa, ctx, layout, dtype):
    """Channels past the pairs, some inside the last piece of the pairs: infinities, NaN with their bits, -0."""
    import torch
    ints = torch.int16 if dtype == BF16 else torch.int32
    for head_d, pairs in ((128, 63), (128, 61), (64, 1), (24, 9), (10, 3)):
        x = torch.randn((5, 3, head_d), device="cuda").to(dt(dtype))
        tail = x[..., 2 * pairs:]
        tail.copy_(torch.tensor([math.inf, 1.0, -0.0, math.nan, -1.0, -math.inf, 0.0, -2.0] * 32,
                                device="cuda")[torch.randint(0, 256, tail.shape, device="cuda")].to(dt(dtype)))
        x.view(ints)[0, 0, 2 * pairs] |= 3  # a NaN of some bits, or a number
        out = ctx.rope(x, torch.arange(5, dtype=torch.int32, device="cuda"), awa.rope_freqs(pairs), layout=layout)
        assert torch.equal(out.view(ints)[..., 2 * pairs:], x.view(ints)[..., 2 * pairs:])
        assert out[..., :2 * pairs].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_queries_and_keys(awa, ctx, dtype):
    """Both tensors of a call, in place inside qkv rows: the same bits as one by one; v stays."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(3)
    tok, hq, hk, d = 37, 12, 3, 64
    buf = torch.randn((tok, (hq + 2 * hk) * d), generator=g, device="cuda").to(dt(dtype))
    was = buf.clone()
    q, k = buf[:, :hq * d].unflatten(1, (hq, d)), buf[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    pos = torch.arange(tok, dtype=torch.int32, device="cuda")
    f = awa.rope_freqs(32)
    wq, wk = ctx.rope(q, pos, f, layout="half"), ctx.rope(k, pos, f, layout="half")
    oq, ok = ctx.rope((q, k), pos, f, layout="half")
    assert torch.equal(oq, wq) and torch.equal(ok, wk)
    ctx.rope((q, k), pos, f, layout="half", out=(q, k))
    assert torch.equal(q, wq) and torch.equal(k, wk) and torch.equal(buf[:, (hq + hk) * d:], was[:, (hq + hk) * d:])
    # heads outside tokens, into such memory
    out = torch.empty((hq, tok, d), dtype=dt(dtype), device="cuda").transpose(0, 1)
    ctx.rope(was[:, :hq * d].unflatten(1, (hq, d)), pos, f, layout="half", out=out)
    assert torch.equal(out, wq)
    with pytest.raises(awa.AwaError):
        ctx.rope((q, q), pos, f, layout="half", out=(q, q))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_gradient(awa, ctx, layout):
    """inverse=True takes gradients back: <g, R x> = <R' g, x>, against differences of the forward pass too."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((6, 2, 20), generator=gen, device="cuda")
    g = torch.randn((6, 2, 20), generator=gen, device="cuda")
    pos = torch.arange(6, dtype=torch.int32, device="cuda") * 7
    f = awa.rope_freqs(8)
    args = dict(layout=layout, scale=1.3)
    grad = ctx.rope(g, pos, f, inverse=True, **args)
    ref, bar = plain_rope(g, pos, f, (8,), layout, 1.3, True)
    within(grad, ref, bar + 2.0 ** -24 * ref.abs())
    # the map is linear, so a difference of any step is the derivative: each of the two passes is off by its
    # bar of at most 4 (|a| + |b| with |x| < 4 and scale 1.3, times 2^-21 and a half step), over 2 h = 2
    for i in (0, 3, 9, 17):
        e = torch.zeros_like(x)
        e[..., i] = 1.0
        up, down = ctx.rope(x + e, pos, f, **args).double(), ctx.rope(x - e, pos, f, **args).double()
        d = ((up - down) / 2 * g.double()).sum(-1)
        assert float((d - grad[..., i].double()).abs().max()) <= 20 * 4 * 13 * 2.0 ** -21


# ------------------------------------------------------------------ far apart

def test_offsets_past_32_bits(awa, ctx):
    """Rows of a buffer of 9 GB (elements past 2^32, bytes past 2^33)."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(6)
    buf = torch.empty(4400 * 2 ** 20, dtype=torch.bfloat16, device="cuda")
    rows = buf.view(4400, 2 ** 20)
    x = torch.randn((4400, 200), generator=g, device="cuda").bfloat16()
    rows[:, 1000:1200] = x
    q, s = ctx.quant_fp8(rows[:, 1000:1200])
    wq, ws = ctx.quant_fp8(x)
    assert torch.equal(q.view(torch.uint8), wq.view(torch.uint8)) and torch.equal(s.view(torch.uint8), ws.view(torch.uint8))
    w = ctx.quant_fp8(torch.randn((300, 200), generator=g, device="cuda"), blocks=True)
    want = ctx.gemm_fp8(q, s, *w)
    assert torch.equal(ctx.gemm_fp8(q, s, *w, out=rows[:, 5:305]), want) and torch.equal(rows[:, 1000:1200], x)
    h = rows[:, 2000:2192].unflatten(1, (3, 64))
    h.copy_(want[:, :192].unflatten(1, (3, 64)))
    pos = torch.arange(4400, dtype=torch.int32, device="cuda")
    for layout in ("half", "interleaved"):
        ref = ctx.rope(h.contiguous(), pos, awa.rope_freqs(32), layout=layout)
        ctx.rope(h, pos, awa.rope_freqs(32), layout=layout, out=h)
        assert torch.equal(h, ref)


def test_most_rows(awa, ctx):
    """2^24 rows: more pieces than one grid of the quantiser holds, and nearly 2^32 threads of the rotation."""
    import torch
    n = 1 << 24
    x = torch.empty((n, 1025), dtype=torch.bfloat16, device="cuda")
    for i in range(0, n, n // 64):  # a part's rows are its first ones, times a power of two of its own
        x[i:i + n // 64].copy_((torch.arange(1025, device="cuda") % 251 - 99).bfloat16() * 2.0 ** (i // (n // 64) - 32))
    q, s = ctx.quant_fp8(x)
    for i in range(0, n, n // 64):
        wq, ws = ctx.quant_fp8(x[i:i + 1])
        assert bool((q[i:i + n // 64].view(torch.int32) == wq.view(torch.int32)).all())
        assert bool((s[:, i:i + n // 64].view(torch.uint8) == ws.view(torch.uint8)).all())
    del x, q, s
    h = torch.ones((n, 1, 256), dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    out = ctx.rope(h, pos, np.array([0.001]), layout="half")
    for i in (0, 12345, n // 2 - 3, n - 10):
        some = ctx.rope(h[i:i + 10].clone(), pos[i:i + 10], np.array([0.001]), layout="half")
        assert torch.equal(out[i:i + 10], some)
    assert bool((out[..., 2:] == 1).all()) and bool((out[..., 0].float() ** 2 + out[..., 1].float() ** 2 - 2).abs().max() < 0.05)


# ------------------------------------------------------------------ together

def layer(ctx, x, w, bias, pos, freqs, stream=None):
    """Rows in 8 bits, the qkv projection, queries and keys rotated in place."""
    q, s = ctx.quant_fp8(x, stream=stream)
    qkv = ctx.gemm_fp8(q, s, *w, bias=bias, stream=stream)
    h = qkv[:, :2 * 512].unflatten(1, (8, 128))
    ctx.rope(h, pos, freqs, pairs=(21, 21, 21), out=h, stream=stream)
    return qkv


def layer_inputs(awa, ctx, m, seed):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, 700), generator=g, device="cuda").bfloat16()
    wt = torch.randn((3 * 512, 700), generator=g, device="cuda") * 0.02
    bias = torch.randn(3 * 512, generator=g, device="cuda")
    pos = torch.randint(0, 99, (m, 3), generator=g, device="cuda", dtype=torch.int32)
    return x, wt, bias, pos, np.tile(awa.rope_freqs(21), 3)


@pytest.mark.parametrize("m", [1, 58, 700])
def test_projection_and_rotation(awa, ctx, m):
    import torch
    x, wt, bias, pos, freqs = layer_inputs(awa, ctx, m, m)
    w = ctx.quant_fp8(wt, blocks=True)
    out = layer(ctx, x, w, bias, pos, freqs)
    va, vw = [q * torch.exp2(e.double()).repeat_interleave(per, 0)[:q.shape[0]].repeat_interleave(128, 1)
              for per, (q, e) in ((1, plain_quant(x, 1)), (128, plain_quant(wt, 128)))]
    assert torch.equal(awa.fp8_values(*ctx.quant_fp8(x), cols=700).double(), va[:, :700])
    assert torch.equal(awa.fp8_values(*w, cols=700).double(), vw[:, :700])
    c = va @ vw.T + bias.double()
    ce = gemm_bar(va, vw, c, torch.bfloat16, 768) + (2.0 ** -24 + 2.0 ** -8) * (c.abs() + bias.abs())
    within(out[:, 1024:], c[:, 1024:], ce[:, 1024:])
    y, bar = plain_rope(c[:, :1024].unflatten(1, (8, 128)), pos, freqs, (21, 21, 21), "interleaved", 1.0, False)
    # a rotated channel is off by both channels' errors before it
    e = ce[:, :1024].unflatten(1, (8, 64, 2)).sum(-1, keepdim=True).expand(-1, -1, -1, 2).flatten(2)
    within(out[:, :1024].unflatten(1, (8, 128)), y, bar + e * 1.01 + 2.0 ** -8 * (y.abs() + e))


def test_captured_and_replayed(awa, ctx):
    """The run as a graph, replayed over changed inputs with eager work between; another context and stream at once."""
    import torch
    x, wt, bias, pos, freqs = layer_inputs(awa, ctx, 130, 9)
    w = ctx.quant_fp8(wt, blocks=True)
    want = layer(ctx, x, w, bias, pos, freqs).clone()
    torch.cuda.synchronize()
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        out = layer(ctx, x, w, bias, pos, freqs)
    x0 = x.clone()
    for k in range(4):
        x.copy_(x0.roll(k, 0) * (k + 1))
        eager = layer(ctx, x, w, bias, pos, freqs)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    x.copy_(x0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    other, side = awa.Context(0), [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [layer(c, x, w, bias, pos, freqs, stream=s) for _ in range(3) for c, s in ((ctx, side[0]), (other, side[1]))]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    other.close()


def test_results_of_another_stream(awa, ctx):
    """A result is not put where the current stream's earlier work, still running, has yet to write."""
    import torch
    x, wt, bias, pos, freqs = layer_inputs(awa, ctx, 700, 3)
    w = ctx.quant_fp8(wt, blocks=True)
    q, s = ctx.quant_fp8(x)
    want = ctx.gemm_fp8(q, s, *w)
    turned = ctx.rope(want.unflatten(1, (12, 128)), pos, freqs, pairs=(21, 21, 21))
    side, big = torch.cuda.Stream(), torch.ones(1 << 28, device="cuda")
    torch.cuda.synchronize()
    for _ in range(8):  # 8 passes over 1 GiB: over a millisecond
        big.mul_(1.0)
    late = [torch.empty_like(t) for t in (q, s, want, turned) for _ in range(4)]
    for t in late:
        t.view(torch.uint8).fill_(85)
    del late, t  # given back before the fills have run
    got = [*ctx.quant_fp8(x, stream=side), ctx.gemm_fp8(q, s, *w, stream=side),
           ctx.rope(want.unflatten(1, (12, 128)), pos, freqs, pairs=(21, 21, 21), stream=side)]
    torch.cuda.synchronize()
    for g, r in zip(got, (q, s, want, turned)):
        assert torch.equal(g.view(torch.uint8), r.view(torch.uint8))


def test_inputs_dropped_before_another_stream_has_read_them(awa, ctx):
    """Inputs given up as the call returns are not overwritten while its stream, still busy, has yet to read them."""
    import torch
    x, wt, bias, pos, freqs = layer_inputs(awa, ctx, 700, 3)
    w = ctx.quant_fp8(wt, blocks=True)
    q, s = ctx.quant_fp8(x)
    qkv = ctx.gemm_fp8(q, s, *w, bias=bias)
    heads, args = qkv.unflatten(1, (12, 128)), dict(pairs=(21, 21, 21))
    want = [q, s, qkv, ctx.rope(heads, pos, freqs, **args)]
    side, big = torch.cuda.Stream(), torch.ones(1 << 28, device="cuda")
    temps = [t.clone() for t in (x, q, s, *w, bias, heads, pos)]
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(8):  # 8 passes over 1 GiB: over a millisecond
            big.mul_(1.0)
    got = [*ctx.quant_fp8(temps[0], stream=side), ctx.gemm_fp8(*temps[1:5], bias=temps[5], stream=side),
           ctx.rope(temps[6], temps[7], freqs, stream=side, **args)]
    shapes = [(t.shape, t.dtype) for t in temps]
    del temps
    late = [torch.empty(*shape, dtype=dtype, device="cuda") for shape, dtype in shapes for _ in range(2)]
    for t in late:
        t.view(torch.uint8).fill_(85)
    torch.cuda.synchronize()
    for g, r in zip(got, want):
        assert torch.equal(g.view(torch.uint8), r.view(torch.uint8))


def test_captured_on_a_given_stream(awa, ctx):
    """The run captured with stream= naming the capture's own stream, temporaries dropped inside it; whole products and
    fp32 rotation too.  Inputs changed between replays, and given back after them."""
    import torch
    x, wt, bias, pos, freqs = layer_inputs(awa, ctx, 130, 21)
    w = ctx.quant_fp8(wt, blocks=True)

    def run(stream=None):
        q, s = ctx.quant_fp8(x, stream=stream)
        c = ctx.gemm_fp8(q, s, *w, dtype=torch.float32, stream=stream)
        turned = ctx.rope(c.unflatten(1, (12, 128)), pos, freqs, pairs=(21, 21, 21), stream=stream)
        return layer(ctx, x, w, bias, pos, freqs, stream), turned, ctx.gemm_fp8(q, s, *w, bias=bias, whole=True, stream=stream)

    run()
    torch.cuda.synchronize()
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=st):
        outs = run(st)
    x0 = x.clone()
    for k in range(4):
        x.copy_(x0.roll(k, 0) * (k + 1))
        eager = run()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))
    del graph, outs
    torch.cuda.synchronize()
