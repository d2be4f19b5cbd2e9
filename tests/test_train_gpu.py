"""GPU tests of the operators of dit_train.h against plain forms in 64 bits.

U = 2^-24 is fp32's half step.  A sum of n terms in fp32, in any order, is off by at most n U times the sum of the
terms' magnitudes.

Layer norm.  A lane adds at most 64 values of a row, a wave and a workgroup 10 more: with n = 80 the mean is off by
n U mean |x - mean| (the second pass corrects the first sum), the variance by (n + 3) U of itself, rstd by half of that
and 2 U; the result's own operations add 6 U: bar U (50 |h w| + 80 |w| + 2 |y|) and half a step of y's type, with
|x - mean| on the mean at most the root mean square, so |h| of 1 on the mean.
Its gradient, from given statistics: h 2 U, a U, the two means n U of their magnitudes' mean; dw and db sum the rows:
at most ceil(M / rows in flight) in a lane, then the 8 waves' 3 and the workgroups' at most 64 + 2.
Weight gradient: products are whole (e4m3 values times a power of two in bf16, dy in bf16 or in three bf16 parts), so
n = M (3 M for fp32) and the splits'.
Attention.  A score (natural units) is off by E = scale d U sum |q| |k| + 4 U |s|; a probability by 2 E of itself
(numerator and sum), n U for the sum over n keys, and half a step of bf16 where it is rounded before it meets v; the
result by the same of sum P |v|, and half a step of its type.  Gradients: with lse rounded to fp32 (U |lse|) and out to its
type (half a step h): dP is off by d U sum |do| |v|, D by (d U + h) sum |do| |out|, dS by P (both) and |dS| (E' + h'),
E' = E + 4 U |lse|, h' half a step of bf16 where dS is rounded; the sums over rows or keys add n U.
"""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BF16, F32, FP8 = "bfloat16", "float32", "fp8"
U = 2.0 ** -24


def dt(name):
    import torch
    return getattr(torch, name)


def half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


def within(out, ref, bar, what=""):
    """out within bar of ref everywhere; NaN where ref is, and only there."""
    import torch
    out = out.double()
    assert out.shape == ref.shape, what
    assert torch.equal(out.isnan(), ref.isnan()), what
    same = out == ref  # infinities
    d = torch.nan_to_num(torch.where(same, -1.0, (out - ref).abs() - bar), nan=-1.0)
    assert float(d.max() if d.numel() else -1) <= 0, f"{what} over the bar by {float(d.max())}"


def gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    import torch
    return torch.randn(shape, generator=g, device="cuda")


# ------------------------------------------------------------------ layer norm

def norm_reference(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    h = (x - mean) * rstd
    y = h * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return y, mean, rstd, h


def check_norm(y, st, x, w, b, eps):
    import torch
    ref, mean, rstd, h = norm_reference(x, w, b, eps)
    wa = torch.ones_like(h) if w is None else w.double().abs().expand_as(h)
    within(y, ref, U * (50 * h.abs() * wa + 80 * wa + 2 * ref.abs()) + half_step(y.dtype) * ref.abs(), "y")
    if st is not None:
        sd = (x.double() - mean).abs().mean(1)
        within(st[:, 0], mean[:, 0], U * (81 * sd + 2 * mean[:, 0].abs()), "mean")
        within(st[:, 1], rstd[:, 0], U * 48 * rstd[:, 0], "rstd")


@pytest.mark.parametrize("tx,ty", [(BF16, BF16), (F32, BF16), (F32, F32), (BF16, F32)])
@pytest.mark.parametrize("rows,cols,ld", [(1, 1, 1), (1, 2, 2), (3, 63, 63), (5, 64, 71), (58, 2560, 2560), (7, 511, 517),
                                          (130, 513, 520), (9, 1025, 1025), (33, 1537, 1540), (17, 2050, 2051),
                                          (12, 2693, 2701), (6, 3100, 3100), (5, 4096, 4099), (3, 4097, 4097),
                                          (4, 8193, 8200), (2, 16384, 16384), (1, 12001, 12001), (5001, 130, 131)])
def test_layer_norm(ctx, tx, ty, rows, cols, ld):
    g = gen(rows + cols)
    x = (randn(g, rows, ld) * 3 + 5 * randn(g, rows, 1)).to(dt(tx))[:, ld - cols:]
    w, b = 1 + 0.1 * randn(g, cols), randn(g, cols)
    for wi, bi in ((w, b), (None, b), (w, None), (None, None)):
        y, st = ctx.layer_norm(x, wi, bi, eps=1e-3, dtype=dt(ty), stats=True)
        assert y.dtype == dt(ty)
        check_norm(y, st, x, wi, bi, 1e-3)


def test_layer_norm_large_mean(ctx):
    """Rows whose mean is 2^12 times their spread: the spread survives."""
    import torch
    g = gen(3)
    x = randn(g, 40, 2560) + 4096.0
    y, st = ctx.layer_norm(x, stats=True)
    ref, mean, rstd, h = norm_reference(x, None, None, 1e-5)
    within(y, ref, U * (50 * h.abs() + 80 + 2 * ref.abs()) + U * ref.abs())
    within(st[:, 1], rstd[:, 0], U * 48 * rstd[:, 0])


def test_layer_norm_constant_rows_and_special_values(ctx):
    import torch
    x = torch.zeros((6, 300), device="cuda")
    x[1] = 7.0
    x[2, 5] = math.inf
    x[3, 299] = math.nan
    x[4] = torch.linspace(-1, 1, 300)
    x[5] = -math.inf
    w, b = torch.full((300,), 2.0, device="cuda"), torch.full((300,), 0.5, device="cuda")
    y, st = ctx.layer_norm(x, w, b, eps=1e-5, stats=True)
    assert bool((y[:2] == 0.5).all()) and bool((st[:2, 0] == torch.tensor([0.0, 7.0], device="cuda")).all())
    for r in (2, 3, 5):
        assert bool(y[r].isnan().all())
    check_norm(y[4:5], st[4:5], x[4:5], w, b, 1e-5)
    y, st = ctx.layer_norm(x[:1], eps=0.0, stats=True)  # 0 / 0
    assert bool(y.isnan().all()) and bool((st[0, 1] == math.inf).all())


@pytest.mark.parametrize("rows,cols", [(70001, 4100), (270003, 40)])
def test_layer_norm_many_rows(ctx, rows, cols):
    """More workgroups than one dimension of the launch takes, not a multiple of the dimensions."""
    g = gen(11)
    x = randn(g, rows, cols).to(dt(BF16))
    y, st = ctx.layer_norm(x, stats=True)
    at = list(range(9)) + list(range(rows // 2 - 9, rows // 2 + 9)) + list(range(65530, 65540)) + list(range(rows - 9, rows))
    check_norm(y[at], st[at], x[at], None, None, 1e-5)
    # every row: no row is left out
    assert float(st[:, 1].min()) > 0.5 and float((y.float().pow(2).mean(1) - 1).abs().max()) < 0.02


def test_layer_norm_in_place_and_rows_around(ctx):
    """y over x; rows and columns beside the result stay as they were."""
    import torch
    g = gen(9)
    for t in (BF16, F32):
        buf = randn(g, 70, 900).to(dt(t))
        keep = buf.clone()
        x = buf[3:60, 7:807]
        want = ctx.layer_norm(x.clone())
        assert ctx.layer_norm(x, out=x) is x
        assert torch.equal(x, want)
        keep[3:60, 7:807] = want
        assert torch.equal(buf, keep)
    assert ctx.layer_norm(torch.zeros((0, 64), device="cuda")).shape == (0, 64)


def norm_grad_reference(dy, x, st, w):
    import torch
    dy, x, st = dy.double(), x.double(), st.double()
    mean, rstd = st[:, :1], st[:, 1:]
    h = (x - mean) * rstd
    a = dy * (1 if w is None else w.double())
    ma, mah = a.mean(1, keepdim=True), (a * h).mean(1, keepdim=True)
    dx = rstd * (a - ma - h * mah)
    bar = rstd * U * (4 * a.abs() + 84 * a.abs().mean(1, keepdim=True) + h.abs() * (90 * (a * h).abs().mean(1, keepdim=True)) +
                      6 * (h * mah).abs())
    n = dy.shape[0] + 80
    return dx, bar, (dy * h).sum(0), n * U * (dy * h).abs().sum(0), dy.sum(0), n * U * dy.abs().sum(0)


def saved(ctx, awa, x):
    """(8-bit rows, scales, their values)."""
    q, s = ctx.quant_fp8(x)
    return q, s, awa.fp8_values(q, s, x.shape[1])


@pytest.mark.parametrize("tdy,tx,tdx", [(BF16, BF16, BF16), (BF16, F32, F32), (F32, F32, BF16), (F32, BF16, F32), (BF16, FP8, BF16),
                                        (F32, FP8, F32)])
@pytest.mark.parametrize("rows,cols,ld", [(1, 1, 1), (2, 2, 2), (3, 63, 63), (58, 2560, 2560), (5, 64, 71), (7, 511, 517),
                                          (130, 513, 520), (9, 1025, 1025), (33, 1537, 1540), (17, 2050, 2051), (12, 2693, 2701),
                                          (31, 3100, 3100), (5, 4096, 4099), (3, 4097, 4097), (4, 6200, 6200), (5, 8192, 8192),
                                          (4, 8193, 8200), (3, 12289, 12289), (2, 16384, 16384), (5001, 130, 131), (2600, 700, 700)])
def test_layer_norm_grad(ctx, awa, tdy, tx, tdx, rows, cols, ld):
    g = gen(rows * 7 + cols)
    x = (randn(g, rows, ld) * 2 + randn(g, rows, 1))
    dy = randn(g, rows, ld).to(dt(tdy))[:, ld - cols:]
    w = 1 + 0.1 * randn(g, cols)
    if tx == FP8:
        xin, xs, x = saved(ctx, awa, x[:, :cols].contiguous())
    else:
        x = x.to(dt(tx))[:, ld - cols:]
        xin, xs = x, None
    _, st = ctx.layer_norm(x.contiguous(), eps=1e-5, stats=True)
    for wi in (w, None):
        dx, dw, db = ctx.layer_norm_grad(dy, xin, st, wi, x_scale=xs, dtype=dt(tdx))
        rx, bx, rw, bw, rb, bb = norm_grad_reference(dy, x, st, wi)
        within(dx, rx, bx + half_step(dx.dtype) * rx.abs(), "dx")
        within(dw, rw, bw, "dw")
        within(db, rb, bb, "db")
        alone, none_w, none_b = ctx.layer_norm_grad(dy, xin, st, wi, x_scale=xs, dtype=dt(tdx), params=False)
        assert none_w is None and none_b is None
        assert alone.equal(dx)


def test_layer_norm_grad_differences(ctx):
    """Against differences of the forward pass in 64 bits: f(x) = sum dy y(x), central differences with step e are off by
    e^2 / 6 times the third derivative; with e = 1e-4 and values of about 1 that is far below 1e-6."""
    import torch
    g = gen(4)
    x, dy, w, b = randn(g, 3, 40), randn(g, 3, 40), 1 + 0.3 * randn(g, 40), randn(g, 40)
    _, st = ctx.layer_norm(x, w, b, stats=True)
    dx, dw, db = ctx.layer_norm_grad(dy, x, st, w)

    def f(x, w, b):
        return (dy.double() * norm_reference(x, w, b, 1e-5)[0]).sum()

    for t, grad, args in ((x, dx, lambda v: (v, w, b)), (w, dw, lambda v: (x, v, b)), (b, db, lambda v: (x, w, v))):
        for i in range(0, t.numel(), 7):
            e = torch.zeros(t.numel(), dtype=torch.float64, device="cuda")
            e[i] = 1e-4
            d = (f(*args(t.double() + e.view_as(t))) - f(*args(t.double() - e.view_as(t)))) / 2e-4
            assert abs(float(d) - float(grad.view(-1)[i])) < 1e-5


def test_layer_norm_grad_in_place_and_no_rows(ctx):
    import torch
    g = gen(5)
    x, dy = randn(g, 37, 600), randn(g, 37, 600)
    _, st = ctx.layer_norm(x, stats=True)
    want = ctx.layer_norm_grad(dy, x, st)
    over = dy.clone()
    got = ctx.layer_norm_grad(over, x, st, dx=over)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    over = x.clone()
    got = ctx.layer_norm_grad(dy, over, st, dx=over)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    dx, dw, db = ctx.layer_norm_grad(dy[:0], x[:0], st[:0])
    assert dx.shape == (0, 600) and not bool(dw.any()) and not bool(db.any())


# ------------------------------------------------------------------ a weight's gradient

def check_weight(dw, db, dy, x, before=None, db_before=None):
    import torch
    dyd, xd = dy.double(), x.double()
    n = dy.shape[0] * (3 if dy.dtype == torch.float32 else 1) + 20
    ref, size = dyd.t() @ xd, dyd.abs().t() @ xd.abs()
    if before is not None:
        ref, size = ref + before.double(), size + before.double().abs()
    within(dw, ref, n * U * size + half_step(dw.dtype) * ref.abs(), "dw")
    if db is not None:
        r, s = dyd.sum(0), dyd.abs().sum(0)
        if db_before is not None:
            r, s = r + db_before.double(), s + db_before.double().abs()
        within(db, r, n * U * s, "db")


@pytest.mark.parametrize("tdy,tw", [(BF16, F32), (BF16, BF16), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("M,N,K,ld", [(1, 1, 1, 1), (2, 3, 5, 3), (31, 64, 128, 64), (32, 65, 129, 70), (33, 127, 100, 127),
                                      (58, 300, 640, 300), (257, 128, 128, 128), (700, 130, 513, 131), (1237, 199, 269, 199),
                                      (2100, 256, 384, 512), (5498, 96, 160, 96), (64, 1000, 2693, 1001),
                                      (600, 4100, 2090, 4103), (1000, 4353, 4090, 4353), (70, 4, 300, 4), (77, 9, 300, 9)])
def test_grad_weight(ctx, awa, tdy, tw, M, N, K, ld):
    import torch
    g = gen(M + N + K)
    dy = randn(g, M, ld).to(dt(tdy))[:, ld - N:]
    x = randn(g, M, K) * torch.exp2(torch.randint(-6, 6, (M, 1), generator=g, device="cuda").float())
    q, s, v = saved(ctx, awa, x)
    dw, db = ctx.grad_weight_fp8(dy, q, s, cols=K, bias=True, dtype=dt(tw))
    check_weight(dw, db, dy, v)
    again, db2 = ctx.grad_weight_fp8(dy, q, s, cols=K, bias=True, dtype=dt(tw))
    assert torch.equal(dw, again) and torch.equal(db, db2)
    assert torch.equal(ctx.grad_weight_fp8(dy, q, s, cols=K, dtype=dt(tw)), dw)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (33, 7, 40), (64, 9, 130), (95, 130, 127), (700, 300, 513), (1300, 515, 700)])
@pytest.mark.parametrize("tdy", [BF16, F32])
def test_what_lies_around(ctx, awa, tdy, M, N, K):
    """NaN beside and behind dy, x and its scales, and in the workspace's memory: nothing of it counts, and what lies beside and
    behind the results stays.  (Columns of 8-bit rows past K reach columns past K only.)"""
    import torch
    g = gen(M + N)
    nan = float("nan")

    def middle(rows, cols, dtype, fill):
        whole = torch.full((rows + 3, cols + 12), fill, device="cuda", dtype=dtype)
        return whole, whole[1:rows + 1, 5:cols + 5]

    def stays(whole, part, fill):
        part.fill_(fill)
        assert bool((whole.isnan() if fill != fill else whole == fill).all())

    x = randn(g, M, K)
    q, s, v = saved(ctx, awa, x)
    q_all = torch.full((M + 5, q.shape[1]), 0x7f, device="cuda", dtype=torch.uint8)
    q_all[:M] = q.view(torch.uint8)
    if q.shape[1] > K:
        q_all[:, K:] = 0x7f
    s_all = torch.full((s.shape[0], M + 5, 4), 0xff, device="cuda", dtype=torch.uint8)
    s_all[:, :M] = s.view(torch.uint8)
    q2, s2 = q_all[:M].view(q.dtype), s_all.view(s.dtype)[:, :M]
    dy = middle(M, N, dt(tdy), nan)[1]
    dy.copy_(randn(g, M, N))
    dw_all, dw = middle(N, K, dt(F32), 7.0)
    junk = torch.full((1 << 23,), nan, device="cuda")
    del junk
    _, db = ctx.grad_weight_fp8(dy, q2, s2, cols=K, bias=True, out=dw)
    check_weight(dw, db, dy, v)
    stays(dw_all, dw, 7.0)

    rows = middle(M, K, dt(tdy), nan)[1]
    rows.copy_(randn(g, M, K))
    y_all, y = middle(M, K, dt(tdy), 7.0)
    w = 1 + 0.1 * randn(g, K)
    _, st = ctx.layer_norm(rows, w, out=y, stats=True)
    check_norm(y, st, rows, w, None, 1e-5)
    want = ctx.layer_norm_grad(rows.contiguous(), v.to(dt(F32)), st, w, dtype=dt(tdy))
    stays(y_all, y, 7.0)
    junk = torch.full((1 << 23,), nan, device="cuda")
    del junk
    dx_all, dx = middle(M, K, dt(tdy), 7.0)
    for a, b in zip(ctx.layer_norm_grad(rows, q2, st, w, x_scale=s2, dx=dx), want):
        assert torch.equal(a, b)
    stays(dx_all, dx, 7.0)


@pytest.mark.parametrize("M", [0, 1, 600])
@pytest.mark.parametrize("tdy", [BF16, F32])
def test_grad_weight_added(ctx, awa, tdy, M):
    """add=True into rows of a wider tensor, whose other columns stay."""
    import torch
    g = gen(M)
    N, K = 77, 301
    q, s, v = saved(ctx, awa, randn(g, M, K))
    dy = randn(g, M, N).to(dt(tdy))
    buf, db = randn(g, N, 400), randn(g, N)
    keep, out, before_b = buf.clone(), buf[:, 50:50 + K], db.clone()
    before = out.clone()
    ctx.grad_weight_fp8(dy, q, s, cols=K, out=out, bias=db, add=True)
    check_weight(out, db, dy, v, before, before_b)
    keep[:, 50:50 + K] = out
    assert torch.equal(buf, keep)
    dw, db = ctx.grad_weight_fp8(dy, q, s, cols=K, bias=True)
    check_weight(dw, db, dy, v)


def test_grad_weight_special_values(ctx, awa):
    """Infinities and NaN reach their rows and columns only; fp32 magnitudes past bf16's bits; scales at their ends."""
    import torch
    g = gen(8)
    x = randn(g, 70, 200)
    x[3] *= 2.0 ** 60
    x[4] *= 2.0 ** -60
    q, s, v = saved(ctx, awa, x)
    dy = randn(g, 70, 40)
    dy[7, 3], dy[9, 5] = math.inf, math.nan
    dw = ctx.grad_weight_fp8(dy, q, s, cols=200)
    ref = dy.double().t() @ v.double()
    clean = [i for i in range(40) if i not in (3, 5)]
    size = dy.double().abs().t() @ v.double().abs()
    within(dw[clean], ref[clean], 230 * U * size[clean])
    assert bool(dw[5].isnan().all())
    assert torch.equal(dw[3].double(), ref[3])  # infinite by x's sign (NaN for a zero)
    q2 = q.clone().view(torch.uint8)
    q2[11, 17] = 0x7f  # NaN
    dw = ctx.grad_weight_fp8(dy[:, clean].contiguous(), q2, s, cols=200)
    assert bool(dw[:, 17].isnan().all()) and not bool(dw[:, :17].isnan().any()) and not bool(dw[:, 18:].isnan().any())


# ------------------------------------------------------------------ attention to states of another length

def batch(g, ql, kl, heads, kv_heads, d, dtype, q_at=None, k_at=None, q_rows=None, k_rows=None):
    q_at = [sum(ql[:i]) for i in range(len(ql))] if q_at is None else q_at
    k_at = [sum(kl[:i]) for i in range(len(kl))] if k_at is None else k_at
    nq = max([a + n for a, n in zip(q_at, ql)], default=0) if q_rows is None else q_rows
    nk = max([a + n for a, n in zip(k_at, kl)], default=0) if k_rows is None else k_rows
    t = dt(dtype)
    return (q_at, k_at, randn(g, nq, heads, d).to(t), randn(g, nk, kv_heads, d).to(t), randn(g, nk, kv_heads, d).to(t),
            randn(g, nq, heads, d).to(t))


def reference(q_at, ql, k_at, kl, q, k, v, mask, scale, do=None):
    """Results and bars in 64 bits: a dict of name -> (reference, bar), sequence by sequence and head by head."""
    import torch
    bf16 = q.dtype == torch.bfloat16
    hs = half_step(q.dtype)
    hp = hs if bf16 else 0.0  # probabilities and dS rounded
    d, per = q.shape[2], q.shape[1] // k.shape[1]
    zq = lambda: torch.zeros(q.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    zk = lambda: torch.zeros(k.shape, dtype=torch.float64, device="cuda")  # noqa: E731
    out, bo, dq, bq = zq(), zq(), zq(), zq()
    dk, bk, dv, bv = zk(), zk(), zk(), zk()
    lse = torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    bl = torch.zeros_like(lse)
    for a, n, ka, m in zip(q_at, ql, k_at, kl):
        rows, keys = slice(a, a + n), torch.arange(ka, ka + m, device="cuda")
        if mask is not None:
            keys = keys[mask[keys].bool()]
        if n == 0 or keys.numel() == 0:
            continue
        for h in range(q.shape[1]):
            Q, K, V = q[rows, h].double(), k[keys, h // per].double(), v[keys, h // per].double()
            S = scale * (Q @ K.T)
            E = scale * d * U * (Q.abs() @ K.abs().T) + 4 * U * S.abs()
            Em = E.amax(1, keepdim=True)
            l = torch.logsumexp(S, 1, keepdim=True)
            P = (S - l).exp()
            o = P @ V
            nk = keys.numel() + 16
            out[rows, h], lse[h, rows] = o, l[:, 0]
            bo[rows, h] = (P * (2 * Em + nk * U + hp)) @ V.abs() + hs * o.abs()
            bl[h, rows] = (Em + nk * U + 4 * U * (1 + l.abs()))[:, 0]
            if do is None:
                continue
            G = do[rows, h].double()
            El = E + Em + 4 * U * l.abs() + nk * U  # a probability's, lse as the forward pass left it
            dP, D = G @ V.T, (G * o).sum(1, keepdim=True)
            dS = P * (dP - D)
            # out as the forward pass left it
            eD = (G.abs() * bo[rows, h]).sum(1, keepdim=True) + d * U * (G.abs() * o.abs()).sum(1, keepdim=True)
            eS = P * (d * U * (G.abs() @ V.abs().T) + eD) * (1 + El + hp) + dS.abs() * (El + hp + 2 * U)
            nq = n * per + 40
            dq[rows, h] = scale * (dS @ K)
            bq[rows, h] = scale * (eS @ K.abs() + nk * U * (dS.abs() @ K.abs())) + (hs + 2 * U) * dq[rows, h].abs()
            dv[keys, h // per] += P.T @ G
            bv[keys, h // per] += (P * (El + hp + nq * U)).T @ G.abs()
            dk[keys, h // per] += scale * (dS.T @ Q)
            bk[keys, h // per] += scale * (eS.T @ Q.abs() + nq * U * (dS.abs().T @ Q.abs()))
    bk, bv = bk + (hs + 2 * U) * dk.abs(), bv + (hs + 2 * U) * dv.abs()
    return {"out": (out, bo), "lse": (lse, bl), "dq": (dq, bq), "dk": (dk, bk), "dv": (dv, bv)}


def check_cross(ctx, g, ql, kl, heads, kv_heads, d, dtype, mask=None, scale=None, grad=True, **places):
    import torch
    q_at, k_at, q, k, v, do = batch(g, ql, kl, heads, kv_heads, d, dtype, **places)
    scale = d ** -0.5 if scale is None else scale
    mask = torch.rand(k.shape[0], generator=g, device="cuda") < 0.8 if mask is True else mask
    plan = ctx.cross_plan(heads, d, ql, kl, kv_heads=kv_heads, q_at=q_at, k_at=k_at)
    out, lse = ctx.cross_attn(plan, q, k, v, mask=mask, scale=scale, lse=True)
    ref = reference(q_at, ql, k_at, kl, q, k, v, mask, scale, do if grad else None)
    rows = [r for a, n in zip(q_at, ql) for r in range(a, a + n)]
    within(out, *ref["out"], "out")
    within(lse[:, rows], ref["lse"][0][:, rows], ref["lse"][1][:, rows], "lse")
    assert torch.equal(ctx.cross_attn(plan, q, k, v, mask=mask, scale=scale), out)
    if grad:
        got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, mask=mask, scale=scale)
        for name, t in zip(("dq", "dk", "dv"), got):
            within(t, *ref[name], name)
        again = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, mask=mask, scale=scale)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    return plan


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,d", [(2, 2, 128), (4, 2, 64), (3, 1, 80), (5, 5, 96), (6, 2, 8), (1, 1, 40)])
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (1, 31), (3, 65), (15, 64), (17, 33), (33, 100), (64, 16), (65, 63), (127, 129),
                                   (128, 128), (129, 65), (200, 300), (2, 1000)])
def test_cross_one_sequence(ctx, dtype, heads, kv_heads, d, nq, nk):
    check_cross(ctx, gen(nq * 31 + nk + d), [nq], [nk], heads, kv_heads, d, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("ql,kl", [([1, 1, 1, 1], [7, 300, 64, 129]), ([5, 0, 130, 1], [40, 12, 0, 90]), ([0, 0], [5, 70]),
                                   ([70, 3], [0, 0]), ([300, 200, 100], [58, 77, 20]), ([2, 3, 1], [2100, 30, 700]), ([], [])])
@pytest.mark.parametrize("masked", [False, True])
def test_cross_batches(ctx, dtype, ql, kl, masked):
    """Ragged batches; sequences without queries, without keys, without either."""
    check_cross(ctx, gen(len(ql) + sum(kl)), ql, kl, 6, 2, 64, dtype, mask=True if masked and sum(kl) else None)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_larger(ctx, dtype):
    """Enough blocks that each way of dividing the work is met, a long axis on either side."""
    check_cross(ctx, gen(1), [1500], [700], 4, 4, 128, dtype, mask=True)
    check_cross(ctx, gen(2), [3000], [58], 2, 1, 128, dtype)
    check_cross(ctx, gen(3), [900, 400, 650], [65, 64, 30], 20, 10, 64, dtype, mask=True)
    check_cross(ctx, gen(4), [1] * 20, [257] * 20, 8, 2, 128, dtype)
    check_cross(ctx, gen(5), [20], [5000], 1, 1, 128, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_shared_keys(ctx, dtype):
    """Several sequences, one text: its gradient is the sum over them.  Places in no order, gaps between them."""
    check_cross(ctx, gen(6), [40, 130, 1, 70], [50, 50, 90, 50], 4, 2, 64, dtype, mask=True, q_at=[300, 20, 9, 200],
                k_at=[100, 100, 0, 100], q_rows=400, k_rows=170)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq", [1, 20, 150])
def test_cross_masks_that_leave_nothing(ctx, dtype, nq):
    """Whole sequences and whole tiles masked; NaN and infinities in masked rows and in rows of no sequence."""
    import torch
    g = gen(nq)
    ql, kl = [nq, nq, nq], [200, 150, 64]
    q_at, k_at, q, k, v, do = batch(g, ql, kl, 4, 2, 64, dtype, k_at=[10, 220, 400], k_rows=480)
    mask = torch.ones(480, dtype=torch.bool, device="cuda")
    mask[10:80] = False       # the first tile, and a piece of the second
    mask[220:370] = False     # a sequence's only keys
    mask[463] = False
    for t in (k, v):
        t[~mask] = math.nan
        t[20] = math.inf
        t[:10] = math.nan
        t[210:220] = math.inf
        t[464:] = math.nan
    plan = ctx.cross_plan(4, 64, ql, kl, kv_heads=2, q_at=q_at, k_at=k_at)
    out, lse = ctx.cross_attn(plan, q, k, v, mask=mask, lse=True)
    ref = reference(q_at, ql, k_at, kl, q, k, v, mask, 0.125, do)
    within(out, *ref["out"], "out")
    within(lse, *ref["lse"], "lse")
    assert bool((lse[:, nq:2 * nq] == -math.inf).all()) and not bool(out[nq:2 * nq].any())
    do[nq:2 * nq] = math.nan  # no key takes part: no gradient, whatever comes back
    got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, mask=mask)
    for name, t in zip(("dq", "dk", "dv"), got):
        within(t, *ref[name], name)
    assert not bool(got[1][~mask].any()) and not bool(got[2][~mask].any()) and not bool(got[0][nq:2 * nq].any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_rows_of_no_sequence_stay(ctx, dtype):
    """Given results keep what they hold in rows of no sequence, made ones hold zeros there; strided tensors."""
    import torch
    g = gen(12)
    ql, kl, q_at, k_at = [20, 33], [70, 10], [5, 40], [3, 90]
    t = dt(dtype)
    rows = randn(g, 100, 3 * 4 * 64).to(t)  # q and its gradient inside wider rows
    q = rows[:, :256].unflatten(1, (4, 64))
    kv = randn(g, 120, 2, 2, 64).to(t)
    k, v = kv[:, 0], kv[:, 1]
    do = randn(g, 4, 100, 64).to(t).transpose(0, 1)  # heads outermost
    plan = ctx.cross_plan(4, 64, ql, kl, kv_heads=2, q_at=q_at, k_at=k_at)
    ref = reference(q_at, ql, k_at, kl, q, k, v, None, 0.125, do)
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    within(out, *ref["out"])
    inside = torch.zeros(100, dtype=torch.bool, device="cuda")
    inside[5:25] = inside[40:73] = True
    kin = torch.zeros(120, dtype=torch.bool, device="cuda")
    kin[3:73] = kin[90:100] = True
    given = torch.full((100, 4, 64), 7.0, dtype=t, device="cuda")
    glse = torch.full((4, 100), 7.0, device="cuda")
    ctx.cross_attn(plan, q, k, v, out=given, lse=glse)
    assert torch.equal(given[inside], out[inside]) and bool((given[~inside] == 7).all())
    assert torch.equal(glse[:, inside], lse[:, inside]) and bool((glse[:, ~inside] == 7).all())
    dq, dk, dv = ctx.cross_attn_grad(plan, do, q, k, v, out, lse)
    for name, x in (("dq", dq), ("dk", dk), ("dv", dv)):
        within(x, *ref[name], name)
    buf = torch.full((120, 2, 2, 64), 7.0, dtype=t, device="cuda")  # dk and dv beside each other
    dq2 = torch.full((100, 12, 64), 7.0, dtype=t, device="cuda")
    ctx.cross_attn_grad(plan, do, q, k, v, out, lse, dq=dq2[:, 4:8], dk=buf[:, 0], dv=buf[:, 1])
    assert torch.equal(dq2[inside][:, 4:8], dq[inside]) and bool((dq2[~inside] == 7).all())
    assert bool((dq2[:, :4] == 7).all()) and bool((dq2[:, 8:] == 7).all())
    assert torch.equal(buf[kin][:, 0], dk[kin]) and torch.equal(buf[kin][:, 1], dv[kin]) and bool((buf[~kin] == 7).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_far_scores(ctx, dtype):
    """Scores of hundreds either way: the softmax neither overflows nor loses the largest."""
    import torch
    g = gen(13)
    q, k, v = 30 * randn(g, 70, 2, 64), 30 * randn(g, 300, 2, 64), randn(g, 300, 2, 64)
    t = dt(dtype)
    q, k, v = q.to(t), k.to(t), v.to(t)
    plan = ctx.cross_plan(2, 64, [70], [300])
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    ref = reference([0], [70], [0], [300], q, k, v, None, 0.125)
    within(out, *ref["out"])
    within(lse, *ref["lse"])


def test_cross_differences(ctx):
    """Gradients against central differences in 64 bits (step 1e-4, third derivatives of about 1: below 1e-6 off)."""
    import torch
    g = gen(14)
    q, k, v, do = randn(g, 5, 2, 8), randn(g, 9, 1, 8), randn(g, 9, 1, 8), randn(g, 5, 2, 8)
    plan = ctx.cross_plan(2, 8, [5], [9], kv_heads=1)
    out, lse = ctx.cross_attn(plan, q, k, v, scale=0.4, lse=True)
    grads = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, scale=0.4)

    def f(q, k, v):
        return (reference([0], [5], [0], [9], q, k, v, None, 0.4)["out"][0] * do.double()).sum()

    for which, t in enumerate((q, k, v)):
        for i in range(0, t.numel(), 5):
            e = torch.zeros(t.numel(), dtype=torch.float64, device="cuda")
            e[i] = 1e-4
            args = [x.double() for x in (q, k, v)]
            hi, lo = list(args), list(args)
            hi[which], lo[which] = args[which] + e.view_as(t), args[which] - e.view_as(t)
            d = float(f(*hi) - f(*lo)) / 2e-4
            assert abs(d - float(grads[which].reshape(-1)[i])) < 1e-5


# ------------------------------------------------------------------ together

def test_a_layer_forward_and_back(ctx, awa):
    """The operators as a layer uses them: norm, 8-bit rows, product, attention to a text, and all the way back,
    against the same chain in 64 bits through autograd (8-bit rows taken as they are: the gradient passes them)."""
    import torch
    g = gen(21)
    M, Kt, Cn, H, D = 300, 40, 256, 2, 64
    x, w, b = randn(g, M, Cn), 1 + 0.1 * randn(g, Cn), 0.1 * randn(g, Cn)
    wq = 0.05 * randn(g, H * D, Cn)
    k, v = randn(g, Kt, H, D), randn(g, Kt, H, D)
    y, st = ctx.layer_norm(x, w, b, stats=True)
    yq, ys = ctx.quant_fp8(y)
    wqq, wqs = ctx.quant_fp8(wq, blocks=True)
    q = ctx.gemm_fp8(yq, ys, wqq, wqs, dtype=torch.float32).unflatten(1, (H, D))
    plan = ctx.cross_plan(H, D, [200, 100], [25, 15])
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    do = randn(g, M, H, D)
    dq, dk, dv = ctx.cross_attn_grad(plan, do, q, k, v, out, lse)
    dwq, dbq = ctx.grad_weight_fp8(dq.flatten(1), yq, ys, bias=True)
    wv = awa.fp8_values(wqq, wqs, Cn)
    dy = dq.flatten(1) @ wv
    dx, dw, db = ctx.layer_norm_grad(dy, x, st, w)

    leaves = [t.double().requires_grad_() for t in (x, w, b, k, v, wv)]
    x6, w6, b6, k6, v6, wq6 = leaves
    y6 = torch.nn.functional.layer_norm(x6, (Cn,), w6, b6, 1e-5)
    y6 = y6 + (awa.fp8_values(yq, ys, Cn).double() - y6).detach()
    q6 = (y6 @ wq6.T).unflatten(1, (H, D))
    o6 = []
    for r, kr in ((slice(0, 200), slice(0, 25)), (slice(200, 300), slice(25, 40))):
        p = torch.softmax(torch.stack([q6[r, h] @ k6[kr, h].T for h in range(H)]) * D ** -0.5, 2)
        o6.append(torch.stack([p[h] @ v6[kr, h] for h in range(H)], 1))
    (torch.cat(o6) * do.double()).sum().backward()
    # each step is off by a few hundred U of magnitudes within a hundred times its result's root mean square
    for got, leaf in ((dx, x6), (dw, w6), (db, b6), (dk, k6), (dv, v6), (dwq, wq6)):
        d = float((got.double() - leaf.grad).norm() / leaf.grad.norm())
        assert d < 1000 * U, d


def test_streams_and_graphs(ctx):
    """Each call on another stream, and captured into one graph that is replayed with new inputs, against eager results."""
    import torch
    g = gen(22)
    ql, kl = [130, 40], [70, 300]
    plan = ctx.cross_plan(4, 64, ql, kl, kv_heads=2)

    def inputs():
        bf = torch.bfloat16
        return [randn(g, 170, 256).to(bf), randn(g, 370, 2, 64).to(bf), randn(g, 370, 2, 64).to(bf), randn(g, 170, 4, 64).to(bf),
                torch.rand(370, generator=g, device="cuda") < 0.9]

    def program(x, k, v, do, mask, stream=None):
        kw = {} if stream is None else {"stream": stream}
        y, st = ctx.layer_norm(x, stats=True, **kw)
        yq, ys = ctx.quant_fp8(y, **kw)
        out, lse = ctx.cross_attn(plan, y.unflatten(1, (4, 64)), k, v, mask=mask, lse=True, **kw)
        dq, dk, dv = ctx.cross_attn_grad(plan, do, y.unflatten(1, (4, 64)), k, v, out, lse, mask=mask, **kw)
        dw, db = ctx.grad_weight_fp8(dq.flatten(1), yq, ys, bias=True, **kw)
        dx, dg, dbeta = ctx.layer_norm_grad(dq.flatten(1), yq, st, x_scale=ys, **kw)
        return [y, st, out, lse, dq, dk, dv, dw, db, dx, dg, dbeta]

    one = inputs()
    want = program(*one)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = program(*one, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    static = [t.clone() for t in one]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        program(*static)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        res = program(*static)
    for _ in range(4):
        new = inputs()
        want = program(*new)
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_two_calls_at_once(ctx):
    """The same plan on two streams at a time, each call with a workspace of its own."""
    import torch
    g = gen(23)
    plan = ctx.cross_plan(4, 64, [1] * 6, [900] * 6, kv_heads=2)
    sets = [[randn(g, 6, 4, 64), randn(g, 5400, 2, 64), randn(g, 5400, 2, 64), randn(g, 6, 4, 64)] for _ in range(2)]
    want = []
    for q, k, v, do in sets:
        out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
        want.append([out, lse, *ctx.cross_attn_grad(plan, do, q, k, v, out, lse)])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for (q, k, v, do), s in zip(sets, streams):
            out, lse = ctx.cross_attn(plan, q, k, v, lse=True, stream=s)
            got.append([out, lse, *ctx.cross_attn_grad(plan, do, q, k, v, out, lse, stream=s)])
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_graphs_of_one_plan(ctx):
    """Two captured graphs of one plan, replayed in turn and at once on two streams: each has a workspace of its own."""
    import torch
    g = gen(24)
    plan = ctx.cross_plan(4, 64, [1] * 5, [1200] * 5, kv_heads=2)

    def inputs():
        return [randn(g, 5, 4, 64), randn(g, 6000, 2, 64), randn(g, 6000, 2, 64), randn(g, 5, 4, 64)]

    def program(q, k, v, do):
        out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
        return [out, lse, *ctx.cross_attn_grad(plan, do, q, k, v, out, lse)]

    sets, graphs, results = [inputs(), inputs()], [], []
    program(*sets[0])
    torch.cuda.synchronize()
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(program(*s))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for s in sets:
            for t, n in zip(s, inputs()):
                t.copy_(n)
        want = [program(*s) for s in sets]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(results, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------ places past 32 bits, other devices

def far_rows(rows, cols, ld, dtype, g):
    """[rows, cols] random values in rows ld elements apart: only they are written."""
    import torch
    t = torch.empty((rows, ld), dtype=dtype, device="cuda")[:, ld - cols:]
    t.copy_(randn(g, rows, cols))
    return t


def test_norm_places_past_32_bits(ctx):
    import torch
    g = gen(31)
    x = far_rows(34000, 70, 1 << 16, torch.bfloat16, g)  # 4.5 GB, 2.2 G elements
    y, st = ctx.layer_norm(x, stats=True)
    check_norm(y, st, x, None, None, 1e-5)
    out = torch.empty((34000, 1 << 16), dtype=torch.bfloat16, device="cuda")[:, :70]
    dx, dw, db = ctx.layer_norm_grad(y, x, st, dx=out)
    rx, bx, rw, bw, rb, bb = norm_grad_reference(y, x, st, None)
    within(dx, rx, bx + half_step(dx.dtype) * rx.abs(), "dx")
    within(dw, rw, bw, "dw")


def test_weight_places_past_32_bits(ctx, awa):
    import torch
    g = gen(32)
    dy = far_rows(2500, 90, 1 << 20, torch.bfloat16, g)  # 5.2 GB
    q, s, v = saved(ctx, awa, randn(g, 2500, 200))
    out = torch.empty((90, 1 << 26), dtype=torch.bfloat16, device="cuda")[:, :200]  # 12 GB
    dw, db = ctx.grad_weight_fp8(dy, q, s, cols=200, out=out, bias=True)
    check_weight(dw, db, dy, v)


@pytest.mark.parametrize("nq", [1, 140])
def test_cross_places_past_32_bits(ctx, nq):
    """A long cache of wide rows, and heads far apart: the last sequences lie past 2^32 bytes."""
    import torch
    g = gen(33)
    ql, kl, k_at = [nq, nq], [300, 130], [2100, 2400]
    cache = torch.empty((2600, 1 << 20), dtype=torch.bfloat16, device="cuda")  # 5.4 GB
    kv = cache[:, (1 << 20) - 256:].unflatten(1, (2, 2, 64))
    kv[2000:].copy_(randn(g, 600, 2, 2, 64))
    k, v = kv[:, 0], kv[:, 1]
    wide = torch.empty((4, 1 << 30), dtype=torch.bfloat16, device="cuda")  # 8.6 GB: a head's rows 2 GB from the next's
    q = wide[:, :2 * nq * 64].unflatten(1, (2 * nq, 64)).transpose(0, 1)
    q.copy_(randn(g, 2 * nq, 4, 64))
    do = randn(g, 2 * nq, 4, 64).to(torch.bfloat16)
    plan = ctx.cross_plan(4, 64, ql, kl, kv_heads=2, k_at=k_at)
    ref = reference([0, nq], ql, k_at, kl, q, k, v, None, 0.125, do)
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    within(out, *ref["out"], "out")
    grads = torch.empty((2600, 1 << 20), dtype=torch.bfloat16, device="cuda")[:, :256].unflatten(1, (2, 2, 64))
    dq, dk, dv = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, dk=grads[:, 0], dv=grads[:, 1])
    within(dq, *ref["dq"], "dq")
    for name, t in (("dk", dk), ("dv", dv)):
        within(t[2100:2530], ref[name][0][2100:2530], ref[name][1][2100:2530], name)


def test_host_tensors_are_refused(ctx, awa):
    import torch
    x, st = torch.randn(5, 128, device="cuda"), torch.zeros(5, 2, device="cuda")
    w = torch.ones(128)
    q8, s8 = ctx.quant_fp8(x)
    plan = ctx.cross_plan(2, 64, [5], [7])
    q, k = torch.randn(5, 2, 64, device="cuda"), torch.randn(7, 2, 64, device="cuda")
    out, lse = ctx.cross_attn(plan, q, k, k, lse=True)
    mask = torch.ones(7, dtype=torch.bool)
    for call in (lambda: ctx.layer_norm(x.cpu()), lambda: ctx.layer_norm(x, w), lambda: ctx.layer_norm(x, out=x.cpu()),
                 lambda: ctx.layer_norm(x, stats=st.cpu()), lambda: ctx.layer_norm_grad(x.cpu(), x, st),
                 lambda: ctx.layer_norm_grad(x, x.cpu(), st), lambda: ctx.layer_norm_grad(x, x, st.cpu()),
                 lambda: ctx.layer_norm_grad(x, x, st, w), lambda: ctx.layer_norm_grad(x, q8.cpu(), st, x_scale=s8),
                 lambda: ctx.layer_norm_grad(x, q8, st, x_scale=s8.cpu()), lambda: ctx.layer_norm_grad(x, x, st, dx=x.cpu()),
                 lambda: ctx.grad_weight_fp8(x.cpu(), q8, s8), lambda: ctx.grad_weight_fp8(x, q8.cpu(), s8),
                 lambda: ctx.grad_weight_fp8(x, q8, s8.cpu()), lambda: ctx.grad_weight_fp8(x, q8, s8, out=torch.zeros(128, 128)),
                 lambda: ctx.grad_weight_fp8(x, q8, s8, bias=torch.zeros(128)), lambda: ctx.cross_attn(plan, q.cpu(), k, k),
                 lambda: ctx.cross_attn(plan, q, k.cpu(), k), lambda: ctx.cross_attn(plan, q, k, k.cpu()),
                 lambda: ctx.cross_attn(plan, q, k, k, mask=mask), lambda: ctx.cross_attn(plan, q, k, k, out=q.cpu()),
                 lambda: ctx.cross_attn_grad(plan, q, q, k, k, out.cpu(), lse), lambda: ctx.cross_attn_grad(plan, q, q, k, k, out, lse.cpu()),
                 lambda: ctx.cross_attn_grad(plan, q, q, k, k, out, lse, dk=k.cpu())):
        with pytest.raises(ValueError, match="device"):
            call()


def test_refusals_with_their_messages(ctx, awa):
    """What the library itself refuses reaches the caller as AwaError with its message."""
    import torch
    x = torch.randn(6, 128, device="cuda")
    y, st = ctx.layer_norm(x, stats=True)
    q8, s8 = ctx.quant_fp8(x)
    plan = ctx.cross_plan(2, 64, [5], [7])
    buf = torch.randn(40, 2, 64, device="cuda")
    q, k = buf[:5], buf[20:27]
    out, lse = ctx.cross_attn(plan, q, k, k, lse=True)
    big = torch.randn(2000, device="cuda")
    for call, text in ((lambda: ctx.layer_norm(x, eps=-1.0), "eps"), (lambda: ctx.layer_norm(x[:5], out=x[1:]), "lie over"),
                       (lambda: ctx.layer_norm_grad(y[:5], x[:5], st[:5], dx=x[1:]), "lie over"),
                       (lambda: ctx.grad_weight_fp8(x, q8, s8, out=x[:1].expand(128, 128)), "ldw"),
                       (lambda: ctx.cross_attn(plan, q, k, k, scale=0.0), "scale"),
                       (lambda: ctx.cross_attn(plan, q, k, k, scale=math.nan), "scale"),
                       (lambda: ctx.cross_attn(plan, q, k, k, out=q), "lie over"),
                       (lambda: ctx.cross_attn(plan, big[1:1 + 640].view(5, 2, 64), k, k), "16-byte"),
                       (lambda: ctx.cross_attn(plan, q, k, k, out=buf[:1].expand(5, 2, 64)), "coincide"),
                       (lambda: ctx.cross_attn_grad(plan, q, q, k, k, out, lse, dk=k), "lie over"),
                       (lambda: ctx.cross_plan(2, 60, [5], [7]), "head_d"), (lambda: ctx.cross_plan(3, 64, [5], [7], kv_heads=2), "kv_heads"),
                       (lambda: ctx.cross_plan(2, 64, [5, 5], [7, 7], q_at=[0, 4]), "overlap"),
                       (lambda: ctx.cross_plan(2, 64, [5, 5], [7, 7], k_at=[0, 3]), "overlap"),
                       (lambda: ctx.cross_plan(2, 64, [-1], [7]), "rows")):
        with pytest.raises(awa.AwaError, match=text):
            call()
