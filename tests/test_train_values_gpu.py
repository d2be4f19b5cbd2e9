"""GPU tests of dit_train.h's operators: values, special values and sizes beside those of test_train_gpu.py, against 64 bits.

U = 2^-24 is fp32's half step.  Attention's bars are those of test_train_gpu.py's text, with `hp` for what P and dS lose
before they meet the tensors: 2^-8 (bf16), or with whole=True 2^-16 (the rest after a bf16 value, at most 2^-8 of it, is rounded to
bf16 too), 0 for fp32.
"""
import math

import pytest

from test_train_gpu import BF16, F32, U, dt, gen, half_step, randn, within

pytestmark = pytest.mark.gpu


def attention(q, k, v, scale, do=None, hp=0.0, mask=None):
    """One sequence in 64 bits: name -> (reference, bar).  q, do [n, heads, d], k, v [m, kv_heads, d], mask [m]."""
    import torch
    hs, d, per = half_step(q.dtype), q.shape[2], q.shape[1] // k.shape[1]
    Q = q.double().transpose(0, 1).contiguous()
    K, V = (t.double().transpose(0, 1).repeat_interleave(per, 0).contiguous() for t in (k, v))
    Kt, Vt = K.transpose(1, 2).contiguous(), V.transpose(1, 2).contiguous()
    S = scale * (Q @ Kt)
    E = scale * d * U * (Q.abs() @ Kt.abs()) + 4 * U * S.abs()
    if mask is not None:
        S = S.masked_fill(~mask, -math.inf)
        E = E.masked_fill(~mask, 0.0)
    Em = E.amax(2, keepdim=True)
    l = torch.logsumexp(S, 2, keepdim=True)
    P = (S - l).exp()
    n, m = Q.shape[1] * per + 40, K.shape[1] + 16
    o = P @ V
    bo = (P * (2 * Em + m * U + hp)) @ V.abs() + hs * o.abs()
    back = lambda t: t.transpose(0, 1)  # noqa: E731
    shared = lambda t: t.unflatten(0, (-1, per)).sum(1).transpose(0, 1)  # noqa: E731
    res = {"out": (back(o), back(bo)), "lse": (l[:, :, 0], (Em + m * U + 4 * U * (1 + l.abs()))[:, :, 0])}
    if do is None:
        return res
    G = do.double().transpose(0, 1).contiguous()
    El = E + Em + 4 * U * l.abs() + m * U
    dP, D = G @ Vt, (G * o).sum(2, keepdim=True)
    dS = P * (dP - D)
    eD = (G.abs() * bo).sum(2, keepdim=True) + d * U * (G.abs() * o.abs()).sum(2, keepdim=True)
    eS = P * (d * U * (G.abs() @ Vt.abs()) + eD) * (1 + El + hp) + dS.abs() * (El + hp + 2 * U)
    dq = scale * (dS @ K)
    bq = scale * (eS @ K.abs() + m * U * (dS.abs() @ K.abs())) + (hs + 2 * U) * dq.abs()
    turn = lambda t: t.transpose(1, 2).contiguous()  # noqa: E731
    dv, dk = shared(turn(P) @ G), shared(scale * (turn(dS) @ Q))
    bv = shared(turn(P * (El + hp + n * U)) @ G.abs()) + (hs + 2 * U) * dv.abs()
    bk = shared(scale * (turn(eS) @ Q.abs() + n * U * (turn(dS).abs() @ Q.abs()))) + (hs + 2 * U) * dk.abs()
    res.update(dq=(back(dq), back(bq)), dk=(dk, bk), dv=(dv, bv))
    return res


# ------------------------------------------------------------------ probabilities of 16 bits

@pytest.mark.parametrize("heads,kv_heads,d", [(3, 3, 8), (4, 2, 64), (2, 1, 96), (2, 2, 128)])
@pytest.mark.parametrize("nq,nk", [(1, 50), (3, 40), (9, 300), (1, 2100), (140, 33), (150, 64), (130, 200), (600, 130)])
def test_whole(ctx, heads, kv_heads, d, nq, nk):
    """Every form of the kernels with whole=True: few columns, one tile, many, keys and queries divided over workgroups."""
    import torch
    g = gen(nq + 7 * nk + d)
    bf = torch.bfloat16
    q, k, v, do = (randn(g, n, h, d).to(bf) for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads), (nq, heads)))
    mask = torch.rand(nk, generator=g, device="cuda") < 0.9
    mask[0] = True
    plan = ctx.cross_plan(heads, d, [nq], [nk], kv_heads=kv_heads)
    for m in (None, mask):
        out, lse = ctx.cross_attn(plan, q, k, v, mask=m, lse=True, whole=True)
        ref = attention(q, k, v, d ** -0.5, do, 2.0 ** -16, m)
        within(out, *ref["out"], "out")
        within(lse, *ref["lse"], "lse")
        got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, mask=m, whole=True)
        for name, t in zip(("dq", "dk", "dv"), got):
            within(t, *ref[name], name)
        assert torch.equal(ctx.cross_attn(plan, q, k, v, mask=m, lse=True)[1], lse)  # scores and sums are the same ones


def test_whole_fp32(ctx):
    """fp32 tensors round nothing on the way: the flag changes no bit."""
    import torch
    g = gen(2)
    q, k, v, do = randn(g, 70, 4, 64), randn(g, 90, 2, 64), randn(g, 90, 2, 64), randn(g, 70, 4, 64)
    plan = ctx.cross_plan(4, 64, [70], [90], kv_heads=2)
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    assert torch.equal(ctx.cross_attn(plan, q, k, v, whole=True), out)
    want = ctx.cross_attn_grad(plan, do, q, k, v, out, lse)
    got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, whole=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------ NaN and infinities that take part

# few columns (undivided and divided keys), one tile, several tiles (undivided and divided)
FORMS = [(1, 40), (3, 3000), (40, 50), (70, 200), (140, 2000)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nk", FORMS)
@pytest.mark.parametrize("where", ["query", "key", "only key"])
def test_nan_among_scores(ctx, dtype, nq, nk, where):
    """A row with a NaN among its scores is NaN, its lse too (it is no row without keys), and so is what follows from it; all else
    is as it would be."""
    import torch
    g = gen(nq + nk)
    q, k, v, do = (randn(g, n, h, 64).to(dt(dtype)) for n, h in ((nq, 4), (nk, 2), (nk, 2), (nq, 4)))
    mask = torch.ones(nk, dtype=torch.bool, device="cuda")
    if where == "query":
        q[nq // 2, 1, 5] = math.nan
    else:
        k[nk - 3, 1, 60] = math.nan
        if where == "only key":
            mask[:] = False
            mask[nk - 3] = True
    plan = ctx.cross_plan(4, 64, [nq], [nk], kv_heads=2)
    out, lse = ctx.cross_attn(plan, q, k, v, mask=mask, lse=True)
    ref = attention(q, k, v, 0.125, do, half_step(q.dtype) if dtype == BF16 else 0.0, mask)
    if where == "query":
        assert bool(ref["lse"][0][1, nq // 2].isnan()) and int(ref["lse"][0].isnan().sum()) == 1
    else:
        assert bool(ref["lse"][0][2:].isnan().all()) and not bool(ref["lse"][0][:2].isnan().any())
    within(out, *ref["out"], "out")
    within(lse, *ref["lse"], "lse")
    got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, mask=mask)
    for name, t in zip(("dq", "dk", "dv"), got):
        if name != "dq":  # keys that take no part get zeros
            ref[name][0][~mask] = 0.0
        within(t, *ref[name], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nk", FORMS)
def test_scores_past_fp32(ctx, dtype, nq, nk):
    """Finite products that the scale takes past fp32 make their row NaN (not one without keys); the other rows stay as they are."""
    import torch
    g = gen(nq + nk)
    q, k, v = (randn(g, n, h, 64) for n, h in ((nq, 2), (nk, 2), (nk, 2)))
    q *= 1e-30  # scores of ordinary sizes
    q[nq - 1, 1], k[:, 1] = 1e5, 1e5 * (1 + 0.01 * randn(g, nk, 64))
    q[: nq - 1, 1] *= 1e-5
    q, k, v = (t.to(dt(dtype)) for t in (q, k, v))
    plan = ctx.cross_plan(2, 64, [nq], [nk])
    out, lse = ctx.cross_attn(plan, q, k, v, scale=1e29, lse=True)
    ref = attention(q, k, v, 1e29, hp=half_step(q.dtype) if dtype == BF16 else 0.0)
    for name in ("out", "lse"):
        for t in ref[name]:
            (t[nq - 1, 1] if name == "out" else t[1, nq - 1:]).fill_(math.nan)
    within(out, *ref["out"], "out")
    within(lse, *ref["lse"], "lse")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq,nk", FORMS + [(64, 300), (97, 64)])
@pytest.mark.parametrize("where", ["query", "key", "finite"])
def test_rows_whose_scores_are_all_minus_infinity(ctx, dtype, nq, nk, where):
    """Zeros, lse -infinity and no gradient, although what made the scores infinite (a query's channel, every key's, finite values
    whose products pass fp32), the values, and what comes back to such rows, are infinite or NaN."""
    import torch
    g = gen(nq + nk)
    heads, kv_heads = (4, 2) if where == "query" else (2, 2)
    q, k, v, do = (randn(g, n, h, 64).to(dt(dtype)) for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads), (nq, heads)))
    none = torch.zeros(nq, heads, dtype=torch.bool, device="cuda")
    if where == "query":
        none[nq // 2, 1] = none[nq - 1, 3] = True
        k[:, :, 5] = k[:, :, 5].abs() + 0.5
    elif where == "key":  # every row of the second head
        none[:, 1] = True
    else:
        none[nq // 2] = True
    clean = [t.clone() for t in (q, k, v, do)]
    if where == "query":
        q[..., 5] = torch.where(none, -math.inf, q[..., 5])
    elif where == "key":
        q[:, 1, 5] = 1.0
        k[:, 1, 5] = -math.inf
        v[::7, 1, 9] = math.inf
    else:
        k[..., 5], clean[1][..., 5] = 3e38, 3e38
        q[..., 5] = torch.where(none, -3e38, 0.0)
        clean[0][..., 5] = 0.0
    do[none] = math.nan
    clean[0][none], clean[3][none] = 0.0, 0.0
    ref = attention(*clean[:3], 0.125, clean[3], half_step(q.dtype) if dtype == BF16 else 0.0)
    for name in ("out", "dq"):
        for t in ref[name]:
            t[none] = 0.0
    for t, value in zip(ref["lse"], (-math.inf, 0.0)):
        t[none.T] = value
    plan = ctx.cross_plan(heads, 64, [nq], [nk], kv_heads=kv_heads)
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    within(out, *ref["out"], "out")
    within(lse, *ref["lse"], "lse")
    for name, t in zip(("dq", "dk", "dv"), ctx.cross_attn_grad(plan, do, q, k, v, out, lse)):
        if name == "dq" and where == "finite":
            # the fifth channel is a sum of terms dS 3e38 with |dS| up to about 1 (P at most 1, dout v of eight on the mean): its
            # partial sums may pass fp32's 3.4e38 whatever the total is, so that it says nothing
            t[..., 5] = torch.where(none, t[..., 5].double(), ref[name][0][..., 5])
        within(t, *ref[name], name)


# ------------------------------------------------------------------ batches of more blocks than are listed by workgroup

LISTED = 65536  # blocks (by heads) of a side up to which a plan lists them for each workgroup


def uniform(g, n, nq, nk, heads, kv_heads, d, dtype):
    """n sequences of nq queries and nk keys: (q, k, v, do) as rows, and the same for `attention` with the sequences as heads."""
    rows = [randn(g, n * m, h, d).to(dt(dtype)) for m, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads), (nq, heads))]
    return rows, [t.unflatten(0, (n, -1)).transpose(0, 1).flatten(1, 2) for t in rows]


def as_rows(t, n, heads):
    """`attention`'s [m, n * heads, d] in the rows' order."""
    return t.unflatten(1, (n, heads)).transpose(0, 1).flatten(0, 1)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,nq,nk,heads,kv_heads", [(9001, 1, 5, 8, 8), (4111, 3, 66, 16, 8), (2061, 40, 70, 32, 16)])
def test_many_blocks(ctx, dtype, n, nq, nk, heads, kv_heads):
    """Few columns and blocks of 128, several blocks of queries' and keys' sides past the list's length."""
    import torch
    g = gen(n)
    d, per = 8, heads // kv_heads
    (q, k, v, do), wide = uniform(g, n, nq, nk, heads, kv_heads, d, dtype)
    groups = heads if nq * per > 32 else kv_heads
    if nq * per > 32 or per == 1:
        assert n * groups > LISTED
    assert n * kv_heads * ((nk + 63) // 64) > LISTED
    mask = torch.rand(n * nk, generator=g, device="cuda") < 0.8
    plan = ctx.cross_plan(heads, d, [nq] * n, [nk] * n, kv_heads=kv_heads)
    some = mask.unflatten(0, (n, nk)).any(1)
    ref = attention(*wide[:3], 0.5, wide[3], half_step(q.dtype) if dtype == BF16 else 0.0,
                    mask.unflatten(0, (n, 1, nk)).repeat_interleave(heads, 0))
    for name in ("out", "dq", "dk", "dv"):  # sequences without keys
        ref[name] = [torch.where(some.repeat_interleave(t.shape[0] // n)[:, None, None], t, 0.0)
                     for t in (as_rows(t, n, heads if name in ("out", "dq") else kv_heads) for t in ref[name])]
    out, lse = ctx.cross_attn(plan, q, k, v, mask=mask, scale=0.5, lse=True)
    within(out, *ref["out"], "out")
    l, bl = (t.unflatten(0, (n, heads)).transpose(0, 1).flatten(1) for t in ref["lse"])
    keep = some.repeat_interleave(nq)
    within(lse[:, keep], l[:, keep], bl[:, keep], "lse")
    assert bool((lse[:, ~keep] == -math.inf).all())
    got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, mask=mask, scale=0.5)
    for name, t in zip(("dq", "dk", "dv"), got):
        if name != "dq":
            ref[name] = [torch.where(mask[:, None, None], r, 0.0) for r in ref[name]]
        within(t, *ref[name], name)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("long_q,long_k", [(1, 5000), (3000, 130), (700, 2000)])
def test_many_blocks_and_divided_ones(ctx, dtype, long_q, long_k):
    """Past the list's length with a sequence whose keys, queries, or both, go to several workgroups and are joined."""
    import torch
    g = gen(long_q)
    n, nk, heads, d = 8500, 4, 8, 16
    assert n * heads > LISTED
    (q, k, v, do), wide = uniform(g, n, 1, nk, heads, heads, d, dtype)
    one = [randn(g, m, heads, d).to(dt(dtype)) for m in (long_q, long_k, long_k, long_q)]
    # the long sequence between the short ones
    at = n // 3
    q, k, v, do = (torch.cat((t[: at * m], o, t[at * m:])) for t, o, m in zip((q, k, v, do), one, (1, nk, nk, 1)))
    plan = ctx.cross_plan(heads, d, [1] * at + [long_q] + [1] * (n - at), [nk] * at + [long_k] + [nk] * (n - at))
    code = 1 if dtype == BF16 else 0
    kept = 2 * ((4 * heads * (n + long_q) + 255) // 256 * 256)  # what the gradients' workspace holds beside parts
    assert plan.work(code, 0) > 0 or long_k < 1000
    assert plan.work(code, 1) - kept > plan.work(code, 0) or long_q == 1
    hp = half_step(q.dtype) if dtype == BF16 else 0.0
    ref, long = attention(*wide[:3], 0.25, wide[3], hp), attention(*one[:3], 0.25, one[3], hp)
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse)
    for name, t in zip(("out", "dq", "dk", "dv"), (out, *got)):
        m, b = (1, long_q) if name in ("out", "dq") else (nk, long_k)
        within(t[at * m:at * m + b], *long[name], name + " of the long one")
        short = torch.cat((t[: at * m], t[at * m + b:]))
        within(short, *(as_rows(r, n, heads) for r in ref[name]), name)
    within(lse[:, at:at + long_q], *long["lse"], "lse of the long one")
    within(torch.cat((lse[:, :at], lse[:, at + long_q:]), 1), *(r.unflatten(0, (n, heads)).transpose(0, 1).flatten(1) for r in ref["lse"]), "lse")


# ------------------------------------------------------------------ tensors side by side

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("nq", [1, 90])
def test_gradients_side_by_side_with_heads_outermost(ctx, dtype, nq):
    """dk and dv in turn for each head of one buffer, dq behind both (and for one query, whose stride does not matter, beside
    keys' rows)."""
    import torch
    g = gen(nq)
    nk = 70
    q, k, v, do = (randn(g, n, 2, 64).to(dt(dtype)) for n in (nq, nk, nk, nq))
    plan = ctx.cross_plan(2, 64, [nq], [nk])
    out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
    want = ctx.cross_attn_grad(plan, do, q, k, v, out, lse)
    buf = torch.full((2, 2 * nk + nq, 64), 7.0, dtype=dt(dtype), device="cuda")
    parts = [t.transpose(0, 1) for t in (buf[:, 2 * nk:], buf[:, :nk], buf[:, nk:2 * nk])]
    got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, dq=parts[0], dk=parts[1], dv=parts[2])
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not bool((buf == 7).all(2).any())
    if nq == 1:
        buf = torch.full((nk, 3, 2, 64), 7.0, dtype=dt(dtype), device="cuda")
        got = ctx.cross_attn_grad(plan, do, q, k, v, out, lse, dq=buf[5:6, 2], dk=buf[:, 0], dv=buf[:, 1])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert bool((buf[:5, 2] == 7).all()) and bool((buf[6:, 2] == 7).all())


# ------------------------------------------------------------------ plans that end before what used them

def test_plans_dropped_before_their_graph(ctx):
    """A captured plan's tables outlive it; a plan that is collected during a capture does not end it."""
    import gc
    import torch
    g = gen(5)
    ql, kl = [3, 70, 1], [500, 90, 2000]
    q, k, v, do = (randn(g, n, h, 64) for n, h in ((74, 4), (2590, 2), (2590, 2), (74, 4)))

    def program(plan):
        out, lse = ctx.cross_attn(plan, q, k, v, lse=True)
        return [out, lse, *ctx.cross_attn_grad(plan, do, q, k, v, out, lse)]

    plan, spare = ctx.cross_plan(4, 64, ql, kl, kv_heads=2), [ctx.cross_plan(4, 64, ql, kl, kv_heads=2)]
    want = program(spare[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        spare.clear()
        gc.collect()
        res = program(plan)
    del plan
    gc.collect()
    # plans of other lengths, in whatever memory has become free
    others = [ctx.cross_plan(4, 64, [1 + i, 70, 1], [500, 90 + i, 2000], kv_heads=2) for i in range(30)]
    for _ in range(4):
        for t in res:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, want))
        others.append(ctx.cross_plan(4, 64, ql, kl, kv_heads=2))
        assert all(torch.equal(a, b) for a, b in zip(program(others[-1]), want))


# ------------------------------------------------------------------ sums that are exact

def whole_numbers(g, top, *shape):
    import torch
    return torch.randint(-top, top + 1, shape, generator=g, device="cuda").float()


# one wave a row to eight, rows of fewer than four columns, one row at a time; few rows and many
@pytest.mark.parametrize("rows,cols", [(1, 3), (5001, 3), (2049, 130), (30001, 520), (4097, 1025), (9999, 1537), (2600, 2050), (12371, 2693),
                                       (1025, 4096), (777, 4097), (3001, 8191), (515, 12289), (511, 16384)])
@pytest.mark.parametrize("tdy,tx", [(BF16, BF16), (F32, F32), (BF16, "fp8"), (F32, "fp8")])
def test_norm_columns_exact(ctx, rows, cols, tdy, tx):
    """dw and db of whole numbers: |dy| up to 4, h up to 8 in halves, so that every sum is a number of halves under 2^24 and
    exact in any order; a row or column that is lost, or taken twice, shows."""
    import torch
    g = gen(rows + cols)
    dy = whole_numbers(g, 4, rows, cols + 1).to(dt(tdy))[:, 1:]
    x = whole_numbers(g, 12, rows, cols)
    st = torch.stack((whole_numbers(g, 4, rows), torch.full((rows,), 0.5, device="cuda")), 1).contiguous()
    assert rows * 4 * 8 * 2 < 2 ** 24
    h = (x.double() - st[:, :1].double()) * 0.5
    if tx == "fp8":  # whole numbers up to 16 have at most the four bits of e4m3
        xin, xs = ctx.quant_fp8(x)
    else:
        xin, xs = x.to(dt(tx)), None
    w = whole_numbers(g, 3, cols)
    _, dw, db = ctx.layer_norm_grad(dy, xin, st, w, x_scale=xs)
    assert torch.equal(dw.double(), (dy.double() * h).sum(0))
    assert torch.equal(db.double(), dy.double().sum(0))


@pytest.mark.parametrize("rows,cols", [(5001, 130), (30001, 64), (12371, 2693), (2600, 8000), (3000, 16384)])
def test_norm_columns_by_their_chain(ctx, rows, cols):
    """dw and db of random data within the sums' length: the rows that a lane adds, 3 halves of a workgroup's waves, at most 66
    parts; a term's own error is 4 U (h 2, its product, a spare one)."""
    g = gen(rows)
    x, dy = randn(g, rows, cols) + randn(g, rows, 1), randn(g, rows, cols)
    _, st = ctx.layer_norm(x, stats=True)
    _, dw, db = ctx.layer_norm_grad(dy, x, st)
    pieces = (cols + 255) // 256
    at_once = 8 if pieces <= 4 else 4 if pieces <= 8 else 2 if pieces <= 16 else 1
    n = -(-rows // (min(-(-rows // at_once), 256) * at_once)) + 3 + 66 + 4
    h = (x.double() - st[:, :1].double()) * st[:, 1:].double()
    within(dw, (dy.double() * h).sum(0), n * U * (dy.double() * h).abs().sum(0), "dw")
    within(db, dy.double().sum(0), n * U * dy.double().abs().sum(0), "db")


# tiles of 128 and 256, whole, divided, and some of each; sizes beside theirs; rows of less than a stage
WEIGHTS = [(1, 5, 7), (31, 130, 260), (33, 7, 500), (700, 300, 600), (1237, 199, 1300), (1237, 1999, 2693), (2047, 640, 2050),
           (1300, 4353, 4353), (5498, 2560, 2560), (4100, 96, 4200)]


@pytest.mark.parametrize("tdy", [BF16, F32])
@pytest.mark.parametrize("M,N,K", WEIGHTS)
def test_weight_sums_exact(ctx, tdy, M, N, K):
    """Whole numbers: |dy| up to 4, x up to 8 times a row's 1, 2 or 4, every sum under 2^24: dW and db are exact."""
    import torch
    g = gen(M + N + K)
    dy = whole_numbers(g, 4, M, N + 3).to(dt(tdy))[:, 2:N + 2]
    x = whole_numbers(g, 8, M, K) * torch.exp2(torch.randint(0, 3, (M, 1), generator=g, device="cuda").float())
    assert M * 4 * 32 < 2 ** 24
    q, s = ctx.quant_fp8(x)
    dw, db = ctx.grad_weight_fp8(dy, q, s, cols=K, bias=True)
    assert torch.equal(dw.double(), dy.double().t().contiguous() @ x.double())
    assert torch.equal(db.double(), dy.double().sum(0))


@pytest.mark.parametrize("M,N,K", [w for w in WEIGHTS if w[0] <= w[2]])
def test_weight_fp32_values_exact(ctx, M, N, K):
    """fp32 dy of 24 bits, each value alone in its sums (column k of x is a power of two in row k mod M and zeros): every bit of
    every row of dy arrives."""
    import torch
    g = gen(M + N)
    dy = torch.randint(-2 ** 24 + 1, 2 ** 24, (M, N), generator=g, device="cuda").float()
    dy = dy * torch.exp2(torch.randint(-40, 20, (M, N), generator=g, device="cuda").float())
    k = torch.arange(K, device="cuda")
    x = torch.zeros(M, K, device="cuda")
    x[k % M, k] = torch.where(k % 3 == 0, -2.0, torch.where(k % 3 == 1, 1.0, 0.25))
    q, s = ctx.quant_fp8(x)
    dw = ctx.grad_weight_fp8(dy, q, s, cols=K)
    assert torch.equal(dw, (dy[k % M] * x[k % M, k][:, None]).t())


def test_norm_squares_past_fp32(ctx):
    """Squares that sum past 2^128: rstd 0, the bias alone; the rows beside are as they would be."""
    import torch
    g = gen(1)
    x, b = randn(g, 5, 300), randn(g, 300)
    x[2] = torch.where(torch.arange(300, device="cuda") % 2 == 0, 1e25, -1e25)
    y, st = ctx.layer_norm(x, None, b, stats=True)
    assert torch.equal(y[2], b) and float(st[2, 1]) == 0.0
    keep = [0, 1, 3, 4]
    assert torch.equal(y[keep], ctx.layer_norm(x[keep], None, b))
