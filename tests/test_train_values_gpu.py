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
