"""The operators of training a layer of one's own around the block, in their plain form and as the library's calls.

A program that fine-tunes a layer which attends to a text encoder's states, or serves it, normalises its rows,
attends from them to states of another length, and on the way back needs the gradients: of the norm, of the
attention, and of the projections' weights, for which it has kept the projections' input as 8-bit rows (quant_fp8)
in place of bf16 ones.  `own` chooses between elementary torch operations and the library's kernels (layer_norm,
layer_norm_grad, grad_weight_fp8, cross_attn and cross_attn_grad of awa_hip.Context).

Inputs come from the seed alone and are made on the GPU: activations N(0, 1) with one value in a thousand eight
times as large and a mean of their own in every row, gains 1 + N(0, 0.02), biases N(0, 0.02), queries, keys, values
and gradients N(0, 1).
"""
import math
import os
import random
import sys

import torch

own = False

DIM, QKV, MLP, HEADS, HEAD_D = 2560, 7680, 6912, 20, 128  # the model's widths
BLOCK = 128    # values per scale of an 8-bit row
E4M3_MAX = 448.0
EPS = 1e-5
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"bf16": 2, "f32": 4}


# ------------------------------------------------------------------ the cases

def _norm(name, rows, cols, x, out, ld=0):
    return {"name": name, "kind": "norm", "rows": rows, "cols": cols, "ld": ld or cols, "x": x, "out": out}


def _norm_grad(name, rows, cols, dy, x, out, ld=0):
    """x: the type of the rows that the forward pass kept ("fp8": e4m3 rows with block scales)."""
    return {"name": name, "kind": "norm_grad", "rows": rows, "cols": cols, "ld": ld or cols, "dy": dy, "x": x, "out": out}


def _weight(name, rows, n, k, dy, out, bias=False):
    return {"name": name, "kind": "weight", "rows": rows, "n": n, "k": k, "dy": dy, "out": out, "bias": bias}


def _cross(name, grad, seqs, q_len, k_len, heads, kv_heads, head_d, dtype, ragged=0, mask=False):
    """seqs sequences of q_len queries and k_len keys, or where ragged is not 0 of up to these, drawn from it.
    The keys of a sequence are the first of its k_len rows; mask: one key in ten takes no part."""
    return {"name": name, "kind": "cross_grad" if grad else "cross", "seqs": seqs, "q_len": q_len, "k_len": k_len,
            "heads": heads, "kv_heads": kv_heads, "head_d": head_d, "dtype": dtype, "ragged": ragged, "mask": mask}


def listed():
    return [
        # the text rows of one layer: the smallest call, bounded by its launch
        _norm("norm_text", 58, DIM, "bf16", "bf16"),
        # a clip of five latent frames of 1080p and its text: the fp32 residual stream, normalised for a projection
        _norm("norm_clip", 5 * 5440 + 58, DIM, "f32", "bf16"),
        # the way back at 1080p, to the fp32 residual stream
        _norm_grad("norm_grad_1080p", 5440 + 58, DIM, "bf16", "f32", "f32"),
        # rows of no round size, kept in 8 bits
        _norm_grad("norm_grad_saved_odd", 12370, 2693, "bf16", "fp8", "bf16", ld=2701),
        # the text's rows: few of them for a whole weight, bound by the weight's gradient
        _weight("weight_text", 58, QKV, DIM, "bf16", "f32", bias=True),
        # 1080p, the MLP's first product: the largest of a layer
        _weight("weight_1080p_mlp_in", 5440 + 58, 2 * MLP, DIM, "bf16", "bf16"),
        # sizes that no tile divides, fp32 gradients
        _weight("weight_odd_f32", 1237, 1999, 2693, "f32", "f32", bias=True),
        # serving: a token each of 32 requests, against an encoder's states of up to 1500 rows, shared heads
        _cross("cross_one_token", False, 32, 1, 1500, HEADS, 4, HEAD_D, "bf16", ragged=1),
        # 1080p, one frame's rows against a prompt
        _cross("cross_1080p_text", False, 1, 5440, 58, HEADS, HEADS, HEAD_D, "bf16"),
        # five frames against long text states
        _cross("cross_clip_long", False, 1, 5 * 5440, 1024, HEADS, HEADS, HEAD_D, "bf16"),
        # a step on four clips of different sizes, each with its own masked prompt
        _cross("cross_grad_clips", True, 4, 5440, 512, HEADS, HEADS, HEAD_D, "bf16", ragged=2, mask=True),
        # fp32 training with shared heads of another width
        _cross("cross_grad_shared_f32", True, 2, 1237, 300, 10, 2, 80, "f32", ragged=3),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(("norm", "norm_grad", "weight", "cross", "cross_grad"))
    either = ("bf16", "f32")
    if kind in ("norm", "norm_grad"):
        cols = _log(rng, 64, 8192)
        rows = _log(rng, 1, min(27000, 60_000_000 // cols))
        ld = cols + rng.choice((0, 0, 8, 13))
        if kind == "norm":
            return _norm("", rows, cols, rng.choice(either), rng.choice(either), ld)
        return _norm_grad("", rows, cols, rng.choice(either), rng.choice(("bf16", "f32", "fp8")), rng.choice(either), ld)
    if kind == "weight":
        rows, n, k = _log(rng, 1, 12000), _log(rng, 64, 14000), _log(rng, 100, 7000)
        dy = rng.choice(either)
        while rows * n * k * (3 if dy == "f32" else 1) > 5498 * 2 * MLP * DIM:
            rows = (rows + 1) // 2
        if rng.random() < 0.5:  # a width that a model has
            n, k = max(64, n // 64 * 64), max(128, k // 128 * 128)
        return _weight("", rows, n, k, dy, rng.choice(either), rng.random() < 0.5)
    grad = kind == "cross_grad"
    head_d, dtype = rng.choice((64, 80, 96, 128)), rng.choice(("bf16", "bf16", "f32"))
    kv_heads = rng.choice((1, 2, 5, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    # a softmax over one key has no gradient, only its rounding: eight keys at least
    seqs, k_len = _log(rng, 1, 32), _log(rng, 16, 2048)
    q_len = 1 if rng.random() < 0.3 else _log(rng, 2, 20000)
    most = 5 * 5440 * 1024 * HEADS * HEAD_D // (4 if grad else 1) // (8 if dtype == "f32" else 1)
    while seqs * q_len * k_len * heads * head_d > most or seqs * q_len * heads * head_d > 60_000_000:
        q_len, seqs = (q_len + 1) // 2, max(1, seqs - 1)
    return _cross("", grad, seqs, q_len, k_len, heads, kv_heads, head_d, dtype, rng.choice((0, rng.randrange(1, 1 << 20))),
                  rng.random() < 0.4)


def _lengths(case):
    """Queries and keys of each sequence: the case's own."""
    s = case["seqs"]
    if not case["ragged"]:
        return [case["q_len"]] * s, [case["k_len"]] * s
    rng = random.Random(case["ragged"])
    q = [rng.randint((case["q_len"] + 1) // 2, case["q_len"]) for _ in range(s)]
    return q, [rng.randint((case["k_len"] + 1) // 2, case["k_len"]) for _ in range(s)]


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
    x = torch.where(torch.rand((rows, cols), generator=g, device="cuda") < 1e-3, 8 * x, x)
    return x + torch.randn((rows, 1), generator=g, device="cuda")


def _saved(x):
    """x as 8-bit rows: (e4m3 [rows][cols padded to blocks], e8m0 scales [groups of four blocks][rows][4])."""
    rows, cols = x.shape
    kp = _padded(cols)
    b = torch.nn.functional.pad(x.float(), (0, kp - cols)).unflatten(1, (-1, BLOCK))
    m, e = torch.frexp(b.abs().amax(2, keepdim=True))  # m 2^e, m in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(m > 0, e - torch.where(m <= 0.875, 9, 8), -127).clamp(min=-127)
    q = torch.ldexp(b, -e).to(torch.float8_e4m3fn).flatten(1)
    s = torch.nn.functional.pad((e[:, :, 0] + 127).to(torch.uint8), (0, 4 * _groups(cols) - kp // BLOCK))
    return q.contiguous(), s.unflatten(1, (-1, 4)).transpose(0, 1).contiguous().view(torch.float8_e8m0fnu)


def _starts(lengths):
    return [sum(lengths[:i]) for i in range(len(lengths))]


def _on_gpu(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def prepare(case, seed):
    g = _generator(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    s = {"case": dict(case)}
    if case["kind"] in ("norm", "norm_grad"):
        x = _activations(case["rows"], case["ld"], g)
        s["weight"], s["bias"] = 1 + 0.02 * normal(case["cols"]), 0.02 * normal(case["cols"])
        if case["kind"] == "norm":
            s["x"] = x.to(DTYPES[case["x"]])[:, : case["cols"]]
            return s
        x = x[:, : case["cols"]] if case["x"] == "fp8" else x.to(DTYPES[case["x"]])[:, : case["cols"]]
        v = x.double()
        mean = v.mean(1)
        s["stats"] = torch.stack((mean, (v.var(1, unbiased=False) + EPS).rsqrt()), 1).float()
        s["x"], s["x_scale"] = _saved(x) if case["x"] == "fp8" else (x, None)
        s["dy"] = normal(case["rows"], case["ld"]).to(DTYPES[case["dy"]])[:, : case["cols"]]
    elif case["kind"] == "weight":
        s["x"], s["x_scale"] = _saved(_activations(case["rows"], case["k"], g))
        s["dy"] = normal(case["rows"], case["n"]).to(DTYPES[case["dy"]])
    else:
        dtype, (ql, kl) = DTYPES[case["dtype"]], _lengths(case)
        s["lengths"] = ql, kl
        s["q_at"], s["q_len"] = _on_gpu(_starts(ql)), _on_gpu(ql)
        s["k_at"], s["k_len"] = torch.arange(len(kl), device="cuda") * case["k_len"], _on_gpu(kl)
        s["q"] = normal(sum(ql), case["heads"], case["head_d"]).to(dtype)
        # keys and values side by side in a projection's rows
        kv = normal(case["seqs"] * case["k_len"], 2, case["kv_heads"], case["head_d"]).to(dtype)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
        s["mask"] = torch.rand(kv.shape[0], generator=g, device="cuda") < 0.9 if case["mask"] else None
        if case["kind"] == "cross_grad":
            s["dout"] = normal(*s["q"].shape).to(dtype)
            s["out"], s["lse"] = _plain_cross(s)
    return s


# ------------------------------------------------------------------ the plain forms

def _values(q, scale, cols):
    """fp32 values of 8-bit rows (a power of two is exact)."""
    b = scale.view(torch.uint8).transpose(0, 1).flatten(1)[:, : q.shape[1] // BLOCK]
    return torch.ldexp(q.float().unflatten(1, (-1, BLOCK)), (b.int() - 127)[:, :, None]).flatten(1)[:, :cols]


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / ((d * d).mean(1, keepdim=True) + EPS).sqrt()
    y = d * rstd * s["weight"] + s["bias"]
    return y.to(DTYPES[s["case"]["out"]]), torch.cat((mean, rstd), 1)


def _plain_norm_grad(s):
    case, dy = s["case"], s["dy"].float()
    x = s["x"].float() if s["x_scale"] is None else _values(s["x"], s["x_scale"], case["cols"])
    mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
    xhat = (x - mean) * rstd
    d = dy * s["weight"]
    dx = rstd * (d - d.mean(1, keepdim=True) - xhat * (d * xhat).mean(1, keepdim=True))
    return dx.to(DTYPES[case["out"]]), (dy * xhat).sum(0), dy.sum(0)


def _plain_weight(s):
    case, dy = s["case"], s["dy"].float()
    dw = (dy.T @ _values(s["x"], s["x_scale"], case["k"])).to(DTYPES[case["out"]])
    return (dw, dy.sum(0)) if case["bias"] else dw


def _rows_of(at, length, most):
    """[sequences][most] row numbers, and whether they are within their sequence."""
    i = torch.arange(most, device=at.device)
    there = i < length[:, None]
    return torch.where(there, at[:, None] + i, 0), there


def _gather(x, rows, there, groups=1):
    """[sequences][heads][rows][head_d] fp32, zeros where no row is; each head `groups` times."""
    y = torch.where(there[:, :, None, None], x[rows].float(), 0.0).transpose(1, 2)
    return y.repeat_interleave(groups, 1)


def _scatter(y, rows, there, count):
    """The rows of y [sequences][heads][rows][head_d] in their places; the last place takes what is no row."""
    out = y.new_zeros((count + 1, y.shape[1], y.shape[3]))
    out[torch.where(there, rows, count)] = y.transpose(1, 2)
    return out[:count]


def _probabilities(s):
    """(P, lse, K, V, rows and places of queries and keys) with scores in fp32."""
    case = s["case"]
    qr, qt = _rows_of(s["q_at"], s["q_len"], max(s["lengths"][0]))
    kr, kt = _rows_of(s["k_at"], s["k_len"], max(s["lengths"][1]))
    if s["mask"] is not None:
        kt = kt & s["mask"][kr]
    groups = case["heads"] // case["kv_heads"]
    q, k, v = _gather(s["q"], qr, qt), _gather(s["k"], kr, kt, groups), _gather(s["v"], kr, kt, groups)
    sc = (q @ k.transpose(2, 3)) * case["head_d"] ** -0.5
    sc = torch.where(kt[:, None, None, :], sc, -math.inf)
    top = sc.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = (sc - top).exp()
    total = e.sum(3, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)  # a row without keys: zeros
    return p, top + total.log(), q, k, v, (qr, qt), (kr, kt)


def _plain_cross(s):
    p, lse, _, _, v, (qr, qt), _ = _probabilities(s)
    n = s["q"].shape[0]
    return _scatter(p @ v, qr, qt, n).to(s["q"].dtype), _scatter(lse, qr, qt, n)[:, :, 0].T.contiguous()


def _plain_cross_grad(s):
    case = s["case"]
    p, _, q, k, v, (qr, qt), (kr, kt) = _probabilities(s)
    do = _gather(s["dout"], qr, qt)
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(3, keepdim=True)) * case["head_d"] ** -0.5

    def shared(x):  # summed over the heads that share a key's
        return x.unflatten(1, (case["kv_heads"], -1)).sum(2)

    n, m, t = s["q"].shape[0], s["k"].shape[0], s["q"].dtype
    return (_scatter(ds @ k, qr, qt, n).to(t), _scatter(shared(ds.transpose(2, 3) @ q), kr, kt, m).to(t),
            _scatter(shared(p.transpose(2, 3) @ do), kr, kt, m).to(t))


# ------------------------------------------------------------------ one pass

_held = []


def _context():
    """The library's handle, which a program makes once."""
    if not _held:
        sys.path.insert(0, os.path.join(os.getcwd(), "seedvr2-2b-ncnn_amd"))
        import awa_hip
        _held.append(awa_hip.Context(0))
    return _held[0]


def _plan(s):
    """The lengths' plan, which a program makes once for a batch and uses in all of its layers."""
    if "plan" not in s:
        case, (ql, kl) = s["case"], s["lengths"]
        s["plan"] = _context().cross_plan(case["heads"], case["head_d"], ql, kl, kv_heads=case["kv_heads"],
                                          k_at=[case["k_len"] * i for i in range(case["seqs"])])
    return s["plan"]


def run(state):
    s, case, kind = state, state["case"], state["case"]["kind"]
    if kind == "norm":
        if own:
            return _context().layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, dtype=DTYPES[case["out"]], stats=True)
        return _plain_norm(s)
    if kind == "norm_grad":
        if own:
            return _context().layer_norm_grad(s["dy"], s["x"], s["stats"], s["weight"], x_scale=s["x_scale"],
                                              dtype=DTYPES[case["out"]])
        return _plain_norm_grad(s)
    if kind == "weight":
        if own:
            return _context().grad_weight_fp8(s["dy"], s["x"], s["x_scale"], cols=case["k"], bias=case["bias"],
                                              dtype=DTYPES[case["out"]])
        return _plain_weight(s)
    if kind == "cross":
        if own:
            return _context().cross_attn(_plan(s), s["q"], s["k"], s["v"], mask=s["mask"], lse=True)
        return _plain_cross(s)
    if own:
        return _context().cross_attn_grad(_plan(s), s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], mask=s["mask"])
    return _plain_cross_grad(s)


def work(case):
    kind = case["kind"]
    if kind == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SIZE[case["x"]] + SIZE[case["out"]]) + 8 * (case["rows"] + case["cols"]), "flops": 8 * n}
    saved = case["rows"] * (_padded(case.get("k", case.get("cols"))) + 4 * _groups(case.get("k", case.get("cols")))) if (
        kind == "weight" or case.get("x") == "fp8") else 0
    if kind == "norm_grad":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (SIZE[case["dy"]] + SIZE.get(case["x"], 0) + SIZE[case["out"]]) + saved + 8 * case["rows"] +
                12 * case["cols"], "flops": 14 * n}
    if kind == "weight":
        m, n, k = case["rows"], case["n"], case["k"]
        return {"bytes": m * n * SIZE[case["dy"]] + saved + n * k * SIZE[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    ql, kl = _lengths(case)
    pairs, size = sum(a * b for a, b in zip(ql, kl)), SIZE[case["dtype"]]
    queries, keys = sum(ql) * case["heads"], sum(kl) * case["kv_heads"]
    wide = (2 * queries + 2 * keys) if kind == "cross" else (4 * queries + 4 * keys)
    return {"bytes": wide * case["head_d"] * size + 4 * queries + (sum(kl) if case["mask"] else 0),
            "flops": (4 if kind == "cross" else 10) * pairs * case["heads"] * case["head_d"]}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_rows(q, scale, cols):
    e = scale.double().permute(1, 0, 2).reshape(q.shape[0], -1)
    return q.double()[:, :cols] * e[:, torch.arange(cols, device=q.device) // BLOCK]


def _exact_norm(s):
    x = s["x"].double()
    var, mean = torch.var_mean(x, 1, correction=0)
    rstd = (var + EPS) ** -0.5
    y = torch.addcmul(s["bias"].double(), (x - mean[:, None]) * rstd[:, None], s["weight"].double())
    return y, torch.stack((mean, rstd), 1)


def _exact_norm_grad(s):
    dy, n = s["dy"].double(), s["case"]["cols"]
    x = s["x"].double() if s["x_scale"] is None else _exact_rows(s["x"], s["x_scale"], n)
    mean, rstd = s["stats"].double().unbind(1)
    h = (x - mean[:, None]) * rstd[:, None]
    a = dy * s["weight"].double()
    # the gradient of y through x directly, through the mean and through the variance
    through_mean = -a.sum(1) / n
    through_var = -(a * h).sum(1) / n
    dx = (a + through_mean[:, None] + through_var[:, None] * h) * rstd[:, None]
    return dx, torch.einsum("rc,rc->c", dy, h), dy.sum(0)


def _exact_weight(s):
    dy = s["dy"].double()
    dw = dy.t().contiguous() @ _exact_rows(s["x"], s["x_scale"], s["case"]["k"])
    return (dw, torch.ones(dy.shape[0], dtype=torch.float64, device=dy.device) @ dy) if s["case"]["bias"] else dw


def _exact_heads(s):
    """For each sequence and head: its rows, its keys that take part, and Q, K, V in 64 bits."""
    case = s["case"]
    per, c = case["heads"] // case["kv_heads"], case["head_d"] ** -0.5
    q0 = 0
    for i, (nq, nk) in enumerate(zip(*s["lengths"])):
        keys = torch.arange(i * case["k_len"], i * case["k_len"] + nk, device="cuda")
        if s["mask"] is not None:
            keys = keys[s["mask"][keys]]
        for h in range(case["heads"]):
            yield (slice(q0, q0 + nq), h, keys, h // per, s["q"][q0:q0 + nq, h].double() * c,
                   s["k"][keys, h // per].double(), s["v"][keys, h // per].double())
        q0 += nq


def _exact_cross(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full((s["q"].shape[1], s["q"].shape[0]), -math.inf, dtype=torch.float64, device="cuda")
    for rows, h, keys, _, q, k, v in _exact_heads(s):
        if keys.numel():
            sc = q @ k.t()
            lse[h, rows] = torch.logsumexp(sc, 1)
            out[rows, h] = torch.softmax(sc, 1) @ v
    return out, lse


def _exact_cross_grad(s):
    c = s["case"]["head_d"] ** -0.5
    dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in ("q", "k", "v"))
    for rows, h, keys, hk, q, k, v in _exact_heads(s):
        p = torch.softmax(q @ k.t(), 1)
        do = s["dout"][rows, h].double()
        dp = do @ v.t()
        ds = p * dp - p * (p * dp).sum(1, keepdim=True)
        dq[rows, h] = c * (ds @ k)
        dk[keys, hk] += ds.t() @ q
        dv[keys, hk] += p.t() @ do
    return dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "norm_grad": _exact_norm_grad, "weight": _exact_weight, "cross": _exact_cross,
            "cross_grad": _exact_cross_grad}[case["kind"]](s)
