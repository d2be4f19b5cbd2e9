"""dit_train.h on the CPU: the refusals of its entry points and the attention's plans (tests/cpp/test_train_args.cpp, which
includes csrc/dit_train.cpp with stubs for the launches and never reads the addresses it passes), and what the binding
refuses."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "seedvr2-2b-ncnn_amd")
HIPCC = "/opt/rocm/bin/hipcc"


def test_refusals_and_plans(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not present")
    exe = str(tmp_path / "test_train_args")
    # the shared header holds device helpers, so hipcc compiles the driver (host code only)
    cmd = [HIPCC, "--offload-arch=gfx950", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "cpp", "test_train_args.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout.split("checks=")[1].split()[0]) > 900


class Entries:
    """Entry points that only count."""

    def __init__(self, calls):
        self.calls = calls

    def __getattr__(self, name):
        if name.endswith("_work"):
            return lambda *args: 0
        return lambda *args: self.calls.append((name, args)) or 0


def meta_context(awa, monkeypatch):
    """(a context for tensors without memory, the calls that reach the library)."""
    import torch
    awa.lib()
    ctx, calls = awa.Context.__new__(awa.Context), []
    ctx.ptr, ctx.device, ctx._on = None, -1, torch.device("meta")
    entries = Entries(calls)
    monkeypatch.setattr(awa, "lib", lambda: entries)
    monkeypatch.setattr(awa.Context, "_stream", lambda self, stream: 0)
    return ctx, calls


def meta_plan(awa, ctx, q_rows, k_rows, heads=4, kv_heads=2, head_d=64):
    plan = awa.CrossPlan.__new__(awa.CrossPlan)
    plan.ptr, plan.device, plan.heads, plan.kv_heads, plan.head_d = 1, ctx.device, heads, kv_heads, head_d
    plan.q_rows = plan._q_count = q_rows
    plan.k_rows = plan._k_count = k_rows
    plan._work = {}
    plan.close = lambda: None
    return plan


def test_binding_refusals(awa, monkeypatch):
    import torch
    ctx, calls = meta_context(awa, monkeypatch)
    bf, f32, e4m3, e8m0, far = torch.bfloat16, torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu, 2 ** 32

    def empty(*shape, dtype=bf):
        return torch.empty(shape, dtype=dtype, device="meta")

    def rows8(rows, cols):
        return empty(rows, (cols + 127) // 128 * 128, dtype=e4m3), empty((cols + 511) // 512, rows, 4, dtype=e8m0)

    st = empty(5, 2, dtype=f32)
    ctx.layer_norm(empty(5, 100), empty(100, dtype=f32), empty(100, dtype=f32), stats=st)
    ctx.layer_norm_grad(empty(5, 100), empty(5, 100, dtype=f32), st)
    x8, s8 = rows8(5, 100)
    ctx.layer_norm_grad(empty(5, 100), x8, st, x_scale=s8)
    ctx.grad_weight_fp8(empty(5, 7), x8, s8, cols=100, bias=True)
    plan = meta_plan(awa, ctx, 10, 20)
    q, k = empty(10, 4, 64), empty(20, 2, 64)
    lse = empty(4, 10, dtype=f32)
    ctx.cross_attn(plan, q, k, k, lse=True)
    ctx.cross_attn_grad(plan, q, q, k, k, q, lse, mask=empty(20, dtype=torch.bool))
    assert [n for n, _ in calls] == ["dit_layer_norm", "dit_layer_norm_grad", "dit_layer_norm_grad", "dit_grad_weight_fp8",
                                     "dit_cross_forward", "dit_cross_grad"]
    refused = [
        lambda: ctx.layer_norm(empty(5)), lambda: ctx.layer_norm(empty(100, 5).T), lambda: ctx.layer_norm(empty(5, 16385)),
        lambda: ctx.layer_norm(empty(far + 5, 100)), lambda: ctx.layer_norm(empty(5, far + 100)),
        lambda: ctx.layer_norm(empty(5, 0)), lambda: ctx.layer_norm(empty(5, 100), empty(100)),
        lambda: ctx.layer_norm(empty(5, 100), empty(99, dtype=f32)),
        lambda: ctx.layer_norm(empty(5, 100), empty(200, dtype=f32)[::2]),
        lambda: ctx.layer_norm(empty(5, 100), bias=empty(1, 100, dtype=f32)),
        lambda: ctx.layer_norm(empty(5, 100), out=empty(5, 101)), lambda: ctx.layer_norm(empty(5, 100), out=empty(5, 100), dtype=f32),
        lambda: ctx.layer_norm(empty(5, 100), stats=empty(5, 3, dtype=f32)),
        lambda: ctx.layer_norm(empty(0, 0)),
        lambda: ctx.layer_norm_grad(empty(5, 100), empty(5, 101), st), lambda: ctx.layer_norm_grad(empty(6, 100), empty(6, 100), st),
        lambda: ctx.layer_norm_grad(empty(5, 100), empty(5, 100), None),
        lambda: ctx.layer_norm_grad(empty(5, 100), x8[:, :100], st, x_scale=s8),
        lambda: ctx.layer_norm_grad(empty(5, 100), x8, st, x_scale=s8[:, :4]),
        lambda: ctx.layer_norm_grad(empty(5, 100), empty(5, 100), st, dx=empty(5, 100), dtype=f32),
        lambda: ctx.grad_weight_fp8(empty(5, 7), x8, s8, cols=129), lambda: ctx.grad_weight_fp8(empty(5, 7), x8, s8, cols=0),
        lambda: ctx.grad_weight_fp8(empty(6, 7), x8, s8), lambda: ctx.grad_weight_fp8(empty(5, 7), x8, s8, cols=100, add=True),
        lambda: ctx.grad_weight_fp8(empty(5, 7), x8, s8, out=empty(7, 128, dtype=f32), add=True, bias=True),
        lambda: ctx.grad_weight_fp8(empty(5, 7), x8, s8, cols=100, out=empty(7, 128)),
        lambda: ctx.grad_weight_fp8(empty(5, far + 7), x8, s8),
        lambda: ctx.grad_weight_fp8(empty(5, 7), x8, s8, bias=empty(8, dtype=f32)),
        lambda: ctx.cross_attn(plan, q[:9], k, k), lambda: ctx.cross_attn(plan, q, k[:19], k), lambda: ctx.cross_attn(plan, q, k, k[:19]),
        lambda: ctx.cross_attn(plan, q, k.float(), k), lambda: ctx.cross_attn(plan, q, k, k.float()),
        lambda: ctx.cross_attn(plan, q[:, :3], k, k), lambda: ctx.cross_attn(plan, q, q, q),
        lambda: ctx.cross_attn(plan, empty(10, 4, 128)[:, :, ::2], k, k), lambda: ctx.cross_attn(plan, q, k, k, out=empty(9, 4, 64)),
        lambda: ctx.cross_attn(plan, q, k, k, out=empty(10, 4, 64, dtype=f32)),
        lambda: ctx.cross_attn(plan, q, k, k, lse=empty(10, 4, dtype=f32)),
        lambda: ctx.cross_attn(plan, q, k, k, mask=empty(19, dtype=torch.bool)),
        lambda: ctx.cross_attn(plan, q, k, k, mask=empty(20, dtype=f32)),
        lambda: ctx.cross_attn_grad(plan, q, q, k, k, q, None), lambda: ctx.cross_attn_grad(plan, q[:9], q, k, k, q, lse),
        lambda: ctx.cross_attn_grad(plan, q, q, k, k, q, lse, dk=empty(21, 2, 64)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    for call in (lambda: ctx.layer_norm(empty(5, 100, dtype=torch.half)), lambda: ctx.cross_attn(plan, q.half(), k.half(), k.half()),
                 lambda: ctx.layer_norm_grad(empty(5, 100, dtype=torch.half), empty(5, 100), st),
                 lambda: ctx.grad_weight_fp8(empty(5, 7, dtype=torch.half), x8, s8)):
        with pytest.raises(TypeError):
            call()
    assert len(calls) == 6
    plan.ptr = None
    with pytest.raises(ValueError, match="closed"):
        ctx.cross_attn(plan, q, k, k)
    other = meta_plan(awa, ctx, 10, 20)
    other.device = 3
    with pytest.raises(ValueError, match="device"):
        ctx.cross_attn(other, q, k, k)


def test_tensors_of_another_stream_are_marked(awa, monkeypatch):
    """Each tensor of a call on a given stream is marked as used there, so that its memory outlives the call."""
    import torch
    ctx, _ = meta_context(awa, monkeypatch)
    monkeypatch.setattr(awa.Context, "_empty", lambda self, dtype, stream, *shape: torch.empty(shape, dtype=dtype, device="meta"))
    marked, stream = [], object()
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: marked.append((t, s)))
    bf, f32 = torch.bfloat16, torch.float32

    def empty(*shape, dtype=bf):
        return torch.empty(shape, dtype=dtype, device="meta")

    def check(*tensors):
        assert all(s is stream for _, s in marked)
        assert {id(t) for t in tensors} <= {id(t) for t, _ in marked}
        marked.clear()

    x, w, b, dy = empty(5, 100), empty(100, dtype=f32), empty(100, dtype=f32), empty(5, 100)
    y, st = ctx.layer_norm(x, w, b, stats=True)
    assert not marked
    check(x, w, b, *ctx.layer_norm(x, w, b, stats=True, stream=stream))
    check(dy, x, st, w, *ctx.layer_norm_grad(dy, x, st, w, stream=stream))
    x8, s8 = empty(5, 128, dtype=torch.float8_e4m3fn), empty(1, 5, 4, dtype=torch.float8_e8m0fnu)
    check(dy, x8, s8, st, *ctx.layer_norm_grad(dy, x8, st, x_scale=s8, stream=stream))
    check(dy, x8, s8, *ctx.grad_weight_fp8(dy, x8, s8, cols=100, bias=True, stream=stream))
    plan = meta_plan(awa, ctx, 10, 20)
    q, do, k, v, mask = empty(10, 4, 64), empty(10, 4, 64), empty(20, 2, 64), empty(20, 2, 64), empty(20, dtype=torch.bool)
    out, lse = ctx.cross_attn(plan, q, k, v, mask=mask, lse=True, stream=stream)
    check(q, k, v, mask, out, lse)
    check(do, q, k, v, mask, out, lse, *ctx.cross_attn_grad(plan, do, q, k, v, out, lse, mask=mask, stream=stream))


def test_cross_plan_refusals(awa):
    ctx = awa.Context.__new__(awa.Context)
    ctx.ptr, ctx.device = None, 0
    for args, kw in (((4, 64, [1.5], [2]), {}), ((4, 64, [[1]], [2]), {}), ((4, 64, [1, 2], [2]), {}), ((4, 64, [1], [2]), {"q_at": [0, 1]}),
                     ((4, 64, [1], [2]), {"k_at": []}), ((2 ** 32 + 4, 64, [1], [2]), {}), ((4, 64, [1], [2]), {"kv_heads": 2 ** 32 + 2}),
                     ((4, 2 ** 32 + 64, [1], [2]), {}), ((4, 64, [1] * 65537, [2] * 65537), {}), ((4, 64, [1], [2]), {"kv_heads": 0})):
        with pytest.raises(ValueError):
            ctx.cross_plan(*args, **kw)
