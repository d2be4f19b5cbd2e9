"""dit_train.h on the CPU beside test_train_cpu.py: what the attention's entry points take and pass on
(tests/cpp/test_cross_args.cpp, which includes csrc/dit_train.cpp with stubs for the launches)."""
import os
import subprocess

import pytest

from test_train_cpu import HIPCC, PKG, ROOT, meta_context, meta_plan


def test_attention_arguments(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not present")
    exe = str(tmp_path / "test_cross_args")
    cmd = [HIPCC, "--offload-arch=gfx950", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "cpp", "test_cross_args.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout.split("checks=")[1].split()[0]) > 20


def test_whole_reaches_the_library(awa, monkeypatch):
    import torch
    ctx, calls = meta_context(awa, monkeypatch)
    plan = meta_plan(awa, ctx, 10, 20)
    for dtype, code in ((torch.bfloat16, awa.AWA_BF16), (torch.float32, awa.AWA_F32)):
        q, k = torch.empty(10, 4, 64, dtype=dtype, device="meta"), torch.empty(20, 2, 64, dtype=dtype, device="meta")
        lse = torch.empty(4, 10, device="meta")
        for whole in (False, True):
            ctx.cross_attn(plan, q, k, k, whole=whole)
            ctx.cross_attn_grad(plan, q, q, k, k, q, lse, whole=whole)
            assert [args[2] for _, args in calls] == 2 * [code | awa.DIT_CROSS_WHOLE if whole else code]
            calls.clear()


def test_a_collected_plan_is_dropped_and_a_closed_one_destroyed(awa, monkeypatch):
    """Collection may come while a stream is captured or a graph lives: it must not free."""
    ctx, calls = meta_context(awa, monkeypatch)
    for end, name in ((lambda p: p.close(), "dit_cross_destroy"), (lambda p: None, "dit_cross_drop")):
        plan = meta_plan(awa, ctx, 10, 20)
        del plan.close  # the class's own
        end(plan)
        del plan
        assert [n for n, _ in calls] == [name]
        calls.clear()
