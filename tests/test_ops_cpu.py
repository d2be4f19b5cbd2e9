"""dit_ops.h on the CPU: the refusals of its entry points (tests/cpp/test_ops_args.cpp, which compiles
csrc/dit_ops.cpp with stubs for the launches and never reads the addresses it passes), the frequencies
against their formulas, and the shapes that the binding refuses."""
import math
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "seedvr2-2b-ncnn_amd")
HIPCC = "/opt/rocm/bin/hipcc"


def test_refusals(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not present")
    exe = str(tmp_path / "test_ops_args")
    # the shared header holds device helpers, so hipcc compiles the driver (host code only)
    cmd = [HIPCC, "--offload-arch=gfx950", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "cpp", "test_ops_args.cpp"),
           os.path.join(PKG, "csrc", "dit_ops.cpp"), "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout.split("checks=")[1].split()[0]) > 100


@pytest.mark.parametrize("n,base,factor", [(1, 10000.0, 1.0), (21, 10000.0, 4.0), (64, 500000.0, 32.0), (128, 2.0, 1.5)])
def test_freqs(awa, n, base, factor):
    i = np.arange(n)
    f = base ** (-i / n)
    close = dict(rtol=1e-14)  # a few roundings of 2^-53 in pow and the products
    np.testing.assert_allclose(awa.rope_freqs(n, base), f, **close)
    np.testing.assert_allclose(awa.rope_freqs(n, base, "linear", factor), f / factor, **close)
    if n > 1:
        g = awa.rope_freqs(n, base, "base", factor)
        assert g[0] == 1.0
        assert math.isclose(g[-1], f[-1] / factor, rel_tol=1e-13)
    trained, lo, hi = 4096.0, 1.0, 32.0
    g = awa.rope_freqs(n, base, "bands", factor, trained, lo, hi)
    turns = trained * f / (2 * np.pi)
    np.testing.assert_allclose(g[turns >= hi], f[turns >= hi], **close)
    np.testing.assert_allclose(g[turns <= lo], f[turns <= lo] / factor, **close)
    t = np.clip((turns - lo) / (hi - lo), 0, 1)
    np.testing.assert_allclose(g, f * (t + (1 - t) / factor), **close)
    assert (np.diff(g) < 0).all()


def test_freqs_refused(awa):
    for args in ((0,), (129,), (8, -1.0), (8, 1e4, "linear", 0.5), (8, 1e4, "bands", 2.0, 0.0)):
        with pytest.raises(awa.AwaError):
            awa.rope_freqs(*args)


def test_binding_refuses_host_tensors(awa):
    """Refused before any device call (a context object without a device)."""
    import torch
    ctx = awa.Context.__new__(awa.Context)
    ctx.ptr, ctx.device = None, 0
    x = torch.zeros((3, 256))
    q, s = torch.zeros((3, 256), dtype=torch.uint8), torch.zeros((1, 3, 4), dtype=torch.uint8)
    w, ws = torch.zeros((5, 256), dtype=torch.uint8), torch.zeros((1, 1, 4), dtype=torch.uint8)
    pos = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ctx.quant_fp8(x), lambda: ctx.gemm_fp8(q, s, w, ws), lambda: ctx.rope(x[:, None], pos, [1.0]),
                 lambda: ctx.quant_fp8(x.T), lambda: ctx.rope(x[:, None], pos.long(), [1.0]),
                 lambda: ctx.rope(x[:, None], pos, [1.0], pairs=(1, 0))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ctx.quant_fp8(x.half()), lambda: ctx.rope(x[:, None].half(), pos, [1.0])):
        with pytest.raises(TypeError):
            call()


def meta_context(awa, monkeypatch):
    """(a context for tensors without memory, the calls that reach the library), whose entry points only count."""
    import torch

    class Entries:
        def __getattr__(self, name):
            return lambda *args: calls.append((name, args)) or 0

    ctx, calls = awa.Context.__new__(awa.Context), []
    ctx.ptr, ctx.device, ctx._on = None, -1, torch.device("meta")
    monkeypatch.setattr(awa, "lib", Entries)
    monkeypatch.setattr(awa.Context, "_stream", lambda self, stream: 0)
    return ctx, calls


def test_binding_refuses_sizes_past_32_bits(awa, monkeypatch):
    """Sizes whose low 32 bits the entry points would take: the rest was neither computed nor refused."""
    import torch
    ctx, calls = meta_context(awa, monkeypatch)
    e4m3, e8m0, far = torch.float8_e4m3fn, torch.float8_e8m0fnu, 2 ** 32

    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")

    def matrix(rows, cols, blocks):
        return (empty(rows, cols, dtype=e4m3),
                empty((cols + 511) // 512, (rows + 127) // 128 if blocks else rows, 4, dtype=e8m0))

    ctx.quant_fp8(empty(5, 128))
    ctx.gemm_fp8(*matrix(5, 128, False), *matrix(7, 128, True))
    ctx.rope(empty(5, 1, 2), empty(5, dtype=torch.int32), [1.0])
    assert [name for name, _ in calls] == ["dit_quant_fp8", "dit_gemm_fp8", "dit_rope"]
    for call in (lambda: ctx.quant_fp8(empty(far + 5, 128)), lambda: ctx.quant_fp8(empty(5, far + 128)),
                 lambda: ctx.quant_fp8(empty(2 ** 24 + 1, 128)), lambda: ctx.quant_fp8(empty(5, 2 ** 20 + 1), blocks=True),
                 lambda: ctx.gemm_fp8(*matrix(far + 5, 128, False), *matrix(7, 128, True)),
                 lambda: ctx.gemm_fp8(*matrix(5, 128, False), *matrix(far + 7, 128, True)),
                 lambda: ctx.gemm_fp8(*matrix(5, far + 128, False), *matrix(7, far + 128, True)),
                 lambda: ctx.rope(empty(far + 5, 1, 2), empty(far + 5, dtype=torch.int32), [1.0]),
                 lambda: ctx.rope(empty(5, far + 1, 2), empty(5, dtype=torch.int32), [1.0])):
        with pytest.raises(ValueError, match="at most"):
            call()
    assert len(calls) == 3


def test_tensors_of_another_stream_are_marked(awa, monkeypatch):
    """Each tensor of a call on a given stream is marked as used there, so that its memory outlives the call."""
    import torch
    ctx, calls = meta_context(awa, monkeypatch)
    monkeypatch.setattr(awa.Context, "_empty", lambda self, dtype, stream, *shape: torch.empty(shape, dtype=dtype, device="meta"))
    marked, stream = [], object()
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: marked.append((t, s)))

    def empty(*shape, dtype=torch.bfloat16):
        return torch.empty(shape, dtype=dtype, device="meta")

    def check(*tensors):
        assert all(s is stream for _, s in marked)
        assert {id(t) for t in tensors} <= {id(t) for t, _ in marked}
        marked.clear()

    x, wt, bias = empty(5, 128), empty(130, 128), empty(130, dtype=torch.float32)
    a, w = ctx.quant_fp8(x), ctx.quant_fp8(wt, blocks=True)
    assert not marked
    check(x, *ctx.quant_fp8(x, stream=stream))
    ctx.quant_fp8(x, q=a[0], scale=a[1], stream=stream)
    check(x, *a)
    check(*a, *w, bias, ctx.gemm_fp8(*a, *w, bias=bias, stream=stream))
    out = empty(5, 130)
    ctx.gemm_fp8(*a, *w, out=out, stream=stream)
    check(*a, *w, out)
    q, k, pos = empty(5, 3, 64), empty(5, 1, 64), empty(5, dtype=torch.int32)
    check(q, k, pos, *ctx.rope((q, k), pos, [1.0] * 32, stream=stream))
    assert len(calls) == 7


def test_freqs_refused_by_the_binding(awa):
    """Numbers of pairs whose low 32 bits are allowed, and kinds that are none."""
    for n in (2 ** 32 + 8, -2 ** 32 + 8):
        with pytest.raises(awa.AwaError):
            awa.rope_freqs(n)
    with pytest.raises(ValueError, match="kind must be one of"):
        awa.rope_freqs(8, kind="cubic")


def test_product_reads_sums_after_their_wait_states(tmp_path):
    """The static check of the other matrix kernels over the 8-bit product's: its sums pass through empty asm
    statements, which the compiler does not wait before."""
    import test_sdpa_asm
    test_sdpa_asm.test_other_mfma_kernels_wait_states(tmp_path, "dit_fp8_gemm")
