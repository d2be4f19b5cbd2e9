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


def test_stream_of_another_device_marks_nothing(awa, monkeypatch):
    """A stream that the call refuses leaves no mark on the tensors given to it."""
    import torch
    own_stream = awa.Context._stream
    ctx, calls = meta_context(awa, monkeypatch)
    monkeypatch.setattr(awa.Context, "_stream", own_stream)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: pytest.fail("marked"))

    class Stream:
        device_index, device, cuda_stream = 5, "cuda:5", 0

    def empty(*shape, dtype=torch.uint8):
        return torch.empty(shape, dtype=dtype, device="meta")

    x, q, s = empty(5, 128, dtype=torch.bfloat16), empty(5, 128), empty(1, 5, 4)
    heads = empty(5, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: ctx.quant_fp8(x, q=q, scale=s, stream=Stream()),
                 lambda: ctx.gemm_fp8(q, s, empty(7, 128), empty(1, 1, 4), out=empty(5, 7, dtype=torch.bfloat16), stream=Stream()),
                 lambda: ctx.rope(heads, empty(5, dtype=torch.int32), [1.0], out=heads, stream=Stream())):
        with pytest.raises(ValueError, match="stream must be of device"):
            call()
    assert not calls


def test_binding_refusals_by_message(awa, monkeypatch):
    """Each check of the binding by its own message; no call of them reaches the library."""
    import torch
    ctx, calls = meta_context(awa, monkeypatch)
    bf16, f32, i32, u8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8

    def empty(*shape, dtype=bf16):
        return torch.empty(shape, dtype=dtype, device="meta")

    def refused(match, call, error=ValueError):
        with pytest.raises(error, match=match):
            call()

    # rows
    x = empty(6, 300)
    q, s = ctx.quant_fp8(x)
    calls.clear()
    refused("contiguous columns", lambda: ctx.quant_fp8(empty(300, 6).T))
    refused("contiguous columns", lambda: ctx.quant_fp8(empty(6, 600)[:, ::2]))
    refused("contiguous columns", lambda: ctx.quant_fp8(empty(300)))
    refused("contiguous columns", lambda: ctx.quant_fp8(empty(2, 6, 300)))
    refused("contiguous columns", lambda: ctx.quant_fp8(empty(6, 0)))
    refused("unsupported dtype", lambda: ctx.quant_fp8(empty(6, 300, dtype=torch.float16)), TypeError)
    for t in (empty(6, 300, dtype=u8), empty(5, 384, dtype=u8), empty(6, 384), empty(6, 400, dtype=u8)[:, :384]):
        refused("q must be", lambda: ctx.quant_fp8(x, q=t, scale=s))
    for t in (empty(1, 5, 4, dtype=u8), empty(2, 6, 4, dtype=u8), empty(1, 6, dtype=i32), empty(1, 6, 8, dtype=u8)[..., :4]):
        refused("scale must be", lambda: ctx.quant_fp8(x, q=q, scale=t))
    refused("scale must be", lambda: ctx.quant_fp8(x, blocks=True, q=q, scale=s))

    # the product: 6 x 384 by 130 x 384
    w, ws = empty(130, 384, dtype=u8), empty(1, 2, 4, dtype=u8)
    gemm = ctx.gemm_fp8
    refused(r"a \[M, K\] and w", lambda: gemm(q[0], s, w, ws))
    refused(r"a \[M, K\] and w", lambda: gemm(q, s, w[0], ws))
    refused("a must be", lambda: gemm(empty(6, 384), s, w, ws))
    refused("a must be", lambda: gemm(empty(12, 384, dtype=u8)[::2], s, w, ws))
    refused("w must be", lambda: gemm(q, s, empty(130, 256, dtype=u8), ws))
    refused("w must be", lambda: gemm(q, s, empty(130, 400, dtype=u8)[:, :384], ws))
    refused("w must be", lambda: gemm(q, s, empty(130, 384), ws))
    for t in (empty(1, 5, 4, dtype=u8), empty(2, 6, 4, dtype=u8), empty(1, 6, 4), empty(1, 6, dtype=i32)):
        refused("a_scale must be a", lambda: gemm(q, t, w, ws))
    for t in (empty(1, 6, 8, dtype=u8)[..., :4], empty(1, 12, 4, dtype=u8)[:, ::2], empty(1, 4, 6, dtype=u8).transpose(1, 2)):
        refused("a_scale must be whole words", lambda: gemm(q, t, w, ws))
    refused("w_scale must be a", lambda: gemm(q, s, w, empty(1, 130, 4, dtype=u8)))
    refused("w_scale must be whole words", lambda: gemm(q, s, w, empty(1, 4, 4, dtype=u8)[:, ::2]))
    wide = empty(6, 640, dtype=u8), empty(130, 640, dtype=u8), empty(2, 2, 4, dtype=u8)
    for t in (torch.empty_strided((2, 6, 4), (26, 4, 1), dtype=u8, device="meta"),
              torch.empty_strided((2, 6, 4), (20, 4, 1), dtype=u8, device="meta")):  # no whole words, groups that overlap
        refused("a_scale must be whole words", lambda: gemm(wide[0], t, *wide[1:]))
    for t in (empty(130), empty(129, dtype=f32), empty(1, 130, dtype=f32), empty(260, dtype=f32)[::2]):
        refused("bias must be", lambda: gemm(q, s, w, ws, bias=t))
    for t in (empty(6, 129), empty(5, 130), empty(130, 6).T, empty(6, 260)[:, ::2], empty(780)):
        refused("out must be", lambda: gemm(q, s, w, ws, out=t))
    refused("out must be", lambda: gemm(q, s, w, ws, out=empty(6, 130), dtype=f32))
    refused("unsupported dtype", lambda: gemm(q, s, w, ws, out=empty(6, 130, dtype=torch.float16)), TypeError)
    refused("unsupported dtype", lambda: gemm(q, s, w, ws, dtype=torch.float16), TypeError)

    # rotation: 6 tokens of 3 heads of 64
    x, pos, f = empty(6, 3, 64), empty(6, dtype=i32), [1.0] * 32

    def rope(x=x, pos=pos, f=f, **args):
        return lambda: ctx.rope(x, pos, f, **args)

    refused("one or two tensors", rope((x, x, x)))
    refused("one or two tensors", rope(()))
    refused("one or two tensors", rope((x, x), out=x))
    refused("one or two tensors", rope(x, out=(x, x)))
    refused(r"must be \[tokens, heads, head_d\]", rope(x[0]))
    refused(r"must be \[tokens, heads, head_d\] of one dtype", rope(empty(6, 3, 128)[..., ::2]))
    for t in (empty(5, 3, 64), empty(6, 3, 32), empty(6, 3, 64, dtype=f32), empty(6, 192), empty(6, 64, 3).transpose(1, 2)):
        refused(r"must be \[tokens, heads, head_d\] of one dtype", rope((x, t)))
    for t in (empty(6, dtype=torch.int64), empty(5, dtype=i32), empty(12, dtype=i32)[::2], empty(6, 1, 1, dtype=i32),
              empty(1, 6, dtype=i32).T.expand(6, 2)):
        refused("positions must be", rope(pos=t))
    refused("must name each axis", rope(pairs=(16, 16)))
    refused("must name each axis", rope(pairs=(31,)))
    refused("must name each axis", rope(pos=empty(6, 3, dtype=i32), pairs=(16, 16)))
    refused("must name each axis", rope(pos=empty(6, 5, dtype=i32), pairs=(8, 8, 8, 4, 4)))
    refused("must name each axis", rope(empty(6, 3, 258), f=[1.0] * 129))
    refused("layout must be", rope(layout="split"))
    for t in (empty(6, 3, 63), empty(6, 3, 64, dtype=f32), empty(6, 3, 128)[..., ::2]):
        refused("out must have", rope(out=t))
    refused("unsupported dtype", rope(empty(6, 3, 64, dtype=torch.float16)), TypeError)

    # each tensor elsewhere than the context's device
    elsewhere = []
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 3 if any(t is e for e in elsewhere) else -1)
    bias, out, turned = empty(130, dtype=f32), empty(6, 130), empty(6, 3, 64)
    rows = empty(6, 300)
    for call, tensors in ((lambda: ctx.quant_fp8(rows, q=q, scale=s), (rows, q, s)),
                          (lambda: gemm(q, s, w, ws, bias=bias, out=out), (q, s, w, ws, bias, out)),
                          (rope(out=turned), (x, pos, turned)), (rope((turned, x)), (x, turned))):
        calls.clear()
        call()
        assert len(calls) == 1
        calls.clear()
        for t in tensors:
            elsewhere[:] = [t]
            refused("must be on device -1", call)
        elsewhere.clear()
    assert not calls


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
