"""Python binding of the C ABI in include/awa_capi.h (ctypes over lib/libseedvr2_awa.so).

This is the binding a Python caller (and the test-suite and bench) uses; the
product is the C ABI itself.  Device buffers are torch tensors on a ROCm
device; the stream is torch's current stream.  There is no fallback: if the
shared library is missing, import fails loudly.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libseedvr2_awa.so")
HEADER_DIR = os.path.join(os.path.dirname(HERE), "include")

AWA_OK, AWA_EARG, AWA_EHIP = 0, -1, -2
AWA_F32, AWA_BF16 = 0, 1
DIT_FP8 = 2
DIT_FP8_WHOLE = DIT_CROSS_WHOLE = 256
HEADS, HEAD_D, DIM, QKV, ROPE_ROT = 20, 128, 2560, 7680, 126

_lib = None
# set by lib(), which imports torch: the module, the 8-bit types that the operators take (values or scales
# first, then plain bytes) and the storage types by torch's
_torch, _e4m3, _e8m0, _storage = None, (), (), {}


class AwaError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"AWA error {code}: {msg}")
        self.code = code


BRANCH_FIELDS = ("qkv_w", "out_w", "out_b", "mlp_w", "mlp_out_w", "nq", "nk", "attn_shift",
                 "attn_scale", "attn_gate", "mlp_shift", "mlp_scale", "mlp_gate")


class DitBranch(C.Structure):
    """dit_branch of include/dit_capi.h (device pointers)."""
    _fields_ = [(n, C.c_void_p) for n in BRANCH_FIELDS]


IO_FIELDS = ("vid_in_w", "vid_in_b", "txt_in_w", "txt_in_b", "out_norm_w", "out_ada_shift",
             "out_ada_scale", "vid_out_w", "vid_out_b")


class DitIoWeights(C.Structure):
    """dit_io_weights of include/dit_capi.h (device pointers)."""
    _fields_ = [(n, C.c_void_p) for n in IO_FIELDS]


class DitTimeWeights(C.Structure):
    """dit_time_weights of include/dit_capi.h (device pointers)."""
    _fields_ = [(n, C.c_void_p) for n in ("w_in", "b_in", "w_hid", "b_hid", "w_out", "b_out")]


# the sizes that include/dit_ops.h accepts; checked here, since ctypes cuts what passes 32 bits
OPS_ROWS_MAX, OPS_COLS_MAX, ROPE_MAX_HEADS = 1 << 24, 1 << 20, 32767
ROPE_MAX_PAIRS, ROPE_MAX_AXES = 128, 4
ROPE_LAYOUTS = {"interleaved": 0, "half": 1}
ROPE_KINDS = {"plain": 0, "linear": 1, "base": 2, "bands": 3}

# and include/dit_train.h
NORM_COLS_MAX, CROSS_SEQ_MAX, CROSS_HEADS_MAX, CROSS_HEAD_D_MAX = 16384, 65536, 1024, 128


# dit_rope_plan of include/dit_ops.h up to its frequencies, and dit_rope_rows
_PLAN = struct.Struct("@7i4xd")
_NO_PAIRS, _NO_FREQS = (0,) * ROPE_MAX_AXES, bytes(8 * ROPE_MAX_PAIRS)
_ROWS = struct.Struct("@PPi4x4q")
_HEADS = struct.Struct("@Pqq")  # dit_heads of include/dit_train.h


class GeomInfo(C.Structure):
    _fields_ = [(n, C.c_int32) for n in
                ("t", "h", "w", "nwin", "sumf", "Lv", "txt_len", "max_S", "n_tiles", "n_items")]


def build():
    """Compile lib/libseedvr2_awa.so with hipcc for gfx950."""
    import subprocess
    subprocess.run(["make", "-s", "-C", HERE, f"-j{min(8, os.cpu_count() or 1)}"], check=True)


def lib():
    global _lib, _torch, _e4m3, _e8m0, _storage
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it (make -C {HERE}) before use")
        # torch ships its own HIP runtime with the same soname
        # (libamdhip64.so.7).  Load it first so the library binds to that one
        # runtime instead of starting a second one from /opt/rocm in the same
        # process: torch's tensors and streams then belong to our runtime too.
        import torch
        L = C.CDLL(LIB_PATH)
        vp, i32p, f32p = C.c_void_p, C.POINTER(C.c_int32), C.POINTER(C.c_float)
        L.awa_create.argtypes = [C.POINTER(vp), C.c_int]
        L.awa_destroy.argtypes = [vp]
        L.awa_destroy.restype = None
        L.awa_last_error.argtypes = [vp]
        L.awa_last_error.restype = C.c_char_p
        L.awa_plan_windows.argtypes = [C.c_int, C.c_int, C.c_int, i32p, C.c_int, i32p, C.c_int]
        L.awa_geom_build.argtypes = [vp, C.c_int, C.c_int, C.c_int, i32p, C.c_int, C.c_int,
                                     C.POINTER(vp), vp]
        L.awa_geom_set.argtypes = [vp, f32p, f32p, f32p, f32p, C.c_int, C.c_int, C.c_int,
                                   C.POINTER(vp), vp]
        L.awa_geom_from_win.argtypes = [vp, C.c_int, C.c_int, C.c_int, C.c_int, i32p, f32p, f32p, C.c_int,
                                        C.POINTER(vp), vp]
        L.awa_geom_query.argtypes = [vp, C.POINTER(GeomInfo)]
        L.awa_geom_read.argtypes = [vp, vp, vp, vp, vp, vp, vp]
        L.awa_geom_destroy.argtypes = [vp]
        L.awa_geom_destroy.restype = None
        L.awa_forward.argtypes = [vp, vp, C.c_int, vp, vp, C.c_int, C.c_int, vp, vp, vp, vp,
                                  C.c_float, vp, vp, vp]
        L.awa_forward_noalloc.argtypes = [vp, vp, C.c_int, vp, vp, C.c_int, C.c_int, vp, vp, vp, vp,
                                          C.c_float, vp, vp, vp]
        L.awa_forward_host.argtypes = [vp, vp, f32p, f32p, C.c_int, C.c_int, f32p, f32p, f32p, f32p,
                                       C.c_float, f32p, f32p]
        L.awa_timing_enable.argtypes = [vp, C.c_int]
        L.awa_timing_read.argtypes = [vp, C.POINTER(C.c_double), C.POINTER(C.c_double),
                                      C.POINTER(C.c_double), C.POINTER(C.c_int)]
        L.dit_pack_mlp_weights.argtypes = [vp, vp, vp, C.c_int, vp, vp]
        L.dit_time_embedding.argtypes = [vp, C.c_float, vp, vp, vp, vp, vp, vp, vp, vp]
        L.dit_layer_forward.argtypes = [vp, vp, C.POINTER(DitBranch), C.POINTER(DitBranch), vp, C.c_int,
                                        C.c_int, C.c_float, vp, C.c_int, C.c_int, vp]
        L.dit_timing_read.argtypes = [vp, C.POINTER(C.c_double), C.POINTER(C.c_double),
                                      C.POINTER(C.c_double), C.POINTER(C.c_int)]
        L.dit_gemm_bf16.argtypes = [vp, vp, vp, vp, C.c_int, C.c_int, C.c_int, vp]
        L.dit_io_create.argtypes = [vp, C.POINTER(DitIoWeights), C.POINTER(vp), vp]
        L.dit_io_destroy.argtypes = [vp, vp]
        L.dit_io_destroy.restype = None
        L.dit_embed.argtypes = [vp, vp, vp, C.c_int, C.c_int, C.c_int, vp, C.c_int, vp, vp]
        L.dit_final.argtypes = [vp, vp, vp, vp, C.c_int, C.c_int, C.c_int, C.c_float, vp, vp]
        L.dit_host_last_error.restype = C.c_char_p
        L.dit_free_host.argtypes = [vp]
        L.dit_free_host.restype = None
        L.dit_read_raw_f.argtypes = [C.c_char_p, C.POINTER(vp), C.POINTER(C.c_int64), C.POINTER(C.c_int64),
                                     C.POINTER(C.c_int)]
        L.dit_read_linear.argtypes = [C.c_char_p, C.c_int, C.POINTER(vp), C.POINTER(vp), C.POINTER(C.c_int),
                                      C.POINTER(C.c_int)]
        L.dit_read_win.argtypes = [C.c_char_p, C.c_int, C.POINTER(C.c_int64), C.POINTER(vp), C.POINTER(vp),
                                   C.POINTER(C.c_int64), C.POINTER(vp), C.POINTER(C.c_int64)]
        L.dit_model_load.argtypes = [vp, C.c_char_p, C.c_int, C.c_int, C.POINTER(vp), vp]
        L.dit_model_load_graph.argtypes = [vp, C.c_char_p, C.c_char_p, C.c_char_p, C.c_int, C.POINTER(vp), vp]
        L.dit_graph_file_info.argtypes = [C.c_char_p, C.c_char_p, C.c_int, C.POINTER(C.c_int), C.POINTER(C.c_int),
                                          C.POINTER(C.c_int)]
        L.dit_read_graph_weight.argtypes = [C.c_char_p, C.c_char_p, C.c_int, C.c_char_p, C.POINTER(vp),
                                            C.POINTER(vp), C.POINTER(C.c_int), C.POINTER(C.c_int)]
        L.dit_model_info.argtypes = [vp, C.POINTER(C.c_int), C.POINTER(C.c_int), C.POINTER(C.c_int)]
        L.dit_model_forward_grid.argtypes = [vp, vp, vp, vp, C.c_int, C.c_float, C.c_float, vp, C.c_int, C.c_int,
                                             C.c_int, vp, C.c_int, vp, vp, vp]
        L.dit_model_destroy.argtypes = [vp, vp]
        L.dit_model_destroy.restype = None
        L.dit_graph_create.argtypes = [vp, vp, vp, vp, C.c_int, C.c_float, C.c_float, vp, C.c_int, C.c_int,
                                       C.c_int, vp, C.c_int, vp, vp, vp, C.POINTER(vp)]
        L.dit_graph_launch.argtypes = [vp, vp, vp]
        L.dit_graph_destroy.argtypes = [vp]
        L.dit_graph_destroy.restype = None
        L.dit_forward_grid.argtypes = [vp, vp, C.POINTER(DitTimeWeights), C.POINTER(C.POINTER(DitBranch)),
                                       C.POINTER(C.POINTER(DitBranch)), C.c_int, vp, vp, C.c_int, C.c_int,
                                       C.c_float, C.c_float, vp, C.c_int, C.c_int, C.c_int, vp, C.c_int, vp,
                                       vp, vp]
        L.awa_cast_f32_to_bf16.argtypes = [vp, vp, vp, C.c_int64, vp]
        L.awa_cast_bf16_to_f32.argtypes = [vp, vp, vp, C.c_int64, vp]
        L.awa_stream_copy.argtypes = [vp, vp, vp, C.c_int64, vp]
        L.awa_reserve.argtypes = [vp, vp, C.c_int]
        L.dit_reserve.argtypes = [vp, vp, C.c_int]
        L.awa_time_phases.argtypes = [vp, vp, C.c_int, vp, vp, C.c_int, C.c_int, vp, vp, vp, vp,
                                      C.c_float, vp, vp, C.c_int, C.POINTER(C.c_double), vp]
        L.dit_quant_fp8.argtypes = [vp, C.c_int, vp, C.c_int64, C.c_int, C.c_int, C.c_int, vp, vp, C.c_int64, vp]
        L.dit_gemm_fp8.argtypes = [vp, vp, vp, C.c_int64, vp, vp, C.c_int64, vp, C.c_int, vp, C.c_int64, C.c_int,
                                   C.c_int, C.c_int, vp]
        L.dit_rope.argtypes = [vp, C.c_int, C.c_char_p, C.c_int, C.c_int, C.c_int, C.c_char_p, vp, vp]
        i64, i64p = C.c_int64, C.POINTER(C.c_int64)
        L.dit_layer_norm.argtypes = [vp, C.c_int, vp, i64, vp, vp, C.c_float, C.c_int, vp, i64, vp, C.c_int, C.c_int, vp]
        L.dit_layer_norm_grad_work.argtypes = [C.c_int, C.c_int]
        L.dit_layer_norm_grad.argtypes = [vp, C.c_int, vp, i64, C.c_int, vp, i64, vp, i64, vp, vp, C.c_int, vp, i64, vp, vp,
                                          vp, i64, C.c_int, C.c_int, vp]
        L.dit_grad_weight_work.argtypes = 5 * [C.c_int]
        L.dit_grad_weight_fp8.argtypes = [vp, C.c_int, vp, i64, vp, vp, i64, C.c_int, vp, i64, vp, C.c_int, vp, i64, C.c_int,
                                          C.c_int, C.c_int, vp]
        L.dit_cross_create.argtypes = [vp, C.c_int, i64p, i64p, i64p, i64p, C.c_int, C.c_int, C.c_int, C.POINTER(vp)]
        L.dit_cross_destroy.argtypes = [vp]
        L.dit_cross_destroy.restype = None
        L.dit_cross_drop.argtypes = [vp]
        L.dit_cross_drop.restype = None
        L.dit_cross_work.argtypes = [vp, C.c_int, C.c_int]
        L.dit_cross_forward.argtypes = [vp, vp, C.c_int] + 3 * [C.c_char_p] + [vp, C.c_float, C.c_char_p, vp, i64, vp, i64, vp]
        L.dit_cross_grad.argtypes = [vp, vp, C.c_int] + 5 * [C.c_char_p] + [vp, i64, vp, C.c_float] + 3 * [C.c_char_p] + [
            vp, i64, vp]
        for fn in (L.dit_layer_norm_grad_work, L.dit_grad_weight_work, L.dit_cross_work):
            fn.restype = i64
        L.dit_rope_freqs.argtypes = [C.c_int, C.c_int] + 5 * [C.c_double] + [vp]
        _torch, _storage = torch, {torch.float32: AWA_F32, torch.bfloat16: AWA_BF16}
        _e4m3, _e8m0 = (torch.float8_e4m3fn, torch.uint8), (torch.float8_e8m0fnu, torch.uint8)
        _lib = L
    return _lib


def _dtype_of(what, t):
    d = _storage.get(t.dtype)
    if d is None:
        raise TypeError(f"{what}: unsupported dtype {t.dtype}")
    return d


def _host_array(ptr, n, dtype):
    """Copy n values from a dit_* host buffer, then free it."""
    ct = {np.float32: C.c_float, np.int32: C.c_int32}[dtype]
    a = np.ctypeslib.as_array(C.cast(ptr, C.POINTER(ct)), shape=(int(n),)).copy() if n else np.zeros(0, dtype)
    lib().dit_free_host(ptr)
    return a


class HostError(RuntimeError):
    pass


def _host_check(rc, what):
    if rc != 0:
        raise HostError(f"{what}: {lib().dit_host_last_error().decode()}")


def read_raw_f(path):
    """dit_read_raw_f: the array with its stored shape."""
    p, n, nd = C.c_void_p(), C.c_int64(), C.c_int()
    shape = (C.c_int64 * 8)()
    _host_check(lib().dit_read_raw_f(str(path).encode(), C.byref(p), C.byref(n), shape, C.byref(nd)), "dit_read_raw_f")
    return _host_array(p, n.value, np.float32).reshape([shape[i] for i in range(nd.value)])


def read_linear(base, has_bias):
    """dit_read_linear: (W [out][in] float32, bias or None)."""
    w, b, no, ni = C.c_void_p(), C.c_void_p(), C.c_int(), C.c_int()
    _host_check(lib().dit_read_linear(str(base).encode(), int(bool(has_bias)), C.byref(w), C.byref(b),
                                      C.byref(no), C.byref(ni)), "dit_read_linear")
    W = _host_array(w, no.value * ni.value, np.float32).reshape(no.value, ni.value)
    return W, (_host_array(b, no.value, np.float32) if has_bias else None)


def read_win(path, txt_len):
    """dit_read_win: dict with header, slices [nwin][6], vid_freq, txt_freq."""
    hdr = (C.c_int64 * 10)()
    sl, vf, tf = C.c_void_p(), C.c_void_p(), C.c_void_p()
    nv, nt = C.c_int64(), C.c_int64()
    _host_check(lib().dit_read_win(str(path).encode(), int(txt_len), hdr, C.byref(sl), C.byref(vf), C.byref(nv),
                                   C.byref(tf), C.byref(nt)), "dit_read_win")
    nwin = hdr[9]
    return {"header": list(hdr), "slices": _host_array(sl, 6 * nwin, np.int32).reshape(nwin, 6),
            "vid_freq": _host_array(vf, nv.value, np.float32), "txt_freq": _host_array(tf, nt.value, np.float32)}


def graph_file_info(param, bin_path, mm_layers=-1):
    """dit_graph_file_info: (n_layers, mm_layers, distinct weights) of a merged graph."""
    n, mm, nw = C.c_int(), C.c_int(), C.c_int()
    _host_check(lib().dit_graph_file_info(str(param).encode(), str(bin_path).encode(), int(mm_layers), C.byref(n),
                                          C.byref(mm), C.byref(nw)), "dit_graph_file_info")
    return n.value, mm.value, nw.value


def read_graph_weight(param, bin_path, name, mm_layers=-1):
    """dit_read_graph_weight: (W [out][in], bias or None) of a linear weight, or
    (vector, None), by its model-directory name."""
    w, b, no, ni = C.c_void_p(), C.c_void_p(), C.c_int(), C.c_int()
    _host_check(lib().dit_read_graph_weight(str(param).encode(), str(bin_path).encode(), int(mm_layers),
                                            name.encode(), C.byref(w), C.byref(b), C.byref(no), C.byref(ni)),
                "dit_read_graph_weight")
    if ni.value == 0:
        return _host_array(w, no.value, np.float32), None
    W = _host_array(w, no.value * ni.value, np.float32).reshape(no.value, ni.value)
    return W, (_host_array(b, no.value, np.float32) if b.value else None)


def header_symbols():
    """Function names declared in include/*.h."""
    import re
    names = []
    for fn in sorted(os.listdir(HEADER_DIR)):
        if fn.endswith(".h"):
            txt = open(os.path.join(HEADER_DIR, fn)).read()
            txt = re.sub(r"/\*.*?\*/", "", txt, flags=re.S)
            names += re.findall(r"^\s*(?:const\s+)?[A-Za-z_][A-Za-z0-9_]*\s*\**\s+\**([a-z_][a-z0-9_]*)\s*\(",
                                txt, flags=re.M)
    return names


def _ptr(a):
    return C.cast(a.ctypes.data, C.POINTER(C.c_int32)) if a is not None else None


def plan_windows(t, h, w, num_windows, shifted):
    """Host-only window planner (awa_plan_windows): returns int32 [nwin, 6]."""
    nw = np.ascontiguousarray(num_windows, np.int32)
    n = lib().awa_plan_windows(t, h, w, _ptr(nw), int(bool(shifted)), None, 0)
    if n < 0:
        raise AwaError(n, "awa_plan_windows rejected the sizes")
    out = np.zeros((max(n, 1), 6), np.int32)
    lib().awa_plan_windows(t, h, w, _ptr(nw), int(bool(shifted)), _ptr(out), n)
    return out[:n]


def rope_freqs(n, base=10000.0, kind="plain", factor=1.0, trained=0.0, low=1.0, high=32.0):
    """dit_rope_freqs: the radians per position of n channel pairs (float64 [n]), for a
    context stretched by `factor` over a trained length where kind is not "plain"."""
    if kind not in ROPE_KINDS:
        raise ValueError(f"rope_freqs: kind must be one of {list(ROPE_KINDS)}")
    n = min(max(int(n), 0), ROPE_MAX_PAIRS + 1)  # what is out of range stays so
    out = np.empty(n, np.float64)
    rc = lib().dit_rope_freqs(ROPE_KINDS[kind], n, float(base), float(factor), float(trained), float(low),
                              float(high), out.ctypes.data)
    if rc != AWA_OK:
        raise AwaError(rc, "dit_rope_freqs rejected the arguments")
    return out


def fp8_values(q, scale, cols=None):
    """The fp32 values of an 8-bit matrix as quant_fp8 returns it (either form), cut to `cols` columns."""
    import torch
    rows, kp = q.shape
    s = scale.view(torch.uint8).transpose(0, 1).flatten(1)[:, :kp // 128].int() - 127
    s = s if s.shape[0] == rows else s.repeat_interleave(128, 0)[:rows]
    v = torch.ldexp(q.view(torch.float8_e4m3fn).float().unflatten(1, (-1, 128)), s[:, :, None]).flatten(1)
    return v if cols is None else v[:, :cols]


def _address(*tensors):
    return [t.data_ptr() if t is not None else None for t in tensors]


def _work_of(t):
    """Address and bytes of a call's workspace."""
    return (t.data_ptr(), t.numel()) if t is not None else (None, 0)


def _stream_ptr(stream=None):
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


class Context:
    """awa_ctx: one per device and stream (owns the op's scratch)."""

    def __init__(self, device=0):
        self.ptr = C.c_void_p()
        rc = lib().awa_create(C.byref(self.ptr), int(device))
        if rc != AWA_OK:
            raise AwaError(rc, f"awa_create(device={device}) failed")
        self.device = int(device)
        self._on = _torch.device("cuda", self.device)

    def error(self):
        return lib().awa_last_error(self.ptr).decode()

    def check(self, rc, what):
        if rc != AWA_OK:
            raise AwaError(rc, f"{what}: {self.error()}")

    def close(self):
        if self.ptr:
            lib().awa_destroy(self.ptr)
            self.ptr = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- timing
    def timing(self, enable=True):
        self.check(lib().awa_timing_enable(self.ptr, int(bool(enable))), "awa_timing_enable")

    def timing_read(self):
        """Summed per-phase ms since the last read: (pack, attention, text, calls)."""
        a, b, c = C.c_double(), C.c_double(), C.c_double()
        n = C.c_int()
        self.check(lib().awa_timing_read(self.ptr, C.byref(a), C.byref(b), C.byref(c), C.byref(n)),
                   "awa_timing_read")
        return a.value, b.value, c.value, n.value

    # ---- geometry
    def build_geometry(self, t, h, w, num_windows, txt_len, shifted, stream=None):
        g = C.c_void_p()
        nw = np.ascontiguousarray(num_windows, np.int32)
        rc = lib().awa_geom_build(self.ptr, t, h, w, _ptr(nw), txt_len, int(bool(shifted)),
                                  C.byref(g), _stream_ptr(stream))
        self.check(rc, "awa_geom_build")
        return Geometry(self, g)

    def set_geometry(self, vidx, cumf, vfreq, tfreq, nwin, Lv, txt_len, stream=None):
        """AwaLayer::set_window_geometry with the reference's float-encoded arrays."""
        arrs = [np.ascontiguousarray(a, np.float32) for a in (vidx, cumf, vfreq, tfreq)]
        fp = [a.ctypes.data_as(C.POINTER(C.c_float)) for a in arrs]
        g = C.c_void_p()
        rc = lib().awa_geom_set(self.ptr, *fp, int(nwin), int(Lv), int(txt_len), C.byref(g),
                                _stream_ptr(stream))
        self.check(rc, "awa_geom_set")
        return Geometry(self, g)

    def geometry_from_win(self, t, h, w, slices, vid_freq, txt_freq, txt_len, stream=None):
        """awa_geom_from_win: a reference Win (grid, nwin x 6 slices, the two
        frequency tables), e.g. as read_win returns a win_*.bin file."""
        sl = np.ascontiguousarray(slices, np.int32).reshape(-1, 6)
        vf = np.ascontiguousarray(vid_freq, np.float32)
        tf = np.ascontiguousarray(txt_freq, np.float32)
        sizes = np.clip(sl[:, 1::2] - sl[:, 0::2], 0, None).prod(axis=1)
        if vf.size != int(sizes.sum()) * ROPE_ROT or tf.size != sl.shape[0] * int(txt_len) * ROPE_ROT:
            raise ValueError("geometry_from_win: frequency tables do not match the windows")
        g = C.c_void_p()
        rc = lib().awa_geom_from_win(self.ptr, int(t), int(h), int(w), sl.shape[0], _ptr(sl),
                                     vf.ctypes.data_as(C.POINTER(C.c_float)),
                                     tf.ctypes.data_as(C.POINTER(C.c_float)), int(txt_len), C.byref(g),
                                     _stream_ptr(stream))
        self.check(rc, "awa_geom_from_win")
        return Geometry(self, g)

    # ---- the op
    def forward(self, geom, vqkv, tqkv, nq_v, nk_v, nq_t, nk_t, eps=1e-5, vattn=None, tattn=None,
                stream=None, noalloc=False):
        """AwaLayer::forward: torch tensors on the device; returns (vattn, tattn).
        noalloc=True calls awa_forward_noalloc (the library's fixed device
        scratch instead of the context's)."""
        import torch
        if vqkv.dtype == torch.bfloat16:
            dtype = AWA_BF16
        elif vqkv.dtype == torch.float32:
            dtype = AWA_F32
        else:
            raise TypeError(f"unsupported dtype {vqkv.dtype}")
        if tqkv.dtype != vqkv.dtype:
            raise TypeError("vqkv and tqkv must share a dtype")
        for t_ in (vqkv, tqkv):
            if not t_.is_cuda or not t_.is_contiguous():
                raise ValueError("inputs must be contiguous device tensors")
        Lv, TXT = vqkv.shape[0], tqkv.shape[0]
        if vqkv.shape[1] != QKV or tqkv.shape[1] != QKV:
            raise ValueError("rows must have 7680 columns (q|k|v)")
        gains = [g.to(device=vqkv.device, dtype=torch.float32).contiguous() for g in (nq_v, nk_v, nq_t, nk_t)]
        if vattn is None:
            vattn = torch.empty((Lv, DIM), dtype=vqkv.dtype, device=vqkv.device)
        if tattn is None:
            tattn = torch.empty((TXT, DIM), dtype=vqkv.dtype, device=vqkv.device)
        fn = lib().awa_forward_noalloc if noalloc else lib().awa_forward
        rc = fn(self.ptr, geom.ptr, dtype, C.c_void_p(vqkv.data_ptr()),
                               C.c_void_p(tqkv.data_ptr()), Lv, TXT,
                               *[C.c_void_p(g.data_ptr()) for g in gains], float(eps),
                               C.c_void_p(vattn.data_ptr()), C.c_void_p(tattn.data_ptr()),
                               _stream_ptr(stream))
        self.check(rc, "awa_forward_noalloc" if noalloc else "awa_forward")
        self._keep = gains  # alive until the stream consumed them
        return vattn, tattn

    def time_phases(self, geom, vqkv, tqkv, nq_v, nk_v, nq_t, nk_t, reps, eps=1e-5, vattn=None,
                    tattn=None, stream=None):
        """awa_time_phases: the op, then each of its kernels (pack, attention,
        text average) `reps` more times back to back between two events;
        returns the mean ms per launch of each, (pack, attention, text)."""
        import torch
        dtype = AWA_BF16 if vqkv.dtype == torch.bfloat16 else AWA_F32
        Lv, TXT = vqkv.shape[0], tqkv.shape[0]
        gains = [g.to(device=vqkv.device, dtype=torch.float32).contiguous() for g in (nq_v, nk_v, nq_t, nk_t)]
        if vattn is None:
            vattn = torch.empty((Lv, DIM), dtype=vqkv.dtype, device=vqkv.device)
        if tattn is None:
            tattn = torch.empty((TXT, DIM), dtype=vqkv.dtype, device=vqkv.device)
        ms = (C.c_double * 3)()
        rc = lib().awa_time_phases(self.ptr, geom.ptr, dtype, C.c_void_p(vqkv.data_ptr()),
                                   C.c_void_p(tqkv.data_ptr()), Lv, TXT,
                                   *[C.c_void_p(g.data_ptr()) for g in gains], float(eps),
                                   C.c_void_p(vattn.data_ptr()), C.c_void_p(tattn.data_ptr()), int(reps),
                                   ms, _stream_ptr(stream))
        self.check(rc, "awa_time_phases")
        return ms[0], ms[1], ms[2]

    # ---- boundary casts
    def cast_f32_to_bf16(self, src, out, stream=None):
        """awa_cast_f32_to_bf16: fp32 device tensor -> 16-bit device tensor (bf16 bits)."""
        if src.numel() != out.numel() or src.element_size() != 4 or out.element_size() != 2:
            raise ValueError("cast_f32_to_bf16: 4-byte source and 2-byte output of one size")
        rc = lib().awa_cast_f32_to_bf16(self.ptr, C.c_void_p(src.data_ptr()), C.c_void_p(out.data_ptr()),
                                        src.numel(), _stream_ptr(stream))
        self.check(rc, "awa_cast_f32_to_bf16")
        return out

    def cast_bf16_to_f32(self, src, out, stream=None):
        """awa_cast_bf16_to_f32: 16-bit device tensor (bf16 bits) -> fp32 device tensor."""
        if src.numel() != out.numel() or src.element_size() != 2 or out.element_size() != 4:
            raise ValueError("cast_bf16_to_f32: 2-byte source and 4-byte output of one size")
        rc = lib().awa_cast_bf16_to_f32(self.ptr, C.c_void_p(src.data_ptr()), C.c_void_p(out.data_ptr()),
                                        src.numel(), _stream_ptr(stream))
        self.check(rc, "awa_cast_bf16_to_f32")
        return out

    def stream_copy(self, src, out, stream=None):
        """awa_stream_copy: device copy of src's bytes into out (the HBM ceiling's copy kernel)."""
        nb = src.numel() * src.element_size()
        if out.numel() * out.element_size() != nb or not (src.is_contiguous() and out.is_contiguous()):
            raise ValueError("stream_copy: contiguous source and output of one byte size")
        rc = lib().awa_stream_copy(self.ptr, C.c_void_p(out.data_ptr()), C.c_void_p(src.data_ptr()), nb,
                                   _stream_ptr(stream))
        self.check(rc, "awa_stream_copy")
        return out

    # ---- the DiT block (include/dit_capi.h)
    def gemm(self, A, W, out=None, stream=None):
        """C = A W^T, bf16 [M,K] x [N,K] -> [M,N] bf16 (the block's GEMM kernel)."""
        import torch
        M, K = A.shape
        N = W.shape[0]
        if out is None:
            out = torch.empty((M, N), dtype=torch.bfloat16, device=A.device)
        rc = lib().dit_gemm_bf16(self.ptr, C.c_void_p(A.data_ptr()), C.c_void_p(W.data_ptr()),
                                 C.c_void_p(out.data_ptr()), M, N, K, _stream_ptr(stream))
        self.check(rc, "dit_gemm_bf16")
        return out

    def pack_mlp(self, w_in, w_gate, stream=None):
        import torch
        mlp = w_in.shape[0]
        out = torch.empty((2 * mlp, w_in.shape[1]), dtype=torch.bfloat16, device=w_in.device)
        rc = lib().dit_pack_mlp_weights(self.ptr, C.c_void_p(w_in.data_ptr()), C.c_void_p(w_gate.data_ptr()),
                                        mlp, C.c_void_p(out.data_ptr()), _stream_ptr(stream))
        self.check(rc, "dit_pack_mlp_weights")
        return out

    def time_embedding(self, t, w_in, b_in, w_hid, b_hid, w_out, b_out, stream=None):
        import torch
        emb = torch.empty(15360, dtype=torch.float32, device=w_in.device)
        ts = (w_in, b_in, w_hid, b_hid, w_out, b_out)
        rc = lib().dit_time_embedding(self.ptr, float(t), *[C.c_void_p(x.data_ptr()) for x in ts],
                                      C.c_void_p(emb.data_ptr()), _stream_ptr(stream))
        self.check(rc, "dit_time_embedding")
        return emb

    # ---- operators around a projection in 8 bits (include/dit_ops.h)
    # stream= (default: the current stream of the context's device) orders nothing: the caller lets that stream wait
    # for what made a call's tensors, and waits for it before reading results or changing inputs.  Tensors may be
    # dropped as soon as a call returns: their memory is marked as used on its stream.
    def _stream(self, stream):
        """The stream of a call: the given one, else the current one of the context's device."""
        if stream is None:
            return _torch._C._cuda_getCurrentRawStream(self.device)
        if stream.device_index != self.device:
            raise ValueError(f"stream must be of device {self.device}, got {stream.device}")
        return stream.cuda_stream

    def _empty(self, dtype, stream, *shape):
        """A result, from the memory of the stream that writes it.  Where that is not the current stream, which
        will read it, it is marked as used there too."""
        if stream is None:
            return _torch.empty(*shape, dtype=dtype, device=self._on)
        self._stream(stream)
        current = _torch.cuda.current_stream(self.device)
        with _torch.cuda.stream(stream):
            t = _torch.empty(*shape, dtype=dtype, device=self._on)
        t.record_stream(current)
        return t

    def _used(self, stream, *tensors):
        """Keeps the memory of a call's tensors from other use until the given stream has passed the call."""
        self._stream(stream)
        for t in tensors:
            if t is not None:
                t.record_stream(stream)

    def _too_large(self, what, *sizes):
        return ValueError(f"{what}: at most {OPS_ROWS_MAX} rows and {OPS_COLS_MAX} columns, got {list(sizes)}")

    def _elsewhere(self, what, t):
        return ValueError(f"{what}: tensors must be on device {self.device}, got {t.device}")

    def _bytes_of(self, what, t, name, kind, *shape):
        """t is a contiguous tensor of this shape of the given 8-bit type (or of plain bytes) on the context's device."""
        if t.dtype not in kind or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be a contiguous {str(kind[0])[6:]} tensor {list(shape)}, got "
                             f"{str(t.dtype)[6:]} {list(t.shape)} with strides {t.stride()}")
        if t.get_device() != self.device:
            raise self._elsewhere(what, t)

    def _scale_ld(self, what, t, name, groups, rows):
        """Words from group to group of a scale tensor [groups, rows, 4], cut from a wider one or not."""
        if t.dtype not in _e8m0 or t.shape != (groups, rows, 4):
            raise ValueError(f"{what}: {name} must be a {str(_e8m0[0])[6:]} tensor [{groups}, {rows}, 4], got "
                             f"{str(t.dtype)[6:]} {list(t.shape)}")
        if t.get_device() != self.device:
            raise self._elsewhere(what, t)
        if t.is_contiguous():
            return rows
        g, r, b = t.stride()
        if b != 1 or (rows > 1 and r != 4) or g % 4 or g < 4 * rows:
            raise ValueError(f"{what}: {name} must be whole words of contiguous rows, got strides {t.stride()}")
        return g // 4

    def quant_fp8(self, x, blocks=False, q=None, scale=None, stream=None):
        """dit_quant_fp8: x [rows, cols] bf16 or fp32 (columns contiguous) to (q, scale): q float8_e4m3fn
        [rows, cols padded to 128], scale float8_e8m0fnu [groups of four column blocks, rows, 4] (blocks=True:
        a scale per 128 x 128 values, [groups, ceil(rows / 128), 4])."""
        lib_ = lib()
        dtype = _dtype_of("quant_fp8", x)
        shape, st = x.shape, x.stride()
        rows, cols = shape if len(shape) == 2 else (0, 0)
        if cols < 1 or (cols > 1 and st[1] != 1):
            raise ValueError("quant_fp8: x must be [rows, cols] with contiguous columns")
        if rows > OPS_ROWS_MAX or cols > OPS_COLS_MAX:
            raise self._too_large("quant_fp8", rows, cols)
        if x.get_device() != self.device:
            raise self._elsewhere("quant_fp8", x)
        kp, groups, srows = (cols + 127) // 128 * 128, (cols + 511) // 512, (rows + 127) // 128 if blocks else rows
        if q is None:
            q = self._empty(_e4m3[0], stream, rows, kp)
        else:
            self._bytes_of("quant_fp8", q, "q", _e4m3, rows, kp)
        if scale is None:
            scale = self._empty(_e8m0[0], stream, groups, srows, 4)
        else:
            self._bytes_of("quant_fp8", scale, "scale", _e8m0, groups, srows, 4)
        if rows:
            if stream is not None:
                self._used(stream, x, q, scale)
            rc = lib_.dit_quant_fp8(self.ptr, dtype, x.data_ptr(), st[0], rows, cols, 128 if blocks else 1,
                                    q.data_ptr(), scale.data_ptr(), srows, self._stream(stream))
            if rc:
                self.check(rc, "dit_quant_fp8")
        return q, scale

    def gemm_fp8(self, a, a_scale, w, w_scale, bias=None, out=None, dtype=None, stream=None, whole=False):
        """dit_gemm_fp8: [M, N] = A W^T (+ bias fp32 [N]) of matrices as quant_fp8 returns them, A by rows and W
        with blocks=True, or of rows cut from them (a[i:j], a_scale[:, i:j]); `dtype` bf16 (default) or fp32, or that
        of `out` (rows may be strided).  whole=True (DIT_FP8_WHOLE): for bf16 too, sums as exact as those of fp32
        results, in their time."""
        lib_ = lib()
        shape, wshape = a.shape, w.shape
        if len(shape) != 2 or len(wshape) != 2:
            raise ValueError("gemm_fp8: a [M, K] and w [N, K]")
        M, K = shape
        N = wshape[0]
        if M > OPS_ROWS_MAX or N > OPS_COLS_MAX or K > OPS_COLS_MAX:
            raise self._too_large("gemm_fp8", M, N, K)
        groups, nb = (K + 511) // 512, (N + 127) // 128
        dev = self.device
        if not (a.dtype in _e4m3 and w.dtype in _e4m3 and wshape[1] == K and a.is_contiguous() and w.is_contiguous() and
                a.get_device() == dev and w.get_device() == dev):
            self._bytes_of("gemm_fp8", a, "a", _e4m3, M, K)
            self._bytes_of("gemm_fp8", w, "w", _e4m3, N, K)
        ld_as = self._scale_ld("gemm_fp8", a_scale, "a_scale", groups, M)
        ld_ws = self._scale_ld("gemm_fp8", w_scale, "w_scale", groups, nb)
        if out is None:
            out = self._empty(dtype or _torch.bfloat16, stream, M, N)
        elif out.shape != (M, N) or (N > 1 and out.stride(1) != 1) or (dtype or out.dtype) != out.dtype:
            raise ValueError(f"gemm_fp8: out must be [{M}, {N}] of dtype {dtype} with contiguous columns")
        elif out.get_device() != self.device:
            raise self._elsewhere("gemm_fp8", out)
        ct = _dtype_of("gemm_fp8", out)
        if bias is not None:
            if bias.dtype != _torch.float32 or bias.shape != (N,) or not bias.is_contiguous():
                raise ValueError(f"gemm_fp8: bias must be a contiguous fp32 tensor [{N}]")
            if bias.get_device() != self.device:
                raise self._elsewhere("gemm_fp8", bias)
        if M:
            if stream is not None:
                self._used(stream, a, a_scale, w, w_scale, bias, out)
            rc = lib_.dit_gemm_fp8(self.ptr, a.data_ptr(), a_scale.data_ptr(), ld_as, w.data_ptr(), w_scale.data_ptr(), ld_ws,
                                   bias.data_ptr() if bias is not None else None, ct | DIT_FP8_WHOLE if whole else ct,
                                   out.data_ptr(), out.stride(0), M, N, K, self._stream(stream))
            if rc:
                self.check(rc, "dit_gemm_fp8")
        return out

    def rope(self, x, positions, freqs, pairs=None, layout="interleaved", scale=1.0, inverse=False, out=None,
             stream=None):
        """dit_rope: x [tokens, heads, head_d] (or a pair of such tensors, queries and keys; channels contiguous)
        rotated at positions int32 [tokens] or [tokens, axes].  freqs: radians per position of each pair
        (rope_freqs, float64), axis after axis; pairs: how many belong to each axis.  inverse=True is the adjoint,
        which takes gradients of the output to those of the input.  out: x itself for a rotation in place."""
        lib_ = lib()
        many = isinstance(x, (tuple, list))
        xs = x if many else (x,)
        outs = (None,) * len(xs) if out is None else out if isinstance(out, (tuple, list)) else (out,)
        if not 1 <= len(xs) <= 2 or len(outs) != len(xs):
            raise ValueError("rope: one or two tensors, and as many outputs")
        first = xs[0]
        dtype = _dtype_of("rope", first)
        shape = first.shape
        if len(shape) != 3:
            raise ValueError("rope: tensors must be [tokens, heads, head_d]")
        tokens, _, head_d = shape
        if tokens > OPS_ROWS_MAX:
            raise self._too_large("rope", tokens)
        f = np.ascontiguousarray(freqs, np.float64)
        n, at = f.size, positions.shape
        axes = at[1] if len(at) == 2 else 1
        pairs = (n,) if pairs is None else tuple(pairs)
        if positions.dtype != _torch.int32 or not 1 <= len(at) <= 2 or at[0] != tokens or not positions.is_contiguous():
            raise ValueError(f"rope: positions must be contiguous int32 [{tokens}] or [{tokens}, axes]")
        if len(pairs) != axes or axes > ROPE_MAX_AXES or sum(pairs) != n or n > ROPE_MAX_PAIRS:
            raise ValueError(f"rope: pairs {pairs} must name each axis of the positions and sum to the {n} freqs")
        if layout not in ROPE_LAYOUTS:
            raise ValueError(f"rope: layout must be one of {list(ROPE_LAYOUTS)}")
        if positions.get_device() != self.device:
            raise self._elsewhere("rope", positions)
        plan = b"".join((_PLAN.pack(ROPE_LAYOUTS[layout], axes, *pairs, *_NO_PAIRS[axes:], 1 if inverse else 0, scale),
                         f.tobytes(), _NO_FREQS[8 * n:]))
        rows, res = b"", []
        for t, o in zip(xs, outs):
            shape, ts = t.shape, t.stride()
            if len(shape) != 3 or t.dtype != first.dtype or shape[0] != tokens or shape[2] != head_d or (
                    head_d > 1 and ts[2] != 1):
                raise ValueError("rope: tensors must be [tokens, heads, head_d] of one dtype with contiguous channels")
            if shape[1] > ROPE_MAX_HEADS:
                raise ValueError(f"rope: at most {ROPE_MAX_HEADS} heads, got {shape[1]}")
            if o is None:
                o = self._empty(t.dtype, stream, *shape)
            elif o.shape != shape or o.dtype != t.dtype or (head_d > 1 and o.stride(2) != 1):
                raise ValueError("rope: out must have x's shape and dtype and contiguous channels")
            if t.get_device() != self.device or o.get_device() != self.device:
                raise self._elsewhere("rope", t)
            res.append(o)
            os_ = o.stride()
            rows += _ROWS.pack(t.data_ptr(), o.data_ptr(), shape[1], ts[0], ts[1], os_[0], os_[1])
        if stream is not None:
            self._used(stream, positions, *xs, *res)
        rc = lib_.dit_rope(self.ptr, dtype, rows, len(xs), tokens, head_d, plan, positions.data_ptr(),
                           self._stream(stream))
        if rc:
            self.check(rc, "dit_rope")
        return tuple(res) if many else res[0]

    # ---- operators that train a layer (include/dit_train.h); streams as above
    def _rows_of(self, what, t, name, rows=None, cols=None):
        """(dtype, elements from row to row) of t [rows, cols] with contiguous columns on the context's device."""
        dtype, shape, st = _dtype_of(what, t), t.shape, t.stride()
        if len(shape) != 2 or shape[1] < 1 or (shape[1] > 1 and st[1] != 1) or (
                rows is not None and (shape[0] != rows or shape[1] != cols)):
            raise ValueError(f"{what}: {name} must be [{'rows' if rows is None else rows}, {'cols' if cols is None else cols}] "
                             f"with contiguous columns, got {list(shape)} with strides {st}")
        if t.get_device() != self.device:
            raise self._elsewhere(what, t)
        return dtype, st[0]

    def _vector(self, what, t, name, *shape):
        """The address of a contiguous fp32 tensor of this shape, or None."""
        if t is None:
            return None
        if t.dtype != _torch.float32 or t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be a contiguous fp32 tensor {list(shape)}")
        if t.get_device() != self.device:
            raise self._elsewhere(what, t)
        return t.data_ptr()

    def layer_norm(self, x, weight=None, bias=None, eps=1e-5, dtype=None, out=None, stats=False, stream=None):
        """dit_layer_norm: each row of x [rows, cols] (bf16 or fp32, columns contiguous) normalised, times weight plus bias
        (fp32 [cols]); `dtype` of the result (default x's), or that of `out` (x itself: in place).  stats=True: (y, stats),
        each row's mean and rstd (fp32 [rows, 2]), which layer_norm_grad takes; a tensor is written."""
        lib_ = lib()
        dx, ldx = self._rows_of("layer_norm", x, "x")
        rows, cols = x.shape
        if rows > OPS_ROWS_MAX or cols > NORM_COLS_MAX:
            raise ValueError(f"layer_norm: at most {OPS_ROWS_MAX} rows and {NORM_COLS_MAX} columns, got {[rows, cols]}")
        w, b = self._vector("layer_norm", weight, "weight", cols), self._vector("layer_norm", bias, "bias", cols)
        if out is None:
            out = self._empty(dtype or x.dtype, stream, rows, cols)
        elif (dtype or out.dtype) != out.dtype:
            raise ValueError(f"layer_norm: out must be of dtype {dtype}")
        dy, ldy = self._rows_of("layer_norm", out, "out", rows, cols)
        st = self._empty(_torch.float32, stream, rows, 2) if stats is True else stats if stats is not False else None
        sp = self._vector("layer_norm", st, "stats", rows, 2)
        if rows:
            if stream is not None:
                self._used(stream, x, weight, bias, out, st)
            rc = lib_.dit_layer_norm(self.ptr, dx, x.data_ptr(), ldx, w, b, eps, dy, out.data_ptr(), ldy, sp, rows, cols,
                                     self._stream(stream))
            if rc:
                self.check(rc, "dit_layer_norm")
        return out if st is None else (out, st)

    def layer_norm_grad(self, dy, x, stats, weight=None, x_scale=None, params=True, dtype=None, dx=None, stream=None):
        """dit_layer_norm_grad: (dx, dweight, dbias) for the gradient dy [rows, cols] of layer_norm's result, its input x
        (bf16, fp32, or 8-bit rows and x_scale as quant_fp8 returns them) and stats.  params=False: dx alone, the others
        None.  `dtype` of dx (default x's, bf16 for 8-bit rows), or that of the given `dx` (dy or x itself: in place)."""
        lib_ = lib()
        what = "layer_norm_grad"
        ddy, lddy = self._rows_of(what, dy, "dy")
        rows, cols = dy.shape
        if rows > OPS_ROWS_MAX or cols > NORM_COLS_MAX:
            raise ValueError(f"{what}: at most {OPS_ROWS_MAX} rows and {NORM_COLS_MAX} columns, got {[rows, cols]}")
        if x_scale is None:
            dtx, ldx = self._rows_of(what, x, "x", rows, cols)
            xs, ld_xs = None, 0
        else:
            self._bytes_of(what, x, "x", _e4m3, rows, (cols + 127) // 128 * 128)
            dtx, ldx = DIT_FP8, 0
            xs, ld_xs = x_scale.data_ptr(), self._scale_ld(what, x_scale, "x_scale", (cols + 511) // 512, rows)
        sp, w = self._vector(what, stats, "stats", rows, 2), self._vector(what, weight, "weight", cols)
        if sp is None:
            raise ValueError(f"{what}: stats must be a contiguous fp32 tensor [{rows}, 2]")
        if dx is None:
            dx = self._empty(dtype or (x.dtype if x_scale is None else _torch.bfloat16), stream, rows, cols)
        elif (dtype or dx.dtype) != dx.dtype:
            raise ValueError(f"{what}: dx must be of dtype {dtype}")
        dtd, lddx = self._rows_of(what, dx, "dx", rows, cols)
        dw = db = work = None
        if params:
            dw, db = self._empty(_torch.float32, stream, cols), self._empty(_torch.float32, stream, cols)
            work = self._work(stream, lib_.dit_layer_norm_grad_work(rows, cols))
        if rows or params:
            if stream is not None:
                self._used(stream, dy, x, x_scale, stats, weight, dx, dw, db)
            rc = lib_.dit_layer_norm_grad(self.ptr, ddy, dy.data_ptr(), lddy, dtx, x.data_ptr(), ldx, xs, ld_xs, sp, w, dtd,
                                          dx.data_ptr(), lddx, *_address(dw, db), *_work_of(work), rows, cols,
                                          self._stream(stream))
            if rc:
                self.check(rc, "dit_layer_norm_grad")
        return dx, dw, db

    def grad_weight_fp8(self, dy, x, x_scale, cols=None, bias=False, dtype=None, out=None, add=False, stream=None):
        """dit_grad_weight_fp8: dW [N, cols] = dy^T X for the gradient dy [M, N] (bf16 or fp32) of X W^T and X [M, cols] in
        8-bit rows as quant_fp8 returns them (cols: X's columns, default all that x holds).  `dtype` fp32 (default) or bf16,
        or that of `out` (rows may be strided).  bias=True: (dW, db), dy's sums over the rows (fp32 [N]); a tensor is
        written.  add=True: added to what `out` (fp32) and a given bias hold."""
        lib_ = lib()
        what = "grad_weight_fp8"
        ddy, lddy = self._rows_of(what, dy, "dy")
        M, N = dy.shape
        shape = x.shape
        if len(shape) != 2:
            raise ValueError(f"{what}: x must be [M, K]")
        K = shape[1] if cols is None else cols
        if K < 1 or (K + 127) // 128 * 128 != shape[1]:
            raise ValueError(f"{what}: x of {shape[1]} columns does not hold {K} padded to 128")
        if M > OPS_ROWS_MAX or N > OPS_COLS_MAX or K > OPS_COLS_MAX:
            raise self._too_large(what, M, N, K)
        self._bytes_of(what, x, "x", _e4m3, M, shape[1])
        ld_s = self._scale_ld(what, x_scale, "x_scale", (K + 511) // 512, M)
        if add and (out is None or bias is True):
            raise ValueError(f"{what}: add needs an out, and a tensor for bias, to add to")
        if out is None:
            out = self._empty(dtype or _torch.float32, stream, N, K)
        elif (dtype or out.dtype) != out.dtype:
            raise ValueError(f"{what}: out must be of dtype {dtype}")
        dtw, ldw = self._rows_of(what, out, "out", N, K)
        db = self._empty(_torch.float32, stream, N) if bias is True else bias if bias is not False else None
        bp = self._vector(what, db, "bias", N)
        work = self._work(stream, lib_.dit_grad_weight_work(ddy, dtw, M, N, K))
        if stream is not None:
            self._used(stream, dy, x, x_scale, out, db)
        rc = lib_.dit_grad_weight_fp8(self.ptr, ddy, dy.data_ptr(), lddy, x.data_ptr(), x_scale.data_ptr(), ld_s, dtw,
                                      out.data_ptr(), ldw, bp, 1 if add else 0, *_work_of(work), M, N, K, self._stream(stream))
        if rc:
            self.check(rc, "dit_grad_weight_fp8")
        return out if db is None else (out, db)

    def cross_plan(self, heads, head_d, q_len, k_len, kv_heads=None, q_at=None, k_at=None):
        """dit_cross_create: the lengths of a batch for cross_attn, of each sequence its query rows q_at .. q_at + q_len and key
        rows k_at .. k_at + k_len (host integers; without q_at or k_at sequences follow one another).  Sequences may share
        the same key rows.  Made once for a batch, with a copy to the device (not while a stream is captured)."""
        return CrossPlan(self, heads, head_d, q_len, k_len, kv_heads, q_at, k_at)

    def _heads_of(self, what, plan, t, name, rows, heads, like=None):
        """t as a dit_heads: [rows or more, heads, head_d] with contiguous channels, of like's dtype and shape."""
        shape, st = t.shape, t.stride()
        if len(shape) != 3 or shape[1] != heads or shape[2] != plan.head_d or shape[0] < rows or st[2] != 1:
            raise ValueError(f"{what}: {name} must be [{rows} rows or more, {heads}, {plan.head_d}] with contiguous channels, got "
                             f"{list(shape)} with strides {st}")
        if like is not None and (t.dtype != like.dtype or shape[0] != like.shape[0]):
            raise ValueError(f"{what}: {name} must have {like.shape[0]} rows of {like.dtype}, got {shape[0]} of {t.dtype}")
        if t.get_device() != self.device:
            raise self._elsewhere(what, t)
        # a stride of one thing only does not matter
        return _HEADS.pack(t.data_ptr(), st[0] if shape[0] > 1 else 0, st[1] if heads > 1 else 0)

    def _cross_inputs(self, what, plan, q, k, v, mask, scale):
        dtype = _dtype_of(what, q)
        if plan.device != self.device or not plan.ptr:
            raise ValueError(f"{what}: the plan is of device {plan.device}, or closed; the context is of device {self.device}")
        if k.dtype != q.dtype:
            raise ValueError(f"{what}: q, k and v must have one dtype, got {q.dtype} and {k.dtype}")
        qkv = (self._heads_of(what, plan, q, "q", plan.q_rows, plan.heads),
               self._heads_of(what, plan, k, "k", plan.k_rows, plan.kv_heads),
               self._heads_of(what, plan, v, "v", plan.k_rows, plan.kv_heads, k))
        if mask is not None:
            if mask.dtype not in (_torch.bool, _torch.uint8) or mask.shape != k.shape[:1] or not mask.is_contiguous():
                raise ValueError(f"{what}: mask must be a contiguous bool tensor [{k.shape[0]}]")
            if mask.get_device() != self.device:
                raise self._elsewhere(what, mask)
        return dtype, qkv, mask.data_ptr() if mask is not None else None, plan.head_d ** -0.5 if scale is None else scale

    def cross_attn(self, plan, q, k, v, mask=None, scale=None, out=None, lse=False, stream=None, whole=False):
        """dit_cross_forward: softmax(scale q k^T) v by the plan's sequences, q [rows, heads, head_d] and k, v [rows, kv_heads,
        head_d] (bf16 or fp32, channels contiguous); mask: bool [key rows], False keys take no part; scale: default
        head_d^-0.5.  lse=True: (out, lse), fp32 [heads, query rows], which cross_attn_grad takes; a tensor is written.  Rows of
        no sequence are zeros in results made here and stay as they are in given ones.  whole=True (DIT_CROSS_WHOLE): bf16
        probabilities meet v with 16 bits in place of 8."""
        lib_ = lib()
        what = "cross_attn"
        dtype, qkv, mp, scale = self._cross_inputs(what, plan, q, k, v, mask, scale)
        if out is None:
            out = self._made(q.dtype, stream, plan.q_whole(q.shape[0]), *q.shape)
        op = self._heads_of(what, plan, out, "out", plan.q_rows, plan.heads, q)
        l = lse if lse is not True and lse is not False else None
        if lse is True:
            l = self._made(_torch.float32, stream, plan.q_whole(q.shape[0]), plan.heads, q.shape[0])
        lp = self._vector(what, l, "lse", plan.heads, q.shape[0])
        work = self._work(stream, plan.work(dtype, 0))
        if stream is not None:
            self._used(stream, q, k, v, mask, out, l)
        rc = lib_.dit_cross_forward(self.ptr, plan.ptr, dtype | DIT_CROSS_WHOLE if whole else dtype, *qkv, mp, scale, op, lp,
                                    q.shape[0], *_work_of(work), self._stream(stream))
        if rc:
            self.check(rc, "dit_cross_forward")
        return out if l is None else (out, l)

    def cross_attn_grad(self, plan, dout, q, k, v, out, lse, mask=None, scale=None, dq=None, dk=None, dv=None, stream=None,
                        whole=False):
        """dit_cross_grad: (dq, dk, dv) for the gradient dout of cross_attn's result, from its inputs and results.  Gradients
        of keys are summed over the heads and sequences that share them; rows of no sequence, and whole, as in cross_attn."""
        lib_ = lib()
        what = "cross_attn_grad"
        dtype, qkv, mp, scale = self._cross_inputs(what, plan, q, k, v, mask, scale)
        dop = self._heads_of(what, plan, dout, "dout", plan.q_rows, plan.heads, q)
        op = self._heads_of(what, plan, out, "out", plan.q_rows, plan.heads, q)
        lp = self._vector(what, lse, "lse", plan.heads, q.shape[0])
        if lp is None:
            raise ValueError(f"{what}: lse must be a contiguous fp32 tensor [{plan.heads}, {q.shape[0]}]")
        if dq is None:
            dq = self._made(q.dtype, stream, plan.q_whole(q.shape[0]), *q.shape)
        filled = plan.k_whole(k.shape[0])
        dk = self._made(k.dtype, stream, filled, *k.shape) if dk is None else dk
        dv = self._made(v.dtype, stream, filled, *v.shape) if dv is None else dv
        grads = (self._heads_of(what, plan, dq, "dq", plan.q_rows, plan.heads, q),
                 self._heads_of(what, plan, dk, "dk", plan.k_rows, plan.kv_heads, k),
                 self._heads_of(what, plan, dv, "dv", plan.k_rows, plan.kv_heads, k))
        work = self._work(stream, plan.work(dtype, 1))
        if stream is not None:
            self._used(stream, dout, q, k, v, out, lse, mask, dq, dk, dv)
        rc = lib_.dit_cross_grad(self.ptr, plan.ptr, dtype | DIT_CROSS_WHOLE if whole else dtype, dop, *qkv, op, lp, q.shape[0],
                                 mp, scale, *grads, *_work_of(work), self._stream(stream))
        if rc:
            self.check(rc, "dit_cross_grad")
        return dq, dk, dv

    def _work(self, stream, size):
        """A call's workspace, from the memory of the stream that uses it."""
        if size < 0:
            raise AwaError(AWA_EARG, "workspace of sizes out of range")
        return self._empty(_torch.uint8, stream, size) if size else None

    def _made(self, dtype, stream, whole, *shape):
        """A result; zeros where not every row of it is written."""
        if whole:
            return self._empty(dtype, stream, *shape)
        if stream is None:
            return _torch.zeros(*shape, dtype=dtype, device=self._on)
        t = self._empty(dtype, stream, *shape)
        with _torch.cuda.stream(stream):
            t.zero_()
        return t

    def reserve(self, geom, dtype="bf16"):
        """awa_reserve: size the op's scratch for geom in this storage dtype."""
        self.check(lib().awa_reserve(self.ptr, geom.ptr, AWA_BF16 if dtype == "bf16" else AWA_F32), "awa_reserve")

    def dit_reserve(self, geom, mlp=6912):
        """dit_reserve: size the layer / embed / final workspaces and the op's scratch."""
        self.check(lib().dit_reserve(self.ptr, geom.ptr, int(mlp)), "dit_reserve")

    def layer(self, geom, vbranch, tbranch, emb, x, Lv, TXT, mlp=6912, txt_vid_only=False, eps=1e-5,
              stream=None):
        """dit_layer_forward in place on x (fp32 [Lv+TXT, 2560]).  Branches are dicts of
        device tensors keyed like dit_branch; pass the same dict for shared layers."""
        vb = DitBranch(**{k: vbranch[k].data_ptr() for k in BRANCH_FIELDS})
        tb = vb if tbranch is vbranch else DitBranch(**{k: tbranch[k].data_ptr() for k in BRANCH_FIELDS})
        rc = lib().dit_layer_forward(self.ptr, geom.ptr, C.byref(vb), C.byref(tb),
                                     C.c_void_p(emb.data_ptr()), int(mlp), int(bool(txt_vid_only)),
                                     float(eps), C.c_void_p(x.data_ptr()), int(Lv), int(TXT),
                                     _stream_ptr(stream))
        self.check(rc, "dit_layer_forward")
        return x

    def io_layers(self, weights, stream=None):
        """dit_io_create from a dict of device tensors keyed like dit_io_weights; the
        returned object keeps the tensors alive (the handle borrows some of them)."""
        w = DitIoWeights(**{k: weights[k].data_ptr() for k in IO_FIELDS})
        h = C.c_void_p()
        self.check(lib().dit_io_create(self.ptr, C.byref(w), C.byref(h), _stream_ptr(stream)), "dit_io_create")
        return DitIo(self, h, weights)

    def embed(self, io, grid, txt, x=None, stream=None):
        """dit_embed: grid fp32 (T, H, W, 33), txt fp32 [TXT, 5120] -> x fp32 [Lv+TXT, 2560]."""
        import torch
        T, H, W, _ = grid.shape
        TXT = txt.shape[0]
        Lv = T * (H // 2) * (W // 2)
        if x is None:
            x = torch.empty((Lv + TXT, DIM), dtype=torch.float32, device=grid.device)
        rc = lib().dit_embed(self.ptr, io.ptr, C.c_void_p(grid.data_ptr()), int(T), int(H), int(W),
                             C.c_void_p(txt.data_ptr()), int(TXT), C.c_void_p(x.data_ptr()), _stream_ptr(stream))
        self.check(rc, "dit_embed")
        return x

    def final(self, io, emb, x, T, H, W, eps=1e-5, out=None, stream=None):
        """dit_final: video rows of x -> fp32 (T, H, W, 16)."""
        import torch
        if out is None:
            out = torch.empty((T, H, W, 16), dtype=torch.float32, device=x.device)
        rc = lib().dit_final(self.ptr, io.ptr, C.c_void_p(emb.data_ptr()), C.c_void_p(x.data_ptr()), int(T),
                             int(H), int(W), float(eps), C.c_void_p(out.data_ptr()), _stream_ptr(stream))
        self.check(rc, "dit_final")
        return out

    def forward_grid(self, io, time_w, layers, geom_even, geom_odd, t, grid, txt, mlp=6912,
                     last_txt_vid_only=False, eps=1e-5, x=None, out=None, stream=None):
        """dit_forward_grid.  time_w: 6 device tensors (w_in, b_in, w_hid, b_hid, w_out, b_out);
        layers: list of (video branch dict, text branch dict) of device tensors."""
        import torch
        T, H, W, _ = grid.shape
        TXT = txt.shape[0]
        Lv = T * (H // 2) * (W // 2)
        if x is None:
            x = torch.empty((Lv + TXT, DIM), dtype=torch.float32, device=grid.device)
        if out is None:
            out = torch.empty((T, H, W, 16), dtype=torch.float32, device=grid.device)
        tw = DitTimeWeights(*[w.data_ptr() for w in time_w])
        cache = {}

        def br(d):
            if id(d) not in cache:
                cache[id(d)] = DitBranch(**{k: d[k].data_ptr() for k in BRANCH_FIELDS})
            return cache[id(d)]
        n = len(layers)
        vb = (C.POINTER(DitBranch) * max(n, 1))(*[C.pointer(br(v)) for v, _ in layers])
        tb = (C.POINTER(DitBranch) * max(n, 1))(*[C.pointer(br(t_)) for _, t_ in layers])
        rc = lib().dit_forward_grid(self.ptr, io.ptr, C.byref(tw), vb, tb, n, geom_even.ptr,
                                    geom_odd.ptr if geom_odd is not None else None, int(mlp),
                                    int(bool(last_txt_vid_only)), float(eps), float(t),
                                    C.c_void_p(grid.data_ptr()), int(T), int(H), int(W),
                                    C.c_void_p(txt.data_ptr()), int(TXT), C.c_void_p(x.data_ptr()),
                                    C.c_void_p(out.data_ptr()), _stream_ptr(stream))
        self.check(rc, "dit_forward_grid")
        return out

    def load_model(self, path, n_layers, mm_layers, stream=None):
        """dit_model_load of a model directory in the reference's layout."""
        h = C.c_void_p()
        self.check(lib().dit_model_load(self.ptr, str(path).encode(), int(n_layers), int(mm_layers), C.byref(h),
                                        _stream_ptr(stream)), "dit_model_load")
        return DitModel(self, h)

    def load_graph_model(self, param, bin_path, model_dir=None, mm_layers=-1, stream=None):
        """dit_model_load_graph: a merged whole-model graph (.param/.bin), the
        timestep MLP from model_dir."""
        h = C.c_void_p()
        self.check(lib().dit_model_load_graph(self.ptr, str(param).encode(), str(bin_path).encode(),
                                              str(model_dir).encode() if model_dir is not None else None,
                                              int(mm_layers), C.byref(h), _stream_ptr(stream)),
                   "dit_model_load_graph")
        return DitModel(self, h)

    def model_forward_grid(self, model, geom_even, geom_odd, t, grid, txt, last_txt_vid_only=False, eps=1e-5,
                           x=None, out=None, stream=None):
        import torch
        T, H, W, _ = grid.shape
        TXT = txt.shape[0]
        Lv = T * (H // 2) * (W // 2)
        if x is None:
            x = torch.empty((Lv + TXT, DIM), dtype=torch.float32, device=grid.device)
        if out is None:
            out = torch.empty((T, H, W, 16), dtype=torch.float32, device=grid.device)
        rc = lib().dit_model_forward_grid(self.ptr, model.ptr, geom_even.ptr,
                                          geom_odd.ptr if geom_odd is not None else None,
                                          int(bool(last_txt_vid_only)), float(eps), float(t),
                                          C.c_void_p(grid.data_ptr()), int(T), int(H), int(W),
                                          C.c_void_p(txt.data_ptr()), int(TXT), C.c_void_p(x.data_ptr()),
                                          C.c_void_p(out.data_ptr()), _stream_ptr(stream))
        self.check(rc, "dit_model_forward_grid")
        return out

    def model_graph(self, model, geom_even, geom_odd, t, grid, txt, x, out, last_txt_vid_only=False,
                    eps=1e-5, stream=None):
        """dit_graph_create: model_forward_grid captured for these buffers (run
        once eagerly, so out already holds the result); DitGraph.launch replays it."""
        T, H, W, _ = grid.shape
        h = C.c_void_p()
        rc = lib().dit_graph_create(self.ptr, model.ptr, geom_even.ptr,
                                    geom_odd.ptr if geom_odd is not None else None,
                                    int(bool(last_txt_vid_only)), float(eps), float(t),
                                    C.c_void_p(grid.data_ptr()), int(T), int(H), int(W),
                                    C.c_void_p(txt.data_ptr()), int(txt.shape[0]), C.c_void_p(x.data_ptr()),
                                    C.c_void_p(out.data_ptr()), _stream_ptr(stream), C.byref(h))
        self.check(rc, "dit_graph_create")
        return DitGraph(self, h.value, (model, geom_even, geom_odd, grid, txt, x, out))

    def dit_timing_read(self):
        a, b, c = C.c_double(), C.c_double(), C.c_double()
        n = C.c_int()
        self.check(lib().dit_timing_read(self.ptr, C.byref(a), C.byref(b), C.byref(c), C.byref(n)),
                   "dit_timing_read")
        return a.value, b.value, c.value, n.value

    def forward_host(self, geom, vqkv, tqkv, nq_v, nk_v, nq_t, nk_t, eps=1e-5):
        """AwaVk::forward: numpy fp32 in and out, synchronous."""
        f = lambda a: np.ascontiguousarray(a, np.float32)
        vqkv, tqkv = f(vqkv), f(tqkv)
        g4 = [f(x) for x in (nq_v, nk_v, nq_t, nk_t)]
        Lv, TXT = vqkv.shape[0], tqkv.shape[0]
        vo = np.empty((Lv, DIM), np.float32)
        to = np.empty((TXT, DIM), np.float32)
        P = lambda a: a.ctypes.data_as(C.POINTER(C.c_float))
        rc = lib().awa_forward_host(self.ptr, geom.ptr, P(vqkv), P(tqkv), Lv, TXT, *[P(x) for x in g4],
                                    float(eps), P(vo), P(to))
        self.check(rc, "awa_forward_host")
        return vo, to


class CrossPlan:
    """dit_cross: the lengths of a batch (see Context.cross_plan).  It may be dropped at any time, after its calls were made: its
    tables go with the making of the next plan, and those that a graph captured stay.  close() frees them at once: when the calls
    that use them have finished, graphs are no longer replayed, and no stream is captured."""

    def __init__(self, ctx, heads, head_d, q_len, k_len, kv_heads=None, q_at=None, k_at=None):
        def integers(v, name):
            a = np.asarray(v)
            if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
                raise ValueError(f"cross_plan: {name} must be a list of integers")
            return np.ascontiguousarray(a, np.int64)

        self.ptr = C.c_void_p()
        ql, kl = integers(q_len, "q_len"), integers(k_len, "k_len")
        qa = np.cumsum(ql) - ql if q_at is None else integers(q_at, "q_at")
        ka = np.cumsum(kl) - kl if k_at is None else integers(k_at, "k_at")
        n = ql.size
        if not n == kl.size == qa.size == ka.size:
            raise ValueError("cross_plan: one length and one place of queries and keys for each sequence")
        kv_heads = heads if kv_heads is None else kv_heads
        if n > CROSS_SEQ_MAX or not (0 < kv_heads <= heads <= CROSS_HEADS_MAX) or not 0 < head_d <= CROSS_HEAD_D_MAX:
            raise ValueError(f"cross_plan: at most {CROSS_SEQ_MAX} sequences, {CROSS_HEADS_MAX} heads of {CROSS_HEAD_D_MAX} "
                             f"channels, got {n}, {heads} ({kv_heads} of keys) of {head_d}")
        rc = lib().dit_cross_create(ctx.ptr, n, *[a.ctypes.data_as(C.POINTER(C.c_int64)) for a in (qa, ql, ka, kl)], heads,
                                    kv_heads, head_d, C.byref(self.ptr))
        ctx.check(rc, "dit_cross_create")
        self.device, self.heads, self.kv_heads, self.head_d = ctx.device, heads, kv_heads, head_d
        self.q_rows = int((qa + ql)[ql > 0].max(initial=0))
        self.k_rows = int((ka + kl)[kl > 0].max(initial=0))
        # rows that belong to a sequence (shared keys counted once)
        self._q_count = int(ql.sum())
        self._k_count = int(sum(dict(zip(ka[kl > 0].tolist(), kl[kl > 0].tolist())).values()))
        self._work = {}

    def q_whole(self, rows):
        """Whether every one of so many query rows belongs to a sequence."""
        return self._q_count == rows

    def k_whole(self, rows):
        return self._k_count == rows

    def work(self, dtype, grad):
        """dit_cross_work, asked once."""
        n = self._work.get((dtype, grad))
        if n is None:
            n = self._work[dtype, grad] = lib().dit_cross_work(self.ptr, dtype, grad)
        return n

    def close(self, later=False):
        """Frees the tables; later: when that is safe."""
        if self.ptr:
            (lib().dit_cross_drop if later else lib().dit_cross_destroy)(self.ptr)
            self.ptr = C.c_void_p()

    def __del__(self):
        try:
            self.close(later=True)
        except Exception:
            pass


class Geometry:
    def __init__(self, ctx, ptr):
        self.ctx = ctx
        self.ptr = ptr

    def info(self):
        gi = GeomInfo()
        rc = lib().awa_geom_query(self.ptr, C.byref(gi))
        if rc != AWA_OK:
            raise AwaError(rc, "awa_geom_query")
        return {n: getattr(gi, n) for n, _ in GeomInfo._fields_}

    def read(self):
        i = self.info()
        sl = np.zeros((i["nwin"], 6), np.int32)
        cumf = np.zeros(i["nwin"] + 1, np.int32)
        vidx = np.zeros(i["sumf"], np.int32)
        vf = np.zeros((i["sumf"], ROPE_ROT), np.float32)
        tf = np.zeros((i["nwin"] * i["txt_len"], ROPE_ROT), np.float32)
        rc = lib().awa_geom_read(self.ctx.ptr, self.ptr, *[C.c_void_p(a.ctypes.data) for a in (sl, cumf, vidx, vf, tf)])
        self.ctx.check(rc, "awa_geom_read")
        return {"slices": sl, "cumf": cumf, "vidx": vidx, "vid_freq": vf, "txt_freq": tf}

    def close(self):
        if self.ptr:
            lib().awa_geom_destroy(self.ptr)
            self.ptr = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DitIo:
    """Handle of dit_io_create; destroyed with the object."""

    def __init__(self, ctx, ptr, weights):
        self.ctx, self.ptr, self._weights = ctx, ptr, weights

    def close(self):
        if self.ptr:
            lib().dit_io_destroy(self.ctx.ptr, self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DitGraph:
    """Handle of dit_graph_create; keeps what the graph reads alive."""

    def __init__(self, ctx, ptr, keep):
        self.ctx, self.ptr, self._keep = ctx, ptr, keep

    def launch(self, stream=None):
        self.ctx.check(lib().dit_graph_launch(self.ctx.ptr, self.ptr, _stream_ptr(stream)), "dit_graph_launch")

    def close(self):
        if self.ptr:
            lib().dit_graph_destroy(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DitModel:
    """Handle of dit_model_load; destroyed with the object."""

    def __init__(self, ctx, ptr):
        self.ctx, self.ptr = ctx, ptr

    def info(self):
        a, b, c = C.c_int(), C.c_int(), C.c_int()
        lib().dit_model_info(self.ptr, C.byref(a), C.byref(b), C.byref(c))
        return {"n_layers": a.value, "mm_layers": b.value, "mlp": c.value}

    def close(self):
        if self.ptr:
            lib().dit_model_destroy(self.ctx.ptr, self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
