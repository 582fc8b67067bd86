"""ctypes binding of libdit_hip.so (include/dit_hip.h) for Python callers.

Device memory and streams come from PyTorch-ROCm tensors; every call goes
through the C ABI of the HIP library.  There is no fallback: if the library
is missing or a call fails, a `DtError` is raised.

Shapes follow PyTorch order at this level; `desc()` converts a tensor to the
ggml-ordered `dt_tensor` descriptor (ne[0] = last PyTorch dim).
"""
from __future__ import annotations

import ctypes
import functools
import os
from ctypes import POINTER, c_char_p, c_float, c_int32, c_int64, c_size_t, c_uint32, c_uint64, c_void_p

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libdit_hip.so")

# ggml type ids
F32, F16, Q8_0, Q4_K, I32, BF16 = 0, 1, 8, 12, 26, 30

# dt_tensor.op ids
(OP_NONE, OP_ADD, OP_SUB, OP_MUL, OP_DIV, OP_SCALE, OP_SIGMOID, OP_NORM, OP_RMS_NORM,
 OP_ROPE, OP_CONCAT, OP_CPY, OP_VIEW, OP_FILL, OP_UNARY, OP_MUL_MAT, OP_FLASH_ATTN_EXT, OP_CONV_2D_DIRECT,
 OP_UPSCALE) = range(19)
FLAG_OUTPUT = 1
GRAPH_ALLOC_RUNS_AT = 1

BIN_ADD, BIN_SUB, BIN_MUL, BIN_DIV = range(4)
(UN_SIGMOID, UN_EXP, UN_LOG, UN_SQRT, UN_SIN, UN_COS, UN_SCALE, UN_CLAMP, UN_SILU,
 UN_FILL) = range(10)


class DtError(RuntimeError):
    pass


class DtTensor(ctypes.Structure):
    pass


DtTensor._fields_ = [
    ("type", c_int32),
    ("op", c_int32),
    ("ne", c_int64 * 4),
    ("nb", c_int64 * 4),
    ("data", c_void_p),
    ("op_params", c_int32 * 16),
    ("src", POINTER(DtTensor) * 4),
    ("flags", c_int32),
    ("id", c_int32),
]

# Every exported symbol with (restype, argtypes).
_S = c_void_p
_I64P = POINTER(c_int64)
_SIGS = {
    "dt_last_error": (c_char_p, []),
    "dt_version": (c_char_p, []),
    "dt_adaln_mod": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_void_p, c_void_p, c_void_p,
                               c_int64, c_float, c_int32, _S]),
    "dt_qk_rmsnorm_rope": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                                     c_int64, c_int64, c_int64, c_int64, c_int64, c_void_p,
                                     c_void_p, c_float, c_void_p, c_int64, c_int32, c_int32,
                                     c_float, c_void_p, c_int32, c_int32, _S]),
    "dt_rope_table_fill": (c_int32, [c_void_p, c_int32, c_int32, c_float, c_float, c_float]),
    "dt_swiglu": (c_int32, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int64,
                            c_int64, c_int32, _S]),
    "dt_gated_residual": (c_int32, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p,
                                    c_int64, c_int64, c_int64, c_int32, _S]),
    "dt_qk_rmsnorm_rope_swiglu": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                                            c_int64, c_int64, c_int64, c_int64, c_int64, c_void_p,
                                            c_void_p, c_float, c_void_p, c_int64, c_int32, c_int32,
                                            c_float, c_void_p, c_int32, c_void_p, c_int64, c_void_p,
                                            c_int64, c_void_p, c_int64, c_int64, c_int64, c_int32, _S]),
    "dt_gated_residual_adaln": (c_int32, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_void_p,
                                          c_int64, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                                          c_int64, c_float, c_int32, _S]),
    "dt_dequant": (c_int32, [c_void_p, c_int32, c_int64, c_int64, c_int64, c_void_p, c_int64,
                             c_int32, _S]),
    "dt_groupnorm_workspace_bytes": (c_size_t, [c_int64, c_int64, c_int64, c_int64]),
    "dt_groupnorm_silu": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_void_p,
                                    c_void_p, c_float, c_int32, c_void_p, c_void_p, c_size_t,
                                    c_int32, _S]),
    "dt_groupnorm_silu_noalloc": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_void_p, c_void_p,
                                            c_float, c_int32, c_void_p, c_int32, _S]),
    "dt_euler_step": (c_int32, [c_void_p, c_void_p, c_float, c_void_p, c_int64, c_int32, _S]),
    "dt_fill_randn": (c_int32, [c_void_p, c_int64, c_uint64, c_float, c_float, _S]),
    "dt_quantize_q8_0": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, _S]),
    "dt_gemm_bf16": (c_int32, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int64,
                               c_int64, c_int64, c_void_p, c_void_p, c_int64, c_int32, _S]),
    "dt_gemm_bf16_config": (c_int32, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64,
                                      c_int64, c_int64, c_int64, c_void_p, c_void_p, c_int64, c_int32,
                                      c_int32, _S]),
    "dt_gemm_bf16_grouped": (c_int32, [c_void_p, c_int32, c_int32, c_int32, _S]),
    "dt_gemm_q8_0": (c_int32, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p,
                               c_int64, c_int64, c_int64, c_int64, c_void_p, c_void_p, c_int64, c_int32,
                               _S]),
    "dt_q8_0_split": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_void_p, c_int64, c_void_p,
                                c_int64, _S]),
    "dt_conv2d_packed_bytes": (ctypes.c_size_t, [c_int64, c_int64, c_int64]),
    "dt_conv2d_pack_weights": (c_int32, [c_void_p, c_int32, c_int64, c_int64, c_int64, c_void_p, _S]),
    "dt_conv2d_workspace_bytes": (ctypes.c_size_t, [c_int64, c_int64, c_int64, c_int64]),
    "dt_conv2d": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_void_p, c_int64, c_int64, c_int32,
                            c_void_p, c_void_p, c_void_p, ctypes.c_size_t, c_int32, _S]),
    "dt_conv2d_gn_stats_bytes": (ctypes.c_size_t, [c_int64, c_int64, c_int64, c_int64, c_int64]),
    "dt_conv2d_gn": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_void_p, c_int64, c_int64, c_int32,
                               c_void_p, c_void_p, c_int64, c_void_p, ctypes.c_size_t, c_void_p, ctypes.c_size_t,
                               c_int32, _S]),
    "dt_groupnorm_silu_from_stats": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_void_p, c_void_p,
                                               c_void_p, c_float, c_int32, c_void_p, c_int32, _S]),
    "dt_op_upscale_nearest": (c_int32, [c_void_p, c_int64, c_int64, c_int64, c_int64, c_int32, c_void_p, c_int32, _S]),
    "dt_flash_attn_qk_bf16": (c_int32, [c_void_p, _I64P, c_void_p, c_void_p, _I64P, c_void_p, c_int64, c_float,
                                        c_void_p, c_int64, c_int32, c_int32, c_float, c_void_p, c_int32,
                                        c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64,
                                        c_int64, _I64P, _I64P, _I64P, c_float, c_int32, _S]),
    "dt_graph_capture": (c_int32, [c_void_p, POINTER(POINTER(DtTensor)), c_int32, POINTER(c_void_p)]),
    "dt_graph_capture_ex": (c_int32, [c_void_p, POINTER(POINTER(DtTensor)), c_int32, c_uint32, POINTER(c_void_p)]),
    "dt_graph_exec_launch": (c_int32, [c_void_p, c_void_p]),
    "dt_graph_exec_free": (c_int32, [c_void_p]),
    "dt_q8_0_split_scale_offset": (c_int64, [c_int64, c_int64]),
    "dt_q8_0_split_bytes": (c_int64, [c_int64, c_int64]),
    "dt_gemm_f32": (c_int32, [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int64, c_int64, c_int64,
                              c_void_p, c_void_p, c_int64, _S]),
    "dt_gemm_bf16_workspace_bytes": (ctypes.c_size_t, [c_int64, c_int64, c_int64]),
    "dt_gemm_bf16_ws": (c_int32, [c_void_p, c_int32, c_void_p, ctypes.c_size_t, _S]),
    "dt_gemm_f32_workspace_bytes": (ctypes.c_size_t, [c_int64, c_int64, c_int64]),
    "dt_gemm_f32_ws": (c_int32, [c_void_p, c_void_p, ctypes.c_size_t, _S]),
    "dt_gemm_f32_grouped": (c_int32, [c_void_p, c_int32, _S]),
    "dt_flash_attn_f32_workspace_bytes": (ctypes.c_size_t, [c_int64, c_int64, c_int64, c_int64, c_int64]),
    "dt_flash_attn_f32": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64,
                                    c_int64, POINTER(c_int64), POINTER(c_int64), POINTER(c_int64),
                                    POINTER(c_int64), c_float, c_void_p, ctypes.c_size_t, _S]),
    "dt_flash_attn_bf16": (c_int32, [c_void_p, c_void_p, c_void_p, c_void_p, c_int64, c_int64,
                                     c_int64, c_int64, c_int64, POINTER(c_int64), POINTER(c_int64),
                                     POINTER(c_int64), POINTER(c_int64), c_float, c_int32, _S]),
    "dt_lora_gemm_workspace_bytes": (ctypes.c_size_t, [c_int64, c_int64, c_int64, c_int64]),
    "dt_lora_gemm": (c_int32, [c_void_p, c_void_p, c_int32, c_void_p, ctypes.c_size_t, _S]),
    "dt_rel_bucket_fill": (c_int32, [c_void_p, c_int64, c_int32, c_int32, c_int32]),
    "dt_attn_fwd_workspace_bytes": (ctypes.c_size_t, [c_void_p]),
    "dt_attn_fwd": (c_int32, [c_void_p, c_void_p, _I64P, c_void_p, c_void_p, ctypes.c_size_t, _S]),
    "dt_attn_bwd_workspace_bytes": (ctypes.c_size_t, [c_void_p]),
    "dt_attn_bwd": (c_int32, [c_void_p, c_void_p, c_void_p, ctypes.c_size_t, _S]),
    "dt_op_binary": (c_int32, [c_int32, POINTER(DtTensor), POINTER(DtTensor), POINTER(DtTensor), _S]),
    "dt_op_unary": (c_int32, [c_int32, POINTER(DtTensor), POINTER(DtTensor), c_float, c_float, _S]),
    "dt_op_norm": (c_int32, [POINTER(DtTensor), POINTER(DtTensor), c_float, _S]),
    "dt_op_rms_norm": (c_int32, [POINTER(DtTensor), POINTER(DtTensor), c_float, _S]),
    "dt_op_rope_ext": (c_int32, [POINTER(DtTensor), c_void_p, POINTER(DtTensor), c_int32, c_int32,
                                 c_float, c_float, c_float, c_float, _S]),
    "dt_op_concat": (c_int32, [POINTER(DtTensor), POINTER(DtTensor), c_int32, POINTER(DtTensor), _S]),
    "dt_op_cpy": (c_int32, [POINTER(DtTensor), POINTER(DtTensor), _S]),
    "dt_backend_init": (c_int32, [c_int32, POINTER(c_void_p)]),
    "dt_backend_free": (c_int32, [c_void_p]),
    "dt_backend_set_stream": (c_int32, [c_void_p, _S]),
    "dt_backend_synchronize": (c_int32, [c_void_p]),
    "dt_buffer_alloc": (c_int32, [c_void_p, c_size_t, POINTER(c_void_p)]),
    "dt_buffer_free": (c_int32, [c_void_p, c_void_p]),
    "dt_tensor_set": (c_int32, [POINTER(DtTensor), c_void_p, c_size_t, c_size_t, _S]),
    "dt_tensor_get": (c_int32, [POINTER(DtTensor), c_void_p, c_size_t, c_size_t, _S]),
    "dt_graph_compute": (c_int32, [c_void_p, POINTER(POINTER(DtTensor)), c_int32]),
    "dt_graph_compute_ex": (c_int32, [c_void_p, POINTER(POINTER(DtTensor)), c_int32, c_uint32]),
    "dt_graph_plan_checked": (c_int32, [POINTER(POINTER(DtTensor)), c_int32, POINTER(c_int32), POINTER(c_int32),
                                        POINTER(c_int32)]),
    "dt_graph_plan": (c_int32, [POINTER(POINTER(DtTensor)), c_int32, POINTER(c_int32)]),
    "dt_graph_plan_ex": (c_int32, [POINTER(POINTER(DtTensor)), c_int32, POINTER(c_int32),
                                   POINTER(c_int32)]),
    "dt_graph_last_stats": (c_int32, [POINTER(c_int32), POINTER(c_int32)]),
    "dt_graph_last_stats_ex": (c_int32, [POINTER(c_int32), POINTER(c_int32), POINTER(c_int32)]),
}

_lib = None


def load(path: str = LIB_PATH):
    """Load the library (once) and declare every signature."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise DtError(f"{path} is not built: run `make -C diffusers-cpp_amd` "
                      "(or __graft_entry__.build())")
    lib = ctypes.CDLL(path)
    for name, (res, args) in _SIGS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def exported_symbols():
    return list(_SIGS)


class _Recorder:
    """Stands in for the loaded library while prepare() runs a wrapper:
    forwards every call and keeps (function, converted arguments)."""

    def __init__(self, lib):
        self._lib = lib
        self.calls = []
        self.keep = []  # scratch tensors the recorded calls point into

    def __getattr__(self, name):
        fn = getattr(self._lib, name)

        def call(*args):
            conv = tuple(a if t is None or isinstance(a, t) else t(a)
                         for a, t in zip(args, fn.argtypes or [None] * len(args)))
            self.calls.append((fn, conv))
            return fn(*conv)

        return call


def _sizing():
    """The library itself: a size asked for once is no part of what prepare() repeats."""
    lib = load()
    return lib._lib if isinstance(lib, _Recorder) else lib


def prepare(wrapper, *args, **kwargs):
    """Run `wrapper(*args, **kwargs)` once (arguments checked, outputs
    allocated, the launch made) and return (result, launch): launch() repeats
    the C-ABI calls that run made, with the same pointers, sizes and stream,
    and no Python work between launches -- for tight loops such as timing
    back-to-back launches.  The tensors the call used must stay alive and
    unchanged in shape while launch is in use; status codes of the repeats
    are not checked (the first call's were)."""
    global _lib
    real = load()
    rec = _Recorder(real)
    _lib = rec
    try:
        result = wrapper(*args, **kwargs)
    finally:
        _lib = real
    calls = rec.calls
    if len(calls) == 1:
        fn, conv = calls[0]
        launch = functools.partial(fn, *conv)
    else:
        def launch():
            for fn, conv in calls:
                fn(*conv)
    launch.keep = rec.keep
    return result, launch


def check(rc: int, what: str = ""):
    if rc != 0:
        msg = load().dt_last_error().decode()
        raise DtError(f"{what or 'dit_hip'} failed (status {rc}): {msg}")


# --------------------------------------------------------------------------
# torch helpers
# --------------------------------------------------------------------------

# A small call's cost is this marshalling (17 us around a 9 us attention
# kernel), so it is kept to lookups: torch and its dtype codes once, the raw
# handle of the current stream, and stride triples (read only by the library).
_TORCH = None
_IO_TYPES = {}


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch
        _IO_TYPES.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16, torch.int32: I32})
        _TORCH = torch
    return _TORCH


def io_type(t) -> int:
    _torch()
    code = _IO_TYPES.get(t.dtype)
    if code is None:
        raise DtError(f"unsupported dtype {t.dtype}")
    return code


_I64x3 = c_int64 * 3


@functools.lru_cache(maxsize=1024)
def _i64x3(a, b, c):
    return _I64x3(a, b, c)


def _strides3(t):
    a = t.stride()
    return _i64x3(a[0], a[1], a[2])


def _p(t):
    return None if t is None else c_void_p(t.data_ptr())


def stream():
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is None:
        return c_void_p(torch.cuda.current_stream().cuda_stream)
    return c_void_p(raw(torch.cuda.current_device()))


def desc(t, op=OP_NONE) -> DtTensor:
    """ggml-ordered descriptor of a torch tensor (at most 4-D)."""
    if t.dim() > 4:
        raise DtError("at most 4 dims")
    d = DtTensor()
    d.type = io_type(t)
    d.op = op
    es = t.element_size()
    shape = list(t.shape)[::-1] + [1] * (4 - t.dim())
    strides = [s * es for s in list(t.stride())[::-1]]
    for i in range(4):
        d.ne[i] = shape[i]
        if i < len(strides):
            d.nb[i] = strides[i]
        else:
            d.nb[i] = (d.nb[i - 1] * d.ne[i - 1]) if i > 0 else es
    d.data = t.data_ptr()
    return d


def _rows(t):
    """(rows, cols, row_stride) of a tensor whose last dim is contiguous and
    whose leading dims collapse to a uniform row stride."""
    if t.stride(-1) != 1:
        raise DtError("last dim must be contiguous")
    cols = t.shape[-1]
    if t.dim() == 1:
        return 1, cols, cols
    rows = 1
    for s in t.shape[:-1]:
        rows *= s
    rs = t.stride(-2)
    expect = rs
    for i in range(t.dim() - 2, -1, -1):
        if t.shape[i] > 1 and t.stride(i) != expect:
            raise DtError("leading dims do not collapse to one row stride")
        expect *= t.shape[i]
    return rows, cols, rs


# --------------------------------------------------------------------------
# fused entry points
# --------------------------------------------------------------------------

def adaln_mod(x, shift, scale, eps=1e-6, out=None):
    torch = _torch()
    rows, cols, xs = _rows(x)
    y = torch.empty_like(x) if out is None else out
    _, _, ys = _rows(y)
    check(load().dt_adaln_mod(_p(x), rows, cols, xs, _p(shift), _p(scale), _p(y), ys, eps,
                              io_type(x), stream()), "dt_adaln_mod")
    return y


def rope_table(n_pos: int, n_dims: int, freq_base: float, device="cuda"):
    """cos/sin table [n_pos, n_dims] (ggml fp32 recurrence), on `device`."""
    torch = _torch()
    host = torch.empty((n_pos, n_dims), dtype=torch.float32)
    check(load().dt_rope_table_fill(c_void_p(host.data_ptr()), n_pos, n_dims, freq_base, 1.0, 1.0),
          "dt_rope_table_fill")
    return host.to(device) if device != "cpu" else host


def qk_rmsnorm_rope(q, k, wq, wk, pos, axis_dim, freq_base, eps=1e-6, table=None,
                    q_out=None, k_out=None):
    """q, k: [tokens, heads, head_dim] views (strides honoured); pos: int32
    [tokens, n_axes] (row stride honoured)."""
    torch = _torch()
    x = q if q is not None else k
    tokens, heads, head_dim = x.shape
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k is not None and k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    o = q_out if q is not None else k_out
    for a, b in ((q, k), (q_out, k_out)):
        if a is not None and b is not None and a.stride() != b.stride():
            raise DtError("q and k (and their outputs) must share strides")
    if x.stride(2) != 1 or o.stride(2) != 1 or pos.stride(1) != 1:
        raise DtError("head_dim and axis columns must be contiguous")
    n_axes = pos.shape[1]
    n_pos = 0 if table is None else table.shape[0]
    check(load().dt_qk_rmsnorm_rope(
        _p(q), _p(k), _p(q_out), _p(k_out), tokens, heads, head_dim, x.stride(0), x.stride(1),
        o.stride(0), o.stride(1), _p(wq), _p(wk), eps, _p(pos), pos.stride(0), n_axes, axis_dim,
        freq_base, _p(table), n_pos, io_type(x), stream()), "dt_qk_rmsnorm_rope")
    return q_out, k_out


def qk_rmsnorm_rope_swiglu(q, k, wq, wk, pos, axis_dim, freq_base, gate, up, eps=1e-6, table=None,
                           q_out=None, k_out=None, out=None):
    """qk_rmsnorm_rope(q, k) and swiglu(gate, up) in one launch -> (q_out,
    k_out, y); q or k may be None (that half is skipped)."""
    torch = _torch()
    x = q if q is not None else k
    tokens, heads, head_dim = x.shape
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k is not None and k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    o = q_out if q is not None else k_out
    y = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device) if out is None else out
    for a, b in ((q, k), (q_out, k_out)):
        if a is not None and b is not None and a.stride() != b.stride():
            raise DtError("q and k (and their outputs) must share strides")
    rows, inner, gs = _rows(gate)
    us, ys = _rows(up)[2], _rows(y)[2]
    n_pos = 0 if table is None else table.shape[0]
    check(load().dt_qk_rmsnorm_rope_swiglu(
        _p(q), _p(k), _p(q_out), _p(k_out), tokens, heads, head_dim, x.stride(0), x.stride(1),
        o.stride(0), o.stride(1), _p(wq), _p(wk), eps, _p(pos), pos.stride(0), pos.shape[1],
        axis_dim, freq_base, _p(table), n_pos, _p(gate), gs, _p(up), us, _p(y), ys, rows, inner,
        io_type(x), stream()), "dt_qk_rmsnorm_rope_swiglu")
    return q_out, k_out, y


def swiglu(gate, up, out=None):
    torch = _torch()
    rows, cols, gs = _rows(gate)
    _, _, us = _rows(up)
    y = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device) if out is None else out
    _, _, ys = _rows(y)
    check(load().dt_swiglu(_p(gate), gs, _p(up), us, _p(y), ys, rows, cols, io_type(gate),
                           stream()), "dt_swiglu")
    return y


def gated_residual(h, o, gate, out=None):
    torch = _torch()
    rows, cols, hs = _rows(h)
    _, _, os_ = _rows(o)
    y = torch.empty(h.shape, dtype=h.dtype, device=h.device) if out is None else out
    _, _, ys = _rows(y)
    check(load().dt_gated_residual(_p(h), hs, _p(o), os_, _p(gate), _p(y), ys, rows, cols,
                                   io_type(h), stream()), "dt_gated_residual")
    return y


def gated_residual_adaln(h, o, gate, shift, scale, eps=1e-6, r_out=None, out=None):
    """r = h + gate * o; y = (1 + scale) * LayerNorm(r) + shift -> (r, y)."""
    torch = _torch()
    rows, cols, hs = _rows(h)
    os_ = _rows(o)[2]
    r = torch.empty(h.shape, dtype=h.dtype, device=h.device) if r_out is None else r_out
    y = torch.empty(h.shape, dtype=h.dtype, device=h.device) if out is None else out
    rs, ys = _rows(r)[2], _rows(y)[2]
    check(load().dt_gated_residual_adaln(_p(h), hs, _p(o), os_, _p(gate), _p(r), rs, _p(shift), _p(scale),
                                         _p(y), ys, rows, cols, eps, io_type(h), stream()),
          "dt_gated_residual_adaln")
    return r, y


def block_bytes(qtype: int) -> tuple[int, int]:
    """(elements per block, bytes per block)"""
    return (32, 34) if qtype == Q8_0 else (256, 144)


def dequant(src, qtype, rows, cols, out_dtype=None, out=None):
    """src: uint8 device tensor of rows*(cols/qk)*block bytes."""
    torch = _torch()
    out_dtype = out_dtype or torch.bfloat16
    qk, bs = block_bytes(qtype)
    y = torch.empty((rows, cols), dtype=out_dtype, device=src.device) if out is None else out
    check(load().dt_dequant(_p(src), qtype, rows, cols, cols // qk * bs, _p(y), y.stride(0),
                            io_type(y), stream()), "dt_dequant")
    return y


def groupnorm_silu(x, groups, w=None, b=None, eps=1e-6, silu=True, out=None, workspace=None):
    """x: [N, C, H, W] contiguous."""
    torch = _torch()
    N, C, H, W = x.shape
    HW = H * W
    lib = load()
    nbytes = lib.dt_groupnorm_workspace_bytes(N, C, HW, groups)
    if workspace is None or workspace.numel() < nbytes:
        workspace = torch.empty(max(nbytes, 8), dtype=torch.uint8, device=x.device)
    y = torch.empty_like(x) if out is None else out
    check(lib.dt_groupnorm_silu(_p(x), N, C, HW, groups, _p(w), _p(b), eps, 1 if silu else 0,
                                _p(y), _p(workspace), workspace.numel(), io_type(x), stream()),
          "dt_groupnorm_silu")
    return y


def groupnorm_silu_noalloc(x, groups, w=None, b=None, eps=1e-6, silu=True, out=None):
    """groupnorm_silu through dt_groupnorm_silu_noalloc (the library's own
    device scratch; nothing allocated but the output when out is None)."""
    torch = _torch()
    N, C, H, W = x.shape
    y = torch.empty_like(x) if out is None else out
    check(load().dt_groupnorm_silu_noalloc(_p(x), N, C, H * W, groups, _p(w), _p(b), eps, 1 if silu else 0,
                                           _p(y), io_type(x), stream()),
          "dt_groupnorm_silu_noalloc")
    return y


def euler_step(x, v, dt, out=None):
    torch = _torch()
    y = torch.empty_like(x) if out is None else out
    check(load().dt_euler_step(_p(x), _p(v), dt, _p(y), x.numel(), io_type(x), stream()),
          "dt_euler_step")
    return y


def quantize_q8_0(x, out=None):
    """x: float32 [rows, cols] (row-contiguous) -> uint8 [rows, cols/32*34]."""
    torch = _torch()
    rows, cols = x.shape
    rb = cols // 32 * 34
    y = torch.empty((rows, rb), dtype=torch.uint8, device=x.device) if out is None else out
    check(load().dt_quantize_q8_0(_p(x), rows, cols, x.stride(0), _p(y), y.stride(0), stream()),
          "dt_quantize_q8_0")
    return y


def _scratch(nbytes, device):
    """Device scratch of one call: back in PyTorch's pool when the wrapper
    returns, in stream order; prepare() keeps it for its repeats."""
    torch = _torch()
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    lib = load()
    if isinstance(lib, _Recorder):
        lib.keep.append(ws)
    return ws


def _scratch_by(t, nbytes):
    """_scratch where t is."""
    ws = t.new_empty(nbytes, dtype=_TORCH.uint8)
    lib = load()
    if isinstance(lib, _Recorder):
        lib.keep.append(ws)
    return ws


def _gemm_ws(nbytes, M, N, K, a):
    """Scratch for a product taken over ranges of K, or None for one that is not split."""
    n = nbytes(M, N, K)
    return _scratch(n, a.device) if n else None


def gemm(a, b, bias=None, addend=None, out=None, out_dtype=None, config=-1):
    """a: bf16 [M, K], b: bf16 [N, K] (rows K-contiguous) -> a @ b.T (+ bias) (+ addend).
    config: tile configuration (0: 256x256, 8 waves, K = 32 stages; 1: 128x128;
    2: 256x256, 4 waves, K = 64 stages; 5: config 2 scheduled; 6: config 5 at
    224x256; 8: config 5 in 8 waves; -1: by shape).  Q8_0 weights: gemm_q8_0."""
    torch = _torch()
    M, K = a.shape
    N = b.shape[0]
    assert b.shape[1] == K and a.stride(1) == 1 and b.stride(1) == 1
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or torch.bfloat16, device=a.device)
    ldd = addend.stride(0) if addend is not None else 0
    ws = _gemm_ws(load().dt_gemm_bf16_workspace_bytes, M, N, K, a) if config == -1 else None
    if ws is not None:
        p = GemmProblem(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), out.data_ptr(), out.stride(0),
                        _p(addend), ldd, _p(bias), M, N, K, None, 0)
        check(load().dt_gemm_bf16_ws(ctypes.cast(ctypes.pointer(p), c_void_p), io_type(out), _p(ws), ws.numel(), stream()), "dt_gemm_bf16_ws")
        return out
    check(load().dt_gemm_bf16_config(_p(a), a.stride(0), _p(b), b.stride(0), _p(out), out.stride(0),
                                     M, N, K, _p(bias), _p(addend), ldd, io_type(out), config,
                                     stream()),
          "dt_gemm_bf16")
    return out


class GemmProblem(ctypes.Structure):
    _fields_ = [("A", c_void_p), ("lda", c_int64), ("B", c_void_p), ("ldb", c_int64),
                ("C", c_void_p), ("ldc", c_int64), ("addend", c_void_p), ("ldd", c_int64),
                ("bias", c_void_p), ("M", c_int64), ("N", c_int64), ("K", c_int64),
                ("b_scale", c_void_p), ("ld_scale", c_int64)]


class Q8Weight:
    """A Q8_0 weight [N, K] in the split layout dt_gemm_q8_0 reads: uint8 codes
    (q + 128) [N, K] and fp32 block scales [K/32, N]."""

    def __init__(self, codes, scales):
        self.codes, self.scales = codes, scales
        self.shape = (codes.shape[0], codes.shape[1])


def q8_0_split(blocks, rows, cols):
    """blocks: uint8 device tensor of rows * cols/32 Q8_0 blocks -> Q8Weight."""
    torch = _torch()
    codes = torch.empty((rows, cols), dtype=torch.uint8, device=blocks.device)
    scales = torch.empty((cols // 32, rows), dtype=torch.float32, device=blocks.device)
    check(load().dt_q8_0_split(_p(blocks), rows, cols, cols // 32 * 34, _p(codes), codes.stride(0),
                               _p(scales), scales.stride(0), stream()), "dt_q8_0_split")
    return Q8Weight(codes, scales)


def gemm_q8_0(a, w, bias=None, addend=None, out=None, out_dtype=None):
    """a: bf16 [M, K]; w: Q8Weight [N, K] -> a @ dequant(w).T (+ bias) (+ addend)."""
    torch = _torch()
    M, K = a.shape
    N = w.shape[0]
    assert w.shape[1] == K and a.stride(1) == 1
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype or torch.bfloat16, device=a.device)
    ldd = addend.stride(0) if addend is not None else 0
    ws = _gemm_ws(load().dt_gemm_bf16_workspace_bytes, M, N, K, a)
    if ws is not None:
        p = GemmProblem(a.data_ptr(), a.stride(0), w.codes.data_ptr(), w.codes.stride(0), out.data_ptr(),
                        out.stride(0), _p(addend), ldd, _p(bias), M, N, K, w.scales.data_ptr(), w.scales.stride(0))
        check(load().dt_gemm_bf16_ws(ctypes.cast(ctypes.pointer(p), c_void_p), io_type(out), _p(ws), ws.numel(), stream()), "dt_gemm_q8_0")
        return out
    check(load().dt_gemm_q8_0(_p(a), a.stride(0), _p(w.codes), w.codes.stride(0), _p(w.scales),
                              w.scales.stride(0), _p(out), out.stride(0), M, N, K, _p(bias), _p(addend), ldd,
                              io_type(out), stream()), "dt_gemm_q8_0")
    return out


def gemm_grouped(items, config=-1):
    """items: list of (a [M,K] bf16, b [N,K] bf16 or Q8Weight, out [M,N]) -> one launch."""
    probs = (GemmProblem * len(items))()
    for i, (a, b, out) in enumerate(items):
        if isinstance(b, Q8Weight):
            probs[i] = GemmProblem(a.data_ptr(), a.stride(0), b.codes.data_ptr(), b.codes.stride(0),
                                   out.data_ptr(), out.stride(0), None, 0, None, a.shape[0], b.shape[0],
                                   a.shape[1], b.scales.data_ptr(), b.scales.stride(0))
        else:
            probs[i] = GemmProblem(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), out.data_ptr(),
                                   out.stride(0), None, 0, None, a.shape[0], b.shape[0], a.shape[1], None, 0)
    ct = io_type(items[0][2])
    check(load().dt_gemm_bf16_grouped(ctypes.cast(probs, c_void_p), len(items), ct, config, stream()),
          "dt_gemm_bf16_grouped")
    return [it[2] for it in items]


class ConvWeight:
    """Conv2d weights [Co, Ci, K, K] packed for dt_conv2d."""

    def __init__(self, packed, co, ci, k):
        self.packed, self.co, self.ci, self.k = packed, co, ci, k


def conv2d_pack(w):
    """w: fp32 or bf16 device tensor [Co, Ci, K, K] -> ConvWeight."""
    torch = _torch()
    co, ci, k, k2 = w.shape
    assert k == k2 and w.is_contiguous()
    n = load().dt_conv2d_packed_bytes(co, ci, k)
    assert n > 0, "unsupported conv weight shape"
    packed = torch.empty(n, dtype=torch.uint8, device=w.device)
    check(load().dt_conv2d_pack_weights(_p(w), io_type(w), co, ci, k, _p(packed), stream()),
          "dt_conv2d_pack_weights")
    return ConvWeight(packed, co, ci, k)


def _conv_ws(x, workspace):
    """A workspace for the DMA conv path: True allocates one, a tensor is used
    as given, None selects the path without one."""
    torch = _torch()
    if workspace is True:
        N, ci, H, W = x.shape
        return _scratch(load().dt_conv2d_workspace_bytes(N, ci, H, W), x.device)
    return workspace


def conv2d(x, w, bias=None, upscale2=False, out=None, workspace=True):
    """x: [N, Ci, H, W] (fp32/bf16, contiguous); w: ConvWeight -> [N, Co, H', W']."""
    torch = _torch()
    N, ci, H, W = x.shape
    assert ci == w.ci and x.is_contiguous()
    Hs, Ws = (2 * H, 2 * W) if upscale2 else (H, W)
    y = torch.empty((N, w.co, Hs, Ws), dtype=x.dtype, device=x.device) if out is None else out
    ws = _conv_ws(x, workspace)
    check(load().dt_conv2d(_p(x), N, ci, H, W, _p(w.packed), w.co, w.k, 1 if upscale2 else 0, _p(bias), _p(y),
                           _p(ws), ws.numel() if ws is not None else 0, io_type(x), stream()), "dt_conv2d")
    return y


def conv2d_gn(x, w, groups, bias=None, upscale2=False, out=None, workspace=True):
    """dt_conv2d + GroupNorm statistics of the output -> (y, stats); stats[:N*groups*16]
    viewed as float64 pairs holds (mean, variance) per (n, g)."""
    torch = _torch()
    N, ci, H, W = x.shape
    assert ci == w.ci and x.is_contiguous()
    Hs, Ws = (2 * H, 2 * W) if upscale2 else (H, W)
    y = torch.empty((N, w.co, Hs, Ws), dtype=x.dtype, device=x.device) if out is None else out
    nb = load().dt_conv2d_gn_stats_bytes(N, w.co, Hs, Ws, groups)
    assert nb > 0, "unsupported conv/GroupNorm shape"
    stats = torch.empty(nb, dtype=torch.uint8, device=x.device)
    ws = _conv_ws(x, workspace)
    check(load().dt_conv2d_gn(_p(x), N, ci, H, W, _p(w.packed), w.co, w.k, 1 if upscale2 else 0, _p(bias), _p(y),
                              groups, _p(stats), nb, _p(ws), ws.numel() if ws is not None else 0, io_type(x),
                              stream()), "dt_conv2d_gn")
    return y, stats


def groupnorm_silu_from_stats(x, stats, groups, w=None, b=None, eps=1e-6, silu=True, out=None):
    torch = _torch()
    N, C = x.shape[0], x.shape[1]
    HW = x.numel() // (N * C)
    y = torch.empty_like(x) if out is None else out
    check(load().dt_groupnorm_silu_from_stats(_p(x), N, C, HW, groups, _p(stats), _p(w), _p(b), eps,
                                              1 if silu else 0, _p(y), io_type(x), stream()),
          "dt_groupnorm_silu_from_stats")
    return y


def flash_attn(q, k, v, scale=None, out=None, out_dtype=None):
    """q: bf16 [B, Sq, H, 128], k, v: [B, Skv, H, 128] (any strides with d
    contiguous) -> softmax(scale q k^T) v as [B, Sq, H, 128]."""
    torch = _torch()
    B, Sq, H, D = q.shape
    Skv = k.shape[1]
    if out is None:
        out = torch.empty((B, Sq, H, D), dtype=out_dtype or torch.bfloat16, device=q.device)
    st = _strides3
    scale = 1.0 / D ** 0.5 if scale is None else scale
    check(load().dt_flash_attn_bf16(_p(q), _p(k), _p(v), _p(out), B, H, Sq, Skv, D, st(q), st(k),
                                    st(v), st(out), scale, io_type(out), stream()),
          "dt_flash_attn_bf16")
    return out


def gemm_f32(a, b, bias=None, addend=None, out=None):
    """a: fp32 [M, K], b: fp32 [N, K] (rows K-contiguous) -> a @ b.T (+ bias) (+ addend), to fp32 accuracy."""
    torch = _torch()
    M, K = a.shape
    N = b.shape[0]
    assert b.shape[1] == K and a.stride(1) == 1 and b.stride(1) == 1
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    ldd = addend.stride(0) if addend is not None else 0
    ws = _gemm_ws(load().dt_gemm_f32_workspace_bytes, M, N, K, a)
    if ws is not None:
        p = GemmProblem(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), out.data_ptr(), out.stride(0),
                        _p(addend), ldd, _p(bias), M, N, K, None, 0)
        check(load().dt_gemm_f32_ws(ctypes.cast(ctypes.pointer(p), c_void_p), _p(ws), ws.numel(), stream()), "dt_gemm_f32")
        return out
    check(load().dt_gemm_f32(_p(a), a.stride(0), _p(b), b.stride(0), _p(out), out.stride(0), M, N, K, _p(bias),
                             _p(addend), ldd, stream()), "dt_gemm_f32")
    return out


def flash_attn_f32(q, k, v, scale=None, out=None):
    """q: fp32 [B, Sq, H, 128], k, v: [B, Skv, H, 128] (d contiguous) ->
    softmax(scale q k^T) v as fp32 [B, Sq, H, 128], in fp32 throughout."""
    torch = _torch()
    B, Sq, H, D = q.shape
    Skv = k.shape[1]
    if out is None:
        out = torch.empty((B, Sq, H, D), dtype=torch.float32, device=q.device)
    st = _strides3
    scale = 1.0 / D ** 0.5 if scale is None else scale
    lib = load()
    nbytes = lib.dt_flash_attn_f32_workspace_bytes(B, H, Sq, Skv, D)
    ws = _scratch(max(nbytes, 16), q.device)
    check(lib.dt_flash_attn_f32(_p(q), _p(k), _p(v), _p(out), B, H, Sq, Skv, D, st(q), st(k), st(v), st(out),
                                scale, _p(ws), ws.numel(), stream()), "dt_flash_attn_f32")
    return out


def flash_attn_qk(q_segments, k, v, pos, axis_dim, freq_base, eps=1e-6, table=None, scale=None, out=None,
                  out_dtype=None):
    """flash_attn with q taken before its QK-RMSNorm + RoPE.  q_segments:
    one or two (q, w) pairs, q bf16 [B, S_i, H, 128] (strides honoured), w
    fp32 [128]; the segments are the query sequence in order (txt then img).
    pos: int32 [sum S_i, n_axes] of the joint sequence."""
    torch = _torch()
    (q0, w0) = q_segments[0]
    q1, w1 = q_segments[1] if len(q_segments) > 1 else (None, None)
    B, S0, H, D = q0.shape
    Sq = S0 + (q1.shape[1] if q1 is not None else 0)
    Skv = k.shape[1]
    if out is None:
        out = torch.empty((B, Sq, H, D), dtype=out_dtype or torch.bfloat16, device=k.device)
    st = _strides3
    scale = 1.0 / D ** 0.5 if scale is None else scale
    n_pos = 0 if table is None else table.shape[0]
    check(load().dt_flash_attn_qk_bf16(
        _p(q0), st(q0), _p(w0), _p(q1), st(q1) if q1 is not None else None, _p(w1), S0 if q1 is not None else Sq,
        eps, _p(pos), pos.stride(0), pos.shape[1], axis_dim, freq_base, _p(table), n_pos, _p(k), _p(v), _p(out),
        B, H, Sq, Skv, D, st(k), st(v), st(out), scale, io_type(out), stream()), "dt_flash_attn_qk_bf16")
    return out


class LoraArgs(ctypes.Structure):
    _fields_ = [("a", c_void_p), ("lda", c_int64), ("a_stride", c_int64), ("b", c_void_p), ("ldb", c_int64),
                ("b_stride", c_int64), ("scale", c_void_p), ("row_adapter", c_void_p), ("adapters", c_int64),
                ("rank", c_int64)]


class Lora:
    """Low-rank adapters of one Linear, side by side: a bf16 [adapters, rank, K] (down),
    b bf16 [adapters, N, rank] (up), scale fp32 [adapters] or None (1)."""

    def __init__(self, a, b, scale=None):
        self.a, self.b, self.scale = a, b, scale


# The calls below check what their tensors are like (types, shapes, strides, devices) once
# for each such description, and keep the arguments' structure without its pointers: of a
# call around a 9 us kernel the checks took 10 us.

def _meta(t):
    return None if t is None else (t.dtype, t.shape, t.stride(), t.get_device())


def _on_device(metas):
    """The launch goes to the current device's current stream: every tensor has to be there."""
    here = _torch().cuda.current_device()
    for m in metas:
        if m is not None and m[3] != here:
            raise DtError(f"a tensor is on {'the host' if m[3] < 0 else 'device %d' % m[3]}, not on the current device {here}")


def _vector(m, dtype, n, what):
    if m is not None and (m[0] != dtype or m[1] != (n,) or (n > 1 and m[2][0] != 1)):
        raise DtError(f"{what} must be contiguous {dtype} [{n}]")


@functools.lru_cache(maxsize=512)
def _lora_plan(x, w, scales, a, b, scale, rows, bias, addend, out, here):
    torch = _torch()
    q8 = scales is not None
    if len(x[1]) != 2 or len(w[1]) != 2 or len(a[1]) != 3 or len(b[1]) != 3 or len(out[1]) != 2:
        raise DtError("x and w must have two dimensions, the adapters three")
    (M, K), N, (n, rank) = x[1], w[1][0], a[1][:2]
    if x[0] != torch.bfloat16 or a[0] != torch.bfloat16 or b[0] != torch.bfloat16 or \
            w[0] != (torch.uint8 if q8 else torch.bfloat16) or (q8 and scales[0] != torch.float32):
        raise DtError("x, w and the adapters must be bf16 (a Q8Weight: uint8 codes, fp32 scales)")
    if w[1][1] != K or a[1] != (n, rank, K) or b[1] != (n, N, rank) or (q8 and scales[1] != (K // 32, N)):
        raise DtError(f"adapters {tuple(a[1])}, {tuple(b[1])} do not fit x {tuple(x[1])} and w {tuple(w[1])}")
    if (K > 1 and (x[2][1] != 1 or w[2][1] != 1 or a[2][2] != 1)) or (rank > 1 and b[2][2] != 1) or \
            (q8 and N > 1 and scales[2][1] != 1):
        raise DtError("rows of x, w and the adapters must be contiguous")
    if rows is None:
        raise DtError("row_adapter must be given (-1: no adapter)")
    _vector(rows, torch.int32, M, "row_adapter")
    _vector(scale, torch.float32, n, "scale")
    _vector(bias, torch.float32, N, "bias")
    for t in (out, addend):
        if t is not None and (t[1] != (M, N) or t[0] != out[0] or (N > 1 and t[2][1] != 1)):
            raise DtError("out and addend must be [M, N] of one dtype with contiguous rows")
    if out[0] not in (torch.bfloat16, torch.float32):
        raise DtError(f"out must be bf16 or fp32, not {out[0]}")
    _on_device((x, w, scales, a, b, scale, rows, bias, addend, out))

    def ld(m, cols):  # the row stride of a tensor of one row is not used
        return max(m[2][-2], cols) if m[1][-2] <= 1 else m[2][-2]

    p = GemmProblem(None, ld(x, K), None, ld(w, K), None, ld(out, N), None, 0 if addend is None else ld(addend, N), None, M,
                    N, K, None, ld(scales, N) if q8 else 0)
    s = LoraArgs(None, ld(a, K), a[2][0], None, ld(b, rank), b[2][0], None, None, n, rank)
    return bytes(p), bytes(s), _sizing().dt_lora_gemm_workspace_bytes(M, N, K, rank), _IO_TYPES[out[0]]


def lora_gemm(x, w, lora, row_adapter, bias=None, addend=None, out=None, out_dtype=None):
    """x: bf16 [M, K], w: bf16 [N, K] or Q8Weight -> x @ w.T (+ bias) (+ addend) +
    scale[a] * (x @ a[a].T) @ b[a].T, each row with the adapter a = row_adapter[m]
    (int32 [M]; outside the adapters: none).  Autograd records nothing, and no
    gradients of the adapters are offered."""
    torch = _torch()
    q8 = isinstance(w, Q8Weight)
    codes, scales = (w.codes, w.scales) if q8 else (w, None)
    a, b, scale = lora.a, lora.b, lora.scale
    if out is None:
        out = x.new_empty((x.shape[0], w.shape[0]), dtype=out_dtype or torch.bfloat16)
    p, s, nbytes, out_type = _lora_plan(_meta(x), _meta(codes), _meta(scales), _meta(a), _meta(b), _meta(scale),
                                        _meta(row_adapter), _meta(bias), _meta(addend), _meta(out),
                                        torch.cuda.current_device())
    p, s = GemmProblem.from_buffer_copy(p), LoraArgs.from_buffer_copy(s)
    p.A, p.B, p.C = x.data_ptr(), codes.data_ptr(), out.data_ptr()
    s.a, s.b, s.row_adapter = a.data_ptr(), b.data_ptr(), row_adapter.data_ptr()
    if bias is not None:
        p.bias = bias.data_ptr()
    if addend is not None:
        p.addend = addend.data_ptr()
    if q8:
        p.b_scale = scales.data_ptr()
    if scale is not None:
        s.scale = scale.data_ptr()
    ws = _scratch_by(x, nbytes) if nbytes else None
    lib = load()
    check(lib.dt_lora_gemm(ctypes.addressof(p), ctypes.addressof(s), out_type, None if ws is None else ws.data_ptr(),
                           nbytes, stream()), "dt_lora_gemm")
    if isinstance(lib, _Recorder):
        lib.keep.extend((p, s))
    return out


class AttnArgs(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("q_strides", _I64x3), ("k_strides", _I64x3),
                ("v_strides", _I64x3), ("batch", c_int64), ("heads", c_int64), ("kv_heads", c_int64),
                ("seq_q", c_int64), ("seq_kv", c_int64), ("head_dim", c_int64), ("kv_len", c_void_p),
                ("kv_mask", c_void_p), ("kv_mask_stride", c_int64), ("rel_table", c_void_p),
                ("rel_table_stride", c_int64), ("q_pos", c_void_p), ("rel_buckets", c_int32),
                ("rel_distance", c_int32), ("rel_two_sided", c_int32), ("io_type", c_int32), ("scale", c_float)]


class AttnGrads(ctypes.Structure):
    _fields_ = [("d_o", c_void_p), ("o", c_void_p), ("lse", c_void_p), ("dq", c_void_p), ("dk", c_void_p),
                ("dv", c_void_p), ("d_o_strides", _I64x3), ("o_strides", _I64x3), ("dq_strides", _I64x3),
                ("dk_strides", _I64x3), ("dv_strides", _I64x3), ("d_rel_table", c_void_p),
                ("d_rel_table_stride", c_int64)]


class RelBias:
    """A learned relative position bias: table fp32 [buckets, heads]; key - query
    falls into the buckets rel_buckets() lists."""

    def __init__(self, table, distance, two_sided=True):
        self.table, self.distance, self.two_sided = table, distance, two_sided


def rel_buckets(n, buckets, distance, two_sided=True):
    """The bucket of every offset key - query in (-n, n), as a host int32 tensor [2 n - 1]."""
    torch = _torch()
    out = torch.empty(max(2 * n - 1, 0), dtype=torch.int32)
    check(load().dt_rel_bucket_fill(c_void_p(out.data_ptr()), n, buckets, distance, 1 if two_sided else 0),
          "dt_rel_bucket_fill")
    return out


@functools.lru_cache(maxsize=512)
def _attn_plan(q, k, v, kv_len, kv_mask, table, q_pos, distance, two_sided, out, here):
    torch = _torch()
    if len(q[1]) != 4 or len(k[1]) != 4 or v[1] != k[1]:
        raise DtError("q must be [B, Sq, H, D], k and v [B, Skv, Hkv, D]")
    B, Sq, H, D = q[1]
    Bk, Skv, Hkv, Dk = k[1]
    if Bk != B or Dk != D:
        raise DtError(f"k {tuple(k[1])} does not fit q {tuple(q[1])}")
    if q[0] not in (torch.bfloat16, torch.float32) or k[0] != q[0] or v[0] != q[0]:
        raise DtError("q, k and v must share a dtype, bf16 or fp32")
    if q[2][3] != 1 or k[2][3] != 1 or v[2][3] != 1:
        raise DtError("the head dim must be contiguous")
    if out[1] != q[1] or out[0] != q[0] or out[2][3] != 1:
        raise DtError("out must have q's shape and dtype, its head dim contiguous")
    a = AttnArgs()
    a.q_strides[:], a.k_strides[:], a.v_strides[:] = q[2][:3], k[2][:3], v[2][:3]
    a.batch, a.heads, a.kv_heads, a.seq_q, a.seq_kv, a.head_dim = B, H, Hkv, Sq, Skv, D
    a.io_type = _IO_TYPES[q[0]]
    _vector(kv_len, torch.int32, B, "kv_len")
    if kv_mask is not None:
        if kv_mask[0] not in (torch.uint8, torch.bool) or kv_mask[1] != (B, Skv) or (Skv > 1 and kv_mask[2][1] != 1):
            raise DtError("kv_mask must be uint8 or bool [B, Skv] with contiguous rows")
        a.kv_mask_stride = kv_mask[2][0]
    if table is not None:
        if table[0] != torch.float32 or len(table[1]) != 2 or table[1][1] != H or (H > 1 and table[2][1] != 1):
            raise DtError("the bias table must be fp32 [buckets, H] with contiguous rows")
        a.rel_table_stride = table[2][0] if table[1][0] > 1 else H
        a.rel_buckets, a.rel_distance, a.rel_two_sided = table[1][0], distance, 1 if two_sided else 0
        _vector(q_pos, torch.int32, B, "q_pos")
    _on_device((q, k, v, kv_len, kv_mask, table, q_pos, out))
    a.scale = 1.0 / D ** 0.5
    # The workspaces go by sizes alone; the pointers stand for the call's own.
    a.q = a.k = a.v = 16
    a.rel_table = None if table is None else 16
    lib, p = _sizing(), ctypes.addressof(a)
    sizes = lib.dt_attn_fwd_workspace_bytes(p), lib.dt_attn_bwd_workspace_bytes(p)
    return bytes(a), *sizes, _i64x3(*out[2][:3])


def _attn_pointers(plan, q, k, v, kv_len, kv_mask, scale, rel, q_pos):
    a = AttnArgs.from_buffer_copy(plan)
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if scale is not None:
        a.scale = scale
    if kv_len is not None:
        a.kv_len = kv_len.data_ptr()
    if kv_mask is not None:
        a.kv_mask = kv_mask.data_ptr()
    if rel is not None:
        a.rel_table = rel.table.data_ptr()
        if q_pos is not None:
            a.q_pos = q_pos.data_ptr()
    return a


def _attn_args(q, k, v, kv_len, kv_mask, scale, rel, q_pos, out):
    plan, fwd, bwd, o_strides = _attn_plan(
        _meta(q), _meta(k), _meta(v), _meta(kv_len), _meta(kv_mask), None if rel is None else _meta(rel.table), _meta(q_pos),
        None if rel is None else rel.distance, None if rel is None else rel.two_sided, _meta(out), _torch().cuda.current_device())
    return _attn_pointers(plan, q, k, v, kv_len, kv_mask, scale, rel, q_pos), fwd, bwd, o_strides


def _attn(q, k, v, kv_len, kv_mask, scale, rel, q_pos, out, return_lse):
    if out is None:
        out = q.new_empty(q.shape)
    a, n, _, o_strides = _attn_args(q, k, v, kv_len, kv_mask, scale, rel, q_pos, out)
    lse = q.new_empty((a.batch, a.heads, a.seq_q), dtype=_TORCH.float32) if return_lse else None
    lib = load()
    ws = _scratch_by(q, n) if n else None
    check(lib.dt_attn_fwd(ctypes.addressof(a), out.data_ptr(), o_strides, None if lse is None else lse.data_ptr(),
                          None if ws is None else ws.data_ptr(), n, stream()), "dt_attn_fwd")
    if isinstance(lib, _Recorder):
        lib.keep.append(a)
    return (out, lse) if return_lse else out


@functools.lru_cache(maxsize=512)
def _grads_plan(q, k, v, kv_len, kv_mask, table, q_pos, distance, two_sided, o, d_o, lse, here):
    if o[1] != q[1] or o[0] != q[0] or o[2][3] != 1 or d_o[1] != q[1] or d_o[0] != q[0] or d_o[2][3] != 1:
        raise DtError("o and d_o must have q's shape and dtype, their head dim contiguous")
    plan, _, bwd, _ = _attn_plan(q, k, v, kv_len, kv_mask, table, q_pos, distance, two_sided, o, here)
    B, Sq, H, D = q[1]
    dense = all(n == 1 or s == want for n, s, want in zip(lse[1], lse[2], (H * Sq, Sq, 1)))
    if lse[0] != _torch().float32 or lse[1] != (B, H, Sq) or not dense and 0 not in lse[1]:
        raise DtError("lse must be the forward pass's: contiguous fp32 [B, H, Sq]")
    _on_device((d_o, o, lse))
    y = AttnGrads()
    y.d_o_strides[:], y.o_strides[:] = d_o[2][:3], o[2][:3]
    y.dq_strides[:] = (Sq * H * D, H * D, D)
    y.dk_strides[:] = y.dv_strides[:] = (k[1][1] * k[1][2] * D, k[1][2] * D, D)
    y.d_rel_table_stride = H
    return plan, bytes(y), bwd


def _attn_bwd(d_o, q, k, v, o, lse, kv_len, kv_mask, scale, rel, q_pos):
    plan, grads, n = _grads_plan(
        _meta(q), _meta(k), _meta(v), _meta(kv_len), _meta(kv_mask), None if rel is None else _meta(rel.table), _meta(q_pos),
        None if rel is None else rel.distance, None if rel is None else rel.two_sided, _meta(o), _meta(d_o), _meta(lse),
        _torch().cuda.current_device())
    a, y = _attn_pointers(plan, q, k, v, kv_len, kv_mask, scale, rel, q_pos), AttnGrads.from_buffer_copy(grads)
    dq, dk, dv = q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(k.shape)
    y.d_o, y.o, y.lse = d_o.data_ptr(), o.data_ptr(), lse.data_ptr()
    y.dq, y.dk, y.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    dt = None
    if rel is not None:
        dt = rel.table.new_empty(rel.table.shape)
        y.d_rel_table = dt.data_ptr()
    lib = load()
    ws = _scratch_by(q, n) if n else None
    check(lib.dt_attn_bwd(ctypes.addressof(a), ctypes.addressof(y), None if ws is None else ws.data_ptr(), n, stream()), "dt_attn_bwd")
    if isinstance(lib, _Recorder):
        lib.keep.extend((a, y))
    return (dq, dk, dv) if rel is None else (dq, dk, dv, dt)


def cross_attn(q, k, v, kv_len=None, kv_mask=None, scale=None, out=None, return_lse=False):
    """softmax over the kept keys of scale q k^T, times v: q [B, Sq, H, D], k and v
    [B, Skv, Hkv, D] (bf16 or fp32, Hkv a divisor of H, D a multiple of 8 up to 128,
    any strides with d contiguous) -> [B, Sq, H, D].  kv_len int32 [B] keeps keys
    below it, kv_mask uint8 or bool [B, Skv] those that are set.  scale: >= 0, by
    default D ** -0.5.  out must not overlap an input.  return_lse: also the log of
    each softmax's sum, fp32 [B, H, Sq], for cross_attn_bwd: autograd records nothing."""
    return _attn(q, k, v, kv_len, kv_mask, scale, None, None, out, return_lse)


def cross_attn_bwd(d_o, q, k, v, o, lse, kv_len=None, kv_mask=None, scale=None):
    """(dq, dk, dv) of cross_attn's o for its gradient d_o."""
    return _attn_bwd(d_o, q, k, v, o, lse, kv_len, kv_mask, scale, None, None)


def rel_attn(q, k, v, rel, q_pos=None, kv_len=None, kv_mask=None, scale=None, out=None, return_lse=False):
    """cross_attn with the bias rel.table[bucket(key - query)] of each head (RelBias)
    added to the scores; query i of batch entry b is at position q_pos[b] + i (int32
    [B]; None: 0), key j at j."""
    return _attn(q, k, v, kv_len, kv_mask, scale, rel, q_pos, out, return_lse)


def rel_attn_bwd(d_o, q, k, v, o, lse, rel, q_pos=None, kv_len=None, kv_mask=None, scale=None):
    """(dq, dk, dv, dtable) of rel_attn's o for its gradient d_o; dtable fp32 [buckets, H]."""
    return _attn_bwd(d_o, q, k, v, o, lse, kv_len, kv_mask, scale, rel, q_pos)


# --------------------------------------------------------------------------
# unfused ops on descriptors
# --------------------------------------------------------------------------

def op_binary(op, a, b, out):
    check(load().dt_op_binary(op, ctypes.byref(desc(a)), ctypes.byref(desc(b)),
                              ctypes.byref(desc(out)), stream()), "dt_op_binary")
    return out


def op_unary(op, a, out, p0=0.0, p1=0.0):
    da = None if a is None else ctypes.byref(desc(a))
    check(load().dt_op_unary(op, da, ctypes.byref(desc(out)), p0, p1, stream()), "dt_op_unary")
    return out


def op_norm(a, out, eps, rms=False):
    fn = load().dt_op_rms_norm if rms else load().dt_op_norm
    check(fn(ctypes.byref(desc(a)), ctypes.byref(desc(out)), eps, stream()), "dt_op_norm")
    return out


def op_rope(a, pos, out, n_dims, freq_base, freq_scale=1.0, attn_factor=1.0, mode=0):
    check(load().dt_op_rope_ext(ctypes.byref(desc(a)), _p(pos), ctypes.byref(desc(out)), n_dims,
                                mode, freq_base, freq_scale, 0.0, attn_factor, stream()),
          "dt_op_rope_ext")
    return out


def op_concat(a, b, dim_ggml, out):
    check(load().dt_op_concat(ctypes.byref(desc(a)), ctypes.byref(desc(b)), dim_ggml,
                              ctypes.byref(desc(out)), stream()), "dt_op_concat")
    return out


def op_cpy(a, out):
    check(load().dt_op_cpy(ctypes.byref(desc(a)), ctypes.byref(desc(out)), stream()), "dt_op_cpy")
    return out
