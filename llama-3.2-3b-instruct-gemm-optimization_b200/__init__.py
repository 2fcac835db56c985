"""Python binding of the b200gemv C ABI (include/b200gemv.h).

The library is the C ABI; this module only marshals arguments.  Device memory
comes from torch tensors (plumbing: allocation, streams); every computation
runs in ``libb200gemv.so``.  There is no fallback: if the library is missing,
``lib()`` raises.

The class names mirror the reference's operator surface:
``GemvOp(in_features, out_features, weight_dtype, scale_mode)`` is the planned
IPluginV3 creator (tensorrt_custom_tactic_kernel_b07f17a4.plan.md:57-58) and
``GemvOp.enqueue(x, W, scales) -> y`` replaces ``run_gemv``
(kernels/gemv_fp8.cu:276-283).  ``I8Op``, ``PagedCache``, ``kv_append`` and
``AttnOp`` (together: ``AttentionBlock``) are the rest of a decoder layer at
any number of rows.
"""
from __future__ import annotations

import ctypes
import struct
from pathlib import Path

HERE = Path(__file__).resolve().parent
LIB_PATH = HERE / "libb200gemv.so"

OK, ERR_INVALID, ERR_UNSUPPORTED, ERR_CUDA, ERR_PEER_TIMEOUT, ERR_OOM, ERR_DEVICE, ERR_SCRATCH_LIMIT = range(8)
STATIC_SCRATCH_BYTES = 2 * 1024 * 1024  # B2G_STATIC_SCRATCH_BYTES
DTYPE = {"fp16": 0, "fp8_e4m3": 1, "bf16": 2, "e4m3": 1}
SCALE = {"none": 0, "tensor_fp16": 1, "channel_fp16": 2, "channel_fp32": 3}
LAYOUT = {"KN": 0, "NK": 1}
FUSE_NONE, FUSE_GATE_UP_SILU, FUSE_RMSNORM_INPUT, FUSE_RESIDUAL_ADD = 0, 1, 2, 4
OPT_MATH, OPT_GRID, OPT_PARTITION, OPT_KSPLIT, OPT_PIPE = 1, 2, 3, 4, 5
PIPE_AUTO, PIPE_REGISTERS, PIPE_TMA = 0, 1, 2
PARTITION_AUTO, PARTITION_UNITS, PARTITION_TILES = 0, 1, 2
MATH_MMA, MATH_FFMA = 0, 1
STACK_OPT_MODE = 1
STACK_MODE_PERSISTENT, STACK_MODE_PER_LAYER, STACK_MODE_PERSISTENT_TMA = 0, 1, 2


class B2GError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {lib().b2g_status_string(status).decode()} (status {status})")


class Fields(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in (
        "in_features", "out_features", "weight_dtype", "scale_mode", "weight_layout", "max_m",
        "fuse", "tp_rank", "tp_size")]


class EnqueueArgs(ctypes.Structure):
    _fields_ = [("m", ctypes.c_int32), ("x", ctypes.c_void_p), ("ldx", ctypes.c_int64),
                ("packed_w", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("residual", ctypes.c_void_p), ("ldr", ctypes.c_int64), ("y", ctypes.c_void_p),
                ("ldy", ctypes.c_int64), ("workspace", ctypes.c_void_p), ("rms_eps", ctypes.c_float),
                ("pdl", ctypes.c_int32), ("prefetch_packed", ctypes.c_void_p),
                ("prefetch_op", ctypes.c_void_p)]


class PlanInfo(ctypes.Structure):
    _fields_ = [("grid", ctypes.c_int32), ("ksplit", ctypes.c_int32),
                ("kblocks_per_vtile", ctypes.c_int32), ("n_tiles", ctypes.c_int32),
                ("total_units", ctypes.c_int64), ("unit_bytes", ctypes.c_int32),
                ("inflight_bytes_per_cta", ctypes.c_int64), ("smem_bytes", ctypes.c_int64), ("max_contrib", ctypes.c_int32),
                ("partition", ctypes.c_int32),
                ("n_slots", ctypes.c_int32), ("x_kblocks", ctypes.c_int32), ("math", ctypes.c_int32),
                ("pipe", ctypes.c_int32), ("n_stages", ctypes.c_int32), ("stage_bytes", ctypes.c_int32)]

    def as_dict(self):
        return {n: getattr(self, n) for n, _ in self._fields_}


class StackFields(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int32), ("intermediate", ctypes.c_int32),
                ("n_layers", ctypes.c_int32), ("weight_dtype", ctypes.c_int32),
                ("scale_mode", ctypes.c_int32), ("max_m", ctypes.c_int32),
                ("rms_eps", ctypes.c_float), ("tp_rank", ctypes.c_int32), ("tp_size", ctypes.c_int32)]


TP_NONE, TP_PUSH, TP_GATHER, TP_REDUCE = 0, 1, 2, 3
TP_MAX_RANKS = 8
TP_MAX_CTAS = 256


class TpComm(ctypes.Structure):
    _fields_ = [("world", ctypes.c_int32), ("rank", ctypes.c_int32), ("max_m", ctypes.c_int32),
                ("width", ctypes.c_int32), ("inbox", ctypes.c_void_p * TP_MAX_RANKS),
                ("counters", ctypes.c_void_p * TP_MAX_RANKS), ("epoch", ctypes.c_void_p)]


class I8RowsArgs(ctypes.Structure):
    _fields_ = [("m", ctypes.c_int32), ("k", ctypes.c_int32), ("dtype", ctypes.c_int32), ("rmsnorm", ctypes.c_int32),
                ("x", ctypes.c_void_p), ("ldx", ctypes.c_int64), ("gamma", ctypes.c_void_p),
                ("rms_eps", ctypes.c_float), ("codes", ctypes.c_void_p), ("ld_codes", ctypes.c_int64),
                ("scales", ctypes.c_void_p)]


class I8Fields(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("in_features", "out_features", "max_m", "dtype", "fuse")]


class I8Args(ctypes.Structure):
    _fields_ = [("m", ctypes.c_int32), ("x", ctypes.c_void_p), ("ldx", ctypes.c_int64), ("gamma", ctypes.c_void_p),
                ("rms_eps", ctypes.c_float), ("x_codes", ctypes.c_void_p), ("ld_codes", ctypes.c_int64),
                ("x_scales", ctypes.c_void_p), ("w_codes", ctypes.c_void_p), ("ldw", ctypes.c_int64),
                ("w_scales", ctypes.c_void_p), ("residual", ctypes.c_void_p), ("ldr", ctypes.c_int64),
                ("y", ctypes.c_void_p), ("ldy", ctypes.c_int64), ("workspace", ctypes.c_void_p)]


class KvCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("stride_page", ctypes.c_int64), ("stride_token", ctypes.c_int64),
                ("stride_head", ctypes.c_int64), ("num_pages", ctypes.c_int32), ("page_size", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


class KvBatch(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int32), ("rows", ctypes.c_int32), ("max_q", ctypes.c_int32),
                ("max_pages", ctypes.c_int32), ("page_table_stride", ctypes.c_int64), ("q_start", ctypes.c_void_p),
                ("seq_lens", ctypes.c_void_p), ("page_table", ctypes.c_void_p)]


class KvAppendArgs(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("q_heads", ctypes.c_int32), ("n_freq", ctypes.c_int32),
                ("interleaved", ctypes.c_int32), ("inv_freq", ctypes.c_void_p),
                ("k", ctypes.c_void_p), ("stride_k", ctypes.c_int64), ("stride_k_head", ctypes.c_int64),
                ("v", ctypes.c_void_p), ("stride_v", ctypes.c_int64), ("stride_v_head", ctypes.c_int64),
                ("q", ctypes.c_void_p), ("stride_q", ctypes.c_int64), ("stride_q_head", ctypes.c_int64),
                ("q_out", ctypes.c_void_p), ("stride_qo", ctypes.c_int64), ("stride_qo_head", ctypes.c_int64)]


class AttnFields(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("q_heads", "kv_heads", "head_dim", "max_batch", "dtype", "cache_dtype")]


class AttnArgs(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("stride_q", ctypes.c_int64), ("stride_q_head", ctypes.c_int64),
                ("out", ctypes.c_void_p), ("stride_o", ctypes.c_int64), ("stride_o_head", ctypes.c_int64),
                ("lse", ctypes.c_void_p), ("scale", ctypes.c_float), ("window", ctypes.c_int32),
                ("workspace", ctypes.c_void_p)]


# Every exported entry point and its ctypes signature (kept in step with
# include/b200gemv.h; the tests check the two agree).
_P, _I32, _I64, _SZ = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_size_t
SIGNATURES = {
    "b2g_status_string": ([ctypes.c_int], ctypes.c_char_p),
    "b2g_version": ([], ctypes.c_int32),
    "b2g_create": ([ctypes.POINTER(Fields), ctypes.POINTER(_P)], ctypes.c_int),
    "b2g_destroy": ([_P], ctypes.c_int),
    "b2g_op_set_option": ([_P, _I32, _I32], ctypes.c_int),
    "b2g_op_query": ([_P, _I32, ctypes.POINTER(PlanInfo)], ctypes.c_int),
    "b2g_plan_for_device": ([ctypes.POINTER(Fields), _I32, _I32, _I32, ctypes.POINTER(PlanInfo),
                             ctypes.POINTER(_SZ), ctypes.POINTER(_SZ)], ctypes.c_int),
    "b2g_prepack_size": ([_P, ctypes.POINTER(_SZ)], ctypes.c_int),
    "b2g_prepack": ([_P, _P, _P, _I64, _P, _P], ctypes.c_int),
    "b2g_quantize_e4m3": ([_P, _I32, _I32, _I32, _I32, _P, _P, _P], ctypes.c_int),
    "b2g_workspace_size": ([_P, _I32, ctypes.POINTER(_SZ)], ctypes.c_int),
    "b2g_workspace_init": ([_P, _P, _P], ctypes.c_int),
    "b2g_enqueue": ([_P, _I32, _P, _P, _P, _P, _P, _P], ctypes.c_int),
    "b2g_enqueue_ex": ([_P, ctypes.POINTER(EnqueueArgs), _P], ctypes.c_int),
    "b2g_device_error": ([ctypes.POINTER(_I32), _I32], ctypes.c_int),
    "b2g_enqueue_static": ([_P, ctypes.POINTER(EnqueueArgs), _P], ctypes.c_int),
    "b2g_tp_comm_bytes": ([_I32, _I32, _I32], _SZ),
    "b2g_tp_comm_layout": ([_P, _I32, _I32, _I32, ctypes.POINTER(_P), ctypes.POINTER(_P), ctypes.POINTER(_P)],
                           ctypes.c_int),
    "b2g_ipc_handle": ([_P, _P], ctypes.c_int),
    "b2g_ipc_open": ([_P, ctypes.POINTER(_P)], ctypes.c_int),
    "b2g_ipc_close": ([_P], ctypes.c_int),
    "b2g_enqueue_tp": ([_P, ctypes.POINTER(EnqueueArgs), ctypes.POINTER(TpComm), _I32, _I32, _P, _P, _I64, _P],
                       ctypes.c_int),
    "b2g_tp_gather": ([ctypes.POINTER(TpComm), _I32, _P, _I32, _P, _I64, _P], ctypes.c_int),
    "b2g_stack_create": ([ctypes.POINTER(StackFields), ctypes.POINTER(_P)], ctypes.c_int),
    "b2g_stack_destroy": ([_P], ctypes.c_int),
    "b2g_stack_ops": ([_P, ctypes.POINTER(_P), ctypes.POINTER(_P)], ctypes.c_int),
    "b2g_stack_set_option": ([_P, _I32, _I32], ctypes.c_int),
    "b2g_stack_set_layer": ([_P, _I32, _P, _P, _P, _P], ctypes.c_int),
    "b2g_stack_workspace_size": ([_P, _I32, ctypes.POINTER(_SZ)], ctypes.c_int),
    "b2g_stack_workspace_init": ([_P, _P, _P], ctypes.c_int),
    "b2g_stack_enqueue": ([_P, _I32, _P, _P, _P, _P], ctypes.c_int),
    "b2g_i8_quantize_rows": ([_P, _P], ctypes.c_int),
    "b2g_i8_quantize_weights": ([_P, _I32, _I32, _I32, _I32, _P, _I64, _P, _P], ctypes.c_int),
    "b2g_i8_create": ([ctypes.POINTER(I8Fields), ctypes.POINTER(_P)], ctypes.c_int),
    "b2g_i8_destroy": ([_P], ctypes.c_int),
    "b2g_i8_workspace_size": ([_P, ctypes.POINTER(_SZ)], ctypes.c_int),
    "b2g_i8_workspace_init": ([_P, _P, _P], ctypes.c_int),
    "b2g_i8_enqueue": ([_P, _P, _P], ctypes.c_int),
    "b2g_kv_append": ([_P, _P, _P, _P], ctypes.c_int),
    "b2g_attn_create": ([ctypes.POINTER(AttnFields), ctypes.POINTER(_P)], ctypes.c_int),
    "b2g_attn_destroy": ([_P], ctypes.c_int),
    "b2g_attn_workspace_size": ([_P, ctypes.POINTER(_SZ)], ctypes.c_int),
    "b2g_attn_workspace_init": ([_P, _P, _P], ctypes.c_int),
    "b2g_attn_enqueue": ([_P, _P, _P, _P, _P],
                         ctypes.c_int),
}

_lib = None


def lib() -> ctypes.CDLL:
    """The C-ABI library.  Raises if it has not been built -- no fallback."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing: build it with build.py (nvcc, sm_100a)")
        L = ctypes.CDLL(str(LIB_PATH))
        for name, (args, res) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        _lib = L
    return _lib


def check(status: int, what: str):
    if status != OK:
        raise B2GError(status, what)


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    import torch
    s = torch.cuda.current_stream() if stream is None else stream
    return ctypes.c_void_p(s.cuda_stream)


def _rows_stride(t):
    """Row stride in elements (a size-1 leading axis may carry any stride)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _code(table, v):
    return table[v] if isinstance(v, str) else int(v)


class GemvOp:
    """One GEMV operator: y[m, N] = epilogue(x[m, K] . W[K, N] * s)."""

    def __init__(self, in_features: int, out_features: int, weight_dtype="fp8_e4m3",
                 scale_mode="channel_fp32", layout="KN", max_m: int = 8, fuse: int = FUSE_NONE,
                 tp_rank: int = 0, tp_size: int = 1, _handle=None):
        self.K, self.N = in_features, out_features
        self.weight_dtype = _code(DTYPE, weight_dtype)
        self.scale_mode = _code(SCALE, scale_mode)
        self.layout = _code(LAYOUT, layout)
        self.max_m, self.fuse = max_m, fuse
        self.planes = 2 if fuse & FUSE_GATE_UP_SILU else 1
        self._owned = _handle is None
        if _handle is None:
            f = Fields(in_features, out_features, self.weight_dtype, self.scale_mode, self.layout,
                       max_m, fuse, tp_rank, tp_size)
            h = ctypes.c_void_p()
            check(lib().b2g_create(ctypes.byref(f), ctypes.byref(h)), "b2g_create")
            self.h = h
        else:
            self.h = _handle

    def __del__(self):
        if getattr(self, "_owned", False) and getattr(self, "h", None) and _lib is not None:
            _lib.b2g_destroy(self.h)
            self.h = None

    # -- planning -------------------------------------------------------
    def set_option(self, key: int, value: int):
        check(lib().b2g_op_set_option(self.h, key, value), "b2g_op_set_option")

    def plan(self, m: int) -> dict:
        info = PlanInfo()
        check(lib().b2g_op_query(self.h, m, ctypes.byref(info)), "b2g_op_query")
        return info.as_dict()

    # -- weights -------------------------------------------------------
    def packed_bytes(self) -> int:
        n = ctypes.c_size_t()
        check(lib().b2g_prepack_size(self.h, ctypes.byref(n)), "b2g_prepack_size")
        return n.value

    def prepack(self, w0, w1=None, out=None, ld: int = 0, stream=None):
        """Repack device weights (op dtype/layout; E4M3 given as uint8) into the stream layout."""
        import torch
        if out is None:
            out = torch.empty(self.packed_bytes(), dtype=torch.uint8, device=w0.device)
        check(lib().b2g_prepack(self.h, _ptr(w0), _ptr(w1), ld, _ptr(out), _stream(stream)),
              "b2g_prepack")
        return out

    # -- workspace ------------------------------------------------------
    def workspace_bytes(self, m=None) -> int:
        n = ctypes.c_size_t()
        check(lib().b2g_workspace_size(self.h, m or self.max_m, ctypes.byref(n)), "b2g_workspace_size")
        return n.value

    def workspace(self, device="cuda", stream=None):
        import torch
        ws = torch.empty(self.workspace_bytes(), dtype=torch.uint8, device=device)
        check(lib().b2g_workspace_init(self.h, _ptr(ws), _stream(stream)), "b2g_workspace_init")
        return ws

    # -- enqueue --------------------------------------------------------
    def enqueue(self, x, packed, scales=None, y=None, workspace=None, residual=None,
                rms_eps: float = 1e-5, pdl: bool = False, stream=None, prefetch=None):
        """y = op(x, W, scales).  prefetch=(next_op, next_packed) warms L2 with the
        start of the weights the next launch in the stream will read."""
        import torch
        m = x.shape[0]
        if y is None:
            y = torch.empty((m, self.N), dtype=torch.float16, device=x.device)
        if workspace is None:
            workspace = self.workspace(x.device, stream)
        if x.stride(-1) != 1 or y.stride(-1) != 1 or (residual is not None and residual.stride(-1) != 1):
            raise ValueError("x, y and residual rows must be contiguous")
        a = EnqueueArgs(m, x.data_ptr(), _rows_stride(x), packed.data_ptr(),
                        0 if scales is None else scales.data_ptr(),
                        0 if residual is None else residual.data_ptr(),
                        0 if residual is None else _rows_stride(residual), y.data_ptr(),
                        _rows_stride(y), workspace.data_ptr(), rms_eps, 1 if pdl else 0,
                        None if prefetch is None else prefetch[1].data_ptr(),
                        None if prefetch is None else prefetch[0].h)
        check(lib().b2g_enqueue_ex(self.h, ctypes.byref(a), _stream(stream)), "b2g_enqueue_ex")
        return y

    def enqueue_tp(self, comm, mode, buf, x, packed, scales=None, y=None, workspace=None, residual=None,
                   rms_eps: float = 1e-5, pdl: bool = False, stream=None, prefetch=None, push_op=None,
                   h_out=None):
        """b2g_enqueue_tp: REDUCE (this op's rows to every rank's inbox, then
        y = the all-reduced rows on every rank), PUSH (the rows to every
        rank's inbox only) or GATHER (stage the all-reduced rows from the
        local inbox, writing them to h_out)."""
        m = x.shape[0]
        a = EnqueueArgs(m, x.data_ptr(), _rows_stride(x), packed.data_ptr(),
                        0 if scales is None else scales.data_ptr(),
                        0 if residual is None else residual.data_ptr(),
                        0 if residual is None else _rows_stride(residual),
                        (x if y is None else y).data_ptr(), self.N if y is None else _rows_stride(y),
                        workspace.data_ptr(), rms_eps, 1 if pdl else 0,
                        None if prefetch is None else prefetch[1].data_ptr(),
                        None if prefetch is None else prefetch[0].h)
        check(lib().b2g_enqueue_tp(self.h, ctypes.byref(a), ctypes.byref(comm), mode, buf,
                                   None if push_op is None else push_op.h,
                                   None if h_out is None else h_out.data_ptr(),
                                   0 if h_out is None else _rows_stride(h_out), _stream(stream)),
              "b2g_enqueue_tp")

    def enqueue_static(self, x, packed, y, scales=None, residual=None, rms_eps: float = 1e-5,
                       stream=None):
        """y = op(x, W, scales) on the library's static scratch (b2g_enqueue_static).

        The library call allocates nothing, so y must be given.  Calls that
        overlap on the device (other streams or threads) race on the scratch.
        """
        if x.stride(-1) != 1 or y.stride(-1) != 1 or (residual is not None and residual.stride(-1) != 1):
            raise ValueError("x, y and residual rows must be contiguous")
        a = EnqueueArgs(x.shape[0], x.data_ptr(), _rows_stride(x), packed.data_ptr(),
                        0 if scales is None else scales.data_ptr(),
                        0 if residual is None else residual.data_ptr(),
                        0 if residual is None else _rows_stride(residual), y.data_ptr(),
                        _rows_stride(y), None, rms_eps, 0, None, None)
        check(lib().b2g_enqueue_static(self.h, ctypes.byref(a), _stream(stream)), "b2g_enqueue_static")
        return y


B200_SMS, B200_SMEM_OPTIN = 148, 232448


def plan_for_device(in_features: int, out_features: int, weight_dtype="fp8_e4m3", scale_mode="channel_fp32",
                    layout="KN", max_m: int = 8, fuse: int = FUSE_NONE, m=None, num_sms: int = B200_SMS,
                    smem_optin: int = B200_SMEM_OPTIN) -> dict:
    """The plan GemvOp would make on a GPU with num_sms SMs (b2g_plan_for_device;
    no device needed), with its packed-weight and workspace bytes."""
    f = Fields(in_features, out_features, _code(DTYPE, weight_dtype), _code(SCALE, scale_mode),
               _code(LAYOUT, layout), max_m, fuse, 0, 1)
    info, pb, wb = PlanInfo(), ctypes.c_size_t(), ctypes.c_size_t()
    check(lib().b2g_plan_for_device(ctypes.byref(f), num_sms, smem_optin, m or max_m, ctypes.byref(info),
                                    ctypes.byref(pb), ctypes.byref(wb)), "b2g_plan_for_device")
    d = info.as_dict()
    d.update(packed_bytes=pb.value, workspace_bytes=wb.value)
    return d


def quantize_e4m3(w16, scale_mode="channel_fp32", layout="KN", stream=None):
    """Device E4M3 quantisation: returns (codes uint8 like w16, scales or None)."""
    import torch
    sm = _code(SCALE, scale_mode)
    lay = _code(LAYOUT, layout)
    K, N = (w16.shape if lay == 0 else w16.shape[::-1])
    q = torch.empty(w16.shape, dtype=torch.uint8, device=w16.device)
    if sm == 0:
        s = None
    elif sm == 1:
        s = torch.empty(1, dtype=torch.float16, device=w16.device)
    elif sm == 2:
        s = torch.empty(N, dtype=torch.float16, device=w16.device)
    else:
        s = torch.empty(N, dtype=torch.float32, device=w16.device)
    check(lib().b2g_quantize_e4m3(_ptr(w16), K, N, lay, sm, _ptr(q), _ptr(s), _stream(stream)),
          "b2g_quantize_e4m3")
    return q, s


def device_error(clear: bool = True) -> int:
    v = ctypes.c_int32()
    check(lib().b2g_device_error(ctypes.byref(v), 1 if clear else 0), "b2g_device_error")
    return v.value


class Stack:
    """The decode-MLP layer stack (RMSNorm -> gate||up+SiLU*up -> down + residual)."""

    def __init__(self, hidden=3072, intermediate=8192, n_layers=28, weight_dtype="fp8_e4m3",
                 scale_mode="channel_fp32", max_m=8, rms_eps=1e-5, tp_rank=0, tp_size=1):
        f = StackFields(hidden, intermediate, n_layers, _code(DTYPE, weight_dtype),
                        _code(SCALE, scale_mode), max_m, rms_eps, tp_rank, tp_size)
        h = ctypes.c_void_p()
        check(lib().b2g_stack_create(ctypes.byref(f), ctypes.byref(h)), "b2g_stack_create")
        self.h = h
        self.hidden, self.intermediate, self.n_layers, self.max_m = hidden, intermediate, n_layers, max_m
        g, d = ctypes.c_void_p(), ctypes.c_void_p()
        check(lib().b2g_stack_ops(self.h, ctypes.byref(g), ctypes.byref(d)), "b2g_stack_ops")
        kw = dict(weight_dtype=weight_dtype, scale_mode=scale_mode, max_m=max_m)
        self.gate_up = GemvOp(hidden, intermediate, fuse=FUSE_GATE_UP_SILU | FUSE_RMSNORM_INPUT,
                              _handle=g, **kw)
        self.down = GemvOp(intermediate, hidden, fuse=FUSE_RESIDUAL_ADD, _handle=d, **kw)
        self._keep = {}

    def __del__(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.b2g_stack_destroy(self.h)
            self.h = None

    def set_mode(self, mode):
        """"per_layer" (two chained launches per layer), "persistent" (one
        cooperative launch) or "persistent_tma" (one cooperative launch, weights
        through the TMA pipeline)."""
        check(lib().b2g_stack_set_option(self.h, STACK_OPT_MODE, _code(
            {"persistent": STACK_MODE_PERSISTENT, "per_layer": STACK_MODE_PER_LAYER,
             "persistent_tma": STACK_MODE_PERSISTENT_TMA}, mode)),
            "b2g_stack_set_option")

    def set_layer(self, layer, packed_gu, scales_gu, packed_d, scales_d):
        self._keep[layer] = (packed_gu, scales_gu, packed_d, scales_d)
        check(lib().b2g_stack_set_layer(self.h, layer, _ptr(packed_gu), _ptr(scales_gu),
                                        _ptr(packed_d), _ptr(scales_d)), "b2g_stack_set_layer")

    def workspace(self, device="cuda", stream=None):
        import torch
        n = ctypes.c_size_t()
        check(lib().b2g_stack_workspace_size(self.h, self.max_m, ctypes.byref(n)),
              "b2g_stack_workspace_size")
        ws = torch.empty(n.value, dtype=torch.uint8, device=device)
        check(lib().b2g_stack_workspace_init(self.h, _ptr(ws), _stream(stream)),
              "b2g_stack_workspace_init")
        return ws

    def enqueue(self, h, act, workspace, stream=None):
        check(lib().b2g_stack_enqueue(self.h, h.shape[0], _ptr(h), _ptr(act), _ptr(workspace),
                                      _stream(stream)), "b2g_stack_enqueue")
        return h


def tp_comm_bytes(world: int, max_m: int, width: int) -> int:
    return lib().b2g_tp_comm_bytes(world, max_m, width)


def tp_comm_layout(base: int, world: int, max_m: int, width: int):
    """(inbox, counters, epoch) device addresses inside a comm buffer at base."""
    i, c, e = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    check(lib().b2g_tp_comm_layout(ctypes.c_void_p(base), world, max_m, width, ctypes.byref(i),
                                   ctypes.byref(c), ctypes.byref(e)), "b2g_tp_comm_layout")
    return i.value, c.value, e.value


IPC_RECORD_BYTES = 72


def ipc_handle(t) -> bytes:
    buf = ctypes.create_string_buffer(IPC_RECORD_BYTES)
    check(lib().b2g_ipc_handle(ctypes.c_void_p(t.data_ptr()), buf), "b2g_ipc_handle")
    return buf.raw


def ipc_open(record: bytes) -> int:
    p = ctypes.c_void_p()
    check(lib().b2g_ipc_open(ctypes.create_string_buffer(record, IPC_RECORD_BYTES), ctypes.byref(p)),
          "b2g_ipc_open")
    return p.value


def ipc_close(addr: int):
    check(lib().b2g_ipc_close(ctypes.c_void_p(addr)), "b2g_ipc_close")


def tp_gather(comm, buf: int, push_op, h, stream=None):
    check(lib().b2g_tp_gather(ctypes.byref(comm), buf, push_op.h, h.shape[0], ctypes.c_void_p(h.data_ptr()),
                              _rows_stride(h), _stream(stream)), "b2g_tp_gather")
    return h


# ---------------------------------------------------------------------------
# 8-bit integer product, paged cache, attention
#
# A decode step's calls take a few microseconds on the device, so what one
# costs in Python is kept small: argument structures are packed into bytes
# (a fifth of a ctypes.Structure's time), a tensor's shape, type and strides
# are read once.
# ---------------------------------------------------------------------------
def _packer(fields):
    """Packs a ctypes.Structure's fields into bytes of its layout (pointers as integers)."""
    code = {ctypes.c_int32: "i", ctypes.c_int64: "q", ctypes.c_void_p: "P", ctypes.c_float: "f"}
    s = struct.Struct("@" + "".join(code[t] for _, t in fields._fields_) + "0q")
    assert s.size == ctypes.sizeof(fields)
    return s.pack


_pack_rows, _pack_i8, _pack_cache, _pack_batch, _pack_append, _pack_attn = map(
    _packer, (I8RowsArgs, I8Args, KvCache, KvBatch, KvAppendArgs, AttnArgs))
_ACT_CODE, _ACT_TYPE, _CACHE_CODE = {}, {}, {}


def _types():
    """torch's types by B2G_DTYPE_* code, and back (torch is imported on first use)."""
    if not _ACT_CODE:
        import torch
        _ACT_TYPE.update({0: torch.float16, 2: torch.bfloat16})
        _CACHE_CODE.update({torch.float16: 0, torch.float8_e4m3fn: 1, torch.bfloat16: 2})
        _ACT_CODE.update({t: c for c, t in _ACT_TYPE.items()})
    return _ACT_TYPE


def _act_code(t):
    _types()
    code = _ACT_CODE.get(t.dtype)
    if code is None:
        raise ValueError(f"expected float16 or bfloat16, got {t.dtype}")
    return code


def _launch(stream, device):
    """(index of the current device, which has to be `device`; the raw stream to
    launch on)."""
    import torch
    if device.type != "cuda":
        raise ValueError(f"tensors on {device}: expected a CUDA device")
    index = device.index
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"tensors are on {device}, the current device is cuda:{torch.cuda.current_device()}")
    if stream is None:
        return index, torch._C._cuda_getCurrentRawStream(index)
    if stream.device != device:
        raise ValueError(f"tensors on {device}, a stream of {stream.device}")
    return index, stream.cuda_stream


def _made(stream, make):
    """A buffer that a call makes for its work on `stream`: allocated under
    that stream, so that the allocator does not hand it on before that work is
    done."""
    if stream is None:
        return make()
    import torch
    with torch.cuda.stream(stream):
        return make()


def _refuse(t, index, dtype, shape, what):
    raise ValueError(f"{what}: expected {list(shape)} {dtype} with contiguous rows on cuda:{index}, got "
                     f"{tuple(t.shape)} {t.dtype} strides {t.stride()} on {t.device}")


def _matrix(t, index, dtype, shape, align, what):
    """The row stride of a matrix with contiguous rows (a single row may carry
    any stride, so it gets an aligned one)."""
    if t.dtype is dtype and t.get_device() == index and t.shape == shape:
        if shape[0] > 1 and t.is_contiguous():
            return shape[1]
        rows, cols = t.stride()
        if cols == 1 or shape[1] == 1:
            return rows if shape[0] > 1 else -(-shape[1] // align) * align
    _refuse(t, index, dtype, shape, what)


def _vector(t, index, dtype, n, what):
    """The address of n elements."""
    if t.dtype is not dtype or t.get_device() != index or t.shape != (n,) or not t.is_contiguous():
        _refuse(t, index, dtype, (n,), what)
    return t.data_ptr()


def _heads(t, index, dtype, shape, what):
    """(address, row stride, head stride) of [rows, heads, dim]."""
    if t.dtype is dtype and t.get_device() == index and t.shape == shape:
        row, head, one = t.stride()
        if one == 1:
            return t.data_ptr(), row, head
    _refuse(t, index, dtype, shape, what)


def _workspace(ws, index, need):
    if ws.get_device() != index or ws.nbytes < need or not ws.is_contiguous():
        raise ValueError(f"the workspace needs {need} contiguous bytes on cuda:{index}")
    return ws.data_ptr()


def _address(t):
    return 0 if t is None else t.data_ptr()


def _codes(rows, cols, device):
    """[rows, cols] int8 whose rows start 16-byte aligned, as the product reads them."""
    import torch
    return torch.empty((rows, -(-cols // 16) * 16), dtype=torch.int8, device=device)[:, :cols]


def quantize_i8_rows(x, gamma=None, rms_eps=None, codes=None, scales=None, stream=None):
    """Codes [m, k] int8 and scales [m] fp32 of 16-bit rows (b2g_i8_quantize_rows).

    With rms_eps the rows are RMS-normalised first (times gamma, if given).
    """
    import torch
    m, k = x.shape
    index, raw = _launch(stream, x.device)
    ldx = _matrix(x, index, x.dtype, (m, k), 8, "x")
    g = 0 if gamma is None else _vector(gamma, index, x.dtype, k, "gamma")
    if codes is None:
        codes = _made(stream, lambda: _codes(m, k, x.device))
    if scales is None:
        scales = _made(stream, lambda: torch.empty(m, dtype=torch.float32, device=x.device))
    ldc = _matrix(codes, index, torch.int8, (m, k), 16, "codes")
    a = _pack_rows(m, k, _act_code(x), rms_eps is not None, x.data_ptr(), ldx, g, rms_eps or 0.0, codes.data_ptr(), ldc,
                   _vector(scales, index, torch.float32, m, "scales"))
    check(lib().b2g_i8_quantize_rows(a, raw), "b2g_i8_quantize_rows")
    return codes, scales


def quantize_i8_weights(w16, layout="KN", stream=None):
    """Codes [N, K] int8 and scales [N] fp32 of 16-bit weights [K, N] (KN) or [N, K] (NK)."""
    import torch
    lay = _code(LAYOUT, layout)
    K, N = (w16.shape if lay == 0 else w16.shape[::-1])
    raw = _launch(stream, w16.device)[1]
    if not w16.is_contiguous():
        raise ValueError("w16 must be contiguous")
    codes = _made(stream, lambda: _codes(N, K, w16.device))
    scales = _made(stream, lambda: torch.empty(N, dtype=torch.float32, device=w16.device))
    check(lib().b2g_i8_quantize_weights(_ptr(w16), K, N, lay, _act_code(w16), _ptr(codes), -(-K // 16) * 16,
                                        _ptr(scales), raw), "b2g_i8_quantize_weights")
    return codes, scales


class I8Op:
    """y[m, N] = epilogue(sx[m] * sw[N] * (x codes [m, K] . w codes [N, K])), any m up to max_m.

    The fusions are GemvOp's: FUSE_RMSNORM_INPUT (rows normalised before they
    are quantised), FUSE_GATE_UP_SILU (w holds the gate rows, then the up
    rows: [2N, K]), FUSE_RESIDUAL_ADD.
    """

    def __init__(self, in_features: int, out_features: int, max_m: int, fuse: int = FUSE_NONE, dtype="fp16"):
        self.K, self.N, self.max_m, self.fuse = in_features, out_features, max_m, fuse
        self.dtype = _code(DTYPE, dtype)
        self.planes = 2 if fuse & FUSE_GATE_UP_SILU else 1
        h, n = ctypes.c_void_p(), ctypes.c_size_t()
        f = I8Fields(in_features, out_features, max_m, self.dtype, fuse)
        check(lib().b2g_i8_create(ctypes.byref(f), ctypes.byref(h)), "b2g_i8_create")
        self.h = h
        check(lib().b2g_i8_workspace_size(self.h, ctypes.byref(n)), "b2g_i8_workspace_size")
        self._ws_bytes = n.value
        self._type = _types()[self.dtype]

    def __del__(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.b2g_i8_destroy(self.h)
            self.h = None

    def workspace_bytes(self) -> int:
        return self._ws_bytes

    def workspace(self, device="cuda", stream=None):
        """A zeroed workspace, for this op only.  Calls that can overlap (other
        streams, graphs replayed at the same time) need one each."""
        import torch
        ws = _made(stream, lambda: torch.empty(self._ws_bytes, dtype=torch.uint8, device=device))
        check(lib().b2g_i8_workspace_init(self.h, _ptr(ws), _stream(stream)), "b2g_i8_workspace_init")
        return ws

    def enqueue(self, x, wq, sw, y=None, workspace=None, residual=None, gamma=None, rms_eps: float = 1e-5,
                stream=None):
        """y of 16-bit rows x [m, K], quantised (and normalised) on the way.  Without
        a workspace one is made and cleared for this call."""
        device, m = x.device, x.shape[0]
        index, raw = _launch(stream, device)
        ldx = _matrix(x, index, self._type, (m, self.K), 8, "x")
        g = 0 if gamma is None else _vector(gamma, index, self._type, self.K, "gamma")
        return self._enqueue(m, device, index, (x.data_ptr(), ldx, g, rms_eps, 0, 0, 0), wq, sw, y, workspace, residual,
                             stream, raw)

    def enqueue_codes(self, xq, sx, wq, sw, y=None, workspace=None, residual=None, stream=None):
        """y of rows that quantize_i8_rows has quantised (one quantisation, several products)."""
        import torch
        device, m = xq.device, xq.shape[0]
        index, raw = _launch(stream, device)
        ldx = _matrix(xq, index, torch.int8, (m, self.K), 16, "xq")
        return self._enqueue(m, device, index, (0, 0, 0, 0.0, xq.data_ptr(), ldx, _vector(sx, index, torch.float32, m, "sx")),
                             wq, sw, y, workspace, residual, stream, raw)

    def _enqueue(self, m, device, index, x_args, wq, sw, y, workspace, residual, stream, raw):
        import torch
        rows, shape = self.planes * self.N, (m, self.N)
        ldw = _matrix(wq, index, torch.int8, (rows, self.K), 16, "wq")
        scales = _vector(sw, index, torch.float32, rows, "sw")
        res, ldr = 0, 0
        if residual is not None:
            res, ldr = residual.data_ptr(), _matrix(residual, index, self._type, shape, 1, "residual")
        if y is None:
            y = _made(stream, lambda: torch.empty(shape, dtype=self._type, device=device))
            ldy = self.N
        else:
            ldy = _matrix(y, index, self._type, shape, 1, "y")
        if workspace is None:
            workspace = self.workspace(device, stream)
        a = _pack_i8(m, *x_args, wq.data_ptr(), ldw, scales, res, ldr, y.data_ptr(), ldy,
                     _workspace(workspace, index, self._ws_bytes))
        status = _lib.b2g_i8_enqueue(self.h, a, raw)
        if status:
            check(status, "b2g_i8_enqueue")
        return y


class PagedCache:
    """A paged key/value cache over two tensors of one shape and strides:
    [pages, page_size, heads, dim] (layout "NHD") or [pages, heads, page_size,
    dim] ("HND"), float16, bfloat16 or float8_e4m3fn.  An 8-bit cache holds
    value / scale[head] (k_scale, v_scale: [heads] float32, None = 1)."""

    def __init__(self, k, v, layout="NHD", k_scale=None, v_scale=None):
        import torch
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride() or k.stride(3) != 1:
            raise ValueError("k and v: two 4-d tensors of one shape, type and strides, the last axis contiguous")
        _types()
        code = _CACHE_CODE.get(k.dtype)
        if code is None or layout not in ("NHD", "HND"):
            raise ValueError(f"cache type {k.dtype}, layout {layout}")
        tok, head = (1, 2) if layout == "NHD" else (2, 1)
        for s in (k_scale, v_scale):
            if s is not None:
                _vector(s, k.get_device(), torch.float32, k.shape[head], "k_scale, v_scale")
        if v.device != k.device:
            raise ValueError("the cache's tensors are on different devices")
        self.k, self.v, self.k_scale, self.v_scale, self.index = k, v, k_scale, v_scale, k.get_device()
        self.page_size, self.kv_heads, self.head_dim, self.dtype = k.shape[tok], k.shape[head], k.shape[3], code
        # The tensors are held above, so their addresses stay theirs.
        self.packed = _pack_cache(k.data_ptr(), v.data_ptr(), _address(k_scale), _address(v_scale), k.stride(0),
                                  k.stride(tok), k.stride(head), k.shape[0], self.page_size, self.kv_heads,
                                  self.head_dim, code)


def _batch(index, rows, q_start, seq_lens, page_table, max_q):
    import torch
    batch = seq_lens.shape[0]
    if page_table.dim() != 2:
        raise ValueError("page_table: expected [batch, pages]")
    pages = page_table.shape[1]
    ld = _matrix(page_table, index, torch.int32, (batch, pages), 1, "page_table")
    return _pack_batch(batch, rows, rows if max_q is None else max_q, pages, ld,
                       _vector(q_start, index, torch.int32, batch + 1, "q_start"),
                       _vector(seq_lens, index, torch.int32, batch, "seq_lens"), page_table.data_ptr())


def _cache(cache, index):
    if cache.index != index:
        raise ValueError(f"the cache is on cuda:{cache.index}, the call's tensors on cuda:{index}")
    return cache.packed


def kv_append(k, v, cache, q_start, seq_lens, page_table, q=None, q_out=None, inv_freq=None,
              interleaved: bool = False, stream=None):
    """Writes the new tokens' k (rotated) and v [rows, kv_heads, dim] into the
    cache's pages, and the rotated q to q_out (default: q itself); b2g_kv_append.

    q_start [batch + 1], seq_lens [batch] (new tokens counted) and page_table
    [batch, pages] are int32.  inv_freq [n] float32 turns the first 2n elements
    of a head by pos * inv_freq (None: no rotation).
    """
    import torch
    rows, dim, t = k.shape[0], cache.head_dim, k.dtype
    index, raw = _launch(stream, k.device)
    shape = (rows, cache.kv_heads, dim)
    heads, qq, qo, n_freq, freq = 0, (0, 0, 0), (0, 0, 0), 0, 0
    if q is not None:
        heads = q.shape[1]
        qq = _heads(q, index, t, (rows, heads, dim), "q")
        qo = qq if q_out is None else _heads(q_out, index, t, (rows, heads, dim), "q_out")
    elif q_out is not None:
        raise ValueError("q_out without q")
    if inv_freq is not None:
        n_freq = inv_freq.shape[0]
        freq = _vector(inv_freq, index, torch.float32, n_freq, "inv_freq")
    a = _pack_append(_act_code(k), heads, n_freq, interleaved, freq, *_heads(k, index, t, shape, "k"),
                     *_heads(v, index, t, shape, "v"), *qq, *qo)
    status = lib().b2g_kv_append(a, _cache(cache, index), _batch(index, rows, q_start, seq_lens, page_table, 1), raw)
    if status:
        check(status, "b2g_kv_append")
    return q if q_out is None else q_out


class AttnOp:
    """Attention of new tokens over a PagedCache (b2g_attn_enqueue): one token
    of a decode step or a chunk of a prompt, ragged over the batch."""

    def __init__(self, q_heads: int, kv_heads: int, head_dim: int, max_batch: int, dtype="fp16", cache_dtype=None):
        self.q_heads, self.kv_heads, self.head_dim, self.max_batch = q_heads, kv_heads, head_dim, max_batch
        self.dtype = _code(DTYPE, dtype)
        self.cache_dtype = self.dtype if cache_dtype is None else _code(DTYPE, cache_dtype)
        h, n = ctypes.c_void_p(), ctypes.c_size_t()
        f = AttnFields(q_heads, kv_heads, head_dim, max_batch, self.dtype, self.cache_dtype)
        check(lib().b2g_attn_create(ctypes.byref(f), ctypes.byref(h)), "b2g_attn_create")
        self.h = h
        check(lib().b2g_attn_workspace_size(self.h, ctypes.byref(n)), "b2g_attn_workspace_size")
        self._ws_bytes = n.value
        self._type = _types()[self.dtype]

    def __del__(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.b2g_attn_destroy(self.h)
            self.h = None

    def workspace_bytes(self) -> int:
        return self._ws_bytes

    def workspace(self, device="cuda", stream=None):
        """A zeroed workspace.  Calls that can overlap (other
        streams, graphs replayed at the same time) need one each."""
        import torch
        ws = _made(stream, lambda: torch.empty(self._ws_bytes, dtype=torch.uint8, device=device))
        check(lib().b2g_attn_workspace_init(self.h, _ptr(ws), _stream(stream)), "b2g_attn_workspace_init")
        return ws

    def enqueue(self, q, cache, q_start, seq_lens, page_table, max_q=None, scale=None, window: int = 0, out=None,
                lse=None, workspace=None, stream=None):
        """out [rows, q_heads, dim] of q (may be q itself); lse [rows, q_heads]
        float32 receives the log-sums.

        max_q: the most new tokens of one sequence (None: unknown), a hint that
        picks the kernel.  scale: default 1 / sqrt(dim).  window: a token sees
        the last `window` positions, its own among them (0: all).  Without a
        workspace one is made and cleared for this call.
        """
        import torch
        rows, device = q.shape[0], q.device
        index, raw = _launch(stream, device)
        shape = (rows, self.q_heads, self.head_dim)
        qq = _heads(q, index, self._type, shape, "q")
        if out is None:
            out = _made(stream, lambda: torch.empty(shape, dtype=self._type, device=device))
            oo = (out.data_ptr(), self.q_heads * self.head_dim, self.head_dim)
        else:
            oo = _heads(out, index, self._type, shape, "out")
        sums = 0
        if lse is not None:
            if lse.dtype is not torch.float32 or lse.get_device() != index or lse.shape != shape[:2] or \
                    not lse.is_contiguous():
                _refuse(lse, index, torch.float32, shape[:2], "lse")
            sums = lse.data_ptr()
        if workspace is None:
            workspace = self.workspace(device, stream)
        a = _pack_attn(*qq, *oo, sums, self.head_dim ** -0.5 if scale is None else scale, window,
                       _workspace(workspace, index, self._ws_bytes))
        status = _lib.b2g_attn_enqueue(self.h, a, _cache(cache, index),
                                       _batch(index, rows, q_start, seq_lens, page_table, max_q), raw)
        if status:
            check(status, "b2g_attn_enqueue")
        return out


class AttentionBlock:
    """The attention half of a decoder layer, beside Stack's MLP half: h (updated
    in place) += out(attention(append(qkv(RMSNorm(h))))), for any number of new
    tokens of each sequence -- a decode step, a prompt chunk, or both.  Rows of
    h behind the last sequence are computed on, from nothing of use.

    wqkv: codes [(q_heads + 2 * kv_heads) * head_dim, hidden] and scales, q
    heads first, then k, then v; wo: codes [hidden, q_heads * head_dim] and
    scales; as quantize_i8_weights leaves them.  gamma: the norm's weights or
    None (1).  inv_freq: the rotation's frequencies (float32, [head_dim / 2]).
    """

    def __init__(self, hidden: int, q_heads: int, kv_heads: int, head_dim: int, max_rows: int, max_batch: int, wqkv, wo,
                 inv_freq, gamma=None, rms_eps: float = 1e-5, dtype="fp16", cache_dtype=None,
                 interleaved: bool = False):
        import torch
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        heads = q_heads + 2 * kv_heads
        self.qkv = I8Op(hidden, heads * head_dim, max_rows, FUSE_RMSNORM_INPUT, dtype)
        self.attn = AttnOp(q_heads, kv_heads, head_dim, max_batch, dtype, cache_dtype)
        self.out = I8Op(q_heads * head_dim, hidden, max_rows, FUSE_RESIDUAL_ADD, dtype)
        self.wqkv, self.wo, self.inv_freq, self.gamma = wqkv, wo, inv_freq, gamma
        self.rms_eps, self.interleaved = rms_eps, interleaved
        self._rows = torch.empty((max_rows, heads, head_dim), dtype=self.qkv._type, device=wqkv[0].device)

    def workspace(self, device="cuda", stream=None):
        """The three ops' workspaces.  Calls that can overlap need their own,
        and a block of their own (it holds the rows between its ops)."""
        return tuple(op.workspace(device, stream) for op in (self.qkv, self.attn, self.out))

    def enqueue(self, h, cache, q_start, seq_lens, page_table, workspace, max_q=None, window: int = 0, stream=None):
        m = h.shape[0]
        if m > self._rows.shape[0]:
            raise ValueError(f"{m} rows: the block was made for {self._rows.shape[0]}")
        rows = self._rows[:m]
        self.qkv.enqueue(h, *self.wqkv, y=rows.view(m, -1), workspace=workspace[0], gamma=self.gamma,
                         rms_eps=self.rms_eps, stream=stream)
        q, k, v = rows.split((self.q_heads, self.kv_heads, self.kv_heads), dim=1)
        kv_append(k, v, cache, q_start, seq_lens, page_table, q=q, inv_freq=self.inv_freq, interleaved=self.interleaved,
                  stream=stream)
        # Each head's result over its q: no row needs another row's q.
        self.attn.enqueue(q, cache, q_start, seq_lens, page_table, max_q=max_q, window=window, out=q,
                          workspace=workspace[1], stream=stream)
        return self.out.enqueue(q.flatten(1), *self.wo, y=h, residual=h, workspace=workspace[2], stream=stream)
