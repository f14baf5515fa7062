"""Python binding of libbsp.so (the C ABI in include/bsp.h), via ctypes; the
decoder-attention entries that are called once a layer and token go through
_bsp_calls.so (csrc/calls.cpp), which costs a call less.

Device memory comes from torch tensors (torch is plumbing here: allocation,
streams, NCCL); every multiply runs in libbsp's sm_100a kernels.  There is no
CPU or torch fallback: if libbsp.so is missing or the call fails, this raises.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
from dataclasses import dataclass
from typing import Optional

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libbsp.so")

BSP_OK, BSP_ERR_INVALID_ARG, BSP_ERR_UNSUPPORTED, BSP_ERR_CUDA, BSP_ERR_TIMEOUT = 0, 1, 2, 3, 4
NAIVE, SNF, DDA = 0, 1, 2
BF16, F32 = 0, 1
STRATEGIES = {"naive": NAIVE, "snf": SNF, "dda": DDA}

# Every symbol the header declares (checked by the CPU test suite).
EXPORTS = [
    "bsp_device_open", "bsp_device_close", "bsp_device_synchronize", "bsp_device_get_error",
    "bsp_device_sm_count", "bsp_last_error_string", "bsp_status_string",
    "bsp_spmm_plan_create", "bsp_spmm_execute", "bsp_spmm_plan_destroy", "bsp_spmm_plan_info",
    "bsp_spmm", "bsp_spmm_host",
    "bsp_sddmm_plan_create", "bsp_sddmm_execute", "bsp_sddmm_plan_destroy",
    "bsp_sddmm_plan_info", "bsp_sddmm", "bsp_sddmm_host",
    "bsp_partition_rows", "bsp_serpentine_assign", "bsp_spmm_host_profile",
    "bsp_sddmm_host_profile", "bsp_spmm_plan_inspect", "bsp_sddmm_plan_inspect",
    "bsp_spmm_noalloc", "bsp_spmm_execute_replicated", "bsp_ipc_export", "bsp_ipc_import",
    "bsp_ipc_close", "bsp_spgemm_plan_create", "bsp_spgemm_pattern", "bsp_spgemm_execute",
    "bsp_spgemm_plan_destroy", "bsp_spgemm_plan_info", "bsp_spgemm_host", "bsp_spgemm_plan_inspect",
    "bsp_attn_plan_create", "bsp_attn_execute", "bsp_attn_plan_destroy", "bsp_attn_plan_info",
    "bsp_attn_host", "bsp_attn_plan_inspect", "bsp_spmm_plan_traffic", "bsp_spmm_plan_entry_rows",
    "bsp_rope_table", "bsp_rope", "bsp_kv_append", "bsp_prompt_plan_create", "bsp_prompt_execute",
    "bsp_prompt_plan_destroy", "bsp_prompt_plan_info", "bsp_prompt_plan_inspect", "bsp_decode_plan_create", "bsp_decode_execute",
    "bsp_decode_plan_destroy", "bsp_decode_plan_info",
]
IPC_HANDLE_BYTES = 64


class BspError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"bsp error {status}: {msg}")
        self.status = status


class BsrDesc(ctypes.Structure):
    _fields_ = [
        ("rows", ctypes.c_int64), ("cols", ctypes.c_int64),
        ("R", ctypes.c_int32), ("C", ctypes.c_int32),
        ("nnzb", ctypes.c_int64),
        ("row_ptr", ctypes.c_void_p), ("col_idx", ctypes.c_void_p), ("values", ctypes.c_void_p),
    ]


class SpmmHostJob(ctypes.Structure):
    """bsp_spmm_host_job: one product of bsp_spmm_host_batch (host arrays)."""
    _fields_ = [
        ("M", ctypes.c_int64), ("K", ctypes.c_int64), ("R", ctypes.c_int32), ("C", ctypes.c_int32),
        ("nnzb", ctypes.c_int64), ("row_ptr", ctypes.c_void_p), ("col_idx", ctypes.c_void_p),
        ("values", ctypes.c_void_p), ("B", ctypes.c_void_p), ("N", ctypes.c_int64), ("C_out", ctypes.c_void_p),
    ]


class RopeScaling(ctypes.Structure):
    """bsp_rope_scaling: how a rotary table is stretched for long contexts."""
    _fields_ = [
        ("kind", ctypes.c_int32), ("factor", ctypes.c_double), ("context", ctypes.c_double),
        ("slow", ctypes.c_double), ("fast", ctypes.c_double), ("magnitude", ctypes.c_double),
    ]


class KvCacheDesc(ctypes.Structure):
    """bsp_kv_cache: a paged 8-bit key/value cache (device pointers)."""
    _fields_ = [
        ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
        ("n_pages", ctypes.c_int64), ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64),
        ("kv_heads", ctypes.c_int32), ("page", ctypes.c_int32), ("d", ctypes.c_int32),
    ]


class Opts(ctypes.Structure):
    _fields_ = [
        ("no_load_balance", ctypes.c_int32), ("group_rows", ctypes.c_int32),
        ("n_tiles", ctypes.c_int32), ("max_ctas", ctypes.c_int32),
        ("timeout_ms", ctypes.c_int32), ("group_mma", ctypes.c_int32),
        ("producers", ctypes.c_int32), ("steps_per_stage", ctypes.c_int32),
    ]


_lib = None


def lib():
    """Load libbsp.so (raises if it was not built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"libbsp.so not built at {LIB_PATH}; run __graft_entry__.build()")
    L = ctypes.CDLL(LIB_PATH)
    P, I64, I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
    S = ctypes.c_int
    sig = {
        "bsp_device_open": (S, [ctypes.c_int, ctypes.POINTER(P)]),
        "bsp_device_close": (S, [P]),
        "bsp_device_synchronize": (S, [P]),
        "bsp_device_get_error": (S, [P, ctypes.POINTER(ctypes.c_uint32)]),
        "bsp_device_sm_count": (ctypes.c_int, [P]),
        "bsp_last_error_string": (ctypes.c_char_p, []),
        "bsp_status_string": (ctypes.c_char_p, [S]),
        "bsp_spmm_plan_create": (S, [P, ctypes.POINTER(BsrDesc), P, P, I64, S, S,
                                     ctypes.POINTER(Opts), ctypes.POINTER(P)]),
        "bsp_spmm_execute": (S, [P, ctypes.POINTER(BsrDesc), P, I64, P, I64, P]),
        "bsp_spmm_plan_destroy": (S, [P]),
        "bsp_spmm_plan_info": (S, [P, ctypes.POINTER(I64)]),
        "bsp_spmm": (S, [P, ctypes.POINTER(BsrDesc), P, I64, P, I64, S, I64, S,
                         ctypes.POINTER(Opts), P]),
        "bsp_spmm_host": (S, [P, I64, I64, I32, I32, I64, P, P, P, P, I64, P, S,
                              ctypes.POINTER(Opts)]),
        "bsp_sddmm_plan_create": (S, [P, ctypes.POINTER(BsrDesc), P, P, I64, S,
                                      ctypes.POINTER(Opts), ctypes.POINTER(P)]),
        "bsp_sddmm_execute": (S, [P, ctypes.POINTER(BsrDesc), P, I64, P, I64, P, P]),
        "bsp_sddmm_plan_destroy": (S, [P]),
        "bsp_sddmm_plan_info": (S, [P, ctypes.POINTER(I64)]),
        "bsp_sddmm": (S, [P, ctypes.POINTER(BsrDesc), P, I64, P, I64, I64, P, S,
                          ctypes.POINTER(Opts), P]),
        "bsp_sddmm_host": (S, [P, I64, I64, I32, I32, I64, P, P, P, P, P, I64, P, S,
                               ctypes.POINTER(Opts)]),
        "bsp_partition_rows": (S, [P, I64, I32, P]),
        "bsp_serpentine_assign": (S, [I64, I32, P, P]),
        "bsp_spmm_host_profile": (S, [P, I64, I64, I32, I32, I64, P, P, P, P, I64, P, S,
                                      ctypes.POINTER(Opts), I32, ctypes.POINTER(ctypes.c_double)]),
        "bsp_sddmm_host_profile": (S, [P, I64, I64, I32, I32, I64, P, P, P, P, P, I64, P, S,
                                       ctypes.POINTER(Opts), I32, ctypes.POINTER(ctypes.c_double)]),
        "bsp_spmm_plan_inspect": (S, [I64, I64, I32, I32, I64, P, P, I64, S, S, ctypes.POINTER(Opts),
                                      I32, I32, P, P, P, P, P, P]),
        "bsp_spmm_noalloc": (S, [ctypes.POINTER(BsrDesc), P, P, P, I64, P, I64, I64, S, S, P]),
        "bsp_spmm_execute_replicated": (S, [P, ctypes.POINTER(BsrDesc), P, I64, P, I64,
                                            ctypes.POINTER(ctypes.c_void_p), I32, P]),
        "bsp_ipc_export": (S, [P, P, P, ctypes.POINTER(ctypes.c_int64)]),
        "bsp_ipc_import": (S, [P, P, ctypes.POINTER(ctypes.c_void_p)]),
        "bsp_ipc_close": (S, [P, P]),
        "bsp_sddmm_plan_inspect": (S, [I64, I64, I32, I32, I64, P, P, I64, S, ctypes.POINTER(Opts),
                                       I32, I32, P, P, P]),
        "bsp_spgemm_plan_create": (S, [P, ctypes.POINTER(BsrDesc), P, P, ctypes.POINTER(BsrDesc),
                                       P, P, ctypes.POINTER(Opts), ctypes.POINTER(P)]),
        "bsp_spgemm_pattern": (S, [P, ctypes.POINTER(I64), P, P]),
        "bsp_spgemm_execute": (S, [P, ctypes.POINTER(BsrDesc), ctypes.POINTER(BsrDesc), P, P]),
        "bsp_spgemm_plan_destroy": (S, [P]),
        "bsp_spgemm_plan_info": (S, [P, ctypes.POINTER(I64)]),
        "bsp_spgemm_host": (S, [P, I64, I64, I64, I32, I32, I32, I64, P, P, P, I64, P, P, P, I64,
                                ctypes.POINTER(I64), P, P, P, ctypes.POINTER(Opts), I32,
                                ctypes.POINTER(ctypes.c_double)]),
        "bsp_spgemm_plan_inspect": (S, [I64, I64, I64, I32, I32, I32, I64, P, P, I64, P, P,
                                        ctypes.POINTER(Opts), I32, I32, P, P, P, P, P, P]),
        "bsp_attn_plan_create": (S, [P, ctypes.POINTER(BsrDesc), P, P, I64, ctypes.POINTER(Opts),
                                     ctypes.POINTER(P)]),
        "bsp_attn_execute": (S, [P, P, I64, P, I64, P, I64, ctypes.c_float, P, I64, P]),
        "bsp_attn_plan_destroy": (S, [P]),
        "bsp_attn_plan_info": (S, [P, ctypes.POINTER(I64)]),
        "bsp_attn_host": (S, [P, I64, I64, I64, P, P, P, P, P, ctypes.c_float, P, ctypes.POINTER(Opts)]),
        "bsp_attn_plan_inspect": (S, [I64, I64, I64, P, P, ctypes.POINTER(Opts), I32, I32, P, P, P, P]),
        "bsp_spmm_plan_traffic": (S, [I64, I64, I32, I32, I64, P, P, I64, S, ctypes.POINTER(Opts), I32, I32,
                                      P, P]),
        "bsp_spmm_plan_entry_rows": (S, [I64, I64, I32, I32, I64, P, P, I64, S, ctypes.POINTER(Opts), I32, I32,
                                         P, ctypes.POINTER(I64)]),
        "bsp_testing_spmm_counters": (S, [P, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(I64),
                                          ctypes.POINTER(I32)]),
        "bsp_testing_spmm_drop_stage": (S, [P, I32]),
        "bsp_spmm_host_batch": (S, [P, I32, ctypes.POINTER(SpmmHostJob), S, ctypes.POINTER(Opts)]),
        "bsp_bsr_upload": (S, [P, I64, I64, I32, I32, I64, P, P, P, ctypes.POINTER(BsrDesc)]),
        "bsp_bsr_free": (S, [P, ctypes.POINTER(BsrDesc)]),
        "bsp_buffer_alloc": (S, [P, I64, ctypes.POINTER(ctypes.c_void_p)]),
        "bsp_buffer_free": (S, [P, P]),
        "bsp_buffer_write": (S, [P, P, P, I64]),
        "bsp_buffer_read": (S, [P, P, P, I64]),
        "bsp_rope_table": (S, [P, I64, I32, ctypes.c_double, ctypes.POINTER(RopeScaling), P, P]),
        "bsp_rope": (S, [P, P, I64, I64, P, P, I64, I64, I32, I32, I32, S, I32, S, P, I64, I64, P]),
        "bsp_kv_append": (S, [P, ctypes.POINTER(KvCacheDesc), P, I64, I64, P, I64, I64, I64, I32, P, P, P, I64, I64,
                              P, I64, I32, S, P, I64, I64, I32, P, I64, I64, P, I64, I64, P]),
        "bsp_prompt_plan_create": (S, [P, I32, P, P, I32, I32, I32, I32, ctypes.POINTER(Opts), ctypes.POINTER(P)]),
        "bsp_prompt_execute": (S, [P, P, I64, I64, P, I64, I64, P, I64, I64, ctypes.c_float, P, I64, I64, P, P]),
        "bsp_prompt_plan_destroy": (S, [P]),
        "bsp_prompt_plan_info": (S, [P, ctypes.POINTER(I64)]),
        "bsp_prompt_plan_inspect": (S, [I32, P, P, I32, I32, I32, I32, ctypes.POINTER(Opts), I32, P, P, P]),
        "bsp_decode_plan_create": (S, [P, I32, I32, I32, I32, I32, ctypes.POINTER(Opts), ctypes.POINTER(P)]),
        "bsp_decode_execute": (S, [P, ctypes.POINTER(KvCacheDesc), P, I64, I64, I32, P, P, I64, I64, ctypes.c_float,
                                   P, I64, I64, P, P]),
        "bsp_decode_plan_destroy": (S, [P]),
        "bsp_decode_plan_info": (S, [P, ctypes.POINTER(I64)]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def _check(status: int):
    if status != BSP_OK:
        raise BspError(status, lib().bsp_last_error_string().decode())


def make_opts(**kw) -> Opts:
    o = Opts()
    for k, v in kw.items():
        if v is not None:
            setattr(o, k, int(v))
    return o


def _ptr(a) -> Optional[int]:
    if a is None:
        return None
    if hasattr(a, "data_ptr"):
        return a.data_ptr()
    return a.ctypes.data


# ------------------------------------------------------------------ device --
class Device:
    """A B200 (sm_100a) opened through the library (reference: IDevice*)."""

    def __init__(self, ordinal: int = 0):
        h = ctypes.c_void_p()
        _check(lib().bsp_device_open(ordinal, ctypes.byref(h)))
        self.handle = h
        self.ordinal = ordinal

    @property
    def sm_count(self) -> int:
        return lib().bsp_device_sm_count(self.handle)

    def synchronize(self):
        _check(lib().bsp_device_synchronize(self.handle))

    def status_bits(self) -> int:
        v = ctypes.c_uint32()
        _check(lib().bsp_device_get_error(self.handle, ctypes.byref(v)))
        return v.value

    def close(self):
        if self.handle:
            lib().bsp_device_close(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_default = {}


def device(ordinal: int = 0) -> Device:
    if ordinal not in _default:
        _default[ordinal] = Device(ordinal)
    return _default[ordinal]


# ---------------------------------------------------------------- BSR data --
@dataclass
class DeviceBSR:
    """A BSR matrix resident on the GPU (torch tensors) plus its host pattern."""

    rows: int
    cols: int
    R: int
    C: int
    row_ptr: "object"   # torch int32 cuda
    col_idx: "object"   # torch int32 cuda
    values: "object"    # torch bf16 cuda, [nnzb*R*C] (or None for a pattern-only mask)
    h_row_ptr: np.ndarray
    h_col_idx: np.ndarray

    @property
    def nnzb(self) -> int:
        return int(self.h_row_ptr[-1])

    def desc(self) -> BsrDesc:
        return BsrDesc(self.rows, self.cols, self.R, self.C, self.nnzb,
                       _ptr(self.row_ptr), _ptr(self.col_idx), _ptr(self.values))

    @staticmethod
    def from_host(rows, cols, R, C, row_ptr, col_idx, values_bf16_bits=None, device_index=0):
        import torch
        dev = torch.device("cuda", device_index)
        rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
        ci = np.ascontiguousarray(col_idx, dtype=np.int32)
        t_rp = torch.from_numpy(rp).to(dev)
        t_ci = torch.from_numpy(ci if ci.size else np.zeros(1, np.int32)).to(dev)
        t_v = None
        if values_bf16_bits is not None:
            v = np.ascontiguousarray(values_bf16_bits, dtype=np.uint16).ravel()
            if v.size == 0:
                v = np.zeros(8, np.uint16)
            t_v = torch.from_numpy(v.view(np.int16)).to(dev).view(torch.bfloat16)
        return DeviceBSR(rows, cols, R, C, t_rp, t_ci, t_v, rp, ci)


def to_device_bf16(bits: np.ndarray, device_index=0):
    import torch
    a = np.ascontiguousarray(bits, dtype=np.uint16)
    return torch.from_numpy(a.view(np.int16)).to(torch.device("cuda", device_index)).view(torch.bfloat16)


def to_host_bits(t) -> np.ndarray:
    import torch
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


def _stream_ptr(stream) -> Optional[int]:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


# -------------------------------------------------------------------- SpMM --
class SpmmPlan:
    """Reusable SpMM plan for one pattern and one N (reference: the planner)."""

    def __init__(self, dev: Device, A: DeviceBSR, N: int, strategy=NAIVE, c_type=BF16, opts=None):
        self.dev, self.N, self.c_type = dev, N, c_type
        self._desc = A.desc()
        h = ctypes.c_void_p()
        o = opts if opts is not None else Opts()
        _check(lib().bsp_spmm_plan_create(dev.handle, ctypes.byref(self._desc),
                                          _ptr(A.h_row_ptr), _ptr(A.h_col_idx), N, c_type,
                                          strategy, ctypes.byref(o), ctypes.byref(h)))
        self.handle = h

    def info(self) -> dict:
        arr = (ctypes.c_int64 * 16)()
        _check(lib().bsp_spmm_plan_info(self.handle, arr))
        keys = ["units", "ctas", "group_rows", "n_tiles", "slab", "kc", "stages", "steps",
                "plan_bytes", "smem_bytes", "tmem_cols", "variant", "producers"]
        return {k: int(arr[i]) for i, k in enumerate(keys)}

    def execute(self, A: DeviceBSR, B, C, stream=None):
        d = A.desc()
        _check(lib().bsp_spmm_execute(self.handle, ctypes.byref(d), _ptr(B), B.stride(0), _ptr(C),
                                      C.stride(0), _stream_ptr(stream)))

    def execute_replicated(self, A: DeviceBSR, B, C, peer_ptrs, stream=None):
        """execute(), and every C store repeated into the peers' C buffers
        (device pointers of the element matching C[0][0] on each peer)."""
        d = A.desc()
        arr = (ctypes.c_void_p * max(len(peer_ptrs), 1))(*[int(x) for x in peer_ptrs])
        _check(lib().bsp_spmm_execute_replicated(self.handle, ctypes.byref(d), _ptr(B), B.stride(0),
                                                 _ptr(C), C.stride(0), arr, len(peer_ptrs),
                                                 _stream_ptr(stream)))

    def close(self):
        if self.handle:
            lib().bsp_spmm_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def spmm(A: DeviceBSR, B, strategy=NAIVE, c_type=BF16, opts=None, dev: Device = None):
    """One-shot C = A @ B on the GPU (B: torch bf16 cuda [K, N]); returns C."""
    import torch
    dev = dev or device(B.device.index or 0)
    N = B.shape[1]
    C = torch.empty((A.rows, N), dtype=torch.float32 if c_type == F32 else torch.bfloat16,
                    device=B.device)
    plan = SpmmPlan(dev, A, N, strategy, c_type, opts)
    plan.execute(A, B, C)
    dev.synchronize()
    plan.close()
    return C


def spmm_host(M, K, R, C, row_ptr, col_idx, values, B, N, strategy=NAIVE, opts=None,
              dev: Device = None, out=None) -> np.ndarray:
    """Host buffers in, host C out (reference planner semantics)."""
    dev = dev or device(0)
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    ci = np.ascontiguousarray(col_idx, dtype=np.int32)
    v = np.ascontiguousarray(values, dtype=np.uint16)
    b = np.ascontiguousarray(B, dtype=np.uint16)
    o = out if out is not None else np.empty((M, N), dtype=np.uint16)
    opt = opts if opts is not None else Opts()
    _check(lib().bsp_spmm_host(dev.handle, M, K, R, C, int(rp[-1]), _ptr(rp), _ptr(ci), _ptr(v),
                               _ptr(b), N, _ptr(o), strategy, ctypes.byref(opt)))
    return o


def spmm_host_batch(jobs, strategy=NAIVE, opts=None, dev: Device = None):
    """Several host-buffer SpMMs in one pipelined call (bsp_spmm_host_batch).
    jobs: sequence of dicts with M, K, R, C, row_ptr, col_idx, values, B, N and
    optionally out (a uint16 M x N array to write); returns the outputs."""
    dev = dev or device(0)
    keep, arr = [], (SpmmHostJob * max(len(jobs), 1))()
    outs = []
    for k, j in enumerate(jobs):
        rp = np.ascontiguousarray(j["row_ptr"], dtype=np.int32)
        ci = np.ascontiguousarray(j["col_idx"], dtype=np.int32)
        v = np.ascontiguousarray(j["values"], dtype=np.uint16)
        b = np.ascontiguousarray(j["B"], dtype=np.uint16)
        o = j.get("out")
        if o is None:
            o = np.empty((j["M"], j["N"]), dtype=np.uint16)
        keep += [rp, ci, v, b, o]
        outs.append(o)
        arr[k] = SpmmHostJob(j["M"], j["K"], j["R"], j["C"], int(rp[-1]), _ptr(rp), _ptr(ci), _ptr(v), _ptr(b),
                             j["N"], _ptr(o))
    opt = opts if opts is not None else Opts()
    _check(lib().bsp_spmm_host_batch(dev.handle, len(jobs), arr, strategy, ctypes.byref(opt)))
    return outs


# ------------------------------------------------------------------- SDDMM --
class SddmmPlan:
    def __init__(self, dev: Device, mask: DeviceBSR, K: int, strategy=NAIVE, opts=None):
        self.dev, self.K = dev, K
        self._desc = mask.desc()
        h = ctypes.c_void_p()
        o = opts if opts is not None else Opts()
        _check(lib().bsp_sddmm_plan_create(dev.handle, ctypes.byref(self._desc),
                                           _ptr(mask.h_row_ptr), _ptr(mask.h_col_idx), K,
                                           strategy, ctypes.byref(o), ctypes.byref(h)))
        self.handle = h

    def info(self) -> dict:
        arr = (ctypes.c_int64 * 16)()
        _check(lib().bsp_sddmm_plan_info(self.handle, arr))
        keys = ["units", "ctas", "_2", "_3", "slab", "kc", "stages", "keep_a", "plan_bytes",
                "smem_bytes", "tmem_cols", "variant", "_12", "nseg_max", "producers"]
        return {k: int(arr[i]) for i, k in enumerate(keys) if not k.startswith("_")}

    def execute(self, mask: DeviceBSR, A, B, out, stream=None):
        d = mask.desc()
        _check(lib().bsp_sddmm_execute(self.handle, ctypes.byref(d), _ptr(A), A.stride(0), _ptr(B),
                                       B.stride(0), _ptr(out), _stream_ptr(stream)))

    def close(self):
        if self.handle:
            lib().bsp_sddmm_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def sddmm(mask: DeviceBSR, A, B, strategy=NAIVE, opts=None, dev: Device = None):
    """One-shot out = mask (.) (A @ B) on the mask's pattern; returns bf16 block values."""
    import torch
    dev = dev or device(A.device.index or 0)
    out = torch.empty(max(mask.nnzb * mask.R * mask.C, 8), dtype=torch.bfloat16, device=A.device)
    plan = SddmmPlan(dev, mask, A.shape[1], strategy, opts)
    plan.execute(mask, A, B, out)
    dev.synchronize()
    plan.close()
    return out[: mask.nnzb * mask.R * mask.C]


def sddmm_host(M, N, R, C, row_ptr, col_idx, mask_values, A, B, K, strategy=NAIVE, opts=None,
               dev: Device = None, out=None) -> np.ndarray:
    dev = dev or device(0)
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    ci = np.ascontiguousarray(col_idx, dtype=np.int32)
    mv = None if mask_values is None else np.ascontiguousarray(mask_values, dtype=np.uint16)
    a = np.ascontiguousarray(A, dtype=np.uint16)
    b = np.ascontiguousarray(B, dtype=np.uint16)
    nnzb = int(rp[-1])
    o = out if out is not None else np.empty(nnzb * R * C, dtype=np.uint16)
    opt = opts if opts is not None else Opts()
    _check(lib().bsp_sddmm_host(dev.handle, M, N, R, C, nnzb, _ptr(rp), _ptr(ci), _ptr(mv),
                                _ptr(a), _ptr(b), K, _ptr(o), strategy, ctypes.byref(opt)))
    return o


# ------------------------------------------------------------------ SpGEMM --
SPGEMM_INFO_KEYS = ["units", "ctas", "steps", "pairs", "out_nnzb", "kc", "stages",
                    "steps_per_stage", "plan_bytes", "smem_bytes", "tmem_cols", "nseg_max",
                    "producers", "boxes"]


class SpgemmPlan:
    """C = A @ B for two BSR matrices (bsr_matrix<T>::spgemm,
    sparse_common/bsr_matrix.hpp:741-810); the plan holds C's pattern."""

    def __init__(self, dev: Device, A: DeviceBSR, B: DeviceBSR, opts=None):
        self.dev = dev
        self.M, self.N, self.Ra, self.Cb = A.rows, B.cols, A.R, B.C
        da, db = A.desc(), B.desc()
        h = ctypes.c_void_p()
        o = opts if opts is not None else Opts()
        _check(lib().bsp_spgemm_plan_create(dev.handle, ctypes.byref(da), _ptr(A.h_row_ptr),
                                            _ptr(A.h_col_idx), ctypes.byref(db), _ptr(B.h_row_ptr),
                                            _ptr(B.h_col_idx), ctypes.byref(o), ctypes.byref(h)))
        self.handle = h
        n = ctypes.c_int64()
        _check(lib().bsp_spgemm_pattern(h, ctypes.byref(n), None, None))
        self.nnzb = int(n.value)
        self.row_ptr = np.zeros(self.M // self.Ra + 1, np.int32)
        self.col_idx = np.zeros(max(self.nnzb, 1), np.int32)
        _check(lib().bsp_spgemm_pattern(h, ctypes.byref(n), _ptr(self.row_ptr), _ptr(self.col_idx)))
        self.col_idx = self.col_idx[: self.nnzb]

    def info(self) -> dict:
        arr = (ctypes.c_int64 * 16)()
        _check(lib().bsp_spgemm_plan_info(self.handle, arr))
        return {k: int(arr[i]) for i, k in enumerate(SPGEMM_INFO_KEYS)}

    def execute(self, A: DeviceBSR, B: DeviceBSR, out, stream=None):
        """out: device bf16, at least nnzb * Ra * Cb elements."""
        da, db = A.desc(), B.desc()
        _check(lib().bsp_spgemm_execute(self.handle, ctypes.byref(da), ctypes.byref(db), _ptr(out),
                                        _stream_ptr(stream)))

    def close(self):
        if self.handle:
            lib().bsp_spgemm_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def spgemm(A: DeviceBSR, B: DeviceBSR, opts=None, dev: Device = None) -> DeviceBSR:
    """One-shot C = A @ B (both BSR on the GPU); returns C as a DeviceBSR."""
    import torch
    dev = dev or device(A.values.device.index or 0)
    plan = SpgemmPlan(dev, A, B, opts)
    out = torch.empty(max(plan.nnzb * A.R * B.C, 8), dtype=torch.bfloat16, device=A.values.device)
    plan.execute(A, B, out)
    dev.synchronize()
    C = DeviceBSR(A.rows, B.cols, A.R, B.C,
                  torch.from_numpy(plan.row_ptr.copy()).to(out.device),
                  torch.from_numpy(plan.col_idx.copy() if plan.nnzb else np.zeros(1, np.int32)).to(out.device),
                  out, plan.row_ptr.copy(), plan.col_idx.copy())
    plan.close()
    return C


def spgemm_host(M, K, N, Ra, Ca, Cb, a_row_ptr, a_col_idx, a_values, b_row_ptr, b_col_idx,
                b_values, opts=None, dev: Device = None, iters=0):
    """Host BSR in, host BSR out: (row_ptr, col_idx, values bf16 bits) of A @ B
    (bsr_matrix<T>::spgemm semantics), plus the mean launch time in ms when
    iters > 0.  Uploads, plans once (C's pattern on the host), runs, downloads."""
    import torch

    dev = dev or device(0)
    A = DeviceBSR.from_host(M, K, Ra, Ca, a_row_ptr, a_col_idx, a_values, dev.ordinal)
    B = DeviceBSR.from_host(K, N, Ca, Cb, b_row_ptr, b_col_idx, b_values, dev.ordinal)
    plan = SpgemmPlan(dev, A, B, opts)
    n = plan.nnzb * Ra * Cb
    out = torch.empty(max(n, 8), dtype=torch.bfloat16, device=A.row_ptr.device)
    plan.execute(A, B, out)
    ms = 0.0
    if iters > 0:
        e0 = torch.cuda.Event(enable_timing=True)
        e1 = torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(iters):
            plan.execute(A, B, out)
        e1.record()
        e1.synchronize()
        ms = e0.elapsed_time(e1) / iters
    dev.synchronize()
    res = (plan.row_ptr.copy(), plan.col_idx.copy(), to_host_bits(out)[:n])
    plan.close()
    return res + (ms,) if iters > 0 else res


def spgemm_host_c(M, K, N, Ra, Ca, Cb, a_row_ptr, a_col_idx, a_values, b_row_ptr, b_col_idx,
                  b_values, opts=None, dev: Device = None, iters=0):
    """The same through the C ABI's host-buffer entry point bsp_spgemm_host
    (a size query, then the product: C's pattern is planned twice)."""
    dev = dev or device(0)
    arp = np.ascontiguousarray(a_row_ptr, dtype=np.int32)
    aci = np.ascontiguousarray(a_col_idx, dtype=np.int32)
    av = np.ascontiguousarray(a_values, dtype=np.uint16)
    brp = np.ascontiguousarray(b_row_ptr, dtype=np.int32)
    bci = np.ascontiguousarray(b_col_idx, dtype=np.int32)
    bv = np.ascontiguousarray(b_values, dtype=np.uint16)
    opt = opts if opts is not None else Opts()
    n = ctypes.c_int64()
    ms = ctypes.c_double(0.0)
    common = (dev.handle, M, K, N, Ra, Ca, Cb, int(arp[-1]), _ptr(arp), _ptr(aci), _ptr(av),
              int(brp[-1]), _ptr(brp), _ptr(bci), _ptr(bv))
    _check(lib().bsp_spgemm_host(*common, 0, ctypes.byref(n), None, None, None, ctypes.byref(opt),
                                 0, None))
    cap = int(n.value)
    orp = np.zeros(M // Ra + 1, np.int32)
    oci = np.zeros(max(cap, 1), np.int32)
    ov = np.zeros(max(cap * Ra * Cb, 8), np.uint16)
    _check(lib().bsp_spgemm_host(*common, cap, ctypes.byref(n), _ptr(orp), _ptr(oci), _ptr(ov),
                                 ctypes.byref(opt), iters, ctypes.byref(ms)))
    res = (orp, oci[:cap], ov[: cap * Ra * Cb])
    return res + (ms.value,) if iters > 0 else res


def inspect_spgemm_plan(M, K, N, Ra, Ca, Cb, a_row_ptr, a_col_idx, b_row_ptr, b_col_idx, opts=None,
                        sm_count=148, max_smem=232448):
    """Run the SpGEMM planner on the host only (no GPU) and return its schedule."""
    arp = np.ascontiguousarray(a_row_ptr, dtype=np.int32)
    aci = np.ascontiguousarray(a_col_idx, dtype=np.int32)
    brp = np.ascontiguousarray(b_row_ptr, dtype=np.int32)
    bci = np.ascontiguousarray(b_col_idx, dtype=np.int32)
    aci = aci if aci.size else np.zeros(1, np.int32)
    bci = bci if bci.size else np.zeros(1, np.int32)
    info = np.zeros(16, np.int64)
    o = opts if opts is not None else Opts()
    args = (M, K, N, Ra, Ca, Cb, int(arp[-1]), _ptr(arp), _ptr(aci), int(brp[-1]), _ptr(brp),
            _ptr(bci), ctypes.byref(o), sm_count, max_smem, _ptr(info))
    _check(lib().bsp_spgemm_plan_inspect(*args, None, None, None, None, None))
    nu, ns, nb, nc = int(info[0]), int(info[2]), int(info[4]), int(info[1])
    orp = np.zeros(M // Ra + 1, np.int32)
    oci = np.zeros(max(nb, 1), np.int32)
    units = np.zeros((max(nu, 1), 48), np.int32)
    steps = np.zeros((max(ns, 1), 16), np.int32)
    cta = np.zeros(nc + 1, np.int32)
    _check(lib().bsp_spgemm_plan_inspect(*args, _ptr(orp), _ptr(oci), _ptr(units), _ptr(steps),
                                         _ptr(cta)))
    d = {k: int(info[i]) for i, k in enumerate(SPGEMM_INFO_KEYS)}
    d.update(out_row_ptr=orp, out_col_idx=oci[:nb], unit_table=units[:nu], step_table=steps[:ns],
             cta_begin=cta)
    return d


# --------------------------------------------------------------- attention --
ATTN_INFO_KEYS = ["units", "ctas", "chunks", "mask_blocks", "S", "d", "parts", "split_units",
                  "plan_bytes", "smem_bytes", "tmem_cols"]


class AttnPlan:
    """Fused block-sparse attention step for one mask pattern and head size:
    O = softmax_rows(scale * Q K^T on the mask's blocks) V (the reference's
    SDDMM -> softmax -> SpMM chain in one kernel)."""

    def __init__(self, dev: Device, mask: DeviceBSR, d: int, opts=None):
        self.dev, self.d, self.S = dev, d, mask.rows
        self._desc = mask.desc()
        h = ctypes.c_void_p()
        o = opts if opts is not None else Opts()
        _check(lib().bsp_attn_plan_create(dev.handle, ctypes.byref(self._desc), _ptr(mask.h_row_ptr),
                                          _ptr(mask.h_col_idx), d, ctypes.byref(o), ctypes.byref(h)))
        self.handle = h

    def info(self) -> dict:
        arr = (ctypes.c_int64 * 16)()
        _check(lib().bsp_attn_plan_info(self.handle, arr))
        return {k: int(arr[i]) for i, k in enumerate(ATTN_INFO_KEYS) if not k.startswith("_")}

    def execute(self, Q, K, V, O, scale=None, stream=None):
        """Q, K, V, O: torch bf16 cuda [S, d] (row strides may exceed d)."""
        sc = float(scale) if scale is not None else 1.0 / float(np.sqrt(self.d))
        _check(lib().bsp_attn_execute(self.handle, _ptr(Q), Q.stride(0), _ptr(K), K.stride(0), _ptr(V),
                                      V.stride(0), sc, _ptr(O), O.stride(0), _stream_ptr(stream)))

    def close(self):
        if self.handle:
            lib().bsp_attn_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def attention(mask: DeviceBSR, Q, K, V, scale=None, opts=None, dev: Device = None):
    """One-shot fused attention step on device tensors; returns O."""
    import torch

    dev = dev or device(Q.device.index or 0)
    O = torch.empty_like(Q)
    plan = AttnPlan(dev, mask, Q.shape[1], opts)
    plan.execute(Q, K, V, O, scale)
    dev.synchronize()
    plan.close()
    return O


def attn_host(S, d, row_ptr, col_idx, Q, K, V, scale=None, opts=None, dev: Device = None):
    """Host arrays in (pattern, Q, K, V bf16 bits), host O out (bsp_attn_host)."""
    dev = dev or device(0)
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    ci = np.ascontiguousarray(col_idx, dtype=np.int32)
    q = np.ascontiguousarray(Q, dtype=np.uint16)
    k = np.ascontiguousarray(K, dtype=np.uint16)
    v = np.ascontiguousarray(V, dtype=np.uint16)
    o = np.empty((S, d), dtype=np.uint16)
    sc = float(scale) if scale is not None else 1.0 / float(np.sqrt(d))
    opt = opts if opts is not None else Opts()
    _check(lib().bsp_attn_host(dev.handle, S, d, int(rp[-1]), _ptr(rp), _ptr(ci), _ptr(q), _ptr(k), _ptr(v),
                               sc, _ptr(o), ctypes.byref(opt)))
    return o


def inspect_attn_plan(S, d, row_ptr, col_idx, opts=None, sm_count=148, max_smem=232448):
    """Run the attention planner on the host only (no GPU)."""
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    ci = np.ascontiguousarray(col_idx, dtype=np.int32)
    ci = ci if ci.size else np.zeros(1, np.int32)
    info = np.zeros(16, np.int64)
    o = opts if opts is not None else Opts()
    args = (S, d, int(rp[-1]), _ptr(rp), _ptr(ci), ctypes.byref(o), sm_count, max_smem, _ptr(info))
    _check(lib().bsp_attn_plan_inspect(*args, None, None, None))
    units = np.zeros((max(int(info[0]), 1), 8), np.int32)
    chunks = np.zeros((max(int(info[2]), 1), 8), np.int32)
    cta = np.zeros(int(info[1]) + 1, np.int32)
    _check(lib().bsp_attn_plan_inspect(*args, _ptr(units), _ptr(chunks), _ptr(cta)))
    dd = {k: int(info[i]) for i, k in enumerate(ATTN_INFO_KEYS) if not k.startswith("_")}
    dd.update(unit_table=units[: int(info[0])], chunk_table=chunks[: int(info[2])], cta_begin=cta)
    return dd


# ------------------------------------------- attention of a decoder model --
ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
ROPE_KINDS = {"none": 0, "linear": 1, "base": 2, "parts": 3}


_calls = None


def _load_calls():
    """The module through which these entries are called with torch tensors
    (csrc/calls.cpp); raises if it was not built."""
    global _calls
    import torch  # noqa: F401  (the module resolves its symbols)

    lib()
    path = os.path.join(HERE, "_bsp_calls.so")
    if not os.path.exists(path):
        raise RuntimeError(f"_bsp_calls.so not built at {path}; run __graft_entry__.build()")
    spec = importlib.util.spec_from_file_location("_bsp_calls", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.setup(BspError, device)
    _calls = m
    return m


def _stream_of(stream, dev: Device):
    """Stream number: the given stream, or the current one of dev's GPU."""
    if stream is None:
        import torch

        return torch.cuda.current_stream(dev.ordinal).cuda_stream
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _empty(shape, dtype, device, stream):
    """An output that a call on `stream` makes: it belongs to that stream, so its
    memory is none that kernels still running on the current one may use."""
    import torch

    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(_stream_of(stream, None), device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _refuse(msg):
    raise BspError(BSP_ERR_INVALID_ARG, msg)


def _rope_layout(layout):
    if layout not in ROPE_LAYOUTS:
        _refuse(f"rotary layout {layout!r}: one of {sorted(ROPE_LAYOUTS)}")
    return ROPE_LAYOUTS[layout]


def rope_table(n_pos, rot, base=10000.0, kind="none", factor=1.0, context=0.0, slow=1.0, fast=32.0, magnitude=1.0,
               dev: Device = None, stream=None):
    """Rotary table [n_pos, rot / 2, 2] of (cos, sin) for `rot` rotated values
    of each head; kind "linear", "base" or "parts" stretches it for contexts
    longer than trained (bsp_rope_table)."""
    import torch

    dev = dev or device(torch.cuda.current_device())
    if kind not in ROPE_KINDS:
        _refuse(f"scaling {kind!r}: one of {sorted(ROPE_KINDS)}")
    if n_pos < 1 or rot < 2:
        _refuse("n_pos and rot must be positive")
    table = _empty((n_pos, rot // 2, 2), torch.float32, torch.device("cuda", dev.ordinal), stream)
    sc = RopeScaling(ROPE_KINDS[kind], factor, context, slow, fast, magnitude)
    _check(lib().bsp_rope_table(dev.handle, n_pos, rot, base, ctypes.byref(sc), _ptr(table), _stream_of(stream, dev)))
    return table


def rope(x, positions, table, layout="half", transpose=False, out=None, dev: Device = None, stream=None):
    """Rotary positions of x [tokens, heads, d] (bf16 or f32): pairs
    (i, i + rot/2) for "half", (2i, 2i + 1) for "interleaved"; the rest of a
    head is copied.  transpose=True gives the gradient of x from that of the
    result.  out may be x."""
    if out is None:
        out = _empty(x.shape, x.dtype, x.device, stream)
    (_calls or _load_calls()).rope(x, positions, table, _rope_layout(layout), bool(transpose), out, dev, stream)
    return out


class KvCache:
    """A paged key/value cache in e4m3: k, v [pages, kv_heads, page, d] (uint8
    or float8_e4m3fn), k_scale, v_scale f32 [pages, kv_heads], powers of two;
    value = code * scale of its (page, head)."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch

        for x, name in ((k, "k"), (v, "v")):
            if not x.is_cuda or x.dim() != 4 or x.dtype not in (torch.uint8, torch.float8_e4m3fn):
                _refuse(f"cache {name} must be a uint8 or float8_e4m3fn cuda tensor [pages, kv_heads, page, d]")
            if x.shape != k.shape or x.stride() != k.stride() or x.stride(3) != 1 or x.stride(2) != x.shape[3]:
                _refuse("cache k and v must have the same shape and strides, the tokens of a page contiguous")
        for x, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if not x.is_cuda or x.dtype is not torch.float32 or x.shape != k.shape[:2] or not x.is_contiguous():
                _refuse(f"cache {name} must be a contiguous f32 cuda tensor [pages, kv_heads]")
        for x, name in ((v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if x.device != k.device:
                _refuse(f"cache {name} is on {x.device}, k on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        n, h, page, d = k.shape
        # strides of single-entry dimensions are never stepped over: give them a valid value
        hs = k.stride(1) if h > 1 else page * d
        ps = k.stride(0) if n > 1 else h * hs
        self.desc = KvCacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), n, ps, hs, h,
                                page, d)
        self.address = ctypes.addressof(self.desc)
        self.kv_heads, self.page, self.d = h, page, d
        self.ordinal = k.device.index

    @staticmethod
    def empty(n_pages, kv_heads, page, d, device_index=None):
        """A cache of n_pages zeroed pages (on the current GPU, or device_index)."""
        import torch

        dv = torch.device("cuda", torch.cuda.current_device() if device_index is None else device_index)
        k, v = (torch.zeros((n_pages, kv_heads, page, d), dtype=torch.uint8, device=dv) for _ in range(2))
        ks, vs = (torch.ones((n_pages, kv_heads), dtype=torch.float32, device=dv) for _ in range(2))
        return KvCache(k, v, ks, vs)


def kv_append(cache: KvCache, k, v, starts, before, pages, table=None, layout="half", q=None, q_out=None, k_out=None,
              dev: Device = None, stream=None):
    """Append the tokens starts[s] .. starts[s + 1] of k and v [tokens,
    kv_heads, d] behind the before[s] tokens that sequence s has in the cache;
    pages[s, i] is the page of its positions i * page ....  With a rotary table
    keys are rotated on the way; q [tokens, heads, d] is rotated to q_out and
    the rotated keys go to k_out where these are given (bsp_kv_append)."""
    (_calls or _load_calls()).kv_append(cache, k, v, starts, before, pages, table, _rope_layout(layout), q, q_out,
                                        k_out, dev, stream)
    return cache


PROMPT_INFO_KEYS = ["units", "ctas", "q_tokens", "kv_tokens", "heads", "kv_heads", "d", "tiles", "plan_bytes",
                    "smem_bytes", "tmem_cols", "packed_heads", "workspace_bytes"]


class PromptPlan:
    """Attention over whole prompts packed one after the other: q_lens[s]
    queries and kv_lens[s] keys of sequence s (host lists; the earlier tokens'
    keys too where a prompt's later part is given, in bf16: no KvCache is read);
    causal: query i sees the keys up to i + (kv_len - q_len).  A plan with a workspace
    (info()["workspace_bytes"]: few rows of many keys are cut along the keys)
    runs on one stream at a time."""

    def __init__(self, dev: Device, q_lens, kv_lens, heads, kv_heads, d, causal=True, opts=None):
        ql = np.ascontiguousarray(q_lens, dtype=np.int32)
        kl = np.ascontiguousarray(kv_lens, dtype=np.int32)
        if ql.ndim != 1 or ql.shape != kl.shape:
            _refuse("q_lens and kv_lens must be lists of one length")
        self.handle = None
        self.dev, self.heads, self.kv_heads, self.d = dev, heads, kv_heads, d
        self.q_tokens, self.kv_tokens = int(ql.sum(dtype=np.int64)), int(kl.sum(dtype=np.int64))
        h = ctypes.c_void_p()
        o = opts if opts is not None else Opts()
        _check(lib().bsp_prompt_plan_create(dev.handle, ql.size, _ptr(ql), _ptr(kl), heads, kv_heads, d,
                                            int(bool(causal)), ctypes.byref(o), ctypes.byref(h)))
        self.handle = h
        self.scale = 1.0 / float(np.sqrt(d))

    def info(self) -> dict:
        arr = (ctypes.c_int64 * 16)()
        _check(lib().bsp_prompt_plan_info(self.handle, arr))
        return {k: int(arr[i]) for i, k in enumerate(PROMPT_INFO_KEYS)}

    def execute(self, q, k, v, o, scale=None, lse=None, stream=None):
        """q, o: bf16 cuda [q_tokens, heads, d]; k, v [kv_tokens, kv_heads, d];
        lse (optional): f32 [q_tokens, heads]."""
        (_calls or _load_calls()).prompt(self, self.dev.ordinal, q, k, v, o, self.scale if scale is None else scale,
                                         lse, stream)

    def close(self):
        if self.handle:
            lib().bsp_prompt_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def inspect_prompt_plan(q_lens, kv_lens, heads, kv_heads, d, causal=True, opts=None, sm_count=148):
    """Run the prompt attention planner on the host only (no GPU)."""
    ql = np.ascontiguousarray(q_lens, dtype=np.int32)
    kl = np.ascontiguousarray(kv_lens, dtype=np.int32)
    if ql.ndim != 1 or ql.shape != kl.shape:
        _refuse("q_lens and kv_lens must be lists of one length")
    info = np.zeros(16, np.int64)
    o = opts if opts is not None else Opts()
    args = (ql.size, _ptr(ql), _ptr(kl), heads, kv_heads, d, int(bool(causal)), ctypes.byref(o), sm_count, _ptr(info))
    _check(lib().bsp_prompt_plan_inspect(*args, None, None))
    units = np.zeros((max(int(info[0]), 1), 12), np.int32)
    cta = np.zeros(int(info[1]) + 1, np.int32)
    _check(lib().bsp_prompt_plan_inspect(*args, _ptr(units), _ptr(cta)))
    dd = {k: int(info[i]) for i, k in enumerate(PROMPT_INFO_KEYS)}
    dd.update(unit_table=units[: int(info[0])], cta_begin=cta)
    return dd


DECODE_INFO_KEYS = ["max_seqs", "ctas", "heads", "kv_heads", "d", "page", "_6", "_7", "workspace_bytes", "smem_bytes"]


class DecodePlan:
    """Attention of one token of each of up to max_seqs sequences over a
    KvCache; the plan is the workspace, lengths are given to execute."""

    def __init__(self, dev: Device, max_seqs, heads, kv_heads, d, page, opts=None):
        self.handle = None
        self.dev, self.max_seqs, self.heads, self.kv_heads, self.d = dev, max_seqs, heads, kv_heads, d
        h = ctypes.c_void_p()
        o = opts if opts is not None else Opts()
        _check(lib().bsp_decode_plan_create(dev.handle, max_seqs, heads, kv_heads, d, page, ctypes.byref(o),
                                            ctypes.byref(h)))
        self.handle = h
        self.scale = 1.0 / float(np.sqrt(d))

    def info(self) -> dict:
        arr = (ctypes.c_int64 * 16)()
        _check(lib().bsp_decode_plan_info(self.handle, arr))
        return {k: int(arr[i]) for i, k in enumerate(DECODE_INFO_KEYS) if not k.startswith("_")}

    def execute(self, cache: KvCache, q, lens, pages, o, scale=None, lse=None, stream=None):
        """q, o: bf16 cuda [sequences, heads, d]; lens: int32 tokens in the
        cache; pages: int32 [sequences, width]; lse (optional): f32
        [sequences, heads]."""
        (_calls or _load_calls()).decode(self, self.dev.ordinal, cache, q, lens, pages, o,
                                         self.scale if scale is None else scale, lse, stream)

    def close(self):
        if self.handle:
            lib().bsp_decode_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ----------------------------------------------------------------- helpers --
def inspect_spmm_plan(M, K, R, C, row_ptr, col_idx, N, strategy=NAIVE, c_type=BF16, opts=None,
                      sm_count=148, max_smem=232448):
    """Run the SpMM planner on the host only (no GPU) and return its schedule."""
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    ci = np.ascontiguousarray(col_idx, dtype=np.int32)
    if ci.size == 0:
        ci = np.zeros(1, np.int32)
    info = np.zeros(16, np.int64)
    o = opts if opts is not None else Opts()
    args = (M, K, R, C, int(rp[-1]), _ptr(rp), _ptr(ci), N, c_type, strategy, ctypes.byref(o),
            sm_count, max_smem, _ptr(info))
    _check(lib().bsp_spmm_plan_inspect(*args, None, None, None, None, None))
    units = np.zeros((int(info[0]), 8), np.int32)
    cta = np.zeros(int(info[1]) + 1, np.int32)
    steps = np.zeros((max(int(info[7]), 1), int(info[15])), np.int32)
    stages = np.zeros((max(int(info[13]), 1), 16), np.int32)
    cta_st = np.zeros(int(info[1]) + 1, np.int32)
    _check(lib().bsp_spmm_plan_inspect(*args, _ptr(units), _ptr(cta), _ptr(steps), _ptr(stages),
                                       _ptr(cta_st)))
    keys = ["units", "ctas", "group_rows", "n_tiles", "slab", "kc", "stages", "steps",
            "plan_bytes", "smem_bytes", "tmem_cols", "variant", "producers", "stage_list", "nsub",
            "step_stride"]
    d = {k: int(info[i]) for i, k in enumerate(keys)}
    d.update(unit_table=units, cta_begin=cta, step_table=steps[: int(info[7])],
             stage_table=stages[: int(info[13])], cta_stage_begin=cta_st)
    # row-stacked plans: stacking order of the block-rows (None = consecutive)
    d["entry_rows"] = None
    if d["variant"] == 1:
        n = ctypes.c_int64(0)
        eargs = (M, K, R, C, int(rp[-1]), _ptr(rp), _ptr(ci), N, strategy, ctypes.byref(o), sm_count, max_smem)
        _check(lib().bsp_spmm_plan_entry_rows(*eargs, None, ctypes.byref(n)))
        if n.value > 0:
            rows = np.zeros(n.value, np.int32)
            _check(lib().bsp_spmm_plan_entry_rows(*eargs, _ptr(rows), ctypes.byref(n)))
            d["entry_rows"] = rows
    return d


def spmm_plan_traffic(M, K, R, C, row_ptr, col_idx, N, strategy=NAIVE, opts=None, sm_count=148,
                      max_smem=232448):
    """Operand bytes / boxes the SpMM plan moves into shared memory (host only):
    dict(a_bytes, b_bytes, a_boxes, b_boxes, variant)."""
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    ci = np.ascontiguousarray(col_idx, dtype=np.int32)
    ci = ci if ci.size else np.zeros(1, np.int32)
    info = np.zeros(16, np.int64)
    tr = np.zeros(4, np.int64)
    o = opts if opts is not None else Opts()
    _check(lib().bsp_spmm_plan_traffic(M, K, R, C, int(rp[-1]), _ptr(rp), _ptr(ci), N, strategy,
                                       ctypes.byref(o), sm_count, max_smem, _ptr(info), _ptr(tr)))
    return dict(a_bytes=int(tr[0]), b_bytes=int(tr[1]), a_boxes=int(tr[2]), b_boxes=int(tr[3]),
                variant=int(info[11]), units=int(info[0]))


def inspect_sddmm_plan(M, N, R, C, row_ptr, col_idx, K, strategy=NAIVE, opts=None, sm_count=148,
                       max_smem=232448):
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    ci = np.ascontiguousarray(col_idx, dtype=np.int32)
    if ci.size == 0:
        ci = np.zeros(1, np.int32)
    info = np.zeros(16, np.int64)
    o = opts if opts is not None else Opts()
    args = (M, N, R, C, int(rp[-1]), _ptr(rp), _ptr(ci), K, strategy, ctypes.byref(o), sm_count,
            max_smem, _ptr(info))
    _check(lib().bsp_sddmm_plan_inspect(*args, None, None))
    units = np.zeros((max(int(info[0]), 1), int(info[12])), np.int32)
    cta = np.zeros(int(info[1]) + 1, np.int32)
    _check(lib().bsp_sddmm_plan_inspect(*args, _ptr(units), _ptr(cta)))
    return dict(units=int(info[0]), ctas=int(info[1]), slab=int(info[4]), kc=int(info[5]),
                stages=int(info[6]), keep_a=int(info[7]), variant=int(info[11]), nseg_max=int(info[13]),
                producers=int(info[14]), unit_table=units[: int(info[0])], cta_begin=cta)


def ipc_export(dev: Device, tensor):
    """(64-byte handle, byte offset) that lets another process on this node map
    the device allocation holding `tensor`."""
    h = ctypes.create_string_buffer(IPC_HANDLE_BYTES)
    off = ctypes.c_int64()
    _check(lib().bsp_ipc_export(dev.handle, _ptr(tensor), h, ctypes.byref(off)))
    return h.raw, int(off.value)


def ipc_import(dev: Device, handle: bytes) -> int:
    """Map a peer process's allocation into this one; returns its base address."""
    base = ctypes.c_void_p()
    buf = ctypes.create_string_buffer(bytes(handle), IPC_HANDLE_BYTES)
    _check(lib().bsp_ipc_import(dev.handle, buf, ctypes.byref(base)))
    return int(base.value)


def ipc_close(dev: Device, base: int) -> None:
    _check(lib().bsp_ipc_close(dev.handle, ctypes.c_void_p(base)))


def partition_rows(row_ptr: np.ndarray, parts: int) -> np.ndarray:
    rp = np.ascontiguousarray(row_ptr, dtype=np.int32)
    bounds = np.zeros(parts + 1, dtype=np.int64)
    _check(lib().bsp_partition_rows(_ptr(rp), rp.size - 1, parts, _ptr(bounds)))
    return bounds


def serpentine_assign(n: int, parts: int):
    owner = np.zeros(max(n, 1), dtype=np.int32)
    slot = np.zeros(max(n, 1), dtype=np.int32)
    _check(lib().bsp_serpentine_assign(n, parts, _ptr(owner), _ptr(slot)))
    return owner[:n], slot[:n]
