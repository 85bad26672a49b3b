"""cllm_inference_amd -- the quantized linear-layer path of cllm_inference on MI355X (gfx950).

Python mirror of the reference's Quant API (include/cllm/core/quant.hpp:90-151 in the
reference) over the C ABI of libcllm_hip.so (include/cllm_hip.h). Same names, argument
meaning and error behaviour: failures raise RuntimeError with the reference's messages.

Host-array functions take and return numpy arrays and are synchronous, like the reference.
The *_dev functions take torch tensors already on the GPU and enqueue on torch's current
stream. There is no CPU fallback: if the HIP library is not built, importing the functions
works but every call raises.
"""
from __future__ import annotations

import ctypes
import enum
import os
from dataclasses import dataclass

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libcllm_hip.so")
QUANT_LIB_PATH = os.path.join(_HERE, "libcllm_quant.so")


class GgmlType(enum.IntEnum):
    """GGUF tensor type ids (reference include/cllm/core/quant.hpp:13-27)."""
    F32 = 0
    F16 = 1
    Q4_0 = 2
    Q4_1 = 3
    Q5_0 = 6
    Q5_1 = 7
    Q8_0 = 8
    Q8_1 = 9
    Q2_K = 10
    Q3_K = 11
    Q4_K = 12
    Q5_K = 13
    Q6_K = 14


# Every symbol include/cllm_hip.h declares: (name, restype, argtypes).
_P = ctypes.c_void_p
_I = ctypes.c_int
_U = ctypes.c_uint32
_I64 = ctypes.c_int64
_SZ = ctypes.c_size_t
SIGNATURES = {
    "cllm_hip_init": (_I, [_I]),
    "cllm_hip_last_error": (ctypes.c_char_p, []),
    "cllm_hip_block_size": (_I, [_U]),
    "cllm_hip_type_size": (_SZ, [_U]),
    "cllm_hip_has_vec_dot": (_I, [_U]),
    "cllm_hip_quantize_row_q8_0": (_I, [_P, _I64, _I, _P, _P, _P]),
    "cllm_hip_vec_dot_rows": (_I, [_P, _U, _I64, _I, _P, _P, _P, _P]),
    "cllm_hip_matmul_quant": (_I, [_P, _P, _U, _P, _I, _I, _P]),
    "cllm_hip_matmul_quant_batch": (_I, [_P, _P, _U, _P, _I, _I, _I, _P]),
    "cllm_hip_dequantize_block": (_I, [_P, _P, _U, _I64]),
    "cllm_hip_dequantize_block_f16": (_I, [_P, _P, _U, _I64]),
    "cllm_hip_register_weights": (_I, [_P, _SZ]),
    "cllm_hip_unregister_weights": (_I, [_P]),
    "cllm_hip_file_mapping_identity": (_I, [_P, _P]),
    "cllm_hip_allocation_count": (ctypes.c_uint64, []),
    "cllm_hip_quantize_q8_0_dev": (_I, [_P, _I64, _I, _P, _P, _P, _P]),
    "cllm_hip_gemv_q8_dev": (_I, [_P, _U, _I, _I, _I, _P, _P, _P, _P, _P, _P]),
    "cllm_hip_matmul_quant_dev": (_I, [_P, _P, _U, _P, _I, _I, _I, _P, _P]),
    "cllm_hip_matmul_quant_static_dev": (_I, [_P, _P, _U, _P, _I, _I, _I, _P, _P]),
    "cllm_hip_static_scratch_bytes": (_SZ, []),
    "cllm_hip_read_stream_dev": (_I, [_P, ctypes.c_uint64, _P]),
    "cllm_hip_matmul_route": (ctypes.c_char_p, [_U, _I, _I, _I]),
    "cllm_hip_matmul_plan": (ctypes.c_char_p, [_U, _I, _I, _I]),
    "cllm_hip_tune": (_I, [ctypes.c_char_p, _P, _I]),
    "cllm_hip_rmsnorm_q8_0_dev": (_I, [_P, _P, ctypes.c_float, _I, _I, _P, _P, _P, _P, _P]),
    "cllm_hip_swiglu_q8_0_dev": (_I, [_P, _P, _I, _I, _P, _P, _P, _P, _P]),
    "cllm_hip_add_dev": (_I, [_P, _P, _I64, _P]),
    "cllm_hip_mfma_act_bytes": (_SZ, [_I, _I]),
    "cllm_hip_quantize_mfma_dev": (_I, [_P, _I, _I, _P, _P]),
    "cllm_hip_rmsnorm_mfma_dev": (_I, [_P, _P, ctypes.c_float, _I, _I, _P, _P, _P]),
    "cllm_hip_swiglu_mfma_dev": (_I, [_P, _P, _I, _I, _P, _P, _P]),
    "cllm_hip_matmul_mfma_dev": (_I, [_U, _I, _I, _P, _P, _P, _P, _I, _P, _P]),
    "cllm_hip_matmul_mfma_plan": (ctypes.c_char_p, [_U, _I, _I, _P, _I]),
    "cllm_hip_gemv_q8_residual_dev": (_I, [_P, _U, _I, _I, _I, _P, _P, _P, _P, _P, _P]),
    "cllm_hip_gemv_q8_multi_dev": (_I, [_U, _I, _I, _P, _P, _P, _P, _I, _P, _P, _P, _P]),
    "cllm_hip_gemv_q8_swiglu_dev": (_I, [_U, _I, _I, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P]),
    "cllm_hip_rmsnorm_gemv_multi_dev": (_I, [_U, _I, _I, _P, _P, _P, _P, _P, _P, ctypes.c_float,
                                             _P]),
    "cllm_hip_rmsnorm_gemv_swiglu_dev": (_I, [_U, _I, _I, _P, _P, _P, _P, _P, _P, ctypes.c_float,
                                              _P, _P]),
    "cllm_hip_group_rows_dev": (_I, [_P, _I, _I, _P, _P, _P]),
    "cllm_hip_moe_route_dev": (_I, [_P, _I64, _P, _I, _I, _I, _I, _I,
                                    ctypes.c_float, _I, _I, _P, _P, _P, _P, _P]),
    "cllm_hip_moe_matmul_ws_bytes": (_SZ, [_U, _I, _I]),
    "cllm_hip_moe_matmul_dev": (_I, [_U, _I, _I, _I, _P, _P, _P, _I, _I, _P, _P, _P, _P, _SZ, _P]),
    "cllm_hip_moe_swiglu_dev": (_I, [_U, _I, _I, _I, _P, _P, _P, _P, _P, _I, _I, _P, _P, _P, _P, _SZ, _P]),
    "cllm_hip_moe_down_ws_bytes": (_SZ, [_U, _I, _I, _I, _I]),
    "cllm_hip_moe_down_dev": (_I, [_U, _I, _I, _I, _P, _P, _P, _I, _I, _P, _P, _P, _P, _P, _P, _P, _SZ, _P]),
    "cllm_hip_moe_plan": (ctypes.c_char_p, [_U, _I, _I, _I, _I, _I]),
    "cllm_hip_lora_ws_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "cllm_hip_lora_dev": (_I, [_U, _I, _I, _P, _P, _P, _I, _I, _P, _P, _P, _I, _P, _P, _P, _P, _P, _SZ, _P]),
    "cllm_hip_gguf_open": (_I, [ctypes.c_char_p, _I, ctypes.POINTER(_P)]),
    "cllm_hip_gguf_close": (_I, [_P]),
    "cllm_hip_gguf_tensor_count": (_I, [_P]),
    "cllm_hip_gguf_find": (_I, [_P, ctypes.c_char_p]),
    "cllm_hip_gguf_tensor": (_I, [_P, _I, ctypes.POINTER(ctypes.c_char_p), ctypes.POINTER(_U),
                                  ctypes.POINTER(_I), ctypes.POINTER(ctypes.c_uint64),
                                  ctypes.POINTER(ctypes.c_uint64), ctypes.POINTER(_P),
                                  ctypes.POINTER(_P)]),
    "cllm_hip_gguf_config": (_I, [_P, _P]),
    "cllm_hip_rope_neox_dev": (_I, [_P, _I, _I, _I, _I, ctypes.c_float, _P]),
    "cllm_hip_rope_neox2_dev": (_I, [_P, _I, _P, _I, _I, _I, _I, ctypes.c_float, _P]),
    "cllm_hip_matmul_quant_residual_dev": (_I, [_P, _P, _U, _P, _I, _I, _I, _P, _P]),
    "cllm_hip_dequantize_rows_dev": (_I, [_P, _U, _I, _P, _I, _P, _P]),
    "cllm_hip_attention_dev": (_I, [_P, _P, _P, _I, _I, _I, _I, _I, _P, _P]),
    "cllm_hip_attention_rope_dev": (_I, [_P, _P, _P, _I, _I, _I, _I, ctypes.c_float, _P, _P]),
    "cllm_hip_attention_plan": (ctypes.c_char_p, [_I, _I, _I, _I, _I]),
    "cllm_hip_kv4_page_bytes": (_SZ, [_I, _I, _I]),
    "cllm_hip_kv4_work_ints": (_SZ, [_I, _I, _I]),
    "cllm_hip_kv4_extend_dev": (_I, [_P, _P, _P, _I, _P, _P]),
    "cllm_hip_kv4_fork_dev": (_I, [_P, _P, _P, _I, _P]),
    "cllm_hip_kv4_truncate_dev": (_I, [_P, _P, _P, _I, _P]),
    "cllm_hip_kv4_compact_dev": (_I, [_P, _P, _P]),
    "cllm_hip_kv4_copy_pages_dev": (_I, [_P, _P, _P, _I, _P]),
    "cllm_hip_kv4_store_dev": (_I, [_P, _I, _P, _P, _P, _I, ctypes.c_float, _P, _P, _I, _I, _P]),
    "cllm_hip_kv4_load_dev": (_I, [_P, _I, _P, _P, _I, _I, _P, _P, _P]),
    "cllm_hip_kv4_attention_ws_bytes": (_SZ, [_P, _I, _I, _I, _I, _I]),
    "cllm_hip_kv4_attention_dev": (_I, [_P, _I, _P, _P, _P, _I, _I, _I, _I, _I, _P, _P, _SZ, _P]),
    "cllm_hip_kv4_attention_plan": (ctypes.c_char_p, [_P, _I, _I, _I, _I, _I]),
    "cllm_hip_logprobs_ws_bytes": (_SZ, [_I, _I, _I]),
    "cllm_hip_logprobs_dev": (_I, [_P, _I64, _I, _I, _P, _I, _P, _P, _P, _P, _P, _P, _P, _SZ, _P]),
}


class ModelConfig(ctypes.Structure):
    """cllm_hip_model_config: ModelConfig (reference gguf.hpp:13-34) plus the file layout."""
    _fields_ = [("arch", ctypes.c_char * 64)] + [
        (n, ctypes.c_uint32) for n in ("n_layers", "n_embd", "n_head", "n_head_kv", "n_ctx",
                                        "n_ff", "vocab_size", "head_dim")] + [
        ("rope_theta", ctypes.c_float), ("norm_eps", ctypes.c_float),
        ("version", ctypes.c_uint32), ("data_offset", ctypes.c_uint64),
        ("data_bytes", ctypes.c_uint64)]

_lib_handle = None


def load_library(path: str = LIB_PATH) -> ctypes.CDLL:
    """Loads libcllm_hip.so (once) and declares every C-ABI signature."""
    global _lib_handle
    if _lib_handle is None:
        if not os.path.exists(path):
            raise RuntimeError(
                f"{path} is missing: build it with `python -m cllm_inference_amd.build`")
        lib = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib_handle = lib
    return _lib_handle


def _check(rc: int) -> None:
    if rc != 0:
        msg = load_library().cllm_hip_last_error().decode()
        raise RuntimeError(msg)


def _ptr(a: np.ndarray | None):
    return None if a is None else a.ctypes.data_as(ctypes.c_void_p)


def file_mapping_identity(addr: int) -> tuple:
    """What the library compares before reusing the device copy of the read-only private file
    mapping that holds host address addr (cllm_hip_file_mapping_identity): (start, end, file
    offset, inode, device, file size, mtime ns, ctime ns, file reachable by its path)."""
    info = (ctypes.c_uint64 * 9)()
    _check(load_library().cllm_hip_file_mapping_identity(ctypes.c_void_p(addr), info))
    return tuple(int(v) for v in info)


def block_size(t: int) -> int:
    return load_library().cllm_hip_block_size(int(t))


def type_size(t: int) -> int:
    return load_library().cllm_hip_type_size(int(t))


def has_vec_dot(t: int) -> bool:
    return bool(load_library().cllm_hip_has_vec_dot(int(t)))


@dataclass
class QuantizedQ8_0:
    """Q8_0 activation rows (reference quant.hpp:118-124): fp32 scales, int8 qs, int32
    per-block sums of qs."""
    scales: np.ndarray
    qs: np.ndarray
    bsums: np.ndarray
    n: int


def quantize_row_q8_0(x: np.ndarray, n: int | None = None) -> QuantizedQ8_0:
    """fp32 -> Q8_0. x is one row of n floats, or an (m, n) array quantized row by row."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    rows = x.reshape(-1, x.shape[-1]) if x.ndim > 1 else x.reshape(1, -1)
    n = rows.shape[1] if n is None else int(n)
    m = rows.shape[0] if x.ndim > 1 else 1
    qs = np.empty((m, n), dtype=np.int8)
    sc = np.empty((m, max(n // 32, 0)), dtype=np.float32)
    bs = np.empty((m, max(n // 32, 0)), dtype=np.int32)
    _check(load_library().cllm_hip_quantize_row_q8_0(_ptr(rows), n, m, _ptr(qs), _ptr(sc),
                                                     _ptr(bs)))
    if x.ndim == 1:
        qs, sc, bs = qs[0], sc[0], bs[0]
    return QuantizedQ8_0(scales=sc, qs=qs, bsums=bs, n=n)


def vec_dot_rows(w: np.ndarray, t: int, qx: QuantizedQ8_0, n: int, n_w_rows: int = 1) -> np.ndarray:
    """vec_dot_row over n_w_rows consecutive weight rows starting at w."""
    w = np.ascontiguousarray(w, dtype=np.uint8)
    out = np.empty(n_w_rows, dtype=np.float32)
    _check(load_library().cllm_hip_vec_dot_rows(
        _ptr(w), int(t), int(n), int(n_w_rows), _ptr(np.ascontiguousarray(qx.qs)),
        _ptr(np.ascontiguousarray(qx.scales)), _ptr(np.ascontiguousarray(qx.bsums)), _ptr(out)))
    return out


def vec_dot_row(w_row: np.ndarray, t: int, qx: QuantizedQ8_0, n: int) -> float:
    """Reference quant.hpp:135-136."""
    return float(vec_dot_rows(w_row, t, qx, n, 1)[0])


def matmul_quant(x: np.ndarray, w: np.ndarray, t: int, bias: np.ndarray | None, in_dim: int,
                 out_dim: int) -> np.ndarray:
    """y[out_dim] = x . W^T (+ bias) -- reference quant.hpp:143-145."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    w = np.ascontiguousarray(w, dtype=np.uint8)
    b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
    y = np.empty(out_dim, dtype=np.float32)
    _check(load_library().cllm_hip_matmul_quant(_ptr(x), _ptr(w), int(t), _ptr(b), int(in_dim),
                                                int(out_dim), _ptr(y)))
    return y


def matmul_quant_batch(x: np.ndarray, w: np.ndarray, t: int, bias: np.ndarray | None,
                       in_dim: int, out_dim: int, n_rows: int) -> np.ndarray:
    """y[n_rows, out_dim] = X . W^T (+ bias) -- reference quant.hpp:149-151."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    w = np.ascontiguousarray(w, dtype=np.uint8)
    b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
    y = np.zeros((max(n_rows, 0), out_dim), dtype=np.float32)
    _check(load_library().cllm_hip_matmul_quant_batch(_ptr(x), _ptr(w), int(t), _ptr(b),
                                                      int(in_dim), int(out_dim), int(n_rows),
                                                      _ptr(y)))
    return y


def _src_ptr(src):
    """A host array's address, a torch tensor's device address, or an int address as it is."""
    if isinstance(src, np.ndarray):
        return _ptr(src)
    if hasattr(src, "data_ptr"):
        return ctypes.c_void_p(src.data_ptr())
    return ctypes.c_void_p(int(src))


def dequantize_block(src, t: int, n: int) -> np.ndarray:
    """The first n elements of the blocks at src as float32 -- reference quant.hpp:99. src is a
    uint8 host array, a device tensor, or a raw address (host or device)."""
    out = np.empty(max(int(n), 0), np.float32)
    _check(load_library().cllm_hip_dequantize_block(_src_ptr(src), _ptr(out), int(t), int(n)))
    return out


def dequantize_block_f16(src, t: int, n: int) -> np.ndarray:
    """The same values as binary16 bits (uint16) -- reference quant.hpp:105."""
    out = np.empty(max(int(n), 0), np.uint16)
    _check(load_library().cllm_hip_dequantize_block_f16(_src_ptr(src), _ptr(out), int(t), int(n)))
    return out


# ---- device (torch) entry points --------------------------------------------------------

def _tp(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    import torch
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def quantize_q8_0_dev(x, qs=None, scales=None, bsums=None):
    """x: float32 (m, k) CUDA tensor -> (qs int8 (m, k), scales f32 (m, k/32), bsums i32)."""
    import torch
    m, k = x.shape
    if qs is None:
        qs = torch.empty((m, k), dtype=torch.int8, device=x.device)
        scales = torch.empty((m, k // 32), dtype=torch.float32, device=x.device)
        bsums = torch.empty((m, k // 32), dtype=torch.int32, device=x.device)
    _check(load_library().cllm_hip_quantize_q8_0_dev(_tp(x), k, m, _tp(qs), _tp(scales),
                                                     _tp(bsums), _stream()))
    return qs, scales, bsums


def gemv_q8_dev(w, t: int, in_dim: int, out_dim: int, qs, scales, bsums, bias=None, y=None):
    """vec_dot of every weight row against already-quantized activation rows (device)."""
    import torch
    m = qs.shape[0]
    if y is None:
        y = torch.empty((m, out_dim), dtype=torch.float32, device=qs.device)
    _check(load_library().cllm_hip_gemv_q8_dev(_tp(w), int(t), int(in_dim), int(out_dim), int(m),
                                               _tp(qs), _tp(scales), _tp(bsums), _tp(bias),
                                               _tp(y), _stream()))
    return y


def gemv_q8_multi_dev(ws, t: int, in_dim: int, out_dims, qs, scales, bsums, ys=None,
                      biases=None):
    """One launch over up to three matrices sharing the quantized activation rows (q/k/v,
    gate/up). Returns the list of outputs [n_rows, out_dims[i]]."""
    import torch
    m = qs.shape[0]
    n_mats = len(ws)
    if ys is None:
        ys = [torch.empty((m, int(n)), dtype=torch.float32, device=qs.device) for n in out_dims]
    wa = (ctypes.c_void_p * n_mats)(*[w.data_ptr() for w in ws])
    ya = (ctypes.c_void_p * n_mats)(*[y.data_ptr() for y in ys])
    na = (ctypes.c_int * n_mats)(*[int(n) for n in out_dims])
    ba = None
    if biases is not None:
        ba = (ctypes.c_void_p * n_mats)(*[0 if b is None else b.data_ptr() for b in biases])
    _check(load_library().cllm_hip_gemv_q8_multi_dev(
        int(t), int(in_dim), n_mats, wa, na, ba, ya, int(m), _tp(qs), _tp(scales), _tp(bsums),
        _stream()))
    return ys


def gemv_q8_swiglu_dev(w_gate, w_up, t: int, in_dim: int, n_ff: int, qs, scales, bsums,
                       h=None, bias_gate=None, bias_up=None):
    """h = silu(gate . a) * (up . a) for the n_ff rows of the gate and up matrices against the
    quantized rows, in one launch (engine.cpp:509-512). Returns h [n_rows, n_ff]."""
    import torch
    m = qs.shape[0]
    if h is None:
        h = torch.empty((m, int(n_ff)), dtype=torch.float32, device=qs.device)
    _check(load_library().cllm_hip_gemv_q8_swiglu_dev(
        int(t), int(in_dim), int(n_ff), _tp(w_gate), _tp(w_up), _tp(bias_gate), _tp(bias_up),
        int(m), _tp(qs), _tp(scales), _tp(bsums), _tp(h), _stream()))
    return h


def rmsnorm_gemv_multi_dev(x, norm_w, eps: float, ws, t: int, in_dim: int, out_dims, ys=None,
                           biases=None):
    """RMSNorm of the one row x (float32 (1, in_dim), in_dim <= 4096) with weight norm_w, then
    gemv_q8_multi_dev on it, in one launch (engine.cpp:475-478); the bits of rmsnorm_q8_0_dev
    followed by gemv_q8_multi_dev. Returns the list of outputs [1, out_dims[i]]."""
    import torch
    n_mats = len(ws)
    if ys is None:
        ys = [torch.empty((1, int(n)), dtype=torch.float32, device=x.device) for n in out_dims]
    wa = (ctypes.c_void_p * n_mats)(*[w.data_ptr() for w in ws])
    ya = (ctypes.c_void_p * n_mats)(*[y.data_ptr() for y in ys])
    na = (ctypes.c_int * n_mats)(*[int(n) for n in out_dims])
    ba = None
    if biases is not None:
        ba = (ctypes.c_void_p * n_mats)(*[0 if b is None else b.data_ptr() for b in biases])
    _check(load_library().cllm_hip_rmsnorm_gemv_multi_dev(
        int(t), int(in_dim), n_mats, wa, na, ba, ya, _tp(x), _tp(norm_w), float(eps), _stream()))
    return ys


def rmsnorm_gemv_swiglu_dev(x, norm_w, eps: float, w_gate, w_up, t: int, in_dim: int, n_ff: int,
                            h=None, bias_gate=None, bias_up=None):
    """RMSNorm of the one row x, then gemv_q8_swiglu_dev on it, in one launch
    (engine.cpp:508-512); the bits of rmsnorm_q8_0_dev followed by gemv_q8_swiglu_dev.
    Returns h [1, n_ff]."""
    import torch
    if h is None:
        h = torch.empty((1, int(n_ff)), dtype=torch.float32, device=x.device)
    _check(load_library().cllm_hip_rmsnorm_gemv_swiglu_dev(
        int(t), int(in_dim), int(n_ff), _tp(w_gate), _tp(w_up), _tp(bias_gate), _tp(bias_up),
        _tp(x), _tp(norm_w), float(eps), _tp(h), _stream()))
    return h


def gemv_q8_residual_dev(w, t: int, in_dim: int, out_dim: int, qs, scales, bsums, y, bias=None):
    """y += vec_dot of every weight row against the quantized rows (device): a matmul and
    the residual add after it (engine.cpp:505-506, 512-513) in one launch."""
    m = qs.shape[0]
    _check(load_library().cllm_hip_gemv_q8_residual_dev(
        _tp(w), int(t), int(in_dim), int(out_dim), int(m), _tp(qs), _tp(scales), _tp(bsums),
        _tp(bias), _tp(y), _stream()))
    return y


def matmul_quant_dev(x, w, t: int, bias, in_dim: int, out_dim: int, y=None):
    """matmul_quant_batch on device tensors: x float32 (m, in_dim), w uint8 GGUF blocks."""
    import torch
    m = x.shape[0]
    if y is None:
        y = torch.empty((m, out_dim), dtype=torch.float32, device=x.device)
    _check(load_library().cllm_hip_matmul_quant_dev(_tp(x), _tp(w), int(t), _tp(bias),
                                                    int(in_dim), int(out_dim), int(m), _tp(y),
                                                    _stream()))
    return y


def matmul_quant_residual_dev(x, w, t: int, bias, in_dim: int, out_dim: int, y):
    """y += matmul_quant_batch(x, w) (+ bias) on device tensors: a matmul and the residual
    add after it (engine.cpp:505-506, 512-513)."""
    m = x.shape[0]
    _check(load_library().cllm_hip_matmul_quant_residual_dev(_tp(x), _tp(w), int(t), _tp(bias),
                                                             int(in_dim), int(out_dim), int(m),
                                                             _tp(y), _stream()))
    return y


def matmul_route(t: int, in_dim: int, out_dim: int, n_rows: int) -> str:
    return load_library().cllm_hip_matmul_route(int(t), int(in_dim), int(out_dim),
                                                int(n_rows)).decode()


def read_stream_dev(t) -> None:
    """Reads the CUDA tensor t's bytes once and computes nothing (cllm_hip_read_stream_dev): the
    one-launch HBM read ceiling a GEMV over the same bytes is measured against."""
    _check(load_library().cllm_hip_read_stream_dev(_tp(t), t.numel() * t.element_size(),
                                                   _stream()))


def matmul_plan(t: int, in_dim: int, out_dim: int, n_rows: int) -> str:
    """The kernel instantiation and split count the batch would run (or the route name)."""
    return load_library().cllm_hip_matmul_plan(int(t), int(in_dim), int(out_dim),
                                               int(n_rows)).decode()


def attention_plan(n_rows: int, pos0: int, n_head: int, n_head_kv: int, head_dim: int) -> str:
    """The attention kernel attention_dev would run for this shape, with its workgroups or
    sequence splits ("none" for an unsupported shape)."""
    return load_library().cllm_hip_attention_plan(int(n_rows), int(pos0), int(n_head),
                                                  int(n_head_kv), int(head_dim)).decode()


def tune(knob: str, *values: int) -> None:
    """Sets a process-wide kernel-choice override (cllm_hip_tune); no values resets it."""
    arr = (ctypes.c_int * max(len(values), 1))(*[int(v) for v in values])
    _check(load_library().cllm_hip_tune(knob.encode(), ctypes.cast(arr, ctypes.c_void_p),
                                        len(values)))


# ---- producers of a device-resident layer ------------------------------------------------

def _q8_buffers(m, n, device, want):
    import torch
    if not want:
        return None, None, None
    return (torch.empty((m, n), dtype=torch.int8, device=device),
            torch.empty((m, n // 32), dtype=torch.float32, device=device),
            torch.empty((m, n // 32), dtype=torch.int32, device=device))


def rmsnorm_q8_0_dev(x, w, eps: float, h=True, quantize=True):
    """RMSNorm of each row of x (float32 (m, n) CUDA tensor) with weight w (n,), fused with
    Q8_0 quantization -- engine.cpp:23-28 then quant.cpp:420-452. Returns (h, qs, scales,
    bsums); h is None when h=False, the Q8_0 triple None when quantize=False."""
    import torch
    m, n = x.shape
    hb = torch.empty_like(x) if h else None
    qs, sc, bs = _q8_buffers(m, n, x.device, quantize)
    _check(load_library().cllm_hip_rmsnorm_q8_0_dev(_tp(x), _tp(w), float(eps), int(n), int(m),
                                                    _tp(hb), _tp(qs), _tp(sc), _tp(bs),
                                                    _stream()))
    return hb, qs, sc, bs


def swiglu_q8_0_dev(gate, up, h=True, quantize=True):
    """silu(gate) * up (engine.cpp:38, 511, 596) fused with Q8_0 quantization; gate and up
    are float32 (m, n) CUDA tensors. Returns (h, qs, scales, bsums) like rmsnorm_q8_0_dev."""
    import torch
    m, n = gate.shape
    hb = torch.empty_like(gate) if h else None
    qs, sc, bs = _q8_buffers(m, n, gate.device, quantize)
    _check(load_library().cllm_hip_swiglu_q8_0_dev(_tp(gate), _tp(up), int(n), int(m), _tp(hb),
                                                   _tp(qs), _tp(sc), _tp(bs), _stream()))
    return hb, qs, sc, bs


def add_dev(x, d):
    """x += d in place (the residual adds, engine.cpp:506, 513)."""
    _check(load_library().cllm_hip_add_dev(_tp(x), _tp(d), int(x.numel()), _stream()))
    return x


# ---- prefill linear layer on the weight-row format ----------------------------------------

def mfma_act_new(in_dim: int, n_rows: int, device="cuda"):
    """A device buffer for n_rows rows of the weight-row kernels' activation format."""
    import torch
    nbytes = load_library().cllm_hip_mfma_act_bytes(int(in_dim), int(n_rows))
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def quantize_mfma_dev(x, act=None):
    """Q8_0 of the rows of x [n_rows, in_dim] into the weight-row format (a new buffer if act
    is None); returns act."""
    m, k = x.shape
    if act is None:
        act = mfma_act_new(k, m, x.device)
    _check(load_library().cllm_hip_quantize_mfma_dev(_tp(x), int(k), int(m), _tp(act), _stream()))
    return act


def rmsnorm_mfma_dev(x, norm_w, eps: float, h=None, act=None):
    """RMSNorm of the rows of x into h (fp32, when given) and the weight-row format; returns
    act."""
    m, k = x.shape
    if act is None:
        act = mfma_act_new(k, m, x.device)
    _check(load_library().cllm_hip_rmsnorm_mfma_dev(_tp(x), _tp(norm_w), float(eps), int(k),
                                                    int(m), _tp(h), _tp(act), _stream()))
    return act


def swiglu_mfma_dev(gate, up, h=None, act=None):
    """silu(gate) * up into h (fp32, when given) and the weight-row format; returns act."""
    m, n = gate.shape
    if act is None:
        act = mfma_act_new(n, m, gate.device)
    _check(load_library().cllm_hip_swiglu_mfma_dev(_tp(gate), _tp(up), int(n), int(m), _tp(h),
                                                   _tp(act), _stream()))
    return act


def matmul_mfma_dev(ws, t: int, in_dim: int, out_dims, act, n_rows: int, ys=None, biases=None):
    """matmul_quant_batch of the matrices ws (device weights, one type and in_dim) over the
    activation rows in act; returns the outputs [n_rows, out_dims[i]]."""
    import torch
    n_mats = len(ws)
    if ys is None:
        ys = [torch.empty((n_rows, int(n)), dtype=torch.float32, device=act.device)
              for n in out_dims]
    wa = (ctypes.c_void_p * n_mats)(*[w.data_ptr() for w in ws])
    ya = (ctypes.c_void_p * n_mats)(*[y.data_ptr() for y in ys])
    na = (ctypes.c_int * n_mats)(*[int(n) for n in out_dims])
    ba = None
    if biases is not None:
        ba = (ctypes.c_void_p * n_mats)(*[0 if b is None else b.data_ptr() for b in biases])
    _check(load_library().cllm_hip_matmul_mfma_dev(int(t), int(in_dim), n_mats, wa, na, ba, ya,
                                                   int(n_rows), _tp(act), _stream()))
    return ys


def matmul_mfma_plan(t: int, in_dim: int, out_dims, n_rows: int) -> str:
    na = (ctypes.c_int * len(out_dims))(*[int(n) for n in out_dims])
    return load_library().cllm_hip_matmul_mfma_plan(int(t), int(in_dim), len(out_dims), na,
                                                    int(n_rows)).decode()


# ---- GGUF files ---------------------------------------------------------------------------

@dataclass
class GgufTensorInfo:
    name: str
    type: int
    shape: tuple          # rows first
    offset: int           # in the data section
    host: int             # address in the mapping
    dev: int              # device address (0 without upload)


class GgufFile:
    """A GGUF file parsed by the library (reference GgufLoader::load, gguf.cpp:122-275);
    with upload=True its data section lives on the device and host tensor pointers into the
    mapping resolve to it in every matmul call."""

    def __init__(self, path: str, upload: bool = False):
        lib = load_library()
        h = ctypes.c_void_p()
        _check(lib.cllm_hip_gguf_open(str(path).encode(), 1 if upload else 0, ctypes.byref(h)))
        self._h = h

    def close(self):
        if self._h:
            _check(load_library().cllm_hip_gguf_close(self._h))
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __len__(self):
        return load_library().cllm_hip_gguf_tensor_count(self._h)

    def tensor(self, i: int) -> GgufTensorInfo:
        name = ctypes.c_char_p()
        t = ctypes.c_uint32()
        nd = ctypes.c_int()
        dims = (ctypes.c_uint64 * 4)()
        off = ctypes.c_uint64()
        host = ctypes.c_void_p()
        dev = ctypes.c_void_p()
        _check(load_library().cllm_hip_gguf_tensor(self._h, int(i), ctypes.byref(name),
                                                   ctypes.byref(t), ctypes.byref(nd), dims,
                                                   ctypes.byref(off), ctypes.byref(host),
                                                   ctypes.byref(dev)))
        return GgufTensorInfo(name.value.decode(), t.value, tuple(dims[:min(nd.value, 4)]),
                              off.value, host.value or 0, dev.value or 0)

    def find(self, name: str) -> int:
        return load_library().cllm_hip_gguf_find(self._h, name.encode())

    def config(self) -> ModelConfig:
        c = ModelConfig()
        _check(load_library().cllm_hip_gguf_config(self._h, ctypes.byref(c)))
        return c


# ---- float ops between the linear layers ------------------------------------------------

def rope_neox_dev(x, n_heads: int, head_dim: int, pos0: int, theta_base: float):
    """NEOX RoPE in place on x (float32 CUDA tensor of n_rows x n_heads x head_dim), row t at
    position pos0 + t -- engine.cpp:41-56."""
    n_rows = x.numel() // (n_heads * head_dim)
    _check(load_library().cllm_hip_rope_neox_dev(_tp(x), int(n_rows), int(n_heads),
                                                 int(head_dim), int(pos0), float(theta_base),
                                                 _stream()))
    return x


def rope_neox2_dev(q, n_head: int, k, n_head_kv: int, head_dim: int, pos0: int,
                   theta_base: float):
    """NEOX RoPE on the queries and the keys in one launch (engine.cpp:481-482)."""
    n_rows = q.numel() // (n_head * head_dim)
    _check(load_library().cllm_hip_rope_neox2_dev(_tp(q), int(n_head), _tp(k), int(n_head_kv),
                                                  int(n_rows), int(head_dim), int(pos0),
                                                  float(theta_base), _stream()))


def attention_dev(q, k_cache, v_cache, pos0: int, n_head: int, n_head_kv: int, head_dim: int,
                  out=None):
    """Grouped-query attention of the query rows q (n_rows x n_head x head_dim) over the
    caches (positions x n_head_kv x head_dim); row t sees positions [0, pos0 + t] --
    engine.cpp:114-146."""
    import torch
    n_rows = q.numel() // (n_head * head_dim)
    if out is None:
        out = torch.empty((n_rows, n_head * head_dim), dtype=torch.float32, device=q.device)
    _check(load_library().cllm_hip_attention_dev(_tp(q), _tp(k_cache), _tp(v_cache), int(n_rows),
                                                 int(pos0), int(n_head), int(n_head_kv),
                                                 int(head_dim), _tp(out), _stream()))
    return out


def attention_rope_dev(q, k_cache, v_cache, pos0: int, n_head: int, n_head_kv: int,
                       head_dim: int, theta_base: float, out=None):
    """A decode step's RoPE and attention in one launch (engine.cpp:486-495): q (one row,
    unrotated, left as it is) and the unrotated key row pos0 of k_cache (rotated in place) get
    the NEOX rotation at position pos0, then the attention over positions [0, pos0]."""
    import torch
    if out is None:
        out = torch.empty((1, n_head * head_dim), dtype=torch.float32, device=q.device)
    _check(load_library().cllm_hip_attention_rope_dev(
        _tp(q), _tp(k_cache), _tp(v_cache), int(pos0), int(n_head), int(n_head_kv),
        int(head_dim), float(theta_base), _tp(out), _stream()))
    return out


def dequantize_rows_dev(w, t: int, in_dim: int, ids, out=None):
    """Rows ids (int32 CUDA tensor) of the weight matrix w (uint8 CUDA tensor) as fp32 --
    the embedding lookup, bit for bit like dequantize_block."""
    import torch
    n = ids.numel()
    if out is None:
        out = torch.empty((n, in_dim), dtype=torch.float32, device=ids.device)
    _check(load_library().cllm_hip_dequantize_rows_dev(_tp(w), int(t), int(in_dim), _tp(ids),
                                                       int(n), _tp(out), _stream()))
    return out


# ---- the paged KV cache in 4 bits -----------------------------------------------------------

class _Kv4CacheStruct(ctypes.Structure):
    """cllm_hip_kv4_cache."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("pages", "table", "lens", "refs", "work")] + [
        (n, ctypes.c_int) for n in ("n_layers", "n_pages", "page_size", "n_head_kv", "head_dim",
                                    "max_seqs", "max_pages")]


def kv4_page_bytes(page_size: int, n_head_kv: int, head_dim: int) -> int:
    """Bytes of a page of one layer (0 for a shape that is not supported)."""
    return int(load_library().cllm_hip_kv4_page_bytes(int(page_size), int(n_head_kv), int(head_dim)))


def _addr(who: str, name: str, t, dtype, device: int, numel: int = -1) -> int:
    """t's address, after a check of what the kernels take from it: dtype, contiguous, on CUDA device
    `device`, of numel elements (when given)."""
    if (t is not None and t.dtype is dtype and t.is_contiguous() and t.get_device() == device
            and (numel < 0 or t.numel() == numel)):
        return t.data_ptr()
    if t is None:
        raise RuntimeError(f"{who}: {name} is None")
    if t.dtype is not dtype:
        raise RuntimeError(f"{who}: {name} must be {dtype}, not {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{who}: {name} must be contiguous")
    if t.get_device() != device:
        raise RuntimeError(f"{who}: {name} is on {t.device}, not on cuda:{device}")
    raise RuntimeError(f"{who}: {name} has {t.numel()} elements, not {numel}")


def _current(who: str, device: int):
    """(torch, the address of torch's current stream on `device`), which must be the current one."""
    import torch
    if device != torch._C._cuda_getDevice():
        if device < 0:
            raise RuntimeError(f"{who}: needs CUDA tensors")
        raise RuntimeError(f"{who}: tensors are on cuda:{device}, the current device is "
                           f"cuda:{torch.cuda.current_device()}")
    return torch, torch._C._cuda_getCurrentRawStream(device)


class Kv4Cache:
    """A paged KV cache in 4 bits (cllm_hip_kv4_cache, include/cllm_hip.h): pages (uint8,
    n_layers x n_pages x page bytes), table (int32, max_seqs x max_pages page ids, -1: none), lens
    (int32, max_seqs) and refs (int32, n_pages). Kv4Cache(...) makes an empty one on the device,
    from_tensors wraps a caller's. The kv4_*_dev functions work on it, on torch's current stream."""

    def __init__(self, n_layers: int, n_pages: int, max_seqs: int, max_pages: int, *,
                 page_size: int = 64, n_head_kv: int, head_dim: int, device="cuda"):
        import torch
        nbytes = kv4_page_bytes(page_size, n_head_kv, head_dim)
        if nbytes == 0 or min(n_layers, n_pages, max_seqs, max_pages) <= 0:
            raise RuntimeError("Kv4Cache: page_size must be a power of two from 32 to 1024, head_dim "
                               "64, 128 or 256, and every count positive")
        i32 = dict(dtype=torch.int32, device=device)
        self._set(torch.empty((n_layers, n_pages, nbytes), dtype=torch.uint8, device=device),
                  torch.full((max_seqs, max_pages), -1, **i32), torch.zeros(max_seqs, **i32),
                  torch.zeros(n_pages, **i32), page_size, n_head_kv, head_dim)

    @classmethod
    def from_tensors(cls, pages, table, lens, refs, *, page_size: int, n_head_kv: int, head_dim: int):
        self = cls.__new__(cls)
        self._set(pages, table, lens, refs, page_size, n_head_kv, head_dim)
        return self

    def _set(self, pages, table, lens, refs, page_size, n_head_kv, head_dim):
        import torch
        who = "Kv4Cache"
        nbytes = kv4_page_bytes(page_size, n_head_kv, head_dim)
        if pages.dim() != 3 or pages.shape[2] != nbytes or nbytes == 0:
            raise RuntimeError(f"{who}: pages must be n_layers x n_pages x {nbytes} bytes")
        if table.dim() != 2:
            raise RuntimeError(f"{who}: table must be max_seqs x max_pages")
        if not pages.is_cuda:
            raise RuntimeError(f"{who}: needs CUDA tensors, not {pages.device}")
        self.device = dev = pages.get_device()
        work = load_library().cllm_hip_kv4_work_ints(pages.shape[1], table.shape[0], table.shape[1])
        self.pages, self.table, self.lens, self.refs = pages, table, lens, refs
        self.work = torch.empty(int(work), dtype=torch.int32, device=pages.device)
        self.struct = _Kv4CacheStruct(
            _addr(who, "pages", pages, torch.uint8, dev), _addr(who, "table", table, torch.int32, dev),
            _addr(who, "lens", lens, torch.int32, dev, table.shape[0]),
            _addr(who, "refs", refs, torch.int32, dev, pages.shape[1]), self.work.data_ptr(),
            pages.shape[0], pages.shape[1], int(page_size), int(n_head_kv), int(head_dim),
            table.shape[0], table.shape[1])
        self._ref = ctypes.addressof(self.struct)
        self._shape = (int(n_head_kv), int(head_dim), table.shape[0])  # of what the calls check
        self._ws = {}  # attention scratch bytes by batch shape

    def attention_ws_bytes(self, *args) -> int:
        """cllm_hip_kv4_attention_ws_bytes for (n_seqs, n_rows, max_rows, max_len, n_head)."""
        n = self._ws.get(args)
        if n is None:
            if len(self._ws) >= 1024:
                self._ws.clear()
            n = self._ws[args] = int(load_library().cllm_hip_kv4_attention_ws_bytes(self._ref, *args))
        return n


def _kv4_batch(who, cache, i32, q_start, slots):
    """(slots, q_start, n_seqs) of a batch, checked."""
    qs = _addr(who, "q_start", q_start, i32, cache.device)
    n_seqs = q_start.numel() - 1
    if n_seqs < 0:
        raise RuntimeError(f"{who}: q_start has n_seqs + 1 elements")
    if slots is not None:
        return _addr(who, "slots", slots, i32, cache.device, n_seqs), qs, n_seqs
    if n_seqs > cache._shape[2]:
        raise RuntimeError(f"{who}: {n_seqs} sequences, {cache._shape[2]} slots")
    return None, qs, n_seqs


def kv4_extend_dev(cache: Kv4Cache, slots, counts, status=None):
    """Adds counts[i] tokens to slot slots[i] (int32 CUDA tensors; slots None: slot i) with the pages
    they need, copies of shared partly filled pages included. Returns status (int32, one element, on
    the device): 0, the number of pages missing, or -1 for bad entries; unless it is 0 nothing has
    changed."""
    who, dev = "kv4_extend", cache.device
    torch, stream = _current(who, dev)
    i32 = torch.int32
    c = _addr(who, "counts", counts, i32, dev)
    n = counts.numel()
    s = None
    if slots is not None:
        s = _addr(who, "slots", slots, i32, dev, n)
    elif n > cache._shape[2]:
        raise RuntimeError(f"{who}: {n} counts, {cache._shape[2]} slots")
    if status is None:
        status = torch.empty(1, dtype=i32, device=cache.pages.device)
    _check(load_library().cllm_hip_kv4_extend_dev(cache._ref, s, c, n, _addr(who, "status", status, i32, dev, 1),
                                                  stream))
    return status


def kv4_fork_dev(cache: Kv4Cache, src, dst) -> None:
    """Slot dst[i] becomes a copy of slot src[i] (int32 CUDA tensors), all at once; the pages are
    shared."""
    who, dev = "kv4_fork", cache.device
    torch, stream = _current(who, dev)
    n = src.numel()
    _check(load_library().cllm_hip_kv4_fork_dev(cache._ref, _addr(who, "src", src, torch.int32, dev),
                                                _addr(who, "dst", dst, torch.int32, dev, n), n, stream))


def kv4_truncate_dev(cache: Kv4Cache, slots, new_lens=None) -> None:
    """Cuts slot slots[i] to new_lens[i] tokens (None: to 0, freeing the sequences) and releases the
    pages past them."""
    who, dev = "kv4_truncate", cache.device
    torch, stream = _current(who, dev)
    n = slots.numel()
    new = None if new_lens is None else _addr(who, "new_lens", new_lens, torch.int32, dev, n)
    _check(load_library().cllm_hip_kv4_truncate_dev(cache._ref, _addr(who, "slots", slots, torch.int32, dev), new,
                                                    n, stream))


def kv4_compact_dev(cache: Kv4Cache, n_live=None):
    """Moves the pages in use to the front of the pool; returns their number (int32, one element, on
    the device)."""
    who, dev = "kv4_compact", cache.device
    torch, stream = _current(who, dev)
    if n_live is None:
        n_live = torch.empty(1, dtype=torch.int32, device=cache.pages.device)
    _check(load_library().cllm_hip_kv4_compact_dev(cache._ref, _addr(who, "n_live", n_live, torch.int32, dev, 1),
                                                   stream))
    return n_live


def kv4_copy_pages_dev(cache: Kv4Cache, src, dst) -> None:
    """Copies page src[i] to page dst[i] (int32 CUDA tensors) in every layer."""
    who, dev = "kv4_copy_pages", cache.device
    torch, stream = _current(who, dev)
    n = src.numel()
    _check(load_library().cllm_hip_kv4_copy_pages_dev(cache._ref, _addr(who, "src", src, torch.int32, dev),
                                                      _addr(who, "dst", dst, torch.int32, dev, n), n, stream))


def kv4_store_dev(cache: Kv4Cache, layer: int, k, v, q_start, slots=None, q=None, n_head: int = 0,
                  theta_base: float = 0.0) -> None:
    """Stores the rows k and v (float32, n_rows x n_head_kv x head_dim) as the last tokens of the
    batch's sequences: sequence i is slot slots[i] (None: slot i) and has rows q_start[i] ..
    q_start[i + 1]. theta_base > 0: the keys, and the query rows q in place, get the NEOX rotation of
    rope_neox2_dev at their positions first."""
    who, dev = "kv4_store", cache.device
    torch, stream = _current(who, dev)
    f32 = torch.float32
    s, qs, n_seqs = _kv4_batch(who, cache, torch.int32, q_start, slots)
    n_kv, hd, _ = cache._shape
    kp = _addr(who, "k", k, f32, dev)
    n = k.numel()
    n_rows = n // (n_kv * hd)
    if n_rows * n_kv * hd != n:
        raise RuntimeError(f"{who}: k has {n} elements, rows have {n_kv * hd}")
    vp = _addr(who, "v", v, f32, dev, n)
    qp = None if q is None else _addr(who, "q", q, f32, dev, n_rows * int(n_head) * hd)
    _check(load_library().cllm_hip_kv4_store_dev(cache._ref, layer, kp, vp, qp, n_head, theta_base, s, qs, n_seqs,
                                                 n_rows, stream))


def kv4_load_dev(cache: Kv4Cache, layer: int, q_start, n_rows: int, slots=None, k=None, v=None):
    """The rows' keys and values as float32 (n_rows x n_head_kv * head_dim), the batch as
    kv4_store_dev's (rows of no sequence are left as they are)."""
    who, dev = "kv4_load", cache.device
    torch, stream = _current(who, dev)
    f32 = torch.float32
    s, qs, n_seqs = _kv4_batch(who, cache, torch.int32, q_start, slots)
    n_rows = int(n_rows)
    shape = (n_rows, cache._shape[0] * cache._shape[1])
    if k is None:
        k = torch.empty(shape, dtype=f32, device=cache.pages.device)
    if v is None:
        v = torch.empty(shape, dtype=f32, device=cache.pages.device)
    n = shape[0] * shape[1]
    _check(load_library().cllm_hip_kv4_load_dev(cache._ref, layer, s, qs, n_seqs, n_rows,
                                                _addr(who, "k", k, f32, dev, n), _addr(who, "v", v, f32, dev, n),
                                                stream))
    return k, v


def kv4_attention_dev(cache: Kv4Cache, layer: int, q, q_start, *, n_head: int, max_rows: int,
                      max_len: int, slots=None, out=None):
    """Grouped-query attention of the rows q (float32, n_rows x n_head x head_dim) over the cache,
    the batch as kv4_store_dev's: row t of a sequence with r rows sees positions [0, len - r + t].
    max_rows and max_len bound a sequence's rows and tokens. Returns out (n_rows x n_head *
    head_dim); a row that sees nothing is 0, one of no sequence is left as it is."""
    who, dev = "kv4_attention", cache.device
    torch, stream = _current(who, dev)
    f32 = torch.float32
    s, qs, n_seqs = _kv4_batch(who, cache, torch.int32, q_start, slots)
    width = n_head * cache._shape[1]
    qp = _addr(who, "q", q, f32, dev)
    n = q.numel()
    n_rows = n // width if width > 0 else 0
    if width <= 0 or n_rows * width != n:
        raise RuntimeError(f"{who}: q has {n} elements, rows have {width}")
    if out is None:
        out = torch.empty((n_rows, width), dtype=f32, device=q.device)
    args = (n_seqs, n_rows, max_rows, max_len, n_head)
    nbytes = cache.attention_ws_bytes(*args)
    # scratch from torch's allocator: a captured call's belongs to its graph
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _check(load_library().cllm_hip_kv4_attention_dev(
        cache._ref, layer, qp, s, qs, n_seqs, n_rows, max_rows, max_len, n_head,
        _addr(who, "out", out, f32, dev, n), ws.data_ptr() if nbytes else None, nbytes, stream))
    return out


def kv4_attention_plan(cache: Kv4Cache, n_seqs: int, n_rows: int, max_rows: int, max_len: int,
                       n_head: int) -> str:
    """The kernel and launch plan of kv4_attention_dev for this shape."""
    return load_library().cllm_hip_kv4_attention_plan(cache._ref, int(n_seqs), int(n_rows), int(max_rows),
                                                      int(max_len), int(n_head)).decode()


# ---- log probabilities ------------------------------------------------------------------------

@dataclass
class LogProbs:
    """What logprobs_dev returns: CUDA tensors (None: not asked for)."""
    logprobs: object      # float32 [n_rows], of the given tokens
    ranks: object         # int32 [n_rows], tokens ahead of them
    entropy: object       # float32 [n_rows]
    lse: object           # float32 [n_rows]
    top_ids: object       # int32 [n_rows, top_k]
    top_logprobs: object  # float32 [n_rows, top_k]


def logprobs_dev(logits, tokens=None, top_k: int = 0) -> LogProbs:
    """Log probabilities of the rows of logits (float32 (n_rows, vocab), unit stride along a row, a
    row stride of vocab or more): of the given tokens (int32 (n_rows,)) with their ranks, the entropy and
    log-sum-exp, and the top_k (at most 64) largest with their ids, equal logits by ids."""
    who, dev = "logprobs", logits.get_device()
    torch, stream = _current(who, dev)
    f32, i32, device = torch.float32, torch.int32, logits.device
    if logits.dim() != 2 or logits.dtype is not f32:
        raise RuntimeError(f"{who}: logits must be float32 n_rows x vocab")
    m, vocab = logits.shape
    stride, along = logits.stride()
    if vocab > 1 and along != 1:
        raise RuntimeError(f"{who}: the logits of a row must lie side by side")
    if m <= 1:
        stride = vocab
    lib = load_library()
    nbytes = int(lib.cllm_hip_logprobs_ws_bytes(m, vocab, top_k))
    tp = lp = ranks = tid = ttop = None
    per_row = 3 if tokens is not None else 2
    per = torch.empty((per_row, m), dtype=f32, device=device).unbind(0)
    if tokens is not None:
        tp = _addr(who, "tokens", tokens, i32, dev, m)
        lp, ranks = per[2], torch.empty(m, dtype=i32, device=device)
    top_ids = torch.empty((m, top_k), dtype=i32, device=device)
    top_lp = torch.empty((m, top_k), dtype=f32, device=device)
    if top_k:
        tid, ttop = top_ids.data_ptr(), top_lp.data_ptr()
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    r = LogProbs(lp, ranks, per[0], per[1], top_ids, top_lp)
    _check(lib.cllm_hip_logprobs_dev(logits.data_ptr(), stride, m, vocab, tp, top_k,
                                     None if lp is None else lp.data_ptr(),
                                     None if ranks is None else ranks.data_ptr(), per[0].data_ptr(),
                                     per[1].data_ptr(), tid, ttop, None if ws is None else ws.data_ptr(), nbytes,
                                     stream))
    return r


@dataclass
class RowGroups:
    """Entries grouped by index: order (int32, n) lists them sorted by group, those of group g at
    order[offsets[g]:offsets[g + 1]], those of no group from offsets[-1] on (offsets: int32, groups + 1)."""
    offsets: object
    order: object


@dataclass
class MoeRoute:
    """A router's choice (cllm_hip_moe_route_dev): ids (int32) and weights (float32), n_rows x top_k, -1 and
    0 for no expert, and the entries row * top_k + j grouped by expert as RowGroups has them."""
    ids: object
    weights: object
    offsets: object
    order: object


def group_rows_dev(ids, n_groups: int) -> RowGroups:
    """The entries of ids (int32 (n,)) grouped by id; ids outside [0, n_groups) are of no group."""
    who, dev = "group_rows", ids.get_device()
    torch, stream = _current(who, dev)
    p = _addr(who, "ids", ids, torch.int32, dev)
    if n_groups < 1:
        raise RuntimeError(f"{who}: n_groups must be positive")
    n = ids.numel()
    g = RowGroups(torch.empty(n_groups + 1, dtype=torch.int32, device=ids.device),
                  torch.empty(n, dtype=torch.int32, device=ids.device))
    _check(load_library().cllm_hip_group_rows_dev(p, n, n_groups, g.offsets.data_ptr(), g.order.data_ptr(), stream))
    return g


def moe_route_dev(logits, top_k: int, bias=None, sigmoid: bool = False, normalise: bool = True,
                  scale: float = 1.0, n_groups: int = 1, top_groups: int = 1) -> MoeRoute:
    """A router's choice of top_k experts for the rows of logits (float32 (n_rows, n_experts), unit stride
    along a row): softmax or sigmoid scores, chosen by logit or, with bias (float32 (n_experts,)), by
    score + bias, from the top_groups best of n_groups groups of experts; weights are the chosen scores,
    normalised to sum 1 or not, times scale."""
    who, dev = "moe_route", logits.get_device()
    torch, stream = _current(who, dev)
    if logits.dim() != 2 or logits.dtype is not torch.float32:
        raise RuntimeError(f"{who}: logits must be float32 n_rows x n_experts")
    m, experts = logits.shape
    stride, along = logits.stride()
    if experts > 1 and along != 1:
        raise RuntimeError(f"{who}: the logits of a row must lie side by side")
    if m <= 1:
        stride = experts
    bp = None if bias is None else _addr(who, "bias", bias, torch.float32, dev, experts)
    # one allocation: ids, order, offsets
    k = max(top_k, 0)
    ints = torch.empty(2 * m * k + experts + 1, dtype=torch.int32, device=logits.device)
    weights = torch.empty((m, k), dtype=torch.float32, device=logits.device)
    ids, order, offsets = ints.split((m * k, m * k, experts + 1))
    r = MoeRoute(ids.view(m, k), weights, offsets, order)
    at = ints.data_ptr()
    _check(load_library().cllm_hip_moe_route_dev(
        logits.data_ptr(), stride, bp, m, experts, top_k, int(sigmoid), int(normalise), scale, n_groups,
        top_groups, at, weights.data_ptr(), at + 8 * m * k, at + 4 * m * k, stream))
    return r


def _moe_args(who, x, w, t, out_dim, groups):
    """(in_dim, rows of x, experts) of an expert product, after the checks of its tensors' sizes."""
    if x.dim() < 2:
        raise RuntimeError(f"{who}: activations must have two dimensions")
    in_dim = x.shape[-1]
    rows = x.numel() // in_dim if in_dim else 0
    experts = groups.offsets.numel() - 1
    if experts < 1:
        raise RuntimeError(f"{who}: offsets must have n_experts + 1 elements")
    per = block_size(t) if has_vec_dot(t) else 0
    if per and in_dim % per == 0:
        need = experts * out_dim * (in_dim // per) * type_size(t)
        for name, m in w:
            if m.numel() * m.element_size() != need:
                raise RuntimeError(f"{who}: {name} has {m.numel() * m.element_size()} bytes, not {need}")
    return in_dim, rows, experts


def moe_matmul_dev(x, w, t: int, out_dim: int, groups: RowGroups, bias=None, per_row: int = 1, y=None):
    """The products of entries with the matrices of their groups: entry e has row e // per_row of x
    (float32 (n_rows, in_dim)) and w (uint8, the GGUF blocks of [n_experts][out_dim] rows of type t). Returns
    y (n_rows * per_row, out_dim); entries of no group leave their row as it is."""
    who, dev = "moe_matmul", x.get_device()
    torch, stream = _current(who, dev)
    f32, i32 = torch.float32, torch.int32
    in_dim, rows, experts = _moe_args(who, x, (("w", w),), t, out_dim, groups)
    n = rows * per_row
    if y is None:
        y = torch.empty((n, out_dim), dtype=f32, device=x.device)
    lib = load_library()
    nbytes = int(lib.cllm_hip_moe_matmul_ws_bytes(t, in_dim, rows))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _check(lib.cllm_hip_moe_matmul_dev(
        t, in_dim, out_dim, experts, _addr(who, "w", w, torch.uint8, dev),
        None if bias is None else _addr(who, "bias", bias, f32, dev, experts * out_dim),
        _addr(who, "x", x, f32, dev), rows, per_row, _addr(who, "offsets", groups.offsets, i32, dev),
        _addr(who, "order", groups.order, i32, dev, n), _addr(who, "y", y, f32, dev, n * out_dim), ws.data_ptr(),
        nbytes, stream))
    return y


def moe_swiglu_dev(x, w_gate, w_up, t: int, n_ff: int, route: MoeRoute, bias_gate=None, bias_up=None, h=None):
    """silu(gate) * up of every row of x (float32 (n_rows, in_dim)) and each of its chosen experts: w_gate and
    w_up are the GGUF blocks (uint8) of [n_experts][n_ff] rows of type t. Returns h (n_rows, top_k, n_ff); what
    has no expert is left as it is."""
    who, dev = "moe_swiglu", x.get_device()
    torch, stream = _current(who, dev)
    f32, i32 = torch.float32, torch.int32
    in_dim, rows, experts = _moe_args(who, x, (("w_gate", w_gate), ("w_up", w_up)), t, n_ff, route)
    if route.ids.dim() != 2 or route.ids.shape[0] != rows:
        raise RuntimeError(f"{who}: x has {rows} rows, the route {tuple(route.ids.shape)}")
    top_k = route.ids.shape[1]
    n = rows * top_k
    if h is None:
        h = torch.empty((rows, top_k, n_ff), dtype=f32, device=x.device)
    lib = load_library()
    nbytes = int(lib.cllm_hip_moe_matmul_ws_bytes(t, in_dim, rows))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _check(lib.cllm_hip_moe_swiglu_dev(
        t, in_dim, n_ff, experts, _addr(who, "w_gate", w_gate, torch.uint8, dev),
        _addr(who, "w_up", w_up, torch.uint8, dev),
        None if bias_gate is None else _addr(who, "bias_gate", bias_gate, f32, dev, experts * n_ff),
        None if bias_up is None else _addr(who, "bias_up", bias_up, f32, dev, experts * n_ff),
        _addr(who, "x", x, f32, dev), rows, top_k, _addr(who, "offsets", route.offsets, i32, dev),
        _addr(who, "order", route.order, i32, dev, n), _addr(who, "h", h, f32, dev, n * n_ff), ws.data_ptr(),
        nbytes, stream))
    return h


def moe_down_dev(h, w, t: int, out_dim: int, route: MoeRoute, bias=None, base=None, y=None):
    """The down projections of h (float32, n_rows x top_k x n_ff) with the chosen experts' matrices (GGUF blocks
    of [n_experts][out_dim] rows of type t), summed over a row's experts with the route's weights, plus base
    (float32 (n_rows, out_dim), the residual; may be y). Returns y (n_rows, out_dim)."""
    who, dev = "moe_down", h.get_device()
    torch, stream = _current(who, dev)
    f32, i32 = torch.float32, torch.int32
    n_ff, n, experts = _moe_args(who, h, (("w", w),), t, out_dim, route)
    if route.ids.dim() != 2 or route.ids.numel() != n:
        raise RuntimeError(f"{who}: h has {n} rows, the route {tuple(route.ids.shape)}")
    rows, top_k = route.ids.shape
    if y is None:
        y = torch.empty((rows, out_dim), dtype=f32, device=h.device)
    lib = load_library()
    nbytes = int(lib.cllm_hip_moe_down_ws_bytes(t, n_ff, out_dim, rows, top_k))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
    _check(lib.cllm_hip_moe_down_dev(
        t, n_ff, out_dim, experts, _addr(who, "w", w, torch.uint8, dev),
        None if bias is None else _addr(who, "bias", bias, f32, dev, experts * out_dim),
        _addr(who, "h", h, f32, dev), rows, top_k, _addr(who, "ids", route.ids, i32, dev, n),
        _addr(who, "weights", route.weights, f32, dev, n), _addr(who, "offsets", route.offsets, i32, dev),
        _addr(who, "order", route.order, i32, dev, n),
        None if base is None else _addr(who, "base", base, f32, dev, rows * out_dim),
        _addr(who, "y", y, f32, dev, rows * out_dim), ws.data_ptr(), nbytes, stream))
    return y


def moe_plan(t: int, n_mats: int, in_dim: int, out_dim: int, n_experts: int, n_entries: int) -> str:
    """The kernel and launch plan of the experts' products of n_entries entries."""
    return load_library().cllm_hip_moe_plan(t, n_mats, in_dim, out_dim, n_experts, n_entries).decode()


def lora_dev(x, a, b, groups: RowGroups, ranks=None, scales=None, base=None, ys=None):
    """Low-rank adapters on the projections of x (float32 (n_rows, in_dim)), rows grouped by adapter: a[i]
    (n_adapters, max_rank, in_dim) and b[i] (n_adapters, out_dims[i], max_rank), float16 or float32, of 1 to 4
    projections; ranks (int32) and scales (float32) (n_adapters,). Returns the list of base[i] + scale * b[i]
    (a[i] x) (base None: zeros), base[i] for rows of no adapter."""
    who, dev = "lora", x.get_device()
    torch, stream = _current(who, dev)
    f32, i32 = torch.float32, torch.int32
    n = len(a)
    if n == 0 or len(b) != n or (base is not None and len(base) != n) or (ys is not None and len(ys) != n):
        raise RuntimeError(f"{who}: a, b, base and ys must have an entry for each projection")
    first = a[0]
    if x.dim() != 2 or first.dim() != 3:
        raise RuntimeError(f"{who}: x must be n_rows x in_dim, a[i] n_adapters x max_rank x in_dim")
    rows, in_dim = x.shape
    shape, dt = first.shape, first.dtype
    adapters, max_rank, k = shape
    half = dt is torch.float16
    if not half and dt is not f32:
        raise RuntimeError(f"{who}: adapters must be float16 or float32")
    if k != in_dim:
        raise RuntimeError(f"{who}: x has rows of {in_dim}, a of {k}")
    ptrs, ints = ctypes.c_void_p * n, ctypes.c_int * n
    outs, ap, bp, yp = ints(), ptrs(), ptrs(), ptrs()
    basep = None if base is None else ptrs()
    new = [] if ys is None else ys
    for i in range(n):
        m, w = a[i], b[i]
        if m.shape != shape or w.dim() != 3 or w.shape[0] != adapters or w.shape[2] != max_rank:
            raise RuntimeError(f"{who}: shapes of adapter {i} do not match: {tuple(m.shape)}, {tuple(w.shape)}")
        ap[i] = _addr(who, "a", m, dt, dev)
        bp[i] = _addr(who, "b", w, dt, dev)
        outs[i] = out = w.shape[1]
        if ys is None:
            y = torch.empty((rows, out), dtype=f32, device=x.device)
            new.append(y)
            yp[i] = y.data_ptr()
        else:
            yp[i] = _addr(who, "y", ys[i], f32, dev, rows * out)
        if basep is not None and base[i] is not None:
            basep[i] = _addr(who, "base", base[i], f32, dev, rows * out)
    ys = new
    lib = load_library()
    nbytes = lib.cllm_hip_lora_ws_bytes(in_dim, n, adapters, max_rank, rows)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _check(lib.cllm_hip_lora_dev(
        1 if half else 0, in_dim, n, ap, bp, outs, adapters, max_rank,
        None if ranks is None else _addr(who, "ranks", ranks, i32, dev, adapters),
        None if scales is None else _addr(who, "scales", scales, f32, dev, adapters),
        _addr(who, "x", x, f32, dev), rows, _addr(who, "offsets", groups.offsets, i32, dev, adapters + 1),
        _addr(who, "order", groups.order, i32, dev, rows), basep, yp, ws.data_ptr(), nbytes, stream))
    return ys
