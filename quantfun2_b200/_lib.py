"""ctypes binding of libqf2b200.so (the C ABI declared in include/qf2b200.h).

The library is built in-tree by ``quantfun2_b200/build.py``.  There is no CPU or
PyTorch fallback: if the shared object is missing, or the current device is not
an sm_100 part, every op raises.
"""
from __future__ import annotations

import ctypes
import functools
import os
import struct
from ctypes import c_float, c_int, c_int64, c_void_p, POINTER
from pathlib import Path

# QF2_LIBRARY may name another build of the same library (same C ABI), e.g. one compiled
# with different tuning macros; the default is the in-tree build.
LIB_PATH = Path(os.environ.get("QF2_LIBRARY") or Path(__file__).resolve().parent / "libqf2b200.so")

QF2_OK = 0
QF2_F32, QF2_F16, QF2_BF16, QF2_I8, QF2_E4M3, QF2_I32 = range(6)
QF2_ROPE_FP16_TRIG = 1
QF2_RMS_EAGER, QF2_RMS_FUSED = 0, 1
QF2_ROTARY_HALF, QF2_ROTARY_INTERLEAVED = 0, 1
QF2_OFFSET_CONST, QF2_OFFSET_ARRAY, QF2_OFFSET_END = 0, 1, 2

_P64 = POINTER(c_int64)
_P32 = POINTER(ctypes.c_int32)



class _Args:
    """An argument struct of include/qf2b200.h whose fields are all 8 bytes, filled by one
    struct.pack: a ctypes call of two dozen arguments costs the host more than a small kernel
    takes.  `fields`: (name, count, format q or d) in order."""

    def __init__(self, fields):
        self.fields = fields
        self._struct = struct.Struct("=" + "".join(f"{n}{f}" for _, n, f in fields))
        self.pack = self._struct.pack

    def pack_named(self, **values) -> bytes:
        flat = []
        for name, n, _ in self.fields:
            v = values.get(name) or 0
            flat += list(v) if isinstance(v, (tuple, list)) else [v] * n
        return self.pack(*flat)


ROTARY_ARGS = _Args([
    ("xq", 1, "q"), ("xq_out", 1, "q"), ("xk", 1, "q"), ("xk_out", 1, "q"), ("positions", 1, "q"), ("inv_freq", 1, "q"),
    ("xq_strides", 3, "q"), ("xq_out_strides", 3, "q"), ("xk_strides", 3, "q"), ("xk_out_strides", 3, "q"),
    ("pos_strides", 2, "q"), ("pos_is_i64", 1, "q"), ("B", 1, "q"), ("S", 1, "q"), ("Hq", 1, "q"), ("Hk", 1, "q"),
    ("D", 1, "q"), ("rotary_dim", 1, "q"), ("layout", 1, "q"), ("inverse", 1, "q"), ("dtype", 1, "q"), ("gain", 1, "d"),
    ("stream", 1, "q")])
MASKED_ATTN_ARGS = _Args([
    ("q", 1, "q"), ("k", 1, "q"), ("v", 1, "q"), ("out", 1, "q"), ("prefix_k", 1, "q"), ("prefix_v", 1, "q"),
    ("q_strides", 3, "q"), ("k_strides", 3, "q"), ("v_strides", 3, "q"), ("out_strides", 3, "q"),
    ("prefix_k_strides", 2, "q"), ("prefix_v_strides", 2, "q"), ("B", 1, "q"), ("Hq", 1, "q"), ("Hkv", 1, "q"),
    ("Sq", 1, "q"), ("Skv", 1, "q"), ("P", 1, "q"), ("D", 1, "q"), ("dtype", 1, "q"), ("left", 1, "q"), ("right", 1, "q"),
    ("kv_lens", 1, "q"), ("prefix_lens", 1, "q"), ("q_offsets", 1, "q"), ("q_offset", 1, "q"), ("q_offset_mode", 1, "q"),
    ("q_ids", 1, "q"), ("k_ids", 1, "q"), ("ids_i64", 1, "q"), ("slopes", 1, "q"), ("bias_table", 1, "q"), ("bias_reach", 1, "q"),
    ("softcap", 1, "d"), ("sm_scale", 1, "d"), ("workspace", 1, "q"), ("workspace_bytes", 1, "q"), ("stream", 1, "q")])


# name -> (restype, argtypes); mirrors include/qf2b200.h
SIGNATURES = {
    "qf2_version": (ctypes.c_char_p, []),
    "qf2_status_string": (ctypes.c_char_p, [c_int]),
    "qf2_last_error": (ctypes.c_char_p, []),
    "qf2_device_check": (c_int, []),
    "qf2_workspace_status": (c_int, [c_void_p, c_void_p]),
    "qf2_rope_apply": (
        c_int,
        [c_void_p, c_void_p, c_int64, _P64, _P64, c_void_p, c_void_p, c_int64, _P64, _P64, c_void_p, _P64,
         c_int64, c_int64, c_int64, c_int, c_int, c_void_p],
    ),
    "qf2_rms_gate_residual": (
        c_int,
        [c_void_p, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_void_p, c_float, c_void_p, c_int64, c_int,
         c_void_p, c_float, c_void_p, c_int64, c_void_p],
    ),
    "qf2_qkv_norm_rope": (
        c_int,
        [c_void_p, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_void_p, _P64, c_void_p, _P64,
         c_void_p, _P64, c_void_p, c_void_p, c_float, c_void_p, _P64, c_void_p],
    ),
    "qf2_rmsnorm": (
        c_int,
        [c_void_p, c_int64, c_int, c_void_p, c_int, c_void_p, c_int64, c_int, c_int64, c_int64, c_float, c_int,
         c_void_p],
    ),
    "qf2_softmax_inplace": (c_int, [c_void_p, c_int64, c_int64, c_int64, c_int, c_void_p]),
    "qf2_sage_workspace_bytes": (
        c_int64, [c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64]),
    "qf2_sage_workspace_layout": (
        c_int, [c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, _P64]),
    "qf2_sageattn": (
        c_int,
        [c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, c_int64, c_int64, c_int64, c_int64,
         c_int64, c_int64, c_float, c_int, c_void_p, c_int64, c_void_p],
    ),
    "qf2_sageattn_varlen": (
        c_int,
        [c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, _P32, _P32, c_int64, c_int64, c_int64,
         c_int64, c_int64, c_int64, c_int64, c_int64, c_float, c_int, c_void_p, c_int64, c_void_p],
    ),
    "qf2_sage_quantize": (
        c_int,
        [c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, _P32, _P32, c_int64, c_int64, c_int64, c_int64, c_int64,
         c_int64, c_int64, c_int64, c_int64, c_int64, c_float, c_int, c_void_p, c_int64, c_void_p],
    ),
    "qf2_sage_attn_quantized": (
        c_int,
        [c_void_p, _P64, _P32, _P32, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64,
         c_int64, c_int64, c_int, c_void_p, c_int64, c_void_p],
    ),
    "qf2_blocktopk_workspace_bytes": (c_int64, [c_int64, c_int64, c_int64, c_int64, c_int64]),
    "qf2_blocktopk_select": (
        c_int,
        [c_void_p, _P64, c_void_p, _P64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int, c_void_p,
         c_void_p, c_int64, c_void_p],
    ),
    "qf2_blocksparse_attn": (
        c_int,
        [c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, c_int64, c_int64, c_int64, c_int64,
         c_int64, c_void_p, c_int64, c_float, c_int, c_void_p, c_int64, c_void_p],
    ),
    "qf2_rotary_apply": (c_int, [ctypes.c_char_p]),
    "qf2_masked_attn_workspace_bytes": (
        c_int64, [c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int64, c_int]),
    "qf2_masked_attn": (c_int, [ctypes.c_char_p]),
    "qf2_masked_attn_status": (c_int, [c_void_p]),
    "qf2_masked_attn_fault_injection": (c_int, [c_int64, c_int]),
    "qf2_masked_attn_plan": (c_int, [ctypes.c_char_p, _P64]),
    "qf2_quantize_rows": (
        c_int, [c_void_p, c_int64, c_int, c_int64, c_int64, c_void_p, c_int64, c_int, c_void_p, c_void_p]),
    "qf2_codes_to_bf16": (c_int, [c_void_p, c_int64, c_int, c_int64, c_int64, c_void_p, c_int64, c_void_p]),
    "qf2_gemm": (
        c_int,
        [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int, c_int,
         c_void_p, c_void_p, c_void_p, c_int, c_void_p, c_int64, c_void_p],
    ),
    "qf2_quantize_weight_rows": (
        c_int, [c_void_p, c_int64, c_int, c_int64, c_int64, c_void_p, c_int64, c_int, c_void_p, c_void_p]),
    "qf2_codes_convert": (
        c_int, [c_void_p, c_int64, c_int, c_int64, c_int64, c_void_p, c_int64, c_int, c_void_p]),
    "qf2_gemm_rows_indexed": (
        c_int,
        [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int64, c_int, c_int,
         c_void_p, c_int64, c_void_p, c_void_p, c_int, c_void_p, c_int64, c_void_p]),
    "qf2_rope_scatter": (
        c_int,
        [c_void_p, _P64, c_void_p, c_int64, c_void_p, c_void_p, _P64, c_int64, c_int64, c_int64, c_int64, c_int64,
         c_int, c_void_p, c_void_p]),
    "qf2_gemm_codes": (
        c_int,
        [c_void_p, c_int64, c_void_p, c_int64, c_int, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int, c_int,
         c_void_p, c_void_p, c_void_p, c_int, c_int64, c_int, c_void_p, c_int64, c_void_p, c_int64, c_int64,
         c_void_p, c_int64, c_void_p],
    ),
    "qf2_gemm_ex": (
        c_int,
        [c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_int64, c_int64, c_int64, c_int, c_int,
         c_void_p, c_void_p, c_void_p, c_int, c_int64, c_int, c_void_p, c_int64, c_void_p, c_int64, c_int64,
         c_void_p, c_int64, c_void_p],
    ),
    "qf2_ln_modulate": (
        c_int,
        [c_void_p, c_int64, c_int, c_void_p, c_void_p, c_int64, c_int64, c_int64, c_int64, c_float, c_void_p,
         c_int64, c_int, c_void_p, c_void_p],
    ),
    "qf2_copy_chunks": (c_int, [c_void_p, c_void_p, c_int64, _P64, _P64, _P64, c_void_p]),
    "qf2_sageattn_noalloc": (
        c_int,
        [c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, c_void_p, _P64, c_int64, c_int64, c_int64, c_int64,
         c_int64, c_int64, c_float, c_int, c_void_p],
    ),
    "qf2_sageattn_noalloc_status": (c_int, [c_void_p]),
    "qf2_sage_fault_injection": (c_int, [c_int64, c_int]),
}

_lib = None


class QF2Error(RuntimeError):
    pass


def load() -> ctypes.CDLL:
    """Load the shared library (once) and bind every declared entry point."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise QF2Error(
            f"{LIB_PATH} is missing; build it with `python quantfun2_b200/build.py` "
            "(there is no CPU fallback)")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def check(status: int, what: str) -> None:
    if status != QF2_OK:
        lib = load()
        msg = lib.qf2_status_string(status).decode()
        if status == -3:
            msg += ": " + lib.qf2_last_error().decode()
        raise QF2Error(f"{what} failed: {msg} ({status})")


def i64(*vals) -> ctypes.Array:
    return (c_int64 * len(vals))(*[int(v) for v in vals])


def ptr32(t) -> ctypes._Pointer:
    return ctypes.cast(c_void_p(t.data_ptr()), _P32)


_device_ok: dict[int, bool] = {}


def require_device(t) -> None:
    """Raise unless `t` lives on an sm_100 CUDA device."""
    import torch

    if not t.is_cuda:
        raise QF2Error("quantfun2_b200 ops run on CUDA tensors only (no CPU fallback)")
    idx = t.device.index if t.device.index is not None else torch.cuda.current_device()
    ok = _device_ok.get(idx)
    if ok is None:
        ok = torch.cuda.get_device_capability(idx) == (10, 0)
        _device_ok[idx] = ok
    if not ok:
        raise QF2Error(f"device {idx} is not compute capability 10.0 (B200); sm_100a kernels only")


def call_on(device, fn, args: bytes) -> int:
    """fn(args) with `device` current (the library launches on the current device)."""
    import torch

    if device.index == torch._C._cuda_getDevice():
        return fn(args)
    with torch.cuda.device(device):
        return fn(args)


def raw_stream(index: int) -> int:
    """Handle of the current stream of device `index`."""
    import torch

    return torch._C._cuda_getCurrentRawStream(index)


def stream_ptr(device=None) -> c_void_p:
    import torch

    return c_void_p(torch.cuda.current_stream(device).cuda_stream)


_autograd = None


def wants_derivative(*tensors) -> bool:
    """Whether a gradient would be asked of any of the tensors (None among them), or one carries
    a forward-mode tangent: the ops have neither, and must not drop them."""
    global _autograd
    if _autograd is None:
        import torch
        from torch.autograd import forward_ad

        _autograd = torch.is_grad_enabled, forward_ad
    grad_enabled, forward_ad = _autograd
    if grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level < 0:
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def overlaps_itself(t) -> bool:
    """Whether elements of t may share memory (expanded or unfolded views)."""
    return not t.is_contiguous() and _folded(t.stride(), t.shape)


def overlap(a, b) -> bool:
    """Whether an element of a may lie on one of b."""
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa <= pb and a.is_contiguous() and pa + a.nbytes <= pb or pb <= pa and b.is_contiguous() and pb + b.nbytes <= pa:
        return False  # (the common case)
    return _overlap(pb - pa, a.stride(), a.shape, a.element_size(), b.stride(), b.shape, b.element_size())


@functools.lru_cache(maxsize=1024)
def _folded(strides, shape) -> bool:
    ext = 1
    for s, n in sorted(zip(strides, shape)):
        if n == 0:
            return False
        if n > 1:
            if s < ext:
                return 0 not in shape
            ext += s * (n - 1)
    return False


@functools.lru_cache(maxsize=1024)
def _overlap(delta, sa, na, ea, sb, nb, eb) -> bool:
    """b begins delta bytes behind a; strides and sizes, bytes of an element.  Slices of one
    buffer are told apart by a stride of theirs: all strides from it on are its multiples, and
    within one step of it a and b lie side by side."""
    if 0 in na or 0 in nb:
        return False
    da = [(s * ea, n - 1) for s, n in zip(sa, na) if n > 1]
    db = [(s * eb, n - 1) for s, n in zip(sb, nb) if n > 1]
    if ea + sum(s * n for s, n in da) <= delta or eb + sum(s * n for s, n in db) <= -delta:
        return False
    strides = {s for s, _ in da + db if s}
    for p in strides:
        if any(s > p and s % p for s in strides):
            continue
        ia, ib = (e + sum(s * n for s, n in d if s < p) for e, d in ((ea, da), (eb, db)))
        if ia <= delta % p and delta % p + ib <= p:
            return False
    return True


_dtype_codes: dict = {}


def dtype_code(dt) -> int:
    if not _dtype_codes:
        import torch

        _dtype_codes.update({torch.float32: QF2_F32, torch.float16: QF2_F16, torch.bfloat16: QF2_BF16})
    code = _dtype_codes.get(dt)
    if code is None:
        raise QF2Error(f"unsupported dtype {dt}")
    return code


def header_symbols(header: str | os.PathLike | None = None) -> list[str]:
    """Function names declared in include/qf2b200.h."""
    import re

    h = Path(header) if header else Path(__file__).resolve().parent.parent / "include" / "qf2b200.h"
    text = h.read_text()
    return sorted(set(re.findall(r"^\s*(?:const\s+)?[a-z0-9_]+\*?\s+\*?(qf2_[a-z0-9_]+)\s*\(", text, re.M)))
