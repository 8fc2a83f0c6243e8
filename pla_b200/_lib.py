"""ctypes binding of libpla_b200.so (the C ABI declared in include/pla_b200.h).

The shared library is built in-tree (``python -m pla_b200.build``); importing
the ops without it, or calling them on a non-CUDA tensor, raises: there is no
CPU or eager-PyTorch fallback anywhere in this package.
"""
from __future__ import annotations

import contextlib
import ctypes
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libpla_b200.so")
TORCH_LIB_PATH = os.path.join(_HERE, "libpla_b200_torch.so")

PLA_F16, PLA_F32, PLA_F64, PLA_BF16 = 0, 1, 2, 3
PLA_OK, PLA_ERR_UNSUPPORTED = 0, 2
PLA_NCHW, PLA_NHWC = 0, 1

DTYPE_CODE = {
    torch.float16: PLA_F16,
    torch.float32: PLA_F32,
    torch.float64: PLA_F64,
    torch.bfloat16: PLA_BF16,
}

# Every symbol include/pla_b200.h declares, with its ctypes signature.
_vp, _i32, _i64, _u32p = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.POINTER(ctypes.c_uint)
_f32p = ctypes.POINTER(ctypes.c_float)
SIGNATURES = {
    "pla_status_string": ([_i32], ctypes.c_char_p),
    "pla_last_cuda_error": ([], ctypes.c_char_p),
    "pla_version": ([], _i32),
    "pla_stencil7x7_forward": ([_vp, _vp, _vp, _vp, _i32, _i32, _i32, _i64, _i64, _i64, _i32, _vp], _i32),
    "pla_stencil7x7_forward_taps": ([_vp, _f32p, _f32p, _vp, _i32, _i32, _i32, _i64, _i64, _i64, _i32, _vp], _i32),
    "pla_depthwise7x7_forward": ([_vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_depthwise_forward": ([_vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_depthwise7x7_forward_many": ([_vp, _i32, _i32, _i32, _vp], _i32),
    "pla_depthwise7x7_layernorm_nhwc": ([_vp, _vp, _vp, _vp, _vp, ctypes.c_float, _vp, _i32, _i32, _i32, _i32, _i32,
                                         _vp], _i32),
    "pla_stencil7x7_iterate": ([_vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_stencil7x7_iterate_noalloc": ([_vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_stencil7x7_iterate_taps": ([_vp, _f32p, _f32p, _vp, _vp, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_stencil7x7_band_step": ([_vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_stencil7x7_band_step_taps": ([_vp, _f32p, _f32p, _vp, _i32, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_stencil7x7_band_step_halo": ([_vp, _f32p, _f32p, _vp, _i32, _i32, _i32, _vp, _i32, _vp, _vp, _vp, _vp,
                                       _vp, ctypes.c_uint, _vp], _i32),
    "pla_ipc_export": ([_vp, _vp, ctypes.POINTER(ctypes.c_uint64)], _i32),
    "pla_ipc_import": ([_vp, ctypes.c_uint64, ctypes.POINTER(ctypes.c_void_p)], _i32),
    "pla_ipc_close": ([_vp, ctypes.c_uint64], _i32),
    "pla_causal_depthwise_forward": ([_vp, _vp], _i32),
    "pla_causal_depthwise_workspace": ([_vp], ctypes.c_size_t),
    "pla_causal_depthwise_backward": ([_vp, _vp, _vp], _i32),
    "pla_causal_depthwise_step": ([_vp, _i64, _vp, _i64, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _vp], _i32),
    "pla_qk_norm_rotate_forward": ([_vp, _vp], _i32),
    "pla_qk_norm_rotate_workspace": ([_vp], ctypes.c_size_t),
    "pla_qk_norm_rotate_backward": ([_vp, _vp, ctypes.c_size_t, _vp], _i32),
    "pla_gated_delta_rule_workspace": ([_vp, _i32], ctypes.c_size_t),
    "pla_gated_delta_rule_forward": ([_vp, _vp], _i32),
    "pla_gated_delta_rule_backward": ([_vp, _vp, _vp], _i32),
    "pla_gated_delta_rule_step": ([_vp, _vp], _i32),
    "pla_read_device_faults": ([_u32p], _i32),
    "pla_clear_device_faults": ([], _i32),
}

class DwProblem(ctypes.Structure):
    """pla_dw_problem (include/pla_b200.h): one problem of pla_depthwise7x7_forward_many."""

    _fields_ = [("x", ctypes.c_void_p), ("w", ctypes.c_void_p), ("b", ctypes.c_void_p), ("y", ctypes.c_void_p),
                ("n", ctypes.c_int), ("c", ctypes.c_int), ("h", ctypes.c_int), ("width", ctypes.c_int)]


def _fields(pointers="", strides="", ints="", floats="", sizes=""):
    return ([(n, ctypes.c_void_p) for n in pointers.split()], [(n, ctypes.c_int64) for n in strides.split()],
            [(n, ctypes.c_int) for n in ints.split()], [(n, ctypes.c_float) for n in floats.split()],
            [(n, ctypes.c_size_t) for n in sizes.split()])


def _struct(name, doc, *groups):
    """A C struct of include/pla_b200.h: groups of fields in the header's order."""
    return type(name, (ctypes.Structure,), {"__doc__": doc, "_fields_": [f for g in groups for part in g for f in part]})


Causal = _struct("Causal", "pla_causal", _fields("x", "x_batch x_token"),
                 _fields("w b cu_seqlens state_in state_out y", "", "batch tokens channels taps sequences silu dtype"))
CausalGradient = _struct("CausalGradient", "pla_causal_gradient", _fields("dy", "dy_batch dy_token"),
                         _fields("dstate_out dx dw db dstate_in workspace", sizes="workspace_bytes"))
NormSide = _struct("NormSide", "pla_norm_side", _fields("x", "x_batch x_token x_head"),
                   _fields("w y dy", "dy_batch dy_token dy_head"), _fields("dw", "", "heads"))


class QkNorm(ctypes.Structure):
    """pla_qk_norm"""

    _fields_ = [("q", NormSide), ("k", NormSide), ("cos_table", ctypes.c_void_p), ("sin_table", ctypes.c_void_p),
                ("positions", ctypes.c_void_p), ("position_batch", ctypes.c_int64)] + [
                    (n, ctypes.c_int) for n in ("position_bytes", "table_rows", "batch", "tokens", "dim", "rot",
                                                "interleaved", "l2")] + [("eps", ctypes.c_float), ("dtype", ctypes.c_int)]


Delta = _struct("Delta", "pla_delta",
                _fields("q k v g beta", "q_batch q_token q_head k_batch k_token k_head v_batch v_token v_head "
                        "g_batch g_token g_head beta_batch beta_token beta_head"),
                _fields("cu_seqlens state_in state_out o", "", "batch tokens sequences hk hv dk dv gates32 dtype", "scale"),
                _fields("workspace", sizes="workspace_bytes"))
DeltaGradient = _struct("DeltaGradient", "pla_delta_gradient", _fields("d_o", "do_batch do_token do_head"),
                        _fields("dstate_out dstate_in dq dk dv dg dbeta"))
DeltaStep = _struct("DeltaStep", "pla_delta_step",
                    _fields("q k v g beta", "q_row q_head k_row k_head v_row v_head g_row g_head beta_row beta_head"),
                    _fields("state", "state_row"), _fields("o", "", "n hk hv dk dv gates32 dtype", "scale"))


_lib = None


class PlaError(RuntimeError):
    """A non-zero status from the C ABI (mirrors the reference's TORCH_CHECK -> RuntimeError)."""


def lib() -> ctypes.CDLL:
    """Load libpla_b200.so once; raise if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build the CUDA library first (python -m pla_b200.build); "
                "this package has no CPU fallback")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (argtypes, restype) in SIGNATURES.items():
            try:
                fn = getattr(handle, name)
            except AttributeError:
                raise ImportError(f"{LIB_PATH} does not export {name}: it is older than the package; "
                                  "rebuild it (python -m pla_b200.build)") from None
            fn.argtypes = argtypes
            fn.restype = restype
        _lib = handle
    return _lib


_ops = None


def ops():
    """``torch.ops.pla_b200``: the torch custom ops of libpla_b200_torch.so
    (csrc/torch_ops.cpp) over the C ABI, loaded once; raise if not built."""
    global _ops
    if _ops is None:
        lib()
        if not os.path.exists(TORCH_LIB_PATH):
            raise ImportError(f"{TORCH_LIB_PATH} is missing: build it first (python -m pla_b200.build)")
        torch.ops.load_library(TORCH_LIB_PATH)
        _ops = torch.ops.pla_b200
    return _ops


def check(status: int, what: str) -> None:
    if status != 0:
        L = lib()
        msg = L.pla_status_string(status).decode()
        detail = L.pla_last_cuda_error().decode()
        raise PlaError(f"{what}: {msg}" + (f" ({detail})" if detail and status == 4 else ""))


def check_faults(device=None) -> None:
    """Raise ``PlaError`` if a kernel on ``device`` (the current one if None) gave up a bounded wait (synchronises).

    Kernels that wait (for an asynchronous copy, for a neighbour's halo) do so
    for about two seconds at most, then record it and end; what they had to
    write is then incomplete.  The word stays set until
    ``pla_clear_device_faults``.
    """
    v = ctypes.c_uint(0)
    with contextlib.nullcontext() if device is None else torch.cuda.device(device):
        check(lib().pla_read_device_faults(ctypes.byref(v)), "pla_read_device_faults")
    if v.value:
        raise PlaError(f"device fault word {v.value:#x}: a bounded wait in a kernel timed out")


def stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def overlaps(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory spans of two CUDA tensors intersect.

    The single-step kernels read each input halo after other CTAs may have
    stored their outputs, so an output that overlaps its input would give
    wrong results; the ops reject it instead.
    """
    if a.numel() == 0 or b.numel() == 0 or a.device != b.device:
        return False

    def span(t):
        lo = hi = t.data_ptr()
        for size, stride in zip(t.shape, t.stride()):
            ext = (size - 1) * stride * t.element_size()
            if ext < 0:
                lo += ext
            else:
                hi += ext
        return lo, hi + t.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


class HostTaps:
    """A 7x7 filter (+ optional bias) copied to host fp32 memory for the *_taps entry points.

    Mirrors the reference's weight cache (data/depthwise_conv_7x7_cuda/
    model_cutlass_autotune_v6.py:507-513, keyed on the parameter's _version
    and storage): the device->host copy (a stream sync) happens only when the
    weight or bias tensor changed since the last call.
    """

    def __init__(self):
        self._key = None
        self.taps = (ctypes.c_float * 49)()
        self.bias = ctypes.c_float(0.0)
        self.has_bias = False

    @staticmethod
    def _tkey(t):
        return None if t is None else (t.data_ptr(), t._version, t.dtype, str(t.device))

    def update(self, weight: torch.Tensor, bias: torch.Tensor | None) -> "HostTaps":
        key = (self._tkey(weight), self._tkey(bias))
        if key != self._key:
            w = weight.detach().reshape(49).float().cpu()
            for k in range(49):
                self.taps[k] = float(w[k])
            self.has_bias = bias is not None
            if bias is not None:
                self.bias.value = float(bias.detach().reshape(-1)[0].float().cpu())
            self._key = key
        return self

    def args(self):
        return self.taps, (ctypes.byref(self.bias) if self.has_bias else None)
