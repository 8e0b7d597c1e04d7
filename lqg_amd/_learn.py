"""ctypes mirror of include/lqg_learn.h: the learned-filter operators (lqg_amd.belief.ssm) and the AdamW step (lqg_amd.optim)."""
import ctypes as C

import torch

from lqg_amd import _abi
from lqg_amd._abi import LqgHipError

T_F32, T_BF16, T_F16, T_F64 = range(4)
TYPES = {torch.float32: T_F32, torch.bfloat16: T_BF16, torch.float16: T_F16, torch.float64: T_F64}
SEQ_TYPES = (torch.float32, torch.bfloat16, torch.float16)


class Seq(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("sb", C.c_int64), ("st", C.c_int64), ("sg", C.c_int64)]


class Param(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("type", C.c_int32), ("pad", C.c_int32)]


class Conv(C.Structure):
    _fields_ = [("type", C.c_int32), ("W", C.c_int32), ("silu", C.c_int32), ("pad", C.c_int32), ("B", C.c_int64), ("T", C.c_int64),
                ("D", C.c_int64), ("x", Seq), ("y", Seq), ("w", Param), ("bias", Param), ("state", C.c_void_p),
                ("state_out", C.c_void_p), ("lengths", C.c_void_p)]


class SelScan(C.Structure):
    _fields_ = [("type", C.c_int32), ("softplus", C.c_int32), ("B", C.c_int64), ("T", C.c_int64), ("D", C.c_int64), ("N", C.c_int64),
                ("G", C.c_int64), ("u", Seq), ("delta", Seq), ("z", Seq), ("Bm", Seq), ("Cm", Seq), ("y", Seq), ("A", Param),
                ("Dskip", Param), ("delta_bias", Param), ("state", C.c_void_p), ("state_out", C.c_void_p), ("lengths", C.c_void_p),
                ("checkpoints", C.c_void_p), ("chunks", C.c_int32), ("channels", C.c_int32)]


class SelScanBars(C.Structure):
    _fields_ = [("dy", Seq), ("dstate_out", C.c_void_p), ("du", C.c_void_p), ("ddelta", C.c_void_p), ("dz", C.c_void_p),
                ("dBm", C.c_void_p), ("dCm", C.c_void_p), ("dA", C.c_void_p), ("dD", C.c_void_p), ("ddelta_bias", C.c_void_p),
                ("dstate", C.c_void_p)]


class AdamW(C.Structure):
    _fields_ = [("type", C.c_int32), ("bits", C.c_int32), ("count", C.c_int32), ("pad", C.c_int32), ("params", C.c_void_p),
                ("grads", C.c_void_p), ("numel", C.c_void_p), ("offset", C.c_void_p), ("exp_avg", C.c_void_p),
                ("exp_avg_sq", C.c_void_p), ("exp_avg_scale", C.c_void_p), ("exp_avg_sq_scale", C.c_void_p), ("lr", C.c_double),
                ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("weight_decay", C.c_double), ("step", C.c_int64),
                ("step_state", C.c_void_p)]


_lib = None


def load():
    """liblqg_hip.so with the entry points of include/lqg_learn.h declared."""
    global _lib
    if _lib is None:
        lib = _abi.load()
        if not hasattr(lib, "lqg_selective_scan"):
            raise LqgHipError(f"{_abi.LIB_PATH} holds no learned-filter operators: build it again "
                              "(python -c 'import __graft_entry__ as g; g.build()')")
        V, Z, I = C.c_void_p, C.c_size_t, C.c_int
        for name, args, res in (
                ("causal_conv", [C.POINTER(Conv), V], I),
                ("causal_conv_grad_workspace", [C.POINTER(Conv)], Z),
                ("causal_conv_grad", [C.POINTER(Conv), Seq, V, V, V, V, V, V, Z, V], I),
                ("causal_conv_step", [C.POINTER(Conv), V], I),
                ("selscan_workspace", [C.POINTER(SelScan)], Z),
                ("selscan_checkpoint_bytes", [C.POINTER(SelScan)], Z),
                ("selscan_grad_workspace", [C.POINTER(SelScan)], Z),
                ("selective_scan", [C.POINTER(SelScan), V, Z, V], I),
                ("selective_scan_grad", [C.POINTER(SelScan), C.POINTER(SelScanBars), V, Z, V], I),
                ("selective_scan_step", [C.POINTER(SelScan), V, V], I),
                ("adamw_step", [C.POINTER(AdamW), V], I),
                ("adamw_advance", [V, C.c_double, C.c_double, V], I)):
            fn = getattr(lib, "lqg_" + name)
            fn.argtypes, fn.restype = args, res
        _lib = lib
    return _lib


def stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def on_device(device):
    """`with` block in which `device` is the current one; free when it already is."""
    return torch.cuda.device(device)


def ptr(t):
    return None if t is None else t.data_ptr()


def seq(t):
    """[B, T, D] or [B, T, G, N] (channel stride 1) -> its view."""
    return Seq(None, 0, 0, 0) if t is None else Seq(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2) if t.dim() == 4 else 0)


def row(t):
    """[B, D] or [B, G, N]: one step -> its view."""
    return Seq(None, 0, 0, 0) if t is None else Seq(t.data_ptr(), t.stride(0), 0, t.stride(1) if t.dim() == 3 else 0)


def param(t):
    return Param(None, 0, 0) if t is None else Param(t.data_ptr(), TYPES[t.dtype], 0)


def scratch(nbytes, device):
    return torch.empty(int(nbytes), dtype=torch.uint8, device=device) if nbytes else None
