"""ctypes binding of libtagi_b200.so (the sm_100a CUDA library).

There is no fallback: if the library is missing or cannot be loaded, importing
any compute function raises, and every call checks the returned status and
raises ``ValueError`` (bad arguments) or ``RuntimeError`` (CUDA errors) with
the library's message.
"""

from __future__ import annotations

import ctypes
import os
from pathlib import Path

import torch

LIB_PATH = Path(os.environ.get("TAGI_B200_LIB", Path(__file__).resolve().parent / "libtagi_b200.so"))

_P, _I, _F, _D, _N, _Z, _U = (ctypes.c_void_p, ctypes.c_int64, ctypes.c_float, ctypes.c_double,
                              ctypes.c_int, ctypes.c_size_t, ctypes.c_uint64)
_CODES = {"p": _P, "i": _I, "f": _F, "d": _D, "n": _N, "z": _Z, "u": _U}

# name -> argument codes (stream last, always 'p'); returns int status unless listed in _RET.
_SIGS = {
    "tagi_fused_var_forward": "pppppp" + "iii" + "iiiiii" + "p",
    "tagi_moment_forward": "pp" + "iiii" + "ppi" + "pppp" + "iiii" + "iii" + "p",
    "tagi_fused_backward_delta": "ppppp" + "iii" + "iiiiii" + "p",
    "tagi_backward_delta_view": "pp" + "iiii" + "pi" + "pp" + "iiii" + "iii" + "p",
    "tagi_conv2d_backward_delta": "ppp" + "pp" + "iiiiiiiii" + "nn" + "pz" + "p",
    "tagi_linear_forward": "pppppp" + "pp" + "iii" + "pz" + "p",
    "tagi_linear_backward_delta": "ppp" + "pp" + "iii" + "pz" + "p",
    "tagi_conv2d_forward": "pppppp" + "pp" + "iiiiiiiii" + "n" + "pz" + "p",
    "tagi_nchw_to_nhwc": "pppp" + "iii" + "p",
    "tagi_fused_weight_grad_workspace_size": "iii",
    "tagi_store_workspace_size": "iii",
    "tagi_fused_weight_grad": "ppppp" + "iii" + "iiiiii" + "pz" + "p",
    "tagi_fused_weight_grad_static": "ppppp" + "iii" + "iiiiii" + "p",
    "tagi_param_grad_workspace_size": "iiin",
    "tagi_param_grad": "pipp" + "iiii" + "iii" + "nn" + "pppp" + "pppp" + "f" + "pz" + "p",
    "tagi_param_grad_t": "pipp" + "iiii" + "iii" + "nn" + "pppp" + "pppp" + "f" + "pz" + "p",
    "tagi_param_grad_bias_given": "pin" + "pp" + "iiii" + "iii" + "pn" + "pppp" + "pppp" + "f"
                                  + "pz" + "p",
    "tagi_apply_param_sums": "pp" + "ii" + "n" + "pppp" + "f" + "p",
    "tagi_bmm_tagi_var": "pppppp" + "iiii" + "iiiiiiiii" + "ff" + "p",
    "tagi_bmm_shared_right": "ppppp" + "iiii" + "iiiiiiiii" + "f" + "p",
    "tagi_bmm_shared_left": "ppppp" + "iiii" + "iiiiiiiii" + "f" + "p",
    "tagi_capped_update": "pppp" + "i" + "f" + "p",
    "tagi_innovation": "ppppp" + "i" + "f" + "p",
    "tagi_relu_forward": "ppppp" + "i" + "p",
    "tagi_jacobian_backward": "ppppp" + "i" + "p",
    "tagi_remax_forward": "ppppp" + "iii" + "p",
    "tagi_add_inplace": "pppp" + "i" + "p",
    "tagi_embedding_forward": "ppppp" + "iiii" + "p",
    "tagi_embedding_backward": "pppp" + "iiii" + "n" + "pp" + "p",
    "tagi_positional_add": "ppp" + "iii" + "p",
    "tagi_avgpool_forward": "pppp" + "iiiii" + "f" + "p",
    "tagi_avgpool_backward": "pppp" + "iiiii" + "f" + "p",
    "tagi_im2col": "pppp" + "iiiiiiii" + "p",
    "tagi_im2col_t": "pp" + "iiiiiiii" + "p",
    "tagi_col2im": "pppp" + "iiiiiiii" + "n" + "p",
    "tagi_bn_channel_sums": "ppp" + "iii" + "p",
    "tagi_bn_finalize": "p" + "i" + "d" + "ppppp" + "nn" + "ff" + "p",
    "tagi_bn_forward": "pppppppppppp" + "iii" + "f" + "p",
    "tagi_bn_train_forward": "ppppppppppppp" + "pp" + "iii" + "nn" + "ff" + "p",
    "tagi_bn_sync_forward": "ppp" + "d" + "p" * 13 + "iii" + "nn" + "ff" + "p",
    "tagi_bn_backward": "ppppppp" + "ppp" + "iii" + "f" + "ppp" + "f" + "p",
    "tagi_bn_apply_grads": "p" + "i" + "n" + "pppppppp" + "f" + "p",
    "tagi_rmsnorm_forward": "ppppppp" + "ii" + "f" + "p",
    "tagi_rmsnorm_backward": "pppppppp" + "ii" + "p",
    "tagi_apply_vector_sums": "pp" + "i" + "n" + "pppp" + "f" + "p",
    "tagi_embedding_lookup": "pn" + "pppp" + "iiii" + "d" + "p",
    "tagi_embedding_grad_workspace_size": "ii",
    "tagi_embedding_grad": "pn" + "pp" + "iiii" + "d" + "n" + "pppp" + "f" + "pz" + "p",
    "tagi_add_rmsnorm_forward": "p" * 11 + "ii" + "f" + "p",
    "tagi_add_rmsnorm_int8": "p" * 12 + "iii" + "f" + "p",
    "tagi_quantize_moments": "ppn" + "pppp" + "iii" + "p",
    "tagi_int8_values": "pppp" + "i" + "ppp" + "ii" + "p",
    "tagi_add_rmsnorm_backward_workspace_size": "ii",
    "tagi_add_rmsnorm_backward": "p" * 8 + "n" + "ppppp" + "f" + "ii" + "pz" + "p",
    "tagi_int8_moment_matmul": "ppppi" + "ppppi" + "pppp" + "iii" + "p",
    "tagi_version": "",
    "tagi_device_arch": "n",
    "tagi_last_error": "",
    "tagi_kernel_launches": "",
    "tagi_tma_launches": "",
    "tagi_tc_launches": "",
    "tagi_device_status": "n",
    "tagi_set_wait_limit_ns": "u",
    "tagi_peer_buffer_bytes": "ni",
    "tagi_peer_buffer_create": "zpp",
    "tagi_peer_buffer_open": "pp",
    "tagi_peer_buffer_close": "pn",
    "tagi_peer_allreduce_f64": "pipnnip" + "p",
    "tagi_peer_status": "n",
}
_RET = {
    "tagi_peer_buffer_bytes": _Z,
    "tagi_fused_weight_grad_workspace_size": _Z,
    "tagi_param_grad_workspace_size": _Z,
    "tagi_store_workspace_size": _Z,
    "tagi_embedding_grad_workspace_size": _Z,
    "tagi_add_rmsnorm_backward_workspace_size": _Z,
    "tagi_last_error": ctypes.c_char_p,
    "tagi_kernel_launches": ctypes.c_uint64,
    "tagi_tma_launches": ctypes.c_uint64,
    "tagi_tc_launches": ctypes.c_uint64,
}

# Status codes (include/tagi_b200.h)
TAGI_OK, TAGI_E_BAD_ARG, TAGI_E_ALIGNMENT = 0, -1, -2
WGRAD_SUMS, WGRAD_DELTAS, WGRAD_UPDATE = 0, 1, 2


class _Lib:
    def __init__(self, path: Path):
        if not path.exists():
            raise ImportError(
                f"libtagi_b200.so not found at {path}; build it with "
                "`python triton-tagi_b200/build_lib.py` (nvcc, sm_100a)")
        self.path = path
        self.dll = ctypes.CDLL(str(path))
        self.fn = {}
        for name, codes in _SIGS.items():
            f = getattr(self.dll, name)
            f.argtypes = [_CODES[c] for c in codes]
            f.restype = _RET.get(name, ctypes.c_int)
            self.fn[name] = f

    hook = None  # optional callable(phase, name, args) used by the benchmark to time launches

    def __call__(self, name: str, *args):
        h = self.hook
        if h is not None:
            h("before", name, args)
        rc = self.fn[name](*args)
        if h is not None:
            h("after", name, args)
        if rc != 0:
            self.fail(name, rc)

    def fail(self, name: str, rc: int):
        msg = self.fn["tagi_last_error"]().decode(errors="replace")
        if rc in (TAGI_E_BAD_ARG, TAGI_E_ALIGNMENT):
            raise ValueError(msg)
        raise RuntimeError(f"{name} failed ({rc}): {msg}")

    def size(self, name: str, *args) -> int:
        return int(self.fn[name](*args))


_instance: _Lib | None = None


def lib() -> _Lib:
    global _instance
    if _instance is None:
        _instance = _Lib(LIB_PATH)
    return _instance


def device_status(reset: bool = False) -> int:
    """0, or the code of a tensor-core kernel wait that timed out (synchronises)."""
    return int(lib().fn["tagi_device_status"](1 if reset else 0))


def check_device_status() -> None:
    """Raise RuntimeError if a tensor-core kernel wait or a peer exchange wait ran
    out since the last check (outputs are then incomplete); clears the words."""
    code = device_status(reset=True)
    if code != 0:
        raise RuntimeError(f"a tensor-core kernel gave up a tile (bounded wait {code} ran out); "
                           "its outputs are incomplete")
    if int(lib().fn["tagi_peer_status"](1)) != 0:
        raise RuntimeError("a peer-memory exchange wait ran out (a rank stopped?); the "
                           "statistics it carried were not reduced")


def set_wait_limit_ns(ns: int) -> None:
    """Limit of the tensor-core kernels' abortable waits (0 restores 2 s); a test hook."""
    rc = lib().fn["tagi_set_wait_limit_ns"](int(ns))
    if rc != 0:
        raise RuntimeError(lib().fn["tagi_last_error"]().decode(errors="replace"))


def kernel_launches() -> int:
    """Kernels launched by libtagi_b200 so far in this process."""
    return int(lib().fn["tagi_kernel_launches"]())


def tc_launches() -> int:
    """Of those, launches of the tcgen05 tensor-core contraction kernel."""
    return int(lib().fn["tagi_tc_launches"]())


def stream(t: torch.Tensor) -> int:
    """Raw cudaStream_t of the current torch stream on ``t``'s device."""
    return torch.cuda.current_stream(t.device).cuda_stream


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def check_cuda_f32(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError("triton_tagi (B200) tensors must live on a CUDA device")
        if t.dtype != torch.float32:
            raise ValueError(f"expected float32 tensor, got {t.dtype}")


def check_f32(*ts: torch.Tensor | None) -> int:
    """Checks that the tensors (None: absent) are float32 on one CUDA device and
    returns its index."""
    dev = None
    for t in ts:
        if t is None:
            continue
        d = t.get_device()
        if t.dtype is not torch.float32:
            raise ValueError(f"expected float32 tensor, got {t.dtype}")
        if d != dev:
            if d < 0:  # the CPU's
                raise ValueError("triton_tagi (B200) tensors must live on a CUDA device")
            if dev is not None:
                raise ValueError(f"tensors live on different devices (cuda:{dev} and cuda:{d})")
            dev = d
    return dev


def check_on(dev: int, *ts: torch.Tensor | None) -> None:
    """Checks that the tensors live on CUDA device ``dev``."""
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors live on different devices (cuda:{dev} and {t.device})"
                             if t.is_cuda else
                             "triton_tagi (B200) tensors must live on a CUDA device")


_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
try:  # torch's shortest way to an uninitialised tensor: 0.8 us, where empty_like takes 1.3
    # and new_empty 1.8, in calls that take 10 to 20 us altogether
    from torch._C._dynamo.guards import _empty_strided_cuda as _fast_empty
except ImportError:
    _fast_empty = None


def call_on(dev: int, name: str, *args) -> None:
    """``lib()(name, *args, stream)`` with device ``dev`` current and its current
    stream: a kernel belongs to the device that is current when it is launched."""
    L = _instance or lib()
    if dev != _current_device():
        with torch.cuda.device(dev):
            L(name, *args, _raw_stream(dev))
    elif L.hook is not None:
        L(name, *args, _raw_stream(dev))
    else:  # L(...) without its detours
        rc = L.fn[name](*args, _raw_stream(dev))
        if rc != 0:
            L.fail(name, rc)


def allocator(dev: int):
    """``new(size, stride, dtype)``: uninitialised tensors on CUDA device ``dev``; size and
    stride are tuples of integers."""
    if _fast_empty is not None and dev == _current_device():
        return _fast_empty
    device = torch.device("cuda", dev)
    return lambda size, stride, dtype: torch.empty_strided(size, stride, dtype=dtype,
                                                           device=device)


def workspace(nbytes: int, like: torch.Tensor) -> tuple[torch.Tensor | None, int | None, int]:
    """Scratch buffer for one call: returns (holder, pointer, bytes).

    The holder only has to live until the call has been enqueued: torch's
    caching allocator hands a freed block only to later work on the same
    stream, which runs after the kernels that used it."""
    if nbytes == 0:
        return None, None, 0
    buf = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    return buf, buf.data_ptr(), nbytes
