"""ctypes binding of the language-model operators (`libtrainkernel_ops.so`, `include/trainkernel_ops.h`).

The library holds hand-written sm_100a kernels that stand beside the generated step kernels: token
log-probabilities and the losses built on them (`losses.py`) and the AdamW update (`optim.py`).  Like
the rest of the package it has no CPU or eager fallback: a missing library is built with nvcc, and
tensors that are not on an sm_100 device raise.  No counterpart in the reference.
"""
from __future__ import annotations

import ctypes
import importlib.util
import subprocess
import sysconfig
import threading
import warnings
from pathlib import Path

import torch

from . import runtime

LIBRARY_PATH = runtime.PACKAGE_DIR / "libtrainkernel_ops.so"
SOURCES = ("tk_token_rows.cu", "tk_adamw.cu", "tk_ops_host.cpp")
HEADERS = ("tk_ops_host.h",)
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}

HOST_PATH = runtime.PACKAGE_DIR / "_ops_host.so"

_lock = threading.RLock()
_library: ctypes.CDLL | None = None
_host = None


class TokenArray(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_batch", ctypes.c_int64), ("stride_token", ctypes.c_int64)]


class TokenRows(ctypes.Structure):
    _fields_ = [("logits", ctypes.c_void_p), ("stride_batch", ctypes.c_int64), ("stride_token", ctypes.c_int64),
                ("batch", ctypes.c_int64), ("length", ctypes.c_int64), ("vocab", ctypes.c_int64),
                ("dtype", ctypes.c_int32), ("target_bytes", ctypes.c_int32), ("targets", TokenArray), ("mask", TokenArray)]


class TokenGrad(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride_batch", ctypes.c_int64), ("stride_token", ctypes.c_int64), ("scale_at", ctypes.c_void_p), ("scale", ctypes.c_float), ("reserved", ctypes.c_int32)]


class PolicyTerms(ctypes.Structure):
    _fields_ = [("old_logprobs", TokenArray), ("advantages", TokenArray), ("ref_logprobs", TokenArray),
                ("clip_low", ctypes.c_float), ("clip_high", ctypes.c_float), ("kl_weight", ctypes.c_float), ("average", ctypes.c_int32)]


class AdamWTensor(ctypes.Structure):
    _fields_ = [("param", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("offset", ctypes.c_int64), ("count", ctypes.c_int64),
                ("weight_decay", ctypes.c_float), ("reserved", ctypes.c_int32)]


class AdamWState(ctypes.Structure):
    _fields_ = [("mean", ctypes.c_void_p), ("square", ctypes.c_void_p), ("mean_scale", ctypes.c_void_p),
                ("root_scale", ctypes.c_void_p), ("steps", ctypes.c_void_p)]


class AdamWOptions(ctypes.Structure):
    _fields_ = [("lr_at", ctypes.c_void_p), ("scale_at", ctypes.c_void_p), ("lr", ctypes.c_double), ("beta1", ctypes.c_double),
                ("beta2", ctypes.c_double), ("eps", ctypes.c_double), ("seed", ctypes.c_uint32), ("bits", ctypes.c_int32)]


def build_library(force: bool = False) -> Path:
    """nvcc-compile the operators for sm_100a into a shared library next to the runtime shim."""
    sources = [runtime.CSRC_DIR / name for name in SOURCES]
    watched = [*sources, *(runtime.CSRC_DIR / name for name in HEADERS), runtime.INCLUDE_DIR / "trainkernel_ops.h"]
    if not force and LIBRARY_PATH.exists() and LIBRARY_PATH.stat().st_mtime >= max(p.stat().st_mtime for p in watched):
        return LIBRARY_PATH
    cuda = runtime._cuda_home()
    if cuda is None:
        raise RuntimeError("trainkernel: CUDA toolkit with nvcc is required to build libtrainkernel_ops.so")
    command = [str(Path(cuda) / "bin" / "nvcc"), "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
               "--threads", "0", "-shared", "-Xcompiler", "-fPIC", "-I", str(runtime.INCLUDE_DIR), "-o", str(LIBRARY_PATH), *map(str, sources)]
    done = subprocess.run(command, capture_output=True, text=True)
    if done.returncode != 0:
        raise RuntimeError(f"trainkernel: building libtrainkernel_ops.so failed:\n{done.stderr[-4000:]}")
    return LIBRARY_PATH


def build_host(force: bool = False) -> Path:
    """Compile `csrc/tk_ops_host_path.cpp`, the short way from a Python call to a launch, against PyTorch's headers."""
    source = runtime.CSRC_DIR / "tk_ops_host_path.cpp"
    library_path = build_library()
    watched = (source, runtime.INCLUDE_DIR / "trainkernel_ops.h")
    if not force and HOST_PATH.exists() and HOST_PATH.stat().st_mtime >= max(p.stat().st_mtime for p in watched):
        return HOST_PATH
    cuda = runtime._cuda_home()
    if cuda is None:
        raise RuntimeError("trainkernel: CUDA toolkit headers are required to build the operators' host path")
    torch_dir = Path(torch.__file__).resolve().parent
    include = [runtime.INCLUDE_DIR, torch_dir / "include", torch_dir / "include" / "torch" / "csrc" / "api" / "include", Path(cuda) / "include",
               sysconfig.get_paths()["include"]]
    command = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
               *(f"-I{path}" for path in include), "-o", str(HOST_PATH), str(source), f"-L{torch_dir / 'lib'}", f"-L{library_path.parent}",
               "-ltrainkernel_ops", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda", "-Wl,-rpath,$ORIGIN"]
    done = subprocess.run(command, capture_output=True, text=True)
    if done.returncode != 0:
        raise RuntimeError(f"trainkernel: building the operators' host path failed:\n{done.stderr[-4000:]}")
    return HOST_PATH


def host():
    """The compiled host path (its calls return None for anything out of the ordinary)."""
    global _host
    with _lock:
        if _host is None:
            library()                           # resident first: the host path links against it
            spec = importlib.util.spec_from_file_location("_ops_host", build_host())
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
            _host = module
        return _host


def host_or_none():
    """The host path, or None with a warning where it cannot be had: it saves microseconds a call, and every operator runs without it."""
    try:
        return host()
    except (RuntimeError, OSError, ImportError) as error:
        warnings.warn(f"trainkernel: the operators run without their compiled host path: {error}", RuntimeWarning, stacklevel=3)
        return None


def library() -> ctypes.CDLL:
    """The loaded operator library with argument types declared; built on first use if missing."""
    global _library
    with _lock:
        if _library is not None:
            return _library
        lib = ctypes.CDLL(str(build_library()))
        p, i32, i64, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float
        rows, grad, array = ctypes.POINTER(TokenRows), ctypes.POINTER(TokenGrad), ctypes.POINTER(TokenArray)
        lib.tk_ops_last_error.restype = ctypes.c_char_p
        lib.tk_ops_launch_count.restype = ctypes.c_uint64
        lib.tk_token_logprobs.argtypes = [rows, p, p, i32, p]
        lib.tk_token_logprobs_and_grad.argtypes = [rows, array, p, grad, i32, p]
        lib.tk_token_logits_grad.argtypes = [rows, array, p, grad, i32, p]
        lib.tk_policy_workspace_bytes.argtypes = [i64, i64]
        lib.tk_policy_workspace_bytes.restype = ctypes.c_size_t
        lib.tk_policy_loss.argtypes = [rows, ctypes.POINTER(PolicyTerms), p, p, p, p, grad, p, i32, p]
        lib.tk_preference_workspace_bytes.argtypes = [i64, i64]
        lib.tk_preference_workspace_bytes.restype = ctypes.c_size_t
        lib.tk_preference_loss.argtypes = [rows, p, i64, f32, f32, p, p, p, p, grad, p, i32, p]
        lib.tk_adamw_update.argtypes = [ctypes.POINTER(AdamWTensor), i32, i32, i32, ctypes.POINTER(AdamWState), ctypes.POINTER(AdamWOptions), i32, i32, p]
        _library = lib
        return lib


def check(code: int) -> None:
    if code:
        raise RuntimeError(library().tk_ops_last_error().decode() or f"trainkernel: operator library error {code}")


_usable: dict[int, bool] = {}
fast = None             # the host path, once a device has been found usable


def require_device(device: torch.device) -> int:
    """The ordinal of an sm_100 CUDA device; raises for anything else, as `compile_program` does."""
    if device.type != "cuda":
        raise RuntimeError("trainkernel: CUDA sm_100a GPU required; this operator has no CPU form")
    global fast
    index = device.index if device.index is not None else torch.cuda.current_device()
    if index not in _usable:
        capability = torch.cuda.get_device_capability(index)
        _usable[index] = capability[0] == 10
        if _usable[index] and (path := host_or_none()) is not None:
            path.allow_device(index)
            fast = path
    if not _usable[index]:
        raise RuntimeError("trainkernel: an sm_100 (B200-class) GPU is required")
    return index
