"""ctypes binding of ``libtcq_b200.so`` (the C ABI declared in ``include/tcq_b200.h``).

The library is built in-tree by ``csrc/Makefile`` (see ``build()``).  There is no
fallback: if the shared object is missing or cannot be loaded, importing the
codec fails with an error that says how to build it.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
import subprocess
import sys
import warnings

_CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc")
LIB_PATH = os.path.join(_CSRC, "libtcq_b200.so")
SHORT_PATH = os.path.join(_CSRC, "tcq_torch.so")

ABI_VERSION = 7

# name -> (restype, argtypes); mirrors include/tcq_b200.h one to one
_vp, _i64, _int, _sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
SIGNATURES = {
    "tcq_abi_version": (_int, []),
    "tcq_strerror": (ctypes.c_char_p, [_int]),
    "tcq_last_cuda_error": (ctypes.c_char_p, []),
    "tcq_workspace_bytes": (_sz, [_i64, _int]),
    "tcq_workspace_min_bytes": (_sz, [_int]),
    "tcq_encode_tb": (_int, [_vp, _i64, _int, _int, _vp, _vp, _vp, _vp, _vp, _sz, _vp]),
    "tcq_encode_tb_static_max_tiles": (_i64, [_int]),
    "tcq_encode_tb_static": (_int, [_vp, _i64, _int, _int, _vp, _vp, _vp, _vp, _vp]),
    "tcq_encode_tb_static_status": (_int, [_vp]),
    "tcq_encode_tb_rows": (_int, [_vp, _vp, _i64, _i64, _int, _int, _vp, _i64, _vp, _vp, _vp, _vp, _sz, _vp]),
    "tcq_viterbi_pass": (_int, [_vp, _i64, _int, _int, _vp, _int, _vp, _vp, _sz, _vp]),
    "tcq_forward_pass": (_int, [_vp, _i64, _int, _int, _vp, _int, _int, _vp, _sz, _vp]),
    "tcq_workspace_status": (_int, [_vp, _sz, _i64, _int, _vp]),
    "tcq_selftest_wait_timeout": (_int, [_vp, _i64, _int, _vp, _sz, _vp]),
    "tcq_selftest_walk_waits": (_int, [_vp, _i64, _int, _vp, _vp, _sz, _vp]),
    "tcq_encode_launches": (_i64, [_i64, _int, _sz]),
    "tcq_decode_packed": (_int, [_vp, _i64, _int, _int, _vp, _vp]),
    "tcq_decode_matvec": (_int, [_vp, _i64, _i64, _int, _int, _vp, _i64, _int, _vp, _i64, _vp]),
    "tcq_decode_symbols": (_int, [_vp, _i64, _i64, _int, _int, _vp, _vp, _vp]),
    "tcq_pack_symbols": (_int, [_vp, _i64, _int, _vp, _vp]),
    "tcq_codebook_lut": (_int, [_int, _vp, _vp]),
    "tcq_ip_workspace_bytes": (_sz, [_i64, _i64]),
    "tcq_ip_forward": (_int, [_vp, _i64, _i64, _vp, _vp, ctypes.c_float, _int, _vp, _vp, _vp, _vp, _vp, _sz, _vp]),
    "tcq_ip_restore": (_int, [_vp, _int, _i64, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp]),
    "tcq_ms_code_pitch": (_sz, [_i64]),
    "tcq_ms_scale_bytes": (_sz, [_i64, _i64, _int]),
    "tcq_ms_quantize": (_int, [_vp, _int, _i64, _i64, _i64, _int, _int, _vp, _vp, _vp, _vp, _vp]),
    "tcq_ms_dequantize": (_int, [_vp, _vp, _vp, _i64, _i64, _int, _vp, _int, _i64, _vp]),
    "tcq_ms_linear_workspace_bytes": (_sz, [_i64, _i64, _i64, _int, _int]),
    "tcq_ms_linear": (_int, [_vp, _int, _i64, _i64, _vp, _vp, _vp, _i64, _i64, _int, _vp, _i64, _vp, _sz, _vp]),
    "tcq_ms_matmul": (_int, [_vp, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _int, _vp, _int, _i64, _vp]),
    "tcq_selftest_ms_linear_waits": (_int, [_i64, _vp, _int, _i64, _i64, _vp, _vp, _vp, _i64, _i64, _int, _vp, _i64, _vp, _sz, _vp]),
    "tcq_selftest_ms_matmul_waits": (_int, [_i64, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _i64, _i64, _int, _vp, _int, _i64, _vp]),
    "tcq_ms_grouped_linear_workspace_bytes": (_sz, [_i64, _i64, _i64, _i64, _int, _int, _int]),
    "tcq_ms_grouped_linear": (_int, [_vp, _int, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _i64, _i64, _int, _vp, _int, _int, _vp, _i64, _vp, _int, _i64,
                                     _vp, _sz, _vp]),
    "tcq_ms_epilogue": (_int, [_vp, _i64, _i64, _vp, _int, _int, _vp, _i64, _vp, _int, _i64, _vp]),
    "tcq_route_workspace_bytes": (_sz, [_i64, _i64]),
    "tcq_route": (_int, [_vp, _int, _i64, _i64, _i64, _i64, _int, _int, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp]),
    "tcq_combine": (_int, [_vp, _int, _i64, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _i64, _vp, _int, _i64, _vp]),
    "tcq_selftest_ms_grouped_waits": (_int, [_i64, _vp, _int, _i64, _i64, _vp, _vp, _i64, _i64, _vp, _vp, _vp, _i64, _i64, _int, _vp, _int, _int, _vp, _i64, _vp, _int,
                                             _i64, _vp, _sz, _vp]),
}

_lib = None


class TcqError(RuntimeError):
    """A C-ABI call returned a negative status."""


def build(verbose: bool = False, jobs: int = 8) -> str:
    """Compile the CUDA sources for sm_100a with nvcc (``make`` in ``csrc/``)."""
    out = None if verbose else subprocess.DEVNULL
    subprocess.check_call(["make", "-C", _CSRC, f"-j{jobs}", "libtcq_b200.so"], stdout=out)
    try:
        subprocess.check_call(["make", "-C", _CSRC, "tcq_torch.so", f"PYTHON={sys.executable}"], stdout=out)
    except subprocess.CalledProcessError as e:               # (a torch without its headers or CUDA libraries: all calls work without it)
        warnings.warn(f"tcq_torch.so was not built ({e}): small calls go through ctypes and take twice the host's time", RuntimeWarning, stacklevel=2)
    return LIB_PATH


def lib() -> ctypes.CDLL:
    """The loaded library, with argument types set.  Raises if it was not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} not found: the CUDA extension is not built. "
                "Run `python -c 'import __graft_entry__ as g; g.build()'` or `make -C <package>/csrc`. "
                "There is no CPU fallback.")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)       # AttributeError here = a declared symbol is not exported
            fn.restype = res
            fn.argtypes = args
        got = handle.tcq_abi_version()
        if got != ABI_VERSION:
            raise ImportError(f"libtcq_b200.so has ABI version {got}, this package needs {ABI_VERSION}: rebuild it")
        _lib = handle
    return _lib


_short = None
SHORT_BINDS = ("tcq_ms_grouped_linear_workspace_bytes", "tcq_ms_grouped_linear", "tcq_route_workspace_bytes", "tcq_route", "tcq_combine", "tcq_ms_linear_workspace_bytes", "tcq_ms_linear",
               "tcq_ms_epilogue")


def short():
    """The extension that takes the small calls where all is well (``csrc/tcq_torch.cpp``), bound to the library; False where it was not built, or (with a warning, once) was built for
    another library, torch or Python: the same calls then go through ctypes, which takes twice as long."""
    global _short
    if _short is None:
        handle, _short = lib(), False
        if os.path.exists(SHORT_PATH):
            try:
                _short = _load_short(handle)
            except ImportError as e:
                warnings.warn(f"{SHORT_PATH} is not used, small calls go through ctypes: {e} (build it anew)", RuntimeWarning, stacklevel=2)
    return _short


def _load_short(handle: ctypes.CDLL):
    import torch
    loader = importlib.machinery.ExtensionFileLoader("tcq_torch", SHORT_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("tcq_torch", SHORT_PATH, loader=loader))
    loader.exec_module(module)
    here = (ABI_VERSION, torch.__version__.split("+")[0], sys.hexversion >> 16)
    if getattr(module, "built_for", None) != here:
        raise ImportError(f"it was built for {getattr(module, 'built_for', 'an unknown version')}, this is {here}")
    module.bind(*(ctypes.cast(getattr(handle, name), ctypes.c_void_p).value for name in SHORT_BINDS))
    return module


def check(code: int, what: str) -> None:
    """Turn a negative status into an exception (ValueError for bad arguments)."""
    if code == 0:
        return
    L = lib()
    msg = L.tcq_strerror(code).decode()
    if code == -7:
        raise TcqError(f"{what}: {msg}: {L.tcq_last_cuda_error().decode()}")
    if code in (-6, -10, -11):
        raise TcqError(f"{what}: {msg}")
    raise ValueError(f"{what}: {msg}")
