"""ctypes bindings of libartemis_synth.so (the C ABI declared in include/artemis_synth.h) and of
libartemis_ops.so (include/artemis_ops.h: the encoder's operators and the optimizer step).

The library is the product: if it is missing or does not load, every op raises -- there is no
CPU or eager-PyTorch fallback (the reference has none either: cupy_module/synth.py:310-311).
"""
from __future__ import annotations

import ctypes
import os

from . import build as _build

_lib = None
_ops = None
_ops_host = None

ABI_VERSION = 1
RADIUS_DEFAULT = -1
RADIUS_NONE = 0
RADIUS_AUTO = -2
RADIUS_SMALL = -3
GIN_ATOMIC = 0
GIN_DETERMINISTIC = 1
FRAME_F32 = 0
FRAME_BF16 = 1

_vp = ctypes.c_void_p
_i = ctypes.c_int

# name -> (restype, argtypes); one entry per declaration in include/artemis_synth.h
SIGNATURES = {
    "artemis_synth_forward": (_i, [_vp] * 5 + [_i] * 7 + [_vp]),
    "artemis_synth_backward": (_i, [_vp] * 9 + [_i] * 8 + [_vp, ctypes.c_size_t, _vp]),
    "artemis_synth_backward_workspace_bytes": (ctypes.c_size_t, [_i] * 7),
    "artemis_synth_forward_ex": (_i, [_vp] * 5 + [_i] * 12 + [_vp]),
    "artemis_synth_backward_ex": (_i, [_vp] * 9 + [_i] * 13 + [_vp, ctypes.c_size_t, _vp]),
    "artemis_synth_backward_workspace_bytes_ex": (ctypes.c_size_t, [_i] * 9),
    "artemis_synth_backward_noalloc": (_i, [_vp] * 9 + [_i] * 13 + [_vp]),
    "artemis_synth_head_forward": (_i, [_vp, _i] + [_vp] * 5 + [_i] * 9 + [_vp]),
    "artemis_synth_head_backward": (_i, [_vp, _i] + [_vp] * 9 + [_i] * 9 + [_vp]),
    "artemis_synth_offset_radius": (_i, [_vp, _vp, ctypes.c_size_t, _vp, _vp]),
    "artemis_synth_set_small_grid_tiles": (ctypes.c_longlong, [ctypes.c_longlong]),
    "artemis_synth_auto_query": (_i, [_i, _i, _i, _vp, _vp, _vp, _vp]),
    "artemis_synth_auto_reset": (None, []),
    "artemis_synth_set_gin_gather": (_i, [_i]),
    "artemis_synth_version": (ctypes.c_char_p, []),
    "artemis_synth_last_error": (ctypes.c_char_p, []),
}


OPS_ABI_VERSION = 1
OPS_F32 = 0
OPS_BF16 = 1
OPS_F16 = 2


class WindowDesc(ctypes.Structure):
    """artemis_ops_window"""
    _fields_ = [(n, _i) for n in ("B", "D", "H", "W", "heads", "head_dim", "wd", "wh", "ww", "shift_d", "shift_h",
                                  "shift_w", "label_maps", "dtype")] + [("scale", ctypes.c_float),
                                                                       ("outside", ctypes.c_float)]


class TensorDesc(ctypes.Structure):
    """artemis_ops_tensor"""
    _fields_ = [(n, _vp) for n in ("param", "grad", "m", "v", "m_base", "v_base")] + [("count", ctypes.c_longlong)]


_ll, _d, _sz = ctypes.c_longlong, ctypes.c_double, ctypes.c_size_t
_win = ctypes.POINTER(WindowDesc)

# name -> (restype, argtypes); one entry per declaration in include/artemis_ops.h
OPS_SIGNATURES = {
    "artemis_ops_layer_norm_forward": (_i, [_vp] * 6 + [_ll, _ll, ctypes.c_float, _i, _vp]),
    "artemis_ops_layer_norm_backward": (_i, [_vp] * 8 + [_ll, _ll, _i, _vp, _sz, _vp]),
    "artemis_ops_layer_norm_workspace_bytes": (_sz, [_ll, _ll, _i]),
    "artemis_ops_window_attention_lse_count": (_sz, [_win]),
    "artemis_ops_window_attention_workspace_bytes": (_sz, [_win, _i, _i]),
    "artemis_ops_window_attention_forward": (_i, [_win] + [_vp] * 6 + [_sz, _vp]),
    "artemis_ops_window_attention_backward": (_i, [_win] + [_vp] * 9 + [_sz, _vp]),
    "artemis_ops_adamw": (_i, [_vp, _i, _i, _i, _d, _d, _d, _d, _d, _ll, ctypes.c_uint, _vp]),
    "artemis_ops_moments_from_8bit": (_i, [_vp, _i, _i, _vp]),
    "artemis_ops_version": (ctypes.c_char_p, []),
    "artemis_ops_last_error": (ctypes.c_char_p, []),
}


class SynthLibraryError(RuntimeError):
    pass


def lib_path() -> str:
    return os.environ.get("ARTEMIS_SYNTH_LIB", _build.LIB_PATH)


def _open(path, signatures):
    if not os.path.exists(path):
        raise SynthLibraryError(
            f"{path} not found: build it with `python -m artemis_amd.build` "
            "(hipcc --offload-arch=gfx950). There is no fallback path.")
    try:
        lib = ctypes.CDLL(path)
    except OSError as e:  # e.g. libamdhip64 missing
        raise SynthLibraryError(f"cannot load {path}: {e}") from e
    for name, (res, args) in signatures.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


def load():
    """Load the shared library once per process; raise loudly when it is absent."""
    global _lib
    if _lib is None:
        _lib = _open(lib_path(), SIGNATURES)
    return _lib


def load_ops():
    """Load libartemis_ops.so once per process; raise loudly when it is absent."""
    global _ops
    if _ops is None:
        _ops = _open(_build.OPS_LIB_PATH, OPS_SIGNATURES)
    return _ops


def load_ops_host():
    """The extension module around libartemis_ops.so (csrc/ops_torch.cpp: the operators on torch tensors), loaded once
    per process; raise loudly when it is absent."""
    global _ops_host
    if _ops_host is None:
        import importlib.util

        import torch  # noqa: F401  (its libraries first)
        load_ops()
        path = _build.OPS_HOST_PATH
        if not os.path.exists(path):
            raise SynthLibraryError(f"{path} not found: build it with `python -m artemis_amd.build`. There is no fallback path.")
        try:
            spec = importlib.util.spec_from_file_location("_artemis_ops", path)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
        except ImportError as e:
            raise SynthLibraryError(f"cannot load {path}: {e}") from e
        _ops_host = module
    return _ops_host


def check(code: int, what: str) -> None:
    if code != 0:
        msg = load().artemis_synth_last_error().decode("utf-8", "replace")
        raise RuntimeError(f"{what} failed (hipError {code}): {msg}")


def version() -> str:
    return load().artemis_synth_version().decode()
