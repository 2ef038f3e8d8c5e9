"""The ragged serving step's binding: gqa_kernels._serving_ext, loaded and bound to the library.

A step makes these calls once per layer, so their checks, allocations and the call itself
are native (csrc/serving_ext.cpp). There is no fallback: a missing binding raises.
"""
import ctypes
import threading

from . import _lib

_ext = None
_lock = threading.Lock()
_ENTRY_POINTS = ("gqa_step_plan", "gqa_qk_norm_rope", "gqa_ragged_fwd", "gqa_ragged_fwd_workspace_bytes", "gqa_verify_drafts",
                 "gqa_verify_greedy", "gqa_verify_workspace_bytes", "gqa_strerror")


def load():
    """Loads (once) and returns the binding, bound to the library that _lib selects."""
    global _ext
    if _ext is None:
        with _lock:
            if _ext is None:
                lib = _lib.load()
                try:
                    from . import _serving_ext
                except ImportError as e:
                    raise RuntimeError("gqa_kernels/_serving_ext.so is missing or does not fit the installed torch: build it "
                                       "with `python gqa-flash-attn-rtx3060_b200/build.py`") from e
                _serving_ext.bind(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRY_POINTS))
                _lib.ON_DEVICE_ERROR.append(_serving_ext.drop_workspaces)
                _ext = _serving_ext
    return _ext
