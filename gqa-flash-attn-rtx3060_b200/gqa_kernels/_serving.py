"""Calls of the ragged serving step's C entry points.

They take one struct each (include/gqa_sm100.h), which is packed here with the struct
module: a step makes these calls once per layer, and one packed argument costs a quarter
of ctypes' conversion of thirty. The workspace of attention and verification is kept per
device and stream; its counters have the same place for every shape, so nothing is
zeroed after its allocation, and it only grows.
"""
import struct
import threading

import torch

from . import _lib

_GQA_ERR_WORKSPACE = 6

# The structs' fields in order; a workspace's two fields come first where there is one.
STEP_PLAN = struct.Struct("@14Pq5i").pack
QK_NORM_ROPE = struct.Struct("@11P10q16i3f").pack
RAGGED = struct.Struct("@11P14q14i4f").pack
VERIFY = struct.Struct("@8P6q5i").pack
_WORKSPACE = struct.Struct("@PN").pack

_raw_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice

_workspaces = {}  # (device index, stream) -> (pointer, bytes)
_buffers = []     # every workspace ever handed out: a captured graph may still use it
_lock = threading.Lock()


def _drop(index):
    with _lock:
        for key in [k for k in _workspaces if k[0] == index]:
            del _workspaces[key]


_lib.ON_DEVICE_ERROR.append(_drop)


def device_index(first, *others):
    """The index of the CUDA device that holds all the tensors (None entries are skipped)."""
    index = first.get_device()
    if index < 0:
        raise ValueError("tensors must be on a CUDA device")
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError("tensors must be on one device" if t.is_cuda else "tensors must be on a CUDA device")
    return index


def call(name, args, index):
    """lib.<name>(args, current stream of the device)."""
    fn = getattr(_lib._lib or _lib.load(), name)
    if _current() == index:
        rc = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def call_with_workspace(name, args, index, query):
    """The same with this stream's workspace in front of the packed arguments. `query(lib,
    args)` gives the bytes that the call needs; it is asked when the workspace is too small."""
    if _current() != index:
        with torch.cuda.device(index):
            return call_with_workspace(name, args, index, query)
    lib = _lib._lib or _lib.load()
    stream = _raw_stream(index)
    ws = _workspaces.get((index, stream))
    rc = getattr(lib, name)(_WORKSPACE(*ws) + args, stream) if ws else _GQA_ERR_WORKSPACE
    if rc == _GQA_ERR_WORKSPACE:
        need = query(lib, _WORKSPACE(0, 0) + args)
        with _lock:
            ws = _workspaces.get((index, stream))
            if ws is None or ws[1] < need:
                n = max(need, 4 << 20, 2 * ws[1] if ws else 0)
                buf = torch.zeros(n, dtype=torch.uint8, device=torch.device("cuda", index))
                _buffers.append(buf)
                ws = _workspaces[(index, stream)] = (buf.data_ptr(), n)
        rc = getattr(lib, name)(_WORKSPACE(*ws) + args, stream)
    if rc:
        if rc not in (1, 2, 3):  # anything but a refusal: the counters are not trusted any more
            _drop(index)
        _lib.check(rc, name)
