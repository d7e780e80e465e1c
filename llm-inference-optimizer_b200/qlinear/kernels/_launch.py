"""Host-side plumbing shared by the linear wrappers: device/stream
selection, the per-stream split-K workspace and the launch flags."""
from __future__ import annotations

import os
import threading

import torch

from .. import _lib

_ws_lock = threading.Lock()
_workspaces: dict[tuple[int, int], torch.Tensor] = {}
_MIN_WS = 1 << 20


def default_flags() -> int:
    """Programmatic dependent launch is on unless QLINEAR_PDL=0: the kernels
    stream their (static) weights while the previous kernel finishes."""
    return 0 if os.environ.get("QLINEAR_PDL", "1") == "0" else _lib.QL_FLAG_PDL


def workspace(device: torch.device, stream: torch.cuda.Stream, nbytes: int) -> torch.Tensor | None:
    """Zero-filled scratch for split-K, one per (device, stream).

    The kernels leave it zero-filled after every call, so it is created once
    and reused; calls on one stream are ordered, so they never overlap.  A
    first (eager) call sizes it, which keeps later CUDA-graph captures free
    of allocations."""
    if nbytes == 0:
        return None
    key = (device.index, stream.cuda_stream)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        with _ws_lock:
            buf = _workspaces.get(key)
            if buf is None or buf.numel() < nbytes:
                size = max(_MIN_WS, 1 << (int(nbytes) - 1).bit_length())
                buf = torch.zeros(size, dtype=torch.uint8, device=device)
                _workspaces[key] = buf
    return buf


_scratches: dict[tuple[int, int], torch.Tensor] = {}
_graph_scratches: dict[tuple[int, int], tuple[int, torch.Tensor]] = {}
_SCRATCH_HEADER = 8192           # ql_tree_attention's counters


# Without the checks of torch.cuda's own: there are CUDA tensors by then.
current_device = torch._C._cuda_getDevice
is_capturing = torch._C._cuda_isCurrentStreamCapturing


def capture_id(device: torch.device, stream: int) -> int:
    """The capture that records what is launched on `stream` of `device`, or 0."""
    if current_device() == device.index:
        return _lib.load().ql_capture_id(stream) if is_capturing() else 0    # eager calls end here
    with on_device(device):
        return _lib.load().ql_capture_id(stream)


def scratch(device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
    """Scratch whose head alone is kept zero by the kernels, one per (device,
    stream handle) as `workspace`, and one for each capture on it: a graph is
    replayed on any stream, beside other graphs and later calls, so it shares
    none.  Its first call clears the head at every replay.  `nbytes` is the
    same on every call."""
    key = (device.index, stream)
    capture = capture_id(device, stream)
    if capture:
        held = _graph_scratches.get(key)
        if held is None or held[0] != capture:
            buf = torch.empty(nbytes, dtype=torch.uint8, device=device)     # of the graph's memory pool
            buf[:_SCRATCH_HEADER].zero_()
            # held so that nothing else that is captured gets this memory; the last capture's goes back to its pool
            held = _graph_scratches[key] = (capture, buf)
        return held[1]
    buf = _scratches.get(key)
    if buf is None:
        with _ws_lock:
            buf = _scratches.get(key)
            if buf is None:
                buf = _scratches[key] = torch.zeros(nbytes, dtype=torch.uint8, device=device)
    return buf


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def ld(t: torch.Tensor, row_len: int) -> int:
    """Leading dimension (elements between rows) of a 2-D tensor with unit
    inner stride.  A single-row tensor may report any row stride (torch
    treats size-1 dims as contiguous whatever their stride), so its row
    length is used instead."""
    return t.stride(0) if t.shape[0] > 1 else row_len


def dtype_code(dt: torch.dtype) -> int:
    if dt == torch.float16:
        return _lib.QL_DTYPE_F16
    if dt == torch.float32:
        return _lib.QL_DTYPE_F32
    if dt == torch.bfloat16:
        return _lib.QL_DTYPE_BF16
    raise TypeError(f"unsupported dtype {dt}")


class on_device:
    """Make `device` current for the C call (the ABI uses the current device)."""

    def __init__(self, device: torch.device):
        self.idx = device.index
        self.prev = None

    def __enter__(self):
        cur = torch.cuda.current_device()
        if cur != self.idx:
            self.prev = cur
            torch.cuda.set_device(self.idx)
        return self

    def __exit__(self, *exc):
        if self.prev is not None:
            torch.cuda.set_device(self.prev)
        return False


_INDEX_BYTES = {torch.int64: 8, torch.int32: 4}
_ACTIVATION_CODES = {torch.float16: _lib.QL_DTYPE_F16, torch.bfloat16: _lib.QL_DTYPE_BF16}


def index_bytes(t: torch.Tensor, what: str) -> int:
    """4 or 8 for an int32 / int64 index tensor."""
    n = _INDEX_BYTES.get(t.dtype)
    if n is None:
        raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
    return n


def activation_code(dtype: torch.dtype, what: str) -> int:
    """dtype code of a 16-bit activation tensor."""
    code = _ACTIVATION_CODES.get(dtype)
    if code is None:
        raise TypeError(f"{what} must be fp16 or bf16, got {dtype}")
    return code


# The current stream's handle of a device, without building a Stream object
# (2 us of the host's time, as much as a launch).
current_raw_stream = torch._C._cuda_getCurrentRawStream


_call_flags: int | None = None


def call_flags() -> int:
    """default_flags, read once: looking at the environment costs as much as an eighth of a launch."""
    global _call_flags
    if _call_flags is None:
        _call_flags = default_flags()
    return _call_flags


def call(entry, packed: bytes, device: torch.device) -> None:
    """entry(packed arguments, current stream) with `device` current (the ABI uses the current device)."""
    index = device.index
    if current_device() == index:
        status = entry(packed, current_raw_stream(index))
    else:
        with on_device(device):
            status = entry(packed, current_raw_stream(index))
    if status != _lib.QL_OK:
        _lib.check(status)
