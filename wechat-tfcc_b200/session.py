"""Per-device launch context: stream, scratch and the device status word.

Plays the part of the reference's thread-default Session
(tfcc/core/framework/tfcc_session.h:28-66, tfcc/cuda/framework/tfcc_cudasession.cpp:36-63):
operators enqueue on its stream and never synchronise; ``sync()`` waits and
surfaces asynchronous device-side failures, as ``Session::sync`` does.
"""
from __future__ import annotations

import threading

import torch

from . import exceptions
from ._lib import lib

_local = threading.local()


class Session:
    def __init__(self, device: torch.device):
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise exceptions.InvalidArgumentError("a B200 session needs a CUDA device")
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._workspaces = {}  # one scratch buffer per stream: calls on two streams may overlap

    @property
    def stream_ptr(self) -> int:
        return torch.cuda.current_stream(self.device).cuda_stream

    @property
    def status_ptr(self) -> int:
        return self._status.data_ptr()

    def scratch_on(self, stream_ptr: int):
        """``(pointer, bytes)`` of the current stream's buffer as it stands, to offer to an entry point that
        checks what it needs before it launches anything; nothing under capture, see :meth:`workspace_on`."""
        ws = self._workspaces.get(stream_ptr)
        if ws is None or _capturing():
            return None, 0
        return ws.data_ptr(), ws.numel()

    def workspace_on(self, nbytes: int):
        """``(pointer, bytes, owner)`` of scratch for one call on the current stream: the stream's buffer
        (:meth:`workspace`), or under capture one of the call's own, so that captured graphs, which may
        be replayed side by side, share none.  ``owner`` has to live until the call is launched."""
        if nbytes and _capturing():
            own = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
            return own.data_ptr(), nbytes, own
        return *self.workspace(nbytes), None

    def workspace(self, nbytes: int):
        """Scratch of at least ``nbytes`` for calls on the current stream (grown
        geometrically, reused by later calls on that stream).  A buffer that is outgrown is
        handed back to torch's allocator, which keeps it out of other streams' hands until
        the kernels queued on this stream have used it."""
        if nbytes == 0:
            return None, 0
        stream = torch.cuda.current_stream(self.device)
        key = stream.cuda_stream
        ws = self._workspaces.get(key)
        if ws is None or ws.numel() < nbytes:
            with torch.cuda.stream(stream):
                new = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=self.device)
            if ws is not None:
                ws.record_stream(stream)
            ws = self._workspaces[key] = new
        return ws.data_ptr(), ws.numel()

    def sync(self) -> None:
        torch.cuda.current_stream(self.device).synchronize()
        st = int(self._status.item())
        if st:
            self._status.zero_()
            if not st & 0xF:  # no wait ran out
                raise exceptions.InvalidArgumentError(
                    f"a cache operator met sequences or pages out of range (bits 0x{st:x})")
            raise exceptions.RuntimeError(-6, f"a kernel abandoned a bounded wait (bits 0x{st:x})")


def launch_context(device):
    """``(session, current stream's handle, guard)`` for a call on a tensor's device.  The launches of
    one decode step take a few microseconds each, so this avoids what a call can do without: the guard
    that makes ``device`` current is a no-op when it already is."""
    index = device.index
    table = getattr(_local, "sessions", None)
    sess = table.get(index) if table is not None else None
    if sess is None:
        sess = get_session(device)
    return sess, _raw_stream(index), _NO_GUARD if _current_device() == index else torch.cuda.device(device)


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()
_capturing = torch.cuda.is_current_stream_capturing
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def get_session(device) -> Session:
    """Thread-default session of ``device`` (created on first use)."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    table = getattr(_local, "sessions", None)
    if table is None:
        table = _local.sessions = {}
    s = table.get(device.index)
    if s is None:
        s = table[device.index] = Session(device)
    return s
