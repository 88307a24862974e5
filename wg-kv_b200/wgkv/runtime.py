"""Per-device state shared by the ops: error word, scratch workspaces, streams.

Workspaces are cached per (device, stream, purpose) and only grow.  Their
leading counters must be zero when a kernel starts and the kernels leave them
zero; a cached buffer records how many leading bytes are known to be zero, and
a call that needs a longer counter prefix (more heads, more rows) zeroes the
extra bytes first, since they may hold an earlier call's partial results.
After a call only its own prefix is known to be zero.
"""
from __future__ import annotations

import threading

import torch

from ._lib import ERR_BITS, check, lib

_lock = threading.Lock()  # held while something that outlives a call is made, not while it is looked up
_err_words: dict = {}
_workspaces: dict = {}


def require_cuda(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (this library has no CPU path)")


def raw_stream(index: int) -> int:
    """``stream_ptr`` of device ``index`` without building a Stream object (a C call)."""
    return torch._C._cuda_getCurrentRawStream(index)


def stream_ptr(device=None) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _new_error_word(index: int) -> torch.Tensor:
    """A zero on device ``index`` that kernels of any stream may flag from now on.

    It is made on a stream of its own and waited for: the current stream may have work queued behind which
    the zero would arrive after another stream's flag, or may be capturing a graph, in whose memory the word
    would be set to zero by every replay.  And it is an ordinary tensor, which check_errors() may reset in or
    out of inference mode."""
    mode = lib.wgkv_thread_capture_mode(2)
    check(min(mode, 0), "wgkv_thread_capture_mode")
    try:
        with torch.cuda.device(index), torch.inference_mode(False):
            stream = torch.cuda.Stream()
            while lib.wgkv_stream_capture_id(stream.cuda_stream):  # torch deals its streams in turns
                stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                w = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
            stream.synchronize()
    finally:
        lib.wgkv_thread_capture_mode(mode)
    return w


def err_word(device) -> torch.Tensor:
    d = torch.device(device)
    key = d.index if d.index is not None else torch.cuda.current_device()
    w = _err_words.get(key)
    if w is None:
        with _lock:  # one word a device, whichever threads ask first: check_errors() reads no other
            w = _err_words.get(key)
            if w is None:
                w = _err_words[key] = _new_error_word(key)
    return w


def check_errors(device=None, reset: bool = True):
    """Synchronise and raise AssertionError if a kernel flagged an error.

    The device-side capacity checks mirror the reference's asserts
    (src/modeling_layers.py:1313-1321, :683-686, :702-704), so the raised type
    is the same."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    w = err_word(dev)
    v = int(w.item())
    if v:
        if reset:
            w.zero_()
        msgs = [m for bit, m in ERR_BITS.items() if v & bit]
        raise AssertionError("wgkv device error: " + "; ".join(msgs))


def workspace(device, purpose: str, nbytes: int, zero_prefix: int = 0) -> torch.Tensor:
    d = torch.device(device)
    key = (d.index, torch.cuda.current_stream(d).cuda_stream, purpose)
    ent = _workspaces.get(key)
    if ent is None or ent[0].numel() < nbytes:
        with torch.inference_mode(False):  # later calls may zero a longer prefix out of inference mode
            ws = torch.empty(max(nbytes, zero_prefix, 256), dtype=torch.uint8, device=d)
        zeroed = 0
    else:
        ws, zeroed = ent
    if zero_prefix > zeroed:
        # stream-ordered: runs after every earlier user of this buffer on this stream
        ws[zeroed:zero_prefix].zero_()
    # this call's kernels may write anything past its own prefix and leave the prefix zero
    _workspaces[key] = (ws, zero_prefix)
    return ws


_counter_scratch: dict = {}  # (device index, stream, purpose) -> (data pointer, bytes, capture id, tensors)


def counter_scratch(index: int, stream: int, purpose: str, nbytes: int, zero_prefix: int):
    """(pointer, bytes) of scratch of the current device whose first ``zero_prefix`` bytes (the same for every
    call of a purpose) are zero and are left zero by the kernels that use it: :func:`workspace` for one raw
    stream, found with one dictionary look-up, and safe under capture.  While a graph is captured its calls
    get scratch of the graph's own (from its memory pool, zeroed by a node of the graph): graphs captured on
    one stream may replay on several at a time, and must not share counters and partial results with one
    another or with the stream's eager calls.  Scratch that was outgrown is kept (sizes double): another
    thread may be about to launch on it.  For the same reason a miss is served under a lock: of two threads
    that miss together the second takes what the first has made, so that no address is handed out whose
    tensor the dictionary does not hold."""
    capture = 0
    key = (index, stream, purpose)
    if torch.cuda.is_current_stream_capturing():
        capture = lib.wgkv_stream_capture_id(stream)
        key = (index, stream, purpose, "capture")
    ent = _counter_scratch.get(key)
    if ent is None or ent[1] < nbytes or ent[2] != capture:
        with _lock:
            ent = _counter_scratch.get(key)
            if ent is None or ent[1] < nbytes or ent[2] != capture:
                size = 1 << (nbytes - 1).bit_length()
                t = torch.empty(size, dtype=torch.uint8, device=torch.device("cuda", index))
                t[:zero_prefix].zero_()  # stream-ordered, before the first kernel that counts in it
                outgrown = ent[3] if ent is not None and ent[2] == capture else ()
                ent = _counter_scratch[key] = (t.data_ptr(), size, capture, (*outgrown, t))
    return ent[0], ent[1]


def num_sms() -> int:
    return int(lib.wgkv_num_sms())
