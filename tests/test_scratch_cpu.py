"""Scratch and error words that several threads ask for at once, with a stand-in for torch's allocator: whoever
gets an address gets memory that stays."""
import contextlib
import gc
import os
import threading
import weakref
from types import SimpleNamespace

import pytest
import torch

from wgkv import kv4, runtime
from wgkv._lib import LIB_PATH, lib


class Block:
    """Stands for a CUDA tensor: an address of its own for as long as it lives."""
    live = weakref.WeakSet()

    def __init__(self, n):
        self.n = n
        Block.live.add(self)

    def data_ptr(self):
        return id(self)

    def __getitem__(self, _):
        return self

    def zero_(self):
        return self


def overlapping(monkeypatch, first_wait=0.5):
    """Lets two allocations of different threads overlap if the code under test allows it: the first to come
    waits for a second for a while, as it may when the allocator gives up the interpreter's lock."""
    second, lock, seen = threading.Event(), threading.Lock(), []

    def allocate(n, **_):
        with lock:
            seen.append(n)
            mine = len(seen)
        if mine == 1:
            second.wait(first_wait)
        else:
            second.set()
        return Block(n)

    stand_in = SimpleNamespace(
        empty=allocate, zeros=allocate, uint8="uint8", int32="int32", device=torch.device,
        inference_mode=torch.inference_mode, cuda=SimpleNamespace(
            is_current_stream_capturing=lambda: False, current_device=lambda: 0, Stream=lambda: Stream(1),
            stream=lambda s: contextlib.nullcontext(), device=lambda d: contextlib.nullcontext()))
    monkeypatch.setattr(runtime, "torch", stand_in)
    monkeypatch.setattr(runtime, "lib", SimpleNamespace(wgkv_thread_capture_mode=lambda m: 0,
                                                        wgkv_stream_capture_id=lambda s: 0))
    return seen


class Stream:
    def __init__(self, raw):
        self.cuda_stream, self.waited = raw, False

    def synchronize(self):
        self.waited = True


def from_threads(calls):
    out = [None] * len(calls)

    def work(i):
        out[i] = calls[i]()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    gc.collect()
    return out


@pytest.mark.parametrize("before,sizes", [(None, (1000, 1000)), (None, (1000, 70000)), (500, (2000, 2000)),
                                          (500, (70000, 1000))])
def test_counter_scratch_of_two_threads_stays_allocated(monkeypatch, before, sizes):
    monkeypatch.setattr(runtime, "_counter_scratch", {})
    if before is not None:  # both threads outgrow what there is
        overlapping(monkeypatch, 0.0)
        runtime.counter_scratch(0, 7, "purpose", before, 256)
    overlapping(monkeypatch)
    got = from_threads([lambda n=n: runtime.counter_scratch(0, 7, "purpose", n, 256) for n in sizes])
    alive = {b.data_ptr(): b.n for b in Block.live}
    for (ptr, nbytes), need in zip(got, sizes):
        assert ptr in alive, "an address was handed out whose memory has no owner"
        assert alive[ptr] >= nbytes >= need


def test_error_word_of_two_threads_is_one(monkeypatch):
    monkeypatch.setattr(runtime, "_err_words", {})
    monkeypatch.setattr(kv4, "_err_ptrs", {})
    seen = overlapping(monkeypatch)
    got = from_threads([lambda: kv4._err_ptr(0), lambda: runtime.err_word("cuda:0").data_ptr(), lambda: kv4._err_ptr(0)])
    word = runtime.err_word("cuda:0").data_ptr()  # what check_errors() reads
    assert got == [word] * 3 and kv4._err_ptr(0) == word and len(seen) == 1


def test_error_word_outlives_its_dictionary_entry(monkeypatch):
    """An address that kernels are given for good belongs to memory that stays for good."""
    monkeypatch.setattr(runtime, "_err_words", {})
    monkeypatch.setattr(kv4, "_err_ptrs", {})
    overlapping(monkeypatch, 0.0)
    ptr = kv4._err_ptr(0)
    runtime._err_words.clear()
    gc.collect()
    assert ptr in {b.data_ptr() for b in Block.live}


@pytest.mark.parametrize("fails", [False, True])
def test_error_word_is_made_outside_of_captures(monkeypatch, fails):
    """On a stream that is not capturing (torch deals its streams in turns), waited for, and with the thread's
    capture mode put back whatever happens."""
    monkeypatch.setattr(runtime, "_err_words", {})
    overlapping(monkeypatch, 0.0)
    mode, streams, inside = [0], [Stream(5), Stream(5), Stream(6)], []

    def exchange(m):
        mode[0], old = m, mode[0]
        return old

    @contextlib.contextmanager
    def current(s):
        inside.append((s.cuda_stream, mode[0]))
        yield
        if fails:
            raise MemoryError

    dealt = iter(streams)
    monkeypatch.setattr(runtime, "lib", SimpleNamespace(wgkv_thread_capture_mode=exchange,
                                                        wgkv_stream_capture_id=lambda s: 77 if s == 5 else 0))
    monkeypatch.setattr(runtime.torch.cuda, "Stream", lambda: next(dealt))
    monkeypatch.setattr(runtime.torch.cuda, "stream", current)
    if fails:
        with pytest.raises(MemoryError):
            runtime.err_word("cuda:0")
        assert not runtime._err_words
    else:
        runtime.err_word("cuda:0")
        assert streams[2].waited
    assert inside == [(6, 2)] and mode == [0]


@pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="libwgkv.so not built")
def test_capture_mode_is_checked():
    assert lib.wgkv_thread_capture_mode(3) == -1 and lib.wgkv_thread_capture_mode(-1) == -1
