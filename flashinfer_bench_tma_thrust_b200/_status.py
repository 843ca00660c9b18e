"""Status words of the short convolution and the state space scan.

Their kernels report what the host cannot see without a synchronisation (a bound of
``cu_seqlens`` outside the packed tokens, a bounded wait that gave up) through two int32
words per device in pinned host memory, which they write directly: nothing is copied or
queued per call, and a captured graph reports like an eager call. Every call reads the words
of its device before it launches and raises for what an earlier call left there.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib

_words: dict = {}  # device index -> (pinned tensor, its words as one 64-bit number, address)
_lock = threading.Lock()


def _entry(index: int):
    e = _words.get(index)
    if e is None:
        with _lock:
            e = _words.get(index)
            if e is None:
                t = torch.zeros(2, dtype=torch.int32, pin_memory=True)
                e = _words[index] = (t, ctypes.c_int64.from_address(t.data_ptr()), t.data_ptr())
    return e


def address(index: int) -> int:
    """Address of the device's words, after raising for what they already hold."""
    e = _words.get(index) or _entry(index)
    if e[1].value:
        raise_for(index)
    return e[2]


def raise_for(index: int) -> None:
    wait, bounds = _entry(index)[0].tolist()
    if wait or bounds:
        what = [w for w, on in (("a bounded wait gave up", wait),
                                ("cu_seqlens is not a non-decreasing sequence within [0, T]",
                                 bounds)) if on]
        raise _lib.GDNError(f"a call on cuda:{index} reported: {'; '.join(what)}; its outputs "
                            "are invalid. Clear with reset_device_status().")


def finish(index: int) -> None:
    """Wait for the current stream and raise for what its calls reported."""
    torch.cuda.current_stream(index).synchronize()
    raise_for(index)


def reset(device=None) -> None:
    """Clear the words of a device (default: the current one) once its queued work is done."""
    index = torch.device("cuda" if device is None else device).index
    if index is None:
        index = torch.cuda.current_device()
    torch.cuda.synchronize(index)
    _entry(index)[1].value = 0
