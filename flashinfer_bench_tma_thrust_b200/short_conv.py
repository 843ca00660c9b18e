"""Short causal depthwise convolution for packed prompts and for single tokens.

The convolution in front of a linear-state operator: it makes GDN's q, k and v (or the state
space scan's x, B and C) from the projected channels. With W taps (2, 3 or 4) and u the inputs
of a sequence behind its W - 1 earlier rows (``state``, or zeros):

    c_t = bias + sum_k weight[:, k] u_{t-W+1+k}        y = silu(c)  (activation=None: c)

``split`` cuts the channels into sections that are returned as dense tensors of their own, and
``l2norm`` divides each head of 128 channels of a section by sqrt(sum of squares + eps), as GDN
wants its q and k:

    (q, k, v), conv_state = short_conv.prefill(x, weight, bias, conv_state, cu_seqlens,
                                               split=(HQ * 128, HQ * 128, HV * 128),
                                               l2norm=(True, True, False))
    out, state = prefill.kernel(q.view(-1, HQ, 128), k.view(-1, HQ, 128), v.view(-1, HV, 128),
                                state, A_log, a, dt_bias, b, cu_seqlens)

    x          bf16 [T, C] (prompts), [B, 1, C] (tokens); rows may be strided
    weight     [C, W] or [C, 1, W], bias [C] or None: bf16 or fp32
    state      bf16 [N, W - 1, C]: the last W - 1 inputs of each sequence, oldest first; or None
    cu_seqlens [N + 1] int32 or int64
    returns    (output or tuple of sections, new_state)

Sums are fp32, outputs bf16, rounded once; how tokens are packed or cut into calls changes no bit
of them. A head of zeros with eps = 0 gives NaN (0 / 0). An empty sequence passes its state
through; outputs of tokens that no sequence covers are not written. Inputs are never modified
(except by ``decode_inplace``). Every call is one launch on the current stream of x's device. The
first ``prefill`` on a device allocates its status words: make it before a stream capture.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _checks as C
from . import _lib, _status

MAX_SECTIONS = 8


_NAMES = ("x", "weight", "bias", "state", "cu_seqlens")
_BF16, _empty, _empty_like = torch.bfloat16, torch.empty, torch.empty_like


def _taps(x, weight, bias):
    """(weight, code, bias, code, W), checked."""
    if weight is None:
        C.require_given(("weight",), (weight,))
    ch, shape = x.shape[-1], weight.shape
    if len(shape) == 3 and shape[1] == 1:
        weight = weight[:, 0]
        shape = weight.shape
    if len(shape) != 2 or shape[0] != ch or not 2 <= shape[1] <= 4:
        raise ValueError(f"weight must be [{ch}, W] with 2 to 4 taps, got {tuple(shape)}")
    w, w_t = C.as_gate("weight", weight)
    if bias is None:
        return w, w_t, None, 0, shape[1]
    if bias.shape != (ch,):
        raise ValueError(f"bias must be [{ch}], got {tuple(bias.shape)}")
    return w, w_t, *C.as_gate("bias", bias), shape[1]


def _state(state, shape):
    if state is None:
        return None
    if state.shape != shape:
        raise ValueError(f"state must be {list(shape)}, got {tuple(state.shape)}")
    return C.as_bf16("state", state)


def _rows(x):
    if x.dtype != torch.bfloat16:
        raise TypeError(f"x must be bfloat16, got {x.dtype}")
    if x.shape[-1] == 0:
        raise ValueError("x has no channels")
    return x if x.stride(-1) == 1 else x.contiguous()


@functools.lru_cache(maxsize=256)
def _sections(ch, split, l2norm):
    """(widths, the library's arrays of widths and norms), checked; `split` and `l2norm` as the
    caller gave them, sequences as tuples."""
    widths = (ch,) if split is None else tuple(int(w) for w in split)
    if not 1 <= len(widths) <= MAX_SECTIONS or min(widths) <= 0 or sum(widths) != ch:
        raise ValueError(f"split must be 1 to {MAX_SECTIONS} positive widths summing to {ch}, "
                         f"got {widths}")
    if l2norm is None or isinstance(l2norm, bool):
        normed = (bool(l2norm),) * len(widths)
    else:
        normed = tuple(bool(v) for v in l2norm)
    if len(normed) != len(widths):
        raise ValueError(f"l2norm must have one entry per section ({len(widths)})")
    at = 0
    for w, n in zip(widths, normed):
        if n and (at % C.HEAD_DIM or w % C.HEAD_DIM):
            raise ValueError("a section with l2norm must begin at and span whole heads of "
                             f"{C.HEAD_DIM} channels, got begin {at}, width {w}")
        at += w
    i32 = ctypes.c_int32 * len(widths)
    return widths, i32(*widths), i32(*normed), ctypes.c_void_p * len(widths)


def _hashable(v):
    return v if v is None or isinstance(v, (bool, tuple)) else tuple(v)


def _activation(activation) -> int:
    if activation is None:
        return 0
    if activation in ("silu", "swish"):
        return 1
    raise ValueError(f"activation must be 'silu' or None, got {activation!r}")


def prefill(x, weight, bias=None, state=None, cu_seqlens=None, *, activation="silu", split=None,
            l2norm=None, eps=1e-6, check=False):
    """The convolution over packed prompts: (output [T, C] or a tuple of sections, new_state
    [N, W - 1, C]). A ``cu_seqlens`` that leaves [0, T] or decreases raises GDNError at the
    next call on the device, or at this one with ``check=True`` (which synchronises)."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError("x must be a [T, C] tensor")
    if cu_seqlens is None:
        raise ValueError("cu_seqlens is required")
    dev = x.device
    C.require_all(dev, _NAMES, (x, weight, bias, state, cu_seqlens))
    w, w_t, b, b_t, taps = _taps(x, weight, bias)
    ch = x.shape[-1]
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a 1-D tensor of length num_seqs + 1")
    cu, cu_t = C.as_index("cu_seqlens", cu_seqlens)
    n, t = cu.numel() - 1, x.shape[0]
    s = _state(state, (n, taps - 1, ch))
    if x.dtype is not _BF16 or x.stride(-1) != 1 or not ch:
        x = _rows(x)
    widths, wa, na, pointers = _sections(ch, _hashable(split), _hashable(l2norm))
    act = _activation(activation)
    if not eps >= 0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    lib = _lib.load()
    with C.on_device(dev):
        status = _status.address(dev.index)
        outs = [_empty(t, v, dtype=_BF16, device=dev) for v in widths]
        new_state = _empty(n, taps - 1, ch, dtype=_BF16, device=dev) \
            if s is None else _empty_like(s)
        rc = lib.gdn_conv_prefill_fwd(
            x.data_ptr(), x.stride(0), w.data_ptr(), w_t, C.ptr(b), b_t, C.ptr(s), cu.data_ptr(),
            cu_t, act, len(widths), wa, na, eps, pointers(*[o.data_ptr() for o in outs]),
            new_state.data_ptr(), t, n, ch, taps, status,
            C.stream_handle(dev))
        if rc:
            _lib.check(rc, "gdn_conv_prefill_fwd")
        if check:
            _status.finish(dev.index)
    return (outs[0] if split is None else tuple(outs)), new_state


def _decode(x, weight, bias, state, activation, split, l2norm, eps, inplace):
    if not isinstance(x, torch.Tensor) or x.dim() != 3 or x.shape[1] != 1:
        raise ValueError("x must be a [B, 1, C] tensor")
    dev = x.device
    C.require_all(dev, _NAMES, (x, weight, bias, state, None))
    w, w_t, b, b_t, taps = _taps(x, weight, bias)
    ch = x.shape[-1]
    n = x.shape[0]
    s = _state(state, (n, taps - 1, ch))
    if x.dtype is not _BF16 or x.stride(-1) != 1 or not ch:
        x = _rows(x)
    widths, wa, na, pointers = _sections(ch, _hashable(split), _hashable(l2norm))
    act = _activation(activation)
    if not eps >= 0:
        raise ValueError(f"eps must be at least 0, got {eps}")
    lib = _lib.load()
    with C.on_device(dev):
        outs = [_empty(n, 1, v, dtype=_BF16, device=dev) for v in widths]
        new_state = state if inplace else (
            _empty(n, taps - 1, ch, dtype=_BF16, device=dev) if s is None
            else _empty_like(s))
        rc = lib.gdn_conv_decode_fwd(
            x.data_ptr(), x.stride(0), w.data_ptr(), w_t, C.ptr(b), b_t, C.ptr(s), act,
            len(widths), wa, na, eps, pointers(*[o.data_ptr() for o in outs]),
            new_state.data_ptr(), n, ch, taps, C.stream_handle(dev))
    if rc:
        _lib.check(rc, "gdn_conv_decode_fwd")
    return (outs[0] if split is None else tuple(outs)), new_state


def decode(x, weight, bias=None, state=None, *, activation="silu", split=None, l2norm=None,
           eps=1e-6):
    """One new token per sequence: (output [B, 1, C] or a tuple of sections, new_state)."""
    return _decode(x, weight, bias, state, activation, split, l2norm, eps, False)


def decode_inplace(x, weight, bias, state, *, activation="silu", split=None, l2norm=None,
                   eps=1e-6):
    """``decode`` that moves ``state`` (bf16, contiguous) on in place; returns (output, state)."""
    if state is None or state.dtype != torch.bfloat16 or not state.is_contiguous():
        raise ValueError("decode_inplace needs a contiguous bf16 state tensor")
    return _decode(x, weight, bias, state, activation, split, l2norm, eps, True)


def reset_device_status(device=None) -> None:
    """Clear the status words of a device after its queued work is done (shared with ``ssm``)."""
    _status.reset(device)
