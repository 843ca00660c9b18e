"""Selective state space scan for packed prompts and for single tokens.

The recurrence with one decay per head, GDN's gate without its delta rule. Per sequence and
head h, which reads group h // (H / G) of B and C, with the state S [P, Ns]:

    d = softplus(dt + dt_bias)        g = exp(-exp(A_log) d)
    S <- g S + d x (outer) B          y = S C + D x

    x            bf16 [T, H, P] (prompts), [B, 1, H, P] (tokens)
    dt           [T, H] / [B, 1, H]     A_log, dt_bias [H], D [H] or None: bf16 or fp32
    B, C         bf16 [T, G, Ns] / [B, 1, G, Ns], H a multiple of G
    state        fp32 [N, H, P, Ns] or None (zeros); tokens: fp32 or bf16
    cu_seqlens   [N + 1] int32 or int64
    returns      (output like x, new_state like state)

P is 1 to 256, Ns 16, 32, 64, 128 or 256. Sums, gates and states are fp32 (a bf16 state is
rounded once per token), outputs bf16. An empty sequence passes its state through; outputs of
tokens that no sequence covers are not written. Inputs are never modified (except by
``decode_inplace``). The first ``prefill`` on a device allocates its status words: make it
before a stream capture.
"""
from __future__ import annotations

import torch

from . import _checks as K
from . import _lib, _status

STATE_DIMS = (16, 32, 64, 128, 256)
MAX_HEAD_DIM = 256


class _Args:
    __slots__ = ("dev", "T", "H", "G", "P", "Ns", "x", "dt", "dt_t", "A", "A_t", "B", "C", "D",
                 "D_t", "dtb", "dtb_t", "state", "cu", "cu_t", "N")


def _aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone()


_NAMES = ("x", "dt", "A_log", "B", "C", "D", "dt_bias", "state", "cu_seqlens")


def _gate(name, t, shape):
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    return K.as_gate(name, t)


def _args(x, dt, A_log, B, C, D, dt_bias, state, cu, lead: int) -> _Args:
    """Checks shared by prompts (lead = 1) and tokens (lead = 2: [B, 1, ...])."""
    a = _Args()
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a torch.Tensor, got {type(x).__name__}")
    dev, shape = x.device, tuple(x.shape)
    if len(shape) != lead + 2 or (lead == 2 and shape[1] != 1):
        raise ValueError("x must be a %s tensor" % ("[T, H, P]" if lead == 1 else "[B, 1, H, P]"))
    K.require_all(dev, _NAMES, (x, dt, A_log, B, C, D, dt_bias, state, cu))
    of_b, head = tuple(B.shape), shape[:lead]
    T, H, P = shape[0], shape[-2], shape[-1]
    if len(of_b) != lead + 2 or of_b[:lead] != head or C.shape != of_b:
        raise ValueError(f"B and C must be {list(head)} + [G, Ns], got {of_b} and "
                         f"{tuple(C.shape)}")
    G, Ns = of_b[-2], of_b[-1]
    if Ns not in STATE_DIMS:
        raise ValueError(f"the state size must be one of {STATE_DIMS}, got {Ns}")
    if not 1 <= P <= MAX_HEAD_DIM:
        raise ValueError(f"the head size must be 1 to {MAX_HEAD_DIM}, got {P}")
    if G <= 0 or H <= 0 or H % G:
        raise ValueError(f"num_heads ({H}) must be a positive multiple of num_groups ({G})")
    a.dev, a.T, a.H, a.P, a.G, a.Ns = dev, T, H, P, G, Ns
    a.x, a.B, a.C = K.as_bf16("x", x), K.as_bf16("B", B), K.as_bf16("C", C)
    if (a.B.data_ptr() | a.C.data_ptr()) % 16:
        a.B, a.C = _aligned(a.B), _aligned(a.C)
    a.dt, a.dt_t = _gate("dt", dt, head + (H,))
    vec = (H,)
    a.A, a.A_t = _gate("A_log", A_log, vec)
    a.dtb, a.dtb_t = _gate("dt_bias", dt_bias, vec)
    a.D, a.D_t = (None, 0) if D is None else _gate("D", D, vec)
    return a


def _prefill_args(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens) -> _Args:
    if cu_seqlens is None:
        raise ValueError("cu_seqlens is required")
    a = _args(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, 1)
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a 1-D tensor of length num_seqs + 1")
    a.cu, a.cu_t = K.as_index("cu_seqlens", cu_seqlens)
    a.N = a.cu.numel() - 1
    a.state = None
    if state is not None:
        if state.shape != (a.N, a.H, a.P, a.Ns):
            raise ValueError(f"state must be [{a.N}, {a.H}, {a.P}, {a.Ns}], "
                             f"got {tuple(state.shape)}")
        if state.dtype != torch.float32:
            state = state.float()
        a.state = _aligned(state.contiguous())
    return a


def prefill_recurrent(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, *, check=False):
    """The scan token by token (one launch): any head size, the independent check of the
    chunked kernel."""
    a = _prefill_args(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens)
    lib = _lib.load()
    with K.on_device(a.dev):
        status = _status.address(a.dev.index)
        out = torch.empty(a.T, a.H, a.P, dtype=torch.bfloat16, device=a.dev)
        new_state = torch.empty(a.N, a.H, a.P, a.Ns, dtype=torch.float32, device=a.dev)
        rc = lib.gdn_ssm_prefill_recurrent_fwd(
            a.x.data_ptr(), a.dt.data_ptr(), a.dt_t, a.A.data_ptr(), a.A_t, a.B.data_ptr(),
            a.C.data_ptr(), K.ptr(a.D), a.D_t, a.dtb.data_ptr(), a.dtb_t, K.ptr(a.state),
            a.cu.data_ptr(), a.cu_t, out.data_ptr(), new_state.data_ptr(), a.T, a.N, a.H, a.G,
            a.P, a.Ns, status, K.stream_handle(a.dev))
        _lib.check(rc, "gdn_ssm_prefill_recurrent_fwd")
        _status.finish(a.dev.index, check)
    return out, new_state


def prefill(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, *, check=False):
    """The scan over packed prompts: (output [T, H, P] bf16, new_state [N, H, P, Ns] fp32).
    A ``cu_seqlens`` that leaves [0, T] or decreases, or a bounded wait that gave up, raises
    GDNError at the next call on the device, or at this one with ``check=True`` (which
    synchronises)."""
    a = _prefill_args(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens)
    lib = _lib.load()
    with K.on_device(a.dev):
        status = _status.address(a.dev.index)
        out = torch.empty(a.T, a.H, a.P, dtype=torch.bfloat16, device=a.dev)
        new_state = torch.empty(a.N, a.H, a.P, a.Ns, dtype=torch.float32, device=a.dev)
        nbytes = lib.gdn_ssm_prefill_workspace_size(a.T, a.N, a.H, a.G, a.P, a.Ns)
        # of this call alone: calls on several streams and captured graphs share nothing
        ws = torch.empty(nbytes, dtype=torch.uint8, device=a.dev) if nbytes else None
        rc = lib.gdn_ssm_prefill_fwd(
            _aligned(a.x).data_ptr(), a.dt.data_ptr(), a.dt_t, a.A.data_ptr(), a.A_t,
            a.B.data_ptr(), a.C.data_ptr(), K.ptr(a.D), a.D_t, a.dtb.data_ptr(), a.dtb_t,
            K.ptr(a.state), a.cu.data_ptr(), a.cu_t, out.data_ptr(), new_state.data_ptr(), a.T,
            a.N, a.H, a.G, a.P, a.Ns, K.ptr(ws), nbytes, status, K.stream_handle(a.dev))
        _lib.check(rc, "gdn_ssm_prefill_fwd")
        _status.finish(a.dev.index, check)
    return out, new_state


def _decode(x, dt, A_log, B, C, D, dt_bias, state, inplace):
    a = _args(x, dt, A_log, B, C, D, dt_bias, state, None, 2)
    shape = (a.T, a.H, a.P, a.Ns)
    s = state
    if state is not None:
        if state.shape != shape:
            raise ValueError(f"state must be {list(shape)}, got {tuple(state.shape)}")
        if not inplace:
            if s.dtype not in (torch.float32, torch.bfloat16):
                s = s.float()
            s = _aligned(s.contiguous())
    s_dtype = torch.float32 if s is None else s.dtype
    lib = _lib.load()
    with K.on_device(a.dev):
        out = torch.empty(a.T, 1, a.H, a.P, dtype=torch.bfloat16, device=a.dev)
        new_state = state if inplace else torch.empty(*shape, dtype=s_dtype, device=a.dev)
        rc = lib.gdn_ssm_decode_fwd(
            a.x.data_ptr(), a.dt.data_ptr(), a.dt_t, a.A.data_ptr(), a.A_t, a.B.data_ptr(),
            a.C.data_ptr(), K.ptr(a.D), a.D_t, a.dtb.data_ptr(), a.dtb_t, K.ptr(s),
            _lib.DTYPE_F32 if s_dtype == torch.float32 else _lib.DTYPE_BF16, out.data_ptr(),
            new_state.data_ptr(), a.T, a.H, a.G, a.P, a.Ns, K.stream_handle(a.dev))
    _lib.check(rc, "gdn_ssm_decode_fwd")
    return out, new_state


def decode(x, dt, A_log, B, C, D, dt_bias, state):
    """One new token per sequence: (output [B, 1, H, P] bf16, new_state of ``state``'s type)."""
    return _decode(x, dt, A_log, B, C, D, dt_bias, state, False)


def decode_inplace(x, dt, A_log, B, C, D, dt_bias, state):
    """``decode`` that updates ``state`` (fp32 or bf16, contiguous, 16-byte aligned) in place;
    returns (output, state)."""
    if state is None or state.dtype not in (torch.float32, torch.bfloat16) \
            or not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("decode_inplace needs a contiguous, 16-byte aligned fp32 or bf16 state")
    return _decode(x, dt, A_log, B, C, D, dt_bias, state, True)


def reset_device_status(device=None) -> None:
    """Clear the status words of a device after its queued work is done (shared with
    ``short_conv``)."""
    _status.reset(device)
