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

``prefill`` takes the chunked kernel where P and Ns are 64 or 128 and T is above 4 N + 8, else
goes token by token. Both give the state to fp32's accuracy (the chunked one: 1e-6 of its size).
The chunked kernel multiplies the state, and the decayed products of C and B, rounded to bf16: its
outputs are off by up to 2^-8 of the sum of their terms' sizes, which is more than their own
rounding where terms cancel. ``prefill_recurrent`` has fp32 there. A dt of -infinity skips a token
(d = 0, g = 1). A NaN or infinity of a token reaches no token before it. From it on, what it enters
is not finite: the same values in both kernels, but NaN in the chunked one where the other may have
an infinity.
"""
from __future__ import annotations

import functools

import torch

from . import _checks as K
from . import _lib, _status

STATE_DIMS = (16, 32, 64, 128, 256)
MAX_HEAD_DIM = 256


_NAMES = ("x", "dt", "A_log", "B", "C", "D", "dt_bias", "state", "cu_seqlens")
_BF16, _F32 = torch.bfloat16, torch.float32
_CODES = K._GATE_CODES


def _aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _gate(name, t, shape):
    """A gate or parameter of the given shape: (contiguous tensor, dtype code)."""
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    code = _CODES.get(t.dtype)
    if code is not None and t.is_contiguous():
        return t, code
    return K.as_gate(name, t)


def _bf16(name, t):
    return t if t.dtype is _BF16 and t.is_contiguous() else K.as_bf16(name, t)


def _args(x, dt, A_log, B, C, D, dt_bias, state, cu, lead: int):
    """Checks shared by prompts (lead = 1) and tokens (lead = 2: [B, 1, ...]). Returns (sizes,
    the tensors to keep, the library's arguments up to dt_bias)."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a torch.Tensor, got {type(x).__name__}")
    shape = x.shape
    if len(shape) != lead + 2 or (lead == 2 and shape[1] != 1):
        raise ValueError("x must be a %s tensor" % ("[T, H, P]" if lead == 1 else "[B, 1, H, P]"))
    K.require_all(x.device, _NAMES, (x, dt, A_log, B, C, D, dt_bias, state, cu))
    if dt is None or A_log is None or B is None or C is None or dt_bias is None:
        K.require_given(("dt", "A_log", "B", "C", "dt_bias"), (dt, A_log, B, C, dt_bias))
    of_b, head = B.shape, shape[:lead]
    T, H, P = shape[0], shape[-2], shape[-1]
    if len(of_b) != lead + 2 or of_b[:lead] != head or C.shape != of_b:
        raise ValueError(f"B and C must be {list(head)} + [G, Ns], got {tuple(of_b)} and "
                         f"{tuple(C.shape)}")
    G, Ns = of_b[-2], of_b[-1]
    if Ns not in STATE_DIMS:
        raise ValueError(f"the state size must be one of {STATE_DIMS}, got {Ns}")
    if not 1 <= P <= MAX_HEAD_DIM:
        raise ValueError(f"the head size must be 1 to {MAX_HEAD_DIM}, got {P}")
    if G <= 0 or H <= 0 or H % G:
        raise ValueError(f"num_heads ({H}) must be a positive multiple of num_groups ({G})")
    x, B, C = _bf16("x", x), _bf16("B", B), _bf16("C", C)
    if (B.data_ptr() | C.data_ptr()) % 16:
        B, C = _aligned(B), _aligned(C)
    if lead == 1 and x.data_ptr() % 16:  # (bulk copies read it)
        x = x.clone()
    dt, dt_t = _gate("dt", dt, shape[:-1])
    vec = (H,)
    A_log, a_t = _gate("A_log", A_log, vec)
    dt_bias, b_t = _gate("dt_bias", dt_bias, vec)
    d_ptr, d_t = None, 0
    if D is not None:
        D, d_t = _gate("D", D, vec)
        d_ptr = D.data_ptr()
    return (T, H, G, P, Ns), (x, dt, A_log, B, C, D, dt_bias), (
        x.data_ptr(), dt.data_ptr(), dt_t, A_log.data_ptr(), a_t, B.data_ptr(), C.data_ptr(),
        d_ptr, d_t, dt_bias.data_ptr(), b_t)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(*sizes):
    return _lib.load().gdn_ssm_prefill_workspace_size(*sizes)


def _prompt_args(x, dt, A_log, B, C, D, dt_bias, state, cu):
    if cu is None:
        raise ValueError("cu_seqlens is required")
    sizes, keep, head = _args(x, dt, A_log, B, C, D, dt_bias, state, cu, 1)
    if cu.dim() != 1 or cu.numel() < 1:
        raise ValueError("cu_seqlens must be a 1-D tensor of length num_seqs + 1")
    cu, cu_t = K.as_index("cu_seqlens", cu)
    n = cu.numel() - 1
    _, H, _, P, Ns = sizes
    if state is not None:
        if state.shape != (n, H, P, Ns):
            raise ValueError(f"state must be [{n}, {H}, {P}, {Ns}], got {tuple(state.shape)}")
        if state.dtype is not _F32:
            state = state.float()
        state = _aligned(state.contiguous())
    return sizes, n, (keep, state, cu), head + (K.ptr(state), cu.data_ptr(), cu_t)


def prefill_recurrent(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, *, check=False):
    """The scan token by token (one launch): any head size, the independent check of the
    chunked kernel."""
    (T, H, G, P, Ns), n, keep, head = _prompt_args(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens)
    lib, dev = _lib.load(), x.device
    with K.on_device(dev):
        status = _status.address(dev.index)
        out = torch.empty_like(keep[0][0])
        new_state = torch.empty(n, H, P, Ns, dtype=_F32, device=dev)
        rc = lib.gdn_ssm_prefill_recurrent_fwd(
            *head, out.data_ptr(), new_state.data_ptr(), T, n, H, G, P, Ns, status,
            K.stream_handle(dev))
        if rc:
            _lib.check(rc, "gdn_ssm_prefill_recurrent_fwd")
        if check:
            _status.finish(dev.index)
    return out, new_state


def prefill(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens, *, check=False):
    """The scan over packed prompts: (output [T, H, P] bf16, new_state [N, H, P, Ns] fp32).
    A ``cu_seqlens`` that leaves [0, T] or decreases, or a bounded wait that gave up, raises
    GDNError at the next call on the device, or at this one with ``check=True`` (which
    synchronises)."""
    (T, H, G, P, Ns), n, keep, head = _prompt_args(x, dt, A_log, B, C, D, dt_bias, state, cu_seqlens)
    lib, dev = _lib.load(), x.device
    with K.on_device(dev):
        status = _status.address(dev.index)
        out = torch.empty_like(keep[0][0])
        new_state = torch.empty(n, H, P, Ns, dtype=_F32, device=dev)
        nbytes = _workspace_bytes(T, n, H, G, P, Ns)
        # of this call alone: calls on several streams and captured graphs share nothing
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = lib.gdn_ssm_prefill_fwd(
            *head, out.data_ptr(), new_state.data_ptr(), T, n, H, G, P, Ns, K.ptr(ws), nbytes,
            status, K.stream_handle(dev))
        if rc:
            _lib.check(rc, "gdn_ssm_prefill_fwd")
        if check:
            _status.finish(dev.index)
    return out, new_state


def _decode(x, dt, A_log, B, C, D, dt_bias, state, inplace):
    (T, H, G, P, Ns), keep, head = _args(x, dt, A_log, B, C, D, dt_bias, state, None, 2)
    dtype = _F32
    if state is not None:
        if state.shape != (T, H, P, Ns):
            raise ValueError(f"state must be {[T, H, P, Ns]}, got {tuple(state.shape)}")
        if not inplace:
            if state.dtype is not _F32 and state.dtype is not _BF16:
                state = state.float()
            state = _aligned(state.contiguous())
        dtype = state.dtype
    lib, dev = _lib.load(), x.device
    with K.on_device(dev):
        out = torch.empty_like(keep[0])
        new_state = state if inplace else (
            torch.empty(T, H, P, Ns, dtype=dtype, device=dev) if state is None
            else torch.empty_like(state))
        rc = lib.gdn_ssm_decode_fwd(
            *head, K.ptr(state), _CODES[dtype], out.data_ptr(), new_state.data_ptr(), T, H, G, P, Ns,
            K.stream_handle(dev))
    if rc:
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
