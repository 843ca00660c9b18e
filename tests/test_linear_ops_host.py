"""Refusals of the short convolution and the state space scan, without a GPU: the C ABI's
checks (made before any CUDA call) and the Python entries' (made before any launch)."""
import ctypes

import pytest
import torch

from flashinfer_bench_tma_thrust_b200 import _checks, _lib, _status, short_conv, ssm

P16 = 4096  # a 16-byte aligned address that nothing reads


def _conv(lib, fn="prefill", C=256, W=4, widths=(128, 128), normed=(1, 0), T=4, N=1, wdt=1,
          cu_dt=2, act=1, ptr=P16, cu=P16, stride=256, outs=None, eps=1e-6):
    k = len(widths)
    wa, na = (ctypes.c_int32 * k)(*widths), (ctypes.c_int32 * k)(*normed)
    oa = (ctypes.c_void_p * k)(*(outs or [ptr] * k))
    if fn == "prefill":
        return lib.gdn_conv_prefill_fwd(ptr, stride, ptr, wdt, None, 0, None, cu, cu_dt, act, k,
                                        wa, na, eps, oa, ptr, T, N, C, W, None, None)
    return lib.gdn_conv_decode_fwd(ptr, stride, ptr, wdt, None, 0, None, act, k, wa, na, eps, oa,
                                   ptr, T, C, W, None)


@pytest.mark.parametrize("fn", ["prefill", "decode"])
def test_conv_abi_refusals(cuda_lib, fn):
    lib = cuda_lib
    assert _conv(lib, fn, T=-1) == -1
    assert _conv(lib, fn, W=1) == -2
    assert _conv(lib, fn, W=5) == -2
    assert _conv(lib, fn, C=0) == -2
    assert _conv(lib, fn, widths=(128, 64)) == -2            # do not sum to C
    assert _conv(lib, fn, widths=(128, 129)) == -2
    assert _conv(lib, fn, widths=(192, 64), normed=(1, 0)) == -2   # not whole heads
    assert _conv(lib, fn, widths=(64, 192), normed=(0, 1)) == -2
    assert _conv(lib, fn, widths=(256, 0), normed=(0, 0)) == -2
    assert _conv(lib, fn, widths=tuple([32] * 9), normed=tuple([0] * 9), C=288) == -1
    assert _conv(lib, fn, wdt=2) == -3
    assert _conv(lib, fn, act=2) == -1
    assert _conv(lib, fn, eps=-1.0) == -1 and _conv(lib, fn, eps=float("nan")) == -1
    assert _conv(lib, fn, ptr=None) == -1
    assert _conv(lib, fn, outs=[P16, None]) == -1
    assert _conv(lib, fn, stride=-1) == -1
    if fn == "prefill":
        assert _conv(lib, fn, cu_dt=0) == -3
        assert _conv(lib, fn, cu=None) == -1
        assert _conv(lib, fn, N=0) == 0
    else:
        assert _conv(lib, fn, T=0) == 0


def _ssm(lib, fn="decode", H=4, G=2, P=64, Ns=64, T=4, N=1, dt=(1, 0, 0, 0), sdt=0, cu_dt=2,
         ptr=P16, B=P16, cu=P16,
         out=None, ws=None, wb=0):
    head = (ptr, ptr, dt[0], ptr, dt[1], B, ptr, ptr, dt[2], ptr, dt[3])
    if fn == "decode":
        return lib.gdn_ssm_decode_fwd(*head, None, sdt, ptr, ptr, T, H, G, P, Ns, None)
    if fn == "chunked":
        return lib.gdn_ssm_prefill_fwd(*head, None, cu, cu_dt, out or ptr, ptr, T, N, H, G, P, Ns,
                                       ws, wb, None, None)
    return lib.gdn_ssm_prefill_recurrent_fwd(*head, None, cu, cu_dt, ptr, ptr, T, N, H, G, P, Ns,
                                             None, None)


@pytest.mark.parametrize("fn", ["decode", "recurrent", "chunked"])
def test_ssm_abi_refusals(cuda_lib, fn):
    lib = cuda_lib
    assert _ssm(lib, fn, T=-1) == -1
    assert _ssm(lib, fn, H=3, G=2) == -2
    assert _ssm(lib, fn, G=0) == -2
    assert _ssm(lib, fn, P=0) == -2
    assert _ssm(lib, fn, P=257) == -2
    assert _ssm(lib, fn, Ns=48) == -2
    for i in range(4):
        codes = [1, 0, 0, 0]
        codes[i] = 3
        assert _ssm(lib, fn, dt=tuple(codes)) == -3
    assert _ssm(lib, fn, ptr=None) == -1
    assert _ssm(lib, fn, B=P16 + 2) == -1       # B goes through in vectors
    if fn == "decode":
        assert _ssm(lib, fn, sdt=2) == -3
        assert _ssm(lib, fn, T=0) == 0
    else:
        assert _ssm(lib, fn, cu_dt=1) == -3
        assert _ssm(lib, fn, cu=None) == -1
        assert _ssm(lib, fn, N=0) == 0


def test_ssm_chunked_workspace_and_alignment(cuda_lib):
    """The workspace covers every segment of any lengths; a missing, small or unaligned one and
    unaligned x or out are refused."""
    lib = cuda_lib
    size = lib.gdn_ssm_prefill_workspace_size
    assert size(100, 1, 32, 16, 128, 128) == 0             # short
    assert size(32768, 8, 32, 16, 128, 128) == 0           # enough chains
    assert size(5000, 1, 4, 2, 80, 64) == 0                # token by token
    assert size(-1, 1, 4, 2, 64, 64) == 0 and size(5000, 1, 3, 2, 64, 64) == 0
    need = size(2500, 1, 2, 1, 64, 128)
    assert need == (2500 // 256 + 1) * 2 * (64 * 128 + 1) * 4  # (segments of two chunks)
    assert size(2500, 0, 2, 1, 64, 128) == 0               # no sequences
    call = dict(T=2500, N=1, H=2, G=1, P=64, Ns=128)
    assert _ssm(lib, "chunked", **call) == -5
    assert _ssm(lib, "chunked", ws=P16, wb=need - 1, **call) == -5
    assert _ssm(lib, "chunked", ws=P16 + 4, wb=need, **call) == -1
    assert _ssm(lib, "chunked", T=100, out=P16 + 2) == -1
    assert _ssm(lib, "chunked", T=0x7fffff01) == -2


@pytest.mark.parametrize("fn", ["prefill", "decode"])
def test_conv_channels_that_leave_32_bits(cuda_lib, fn):
    """Channel numbers are 32-bit and a block's last thread lies up to 1024 behind C."""
    for C in (0x7fffffff - 2047, 0x7fffffff - 1000, 0x7fffffff):
        assert _conv(cuda_lib, fn, C=C, widths=(C,), normed=(0,), stride=C) == -2


def test_scan_wait_refusals(cuda_lib):
    call = cuda_lib.gdn_selftest_scan_wait
    assert call(0, 0, P16, P16, None) == -1 and call((1 << 20) + 1, 0, P16, P16, None) == -1
    assert call(1, 0, None, P16, None) == -1 and call(1, 0, P16, None, None) == -1


def test_cpu_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        short_conv.prefill(z(4, 8, dtype=torch.bfloat16), z(8, 4), None, None,
                           z(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        short_conv.decode(z(4, 1, 8, dtype=torch.bfloat16), z(8, 4))
    x = z(4, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ssm.prefill(x, z(4, 2), z(2), z(4, 1, 16), z(4, 1, 16), None, z(2), None,
                    z(2, dtype=torch.int32))


@pytest.fixture
def any_device(monkeypatch):
    """Let CPU tensors through the device check: everything refused below is refused before
    the launch."""
    monkeypatch.setattr(_checks, "require_all", lambda device, names, tensors: None)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


CU = torch.tensor([0, 4], dtype=torch.int32)


@pytest.mark.parametrize("change,error", [
    (dict(x=_bf(4, 1, 256)), ValueError),
    (dict(x=torch.zeros(4, 256)), TypeError),
    (dict(weight=torch.zeros(255, 4)), ValueError),
    (dict(weight=torch.zeros(256, 5)), ValueError),
    (dict(weight=torch.zeros(256, 1)), ValueError),
    (dict(weight=torch.zeros(256, 4, dtype=torch.int32)), TypeError),
    (dict(bias=torch.zeros(255)), ValueError),
    (dict(state=_bf(1, 4, 256)), ValueError),
    (dict(state=_bf(2, 3, 256)), ValueError),
    (dict(state=torch.zeros(1, 3, 256)), TypeError),
    (dict(cu_seqlens=None), ValueError),
    (dict(cu_seqlens=CU.float()), TypeError),
    (dict(cu_seqlens=CU[:0]), ValueError),
    (dict(split=(128, 64)), ValueError),
    (dict(split=(256, 0)), ValueError),
    (dict(split=(32,) * 8 + (0,)), ValueError),
    (dict(split=(64, 192), l2norm=(True, False)), ValueError),
    (dict(split=(64, 128, 64), l2norm=(False, True, False)), ValueError),
    (dict(split=(128, 128), l2norm=(True,)), ValueError),
    (dict(activation="gelu"), ValueError),
    (dict(eps=-1e-6), ValueError),
    (dict(eps=float("nan")), ValueError),
])
def test_conv_prefill_refusals(any_device, change, error):
    args = dict(x=_bf(4, 256), weight=torch.zeros(256, 4), bias=None, state=None, cu_seqlens=CU)
    args.update(change)
    with pytest.raises(error):
        short_conv.prefill(**args)


def test_conv_decode_refusals(any_device):
    w = torch.zeros(256, 4)
    with pytest.raises(ValueError):
        short_conv.decode(_bf(4, 256), w)
    with pytest.raises(ValueError):
        short_conv.decode(_bf(4, 2, 256), w)
    with pytest.raises(ValueError):
        short_conv.decode(_bf(4, 1, 256), w, None, _bf(3, 3, 256))
    with pytest.raises(ValueError):
        short_conv.decode_inplace(_bf(4, 1, 256), w, None, None)
    with pytest.raises(ValueError):
        short_conv.decode_inplace(_bf(4, 1, 256), w, None, _bf(4, 3, 512)[..., ::2])


@pytest.mark.parametrize("change,error", [
    (dict(x=_bf(5, 4, 64)), ValueError),
    (dict(x=torch.zeros(4, 4, 64)), TypeError),
    (dict(x=_bf(4, 3, 64), dt=torch.zeros(4, 3)), ValueError),       # H not a multiple of G
    (dict(x=_bf(4, 4, 257)), ValueError),
    (dict(B=_bf(4, 2, 48), C=_bf(4, 2, 48)), ValueError),
    (dict(B=_bf(4, 2, 64)), ValueError),
    (dict(B=torch.zeros(4, 2, 128)), TypeError),
    (dict(dt=torch.zeros(4, 2)), ValueError),
    (dict(dt=torch.zeros(4, 4, dtype=torch.int64)), TypeError),
    (dict(A_log=torch.zeros(3)), ValueError),
    (dict(dt_bias=torch.zeros(4, 1)), ValueError),
    (dict(D=torch.zeros(4, 64)), ValueError),
    (dict(state=torch.zeros(1, 4, 128, 64)), ValueError),
    (dict(state=torch.zeros(2, 4, 64, 128)), ValueError),
    (dict(cu_seqlens=CU.float()), TypeError),
    (dict(cu_seqlens=CU[None]), ValueError),
])
def test_ssm_prefill_refusals(any_device, change, error):
    args = dict(x=_bf(4, 4, 64), dt=torch.zeros(4, 4), A_log=torch.zeros(4), B=_bf(4, 2, 128),
                C=_bf(4, 2, 128), D=None, dt_bias=torch.zeros(4), state=None, cu_seqlens=CU)
    args.update(change)
    for fn in (ssm.prefill, ssm.prefill_recurrent):
        with pytest.raises(error):
            fn(**args)


def test_ssm_decode_refusals(any_device):
    z = torch.zeros
    args = dict(x=_bf(4, 1, 4, 64), dt=z(4, 1, 4), A_log=z(4), B=_bf(4, 1, 2, 64),
                C=_bf(4, 1, 2, 64), D=None, dt_bias=z(4), state=z(4, 4, 64, 64))
    for change in (dict(x=_bf(4, 4, 64)), dict(x=_bf(4, 2, 4, 64)), dict(dt=z(4, 4)),
                   dict(state=z(3, 4, 64, 64))):
        with pytest.raises(ValueError):
            ssm.decode(**{**args, **change})
    for state in (None, z(4, 4, 64, 64, dtype=torch.float16), z(4, 4, 64, 128)[..., ::2]):
        with pytest.raises(ValueError):
            ssm.decode_inplace(**{**args, "state": state})


def test_required_tensors_that_are_none(any_device):
    z = torch.zeros
    prompt = dict(x=_bf(4, 4, 64), dt=z(4, 4), A_log=z(4), B=_bf(4, 2, 128), C=_bf(4, 2, 128), D=None,
                  dt_bias=z(4), state=None, cu_seqlens=CU)
    token = dict(x=_bf(4, 1, 4, 64), dt=z(4, 1, 4), A_log=z(4), B=_bf(4, 1, 2, 64),
                 C=_bf(4, 1, 2, 64), D=None, dt_bias=z(4), state=None)
    for name in ("dt", "A_log", "B", "C", "dt_bias"):
        for fn, args in ((ssm.prefill, prompt), (ssm.prefill_recurrent, prompt), (ssm.decode, token)):
            with pytest.raises(TypeError, match=f"^{name} must be a torch.Tensor"):
                fn(**{**args, name: None})
    with pytest.raises(TypeError, match="^weight must be a torch.Tensor"):
        short_conv.prefill(_bf(4, 256), None, None, None, CU)
    with pytest.raises(TypeError, match="^weight must be a torch.Tensor"):
        short_conv.decode(_bf(4, 1, 256), None)


def test_status_words_raise_and_name_the_cause(monkeypatch):
    words = torch.zeros(2, dtype=torch.int32)
    monkeypatch.setitem(_status._words, 99, (words, ctypes.c_int64.from_address(words.data_ptr()),
                                             words.data_ptr()))
    assert _status.address(99) == words.data_ptr()
    words[1] = 1
    with pytest.raises(_lib.GDNError, match="cu_seqlens"):
        _status.address(99)
    words[:] = torch.tensor([1, 0])
    with pytest.raises(_lib.GDNError, match="wait"):
        _status.address(99)


def _report(counts, name="ssm_chunk_kernelILi{}ELi64ELb0EEEv"):
    return "".join(f"ptxas info    : Compiling entry function '_ZN3gdn{name.format(64 + i)}' for "
                   "'sm_100a'\nptxas info    : Function properties\n    0 bytes stack frame\n"
                   f"ptxas info    : Used {n} registers, used 3 barriers\n"
                   for i, n in enumerate(counts))


def test_the_build_checks_the_registers_that_a_kernel_hands_out():
    from flashinfer_bench_tma_thrust_b200 import build

    stem = "ssm_prefill_chunked"
    other = _report([90], "ssm_chunk_kernelILi{}ELi64ELb1EEEv")  # (not one of them)
    build.check_registers(stem, _report([96] * 4) + other)
    for bad in (_report([96, 96, 88, 96]), _report([96] * 3), other, ""):
        with pytest.raises(RuntimeError, match="96 registers"):
            build.check_registers(stem, bad)
    build.check_registers("short_conv", "")
    source = (build.CSRC / f"{stem}.cu").read_text()
    assert f"kLaunchRegs = {build.LAUNCH_REGISTERS[stem][1]}," in source
