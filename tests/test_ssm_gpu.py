"""The state space scan on the GPU against its definition in fp64."""
import pytest
import torch

from flashinfer_bench_tma_thrust_b200 import GDNError, _lib, short_conv, ssm
from oracle.ssm_oracle import BF16, assert_within, scan

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status():
    ssm.reset_device_status()
    yield
    ssm.reset_device_status()


def make(lengths, H=4, G=2, P=64, Ns=64, state=True, skip=True, gdtype=torch.float32, gates="slow",
         seed=0):
    g = torch.Generator().manual_seed(seed)
    T, N = sum(lengths), len(lengths)
    silu = torch.nn.functional.silu
    x = silu(torch.randn(T, H, P, generator=g)).bfloat16()
    B = silu(torch.randn(T, G, Ns, generator=g)).bfloat16()
    C = silu(torch.randn(T, G, Ns, generator=g)).bfloat16()
    if gates == "slow":    # softplus from 0.001 to 0.1: the state lives for many tokens
        dt = (torch.randn(T, H, generator=g) * 0.5).to(gdtype)
        d = torch.exp(torch.rand(H, generator=g) * 4.6 - 6.9)
        dtb = d + torch.log(-torch.expm1(-d))
        A_log = torch.log(torch.rand(H, generator=g) * 15 + 1)
    else:                  # "fast": decays to nothing within a few tokens, also below fp32
        dt = (torch.randn(T, H, generator=g) * 3).to(gdtype)
        dtb = torch.rand(H, generator=g) * 30 - 5
        A_log = torch.log(torch.rand(H, generator=g) * 15 + 1)
    D = torch.randn(H, generator=g) if skip else None
    s = torch.randn(N, H, P, Ns, generator=g) if state else None
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return [x, dt, A_log, B, C, D, dtb, s, cu]


def dev(ts):
    return [t.cuda() if isinstance(t, torch.Tensor) else t for t in ts]


def check_prompt(got, a, chunked, bounds=None):
    out, ns = got
    assert out.dtype == torch.bfloat16 and ns.dtype == torch.float32
    y, ye, fin, fe = scan(*a[:8], bounds or a[8].tolist(), chunk_products=chunked)
    assert_within(out, y, ye, "output", rounding=BF16)
    assert_within(ns, fin, fe, "state")


LENGTHS = [[1], [2, 0, 5], [127, 1], [128], [129], [300, 0, 0, 64, 3], [0]]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("gates", ["slow", "fast"])
def test_recurrent_prompt(lengths, gates):
    a = make(lengths, gates=gates, seed=len(lengths))
    check_prompt(ssm.prefill_recurrent(*dev(a), check=True), a, False)


@pytest.mark.parametrize("lengths", LENGTHS + [[513, 40]])
@pytest.mark.parametrize("P,Ns", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("gates", ["slow", "fast"])
def test_chunked_prompt(lengths, P, Ns, gates):
    a = make(lengths, P=P, Ns=Ns, gates=gates, seed=len(lengths) + P)
    check_prompt(ssm.prefill(*dev(a), check=True), a, True)


@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (3, 3), (10, 2), (6, 2)])
@pytest.mark.parametrize("P", [64, 128])
def test_chunked_heads(H, G, P):
    """Groups of odd size: a column block of two heads with one of them missing."""
    a = make([200, 128], H=H, G=G, P=P, Ns=64, state=False, skip=False, gdtype=torch.bfloat16,
             seed=H)
    check_prompt(ssm.prefill(*dev(a), check=True), a, True)


@pytest.mark.parametrize("lengths", [[2500], [1500, 0, 1100, 7], [1024, 1024], [2049], [1100],
                                     [20000], [0, 9000, 1]])
@pytest.mark.parametrize("P,Ns", [(64, 128), (128, 64)])
def test_chunked_segments(lengths, P, Ns):
    """Few heads and long sequences: cut into segments (two launches)."""
    a = make(lengths, H=2, G=1, P=P, Ns=Ns, seed=3)
    T, N = sum(lengths), len(lengths)
    from flashinfer_bench_tma_thrust_b200 import _lib
    assert (_lib.load().gdn_ssm_prefill_workspace_size(T, N, 2, 1, P, Ns) > 0)
    check_prompt(ssm.prefill(*dev(a), check=True), a, True)


@pytest.mark.parametrize("H,lengths,length,parts", [
    (24, [1400, 600], 512, 2), (17, [1500, 900, 700], 640, 2), (32, [1000, 2000], 1024, 2)])
def test_chunked_segments_in_parts(H, lengths, length, parts):
    """More heads: the segments' states in parts, also of unequal sizes (2 and 3 chunks of 5)."""
    a = make(lengths, H=H, G=H, seed=H)
    T, N = sum(lengths), len(lengths)
    from flashinfer_bench_tma_thrust_b200 import _lib
    assert _lib.load().gdn_ssm_prefill_workspace_size(T, N, H, H, 64, 64) == \
        (T // length + N) * parts * H * (64 * 64 + 1) * 4
    check_prompt(ssm.prefill(*dev(a), check=True), a, True)


def test_chunked_uncovered_rows_and_neighbours():
    """Rows in front of, between and behind the sequences hold NaN: they reach nothing, and
    their outputs are not written."""
    a = make([400], seed=31)
    bounds = [5, 140, 140, 300]
    for i in (0, 3, 4):
        a[i][:5] = float("nan")
        a[i][300:] = float("nan")
    a[1][:5] = float("nan")
    a[1][300:] = float("nan")
    a[7] = torch.randn(3, 4, 64, 64, generator=torch.Generator().manual_seed(32))
    a[8] = torch.tensor(bounds, dtype=torch.int32)
    d = dev(a)
    for fn, chunked in ((ssm.prefill, True), (ssm.prefill_recurrent, False)):
        fill = torch.full((400, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        at = fill.data_ptr()
        del fill
        got = fn(*d, check=True)
        check_prompt(got, a, chunked, bounds)
        if got[0].data_ptr() == at:
            assert (got[0][:5] == 7).all() and (got[0][300:] == 7).all()
        assert not torch.isnan(got[0][5:300]).any() and not torch.isnan(got[1]).any()


@pytest.mark.parametrize("lengths", [[1], [2, 3], [12], [13], [4] * 9, [5] * 9, [1] * 40])
def test_short_prompts(lengths):
    """Both sides of the rule that gives short prompts to the token-by-token kernel."""
    a = make(lengths, H=3, G=1, P=64, Ns=128, seed=35)
    check_prompt(ssm.prefill(*dev(a), check=True), a, True)


def test_masked_tokens():
    """dt of -infinity: the token adds nothing and the state keeps its value; whole sequences,
    chunks and single tokens of it."""
    a = make([300, 140], seed=36)
    a[1][128:270] = float("-inf")
    a[1][300:] = float("-inf")
    for fn, chunked in ((ssm.prefill, True), (ssm.prefill_recurrent, False)):
        got = fn(*dev(a), check=True)
        check_prompt(got, a, chunked)
        assert torch.equal(got[1][1].cpu(), a[7][1])
    t = slice(300, 302)
    tok = [a[0][t, None], a[1][t, None], a[2], a[3][t, None], a[4][t, None], a[5], a[6], a[7]]
    out, ns = ssm.decode(*dev(tok))
    assert torch.equal(ns.cpu(), a[7]) and not torch.isnan(out).any()


def test_chunked_many_sequences():
    lengths = [(i * 37) % 140 for i in range(200)]
    a = make(lengths, H=2, G=1, seed=33)
    check_prompt(ssm.prefill(*dev(a), check=True), a, True)


def test_chunked_matches_recurrent_on_long_prompts():
    """The two kernels at sizes beyond the oracle: outputs within two bf16 roundings and the
    chunked form's bf16 operands, states within fp32's terms of both (relative to the whole)."""
    a = dev(make([3000, 0, 5000, 129], H=32, G=16, P=128, Ns=128, seed=34))
    o1, s1 = ssm.prefill(*a, check=True)
    o2, s2 = ssm.prefill_recurrent(*a)
    assert ((o1.double() - o2.double()).norm() / o2.double().norm()) < 2 ** -8
    assert ((s1 - s2).norm() / s2.norm()) < 64 * 2 ** -23


SIZES = [(1, 16), (8, 16), (40, 32), (64, 64), (80, 128), (128, 128), (100, 256), (256, 256), (3, 64)]


@pytest.mark.parametrize("P,Ns", SIZES)
def test_recurrent_sizes(P, Ns):
    a = make([9, 4], H=6, G=2, P=P, Ns=Ns, seed=P + Ns)
    check_prompt(ssm.prefill_recurrent(*dev(a)), a, False)


@pytest.mark.parametrize("P,Ns", SIZES)
@pytest.mark.parametrize("batch", [1, 5])
@pytest.mark.parametrize("sdtype", [torch.float32, torch.bfloat16])
def test_token(P, Ns, batch, sdtype):
    a = make([1] * batch, H=6, G=3, P=P, Ns=Ns, seed=P + Ns)
    a[7] = a[7].to(sdtype)
    tok = [a[0][:, None], a[1][:, None], a[2], a[3][:, None], a[4][:, None], a[5], a[6], a[7]]
    out, ns = ssm.decode(*dev(tok))
    assert out.shape == (batch, 1, 6, P) and ns.dtype == sdtype and ns.shape == a[7].shape
    y, ye, fin, fe = scan(*a[:8], list(range(batch + 1)))
    assert_within(out, y, ye, "output", rounding=BF16)
    assert_within(ns, fin, fe, "state", rounding=BF16 if sdtype == torch.bfloat16 else 0.0)


@pytest.mark.parametrize("gates", ["slow", "fast"])
@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (5, 5), (8, 2)])
def test_token_heads_and_gates(H, G, gates):
    a = make([1] * 3, H=H, G=G, gates=gates, gdtype=torch.bfloat16, skip=False, seed=H)
    tok = [a[0][:, None], a[1][:, None], a[2], a[3][:, None], a[4][:, None], None, a[6], a[7]]
    out, ns = ssm.decode(*dev(tok))
    y, ye, fin, fe = scan(*a[:8], [0, 1, 2, 3])
    assert_within(out, y, ye, "output", rounding=BF16)
    assert_within(ns, fin, fe, "state")
    tok[7] = None
    out, ns = ssm.decode(*dev(tok))
    y, ye, fin, fe = scan(*a[:7], None, [0, 1, 2, 3])
    assert_within(out, y, ye, "output, no state", rounding=BF16)
    assert_within(ns, fin, fe, "state, no state")


@pytest.mark.parametrize("sdtype", [torch.float32, torch.bfloat16])
def test_token_in_place_and_inputs_unchanged(sdtype):
    a = make([1] * 4, seed=21)
    a[7] = a[7].to(sdtype)
    tok = dev([a[0][:, None], a[1][:, None], a[2], a[3][:, None], a[4][:, None], a[5], a[6], a[7]])
    before = [t.clone() for t in tok]
    out, ns = ssm.decode(*tok)
    assert all(torch.equal(u, v) for u, v in zip(tok, before))
    out2, ns2 = ssm.decode_inplace(*tok)
    assert ns2 is tok[7] and torch.equal(out, out2) and torch.equal(ns, ns2)


def test_strided_and_unaligned_inputs():
    """x, B and C as slices of one wide row, at starts that 16 bytes do not divide."""
    a = make([37, 12], seed=22)
    T = 49
    wide = torch.full((T, 1 + 4 * 64 + 3 + 2 * 64 + 2 * 64 + 5), float("nan"), dtype=torch.bfloat16)
    at = [1, 1 + 256 + 3, 1 + 256 + 3 + 128]
    for i, o, w in ((0, at[0], 256), (3, at[1], 128), (4, at[2], 128)):
        wide[:, o:o + w] = a[i].reshape(T, w)
    wd = wide.cuda()
    d = dev(a)
    want = ssm.prefill(*d)
    d[0] = wd[:, at[0]:at[0] + 256].unflatten(1, (4, 64))
    d[3] = wd[:, at[1]:at[1] + 128].unflatten(1, (2, 64))
    d[4] = wd[:, at[2]:at[2] + 128].unflatten(1, (2, 64))
    got = ssm.prefill(*d)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    tok = [d[0][:5, None], d[1][:5, None], d[2], d[3][:5, None], d[4][:5, None], d[5], d[6], None]
    same = [t.contiguous() if isinstance(t, torch.Tensor) else t for t in tok]
    for u, v in zip(ssm.decode(*tok), ssm.decode(*same)):
        assert torch.equal(u, v)


@pytest.mark.parametrize("cu", [[0, 5, 99], [-3, 4, 10], [0, 7, 2, 10]])
def test_bad_cu_seqlens_is_reported(cu):
    a = make([10], state=False, seed=23)
    a[8] = torch.tensor(cu, dtype=torch.int64)
    for fn in (ssm.prefill, ssm.prefill_recurrent):
        with pytest.raises(GDNError, match="cu_seqlens"):
            fn(*dev(a), check=True)
        with pytest.raises(GDNError, match="cu_seqlens"):
            fn(*dev(a))
        ssm.reset_device_status()


def test_empty_calls():
    a = make([0, 0], seed=24)
    for fn in (ssm.prefill, ssm.prefill_recurrent):
        out, ns = fn(*dev(a))
        assert out.shape == (0, 4, 64) and torch.equal(ns.cpu(), a[7])
        out, ns = fn(*dev(a[:7]), None, torch.zeros(1, dtype=torch.int32).cuda())
        assert ns.shape == (0, 4, 64, 64)
    tok = dev([a[0][:, None], a[1][:, None], a[2], a[3][:, None], a[4][:, None], a[5], a[6],
               a[7][:0]])
    out, ns = ssm.decode(*tok)
    assert out.shape == (0, 1, 4, 64) and ns.shape == (0, 4, 64, 64)


@pytest.mark.parametrize("ptype", [torch.bfloat16, torch.float16, torch.float64])
def test_parameter_types(ptype):
    """A_log, D and dt_bias of other types: bf16 as they are, others through fp32."""
    a = make([200, 3], seed=28)
    a = [t.to(ptype) if i in (2, 5, 6) else t for i, t in enumerate(a)]
    exact = [t.float() if i in (2, 5, 6) else t for i, t in enumerate(a)]
    check_prompt(ssm.prefill(*dev(a), check=True), exact, True)
    check_prompt(ssm.prefill_recurrent(*dev(a), check=True), exact, False)
    tok = [t[:2, None] if i in (0, 1, 3, 4) else t for i, t in enumerate(a[:8])]
    out, ns = ssm.decode(*dev(tok))
    one = [t[:2] if i in (0, 1, 3, 4) else t for i, t in enumerate(exact[:8])]
    y, ye, fin, fe = scan(*one, [0, 1, 2])
    assert_within(out[:, 0], y, ye, "output", rounding=BF16)
    assert_within(ns, fin, fe, "state")


def test_tokens_without_sequences():
    """Rows that no sequence covers, as all are where there is none: nothing runs."""
    a = dev(make([700], seed=27))
    for fn in (ssm.prefill, ssm.prefill_recurrent):
        out, ns = fn(*a[:7], None, torch.zeros(1, dtype=torch.int32, device="cuda"), check=True)
        assert out.shape == (700, 4, 64) and ns.shape == (0, 4, 64, 64)


def test_large_offsets():
    """A state past 2^31 elements: the last sequences of a large batch."""
    n, H, P, Ns = 2300, 64, 128, 128
    s = torch.zeros(n, H, P, Ns, device="cuda")
    assert s.numel() > 2 ** 31
    s[-1] = torch.randn(H, P, Ns, device="cuda")
    x = torch.randn(n, 1, H, P, device="cuda").bfloat16()
    B, C = (torch.randn(n, 1, 1, Ns, device="cuda").bfloat16() for _ in range(2))
    dt, A_log, dtb = torch.randn(n, 1, H).cuda(), torch.zeros(H).cuda(), torch.zeros(H).cuda()
    out, ns = ssm.decode_inplace(x, dt, A_log, B, C, None, dtb, s.clone())
    for i in (0, n - 1):
        y, ye, fin, fe = scan(x[i], dt[i], A_log, B[i], C[i], None, dtb, s[i:i + 1], [0, 1])
        assert_within(out[i], y, ye, "output", rounding=BF16)
        assert_within(ns[i:i + 1], fin, fe, "state")


def test_layer_prompt_then_tokens():
    """The run of a layer: convolution with split, scan, then single tokens in place for both,
    against the whole text as one prompt through the definition."""
    H, G, P, Ns, W = 6, 2, 64, 64, 4
    split = (H * P, G * Ns, G * Ns)
    ch = sum(split)
    g = torch.Generator().manual_seed(25)
    total, cut = [150, 40], [140, 30]
    u = torch.randn(sum(total), ch, generator=g).bfloat16().cuda()
    w, b = (torch.randn(ch, W, generator=g) / 2).cuda(), torch.zeros(ch).cuda()
    dt = (torch.randn(sum(total), H, generator=g) * 0.5 - 3).cuda()
    A_log, D, dtb = (torch.randn(H, generator=g).cuda() for _ in range(3))
    starts = [0, total[0]]
    idx = torch.cat([torch.arange(s, s + c) for s, c in zip(starts, cut)]).cuda()
    cu = torch.tensor([0, cut[0], sum(cut)], dtype=torch.int32).cuda()

    (x, B, C), cs = short_conv.prefill(u[idx], w, b, None, cu, split=split)
    view = lambda x, B, C, lead: (x.view(*lead, H, P), B.view(*lead, G, Ns), C.view(*lead, G, Ns))  # noqa: E731
    xv, Bv, Cv = view(x, B, C, (sum(cut),))
    outs, xs = [], [(xv, Bv, Cv)]
    y, st = ssm.prefill(xv, dt[idx], A_log, Bv, Cv, D, dtb, None, cu, check=True)
    outs.append(y)
    for k in range(10):
        t = torch.tensor([s + c + k for s, c in zip(starts, cut)]).cuda()
        parts, _ = short_conv.decode_inplace(u[t][:, None], w, b, cs, split=split)
        xt, Bt, Ct = view(*parts, (2, 1))
        y, _ = ssm.decode_inplace(xt, dt[t][:, None], A_log, Bt, Ct, D, dtb, st)
        outs.append(y[:, 0])
        xs.append((xt[:, 0], Bt[:, 0], Ct[:, 0]))

    for n in range(2):
        lo, hi = (0, cut[0]) if n == 0 else (cut[0], sum(cut))
        seq = lambda parts: torch.cat([parts[0][lo:hi]] + [p[n:n + 1] for p in parts[1:]])  # noqa: E731
        xa, Ba, Ca = (seq([p[i] for p in xs]) for i in range(3))
        rows = slice(starts[n], starts[n] + total[n])
        y, ye, fin, fe = scan(xa, dt[rows], A_log, Ba, Ca, D, dtb, None, [0, total[n]],
                              chunk_products=True)
        assert_within(seq(outs), y, ye, f"sequence {n}", rounding=BF16)
        assert_within(st[n:n + 1], fin, fe, f"state {n}")


def test_graph_and_other_stream():
    a = dev(make([150, 8], seed=26))
    x2 = torch.randn_like(a[0])
    tok = lambda x: [x[:2, None], a[1][:2, None], a[2], a[3][:2, None], a[4][:2, None], a[5], a[6], a[7]]  # noqa: E731
    want, wantd = ssm.prefill(x2, *a[1:]), ssm.decode(*tok(x2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ssm.prefill(x2, *a[1:])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, gotd = ssm.prefill(*a), ssm.decode(*tok(a[0]))
    a[0].copy_(x2)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for u, v in ((want, other), (want, got), (wantd, gotd)):
        assert torch.equal(u[0], v[0]) and torch.equal(u[1], v[1])


# bf16 states in several batches per warp: 600 sequences of 8 heads, the last batch full or not
@pytest.mark.parametrize("P,Ns", [(64, 128), (100, 64), (128, 128), (256, 16), (250, 256)])
def test_token_bf16_states_in_batches(P, Ns):
    B, H, G = 600, 8, 2
    a = make([1] * B, H=H, G=G, P=P, Ns=Ns, seed=P + Ns, state=False)
    a[7] = torch.randn(B, H, P, Ns, generator=torch.Generator().manual_seed(P)).bfloat16()
    tok = dev([a[0][:, None], a[1][:, None], a[2], a[3][:, None], a[4][:, None], a[5], a[6], a[7]])
    out, ns = ssm.decode(*tok)
    assert torch.equal(tok[7].cpu(), a[7])
    some = [0, 1, 299, 598, 599]
    y, ye, fin, fe = scan(*[a[i][some] if i in (0, 1, 3, 4, 7) else a[i] for i in range(8)],
                          list(range(len(some) + 1)))
    assert_within(out[some], y, ye, "output", rounding=BF16)
    assert_within(ns[some], fin, fe, "state", rounding=BF16)
    # all of them: as one sequence alone, which takes one batch per warp (the same operations)
    for i in (7, 300, 599):
        alone = ssm.decode(*[t[i:i + 1] if k in (0, 1, 3, 4, 7) else t for k, t in enumerate(tok)])
        assert torch.equal(alone[0], out[i:i + 1]) and torch.equal(alone[1], ns[i:i + 1])
    again, same = ssm.decode_inplace(*tok)
    assert same is tok[7] and torch.equal(again, out) and torch.equal(same, ns)


@pytest.mark.parametrize("T,segments", [(400, False), (3000, True)])
@pytest.mark.parametrize("bad", ["beyond", "before", "decreasing", "all twice"])
def test_bad_bounds_in_the_chunked_kernel(T, segments, bad):
    """Bounds outside [0, T] are clamped and decreasing ones taken as empty; the call is reported,
    and after a reset the next one is right."""
    cu = {"beyond": [0, T // 2, T + 99], "before": [-3, T // 3, T], "decreasing": [0, T - 10, 20, T],
          "all twice": [0, T, 0, T]}[bad]
    a = make([T], H=2, G=1, P=64, Ns=128, state=False, seed=51)
    n = len(cu) - 1
    assert (_lib.load().gdn_ssm_prefill_workspace_size(T, n, 2, 1, 64, 128) > 0) == segments
    assert T > 4 * n + 8
    a[7] = torch.randn(n, 2, 64, 128, generator=torch.Generator().manual_seed(52))
    good = dev(a[:7] + [a[7][:1], a[8]])
    a[8] = torch.tensor(cu, dtype=torch.int64)
    d = dev(a)
    with pytest.raises(GDNError, match="cu_seqlens"):
        ssm.prefill(*d, check=True)
    with pytest.raises(GDNError, match="cu_seqlens"):   # sticky until cleared
        ssm.prefill(*good)
    ssm.reset_device_status()
    a = a[:7] + [a[7][:1], torch.tensor([0, T], dtype=torch.int32)]
    check_prompt(ssm.prefill(*good, check=True), a, True)


def test_a_wait_that_nothing_ends_gives_up():
    """The chunked kernel's bounded wait: it reports, later ones do not wait, the context lives."""
    call = _lib.load().gdn_selftest_scan_wait
    stream = torch.cuda.current_stream().cuda_stream
    for arrive in (0, 1):
        status = torch.zeros(2, dtype=torch.int32, device="cuda")
        waited = torch.full((2,), -1, dtype=torch.int64, device="cuda")
        _lib.check(call(5000, arrive, status.data_ptr(), waited.data_ptr(), stream), "scan_wait")
        torch.cuda.synchronize()
        assert status.tolist() == [1 - arrive, 0]
        # 5000 polls of 2 us at most: 10 ms, with the timer's steps of a microsecond or so besides
        assert (waited >= 0).all() and (waited <= 100e6).all()
        assert waited[arrive] > 0
        if not arrive:
            assert waited[1] < 20e3
    assert (torch.ones(8, device="cuda") * 2).sum().item() == 16


BAD = [float("nan"), float("inf"), -float("inf")]


@pytest.mark.parametrize("P,Ns,H,G", [(64, 64, 3, 1), (128, 128, 2, 2), (64, 128, 4, 2)])
@pytest.mark.parametrize("where", ["x", "B", "C", "dt"])
def test_what_is_not_finite_reaches_no_earlier_token(P, Ns, H, G, where):
    """A NaN or infinity of a token: the values of the tokens before it, of the other sequences and
    of the channels that it does not enter keep their bits; the others are not finite, as in the
    recurrence, output by output and state by state."""
    lengths = [300, 135]
    clean = make(lengths, H=H, G=G, P=P, Ns=Ns, seed=61)
    index = {"x": 0, "dt": 1, "B": 3, "C": 4}[where]
    want = ssm.prefill(*dev(clean), check=True)
    for k, j in enumerate([0, 5, 31, 32, 63, 100, 127, 128, 140, 255, 256, 299, 301, 434]):
        a = [t.clone() if isinstance(t, torch.Tensor) else t for t in clean]
        spot = a[index][j].view(-1)
        spot[(37 * k + 5) % spot.numel()] = BAD[k % 3] if where != "dt" else BAD[k % 2]
        d = dev(a)
        out, ns = ssm.prefill(*d, check=True)
        out_r, ns_r = ssm.prefill_recurrent(*d)
        ok, ok_s = torch.isfinite(out), torch.isfinite(ns)
        assert torch.equal(ok, torch.isfinite(out_r)) and torch.equal(ok_s, torch.isfinite(ns_r))
        assert not ok.all() and (where == "C" or not ok_s.all())
        lo = 0 if j < 300 else 300
        assert ok[lo:j].all() and ok[:lo].all() and (j >= 300 or ok[300:].all())
        assert torch.equal(out[ok], want[0][ok]) and torch.equal(ns[ok_s], want[1][ok_s])


@pytest.mark.parametrize("value", BAD)
def test_what_is_not_finite_in_segments_and_many_places(value):
    """The same over segments of one sequence, with many such values, several to a chunk and column."""
    clean = make([3000], H=2, G=1, P=64, Ns=128, seed=62)
    g = torch.Generator().manual_seed(63)
    a = [t.clone() if isinstance(t, torch.Tensor) else t for t in clean]
    first = torch.full((2, 64), 3000)
    for _ in range(60):
        t, h, p = (int(torch.randint(n, (1,), generator=g)) for n in (3000, 2, 64))
        a[0][t, h, p] = value
        first[h, p] = min(int(first[h, p]), t)
    want, got = ssm.prefill(*dev(clean), check=True), ssm.prefill(*dev(a), check=True)
    ok = torch.arange(3000)[:, None, None] < first
    assert torch.equal(torch.isfinite(got[0]).cpu(), ok)
    assert torch.equal(torch.isfinite(got[1]).cpu(), (first == 3000)[None, :, :, None].expand(1, 2, 64, 128))
    assert torch.equal(got[0].cpu()[ok], want[0].cpu()[ok])


def test_graphs_with_segments_beside_each_other():
    """Two captured calls with workspaces, replayed at once on two streams, and eager calls between."""
    a, b = (dev(make(L, H=2, G=1, P=64, Ns=128, seed=71)) for L in ([2500], [1500, 0, 1100]))
    want = [ssm.prefill(*v, check=True) for v in (a, b)]
    graphs, got = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, v in zip(graphs, (a, b)):
        with torch.cuda.graph(g):
            got.append(ssm.prefill(*v))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        again = ssm.prefill(*a)
    torch.cuda.synchronize()
    for u, v in ((got[0], want[0]), (got[1], want[1]), (again, want[0])):
        assert torch.equal(u[0], v[0]) and torch.equal(u[1], v[1])


def test_prompts_past_2_31_elements():
    """x and y of more than 2^31 elements: the last sequence as it is alone."""
    T, H, P, Ns, last = 140000, 128, 128, 64, 900
    g = torch.Generator("cuda").manual_seed(72)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x, B, C, dt = new(T, H, P), new(T, 1, Ns), new(T, 1, Ns), new(T, H)
    A_log, dtb = torch.zeros(H, device="cuda"), torch.full((H,), -3.0, device="cuda")
    assert x.numel() > 2 ** 31 and (T - last) * H * P > 2 ** 31
    cu = torch.tensor([0, 100, T - last, T], dtype=torch.int32, device="cuda")
    out, ns = ssm.prefill(x, dt, A_log, B, C, None, dtb, None, cu, check=True)
    tail = slice(T - last, T)
    one = torch.tensor([0, last], dtype=torch.int32, device="cuda")
    want, end = ssm.prefill(x[tail], dt[tail], A_log, B[tail], C[tail], None, dtb, None, one, check=True)
    assert torch.equal(out[tail], want) and torch.equal(ns[2], end[0])
