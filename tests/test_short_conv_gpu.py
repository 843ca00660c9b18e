"""The short convolution on the GPU against its definition in fp64."""
import pytest
import torch

from flashinfer_bench_tma_thrust_b200 import GDNError, prefill, short_conv
from oracle import gdn_oracle
from oracle.ssm_oracle import BF16, assert_within, conv

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_status():
    short_conv.reset_device_status()
    yield
    short_conv.reset_device_status()


def make(lengths, C, W, state=True, bias=True, wdtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    T, N = sum(lengths), len(lengths)
    x = torch.randn(T, C, generator=g).bfloat16()
    w = (torch.randn(C, W, generator=g) * W ** -0.5).to(wdtype)
    b = torch.randn(C, generator=g).to(wdtype) if bias else None
    s = torch.randn(N, W - 1, C, generator=g).bfloat16() if state else None
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return x, w, b, s, cu


def dev(*ts):
    return [t.cuda() if isinstance(t, torch.Tensor) else t for t in ts]


def check(got, new_state, x, w, b, s, bounds, activation="silu", split=None, norm=None, eps=1e-6):
    split = split or (x.shape[1],)
    norm = norm or (False,) * len(split)
    want, states = conv(x, w, b, s, bounds, activation, split, norm, eps)
    got = got if isinstance(got, tuple) else (got,)
    for i, (o, (v, e)) in enumerate(zip(got, want)):
        assert o.dtype == torch.bfloat16 and o.is_contiguous()
        assert_within(o, v, e, f"section {i}", rounding=BF16)
    assert torch.equal(new_state.cpu().double(), states)


LENGTHS = [[1], [2], [3], [5, 0, 1, 2, 3, 4, 0, 7], [64, 1, 65], [200], [0, 0], [7, 130, 9, 33]]


@pytest.mark.parametrize("lengths", LENGTHS)
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("state", [True, False])
def test_prompt(lengths, W, state):
    x, w, b, s, cu = make(lengths, 264, W, state)
    got, ns = short_conv.prefill(*dev(x, w, b, s, cu), check=True)
    check(got, ns, x, w, b, s, cu.tolist())


@pytest.mark.parametrize("C,split,norm", [
    (512, (128, 128, 256), (True, True, False)),
    (512, (128, 384), (False, True)),
    (1160, (128, 1024, 8), (True, True, False)),
    (357, (128, 229), (True, False)),            # odd channels: no vector access
    (333, (100, 33, 200), (False, False, False)),
    (1, (1,), (False,)),
    (2304, (1024, 1024, 256), (True, False, True)),
])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_sections_and_norms(C, split, norm, wdtype):
    x, w, b, s, cu = make([3, 70, 1], C, 4, wdtype=wdtype, seed=C)
    got, ns = short_conv.prefill(*dev(x, w, b, s, cu), split=split, l2norm=norm)
    check(got, ns, x, w, b, s, cu.tolist(), split=split, norm=norm)
    xt = x[:9, None]
    st = torch.randn(9, 3, C, generator=torch.Generator().manual_seed(1)).bfloat16()
    got, ns = short_conv.decode(*dev(xt, w, b, st), split=split, l2norm=norm)
    assert got[0].shape == (9, 1, split[0])
    check(got, ns, x[:9], w, b, st, list(range(10)), split=split, norm=norm)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), -3e38, 3e38])
def test_one_channel_leaves_its_neighbours_alone(bad):
    """A channel's extreme value reaches that channel's outputs, of its own and the next W - 1
    tokens, and nothing else; silu of a value far below zero is next to nothing."""
    x, w, b, s, cu = make([40], 256, 4, bias=False)
    w[:, :3], w[:, 3] = 0, 1
    want, _ = short_conv.prefill(*dev(x, w, None, s, cu))
    for ch in (6, 7):
        y = x.clone()
        y[20, ch] = bad
        for cols in (256, 255):  # in vectors, and channel by channel
            got, _ = short_conv.prefill(*dev(y[:, :cols].contiguous(), w[:cols], None,
                                             s[..., :cols].contiguous(), cu), check=True)
            other = torch.ones(40, cols, dtype=torch.bool)
            other[20:24, ch] = False
            assert torch.equal(got.cpu()[other], want[:, :cols].cpu()[other])
            v = got[20, ch].item()
            if bad != bad:
                assert v != v
            elif bad < 0:
                assert abs(v) < 1e-16
            else:
                assert v == pytest.approx(bad, rel=2 ** -8)  # (bf16's own rounding of it)


FAR = 2.0 ** -14  # silu's exponent |v| log2(e) < 150 rounds by 2^-17, its exponential by 2 ulp


def passed_through(values, C=256):
    """Arguments of a convolution that hands each channel its input (one tap of one)."""
    w = torch.zeros(C, 2)
    w[:, 1] = 1
    x = values.bfloat16()
    return dev(x, w, None, None, torch.tensor([0, x.shape[0]], dtype=torch.int32))


@pytest.mark.parametrize("rows", [1, 50, 1300])
def test_silu_far_below_zero(rows):
    """silu is v e^v where e^-v is large: relative accuracy down to the least normal number, also
    next to ordinary channels, and zero behind it."""
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 256, generator=g) * 3
    far = torch.rand(rows, 256, generator=g) < 0.3
    x = torch.where(far, -40 - 51 * torch.rand(rows, 256, generator=g), x).bfloat16()
    x[:, 3], x[-1, 200], x[0, 77] = -200, float("-inf"), -3e38
    got = short_conv.prefill(*passed_through(x))[0]
    v = x.double()
    want = torch.where(v > -700, v * torch.sigmoid(v), 0.0)
    assert_within(got, want, FAR * want.abs(), "silu", rounding=BF16)
    one = short_conv.decode(x[:, None].cuda(), *passed_through(x)[1:2])[0]
    assert torch.equal(one[:, 0], got)


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("rows", [3, 1300])
@pytest.mark.parametrize("activation", ["silu", None])
def test_norm_of_heads_whose_squares_leave_fp32(eps, rows, activation):
    """Heads of values whose squares underflow or overflow: the norm is still that of the head."""
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 256, generator=g)
    if activation:
        x[0::3] = -44 - 30 * torch.rand(x[0::3].shape, generator=g)
    else:
        x[0::3] *= 1e-25
    x[1::3, :128] *= 1e30
    x = x.bfloat16()
    args = passed_through(x)
    got = short_conv.prefill(*args, activation=activation, l2norm=True, eps=eps)[0]
    v = x.double()
    v = (v * torch.sigmoid(v) if activation else v).unflatten(1, (-1, 128))
    e = torch.tensor(eps).double()  # (as fp32 has it)
    want = (v / (v.pow(2).sum(-1, keepdim=True) + e).sqrt()).flatten(1)
    # twice silu's error (value and norm) and the norm's own 140 roundings of a sum
    assert_within(got, want, (2 * FAR + 140 * 2.0 ** -24) * want.abs(), "normed", rounding=BF16)
    one = short_conv.decode(x[:, None].cuda(), args[1], activation=activation, l2norm=True, eps=eps)
    assert (one[0][:, 0].double() - got.double()).abs().le(2.0 ** -7 * got.double().abs()).all()


def test_zero_head_norm_and_eps():
    """A head of zeros stays zero; eps enters under the root."""
    x, w, _, _, cu = make([5], 256, 4, bias=False, seed=3)
    x[:, :128] = 0
    got, ns = short_conv.prefill(*dev(x, w), None, None, cu.cuda(), l2norm=True, eps=0.25)
    check(got, ns, x, w, None, None, cu.tolist(), norm=(True,), eps=0.25)
    assert (got[:, :128] == 0).all()


@pytest.mark.parametrize("activation", ["silu", None])
def test_no_bias_no_activation_3d_weight_int64(activation):
    x, w, _, s, cu = make([4, 9], 64, 4, seed=4)
    got, ns = short_conv.prefill(x.cuda(), w[:, None].cuda(), None, s.cuda(), cu.long().cuda(),
                                 activation=activation)
    check(got, ns, x, w, None, s, cu.tolist(), activation=activation)


@pytest.mark.parametrize("offset,width", [(0, 800), (8, 800), (3, 777)])
def test_strided_rows(offset, width):
    """x as a slice of wider rows: its own stride and start (aligned or not)."""
    x, w, b, s, cu = make([20, 21], 256, 4, seed=5)
    wide = torch.full((41, width), float("nan"), dtype=torch.bfloat16)
    wide[:, offset:offset + 256] = x
    view = wide.cuda()[:, offset:offset + 256]
    got, ns = short_conv.prefill(view, *dev(w, b, s, cu))
    check(got, ns, x, w, b, s, cu.tolist())
    got, ns = short_conv.decode(view[:2, None], *dev(w, b, s))
    check(got, ns, x[:2], w, b, s, [0, 1, 2])
    t = x.cuda().t().contiguous().t()            # channels not adjacent
    got, ns = short_conv.prefill(t, *dev(w, b, s, cu))
    check(got, ns, x, w, b, s, cu.tolist())


def test_prompt_in_pieces_then_tokens_equals_one_prompt():
    """A prompt cut in two with the state carried, then single tokens in place, gives the bits
    of the whole prompt."""
    x, w, b, s, cu = make([40], 512, 4, seed=6)
    x, w, b, s, cu = dev(x, w, b, s, cu)
    kw = dict(split=(128, 128, 256), l2norm=(True, True, False))
    whole, end = short_conv.prefill(x, w, b, s, cu, **kw)
    parts, st = [], s
    for lo, hi in ((0, 2), (2, 3), (3, 30)):
        o, st = short_conv.prefill(x[lo:hi], w, b, st, torch.tensor([0, hi - lo]).cuda(), **kw)
        parts.append(o)
    for t in range(30, 40):
        o, st2 = short_conv.decode_inplace(x[t:t + 1, None], w, b, st, **kw)
        assert st2 is st
        parts.append(tuple(v[:, 0] for v in o))
    for i in range(3):
        assert torch.equal(torch.cat([p[i] for p in parts]), whole[i])
    assert torch.equal(st, end)


def test_decode_without_state_and_inputs_unchanged():
    x, w, b, s, _ = make([1] * 5, 256, 4, seed=7)
    xd, wd, bd, sd = dev(x, w, b, s)
    got, ns = short_conv.decode(xd[:, None], wd, bd)
    check(got, ns, x, w, b, None, list(range(6)))
    got, ns = short_conv.decode(xd[:, None], wd, bd, sd)
    assert torch.equal(sd.cpu(), s) and torch.equal(xd.cpu(), x)
    got2, ns2 = short_conv.decode_inplace(xd[:, None], wd, bd, sd)
    assert torch.equal(got, got2) and torch.equal(ns, ns2) and ns2 is sd


def test_uncovered_rows_and_neighbours():
    """Tokens in front of and behind the sequences are not written and not read; a NaN stays in
    its own sequence, channel and the W - 1 tokens behind it."""
    x, w, b, s, _ = make([30], 256, 4, seed=8)
    x[0:3] = float("nan")
    x[25:] = float("nan")
    x[10, 7] = float("nan")
    cu = torch.tensor([3, 12, 12, 25], dtype=torch.int32)
    s3 = torch.randn(3, 3, 256, generator=torch.Generator().manual_seed(9)).bfloat16()
    xd, wd, bd, sd, cud = dev(x, w, b, s3, cu)
    # the allocator hands the freed block out again: its values show what is not written
    fill = torch.full((30, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    at = fill.data_ptr()
    del fill
    got, ns = short_conv.prefill(xd, wd, bd, sd, cud, check=True)
    want, states = conv(x, w, b, s3, cu.tolist(), True, (256,), (False,), 1e-6)
    assert_within(got, want[0][0], want[0][1], "covered", rounding=BF16)
    nan = torch.isnan(got.cpu())
    expect = torch.isnan(want[0][0])
    assert torch.equal(nan[3:25], expect[3:25])
    if got.data_ptr() == at:
        assert (got[:3] == 7).all() and (got[25:] == 7).all()
    assert torch.equal(torch.isnan(ns.cpu()), torch.isnan(states))


@pytest.mark.parametrize("cu", [[0, 5, 99], [-3, 4, 10], [0, 7, 2, 10]])
def test_bad_cu_seqlens_is_reported(cu):
    x, w, b, _, _ = make([10], 256, 4, seed=10)
    args = (*dev(x, w, b), None, torch.tensor(cu, dtype=torch.int64).cuda())
    with pytest.raises(GDNError, match="cu_seqlens"):
        short_conv.prefill(*args, check=True)
    with pytest.raises(GDNError, match="cu_seqlens"):   # sticky until cleared
        short_conv.prefill(*args)
    short_conv.reset_device_status()
    good = torch.tensor([0, 10]).cuda()
    short_conv.prefill(*dev(x, w, b), None, good, check=True)


def test_many_sequences():
    lengths = [(i * 7) % 5 for i in range(3000)]
    x, w, b, s, cu = make(lengths, 64, 4, seed=11)
    got, ns = short_conv.prefill(*dev(x, w, b, s, cu), check=True)
    check(got, ns, x, w, b, s, cu.tolist())


def test_empty_calls():
    x, w, b, s, _ = make([0, 0], 256, 4, seed=12)
    got, ns = short_conv.prefill(*dev(x, w, b, s), torch.zeros(3, dtype=torch.int32).cuda())
    assert got.shape == (0, 256) and torch.equal(ns.cpu(), s)
    got, ns = short_conv.prefill(*dev(x, w, b), None, torch.zeros(1, dtype=torch.int32).cuda())
    assert got.shape == (0, 256) and ns.shape == (0, 3, 256)
    got, ns = short_conv.decode(torch.empty(0, 1, 256, dtype=torch.bfloat16, device="cuda"),
                                *dev(w, b))
    assert got.shape == (0, 1, 256) and ns.shape == (0, 3, 256)


def test_graph_and_other_stream():
    """A captured call replayed on new inputs, and a call on a side stream, give the eager
    call's bits."""
    x, w, b, s, cu = dev(*make([33, 8], 512, 4, seed=13))
    x2 = torch.randn_like(x)
    kw = dict(split=(128, 128, 256), l2norm=(True, True, False))
    want = short_conv.prefill(x2, w, b, s, cu, **kw)
    wantd = short_conv.decode(x2[:2, None], w, b, s, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = short_conv.prefill(x2, w, b, s, cu, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = short_conv.prefill(x, w, b, s, cu, **kw)
        gotd = short_conv.decode(x[:2, None], w, b, s, **kw)
    x.copy_(x2)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, c in ((want, other), (want, got), (wantd, gotd)):
        assert all(torch.equal(u, v) for u, v in zip(a[0], c[0])) and torch.equal(a[1], c[1])


def test_feeds_gdn_prefill():
    """Convolution, split, silu and norms in front of the GDN prefill, as a layer runs them."""
    HQ, HV = 2, 4
    lengths = [70, 0, 9]
    C = (2 * HQ + HV) * 128
    x, w, b, s, cu = make(lengths, C, 4, seed=14)
    g = torch.Generator().manual_seed(15)
    T = sum(lengths)
    A_log = torch.log(torch.rand(HV, generator=g) * 15 + 1)
    dtb = torch.rand(HV, generator=g) * 2 - 1
    a, bb = torch.randn(T, HV, generator=g).bfloat16(), torch.randn(T, HV, generator=g).bfloat16()
    split, norm = (HQ * 128, HQ * 128, HV * 128), (True, True, False)
    (q, k, v), ns = short_conv.prefill(*dev(x, w, b, s, cu), split=split, l2norm=norm)
    out, state = prefill.kernel(q.view(T, HQ, 128), k.view(T, HQ, 128), v.view(T, HV, 128), None,
                                *dev(A_log, a, dtb, bb, cu), None, check=True)
    want, wstate = gdn_oracle.prefill(q.cpu().view(T, HQ, 128), k.cpu().view(T, HQ, 128),
                                      v.cpu().view(T, HV, 128), None, A_log, a, dtb, bb, cu)
    check((q, k, v), ns, x, w, b, s, cu.tolist(), split=split, norm=norm)
    assert ((out.float().cpu() - want.float()).abs() <= 1e-2 + 1e-2 * want.float().abs()).all()
    assert ((state.cpu() - wstate).norm() / wstate.norm()) < 1e-3


# Prompts whose tiles hold several batches of tokens: (lengths, channels, split, norm).
LONG = [
    # runs of 12 tokens (three batches), bounds inside batches and tiles
    ([700, 3, 0, 1, 995, 701], 1160, (128, 1024, 8), (True, True, False)),
    # runs of 24 (the ring of four batches comes round)
    ([1, 2500, 18, 1481], 2304, (1024, 1024, 256), (True, False, True)),
    # the rule for longer runs (32 here, eight batches)
    ([29000, 5, 1500], 128, (128,), (True,)),
    # runs of 40, odd channels (no vector access)
    ([9001, 0, 13999], 357, (128, 229), (True, False)),
]


@pytest.mark.parametrize("lengths,C,split,norm", LONG)
@pytest.mark.parametrize("W", [2, 3, 4])
def test_long_prompts(lengths, C, split, norm, W):
    x, w, b, s, cu = make(lengths, C, W, seed=C + W)
    got, ns = short_conv.prefill(*dev(x, w, b, s, cu), split=split, l2norm=norm, check=True)
    check(got, ns, x, w, b, s, cu.tolist(), split=split, norm=norm)


def test_long_prompt_of_unaligned_rows():
    lengths, C = [700, 3, 995, 702], 1160
    x, w, b, s, cu = make(lengths, C, 4, seed=41)
    wide = torch.full((2400, C + 7), float("nan"), dtype=torch.bfloat16)
    wide[:, 3:3 + C] = x
    kw = dict(split=(128, 1024, 8), l2norm=(True, True, False))
    w, b, s, cu = dev(w, b, s, cu)
    got, ns = short_conv.prefill(wide.cuda()[:, 3:3 + C], w, b, s, cu, **kw)
    want, want_ns = short_conv.prefill(x.cuda(), w, b, s, cu, **kw)
    assert all(torch.equal(u, v) for u, v in zip(got, want)) and torch.equal(ns, want_ns)


@pytest.mark.parametrize("rows", [1303, 5])
@pytest.mark.parametrize("W", [2, 3, 4])
def test_many_tokens(rows, W):
    """Several sequences per thread, the last thread with fewer: also in place."""
    C, split, norm = 1160, (128, 1024, 8), (True, True, False)
    x, w, b, s, _ = make([1] * rows, C, W, seed=rows + W)
    xd, wd, bd, sd = dev(x[:, None], w, b, s)
    got, ns = short_conv.decode(xd, wd, bd, sd, split=split, l2norm=norm)
    check(tuple(v[:, 0] for v in got), ns, x, w, b, s, list(range(rows + 1)), split=split, norm=norm)
    again, same = short_conv.decode_inplace(xd, wd, bd, sd, split=split, l2norm=norm)
    assert same is sd and torch.equal(sd, ns)
    assert all(torch.equal(u, v) for u, v in zip(got, again))


def test_bits_do_not_depend_on_packing():
    """A long prompt as a whole, among others, in pieces and token by token: the same bits, normed
    heads too."""
    C, T = 1160, 2400
    kw = dict(split=(128, 1024, 8), l2norm=(True, True, False))
    x, w, b, s, _ = make([T], C, 4, seed=42)
    x, w, b, s = dev(x, w, b, s)
    cu = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    whole, end = short_conv.prefill(x, w, b, s, cu(0, T), **kw)
    # behind another sequence of 7 tokens: other tiles, other batches
    both, _ = short_conv.prefill(torch.cat([x[:7], x]), w, b, torch.cat([s, s]), cu(0, 7, T + 7), **kw)
    assert all(torch.equal(u[7:], v) for u, v in zip(both, whole))
    parts, st = [], s
    for lo, hi in ((0, 1201), (1201, 1204), (1204, T)):
        o, st = short_conv.prefill(x[lo:hi], w, b, st, cu(0, hi - lo), **kw)
        parts.append(o)
    assert all(torch.equal(torch.cat([p[i] for p in parts]), whole[i]) for i in range(3))
    assert torch.equal(st, end)
    # every token with its own earlier rows as its state
    rows = torch.cat([s[0], x])
    before = torch.stack([rows[k:k + T] for k in range(3)], 1).contiguous()
    tokens, _ = short_conv.decode(x[:, None], w, b, before, **kw)
    assert all(torch.equal(u[:, 0], v) for u, v in zip(tokens, whole))


def test_prompts_past_2_31_elements():
    """x and its sections of more than 2^31 elements: the last sequence as it is alone."""
    T, C, last = 270000, 8192, 2000
    g = torch.Generator("cuda").manual_seed(43)
    x = torch.randn(T, C, generator=g, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(C, 4, generator=g, device="cuda") / 2
    assert (T - last) * C > 2 ** 31
    cu = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got, ns = short_conv.prefill(x, w, None, None, cu(0, T - last, T), l2norm=True, check=True)
    want, end = short_conv.prefill(x[T - last:], w, None, None, cu(0, last), l2norm=True, check=True)
    assert torch.equal(got[T - last:], want) and torch.equal(ns[1], end[0])
