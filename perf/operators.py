"""Cases that measure the short causal convolution and the selective state space scan.

Four operators: each of the two for packed prompts (`cu_seqlens`) and for one new token per
sequence. `run` computes them in their plain form (elementary torch operations in fp32,
rounded once at the end), or, where `own` is true, through the package's entry points.

With W taps, a sequence's inputs u_t (its W - 1 earlier inputs first, zeros without a state):

    convolution   c_t = bias + sum_k weight[:, k] u_{t-W+1+k},  y_t = silu(c_t),
                  sections of the channels returned apart; a section that is normalised has
                  each head of 128 channels divided by sqrt(sum of squares + 1e-6)
    scan          d = softplus(dt + dt_bias), g = exp(-exp(A_log) d)
                  S <- g S + d x (outer) B,  y = S C + D x       (S is [P, N] per head)
"""
import math

import torch

own = False

L2_EPS = 1e-6
CHUNK = 128  # tokens per chunk of the scan's plain form


def listed():
    return [
        # one sequence's next prompt piece of a few tokens: latency
        dict(name="conv prompt 7 tokens", op="conv_prompt", lengths="7", sections="2048,2048,4096",
             normed=2, taps=4, state=True, wdtype="bf16"),
        # the packed prompts of the varlen benchmark (8 sequences), q | k | v of 16 / 32 heads
        dict(name="conv prompt qkv varlen", op="conv_prompt",
             lengths="1013,3789,2400,1777,4001,2662,3001,1036", sections="2048,2048,4096",
             normed=2, taps=4, state=True, wdtype="bf16"),
        # long prompts, x | B | C of 64 heads of 64 channels and 8 groups of 128
        dict(name="conv prompt xBC long", op="conv_prompt", lengths="32768,32768",
             sections="4096,1024,1024", normed=0, taps=4, state=False, wdtype="f32"),
        # one stream's next token: latency
        dict(name="conv token 1 stream", op="conv_token", batch=1, sections="2048,2048,4096",
             normed=2, taps=4, wdtype="bf16"),
        # a serving batch's next tokens
        dict(name="conv token 1024 streams", op="conv_token", batch=1024,
             sections="2048,2048,4096", normed=2, taps=4, wdtype="bf16"),
        # one short prompt: latency
        dict(name="scan prompt 100 tokens", op="scan_prompt", lengths="100", heads=32, groups=16,
             head_dim=128, state_dim=128, state=True, skip=True, gdtype="bf16"),
        # the packed prompts of the varlen benchmark, 16 groups and 32 heads of 128
        dict(name="scan prompt varlen", op="scan_prompt",
             lengths="1013,3789,2400,1777,4001,2662,3001,1036", heads=32, groups=16,
             head_dim=128, state_dim=128, state=True, skip=True, gdtype="bf16"),
        # one long document: few (sequence, head) chains
        dict(name="scan prompt 1 x 32768", op="scan_prompt", lengths="32768", heads=64, groups=8,
             head_dim=64, state_dim=128, state=False, skip=True, gdtype="f32"),
        # the long-context benchmark's sequences
        dict(name="scan prompt 4 x 32768", op="scan_prompt", lengths="32768,32768,32768,32768",
             heads=32, groups=16, head_dim=128, state_dim=128, state=False, skip=False,
             gdtype="bf16"),
        # one stream's next token: latency
        dict(name="scan token 1 stream", op="scan_token", batch=1, heads=32, groups=16,
             head_dim=128, state_dim=128, skip=True, sdtype="f32", gdtype="bf16"),
        # the decode benchmark's batch
        dict(name="scan token 256 streams", op="scan_token", batch=256, heads=32, groups=16,
             head_dim=128, state_dim=128, skip=True, sdtype="f32", gdtype="bf16"),
        # heads of 64 channels, a state kept in bf16
        dict(name="scan token 300 bf16 state", op="scan_token", batch=300, heads=80, groups=1,
             head_dim=64, state_dim=128, skip=True, sdtype="bf16", gdtype="f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(rng, most):
    """Ragged lengths of `most` tokens at most together; now and then an empty sequence."""
    total = _log(rng, 1, most)
    n = _log(rng, 1, max(1, min(64, total)))
    cuts = sorted(rng.randint(0, total) for _ in range(n - 1))
    parts = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    return ",".join(str(p) for p in parts)


def _sections(rng):
    if rng.random() < 0.5:  # q | k | v: key heads, value heads of 128
        hq = rng.choice([1, 2, 4, 8, 16])
        hv = hq * rng.choice([1, 2, 4])
        return "%d,%d,%d" % (128 * hq, 128 * hq, 128 * hv), 2
    heads = rng.randint(2, 64)  # x | B | C
    bc = 64 * rng.choice([1, 2, 4, 8, 16])
    return "%d,%d,%d" % (64 * heads, bc, bc), 0


def draw(rng):
    op = rng.choice(["conv_prompt", "conv_token", "scan_prompt", "scan_prompt", "scan_token"])
    if op.startswith("conv"):
        sections, normed = _sections(rng)
        case = dict(op=op, sections=sections, normed=normed, taps=rng.choice([2, 3, 4, 4]),
                    wdtype=rng.choice(["bf16", "f32"]))
        if op == "conv_prompt":
            case.update(lengths=_lengths(rng, 32768), state=rng.random() < 0.5)
        else:
            case.update(batch=_log(rng, 1, 1024))
        return case
    groups = rng.choice([1, 2, 4, 8, 16])
    heads = groups * rng.randint(1, max(1, 32 // groups))
    case = dict(op=op, heads=heads, groups=groups, head_dim=rng.choice([64, 128]),
                state_dim=rng.choice([64, 128]), skip=rng.random() < 0.7,
                gdtype=rng.choice(["bf16", "f32"]))
    if op == "scan_prompt":
        case.update(lengths=_lengths(rng, 32768), state=rng.random() < 0.5)
    else:
        case.update(batch=_log(rng, 1, 256), sdtype=rng.choice(["f32", "f32", "bf16"]))
    return case


def _ints(text):
    return [int(v) for v in text.split(",")]


_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case)
    if "lengths" in case:
        lengths = _ints(case["lengths"])
        s["lens"] = lengths  # a program that packs prompts knows their lengths
        s["cu"] = torch.tensor([0] + lengths, device="cuda").cumsum(0).to(torch.int32)
        lead, n = (sum(lengths),), len(lengths)
    else:
        lead, n = (case["batch"], 1), case["batch"]
    if case["op"].startswith("conv"):
        widths = _ints(case["sections"])
        c, w = sum(widths), case["taps"]
        wd = _DTYPES[case["wdtype"]]
        s["split"] = widths
        s["norm"] = [i < case["normed"] for i in range(len(widths))]
        s["x"] = normal(*lead, c)
        s["weight"] = normal(c, w, scale=w ** -0.5, dtype=wd)
        s["bias"] = normal(c, scale=0.1, dtype=wd)
        s["conv_state"] = normal(n, w - 1, c) if case.get("state", True) else None
        return s
    h, p, k, grp = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
    gd = _DTYPES[case["gdtype"]]
    silu = torch.nn.functional.silu  # x, B and C come out of a convolution with silu
    s["x"] = silu(normal(*lead, h, p))
    s["B"] = silu(normal(*lead, grp, k))
    s["C"] = silu(normal(*lead, grp, k))
    s["dt"] = normal(*lead, h, scale=0.5, dtype=gd)
    u = torch.rand(h, generator=g, device="cuda")
    d = torch.exp(u * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    s["dt_bias"] = d + torch.log(-torch.expm1(-d))  # softplus(dt_bias) spans 0.001 to 0.1
    s["A_log"] = torch.log(torch.rand(h, generator=g, device="cuda") * 15 + 1)
    s["D"] = normal(h, dtype=torch.float32) if case["skip"] else None
    sd = _DTYPES[case.get("sdtype", "f32")]
    s["scan_state"] = normal(n, h, p, k, scale=0.5, dtype=sd) if case.get("state", True) else None
    return s


def _own(s):
    from flashinfer_bench_tma_thrust_b200 import short_conv, ssm

    op = s["op"]
    if op == "conv_prompt":
        return short_conv.prefill(s["x"], s["weight"], s["bias"], s["conv_state"], s["cu"],
                                  split=s["split"], l2norm=s["norm"], eps=L2_EPS)
    if op == "conv_token":
        return short_conv.decode(s["x"], s["weight"], s["bias"], s["conv_state"],
                                 split=s["split"], l2norm=s["norm"], eps=L2_EPS)
    if op == "scan_prompt":
        return ssm.prefill(s["x"], s["dt"], s["A_log"], s["B"], s["C"], s["D"], s["dt_bias"],
                           s["scan_state"], s["cu"])
    return ssm.decode(s["x"], s["dt"], s["A_log"], s["B"], s["C"], s["D"], s["dt_bias"],
                      s["scan_state"])


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"conv_prompt": _conv_prompt, "conv_token": _conv_token,
                "scan_prompt": _scan_prompt, "scan_token": _scan_token}[state["op"]](state)


# ------------------------------------------------------------------ plain forms

def _sections_out(s, y):
    """silu, the sections and their norms, each rounded once."""
    y = y * torch.sigmoid(y)
    parts = torch.split(y, s["split"], dim=-1)

    def finish(part, norm):
        if norm:
            heads = part.unflatten(-1, (-1, 128))
            heads = heads / torch.sqrt((heads * heads).sum(-1, keepdim=True) + L2_EPS)
            part = heads.flatten(-2)
        return part.to(torch.bfloat16)

    return tuple(finish(p, n) for p, n in zip(parts, s["norm"]))


def _conv_prompt(s):
    x, cu, w = s["x"], s["cu"].long(), s["taps"]
    t, c = x.shape
    n = cu.numel() - 1
    # every sequence's rows with the W - 1 rows before it, one after the other
    rows = torch.zeros(t + n * (w - 1), c, device=x.device)
    tok = torch.arange(t, device=x.device)
    seq = torch.searchsorted(cu[1:], tok, right=True)
    at = tok + (seq + 1) * (w - 1)
    rows[at] = x.float()
    before = cu[:-1, None] + torch.arange(n, device=x.device)[:, None] * (w - 1) \
        + torch.arange(w - 1, device=x.device)
    if s["conv_state"] is not None:
        rows[before.reshape(-1)] = s["conv_state"].float().reshape(-1, c)
    weight = s["weight"].float()
    y = s["bias"].float() + sum(rows[at - (w - 1) + k] * weight[:, k] for k in range(w))
    last = before + (cu[1:] - cu[:-1])[:, None]
    return _sections_out(s, y), rows[last].to(x.dtype)


def _conv_token(s):
    rows = torch.cat([s["conv_state"], s["x"]], dim=1).float()  # [B, W, C]
    y = s["bias"].float() + (rows * s["weight"].float().t()).sum(1, keepdim=True)
    return _sections_out(s, y), rows[:, 1:].to(s["x"].dtype)


def _gates(s):
    """d and log g, in 64 bits (their sums run over long chunks)."""
    v = s["dt"].double() + s["dt_bias"].double()
    d = torch.where(v > 20, v, torch.log1p(torch.exp(v)))
    return d, -torch.exp(s["A_log"].double()) * d


def _scan_prompt(s):
    x, cu, h, p, k = s["x"], s["cu"].long(), s["heads"], s["head_dim"], s["state_dim"]
    dev, t, n, rep = x.device, x.shape[0], len(s["lens"]), s["heads"] // s["groups"]
    counts = [-(-v // CHUNK) for v in s["lens"]]
    total, longest = sum(counts), max(counts + [0])
    d, lg = _gates(s)
    lens = cu[1:] - cu[:-1]
    ends = ((lens + CHUNK - 1) // CHUNK).cumsum(0)  # chunks up to the sequence's end
    first = ends - (lens + CHUNK - 1) // CHUNK
    # the tokens of each chunk; places behind a sequence's end point at row t, which is zero
    chunk = torch.arange(total, device=dev)
    seq = torch.searchsorted(ends, chunk, right=True)
    tok = (cu[seq] + (chunk - first[seq]) * CHUNK)[:, None] + torch.arange(CHUNK, device=dev)
    tok = torch.where(tok < cu[seq + 1][:, None], tok, t)

    def rows(v):
        return torch.cat([v, v.new_zeros(1, *v.shape[1:])])[tok]

    xc = rows(x).float().permute(0, 2, 1, 3)                                  # [nc, H, L, P]
    bc = rows(s["B"]).float().permute(0, 2, 1, 3).repeat_interleave(rep, 1)   # [nc, H, L, N]
    cc = rows(s["C"]).float().permute(0, 2, 1, 3).repeat_interleave(rep, 1)
    dc = rows(d).permute(0, 2, 1)                                             # [nc, H, L]
    cum = rows(lg).permute(0, 2, 1).cumsum(-1)
    # what each chunk adds to the state, and what the whole chunk leaves of it
    f = (dc * torch.exp(cum[..., -1:] - cum)).float()
    add = (xc * f[..., None]).transpose(-1, -2) @ bc                          # [nc, H, P, N]
    left = torch.exp(cum[..., -1]).float()
    # the state before each chunk: a recurrence over the chunks of all sequences side by side
    st = x.new_zeros(n, h, p, k, dtype=torch.float32) if s["scan_state"] is None \
        else s["scan_state"].float().clone()
    into = torch.empty(total + 1, h, p, k, device=dev)
    for i in range(longest):
        live = first + i < ends
        at = torch.where(live, first + i, total)
        into[at] = st
        at = at.clamp(max=max(total - 1, 0))
        st = torch.where(live[:, None, None, None], left[at][..., None, None] * st + add[at], st)
    del add
    # inside the chunk
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=dev).tril()
    decay = (cum[..., :, None] - cum[..., None, :]).float()
    m = torch.exp(decay.masked_fill(~lower, -torch.inf)) * dc.float()[..., None, :]
    y = (m * (cc @ bc.transpose(-1, -2))) @ xc
    y = y + torch.exp(cum).float()[..., None] * (cc @ into[:total].transpose(-1, -2))
    if s["D"] is not None:
        y = y + s["D"][:, None, None] * xc
    out = x.new_empty(t + 1, h, p)
    out[tok] = y.permute(0, 2, 1, 3).to(x.dtype)
    return out[:t], st


def _scan_token(s):
    rep = s["heads"] // s["groups"]
    d, lg = _gates(s)
    x = s["x"].float()[:, 0]                                     # [B, H, P]
    b = s["B"].float()[:, 0].repeat_interleave(rep, 1)           # [B, H, N]
    c = s["C"].float()[:, 0].repeat_interleave(rep, 1)
    st = torch.exp(lg).float()[:, 0, :, None, None] * s["scan_state"].float() \
        + (d.float()[:, 0, :, None] * x)[..., None] * b[:, :, None, :]
    y = (st * c[:, :, None, :]).sum(-1)
    if s["D"] is not None:
        y = y + s["D"][:, None] * x
    return y[:, None].to(s["x"].dtype), st.to(s["scan_state"].dtype)


# ------------------------------------------------------------------ 64 bits, from the definition

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"].startswith("conv"):
            return _exact_conv(s)
        return _exact_scan(s)


def _exact_conv(s):
    """One sequence after the other: its rows behind its W - 1 earlier ones, tap by tap."""
    x, w = s["x"], s["taps"]
    c = x.shape[-1]
    bounds = s["cu"].tolist() if "cu" in s else list(range(x.shape[0] + 1))
    if "cu" not in s:  # one row per sequence: all sequences at once
        old = s["conv_state"].double()
        hist = torch.cat([old, x.double()], 1)
        y = torch.einsum("bkc,ck->bc", hist, s["weight"].double()) + s["bias"].double()
        return _exact_sections(s, y[:, None]), hist[:, 1:]
    outs, states = [], []
    for n in range(len(bounds) - 1):
        mine = x[bounds[n]:bounds[n + 1]].double()
        old = mine.new_zeros(w - 1, c) if s["conv_state"] is None else s["conv_state"][n].double()
        hist = torch.cat([old, mine])
        y = s["bias"].double().repeat(mine.shape[0], 1)
        for k in range(w):
            y.addcmul_(hist[k:k + mine.shape[0]], s["weight"].double()[:, k])
        outs.append(y)
        states.append(hist[mine.shape[0]:])
    return _exact_sections(s, torch.cat(outs)), torch.stack(states)


def _exact_sections(s, y):
    y = y / (1 + torch.exp(-y))
    outs, at = [], 0
    for width, norm in zip(s["split"], s["norm"]):
        part = y[..., at:at + width]
        at += width
        if norm:
            r = part.reshape(*part.shape[:-1], width // 128, 128)
            part = (r / (r.pow(2).sum(-1, keepdim=True) + L2_EPS).sqrt()).reshape(part.shape)
        outs.append(part)
    return tuple(outs)


def _exact_scan(s):
    """Token by token, all sequences side by side; an ended one keeps its state."""
    h, p, k, rep = s["heads"], s["head_dim"], s["state_dim"], s["heads"] // s["groups"]
    packed = "cu" in s
    x = s["x"] if packed else s["x"][:, 0]
    b, c, dt = (s[v] if packed else s[v][:, 0] for v in ("B", "C", "dt"))
    t, dev = x.shape[0], x.device
    start = s["cu"][:-1].long() if packed else torch.arange(t, device=dev)
    end = s["cu"][1:].long() if packed else start + 1
    d = torch.logaddexp(dt.double() + s["dt_bias"].double(), dt.new_zeros((), dtype=torch.float64))
    decay = torch.exp(-d * torch.exp(s["A_log"].double()))
    st = torch.zeros(start.numel(), h, p, k, dtype=torch.float64, device=dev) \
        if s["scan_state"] is None else s["scan_state"].double().clone()
    y = torch.zeros(t + 1, h, p, dtype=torch.float64, device=dev)
    for i in range(max(s["lens"]) if packed else 1):
        live = start + i < end
        at = torch.where(live, start + i, 0)
        on = live[:, None].double()
        keep = torch.where(live[:, None], decay[at], 1.0)
        st.mul_(keep[..., None, None])
        st.addcmul_((x[at].double() * (d[at] * on)[..., None])[..., None],
                    b[at].double().repeat_interleave(rep, 1)[:, :, None, :])
        cv = c[at].double().repeat_interleave(rep, 1)
        y[torch.where(live, at, t)] = torch.matmul(st, cv[..., None])[..., 0]
    y = y[:t]
    if s["D"] is not None:
        y = y + s["D"].double()[:, None] * x.double()
    return (y if packed else y[:, None]), st


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if "lengths" in case:
        lens = _ints(case["lengths"])
        t, n = sum(lens), len(lens)
    else:
        t = n = case["batch"]
    if case["op"].startswith("conv"):
        c, w = sum(_ints(case["sections"])), case["taps"]
        states = 2 if case.get("state", True) else 1
        wb = 2 if case["wdtype"] == "bf16" else 4
        return {"bytes": 2 * 2 * t * c + states * 2 * n * (w - 1) * c + wb * c * (w + 1),
                "flops": 2 * w * t * c}
    h, p, k = case["heads"], case["head_dim"], case["state_dim"]
    gb = 2 if case["gdtype"] == "bf16" else 4
    sb = 2 if case.get("sdtype") == "bf16" else 4
    states = 2 if case.get("state", True) else 1
    # the recurrence's own operations: decay, outer product and readout of each state element
    return {"bytes": 2 * 2 * t * h * p + 2 * 2 * t * case["groups"] * k + gb * t * h
            + states * sb * n * h * p * k, "flops": 5 * t * h * p * k}
