"""64-bit oracles of the short causal convolution and the state space scan — TEST
INFRASTRUCTURE ONLY.

Each returns the exact values of the definition (tap by tap, token by token, fp64) and, beside
each, a bound on what fp32 arithmetic may be off by. The bounds follow the operations: a
product or sum rounds by at most u = 2^-24 of its value, so a value computed from terms of
absolute sum A is off by at most (number of operations) u A, and an error E in a state that
decays by g is carried on as g E.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24
BF16 = 2.0 ** -8      # rounding to bf16: at most half a step, relative to the value


def _bounds(cu):
    return [int(v) for v in cu.tolist()]


def conv(x, weight, bias, state, bounds, activation, split, l2norm, eps):
    """x [T, C] over the sequences [bounds[n], bounds[n+1]). Returns ([(section, bound)],
    new_state). Rows of no sequence are NaN."""
    t, c = x.shape
    w = weight.shape[1]
    x, weight = x.double().cpu(), weight.double().cpu()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double().cpu()
    y = torch.full((t, c), float("nan"), dtype=torch.float64)
    mag = torch.zeros(t, c, dtype=torch.float64)
    states = torch.zeros(len(bounds) - 1, w - 1, c, dtype=torch.float64)
    for n in range(len(bounds) - 1):
        lo, hi = bounds[n], max(bounds[n], bounds[n + 1])
        old = torch.zeros(w - 1, c, dtype=torch.float64) if state is None else state[n].double().cpu()
        hist = torch.cat([old, x[lo:hi]])
        states[n] = hist[hi - lo:]
        for i in range(hi - lo):
            terms = hist[i:i + w] * weight.t()
            y[lo + i] = terms.sum(0) + b
            mag[lo + i] = terms.abs().sum(0) + b.abs()
    # W + 1 roundings of the sum; silu has a slope of at most 1.1 and costs about 8 more
    err = 16 * U * mag
    if activation:
        y = y * torch.sigmoid(y)
    out, at = [], 0
    for width, norm in zip(split, l2norm):
        v, e = y[:, at:at + width], err[:, at:at + width]
        at += width
        if norm:
            v, e = v.unflatten(1, (-1, 128)), e.unflatten(1, (-1, 128))
            r = (v.pow(2).sum(-1, keepdim=True) + eps).sqrt()
            v = v / r
            # d(y / r) <= dy / r + |y| / r * |dr| / r, |dr| <= |dy|_2; the norm's own rounding
            e = e / r + v.abs() * e.norm(dim=-1, keepdim=True) / r + 140 * U * v.abs()
            v, e = v.flatten(1), e.flatten(1)
        out.append((v, e))
    return out, states


def gates(dt, dt_bias, A_log):
    """(d, log g, relative error of d, relative error of g) of the fp32 gates. The sum v rounds
    by u |v|, which softplus hands on as at most that much of d (its relative slope is at most
    1); exp and log1p err by at most 2 u each, with two more for the sum and the branch. log g
    has the error of exp(A_log) (2 u) and of the product (u) besides; exp turns a relative
    error of its argument z into |z| times it, and adds 2 u."""
    v = (dt.double().cpu() + dt_bias.double().cpu()).clamp(min=-700.0)  # softplus(-700) = 0 here
    d = torch.nn.functional.softplus(v, threshold=1e9)
    lg = -torch.exp(A_log.double().cpu()) * d
    de = (6 + v.abs()) * U
    return d, lg, de, lg.abs() * (de + 4 * U) + 3 * U


def scan(x, dt, A_log, B, C, D, dt_bias, state, bounds, chunk_products=False):
    """x [T, H, P]. Returns (y, y's bound, state, state's bound) in fp64; rows of no sequence
    are NaN. ``chunk_products``: the bounds of the chunked tensor-core form, whose state terms
    (fp32 products, exactly split) are summed in fp32 by a unit that may truncate, and whose
    output terms are products with one operand rounded to bf16."""
    t, h, p = x.shape
    g_, ns = B.shape[1], B.shape[2]
    rep = h // g_
    x, B, C = x.double().cpu(), B.double().cpu(), C.double().cpu()
    B, C = B.repeat_interleave(rep, 1), C.repeat_interleave(rep, 1)
    d, lg, de, ge = gates(dt, dt_bias, A_log)
    skip = torch.zeros(h, dtype=torch.float64) if D is None else D.double().cpu()
    n_seq = len(bounds) - 1
    y = torch.full((t, h, p), float("nan"), dtype=torch.float64)
    ye = torch.zeros(t, h, p, dtype=torch.float64)
    fin = torch.zeros(n_seq, h, p, ns, dtype=torch.float64)
    fe = torch.zeros(n_seq, h, p, ns, dtype=torch.float64)
    term = 64 * 2.0 ** -23 if chunk_products else 0.0
    for n in range(n_seq):
        s = torch.zeros(h, p, ns, dtype=torch.float64) if state is None else state[n].double().cpu()
        s_abs, e = s.abs(), torch.zeros_like(s)
        for i in range(bounds[n], bounds[n + 1]):
            g = torch.exp(lg[i])[:, None, None]
            add = (d[i][:, None] * x[i])[:, :, None] * B[i][:, None, :]
            s = g * s + add
            # the decayed state by g's error and two roundings, the term by d's and three
            e = g * e + (ge[i][:, None, None] + 2 * U) * g * s_abs \
                + (de[i][:, None, None] + 3 * U + term) * add.abs()
            s_abs = g * s_abs + add.abs()
            y[i] = (s * C[i][:, None, :]).sum(-1) + skip[:, None] * x[i]
            mag = (s_abs * C[i].abs()[:, None, :]).sum(-1)
            ye[i] = (e * C[i].abs()[:, None, :]).sum(-1) + (ns + 8) * U * mag \
                + 4 * U * (skip[:, None] * x[i]).abs()
            if chunk_products:
                ye[i] += (BF16 + 2.0 ** -14) * mag
        fin[n], fe[n] = s, e
    return y, ye, fin, fe


def assert_within(got, ref, bound, what, rounding=0.0):
    """|got - ref| <= rounding |ref| + bound, element by element; NaN in `ref` is not looked at."""
    got = got.detach().double().cpu().reshape(ref.shape)
    look = ~torch.isnan(ref)
    off = (got - ref).abs() - (rounding * ref.abs() + bound + 1e-38)
    bad = look & ~(off <= 0)
    if bad.any():
        i = int(torch.where(bad, torch.nan_to_num(off, nan=float("inf")), -torch.inf).argmax())
        raise AssertionError(
            f"{what}: {int(bad.sum())} of {int(look.sum())} values out of bounds; worst at flat "
            f"index {i}: got {got.flatten()[i].item():.9g}, want {ref.flatten()[i].item():.9g}, "
            f"bound {bound.flatten()[i].item():.3g}")
