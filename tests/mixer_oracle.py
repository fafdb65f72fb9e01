"""Rotations, the short convolution and the scan from their definitions, in 64 bits on the host, and the error a kernel
may make."""
from __future__ import annotations

import math

import torch

# Half a step of the activation types, relative to the value, and of fp32.
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -24
# Half the step of values below the normal range (bf16's is as far down as fp32's).
SMALL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def rounded(y, mag, dtype):
    """What one rounding of y to dtype may be off by, where y itself is off by mag."""
    return U[dtype] * (y.abs() + mag) + mag + SMALL[dtype]


def rotate(x, positions, angles, layout, scale=1.0, weight=None, eps=1e-6):
    """(out, bound) of heads x [T, H, D] at positions [T] with angles [R / 2] radians a position.

    The bound: a norm's sum of D squares is off by (D / 16 + 4) U32 of itself (16 products in a lane, then a tree), its
    root by half of that; root, reciprocal and two products add 6 U32. Turns are reduced in 64 bits; as a float the rest is
    off by 2^-26 turns or 2 pi 2^-26 < 2^-23 in the angle, sine and cosine by 2^-22 more: 2^-21 of |u| + |v| with the
    products' own rounding (4 U32 = 2^-22)."""
    dtype, x = x.dtype, x.double().cpu()
    T, H, D = x.shape
    off = torch.zeros_like(x)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double().cpu()
        off = ((D / 16 + 4) / 2 + 6) * U32 * x.abs()
    angles = torch.as_tensor(angles, dtype=torch.float64).cpu()
    R = 2 * len(angles)
    a = positions.double().cpu()[:, None, None] * angles
    i = torch.arange(R // 2)
    first, second = (i, i + R // 2) if layout == "half" else (2 * i, 2 * i + 1)
    u, v = x[..., first], x[..., second]
    out, mag = x.clone(), off.clone()
    out[..., first] = scale * (u * torch.cos(a) - v * torch.sin(a))
    out[..., second] = scale * (v * torch.cos(a) + u * torch.sin(a))
    pair = scale * (u.abs() + v.abs()) * (2.0 ** -21 + 2.0 ** -22) + scale * (off[..., first] + off[..., second])
    # positions times angles in 64 bits: off by 2^-52 of the product, in the oracle and in the kernel
    pair = pair + scale * (u.abs() + v.abs()) * a.abs() * 2.0 ** -51
    mag[..., first], mag[..., second] = pair, pair
    return out, 1.01 * rounded(out, mag, dtype)


def silu(u):
    return u / (1 + torch.exp(-u))


def silu_off(u):
    """What a kernel's silu(u) may be off by itself: the exponent's product and constant are off by 2 U32 of 1.45 |u|, the
    exponential, sum, reciprocal and product by 8 U32."""
    return silu(u).abs() * (4 * u.abs() + 8) * U32


def spans(T, cu):
    return [(i, i + 1) for i in range(T)] if cu is None else list(zip(cu, cu[1:]))


def conv(x, weight, bias, state, rows, cu=None, held=None, act=True):
    """(out, bound, kept inputs) of x [T, C]: sequence i is row rows[i] of state [rows, W - 1, C]. Tokens of no sequence: nan.

    The bound: W products and sums in fp32 are off by (W + 1) U32 of the sum of their magnitudes."""
    dtype, W = x.dtype, weight.shape[1]
    x, w, state = x.double().cpu(), weight.double().cpu(), state.double().cpu().clone()
    b = torch.zeros(x.shape[1], dtype=torch.float64) if bias is None else bias.double().cpu()
    out, mag = torch.full_like(x, math.nan), torch.zeros_like(x)
    for i, ((s, e), r) in enumerate(zip(spans(len(x), cu), rows)):
        if e <= s:
            continue
        seen = torch.cat([state[r] if held is None or held[i] else torch.zeros_like(state[r]), x[s:e]])
        y, m = b.expand(e - s, -1).clone(), b.abs().expand(e - s, -1).clone()
        for j in range(W):
            y += w[:, j] * seen[j:j + e - s]
            m += (w[:, j] * seen[j:j + e - s]).abs()
        m *= (W + 1) * U32
        out[s:e], mag[s:e] = (silu(y), 1.1 * m + silu_off(y)) if act else (y, m)  # |silu'| <= 1.1
        state[r] = seen[-(W - 1):]
    return out, 1.01 * rounded(out, mag, dtype), state


def scan(x, dt, A, B, C, state, rows, cu=None, D=None, z=None, dt_bias=None, softplus=True, held=None, chunk=False):
    """(out, bound, states, their bound). Tokens of no sequence: nan.

    The bounds follow the recursion with magnitudes: M is S with every term's magnitude, E what S is off by.
      step     s = dt + bias is off by U32 |s|, softplus has slope over value at most 1 and its functions add 6 U32: the step
               is off by d = (|s| + 8) U32 of itself; a step taken as it is by U32.
      decay    exp(A dt): the exponent by |A dt| (d + U32), the function by 4 U32.
      term     dt x b: d + 3 U32.  Each sum: 2 U32 of M.
      output   N products and sums over S: (N / 4 + 8) U32 of sum |C| M, plus sum |C| E.
    In chunks of 64 (chunk), decays are exponentials of sums of up to 64 exponents: a sum of magnitude at most a = the largest
    sum over 64 tokens is off by 12 a U32 (scans of 6 steps, both ways) beside the steps' own, and terms beyond a decay
    of e^-88 vanish; the state's terms are products of parts that keep 2^-22 of them (three of 8 bits, two of 11), its 64
    sums and those of the chunk's halves 70 U32, and up to 16 runs' states that are joined 4 U32 each; the output's weights and
    states are in two parts, 2^-15 of them at most."""
    dtype = x.dtype
    T, H, P = x.shape
    N, R = B.shape[2], H // B.shape[1]
    f = lambda t: t.double().cpu()  # noqa: E731
    x, A, state = f(x), f(A), f(state).clone()
    raw = f(dt) + (0 if dt_bias is None else f(dt_bias))
    step = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30)))) if softplus else raw
    d = (raw.abs() + 8) * U32 if softplus else torch.full_like(raw, U32)
    keep = torch.exp(step * A)
    keep_off = (step * A).abs() * (d + U32) + 4 * U32
    Bs, Cs = (f(t).repeat_interleave(R, 1) for t in (B, C))
    out, mag = torch.full_like(x, math.nan), torch.zeros_like(x)
    state_off = torch.zeros_like(state)
    for i, ((s, e), r) in enumerate(zip(spans(T, cu), rows)):
        if e <= s:
            continue
        S = state[r] if held is None or held[i] else torch.zeros_like(state[r])
        M, E = S.abs(), torch.zeros_like(S)
        sums = (step[s:e] * A).abs().cumsum(0)
        window = sums.clone()
        window[64:] -= sums[:-64]
        most = window.max(0).values[:, None, None]
        for t in range(s, e):
            k, ko = keep[t][:, None, None], keep_off[t][:, None, None]
            dx = step[t][:, None] * x[t]
            term = dx[..., None] * Bs[t][:, None, :]
            S = k * S + term
            E = k * (E + ko * M) + (d[t][:, None, None] + 4 * U32) * term.abs()
            M = k * M + term.abs()
            E = E + 2 * U32 * M
            if chunk:
                extra = 1.1 * (2.0 ** -22 + (134 + 13 * most) * U32) / 64  # of M, spread over the chunk's tokens
                E = E + extra * M
            out[t] = (S * Cs[t][:, None, :]).sum(-1)
            y_mag = (M * Cs[t][:, None, :].abs()).sum(-1)
            mag[t] = (E * Cs[t][:, None, :].abs()).sum(-1) + (N / 4 + 8) * U32 * y_mag
            if chunk:
                mag[t] += (2.0 ** -15 + (200 + 13 * most[..., 0]) * U32) * y_mag + 64 * extra[..., 0] * y_mag
        if chunk:
            E = E + 64 * extra * M
        state[r], state_off[r] = S, E
    if D is not None:
        out += f(D)[:, None] * x
        mag += 2 * U32 * ((f(D)[:, None] * x).abs() + out.abs())
    if z is not None:
        z = f(z)
        mag = (mag + 2 * U32 * out.abs()) * silu(z).abs() + out.abs() * silu_off(z)
        out = out * silu(z)
    mag = torch.nan_to_num(mag)
    return out, 1.01 * rounded(out, mag, dtype), state, 1.01 * state_off + 1e-38


def check(got, want, bound, label=""):
    """got against want (float64 on the host) within bound; rows where want is nan are not looked at. A value past the type's
    largest by more than half a step is its infinity. Returns the worst share."""
    top = torch.finfo(got.dtype).max
    top += top * torch.finfo(got.dtype).eps / 4  # half a step: from here on values round to infinity
    got = got.double().cpu()
    there = ~torch.isnan(want)
    over = torch.isinf(got) & (got.sign() == want.sign()) & (want.abs() + bound >= top)
    assert (torch.isfinite(got) | over)[there].all(), f"{label}: non-finite outputs"
    assert (over | (want.abs() - bound < top))[there].all(), f"{label}: finite outputs past the type's largest"
    share = ((got - want).abs() / bound)[there & ~over]
    worst = share.max().item() if share.numel() else 0.0
    assert worst <= 1, f"{label}: off by {worst:.3g} of the bound"
    return worst
