"""The sequence operators from their definitions in float64 on the CPU, and how far a float32 evaluation rounded once
to the result's type may be from them.

U is the unit roundoff of float32 (2^-24).  Every bound below adds up, rounding by rounding, what the operator's
float32 arithmetic can lose against the exact formula; ``rounded`` adds the final rounding to the result's type (half a
step: finfo.eps / 2 relative, and half the smallest subnormal)."""
import math

import torch

U = 2.0 ** -24


def rounded(value, bound, dtype):
    info = torch.finfo(dtype)
    return bound * (1 + info.eps) + info.eps / 2 * value.abs() + info.smallest_normal * info.eps / 2


def check(got, value, bound, what=""):
    """got within rounded(bound) of value everywhere; NaN and infinities in the same places."""
    got = got.detach().cpu()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    g = got.double()
    fine = torch.isfinite(value)
    assert torch.equal(torch.isnan(g), torch.isnan(value)), f"{what}: NaN in other places"
    inf = torch.isinf(value)
    assert torch.equal(g[inf], value[inf]), f"{what}: infinities differ"
    off = (g - value).abs()[fine]
    limit = rounded(value, bound, got.dtype)[fine]
    if off.numel():
        worst = int(torch.argmax(off - limit))
        assert bool((off <= limit).all()), f"{what}: {off[worst]:.3e} off, {limit[worst]:.3e} allowed"


def act(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu":
        return 0.5 * x * torch.erfc(-x / math.sqrt(2.0))
    return x


def act_bound(x, y, bound, name):
    """What an error ``bound`` of x becomes behind the activation, and the activation's own.

    relu: slope <= 1.  silu: slope <= 1.1; exp of an argument rounded to |x| U, one unit in the last place of exp and
    of the reciprocal, two roundings: (|x| + 8) U |y|.  gelu: slope <= 1.13; 1 + erf is formed near 1 for negative x,
    so its error is absolute: 4 units (erf to 2, the sum to 1, the argument) of |x| U, and 4 U |y| for the products."""
    if name == "silu":
        return 1.1 * bound + (x.abs() + 8) * U * y.abs()
    if name == "gelu":
        return 1.13 * bound + 8 * U * x.abs() + 4 * U * y.abs()
    return bound


def valid_frames(lengths, n, frames):
    return [frames] * n if lengths is None else [max(0, min(frames, int(t))) for t in lengths]


# ----------------------------------------------------------------------------------------------------------- group norm
def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, lengths=None):
    x = x.double()
    c = x.shape[-1]
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    per = c // groups
    frames = x.shape[1] if x.dim() > 2 else 1
    for i, t in enumerate(valid_frames(lengths, x.shape[0], frames)):
        rows = (x[i, :t] if x.dim() > 2 else x[i:i + 1]).reshape(-1, c)
        if rows.shape[0] == 0:
            continue
        out, off = torch.empty_like(rows), torch.empty_like(rows)
        # a thread takes at most every row of the clip, one after the other; then a few joins
        steps = min(rows.shape[0], 512) + 16
        for g in range(groups):
            cols = slice(g * per, (g + 1) * per)
            part = rows[:, cols]
            m = part.mean()
            v = ((part - m) ** 2).mean()
            r = 1 / torch.sqrt(v + eps)
            # running mean: each step adds at most U (|mean| + 2 |d|) / 1, averaged over the steps: steps / 2 of it
            dm = U * steps * (m.abs() + (part - m).abs().max())
            # each square to 4 U, each addition U: (steps + 4) U of the sum; the mean's error twice in the deviation
            dv = (steps + 8) * U * v + 2 * dm * torch.sqrt(v) + dm * dm
            dr = 0.5 * dv / (v + eps) + 4 * U
            n = (part - m) * r
            s = n * w[cols] + b[cols]
            e = w[cols].abs() * (r * (dm + U * (part - m).abs()) + n.abs() * (dr + 2 * U)) + U * s.abs()
            out[:, cols] = act(s, activation)
            off[:, cols] = act_bound(s, out[:, cols], e, activation)
        if x.dim() > 2:
            y[i, :t], bound[i, :t] = out.reshape(x[i, :t].shape), off.reshape(x[i, :t].shape)
        else:
            y[i], bound[i] = out[0], off[0]
    return y, bound


# --------------------------------------------------------------------------------------------------- causal convolution
def causal_conv1d(x, weight, bias=None, activation=None, state=None, lengths=None, reverse=False):
    """(y, bound, state): the state is copied, never computed."""
    n, frames, c = x.shape
    k = weight.shape[1]
    w = weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    y, bound = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    last = torch.empty((n, k - 1, c), dtype=x.dtype)
    for i, t in enumerate(valid_frames(lengths, n, frames)):
        part = x[i, :t].flip(0) if reverse else x[i, :t]
        past = torch.zeros((k - 1, c), dtype=x.dtype) if state is None else state[i]
        line = torch.cat([past, part])
        last[i] = line[t:]
        line = line.double()
        terms = torch.stack([w[:, j] * line[j:j + t] for j in range(k)])
        s = terms.sum(0) + b
        e = (k + 1) * U * (terms.abs().sum(0) + b.abs())          # k fused steps, the largest partial sum below this
        out = act(s, activation)
        e = act_bound(s, out, e, activation)
        y[i, :t], bound[i, :t] = (out.flip(0), e.flip(0)) if reverse else (out, e)
    return y, bound, last


# ------------------------------------------------------------------------------------------------------- selective scan
def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, dt_softplus=False, state=None, lengths=None,
                   reverse=False):
    """(y, bound, state, bound of the state), frame after frame in float64."""
    n, frames, c = x.shape
    m = A.shape[1]
    B, C = (v.unsqueeze(2) if v.dim() == 3 else v for v in (B, C))
    per = c // B.shape[2]
    a = A.double()
    y, bound = torch.zeros(x.shape, dtype=torch.float64), torch.zeros(x.shape, dtype=torch.float64)
    ends, end_bounds = torch.zeros((n, c, m), dtype=torch.float64), torch.zeros((n, c, m), dtype=torch.float64)
    skip = torch.zeros(c, dtype=torch.float64) if D is None else D.double()
    for i, t in enumerate(valid_frames(lengths, n, frames)):
        h = torch.zeros((c, m), dtype=torch.float64) if state is None else state[i].double()
        e = torch.zeros_like(h)
        top = h.abs()
        for j in (range(t - 1, -1, -1) if reverse else range(t)):
            raw = dt[i, j].double()
            d = raw + (0 if dt_bias is None else dt_bias.double())
            # the sum dt + bias is rounded; softplus adds 16 U relative of its value
            de = U * d.abs()
            if dt_softplus:
                d = torch.logaddexp(d, torch.zeros_like(d))
                de = de + 16 * U * d
            b = B[i, j].double().repeat_interleave(per, 0)
            cc = C[i, j].double().repeat_interleave(per, 0)
            xx = x[i, j].double()
            p = torch.exp(d[:, None] * a)
            u = (d * xx)[:, None] * b
            new = p * h + u
            # decay: exponent off by |A| de and two roundings, exp2 to two units; input: de |x B| and two roundings; one
            # fused sum.  A recording scanned in runs joins them with exp(A S), S the sum of a run's steps: each addition
            # of S is off by U S, which its factor exp(-|A| S) turns into at most 0.37 U of the state it carries over.
            e = p * e + p * h.abs() * (a.abs() * de[:, None] + 3 * U * (d[:, None] * a).abs() + 2 * U)
            e = e + (de * xx.abs())[:, None] * b.abs() + 2 * U * u.abs() + U * new.abs()
            top = torch.maximum(top, new.abs())
            e = e + 0.37 * U * top
            h = new
            s = (cc * h).sum(1) + skip * xx
            f = (cc.abs() * e).sum(1) + (m + 4) * U * ((cc * h).abs().sum(1) + (skip * xx).abs())
            if z is not None:
                zz = z[i, j].double()
                g = act(zz, "silu")
                f = g.abs() * f + act_bound(zz, g, 0, "silu") * s.abs() + U * (g * s).abs()
                s = s * g
            y[i, j], bound[i, j] = s, f
        ends[i], end_bounds[i] = h, e
    return y, bound, ends, end_bounds
