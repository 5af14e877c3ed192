"""64-bit CPU oracle of the sequence operators (``horizonnet_amd.sequence``), written from their definitions, one step after the other.

Next to each result it carries a bound of what float32 arithmetic may add to it, by running error analysis: every rounded operation adds
at most ``u = 2**-24`` of its result and errors already there are carried by the same linear maps as the values."""
import math

import numpy as np
import torch

U = 2.0 ** -24


def rounding(dtype):
    """Half a step of the stored type, relative."""
    return torch.finfo(dtype).eps / 2


def recurrence(f, v, o, h0, lengths, direction, dy=None, dlast=None, eps=16 * U):
    """-> {"y", "last"[, "df", "dv", "do", "dh0"]} of float64 tensors, and the same keys of absolute bounds.  `eps`: relative error of a gate
    (exponential, reciprocal, product) with one further product; it is spent once per step."""
    T, B, C = f.shape
    if direction == "both":
        c = C // 2
        cut = lambda t, s: None if t is None else t[..., s]  # noqa: E731
        a, ea = recurrence(*(cut(t, slice(0, c)) for t in (f, v, o, h0)), lengths, "forward", cut(dy, slice(0, c)), cut(dlast, slice(0, c)), eps)
        b, eb = recurrence(*(cut(t, slice(c, C)) for t in (f, v, o, h0)), lengths, "reverse", cut(dy, slice(c, C)), cut(dlast, slice(c, C)), eps)
        return {k: torch.cat([a[k], b[k]], -1) for k in a}, {k: torch.cat([ea[k], eb[k]], -1) for k in ea}
    f, v = f.double(), v.double()
    a, rest = torch.sigmoid(f), torch.sigmoid(-f)
    s, srest = (torch.ones_like(f), torch.zeros_like(f)) if o is None else (torch.sigmoid(o.double()), torch.sigmoid(-o.double()))
    live = torch.ones(T, B, 1, dtype=torch.bool) if lengths is None else (torch.arange(T)[:, None] < lengths[None].clamp(0, T))[..., None]
    zero = torch.zeros(())
    h = torch.zeros(B, C, dtype=torch.float64) if h0 is None else h0.double()
    m = torch.zeros_like(h)
    order = list(range(T)) if direction == "forward" else list(range(T - 1, -1, -1))
    hs, ms, before, mbefore = (torch.zeros(T, B, C, dtype=torch.float64) for _ in range(4))
    for t in order:
        before[t], mbefore[t] = h, m
        n = a[t] * h + rest[t] * v[t]
        e = a[t] * m + eps * (a[t] * h.abs() + (rest[t] * v[t]).abs() + n.abs())
        h, m = torch.where(live[t], n, h), torch.where(live[t], e, m)
        hs[t], ms[t] = h, m
    got = {"y": torch.where(live, s * hs, zero.double()), "last": h}
    off = {"y": torch.where(live, s * ms + eps * (s * hs).abs(), zero.double()), "last": m}
    if dy is not None or dlast is not None:
        dy = torch.zeros_like(f) if dy is None else dy.double()
        dy = torch.where(live, dy, zero.double())
        e = torch.zeros(B, C, dtype=torch.float64) if dlast is None else dlast.double()
        me = torch.zeros_like(e)
        df, dv, do, xf, xv, xo = (torch.zeros_like(f) for _ in range(6))
        for t in reversed(order):
            dh = dy[t] * s[t] + e
            md = me + eps * ((dy[t] * s[t]).abs() + dh.abs())
            gap = before[t] - v[t]
            df[t], dv[t], do[t] = dh * gap * a[t] * rest[t], dh * rest[t], dy[t] * hs[t] * s[t] * srest[t]
            xf[t] = (md * gap.abs() + dh.abs() * (mbefore[t] + U * (before[t].abs() + v[t].abs()))) * a[t] * rest[t] + 4 * eps * df[t].abs()
            xv[t] = md * rest[t] + 2 * eps * dv[t].abs()
            xo[t] = dy[t].abs() * s[t] * srest[t] * ms[t] + 4 * eps * do[t].abs()
            e = torch.where(live[t], a[t] * dh, e)
            me = torch.where(live[t], a[t] * md + eps * (a[t] * dh).abs(), me)
        z = lambda t: torch.where(live, t, zero.double())  # noqa: E731
        got.update(df=z(df), dv=z(dv), do=z(do), dh0=e)
        off.update(df=z(xf), dv=z(xv), do=z(xo), dh0=me)
    return got, off


def activation(z, name):
    """-> value, slope, bound of the slope's own slope."""
    if name == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    if name == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), 0.8
    p = torch.sigmoid(z)
    return (p, p * torch.sigmoid(-z), 0.1) if name == "sigmoid" else (z * p, p * (1 + z * torch.sigmoid(-z)), 0.5)


def linear(x, wg, wu, bg, bu, name, dy=None):
    """-> {"y"[, "dx", "dwg", "dwu", "dbg", "dbu"]} and absolute bounds: a sum of n products in float32, in any order, is off by at most
    (n + 2) u sum |terms|; the activation and its slope add 32 u of themselves and what their argument is off; dg and du are rounded to the
    inputs' type before the products of the backward pass."""
    half = rounding(x.dtype) if x.dtype != torch.float32 else 0.0
    x, wg, wu = x.double(), wg.double(), wu.double()
    K, F, M = x.shape[1], wg.shape[0], x.shape[0]
    g, u = x @ wg.t(), x @ wu.t()
    mg, mu = (K + 2) * U * (x.abs() @ wg.abs().t()), (K + 2) * U * (x.abs() @ wu.abs().t())
    if bg is not None:
        g = g + bg.double()
    if bu is not None:
        u = u + bu.double()
    mg, mu = mg + U * g.abs(), mu + U * u.abs()
    a, slope, bend = activation(g, name)
    ma, ms = 1.2 * mg + 32 * U * a.abs(), bend * mg + 32 * U * (1 + g.abs()) * (slope != 0)
    if name == "gelu":
        ma = ma + 32 * U * (g / (1 + g.abs())).abs()          # (the distribution function is below 1 to 32 u; |z| cdf(z) is at most |z|)
    if name == "relu":
        ms = (g.abs() <= mg).double()
    got, off = {"y": a * u}, {"y": ma * u.abs() + a.abs() * mu + ma * mu + 2 * U * (a * u).abs()}
    if dy is None:
        return got, off
    dy = dy.double()
    du, dg = dy * a, dy * u * slope
    xdu = dy.abs() * ma + 2 * U * du.abs()
    xdg = dy.abs() * (mu * slope.abs() + u.abs() * ms + mu * ms) + 4 * U * dg.abs()
    rdu, rdg = xdu + half * (du.abs() + xdu), xdg + half * (dg.abs() + xdg)
    got.update(dx=dg @ wg + du @ wu, dwg=dg.t() @ x, dwu=du.t() @ x, dbg=dg.sum(0), dbu=du.sum(0))
    off.update(dx=rdg @ wg.abs() + rdu @ wu.abs() + (2 * F + 2) * U * (dg.abs() @ wg.abs() + du.abs() @ wu.abs()),
               dwg=rdg.t() @ x.abs() + (M + 2) * U * (dg.abs().t() @ x.abs()), dwu=rdu.t() @ x.abs() + (M + 2) * U * (du.abs().t() @ x.abs()),
               dbg=xdg.sum(0) + (M + 2) * U * dg.abs().sum(0), dbu=xdu.sum(0) + (M + 2) * U * du.abs().sum(0))
    return got, off


def dropout_keep(n, p, seed, start=0):
    """bool [n]: which elements start .. start + n - 1 are kept."""
    with np.errstate(over="ignore"):
        x = np.arange(start, start + n, dtype=np.uint64) + np.uint64(seed * 0x9E3779B97F4A7C15 % 2 ** 64)
        for factor in (0xFF51AFD7ED558CCD, 0xC4CEB9FE1A85EC53):
            x = (x ^ (x >> np.uint64(33))) * np.uint64(factor)
        x ^= x >> np.uint64(33)
    return torch.from_numpy((x & np.uint64(0xFFFFFFFF)) >= np.uint64(int(float(np.float32(p)) * 2 ** 32)))


def dropout(x, p, seed, residual=None):
    """-> y and its bound: the factor 1 / (1 - p) is off by 2 u, its product and the sum by u each."""
    p32 = float(np.float32(p))
    t = torch.where(dropout_keep(x.numel(), p, seed).view(x.shape), x.double() / (1 - p32), torch.zeros((), dtype=torch.float64))
    y = t if residual is None else t + residual.double()
    return y, 4 * U * t.abs() + U * y.abs()
