"""The gated core's operators in 64 bits, and how far an fp32 evaluation with one final rounding may be from them."""
import math

import torch

f64 = torch.float64
EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, f64: 0.0}      # half a step, relative
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, f64: 0.0}                  # half a step below fp16's smallest normal
E32 = 2.0 ** -24
ACTS = ('none', 'relu', 'tanh', 'silu', 'gelu')


def act64(z, act):
    """(value, slope)"""
    if act == 'relu':
        return z.clamp(min=0), (z > 0).to(f64)
    if act == 'tanh':
        return torch.tanh(z), 1 / torch.cosh(z) ** 2
    if act == 'silu':
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == 'gelu':
        c = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def linear64(x, w, b=None, act='none', r=None):
    """y, its tolerance, slope and the tolerance of the slope as the backward pass sees it.
    An fp32 sum of K products is off by at most (K + 1) E32 sum |x w|; activations have slopes and curvatures of at most 1.13 and are
    themselves off by less than 16 E32 of |z| or of 1 (exp2 and reciprocal: an ulp each, the argument's scaling another, the normal
    tail 7.5e-8); the result is rounded once."""
    dt, K = x.dtype, x.shape[1]
    x, w = x.to(f64), w.to(f64)
    z = x @ w.t().contiguous()
    ez = (K + 2) * E32 * (x.abs() @ w.abs().t().contiguous())
    if b is not None:
        z = z + b.to(f64)
        ez = ez + 2 * E32 * b.to(f64).abs()
    y, slope = act64(z, act)
    tol = 1.13 * ez + (0 if act in ('none', 'relu') else 16 * E32 * torch.maximum(z.abs(), y.abs()))
    if r is not None:
        y = y + r.to(f64)
        tol = tol + E32 * y.abs()
    tol = tol * (1 + EPS[dt]) + EPS[dt] * y.abs() + TINY[dt]
    if act == 'none':
        ts = torch.zeros_like(z)
    elif act == 'relu':
        ts = (z.abs() <= ez).to(f64)                       # the gate of a pre-activation within rounding of zero is not determined
    else:
        ts = 1.13 * ez + 16 * E32 * (1 + z.abs()) + (2.0 ** -15 if dt != torch.float32 else 0)
    return y, tol, slope, ts


def linear_grads64(dy, x, w, slope, ts):
    """dx, dw, db and tolerances: dz is rounded to the storage type, sums are fp32, results are rounded once."""
    dt, (M, N) = dy.dtype, dy.shape
    dy, x, w = dy.to(f64), x.to(f64), w.to(f64)
    dz = dy * slope
    ef = dy.abs() * ts + E32 * dz.abs()                    # before dz is rounded: what db sums
    ez = ef + EPS[dt] * (dz.abs() + ef) + TINY[dt]
    mm = lambda a, b: a.contiguous() @ b.contiguous()
    dx, dw, db = mm(dz, w), mm(dz.t(), x), dz.sum(0)
    end = lambda v, e: e * (1 + EPS[dt]) + EPS[dt] * v.abs() + TINY[dt]
    az = dz.abs() + ez
    tx = end(dx, mm(ez, w.abs()) + (N + 2) * E32 * mm(az, w.abs()))
    tw = end(dw, mm(ez.t(), x.abs()) + (M + 2) * E32 * mm(az.t(), x.abs()))
    tb = end(db, ef.sum(0) + (M + 2) * E32 * (dz.abs() + ef).sum(0))
    return (dx, tx), (dw, tw), (db, tb)


def scan64(gate, value, h0, masks, dout=None, dlast=None):
    """States and gradients step by step, each with a running bound of the error: a step of the fp32 evaluation is off by at most C E32
    of its operands (gate: exp2, reciprocal and their arguments; product, sum), whatever the order in which steps are composed --
    composing (A, B) pairs applies the same factors once more, hence C = 32 instead of 16."""
    C = 32 * E32
    dt, (T, N, H) = gate.dtype, gate.shape
    g, v = gate.to(f64), value.to(f64)
    f, nf = torch.sigmoid(g), torch.sigmoid(-g)
    m = torch.ones(T, N, 1, dtype=f64, device=g.device) if masks is None else masks.to(f64).reshape(T, N, 1)
    h = torch.zeros(N, H, dtype=f64, device=g.device) if h0 is None else h0.to(f64)
    e = torch.zeros_like(h)
    drop = lambda k, t: torch.where(k == 0, torch.zeros_like(t), k * t)
    hs, es, hp, ep = [], [], [], []
    for t in range(T):
        hp.append(drop(m[t], h)), ep.append(drop(m[t].abs(), e))
        a = f[t]
        b = nf[t] * v[t]
        h = a * hp[-1] + b
        e = a * ep[-1] + C * (a * hp[-1].abs() + b.abs())
        hs.append(h), es.append(e)
    st = lambda q: torch.stack(q) if q else torch.zeros(0, N, H, dtype=f64, device=g.device)
    end = lambda x, k: k * (1 + EPS[dt]) + EPS[dt] * x.abs() + TINY[dt]
    out, eo = st(hs), st(es)
    res = dict(out=(out, end(out, eo)), last=(h, e + E32 * h.abs()))
    if dout is None:
        return res
    d, E = dout.to(f64), torch.zeros(N, H, dtype=f64, device=g.device) if dlast is None else dlast.to(f64)
    q = torch.zeros_like(E)
    dg, dv, tg, tv = [], [], [], []
    for t in range(T - 1, -1, -1):
        D = d[t] + E
        eD = q + C * (d[t].abs() + E.abs())
        w, ew = hp[t] - v[t], ep[t] + C * (hp[t].abs() + v[t].abs())
        k = f[t] * nf[t]
        dg.append(D * w * k), tg.append(k * (eD * w.abs() + (D.abs() + eD) * ew) + C * (D * w * k).abs())
        dv.append(D * nf[t]), tv.append(nf[t] * eD + C * (D * nf[t]).abs())
        E = drop(m[t], D * f[t])
        q = m[t].abs() * f[t] * eD + C * E.abs()
    dg, tg, dv, tv = (st(s[::-1]) for s in (dg, tg, dv, tv))
    res.update(dgate=(dg, end(dg, tg)), dvalue=(dv, end(dv, tv)), dh0=(E, q + E32 * E.abs()))
    return res


def check(got, ref, what):
    r, tol = ref
    assert got.shape == r.shape, (what, got.shape, r.shape)
    if got.numel() == 0:
        return
    d = (got.to(f64) - r).abs()
    over = d - tol
    i = int(over.argmax())
    assert bool((d <= tol).all()), '%s: off by %.3g at %d where %.3g is allowed (value %.6g)' % (
        what, d.flatten()[i], i, tol.flatten()[i], r.flatten()[i])
