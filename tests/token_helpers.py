"""The token operators in float64, with error bounds for the kernels' results.

Every reference returns (value, bound): the bound is a worst case over the roundings that the
kernels make, element by element.  Notation: u = eps / 2 of the storage type (one rounding of
a stored value or of a 16-bit MFMA operand), f = 2^-24 (one float32 rounding); a float32 sum of n
terms in any order is off by at most n f times the sum of the terms' magnitudes.  TINY covers
results below fp16's normal range, where a rounding is off by up to half of 2^-24.
"""
import math

import torch

F = 2.0 ** -24
TINY = 2.0 ** -25
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def d(t):
    return None if t is None else t.detach().double()


def check(got, want, bound, what):
    """Every element within its bound; non-finite values equal."""
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    same = torch.where(fin, torch.zeros_like(want), want)
    assert torch.equal(torch.where(torch.isnan(want), torch.isnan(got), got == same) | fin, torch.ones_like(fin)), \
        f"{what}: non-finite values differ"
    err = torch.where(fin, (got - want).abs(), torch.zeros_like(want))
    bad = ~(err <= bound.expand_as(err)) & fin
    if bad.any():
        i = tuple(int(j) for j in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements outside their bound, first at {i}: "
                             f"got {float(got[i])}, want {float(want[i])} +- {float(bound.expand_as(err)[i])}")


# ---- linear ---------------------------------------------------------------------------------
def act64(z, act):
    if act == "silu":
        return z * torch.special.expit(z)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    return z.clamp(min=0) if act == "relu" else z


def slope64(z, act):
    if act == "silu":
        s = torch.special.expit(z)
        return s + z * s * (1 - s)
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return (z > 0).double() if act == "relu" else torch.ones_like(z)


def _final(v, err, dt):
    """Bound of a value known to `err` and rounded once to dt."""
    return err + half_step(dt) * (v.abs() + err) + TINY


def linear(x, w, b, act, res):
    """(y, bound, z, bound).  z is a sum of k products and the bias; an activation's slope is at
    most 1.13, and its float32 evaluation (a few correctly rounded steps of magnitudes below |z| + 1)
    adds at most 16 f (|z| + 1)."""
    dt = x.dtype
    xd, wd = d(x).reshape(-1, x.shape[-1]), d(w)
    z = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if b is not None:
        z = z + d(b)
        mag = mag + d(b).abs()
    ez = (x.shape[-1] + 8) * F * mag
    y = act64(z, act)
    ey = 1.13 * ez + (16 * F * (z.abs() + 1) if act != "none" else 0)
    if res is not None:
        r = d(res).reshape(-1, w.shape[0])
        r = r[torch.arange(z.shape[0], device=z.device) % r.shape[0]]
        y, ey = y + r, ey + F * (y.abs() + r.abs())
    shape = (*x.shape[:-1], w.shape[0])
    return (y.reshape(shape), _final(y, ey, dt).reshape(shape), z.reshape(shape), _final(z, ez, dt).reshape(shape))


def linear_grads(dy, x, w, act, z, res_rows=0):
    """[(gradient, bound)] for x, w, the bias and the residual, at the stored z.  dz is rounded to
    the storage type when there is an activation; its slope (below 1.13) is off by at most 32 f (1 + |z|)."""
    dt, k, n = x.dtype, x.shape[-1], w.shape[0]
    dyd, xd, wd = d(dy).reshape(-1, n), d(x).reshape(-1, k), d(w)
    m = xd.shape[0]
    zd = d(z).reshape(-1, n) if z is not None else torch.zeros_like(dyd)
    dz = dyd * slope64(zd, act)
    raw = dyd.abs() * 32 * F * (1 + zd.abs()) if act != "none" else torch.zeros_like(dz)
    edz = raw + (half_step(dt) * (dz.abs() + raw) + TINY if act != "none" else 0)
    out = []
    dx = dz @ wd
    out.append((dx.reshape(x.shape), _final(dx, edz @ wd.abs() + (n + 8) * F * ((dz.abs() + edz) @ wd.abs()), dt).reshape(x.shape)))
    dw = dz.t() @ xd
    out.append((dw, _final(dw, edz.t() @ xd.abs() + (m + 8) * F * ((dz.abs() + edz).t() @ xd.abs()), dt)))
    db = dz.sum(0)
    out.append((db, raw.sum(0) + (m + 8) * F * (dz.abs() + raw).sum(0)))  # + the rounding of its own dtype
    if res_rows:
        idx = torch.arange(m, device=dy.device) % res_rows
        dr = torch.zeros(res_rows, n, dtype=torch.float64, device=dy.device).index_add_(0, idx, dyd)
        mag = torch.zeros_like(dr).index_add_(0, idx, dyd.abs())
        out.append((dr, _final(dr, (m / res_rows + 9) * F * mag, dt)))
    return out


# ---- layer norm --------------------------------------------------------------------------------
def _norm_parts(x, eps):
    xd = d(x)
    c = x.shape[-1]
    mean = xd.mean(-1, keepdim=True)
    r = ((xd - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    h = (xd - mean) * r
    # the mean is off by at most c f mean|x|, a difference by f |x - mean| more; r relatively by (c + 8) f
    emean = (c + 2) * F * xd.abs().mean(-1, keepdim=True)
    eh = r * emean + h.abs() * (c + 16) * F
    return mean, r, h, emean, eh


def layer_norm(x, w, b, eps):
    _, r, h, _, eh = _norm_parts(x, eps)
    wd = d(w) if w is not None else torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
    bd = d(b) if b is not None else torch.zeros_like(wd)
    y = h * wd + bd
    return y, _final(y, (eh + 2 * F * h.abs()) * wd.abs() + 2 * F * y.abs() + F * bd.abs(), x.dtype)


def layer_norm_grads(dy, x, w, eps):
    c = x.shape[-1]
    _, r, h, _, eh = _norm_parts(x, eps)
    wd = d(w) if w is not None else torch.ones(c, dtype=torch.float64, device=x.device)
    dyd = d(dy)
    g = dyd * wd
    mg, mgh = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = r * (g - mg - h * mgh)
    emgh = (g.abs() * eh).mean(-1, keepdim=True) + (c + 8) * F * (g * h).abs().mean(-1, keepdim=True)
    e = r * ((c + 8) * F * g.abs().mean(-1, keepdim=True) + eh * mgh.abs() + (h.abs() + eh) * emgh +
             8 * F * (g.abs() + mg.abs() + (h * mgh).abs()))
    e = e + (c + 16) * F * dx.abs()
    m = max(x.numel() // c, 1)
    f2 = lambda t: t.reshape(-1, c)  # noqa: E731
    dw, ew = f2(dyd * h).sum(0), f2(dyd.abs() * eh).sum(0) + (m + 8) * F * f2((dyd * h).abs() + dyd.abs() * eh).sum(0)
    db, eb = f2(dyd).sum(0), (m + 8) * F * f2(dyd.abs()).sum(0)
    return [(dx, _final(dx, e, x.dtype)), (dw, ew), (db, eb)]


# ---- attention ---------------------------------------------------------------------------------
def attention(q, k, v, scale=None, causal=False, lengths=None, q_lengths=None, do=None, grad_tiny=(TINY, TINY)):
    """{"o": (o, bound), "lse": .., "dq": .., "dk": .., "dv": ..} by batch element and head.

    A score is off by es = (D + 8) f scale sum|q k| + 4 f |s| (its product, the scaling into a
    power of two, the maximum subtracted); P relatively by es of its row's largest, twice (numerator
    and denominator), n f for the denominator's sum and 8 f per key block for the rescaling; for the
    16-bit types the P and dS that enter a product are rounded once more (u, TINY in fp16's subnormal
    range; the backward pass's own, of P and of dS: grad_tiny).  delta inherits o's bound."""
    dt, u = q.dtype, half_step(q.dtype)
    b, nq, h, dd = q.shape
    nk, hk = k.shape[1], k.shape[2]
    rep, scale = h // hk, dd ** -0.5 if scale is None else scale
    u = u if dt != torch.float32 else 0.0
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=q.device)  # noqa: E731
    o, eo = z(q), z(q) + TINY
    lse = torch.full((b, h, nq), -math.inf, dtype=torch.float64, device=q.device)
    else_ = torch.zeros_like(lse)
    out = {"o": (o, eo), "lse": (lse, else_)}
    if do is not None:
        gr = {n: (z(t), z(t)) for n, t in (("dq", q), ("dk", k), ("dv", v))}
        out.update(gr)
    for i in range(b):
        kl = nk if lengths is None else min(max(int(lengths[i]), 0), nk)
        ql = nq if q_lengths is None else min(max(int(q_lengths[i]), 0), nq)
        if not kl or not ql:
            continue
        hid = torch.zeros(ql, kl, dtype=torch.bool, device=q.device)
        if causal:
            hid = torch.ones(ql, kl, dtype=torch.bool, device=q.device).triu(kl - ql + 1)
        for j in range(h):
            Q, K, V = d(q[i, :ql, j]), d(k[i, :kl, j // rep]), d(v[i, :kl, j // rep])
            s = (Q @ K.t()) * scale
            es = (dd + 8) * F * scale * (Q.abs() @ K.abs().t()) + 4 * F * s.abs()
            s = s.masked_fill(hid, -math.inf)
            es = es.masked_fill(hid, 0)
            L = torch.logsumexp(s, 1, keepdim=True)
            seen = L > -math.inf
            P = torch.exp(s - torch.where(seen, L, torch.zeros_like(L)))
            row = es.amax(1, keepdim=True)
            rel = 2 * row + (kl + 32) * F + 8 * F * (kl / 32 + 1)
            O = P @ V
            tiny = TINY * (~hid).double() if u else torch.zeros_like(P)
            eO = (rel + u) * (P @ V.abs()) + tiny @ V.abs() + (rel + 4 * F) * O.abs()
            fO = _final(O, eO, dt)
            o[i, :ql, j], eo[i, :ql, j] = O, fO
            lse[i, j, :ql] = L[:, 0]
            else_[i, j, :ql] = torch.where(seen, rel + 4 * F * (L.abs() + 1), torch.zeros_like(L))[:, 0]
            if do is None:
                continue
            G = d(do[i, :ql, j])
            dP = G @ V.t()
            edP = (dd + 8) * F * (G.abs() @ V.abs().t())
            delta = (G * O).sum(1, keepdim=True)
            edelta = (G.abs() * fO).sum(1, keepdim=True) + (dd + 8) * F * (G.abs() * (O.abs() + fO)).sum(1, keepdim=True)
            relP = es + rel + torch.where(seen, 8 * F * (L.abs() + 1), torch.zeros_like(L))
            tP, tS = ((~hid).double() * (t if u else 0) for t in grad_tiny)
            eP = P * (relP + u) + tP
            dS = P * (dP - delta)
            edS = P * ((relP + 2 * F) * (dP - delta).abs() + edP + edelta)
            edS = edS + u * (dS.abs() + edS) + tS
            dQ, dK, dV = scale * (dS @ K), scale * (dS.t() @ Q), P.t() @ G
            n = kl + ql + 16
            add = {"dq": (i, slice(0, ql), j), "dk": (i, slice(0, kl), j // rep), "dv": (i, slice(0, kl), j // rep)}
            for name, val, err in (("dq", dQ, scale * (edS @ K.abs() + n * F * ((dS.abs() + edS) @ K.abs()))),
                                   ("dk", dK, scale * (edS.t() @ Q.abs() + rep * n * F * ((dS.abs() + edS).t() @ Q.abs()))),
                                   ("dv", dV, eP.t() @ G.abs() + rep * n * F * ((P + eP).t() @ G.abs()))):
                gr[name][0][add[name]] += val
                gr[name][1][add[name]] += err
    if do is not None:
        for name in ("dq", "dk", "dv"):
            out[name] = (gr[name][0], _final(gr[name][0], gr[name][1], dt))
    return out
