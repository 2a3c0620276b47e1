"""The network-block operators in float64 on the CPU, with bounds for what their float32 sums and single roundings may add.

Every function returns (value, error bound).  u = half a step of the type, relative; SUB half its smallest step, absolute;
F = 2^-24, half a step of float32.  A sum of K products in float32 is off by at most (K + 8) F times the sum of their
magnitudes, in whatever order it is made."""
import math

import torch

F = 2.0 ** -24
# one activation in float32 or by the hardware's exp2 and reciprocal: relative, for the |g| < 16 of the tests.  The
# argument of exp carries a relative 2 F to 4 F, times its size (up to 16 * (1 + .045 * 256) for gelu, where the result
# itself vanishes); the functions add a few F.
ACT = {torch.float32: 64 * F, torch.bfloat16: 512 * F, torch.float16: 512 * F}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2, float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps / 2


def act(kind, g, alpha=0.2):
    if kind == "lrelu":
        d = torch.where(g > 0, 1.0, alpha).to(g.dtype)
        return g * d, d
    if kind == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if kind == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def mm(a, ea, b, eb=None):
    """(a +- ea) @ (b +- eb) summed in float32."""
    v, mag = a @ b, a.abs() @ b.abs()
    e = ea @ b.abs() if ea is not None else 0
    if eb is not None:
        e = e + (a.abs() + (ea if ea is not None else 0)) @ eb
    return v, e + (a.shape[1] + 8) * F * (mag + e)


def rounded(v, e, dtype):
    u, sub = half_step(dtype)
    return v, e + u * (v.abs() + e) + sub


def gated(x, wg, wu, kind, alpha, dtype):
    """(gate, its error), (up, its error), (h, its error), none of them rounded."""
    g, eg = mm(x, None, wg)
    u, eu = mm(x, None, wu)
    a, _ = act(kind, g, alpha)
    ea = 1.2 * eg + ACT[dtype] * (a.abs() + 1.2 * eg) + 1e-37        # |act'| < 1.13
    h = a * u
    return (g, eg), (u, eu), (h, ea * (u.abs() + eu) + a.abs() * eu + 2 * F * h.abs())


def ffn(x, wg, wu, wd, kind, alpha, dtype):
    (g, eg), (u, eu), (h, eh) = gated(x, wg, wu, kind, alpha, dtype)
    out = rounded(*mm(*rounded(h, eh, dtype), wd), dtype)
    return {"out": out, "pre_gate": (g, eg), "pre_up": (u, eu)}


def ffn_back(x, wg, wu, wd, g, u, dout, kind, alpha, dtype):
    a, d = act(kind, g, alpha)
    ea, ed = ACT[dtype] * a.abs() + 1e-37, 2 * ACT[dtype] * (d.abs() + a.abs()) + 1e-37
    dh, edh = mm(dout, None, wd.t())

    def through(f, ef):                  # dh * f, rounded
        v = dh * f
        return rounded(v, edh * (f.abs() + ef) + dh.abs() * ef + 3 * F * v.abs(), dtype)

    dg, du = through(u * d, ed * u.abs()), through(a, ea)
    h = rounded(a * u, ea * u.abs() + 2 * F * (a * u).abs(), dtype)
    both = mm(torch.cat([dg[0], du[0]], 1), torch.cat([dg[1], du[1]], 1), torch.cat([wg, wu], 1).t())
    return {"dx": rounded(*both, dtype),
            "dw_gate": rounded(*mm(x.t(), None, *dg), dtype),
            "dw_up": rounded(*mm(x.t(), None, *du), dtype),
            "dw_down": rounded(*mm(h[0].t(), h[1].t(), dout), dtype)}


# ---- norms.  One float32 operation adds F times the magnitudes it combines; a row's sum is a tree of at most 32 + 6 + 16
# ---- levels, twice in a row where a mean goes before, and a dozen products follow: 160 F covers a chain. ------------------
N = 160 * F


def hat(kind, v, ev, eps):
    """Normed rows without a weight, the rows' factor, the error of both (the factor's relative)."""
    d = v.shape[1]
    c, ec = v, ev + N * v.abs()
    if kind == "layer":
        c = v - v.mean(1, keepdim=True)
        ec = ev + ev.mean(1, keepdim=True) + N * (v.abs() + v.abs().mean(1, keepdim=True))
    q = c.pow(2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(q + eps)
    er = ((c.abs() * ec).mean(1, keepdim=True) + ec.pow(2).mean(1, keepdim=True)) / (q + eps) + N
    assert d == v.shape[1]
    return c * r, r, ec * r * (1 + er) + (c * r).abs() * er, er


def rows_of(gate, rpg, T):
    return gate[torch.arange(T) // rpg]


def norm(x, b, gate, rpg, w_post, w_pre, kind, eps, rs, bs, off, dtype):
    """y and n; b, gate, w_post, w_pre may be None."""
    one = torch.ones(x.shape[1], dtype=torch.float64)
    v, ev = rs * x, 2 * F * (rs * x).abs()
    if b is not None:
        bh, _, eb, _ = hat(kind, b, torch.zeros_like(b), eps)
        f = (one if w_post is None else w_post + off) * bs
        f = f * (rows_of(gate, rpg, x.shape[0]) if gate is not None else torch.ones_like(x))
        v = v + bh * f
        ev = ev + eb * f.abs() + 6 * F * ((bh * f).abs() + v.abs())
    vh, _, evh, _ = hat(kind, v, ev, eps)
    w = one if w_pre is None else w_pre + off
    n, en = vh * w, evh * w.abs() + 4 * F * (vh * w).abs()
    u, sub = half_step(dtype)
    # n's rounding leaves off at most u of it, that part's own rounding u of that
    return {"y": rounded(v, ev, dtype), "n": rounded(n, en, dtype), "n_and_lo": (n, en + 2 * u * u * (n.abs() + en) + 2 * sub)}


def through_hat(kind, z, ez, vh, evh, r, er):
    """The gradient of a row's hat."""
    p = (z * vh).mean(1, keepdim=True)
    ep = (ez * vh.abs() + (z.abs() + ez) * evh).mean(1, keepdim=True) + N * (z * vh).abs().mean(1, keepdim=True)
    t = z - vh * p
    et = ez + vh.abs() * ep + evh * (p.abs() + ep) + N * (z.abs() + (vh * p).abs())
    if kind == "layer":
        m = z.mean(1, keepdim=True)
        em = ez.mean(1, keepdim=True) + N * z.abs().mean(1, keepdim=True)
        t, et = t - m, et + em + N * m.abs()
    return t * r, (et * (1 + er) + t.abs() * er) * r + 2 * F * (t * r).abs()


def norm_back(y, b, gate, rpg, w_post, w_pre, dy, dn, kind, eps, rs, bs, off, dtype):
    """Gradients; every array but y and one of dy, dn may be None.  y is what the call reads (exact)."""
    T, d = y.shape
    one = torch.ones(d, dtype=torch.float64)
    out = {}
    t, et = (dy, torch.zeros_like(y)) if dy is not None else (torch.zeros_like(y), torch.zeros_like(y))
    sums = (T + 24) * F                         # a column's sum over the rows

    def total(v, e, rows=None):
        e = e + sums * (v.abs() + e)
        if rows is None:
            return rounded(v.sum(0), e.sum(0), dtype)
        n = -(-T // rows)
        pad = torch.zeros(2, n * rows, d, dtype=torch.float64)
        pad[0, :T], pad[1, :T] = v, e
        return rounded(pad[0].view(n, rows, d).sum(1), pad[1].view(n, rows, d).sum(1), dtype)

    if dn is not None:
        yh, r, eyh, er = hat(kind, y, torch.zeros_like(y), eps)
        w = one if w_pre is None else w_pre + off
        out["dw_pre"] = total(dn * yh, dn.abs() * eyh + F * (dn * yh).abs())
        g, eg = through_hat(kind, dn * w, 2 * F * (dn * w).abs(), yh, eyh, r, er)
        t, et = t + g, et + eg + F * (t + g).abs()
    out["dx"] = rounded(rs * t, abs(rs) * et + 2 * F * (rs * t).abs(), dtype)
    if b is not None:
        bh, r, ebh, er = hat(kind, b, torch.zeros_like(b), eps)
        w = one if w_post is None else w_post + off
        G = rows_of(gate, rpg, T) if gate is not None else torch.ones_like(y)
        q, eq = bs * t, abs(bs) * et + 2 * F * (bs * t).abs()
        out["dgate"] = total(q * bh * w, (eq * (bh.abs() + ebh) + q.abs() * ebh) * w.abs() + 4 * F * (q * bh * w).abs(), rpg)
        out["dw_post"] = total(q * G * bh, (eq * (bh.abs() + ebh) + q.abs() * ebh) * G.abs() + 3 * F * (q * G * bh).abs())
        z = q * G * w
        g, eg = through_hat(kind, z, eq * (G * w).abs() + 4 * F * z.abs(), bh, ebh, r, er)
        out["dbranch"] = rounded(g, eg, dtype)
    return out


def check(got, want, what):
    v, e = want
    got = got.detach().cpu().double()
    assert got.shape == v.shape, (what, got.shape, v.shape)
    assert torch.isfinite(got).all(), what
    bad = (got - v).abs() > e
    if bad.any():
        i = tuple(int(k) for k in torch.nonzero(bad)[0])
        raise AssertionError("%s: %d of %d values beyond their bound; at %r: %.9g, want %.9g +- %.3g"
                             % (what, int(bad.sum()), v.numel(), i, got[i], v[i], e[i]))
