"""Plain 64-bit forms of the block operators (group norm with an activation, gated recurrence, dropout) and bounds of how
far a kernel that computes in 32 bits may be from them.

The bounds follow the arithmetic.  U = 2^-24 is a rounding to fp32.  A result in a narrower type adds half a step of that type,
half(type) |value|.  The subnormal range of fp16 adds half its smallest step."""
import numpy as np
import torch

U = 2.0 ** -24
NONE, SILU, SIGMOID, RELU = 0, 1, 2, 3


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 1e-38


def close(got, want, err, what=""):
    """|got - want| <= err + half a step of got's type, element by element (err: of the value before that last rounding)."""
    got64, want = got.detach().double().cpu(), want.double()
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    lim = err + half(got.dtype) * (want.abs() + err) + tiny(got.dtype)
    bad = ~((got64 - want).abs() <= lim)
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got64 - want).abs() / lim).nan_to_num(9e9).max()))


def act(v, which):
    return (v, v * torch.sigmoid(v), torch.sigmoid(v), torch.clamp(v, min=0))[which]


def act_grad(v, which):
    p, q = torch.sigmoid(v), torch.sigmoid(-v)
    return (torch.ones_like(v), p * (1 + v * q), p * q, (v > 0).to(v.dtype))[which]


def _live(B, S, lengths):
    n = torch.full((B,), S) if lengths is None else lengths.clamp(0, S).long()
    return n, torch.arange(S)[None, :, None] < n[:, None, None]


def group_norm(x, gamma, beta, groups, eps, which, first, lengths=None, dy=None):
    """Everything in 64 bits, each value with its bound: {"y": (value, err), "stats": ..., "dx": ..., "dgamma": ..., "dbeta": ...}."""
    x = x.double()
    B, S, C = x.shape
    D = C // groups
    ga = torch.ones(C, dtype=torch.float64) if gamma is None else gamma.double()
    be = torch.zeros(C, dtype=torch.float64) if beta is None else beta.double()
    n, live = _live(B, S, lengths)
    x = torch.where(live, x, 0.0)
    u = torch.where(live, act(x, which), 0.0) if first else x
    eu = 8 * U * u.abs() if first else torch.zeros_like(u)                 # a sigmoid is right to a few roundings
    N = (n * D).clamp(min=1).view(B, 1, 1).double()

    def tot(v):                                  # sums over a group, [B, 1, groups]
        return v.view(B, S, groups, D).sum((1, 3)).view(B, 1, groups)

    def at(v):
        return v.repeat_interleave(D, -1)

    mean = tot(u) / N
    dev = torch.where(live, u - at(mean), 0.0)
    var = tot(dev ** 2) / N
    some = (n > 0).view(B, 1, 1)
    rstd = torch.where(some, 1 / torch.sqrt(var + eps), 0.0)
    # The mean of values of size m is right to 64 U m: at most 64 terms are added one after the other in 32 bits.  A deviation
    # carries that and its own rounding; the variance, a mean of squares, twice the deviations' share and 64 roundings.
    m = tot(u.abs()) / N
    emean = 64 * U * m + tot(eu) / N
    ed = at(emean) + eu + 2 * U * (u.abs() + at(m))
    evar = tot(torch.where(live, 2 * dev.abs() * ed + ed ** 2, 0.0)) / N + 128 * U * var
    erstd = rstd * (0.5 * evar / (var + eps) + 4 * U)
    xh = dev * at(rstd)
    exh = ed * at(rstd) + dev.abs() * at(erstd) + 2 * U * xh.abs()
    z = xh * ga + be
    ez = exh * ga.abs() + 2 * U * (z.abs() + be.abs())
    y = z if first else act(z, which)
    ey = ez if first else 1.2 * ez + 8 * U * y.abs()                       # |act'| <= 1.1 for all of them
    out = {"y": (torch.where(live, y, 0.0), torch.where(live, ey, 0.0)),
           "stats": (torch.stack([mean, rstd], -1).view(B, groups, 2), torch.stack([emean + U * mean.abs(), erstd + U * rstd], -1).view(B, groups, 2))}
    if dy is None:
        return out
    dy = torch.where(live, dy.double(), 0.0)
    post = NONE if first else which
    k = act_grad(z, post)
    dz = dy * k
    curve = {NONE: 0.0, SILU: 0.6, SIGMOID: 0.2, RELU: 0.0}                # |act''| at most
    edz = dy.abs() * (curve[post] * ez + 8 * U * (k.abs() + 1))            # silu' is a sum of terms below 1.3
    g, eg = dz * ga, edz * ga.abs() + 2 * U * (dz * ga).abs()
    c1, c2 = tot(torch.where(live, g, 0.0)) / N, tot(torch.where(live, g * xh, 0.0)) / N
    e1 = tot(torch.where(live, eg + 128 * U * g.abs(), 0.0)) / N
    e2 = tot(torch.where(live, eg * xh.abs() + g.abs() * exh + 128 * U * (g * xh).abs(), 0.0)) / N
    inner = g - at(c1) - xh * at(c2)
    einner = eg + at(e1) + exh * at(c2).abs() + xh.abs() * at(e2) + 4 * U * (g.abs() + at(c1).abs() + (xh * at(c2)).abs())
    du = at(rstd) * inner
    edu = at(rstd) * einner + at(erstd) * inner.abs() + 2 * U * du.abs()
    pre = which if first else NONE
    kp = act_grad(x, pre)
    out["dx"] = (torch.where(live, du * kp, 0.0), torch.where(live, edu * kp.abs() + du.abs() * 8 * U * (kp.abs() + 1) + 2 * U * (du * kp).abs(), 0.0))
    for name, v, e in (("dgamma", dz * xh, edz * xh.abs() + dz.abs() * exh), ("dbeta", dz, edz)):
        out[name] = (torch.where(live, v, 0.0).sum((0, 1)), torch.where(live, e + 128 * U * v.abs(), 0.0).sum((0, 1)))
    return out


def recurrence(x, gate, h0=None, lengths=None, reverse=False, dh=None, dlast=None):
    """{"h", "last"} and, with dh, {"dx", "dgate", "dh0"}: (value, err).  The bound walks along: a frame adds K roundings of
    its terms to what it takes over from the one before, K = 16 for the sigmoid (4), the products and sums (4), and the
    regrouping of a scan, which rounds every product of gates once more per level that joins them (8)."""
    K = 16 * U
    x, gate = x.double(), gate.double()
    B, S, C = x.shape
    n, live = _live(B, S, lengths)
    x, gate = torch.where(live, x, 0.0), torch.where(live, gate, 0.0)
    a, na = torch.where(live, torch.sigmoid(gate), 1.0), torch.where(live, torch.sigmoid(-gate), 0.0)
    order = list(range(S - 1, -1, -1) if reverse else range(S))
    h, eh, before, eb = (torch.zeros_like(x) for _ in range(4))
    v = torch.zeros(B, C, dtype=torch.float64) if h0 is None else h0.double()
    e = torch.zeros_like(v)
    for t in order:
        before[:, t], eb[:, t] = v, e
        e = torch.where(live[:, t], a[:, t] * e + K * (a[:, t] * v.abs() + (na[:, t] * x[:, t]).abs()), e)
        v = torch.where(live[:, t], a[:, t] * v + na[:, t] * x[:, t], v)
        h[:, t], eh[:, t] = v, e
    out = {"h": (torch.where(live, h, 0.0), torch.where(live, eh, 0.0)), "last": (v, e)}
    if dh is None:
        return out
    dh = torch.where(live, dh.double(), 0.0)
    D, eD = torch.zeros_like(x), torch.zeros_like(x)
    v = torch.zeros(B, C, dtype=torch.float64) if dlast is None else dlast.double()
    e = torch.zeros_like(v)
    for t in reversed(order):
        D[:, t] = dh[:, t] + v
        eD[:, t] = e + 2 * U * (dh[:, t].abs() + v.abs())
        e = torch.where(live[:, t], a[:, t] * eD[:, t] + K * a[:, t] * (dh[:, t].abs() + v.abs()), e)
        v = torch.where(live[:, t], a[:, t] * D[:, t], v)
    dx, f = na * D, a * na * (before - x)
    out["dx"] = torch.where(live, dx, 0.0), torch.where(live, na * eD + 8 * U * dx.abs(), 0.0)
    out["dgate"] = (torch.where(live, f * D, 0.0),
                    torch.where(live, f.abs() * eD + a * na * (eb + 2 * U * (before.abs() + x.abs())) * (D.abs() + eD) + 16 * U * (f * D).abs(), 0.0))
    out["dh0"] = v, e
    return out


def philox(c, k, rounds=10):
    """Philox4x32 on numpy uint64 words."""
    low, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(v, np.uint64) for v in c]
    for i in range(rounds):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        w = [np.uint64((k[0] + i * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((k[1] + i * 0xBB67AE85) & 0xFFFFFFFF)]
        c = [(q >> s) ^ c[1] ^ w[0], q & low, (p >> s) ^ c[3] ^ w[1], p & low]
    return c


def keep(shape, p, seed, step, site):
    """The dropout's mask of a [B, S, C] tensor."""
    B, S, C = shape
    per = -(-C // 8)
    block = np.arange(B * S * per, dtype=np.uint64)
    m = 0xFFFFFFFF
    w = philox([block & np.uint64(m), block >> np.uint64(32), np.full_like(block, step & m), np.full_like(block, site)],
               [seed & m, seed >> 32 & m])
    bits = np.stack(w, -1).astype("<u4").view("<u2").reshape(B, S, per * 8)[..., :C]
    return torch.from_numpy((bits >= int(np.floor(p * 65536 + 0.5))).copy())


def dropout(x, p, seed, step, site, residual=None):
    thr = int(np.floor(p * 65536 + 0.5))
    scale = 65536 / (65536 - thr) if thr < 65536 else 0.0
    y = torch.where(keep(x.shape, p, seed, step, site), x.double() * scale, 0.0)
    err = 2 * U * y.abs()                                                  # the factor and the product
    if residual is not None:
        y = y + residual.double()
        err = err + U * y.abs()
    return y, err
