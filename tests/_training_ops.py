"""Float64 statements of the training operators and the error bounds that their tests hold them to.

Bounds count roundings.  A product of a kind with unit roundoff u (bf16 2^-8, fp16 2^-11, fp32 2^-24) summed over K terms in Float32
differs from the exact sum by at most (K + 16) 2^-23 times the sum of the absolute terms: one rounding of at most 2^-23 per addition (twice
IEEE's half step: the matrix unit may truncate), 16 for the products themselves.  A value stored in the kind adds u times itself, and fp16
adds 2^-24 (subnormal spacing 2^-24, half of it, twice for safety)."""
import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}
# act, its derivative, bounds of |act'| and |act''| over the reals
S2P = math.sqrt(2 / math.pi)


def _gelu_tanh(g):
    return 0.5 * g * (1 + torch.tanh(S2P * (g + 0.044715 * g ** 3)))


def _gelu_tanh_slope(g):
    t = torch.tanh(S2P * (g + 0.044715 * g ** 3))
    return 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * S2P * (1 + 3 * 0.044715 * g * g)


ACTS = {
    "identity": (lambda g: g, lambda g: torch.ones_like(g), 1.0, 0.0),
    "tanh": (torch.tanh, lambda g: 1 - torch.tanh(g) ** 2, 1.0, 0.8),
    "rbf": (lambda g: torch.exp(-g * g), lambda g: -2 * g * torch.exp(-g * g), 0.9, 2.0),
    "relu": (lambda g: g.clamp_min(0), lambda g: (g > 0).to(g.dtype), 1.0, 0.0),
    "sigmoid": (torch.sigmoid, lambda g: torch.sigmoid(g) * torch.sigmoid(-g), 0.25, 0.1),
    "swish": (lambda g: g * torch.sigmoid(g), lambda g: torch.sigmoid(g) * (1 + g * torch.sigmoid(-g)), 1.1, 0.5),
    "gelu_tanh": (_gelu_tanh, _gelu_tanh_slope, 1.13, 0.9),
    "gelu_erf": (lambda g: 0.5 * g * (1 + torch.erf(g / math.sqrt(2))),
                 lambda g: 0.5 * (1 + torch.erf(g / math.sqrt(2))) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi), 1.13, 0.8),
}
# Float32 evaluation of act and act' out of a handful of library calls and products, each within a few units in the last place, with
# cancellation at most against terms of size 1 + |g|
FN = 32 * 2.0 ** -24


def gated(x, wg, wu, wd, act, dy=None):
    """{name: (value, bound)} of y, gate, up and, with dy, dx, dwg, dwu, dwd, in Float64"""
    kind = x.dtype
    u, tiny = UNIT[kind], TINY[kind]
    f, fs, l1, l2 = ACTS[act]
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))

    def gamma(k):
        return (k + 16) * 2.0 ** -23

    def store(v, e):
        return e * (1 + u) + u * v.abs() + tiny

    D, F, O, T = x.shape[1], wg.shape[0], wd.shape[0], x.shape[0]
    g, up = x @ wg.T, x @ wu.T
    eg, eu = gamma(D) * (x.abs() @ wg.abs().T), gamma(D) * (x.abs() @ wu.abs().T)
    a, s = f(g), fs(g)
    ea = l1 * eg + FN * (1 + g.abs())
    es = l2 * eg + FN * (1 + g.abs())
    if act == "relu":
        ea, es = eg, (g.abs() <= eg).double()
    if act == "identity":
        ea, es = eg, torch.zeros_like(g)
    h = a * up
    eh = store(h, ea * (up.abs() + eu) + a.abs() * eu + 2.0 ** -22 * h.abs())
    y = h @ wd.T
    ey = store(y, (eh + gamma(F) * (h.abs() + eh)) @ wd.abs().T)
    out = {"y": (y, ey), "gate": (g, eg + 2.0 ** -23 * g.abs()), "up": (up, eu + 2.0 ** -23 * up.abs())}
    if dy is None:
        return out
    dy = dy.double()
    dh = dy @ wd
    edh = gamma(O) * (dy.abs() @ wd.abs())
    dg, du = dh * up * s, dh * a
    edg = store(dg, edh * (up.abs() + eu) * (s.abs() + es) + dh.abs() * (eu * (s.abs() + es) + up.abs() * es) + 2.0 ** -21 * dg.abs())
    edu = store(du, edh * (a.abs() + ea) + dh.abs() * ea + 2.0 ** -22 * du.abs())

    def product(p, ep, q, k):
        return p @ q, store(p @ q, (ep + gamma(k) * (p.abs() + ep)) @ q.abs())

    v1, e1 = product(dg, edg, wg, 2 * F)
    v2, e2 = product(du, edu, wu, 2 * F)
    out["dx"] = (v1 + v2, e1 + e2)
    out["dwg"] = product(dg.T, edg.T, x, T)
    out["dwu"] = product(du.T, edu.T, x, T)
    v, e = product(h.T, eh.T, dy, T)
    out["dwd"] = (v.T, e.T)
    return out


def within(got, want):
    """largest error over its bound; NaN and infinities count as infinite unless the reference has them too"""
    value, bound = want
    if value.numel() == 0:
        return 0.0
    d = (got.double() - value).abs()
    return float(torch.where(torch.isfinite(d), d / bound.clamp_min(1e-300), torch.inf).max())


BLOCK = 256


def blocks(x, fill=0.0):
    """(number of blocks, 256), the last one padded"""
    n = x.numel()
    k = -(-n // BLOCK)
    return torch.nn.functional.pad(x.reshape(-1), (0, k * BLOCK - n), value=fill).view(k, BLOCK)


def value_m(q, a):
    q = blocks(q.double())
    return (a.double()[:, None] * q.sign() * (q / 127) ** 2)


def value_v(r, c):
    return c.double()[:, None] * (blocks(r.double()) / 255) ** 4


def adamw(p, g, m, v, t, eta, beta, eps, wd, factor=1.0):
    """one step in Float64: (p, m, v)"""
    g = g.double() * factor
    m, v = beta[0] * m.double() + (1 - beta[0]) * g, beta[1] * v.double() + (1 - beta[1]) * g * g
    step = eta * (m / (1 - beta[0] ** t)) / ((v / (1 - beta[1] ** t)).sqrt() + eps)
    return p.double() * (1 - eta * wd) - step, m, v, step
