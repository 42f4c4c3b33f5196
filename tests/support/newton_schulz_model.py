"""How far a Newton-Schulz result may be off: a model of the kernels' roundings and the plain fp32
form, both compared with the definition in 64 bits on the same input."""
import math

import torch

from .muon_oracle import NS, exact, rel, triples

PRODUCTS = ("gram", "square", "apply")


def _planes(v, exponent):
    """Two fp16 terms of v * 2^exponent, scaled back."""
    s = 2.0 ** exponent
    hi = (v * s).half().float()
    lo = (v * s - hi).half().float()
    return hi / s, lo / s


def _product(x, w, terms):
    """The matrix units' order: 32 summed values at a time to an fp32 accumulator, once per term."""
    out = torch.zeros(x[0].shape[0], w[0].shape[1], device=x[0].device)
    for k in range(0, x[0].shape[1], 32):
        for i, j in terms:
            out += x[i][:, k:k + 32] @ w[j][k:k + 32]
    return out


def modelled(x, wide=True, steps=5, coefficients=NS, eps=1e-7, device="cpu", drop=None):
    """The result before it is rounded to the output's type.  ``wide``: products of both terms (without
    lo lo), else of the first ones.  ``drop``: (product, term) that a wrong kernel would leave out,
    a term being (0, 1) or (1, 0)."""
    y = x.detach().to(device).double()
    y = (y / (y.norm() + eps)).float()
    if x.shape[0] > x.shape[1]:
        y = y.T
    terms = {p: [t for t in ([(0, 0), (0, 1), (1, 0)] if wide else [(0, 0)]) if drop != (p, t)] for p in PRODUCTS}
    y = _planes(y, 14)
    for a, b, c in triples(steps, coefficients):
        g = _product(y, (y[0].T, y[1].T), terms["gram"])
        d = g.diagonal().clone()
        o = _planes(g - torch.diag(d), 14)
        off = o[0] + o[1]
        s = _product(o, (o[0].T, o[1].T), terms["square"])
        p = c * (s + (d[:, None] + d[None, :]) * off) + b * off
        e = c * (s.diagonal() + d * d) + b * d + a
        p = _planes(p - torch.diag(p.diagonal()), 12)
        y = _planes(e[:, None] * (y[0] + y[1]) + _product(p, y, terms["apply"]), 14)
    y = y[0] + y[1]
    return y.T if x.shape[0] > x.shape[1] else y


def plain(x, steps=5, coefficients=NS, eps=1e-7, device="cpu"):
    """The definition with fp32 products."""
    y = x.detach().to(device).double()
    y = (y / (y.norm() + eps)).float()
    if x.shape[0] > x.shape[1]:
        y = y.T
    for a, b, c in triples(steps, coefficients):
        g = y @ y.T
        y = a * y + (b * g + c * (g @ g)) @ y
    return y.T if x.shape[0] > x.shape[1] else y


def bound(x, want, out_dtype=torch.float32, wide=True, device="cpu", **kw):
    """Largest relative distance of a result of ``out_dtype`` from ``want``, the 64-bit value.

    Before its last rounding a result is off by the same roundings as the model, in another order, or
    by those of the plain form: each is one draw of them, of which where x has few directions only a
    few numbers count, so four times the larger of both bounds another draw.  fp32 itself adds half a
    step.  Rounding then: with y the value and e the exact one, every element has |round(y) - e| <=
    |round(y) - y| + |y - e| <= |round(e) - y| + |y - e| <= |round(e) - e| + 2 |y - e|."""
    off = rel(modelled(x, wide, device=device, **kw), want)
    if wide:
        off = max(off, rel(plain(x, device=device, **kw), want))
    off = 4 * off + 2.0 ** -24
    if out_dtype == torch.float32:
        return off
    return rel(want.to(out_dtype), want) + 2 * off


def spectra(m, n, seed=0):
    """Inputs by name: friendly ones, and those whose weak directions drown in the roundings of the
    strong ones (few directions over a low floor, one dominant column, falling singular values)."""
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g)

    few, many = min(8, m, n), min(32, m, n)
    short = min(m, n)
    out = {"noise": r(m, n),
           "gradient": (r(m, few) / torch.arange(1, few + 1)) @ r(few, n) + 0.2 * r(m, n)}
    for floor in (1e-1, 1e-2, 1e-3):
        out[f"low_rank_{floor:g}"] = r(m, many) @ r(many, n) / math.sqrt(many) + floor * r(m, n)
    for f in (1e1, 1e3, 1e4, 1e5):
        x = r(m, n)
        (x if n >= m else x.T)[:, min(3, max(m, n) - 1)] *= f
        out[f"column_{f:g}"] = x
    q = torch.linalg.qr(r(short, short))[0] * torch.logspace(0, -5, short)
    out["falling"] = q @ r(short, n) if m <= n else r(m, short) @ q
    return out
