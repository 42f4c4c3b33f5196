"""Plain forms the Newton-Schulz / Muon tests compare with: the definition in 64 bits, and a model
of the kernels' roundings in fp32 whose own error sets the tolerances."""
import torch

NS = (3.4445, -4.7750, 2.0315)


def triples(steps, coefficients):
    c = list(coefficients)
    return [c] * steps if len(c) == 3 and not hasattr(c[0], "__len__") else c


def exact(x, steps=5, coefficients=NS, eps=1e-7, device="cpu"):
    y = x.detach().to(device).double()
    y = y / (y.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = y.shape[-2] > y.shape[-1]
    if tall:
        y = y.transpose(-2, -1)
    for a, b, c in triples(steps, coefficients):
        g = y @ y.transpose(-2, -1)
        y = a * y + (b * g + c * (g @ g)) @ y
    return y.transpose(-2, -1) if tall else y


def _planes(v, scale):
    """value -> the sum of two fp16 terms, and the first of them."""
    hi = (v * scale).half().float()
    lo = (v * scale - hi).half().float()
    return (hi + lo) / scale, hi / scale


def modelled(x, wide, steps=5, coefficients=NS, eps=1e-7, sums=None, device="cpu"):
    """fp32 accumulation, planes of two fp16 terms (scaled by 2^13, a power of two that keeps every
    value of these tests in range), products of both terms (wide) or of the first (narrow), exact
    diagonals."""
    y = x.detach().to(device).double()
    y = (y / (y.square().sum() .sqrt() + eps)).float()
    if y.shape[0] > y.shape[1]:
        y = y.T
    y, yh = _planes(y, 2.0 ** 13)
    pick = (lambda v, h: v) if wide else (lambda v, h: h)
    for a, b, c in triples(steps, coefficients):
        f = pick(y, yh)
        gram = f @ f.T
        d = gram.diagonal().clone()
        o, oh = _planes(gram - torch.diag(d), 2.0 ** 13)
        f2 = pick(o, oh)
        poly = b * (o + torch.diag(d)) + c * (f2 @ f2 + (d[:, None] + d[None, :]) * o + torch.diag(d * d))
        e = poly.diagonal().clone()
        p, ph = _planes(poly - torch.diag(e), 2.0 ** 12)
        if sums is not None:
            sums.append((abs(a), float((p.abs() @ y.abs()).norm()), y.shape[0]))
        y, yh = _planes((a + e)[:, None] * y + pick(p, ph) @ f, 2.0 ** 13)
    return y.T if x.shape[0] > x.shape[1] else y


def rel(a, b):
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


def gradient(m, n, seed, batch=()):
    """A few strong directions over a floor of noise."""
    g = torch.Generator().manual_seed(seed)
    r = min(8, m, n)
    s = torch.randn(*batch, m, r, generator=g) / torch.arange(1, r + 1)
    return (s @ torch.randn(*batch, r, n, generator=g) + 0.2 * torch.randn(*batch, m, n, generator=g)) * 1e-3


def tolerance(x, wide, out_dtype, **kw):
    """Four times the rounding model's own error (the rare worse draw), the rounding of the sums that
    the model does not share, and the rounding of the result: at most half a step per element.

    Sums: the matrix units add 32 products at a time to an fp32 accumulator, for a wide product three
    times, so an entry of P Y goes through n = 3 ceil(m / 32) roundings of at most 2^-24 of the partial
    sum, itself at most (|P| |Y|)_ij; the model's own sums are blocked and round less often.  Unbiased
    and independent, n of them come to sqrt(n) 2^-24 (|P| |Y|)_ij at most in the mean square, and four
    times that covers the draw.  A difference in Y grows by at most |a| in each later step (the
    polynomial's steepest slope), as it does where x has few directions: there the error is this term."""
    half_step = torch.finfo(out_dtype).eps / 2
    sums, want = [], exact(x, **kw)
    off = 4 * rel(modelled(x, wide, sums=sums, **kw), want)
    grown = 0.0
    for a, size, m in sums:
        n = 3 * (-(-m // 32))
        grown = a * grown + 4 * n ** 0.5 * 2.0 ** -24 * size
    return off + grown / max(float(want.norm()), 1e-30) + half_step + 2.0 ** -22
