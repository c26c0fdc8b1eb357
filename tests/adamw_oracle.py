"""The AdamW step, its 8-bit codes and their tolerances in plain 64-bit torch (CPU), for the tests.

Written from the formulas; nothing here comes from the package."""
import math

import torch

U = 2.0 ** -24  # half a step of fp32, relative
TINY = 2.0 ** -125
BLOCK, M_BITS, ROOT_BITS = 64, 3, 4
MASK = 0xFFFFFFFF


def pad64(n):
    return -(-n // BLOCK) * BLOCK


def place(tensors):
    """(flat fp64 vector with every tensor at a multiple of 64, offsets)"""
    offs, total = [], 0
    for t in tensors:
        offs.append(total)
        total += pad64(t.numel())
    out = torch.zeros(total, dtype=torch.float64)
    for t, o in zip(tensors, offs):
        out[o:o + t.numel()] = memory_order(t).double().cpu()
    return out, offs


def memory_order(t):
    """A dense tensor's elements in their order in memory."""
    return t.detach().as_strided((t.numel(),), (1,))


def hash_bits(numel, t, start=0):
    i = torch.arange(start, start + numel, dtype=torch.int64)
    x = ((i & MASK) + (i >> 32) * 0x27D4A62F + t * 0x632BE5AB) & MASK
    x = ((x ^ (x >> 16)) * 0x6E7A3B15) & MASK
    x = ((x ^ (x >> 15)) * 0x35D2C1A7) & MASK
    x = x ^ (x >> 16)
    return x & 0xFFFF, x >> 16


def code_values(codes, scales, mantissa):
    """What codes stand for (fp64)."""
    c = codes.long()
    sign = torch.ones(c.shape, dtype=torch.float64)
    if mantissa == M_BITS:
        sign[c >= 128] = -1.0
        c = c % 128
    one = 1 << mantissa
    e = c // one
    units = torch.where(e == 0, c.double(), (one + c % one).double() * 2.0 ** (e - 1).double())
    s = scales.double().repeat_interleave(BLOCK)
    unit = torch.where(s == 0, torch.zeros_like(s), 2.0 ** (s - 127))
    unit[s == 255] = math.nan
    return sign * units * unit


def code_bounds(x, mantissa, r16, slack):
    """The two values (fp64) that rounding may give where x is known to ``slack`` (relative): they are
    the same unless the rounding's border lies within it.  Blocks with values that are not finite: NaN.
    Also the mask of blocks whose scale is not decided (their largest value lies at a border)."""
    one = 1 << mantissa
    a = x.abs().view(-1, BLOCK)
    bad = ~torch.isfinite(a).all(1)
    a = torch.where(bad[:, None], torch.zeros_like(a), a)
    top = a.amax(1)
    largest = (2 * one - 1) * 2.0 ** 14
    k = torch.log2(torch.clamp(top, min=2.0 ** -149) / largest)
    open_ = (k - k.round()).abs() < 4 * slack  # includes exact powers: those are decided by tests of their own
    unit = 2.0 ** torch.clamp(torch.ceil(k), min=-126.0)
    y = (a / unit[:, None]).view(-1)

    def cut(y):
        e = torch.clamp(torch.floor(torch.log2(torch.clamp(y, min=1.0))) - mantissa, min=0.0)
        q = 2.0 ** e
        return torch.floor(y / q + (r16.double() + 0.5) / 65536.0) * q

    out = []
    for f in (1.0 - slack, 1.0 + slack):
        c = cut(y * f)
        if mantissa == ROOT_BITS:
            c = torch.where((a.view(-1) > 0) & (c < 1), torch.ones_like(c), c)
        v = c * unit.repeat_interleave(BLOCK)
        v = torch.where(x < 0, -v, v)
        v[bad.repeat_interleave(BLOCK)] = math.nan
        out.append(v)
    return out[0], out[1], open_.repeat_interleave(BLOCK)


def norm(grads):
    return math.sqrt(sum(float(g.detach().double().square().sum()) for g in grads))


def step(w, g, m, v, t, lr, b1, b2, eps, wd, decay, grad_scale=1.0, clip=0.0, total=None):
    """One step on flat fp64 vectors: ``t`` its number (from 1), ``decay`` a 0/1 vector, ``total`` the
    norm of all gradients.  Returns (w, m, v, root, tolerances of w, m, v, root).

    Tolerances: u = 2^-24 for every fp32 rounding.  g*scale: 1 for the product and, with clipping, 4 for
    the norm's rounding, its product with grad_scale, the quotient and the product.  m: 1 for each of
    b1, 1-b1, the product and the final sum, so 12 u of the sum of magnitudes holds; v: the square
    doubles g's, 16 u.  Roots halve and add one: 9 u.  lr*sqrt(1-b2^t)/(1-b1^t): t log b rounds by 1 u,
    expm1 by up to 4, root, product and quotient 1 each: 12 u.  The update's quotient adds 3, its sums with
    the decay 2 of what they sum; the weight's own rounding is 1 of the result."""
    s = grad_scale
    if clip:
        scaled = total * abs(grad_scale)
        s = s if scaled <= clip else s * clip / scaled if math.isfinite(scaled) else math.nan
    x = g * s
    m1, v1 = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    root = v1.sqrt()
    bc1, bc2 = (-math.expm1(t * math.log(b)) if b else 1.0 for b in (b1, b2))
    a = lr * math.sqrt(bc2) / bc1
    q = m1 / (root + eps)
    w1 = w - (lr * wd * decay * w + a * q)
    tm = 12 * U * (b1 * m.abs() + (1 - b1) * x.abs()) + TINY
    tv = 16 * U * v1 + TINY
    tr = 9 * U * root + 2.0 ** -62
    tw = U * (2 * w.abs() + w1.abs()) + 8 * U * lr * wd * w.abs() + 30 * U * a * q.abs() + a * tm / (root + eps) + TINY
    return w1, m1, v1, root, tw, tm, tv, tr


def within(got, want, tol):
    """Elementwise, NaN and infinities equal where expected."""
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    over = (got[ok] - want[ok]).abs() - tol.expand_as(want)[ok]
    assert not over.numel() or float(over.max()) <= 0.0, f"off by {float(over.max())} more than allowed"
