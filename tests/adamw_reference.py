"""Plain 64-bit forms of the optimizer operators (include/gsx_optim.h) on the CPU, and how far 32-bit arithmetic may be from them.

Every bound counts roundings: U = 2^-24, half a step of float32.  A sum's bound is relative to the sum of its terms' magnitudes (terms may cancel)."""
import math

import torch

U = 2.0 ** -24
RUN, TOP, FLOOR = 128, 448.0, 2.0 ** -120
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}   # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}  # ... of the subnormal numbers, at most
GRID = torch.tensor([f * 2.0 ** -9 for f in range(8)] + [(8 + f) * 2.0 ** (e - 10) for e in range(1, 16) for f in range(8)], dtype=torch.float64)[:127]


def mix(x):
    x = x ^ (x >> 16)
    x = x * 0x9E46A9E5 % 2 ** 32
    x = x ^ (x >> 15)
    x = x * 0xF4B0A2DB % 2 ** 32
    return x ^ (x >> 16)


def draws(seed, step, ordinal, first, n):
    """u of the first and of the second moment for values first .. first + n - 1 of tensor `ordinal`."""
    key = mix((mix((seed + 0x9E3779B9 * step) % 2 ** 32) + 0xC2A6F0B5 * ordinal) % 2 ** 32)
    i = torch.arange(first, first + n, dtype=torch.int64)
    w = mix((i + key + 0x61C8864F * (i >> 32)) % 2 ** 32)
    return (w >> 16).double() / 65536, (w % 65536).double() / 65536


def rounded(y, positive, u):
    """y (|y| <= 448) to the numbers of the format; u None: to nearest, ties to even."""
    a = y.abs().clamp(max=TOP)
    low = (torch.searchsorted(GRID, a, right=True) - 1).clamp(max=125)
    lo, hi = GRID[low], GRID[low + 1]
    if u is None:
        up = (a - lo > hi - a) | ((a - lo == hi - a) & (low % 2 == 1))
    else:
        up = (a - lo) / (hi - lo) + u >= 1.0
    c = torch.where(up, hi, lo)
    if positive:
        c = torch.where((y > 0) & (c == 0), GRID[1], c)
    return torch.copysign(c, y)


def runs(n):
    return -(-n // RUN)


def spread(scale, n):
    return scale.repeat_interleave(RUN)[:n]


def scales(x):
    n = x.numel()
    full = torch.zeros(runs(n) * RUN, dtype=torch.float64)
    full[:n] = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    return (full.view(-1, RUN).amax(1) / TOP).clamp(min=FLOOR)


def pack(x, positive, u=None):
    """(codes as float8_e4m3fn, scales as float32) of a flat tensor: a valid 8-bit state near x."""
    s = scales(x.double()).float()
    y = x.double() / spread(s, x.numel()).double()
    return rounded(y.clamp(-TOP, TOP), positive, u).to(torch.float8_e4m3fn), s


def adamw(p, g, m, v, lr, wd, step, b1=0.9, b2=0.999, eps=1e-15, factor=1.0):
    """New p, m, v, r and the magnitudes their errors are relative to.  All float64; m, v the old moments; r = sqrt(v)."""
    g = g * factor
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    mm = (b1 * m).abs() + ((1 - b1) * g).abs()
    r = v1.sqrt()
    denom = r / math.sqrt(1 - b2 ** step) + eps
    k = lr / (1 - b1 ** step)
    q = p * (1 - lr * wd) - k * m1 / denom
    # p: lr wd p takes 3 roundings of its own, the two subtractions one each; the step's quotient: beta and 1 - beta (1 each), the factor (2: itself, its product),
    # the sums (2), 1 / (1 - beta1^t) and 1 / sqrt(1 - beta2^t) (5 each: beta's logarithm times t, expm1 of up to 2 ulp, root, quotient), the root of v (half of
    # 6, 1), its product, the sum, the quotient, lr: 30 at most
    pp = U * (2 * q.abs() + 2 * p.abs() + 4 * (lr * wd * p).abs()) + 32 * U * torch.nan_to_num(k * mm / denom, 0.0)
    return q, m1, v1, r, pp, mm


def check_codes(codes, scale, x, tol, positive, u, what=""):
    """codes / scale (from the device, on the CPU, flat) against the 64-bit values x, each known within +- tol."""
    n = x.numel()
    bad = ~torch.isfinite(x)
    got = codes.float().double()
    assert torch.equal(torch.isnan(got), bad), what + ": NaN codes are those of the values that are not finite"
    s = scales(x)
    fin_tol = torch.where(bad, torch.zeros_like(tol), tol)
    # the largest magnitude of a run is off by at most the largest of its values' bounds; the quotient by 448 one rounding more
    top_tol = torch.zeros(runs(n) * RUN, dtype=torch.float64)
    top_tol[:n] = fin_tol
    err = (scale.double() - s).abs()
    assert bool((err <= top_tol.view(-1, RUN).amax(1) / TOP + 2 * U * s).all()), "%s: scales off by %g" % (what, float((err / s).max()))
    sd = spread(scale.double(), n)
    ok = ~bad
    y, dy = torch.where(ok, x, torch.zeros_like(x)) / sd, fin_tol / sd
    dy = dy + 3 * U * y.abs() + 2.0 ** -149
    a = y.abs()
    lo, hi = rounded((a - dy).clamp(min=0, max=TOP), False, u), rounded((a + dy).clamp(max=TOP), False, u)
    if positive:   # a value that may be above zero is not stored as zero, one that may be zero may be
        hi = torch.where((a > 0) & (hi == 0), GRID[1], hi)
        assert bool((got[ok & (a > 0) & (a > dy)] > 0).all()), what + ": a root above zero stored as zero"
        lo = torch.where((a > dy) & (lo == 0), GRID[1], lo)
    g = got.abs()
    inside = (g >= lo) & (g <= hi) & ((torch.sign(got) == torch.sign(y)) | (got == 0) | (a <= dy))
    assert bool(inside[ok].all()), "%s: %d of %d codes are not the rounded value: %s" % (
        what, int((~inside & ok).sum()), n, [(float(y[i]), float(got[i]), float(lo[i]), float(hi[i])) for i in (~inside & ok).nonzero().flatten()[:4].tolist()])
