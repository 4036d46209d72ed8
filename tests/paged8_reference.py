"""A cache in 8 bits in plain 64-bit arithmetic on the CPU: what stores leave in it, block by block, and what attention to it gives.  Codes
are kept as the numbers they stand for."""
import math

import torch

DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
LEAST = 2.0 ** -100


def nearest(y, code):
    """The nearest code, the even one of two."""
    if code == "int8":
        return torch.round(y)
    e = torch.frexp(y)[1].clamp_min(-5).to(torch.float64) - 4.0            # e4m3 numbers from 2^(e + 3) on are multiples of 2^e, at least 2^-9
    step = torch.exp2(e)
    return torch.round(y / step) * step


def scale_of(a, code):
    """a / Q, rounded up to four significant bits"""
    if a == 0.0:
        return LEAST
    m, e = math.frexp(a / LARGEST[code])
    return max(math.ceil(m * 16.0) / 16.0 * 2.0 ** e, LEAST)


def store(codes, scales, x, table, cu, start, block, code):
    """codes [pages, Hkv, page, D] and scales [pages, Hkv, blocks], float64, are changed; x [rows, Hkv, D]."""
    pages, H, page, _ = codes.shape
    Q = LARGEST[code]
    for b in range(len(cu) - 1):
        first, n = start[b], cu[b + 1] - cu[b]
        for at in range(first // block * block, first + n, block):
            lo, hi = max(first, at), min(first + n, at + block)
            if lo >= hi or at < 0 or at // page >= len(table[b]) or not 0 <= table[b][at // page] < pages:
                continue
            p, t = table[b][at // page], at % page
            for h in range(H):
                new = x[cu[b] + lo - first:cu[b] + hi - first, h].double()
                a = float(new.abs().max()) if torch.isfinite(new).all() else math.inf
                s, lost = float(scales[p, h, t // block]), a == math.inf
                if lo == at:
                    s = scale_of(a, code) if not lost else math.nan
                else:
                    lost = lost or not LEAST <= s < math.inf
                    grow = 0
                    while not lost and a > Q * s * 2.0 ** grow:
                        grow += 1
                    old = codes[p, h, t:t + lo - at]
                    if grow:
                        codes[p, h, t:t + lo - at] = nearest(old * 2.0 ** -grow, code)
                    s = s * 2.0 ** grow
                scales[p, h, t // block] = math.nan if lost else s
                codes[p, h, t + lo - at:t + hi - at] = 0.0 if lost else nearest(new / s, code)


def numbers(codes, scales):
    """[pages, Hkv, page, D] float64"""
    return codes * scales.repeat_interleave(codes.shape[2] // scales.shape[2], 2)[..., None]


def to_device(codes, scales, code):
    return codes.float().to(DTYPES[code]).cuda(), scales.float().cuda()


def from_device(codes):
    return codes.cpu().float().double()


def random_cache(g, pages, Hkv, page, D, block, code):
    """Codes of all sizes and scales far apart, float64."""
    s = torch.exp2(torch.randint(-12, 4, (pages, Hkv, page // block), generator=g).double()) * (8 + torch.randint(0, 8, (pages, Hkv, page // block), generator=g)) / 8.0
    y = torch.randn((pages, Hkv, page, D), generator=g).double() * LARGEST[code] / 3.0
    return nearest(y.clamp(-LARGEST[code], LARGEST[code]), code), s
