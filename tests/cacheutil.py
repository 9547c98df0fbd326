"""What the tests of the quantized key/value cache share: the definition of its
codes in plain torch, and caches that hold given rows."""
import torch

CODES = [torch.int8, torch.float8_e4m3fn]
BF, HF = torch.bfloat16, torch.float16


def two_to(n):
    """2^n, fp64, by its bits."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def quantize(x, codes):
    """Rows [..., D] -> codes and biased exponents, in 64 bits: the least power of two, 2^-126 at
    least, that takes the largest magnitude to 127 (int8) or 448 (e4m3)."""
    x = x.double()
    top = x.abs().amax(-1)
    m, ex = torch.frexp(top)  # top = m 2^ex, m in [1/2, 1)
    e = ex - 7 + (m > 127 / 128) if codes == torch.int8 else ex - 9 + (m > 0.875)
    e = torch.where(top == 0, torch.full_like(e, -126), e).clamp(min=-126)
    y = x * two_to(-e)[..., None]
    if codes == torch.int8:
        return y.round().to(torch.int8), (e + 127).to(torch.uint8)
    step = two_to(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
    return ((y / step).round() * step).float().to(codes), (e + 127).to(torch.uint8)


def value(codes, exps):
    """What codes stand for, fp64 (e4m3 by its bits; NaN where E is 255)."""
    if codes.dtype == torch.int8:
        c = codes.double()
    else:
        u = codes.view(torch.uint8).int()
        ex, m = (u >> 3) & 15, (u & 7).double()
        c = torch.where(ex == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * two_to(ex - 7))
        c = torch.where((u & 127) == 127, torch.full_like(c, float("nan")), c)
        c = torch.where(u >= 128, -c, c)
    c = c * two_to(exps.int() - 127)[..., None]
    return c.masked_fill((exps == 255)[..., None], float("nan"))


def garbage(qimg, n_pages, page, hk, d, codes, g, dev="cuda:0"):
    """A cache whose every byte is noise, NaN codes and exponents of 255 among them."""
    def noise(*shape):
        return torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.uint8)

    k, v = (noise(n_pages, hk, page, d).view(codes) for _ in range(2))
    ke, ve = noise(n_pages, hk, page), noise(n_pages, hk, page)
    ke[::2] = 255
    ve[::3] = 255
    return qimg.KvCache(k, v, ke, ve)


def fill(cache, lens, k, v, g, spare=3):
    """The rows k and v [sum(lens), Hk, D] in pages of the cache in random order; returns the block
    table, whose unused entries name a page outside the cache."""
    n, hk, page, d = cache.k.shape
    dev = cache.k.device
    each = [-(-x // page) for x in lens]
    assert sum(each) + spare <= n
    order = torch.randperm(n, generator=g, device=dev)
    table = torch.full((len(lens), max(each + [1])), n + 7, dtype=torch.int32, device=dev)
    slots, at = [], 0
    for b, x in enumerate(lens):
        mine = order[at:at + each[b]]
        at += each[b]
        table[b, :each[b]] = mine.int()
        i = torch.arange(x, device=dev)
        slots.append(mine[i // page] * page + i % page)
    slots = torch.cat(slots) if slots else torch.zeros(0, dtype=torch.long, device=dev)
    for dst, exps, rows in ((cache.k, cache.k_exp, k), (cache.v, cache.v_exp, v)):
        c, e = quantize(rows, cache.k.dtype)
        dst.view(torch.uint8)[slots // page, :, slots % page] = c.view(torch.uint8)
        exps[slots // page, :, slots % page] = e
    return table, slots
