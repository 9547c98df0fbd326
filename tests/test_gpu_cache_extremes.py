"""GPU: the quantized key/value cache at the ends of its values' ranges, against the
definition in 64 bits."""
import pytest
import torch

from cacheutil import BF, CODES, quantize, value
from test_gpu_attention_cache import Case, _check, _i32

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# Rows of a sequence on average: 14, 70 and 710 of a kv head, for tiles of 16, 32 and 128 rows
TILES = [dict(lq=[2, 1], lk=[90, 300], hq=28, hk=4), dict(lq=[10, 3], lk=[100, 700], hq=28, hk=4),
         dict(lq=[150, 60, 3], lk=[200, 60, 2000], hq=80, hk=8)]


def _top_codes(rows, codes):
    """The definition's codes and exponents; the largest code's next below where it would be 2^128."""
    c, e = quantize(rows, codes)
    v = value(c, e)
    less = torch.tensor(63.0 if codes == torch.int8 else 240.0, device=DEV)
    edge = (torch.sign(v) * less).to(codes)
    over = v.abs() >= 2.0 ** 128
    assert bool(over.any())
    return torch.where(over, edge.view(torch.uint8), c.view(torch.uint8)).view(codes), e


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, BF], ids=str)
def test_the_largest_rows_stay_finite(qimg, codes, dtype):
    """Rows up to the type's largest value: no finite value comes back as an infinity."""
    top = torch.finfo(dtype).max
    x = torch.linspace(-1, 1, 64, dtype=torch.float64, device=DEV).view(1, 1, 64)
    f = torch.linspace(0.9, 1, 16, dtype=torch.float64, device=DEV).view(16, 1, 1)
    rows = (x * f * top).to(dtype)
    rows[3] = (x * 127 * 2.0 ** 121).to(dtype)     # the largest amaxes of smaller exponents
    rows[4] = (x * 448 * 2.0 ** 119).to(dtype)
    assert bool(rows.isfinite().all())
    table, lens, cu = _i32(0).view(1, 1), _i32(16), _i32(0, 16)
    slots = torch.arange(16, dtype=torch.int32, device=DEV)
    want, exps = _top_codes(rows, codes)
    for heads in (False, True):
        cache = qimg.kv_cache(1, 16, 1, 64, codes, DEV)
        if heads:  # k and v of packed heads, without a norm or positions
            qimg.norm_rope_cache(torch.cat((rows, rows), 1), 0, cache, slots)
        else:
            qimg.kv_cache_write(cache, rows, rows, slots)
        torch.cuda.synchronize()
        for c, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)):
            assert torch.equal(e[0].t(), exps)
            same = c[0].transpose(0, 1).view(torch.uint8) == want.view(torch.uint8)
            zero = (rows == 0) if codes != torch.int8 else torch.zeros_like(same)  # (of either sign)
            assert bool((same | zero).all()), int((~same).sum())
        for t in (torch.float32, BF):
            for back in qimg.kv_cache_read(cache, table, lens, cu, 16, out_dtype=t):
                assert bool(back.isfinite().all())
                assert torch.equal(back.double(), value(want, exps))


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("tiles", range(3))
def test_the_largest_values_behind_a_mask(qimg, codes, tiles):
    """V of the largest finite values at a key that the last query of a sequence alone sees: the
    others' results stay as they are."""
    t = TILES[tiles]
    c = Case(qimg, codes=codes, seed=31, **t)
    base = c.run(qimg)
    n, hk, page, d = c.cache.k.shape
    key = t["lk"][0] - 1
    slot = int(c.table[0, key // page]) * page + key % page
    v = torch.full((1, hk, d), torch.finfo(torch.float32).max, device=DEV)
    v[..., ::2] *= -1
    k = torch.zeros_like(v)
    qimg.kv_cache_write(c.cache, k, v, _i32(slot))
    got = c.run(qimg)
    torch.cuda.synchronize()
    keep = torch.ones(sum(t["lq"]), dtype=torch.bool, device=DEV)
    keep[t["lq"][0] - 1] = False
    assert torch.equal(got[keep], base[keep])
    c.k[key] = 0
    c.v[key] = v[0].sign() * (63 * 2.0 ** 122 if codes == torch.int8 else 240 * 2.0 ** 120)
    _check(got, *c.oracle())


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("tiles", range(3))
@pytest.mark.parametrize("scale", [-50, -70, -76])
def test_small_values_of_small_weights(qimg, codes, tiles, scale):
    """Thousands of keys at 2^-14 of one key's weight, whose v is zeros: averages of 2^-79 keep
    their digits, whatever the codes and the tiles' rows."""
    t = TILES[tiles]
    c = Case(qimg, t["lq"], [8000] + t["lk"][1:], hq=t["hq"], hk=t["hk"], codes=codes, seed=32, scale=2.0 ** scale)
    page, hk, d = c.cache.k.shape[2], c.hk, c.q.shape[2]
    c.q.fill_(1)
    c.cache.k.view(torch.uint8).zero_()
    c.cache.k_exp.fill_(127)
    c.k.zero_()
    heavy = torch.full((len(t["lq"]), hk, d), 0.875, device=DEV)  # a score of 14.3 log 2
    qimg.kv_cache_write(c.cache, heavy, torch.zeros_like(heavy), (c.table[:, 0] * page).int())
    at = torch.tensor(c.ck[:len(t["lq"])], device=DEV)
    c.k[at], c.v[at] = 0.875, 0.0
    got = c.run(qimg)
    torch.cuda.synchronize()
    want, mag, far = c.oracle()
    assert float(mag[t["lq"][0] - 1].min()) > 2.0 ** -79
    _check(got, want, mag, far)
