"""GPU parity: norms and rotary positions of packed heads (qimg_norm_rope_packed), the
same into a quantized cache (qimg_norm_rope_cache), rows into it (qimg_kv_cache_write)
and out of it (qimg_kv_cache_read), against their definitions in 64 bits.

Tolerance of a normed value, in units of 2^-24 relative: the sum of D squares comes
from eight fused steps and five additions at most (14, and 7 in the root), the mean,
eps, root and reciprocal are one rounding each (2 for those under the root's half
weight and after it: 3 in all), times x and w 2 more: 12. A turned value is a product and
a fused one of such: 2 more. 16 covers them, times the magnitudes that are added."""
import pytest
import torch

from cacheutil import BF, CODES, HF, fill, garbage, quantize, two_to, value

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, BF, HF]
EPS = 1e-6


def _table(rows, r):
    f = torch.pow(10000.0, -torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)
    a = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.stack((a.cos(), a.sin()), -1).float()


def _definition(x, nq, nk, wq, wk, table, pos, interleaved, eps=EPS):
    """fp64 heads, and the magnitudes that are added for each value (0: copied)."""
    x = x.double()
    d = x.shape[-1]
    mag = torch.zeros_like(x)
    for lo, hi, w in ((0, nq, wq), (nq, nq + nk, wk)):
        if w is not None:
            x[:, lo:hi] = x[:, lo:hi] / ((x[:, lo:hi] ** 2).sum(-1, keepdim=True) / d + eps).sqrt() * w.double()
            mag[:, lo:hi] = x[:, lo:hi].abs()
    out = x.clone()
    if table is not None:
        r, n = 2 * table.shape[1], nq + nk
        cs = table.double()[pos.long()][:, None]
        c, s = cs[..., 0], cs[..., 1]
        ia = slice(0, r, 2) if interleaved else slice(0, r // 2)
        ib = slice(1, r, 2) if interleaved else slice(r // 2, r)
        a, b = x[:, :n, ia], x[:, :n, ib]
        out[:, :n, ia], out[:, :n, ib] = a * c - b * s, b * c + a * s
        mag[:, :n, ia], mag[:, :n, ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, mag


def _tol(want, mag, dtype):
    i = torch.finfo(dtype)
    return 16 * 2.0 ** -24 * mag + (want.abs() + 16 * 2.0 ** -24 * mag) * i.eps / 2 + i.smallest_normal * i.eps / 2


def _check(got, want, mag):
    off = (got.double() - want).abs() - _tol(want, mag, got.dtype)
    assert float(off.max()) <= 0, f"max excess {float(off.max())}"


def _make(t, nq, nk, d, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.randn(t, nq + 2 * nk, d, generator=g, device=DEV)
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(BF) for _ in range(2))
    return x, wq, wk, g


SHAPES = [(1, 28, 4, 128, 128), (7, 3, 0, 64, 64), (33, 0, 5, 64, 32), (100, 4, 2, 80, 40), (1001, 24, 24, 128, 64),
          (3, 1, 1, 8, 8), (5, 2, 1, 256, 256), (9, 3, 2, 200, 48)]


@pytest.mark.parametrize("t,nq,nk,d,r", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_packed(qimg, t, nq, nk, d, r, interleaved):
    x0, wq, wk, g = _make(t, nq, nk, d, t + nq + d)
    table = _table(500, r)
    pos = torch.randint(0, 500, (t,), generator=g, device=DEV, dtype=torch.int32)
    for tin in TYPES:
        for tout in TYPES:
            x = x0.to(tin)
            got = qimg.norm_rope_packed(x, nq, nk, wq, wk, EPS, table, pos, interleaved, out_dtype=tout)
            torch.cuda.synchronize()
            _check(got, *_definition(x, nq, nk, wq, wk, table, pos, interleaved))


def test_without_a_norm_or_a_rotation(qimg):
    x, wq, wk, g = _make(50, 5, 2, 128, 3)
    table, pos = _table(100, 128), torch.arange(50, device=DEV, dtype=torch.int32)
    for q, k, tb in ((None, wk, table), (wq, None, None), (None, None, table), (None, None, None)):
        got = qimg.norm_rope_packed(x, 5, 2, q, k, EPS, tb, None if tb is None else pos)
        _check(got, *_definition(x, 5, 2, q, k, tb, pos, False))
    plain = qimg.rope_packed(x, table, pos, 7)  # without norms: the same values
    assert torch.equal(qimg.norm_rope_packed(x, 5, 2, cos_sin=table, positions=pos), plain)


@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_views_and_tokens_without_a_position(qimg, d, interleaved):
    """Heads of longer rows and head-major ones, in their place; what lies between them and
    tokens whose position is outside the table stay as they were."""
    x, wq, wk, g = _make(77, 6, 2, d, 4)
    table = _table(40, 32)
    pos = torch.randint(0, 40, (77,), generator=g, device=DEV, dtype=torch.int32)
    pos[5], pos[70] = -1, 40
    room = torch.full((77, 12, d + 8), 9.0, device=DEV)
    view = room[:, 1:11, :d]
    view.copy_(x)
    got = qimg.norm_rope_packed(view, 6, 2, wq, wk, EPS, table, pos, interleaved, out=view)
    want, mag = _definition(x, 6, 2, wq, wk, table, pos.clamp(0, 39), interleaved)
    for t in (5, 70):
        want[t], mag[t] = x[t].double(), 0
    torch.cuda.synchronize()
    _check(got, want, mag)
    assert bool((room[:, 0] == 9).all() and (room[:, 11] == 9).all() and (room[:, :, d:] == 9).all())
    heads = torch.zeros(10, 77, d, dtype=BF, device=DEV)
    qimg.norm_rope_packed(x, 6, 2, wq, wk, EPS, table, pos, interleaved, out=heads.permute(1, 0, 2))
    want[[5, 70]], mag[[5, 70]] = 0, 0
    _check(heads.permute(1, 0, 2), want, mag)


def test_small_and_large_values(qimg):
    """A head of zeros, of values whose squares only eps exceeds, and of 1e18."""
    x, wq, wk, g = _make(4, 1, 1, 128, 5)
    x[0], x[1], x[2] = 0, x[1] * 1e-12, x[2] * 1e18
    got = qimg.norm_rope_packed(x, 1, 1, wq, wk, EPS)
    _check(got, *_definition(x, 1, 1, wq, wk, None, None, False))
    assert bool((got[0] == 0).all())
    bad = x.clone()
    bad[3, 0, 7] = float("nan")
    out = qimg.norm_rope_packed(bad, 1, 1, wq, wk, EPS)
    assert bool(out[3, 0].isnan().all()) and torch.equal(out[3, 1:], got[3, 1:]) and torch.equal(out[:3], got[:3])


def _rows_of_cache(cache, slots):
    page = cache.k.shape[2]
    s = slots.long()
    return [value(c.view(torch.uint8)[s // page, :, s % page].view(c.dtype), e[s // page, :, s % page])
            for c, e in ((cache.k, cache.k_exp), (cache.v, cache.v_exp))]


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("tin", TYPES, ids=str)
@pytest.mark.parametrize("d,page,hk,t", [(128, 16, 4, 1), (64, 256, 3, 50), (128, 64, 24, 333), (64, 32, 1, 1000)])
def test_write_is_the_definition(qimg, codes, tin, d, page, hk, t):
    """Codes and exponents bit for bit; the rest of the cache stays as it was."""
    g = torch.Generator(device=DEV)
    g.manual_seed(t + d)
    n = -(-t // page) * 2 + 1
    cache = garbage(qimg, n, page, hk, d, codes, g)
    want = qimg.KvCache(*(x.clone() for x in cache))
    # rows from 2^-149 to 2^120 (fp16: what it holds), zeros, values on the border of two exponents and of two codes
    k, v = (torch.randn(t, hk, d, generator=g, device=DEV) for _ in range(2))
    k = k * torch.exp2(torch.randint(-20 if tin == HF else -140, 14 if tin == HF else 115, (t, hk, 1), generator=g, device=DEV))
    v[t // 3] = 0
    v[t // 2, 0] = torch.arange(d, device=DEV) * 0.5
    v[t // 2, hk - 1, :2] = torch.tensor([127.0, -448.0], device=DEV)
    k, v = k.to(tin), v.to(tin)
    slots = torch.randperm(n * page, generator=g, device=DEV)[:t].int()
    qimg.kv_cache_write(cache, k, v, slots)
    torch.cuda.synchronize()
    for dst, exps, rows in ((want.k, want.k_exp, k), (want.v, want.v_exp, v)):
        c, e = quantize(rows, codes)
        s = slots.long()
        dst.view(torch.uint8)[s // page, :, s % page] = c.view(torch.uint8)
        exps[s // page, :, s % page] = e
    for a, b, name in zip(cache, want, ("k", "v", "k_exp", "v_exp")):
        a, b = (x.view(torch.uint8) if x.dtype != torch.int8 else x for x in (a, b))
        same = (a == b) | ((a == 128) & (b == 0)) | ((a == 0) & (b == 128)) if name in "kv" and codes != torch.int8 else a == b
        assert bool(same.all()), f"{name}: {int((~same).sum())} differ"


@pytest.mark.parametrize("codes", CODES, ids=str)
def test_fp16_rows_stay_in_fp16(qimg, codes):
    """Magnitudes up to 65504 come back as fp16 values, never as infinity."""
    cache = qimg.kv_cache(1, 16, 1, 64, codes, DEV)
    k = torch.linspace(-65504, 65504, 64, device=DEV).to(HF).view(1, 1, 64).repeat(16, 1, 1)
    k *= torch.linspace(0.9, 1, 16, device=DEV).view(16, 1, 1).to(HF)
    qimg.kv_cache_write(cache, k, k, torch.arange(16, device=DEV, dtype=torch.int32))
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([16], dtype=torch.int32, device=DEV)
    back, _ = qimg.kv_cache_read(cache, table, lens, torch.tensor([0, 16], dtype=torch.int32, device=DEV), 16, out_dtype=HF)
    unit = 1024.0 if codes == torch.int8 else 2.0 ** 12 * 2  # the largest steps (e4m3: 2^5 times 2^8)
    assert bool(back.isfinite().all()) and float((back.double() - k.double()).abs().max()) <= unit


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,nq,hk,d,r,page", [(1, 28, 4, 128, 128, 64), (60, 3, 3, 64, 32, 16), (700, 8, 2, 128, 64, 128)])
def test_norm_rope_cache(qimg, codes, interleaved, t, nq, hk, d, r, page):
    x0, wq, wk, g = _make(t, nq, hk, d, t)
    n = -(-t // page) + 3
    table = _table(3000, r)
    pos = torch.randint(0, 3000, (t,), generator=g, device=DEV, dtype=torch.int32)
    for tin, tout in ((torch.float32, BF), (BF, BF), (HF, HF), (BF, torch.float32)):
        x = x0.to(tin)
        cache = garbage(qimg, n, page, hk, d, codes, g)
        before = qimg.KvCache(*(c.clone() for c in cache))
        slots = torch.randperm(n * page, generator=g, device=DEV)[:t].int()
        got = qimg.norm_rope_cache(x, nq, cache, slots, wq, wk, EPS, table, pos, interleaved, out_dtype=tout)
        torch.cuda.synchronize()
        want, mag = _definition(x, nq, hk, wq, wk, table, pos, interleaved)
        _check(got, want[:, :nq], mag[:, :nq])
        k, v = _rows_of_cache(cache, slots)
        wk64, mk = want[:, nq:nq + hk], mag[:, nq:nq + hk]
        unit = two_to(quantize(wk64, codes)[1].int() - 127)[..., None]
        # half a step of the code of a value that is itself 16 * 2^-24 of mag off (whose exponent may
        # then be the next: a step up to twice as long where the largest is next to 127 or 448)
        y = (wk64 / unit).abs().clamp(min=2.0 ** -6)
        step = unit if codes == torch.int8 else unit * two_to(torch.frexp(y * (1 + 2.0 ** -18))[1] - 4)
        top = wk64.abs().amax(-1, keepdim=True) / unit
        near = (top > (127 if codes == torch.int8 else 448) * (1 - 2.0 ** -18)).double()
        off = (k - wk64).abs() - (0.5 + 0.5 * near) * step - 16 * 2.0 ** -24 * mk
        assert float(off.max()) <= 0
        vc, ve = quantize(x[:, nq + hk:], codes)
        assert torch.equal(v, value(vc, ve))
        # nothing else of the cache has changed
        rest = torch.ones(n * page, dtype=torch.bool, device=DEV)
        rest[slots.long()] = False
        rest = rest.view(n, 1, page)
        for a, b in zip(cache, before):
            a, b = a.view(torch.uint8), b.view(torch.uint8)
            keep = rest.expand(n, hk, page) if a.dim() == 3 else rest.unsqueeze(-1).expand(n, hk, page, d)
            assert torch.equal(a[keep], b[keep])
        # the same rows by rope and a write: the same codes
        rows = qimg.norm_rope_packed(x, nq, hk, wq, wk, EPS, table, pos, interleaved, out_dtype=torch.float32)
        other = qimg.KvCache(*(c.clone() for c in before))
        if tin != HF:  # (whose rows are held inside fp16's range)
            qimg.kv_cache_write(other, rows[:, nq:nq + hk], rows[:, nq + hk:], slots)
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, other))


@pytest.mark.parametrize("codes", CODES, ids=str)
def test_tokens_without_a_slot_or_a_position(qimg, codes):
    x, wq, wk, g = _make(10, 4, 2, 64, 8)
    cache = garbage(qimg, 2, 16, 2, 64, codes, g)
    before = qimg.KvCache(*(c.clone() for c in cache))
    table = _table(10, 64)
    pos = torch.arange(10, dtype=torch.int32, device=DEV)
    pos[3] = 10
    slots = torch.tensor([-1, 32, 5, 6, -2 ** 31, 2 ** 31 - 1, 7, 8, 9, 31], dtype=torch.int32, device=DEV)
    out = torch.full((10, 4, 64), 5.0, device=DEV)
    qimg.norm_rope_cache(x, 4, cache, slots, wq, wk, EPS, table, pos, out=out)
    torch.cuda.synchronize()
    assert bool((out[3] == 5).all()) and not bool((out[[0, 1, 4, 5]] == 5).any())
    written = torch.zeros(32, dtype=torch.bool, device=DEV)
    written[[5, 7, 8, 9, 31]] = True
    for a, b in zip((cache.k_exp, cache.v_exp), (before.k_exp, before.v_exp)):
        a, b = a.transpose(1, 2).reshape(32, 2), b.transpose(1, 2).reshape(32, 2)
        assert torch.equal(a[~written], b[~written])
    k, v = _rows_of_cache(cache, slots[[2, 6, 7, 8, 9]])
    assert bool(k.isfinite().all() and v.isfinite().all())


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_rows_that_are_not_finite(qimg, codes, bad):
    """k of such a token and head is NaN whichever of the two held it, v zeros or itself; others are whole."""
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    k, v = (torch.randn(6, 3, 128, generator=g, device=DEV) for _ in range(2))
    ref = qimg.kv_cache(1, 16, 3, 128, codes, DEV)
    slots = torch.arange(6, dtype=torch.int32, device=DEV)
    qimg.kv_cache_write(ref, k, v, slots)
    k[1, 0, 100], v[2, 1, 3], k[4, 2, 0], v[4, 2, 127] = bad, bad, bad, bad
    cache = qimg.kv_cache(1, 16, 3, 128, codes, DEV)
    qimg.kv_cache_write(cache, k, v, slots)
    torch.cuda.synchronize()
    got, want = _rows_of_cache(cache, slots), _rows_of_cache(ref, slots)
    for t, h in ((1, 0), (2, 1), (4, 2)):
        assert int(cache.k_exp[0, h, t]) == 255 and bool(got[0][t, h].isnan().all())
        want[0][t, h] = float("nan")
    for t, h in ((2, 1), (4, 2)):
        want[1][t, h] = 0
    for a, b in zip(got, want):
        assert torch.equal(a.nan_to_num(1e30), b.nan_to_num(1e30))


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_code_reads_back(qimg, codes, dtype):
    """Codes times powers of two are exact in 16 bits too, where the type has the range; fp16
    rounds below 2^-14 once."""
    exps = torch.tensor([1, 60, 100, 103, 104, 113, 120, 126, 127, 128, 134], device=DEV)
    if dtype != HF:
        exps = torch.cat((exps, torch.tensor([200, 245], device=DEV)))
    n = exps.numel()
    c = torch.arange(256, device=DEV).to(torch.uint8).view(1, 2, 1, 128).repeat(1, 1, 16, 1)
    cache = qimg.kv_cache(1, 16, 2, 128, codes, DEV)
    cache.k.view(torch.uint8).copy_(c)
    cache.v.view(torch.uint8).copy_(c.flip(3))
    cache.k_exp[0, :, :n], cache.v_exp[0, :, :n] = exps.to(torch.uint8), exps.to(torch.uint8)
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    got = qimg.kv_cache_read(cache, torch.zeros(1, 1, dtype=torch.int32, device=DEV), lens,
                             torch.tensor([0, n], dtype=torch.int32, device=DEV), n, out_dtype=dtype)
    torch.cuda.synchronize()
    for a, codes_, e in ((got[0], cache.k, cache.k_exp), (got[1], cache.v, cache.v_exp)):
        want = value(codes_, e)[0].transpose(0, 1)[:n]
        assert torch.equal(a.nan_to_num(77.0), want.to(dtype).nan_to_num(77.0))
        assert torch.equal(a.isnan(), want.isnan())


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("page,hk,d", [(16, 4, 128), (256, 1, 64), (32, 24, 64), (64, 3, 128)])
@pytest.mark.parametrize("lens", [[1], [0], [5, 0, 300, 1, 0, 77], [1000, 31, 32, 33], [3] * 100], ids=str)
def test_read(qimg, codes, page, hk, d, lens):
    g = torch.Generator(device=DEV)
    g.manual_seed(sum(lens) + page)
    k, v = (torch.randn(sum(lens), hk, d, generator=g, device=DEV) for _ in range(2))
    cache = garbage(qimg, sum(-(-x // page) for x in lens) + 3, page, hk, d, codes, g)
    table, slots = fill(cache, lens, k, v, g)
    room = [x + 2 for x in lens]  # rows between the sequences stay as they are
    cu = [0]
    for x in room:
        cu.append(cu[-1] + x)
    total = cu[-1] + 5
    kl, cu_d = torch.tensor(lens, dtype=torch.int32, device=DEV), torch.tensor(cu, dtype=torch.int32, device=DEV)
    ko = torch.full((total, hk, d + 8), 9.0, dtype=BF, device=DEV)
    vo = torch.full((hk, total, d), 9.0, dtype=BF, device=DEV)
    qimg.kv_cache_read(cache, table, kl, cu_d, total, k_out=ko[:, :, :d], v_out=vo.transpose(0, 1))
    torch.cuda.synchronize()
    rows = torch.tensor([cu[b] + i for b, x in enumerate(lens) for i in range(x)], device=DEV, dtype=torch.long)
    wk, wv = _rows_of_cache(cache, slots)
    assert torch.equal(ko[rows][:, :, :d].double(), wk) and torch.equal(vo[:, rows].transpose(0, 1).double(), wv)
    keep = torch.ones(total, dtype=torch.bool, device=DEV)
    keep[rows] = False
    assert bool((ko[keep] == 9).all() and (ko[:, :, d:] == 9).all() and (vo[:, keep] == 9).all())


def test_read_within_its_lists(qimg):
    """Lengths past the table, pages outside the cache and offsets that are no list of sequences read
    and write nothing outside the tensors."""
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    k = torch.randn(64, 2, 64, generator=g, device=DEV)
    cache = qimg.kv_cache(4, 16, 2, 64, torch.int8, DEV)
    qimg.kv_cache_write(cache, k, k, torch.arange(64, dtype=torch.int32, device=DEV))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    out = [torch.full((40, 2, 64), 9.0, device=DEV) for _ in range(2)]
    qimg.kv_cache_read(cache, i32(1, -1, 4, 2).view(2, 2), i32(1000, 20), i32(0, 36, 60), 40, k_out=out[0], v_out=out[1])
    torch.cuda.synchronize()
    want = torch.full((40, 2, 64), 9.0, dtype=torch.float64, device=DEV)
    val = value(cache.k, cache.k_exp)
    want[:16] = val[1].transpose(0, 1)          # page 1; page -1 and what lies behind the table are left
    assert torch.equal(out[0].double(), want)   # (sequence 1 begins in page 4, outside; rows 36 .. 39)
    for cu in ([30, 10, 20], [-5, 100, 50], [2 ** 31 - 1, -2 ** 31, 0]):
        qimg.kv_cache_read(cache, i32(1, 2, 0, 3).view(2, 2), i32(32, 32), i32(*cu), 40, k_out=out[0], v_out=out[1])
    torch.cuda.synchronize()
