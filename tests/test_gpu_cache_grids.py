"""GPU: the operators around a quantized key/value cache at sizes of more workgroups than one
launch takes (2^22 of 256 threads; a grid has less than 2^32 threads). Each result is held
against the same call on a part of the rows, whose sizes the other tests hold against the
definitions."""
import pytest
import torch

from cacheutil import BF
from test_gpu_attention_cache import Case, _check, _i32

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def _room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory")


def _same(a, b):
    """Equal bits, without a copy of the whole (and never of more than 2^31 elements at a time)."""
    a, b = a.flatten(), b.flatten()
    return all(torch.equal(x, y) for x, y in zip(a.split(1 << 30), b.split(1 << 30)))


# 32 heads of at most 64, 16 of 128 and 8 of 256 a workgroup: two launches, the last with sizes past 2^32 threads
@pytest.mark.parametrize("t,nq,nk,d", [((1 << 27) + 3, 1, 0, 8), ((1 << 24) + 5, 1, 2, 128), ((1 << 24) + 5, 1, 1, 136),
                                       ((1 << 29) + 70, 1, 0, 8)])
def test_norm_rope_packed(qimg, t, nq, nk, d):
    h = nq + 2 * nk
    _room((2 * 2 * t * h * d + 4 * t >> 30) + 8)
    g = torch.Generator(device=DEV)
    g.manual_seed(d)
    x = torch.empty(t, h, d, dtype=BF, device=DEV)
    x.view(torch.int16).random_(0x3000, 0x4100, generator=g)  # 5e-10 to 8
    w = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(BF)
    a = torch.rand(1000, d // 2, generator=g, device=DEV) * 6
    cs = torch.stack((a.cos(), a.sin()), -1)
    pos = torch.arange(t, dtype=torch.int32, device=DEV) % 1000
    got = qimg.norm_rope_packed(x, nq, nk, w, w, 1e-6, cs, pos)
    per, launch = 1 << 20, (1 << 22) * (32 if d <= 64 else 16 if d <= 128 else 8) // h
    assert launch < t
    for lo in (0, t // 2, min(launch - per // 2, t - per), t - per):
        part = qimg.norm_rope_packed(x[lo:lo + per], nq, nk, w, w, 1e-6, cs, pos[lo:lo + per].contiguous())
        assert _same(got[lo:lo + per].view(torch.int16), part.view(torch.int16)), lo


@pytest.mark.parametrize("norm", [False, True])
def test_rows_into_the_cache(qimg, norm):
    """2^26 tokens and more of one head of 128: those behind the first launch reach their slots."""
    t, d, page = (1 << 26) + 100, 128, 16
    _room(8)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    rows = torch.randn(8 * t + 4 * d, generator=g, device=DEV, dtype=BF)  # token t's values from 8 t on
    slots = torch.full((t,), -1, dtype=torch.int32, device=DEV)
    at = torch.tensor([0, 5, (1 << 26) - 1, 1 << 26, t - 2, t - 1], device=DEV)
    mine = torch.arange(6, dtype=torch.int32, device=DEV) * 3
    slots[at] = mine
    big, small = (qimg.kv_cache(2, page, 1, d, device=DEV) for _ in range(2))
    if norm:
        x = rows.as_strided((t, 2, d), (8, d, 1))
        w = torch.ones(d, dtype=BF, device=DEV)
        qimg.norm_rope_cache(x, 0, big, slots, None, w)
        qimg.norm_rope_cache(x[at], 0, small, mine, None, w)
    else:
        k, v = rows.as_strided((t, 1, d), (8, d, 1)), rows[d:].as_strided((t, 1, d), (8, d, 1))
        qimg.kv_cache_write(big, k, v, slots)
        qimg.kv_cache_write(small, k[at], v[at], mine)
    torch.cuda.synchronize()
    assert bool((small.k.view(torch.uint8) != 0).any())
    for a, b in zip(big, small):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("total", [(1 << 27) + 1000, (1 << 29) + 1000])
def test_rows_back_from_the_cache(qimg, total):
    """Sequences that begin behind 2^27 and 2^29 rows; most rows belong to none."""
    d, page = 64, 16
    _room((2 * 2 * d * total >> 30) + 4)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    cache = qimg.kv_cache(4, page, 1, d, device=DEV)
    rows = torch.randn(64, 1, d, generator=g, device=DEV)
    qimg.kv_cache_write(cache, rows, 2 * rows, torch.arange(64, dtype=torch.int32, device=DEV))
    table = _i32(3, 1, 0, 2, 2, 3).view(3, 2)
    lens, cu = _i32(20, 32, 31), _i32(0, total - 500, total - 100, total)
    small = qimg.kv_cache_read(cache, table, lens, _i32(0, 20, 52, 83), 83)
    out = [torch.empty(total, 1, d, dtype=BF, device=DEV) for _ in range(2)]
    for o in out:
        o[-600:] = 7
    qimg.kv_cache_read(cache, table, lens, cu, total, k_out=out[0], v_out=out[1])
    torch.cuda.synchronize()
    for o, s in zip(out, small):
        assert torch.equal(o[:20], s[:20])
        assert torch.equal(o[total - 500:total - 468], s[20:52])
        assert torch.equal(o[total - 100:total - 69], s[52:])
        assert bool((o[total - 600:total - 500] == 7).all() and (o[total - 468:total - 100] == 7).all()
                    and (o[total - 69:] == 7).all())


@pytest.mark.parametrize("lq", [[1, 2, 1], [81]])
def test_a_prefix_of_many_keys(qimg, lq):
    """A prefix of more than 2^28 keys, whose 16-bit rows are made by two launches, beside the
    sequences' own tiles or without them: the last page's alone have weights, the others' sum to
    2^28 e^-60 < 2^-57 of theirs."""
    page, d = 256, 64
    _room(100)
    n = (1 << 28) // page + 9
    c = Case(qimg, lq, [0] * len(lq), page, hq=128, hk=1, d=d, page=page, seed=3)
    c.q = c.q.abs() + 0.5
    last = int(c.prefix_table[0])
    other = (last + 1) % c.cache.k.shape[0]
    low = torch.full((page, 1, d), -8.0, device=DEV)
    qimg.kv_cache_write(c.cache, low, torch.randn_like(low), other * page + torch.arange(page, dtype=torch.int32, device=DEV))
    top = c.q[:, :, None].double() @ torch.cat((c.k[:, 0], low[:1, 0].double())).t() / d ** 0.5
    assert float((top[..., :-1].amax(-1) - top[..., -1:].squeeze(-1)).min()) > 60
    want = c.oracle()
    c.prefix_table = torch.full((n,), other, dtype=torch.int32, device=DEV)
    c.prefix_table[-1] = last
    c.prefix = n * page
    need = qimg.attention_cache_scratch_bytes(sum(lq), len(lq), 128, 1, d, page, c.table.shape[1], n)
    assert need > 4 * d * page * n  # the prefix's tiles have 128 rows
    got = c.run(qimg)
    torch.cuda.synchronize()
    _check(got, *want)
