"""GPU parity: attention over the pages of a quantized cache, without and behind a shared
prefix (qimg_attention_cache), against the definition in 64 bits on the values that the
codes stand for.

Tolerance, from the arithmetic (that of packed attention, since codes enter the products
exactly): with u = eps / 2 of q's type P is rounded to the type (relative u on every p_j,
and on the same rounded values in the row sum) and the result once more; both are bounded
by u sum_j p_j |v_j - o| + u |o| <= 2 u (sum_j p_j |v_j| + |o|). The fp32 parts add less:
a score's error, about sum |q k| D 2^-24, moves p by that much, covered by 2^-20
sum_j p_j |v_j| (scores here stay below 64 in magnitude). fp16 weights below 2^-21 of the
largest are off by up to 2^-32 of it each: with n keys 2^-32 n max|v| more."""
import math

import pytest
import torch

from cacheutil import BF, CODES, HF, fill, garbage, value

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return _i32(*c), c


class Case:
    """Queries, a cache of noise that holds the sequences' and the prefix' rows, their tables."""

    def __init__(self, qimg, lq, lk, prefix=0, hq=28, hk=4, d=128, dtype=BF, codes=torch.int8, page=64, seed=0, scale=1.0):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        self.lq, self.lk, self.prefix, self.hk = lq, lk, prefix, hk
        self.q = torch.randn(sum(lq), hq, d, generator=g, device=DEV).to(dtype)
        lens = lk + [prefix]
        n = sum(lens)
        k = torch.randn(n, hk, d, generator=g, device=DEV) + 0.5
        v = torch.randn(n, hk, d, generator=g, device=DEV) * scale
        self.cache = garbage(qimg, sum(-(-x // page) for x in lens) + 3, page, hk, d, codes, g)
        table, slots = fill(self.cache, lens, k, v, g)
        self.table = table[:-1].contiguous()
        self.prefix_table = table[-1, :max(1, -(-prefix // page))].contiguous()
        s = slots.long()
        self.k, self.v = (value(c.view(torch.uint8)[s // page, :, s % page].view(c.dtype), e[s // page, :, s % page])
                          for c, e in ((self.cache.k, self.cache.k_exp), (self.cache.v, self.cache.v_exp)))
        self.cu_q, self.cq = _cu(lq)
        self.ck = _cu(lens)[1]
        self.k_lens = _i32(*lk)

    def run(self, qimg, causal=True, with_prefix=None, **kw):
        if self.prefix if with_prefix is None else with_prefix:
            kw.update(prefix_table=self.prefix_table, prefix_len=_i32(self.prefix))
        return qimg.attention_cache(self.q, self.cache, self.cu_q, self.table, self.k_lens, causal=causal, **kw)

    def oracle(self, causal=True, scale=None):
        """The definition, sum_j p_j |v_j| and max |v| n beside it."""
        d = self.q.shape[2]
        scale = 1.0 / math.sqrt(d) if scale is None else scale
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=DEV)
        mag, far = torch.zeros_like(out), torch.zeros_like(out)
        group, p0, pn = self.q.shape[1] // self.hk, self.ck[-2], self.prefix
        for b, (nq, nk) in enumerate(zip(self.lq, self.lk)):
            if nq == 0 or nk + pn == 0:
                continue
            at = torch.cat((torch.arange(p0, p0 + pn, device=DEV), torch.arange(self.ck[b], self.ck[b] + nk, device=DEV)))
            vis = torch.ones(nq, pn + nk, dtype=torch.bool, device=DEV)
            own = torch.arange(nk, device=DEV)
            if causal:
                vis[:, pn:] = own[None] <= torch.arange(nq, device=DEV)[:, None] + (nk - nq)
            none = ~vis.any(-1)
            for h in range(self.q.shape[1]):
                kk, vv = self.k[at, h // group], self.v[at, h // group]
                x = self.q[self.cq[b]:self.cq[b + 1], h].double() @ kk.t() * scale
                p = torch.softmax(x.masked_fill(~vis, -math.inf), dim=-1)
                p[none] = 0
                out[self.cq[b]:self.cq[b + 1], h] = p @ vv
                mag[self.cq[b]:self.cq[b + 1], h] = p @ vv.abs()
                far[self.cq[b]:self.cq[b + 1], h] = vv.abs().amax() * (pn + nk)
        return out, mag, far


def _check(got, want, mag, far):
    i = torch.finfo(got.dtype)
    u = i.eps / 2
    tol = 2 * u * (mag + want.abs()) + 2.0 ** -20 * mag + i.tiny + (2.0 ** -32 * far if got.dtype == HF else 0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"max excess {float((err - tol).max())}, max err {float(err.max())}"


def _run(qimg, lq, lk, causal=True, **kw):
    c = Case(qimg, lq, lk, **kw)
    got = c.run(qimg, causal)
    torch.cuda.synchronize()
    _check(got, *c.oracle(causal))
    return got


LENS = [([1], [1]), ([1], [0]), ([1, 1, 1], [15, 16, 17]), ([1], [33]), ([1, 0, 2], [64, 5, 1]), ([1] * 5, [31, 32, 0, 127, 129]),
        ([3], [2]), ([5, 1], [5, 300]), ([0, 0, 7], [9, 0, 100]), ([1] * 70, list(range(70)))]


@pytest.mark.parametrize("lq,lk", LENS, ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 256])
def test_tokens(qimg, lq, lk, d, page):
    for i, (dtype, codes) in enumerate([(BF, CODES[0]), (BF, CODES[1]), (HF, CODES[0]), (HF, CODES[1])]):
        _run(qimg, lq, lk, causal=i != 1, d=d, page=page, dtype=dtype, codes=codes, seed=len(lq) + i)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("codes", CODES, ids=str)
def test_long_caches_in_ranges(qimg, page, codes):
    """Keys cut into ranges and joined: unlike lengths, one long sequence, many."""
    for dtype in (BF, HF):
        _run(qimg, [1] * 6, [5000, 17, 1025, 2048, 0, 4097], page=page, codes=codes, dtype=dtype, seed=page)
    _run(qimg, [1], [20000], page=page, codes=codes, seed=1)
    _run(qimg, [2] * 40, [700 + 13 * i for i in range(40)], hq=8, hk=8, d=64, page=page, codes=codes, seed=2)


@pytest.mark.parametrize("hq,hk", [(1, 1), (7, 1), (5, 5), (24, 8), (32, 1), (40, 2)])
@pytest.mark.parametrize("lq,lk", [([1, 4], [700, 90]), ([9], [2000])], ids=str)
def test_head_groups(qimg, hq, hk, lq, lk):
    _run(qimg, lq, lk, hq=hq, hk=hk, seed=hq)
    _run(qimg, lq, lk, hq=hq, hk=hk, seed=hq, codes=CODES[1], dtype=HF, d=64, page=16)


PIECES = [([70, 9], [70, 200]), ([300], [300]), ([128, 129, 1, 40], [1000, 129, 800, 41]), ([512], [3000]), ([64] * 12, [64] * 12),
          ([257, 0, 13], [100, 50, 2000])]


@pytest.mark.parametrize("lq,lk", PIECES, ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_pieces_of_prompts(qimg, lq, lk, d, causal):
    for i, (dtype, codes) in enumerate([(BF, CODES[0]), (BF, CODES[1]), (HF, CODES[0]), (HF, CODES[1])]):
        _run(qimg, lq, lk, causal, d=d, page=(16, 32, 64, 128)[i], dtype=dtype, codes=codes, seed=len(lq) + d)


@pytest.mark.parametrize("lq,lk", PIECES[1:] + [([1, 0, 160], [3, 9, 900])], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_pieces_of_many_rows(qimg, lq, lk, d):
    """Ten q heads to a kv head and eight of those: tiles of 128 rows."""
    for i, (dtype, codes) in enumerate([(BF, CODES[0]), (BF, CODES[1]), (HF, CODES[0]), (HF, CODES[1])]):
        _run(qimg, lq, lk, i != 1, hq=80, hk=8, d=d, page=(256, 16, 32, 64)[i], dtype=dtype, codes=codes, seed=len(lq) + d)


PREFIXES = [([1], [1], 1), ([1] * 3, [5, 0, 40], 100), ([1] * 20, [0] * 20, 700), ([2, 0, 3], [40, 3, 0], 33), ([1] * 40, list(range(1, 41)), 2000),
            ([200, 31], [200, 300], 500), ([1] * 5, [1, 2, 3, 4, 5], 0), ([4] * 30, [64 * i for i in range(30)], 3000),
            ([1] * 130, [1 + i % 50 for i in range(130)], 9000)]


@pytest.mark.parametrize("lq,lk,prefix", PREFIXES, ids=lambda x: str(x)[:40])
@pytest.mark.parametrize("d", [64, 128])
def test_prefix(qimg, lq, lk, prefix, d):
    for i, (dtype, codes) in enumerate([(BF, CODES[0]), (BF, CODES[1]), (HF, CODES[0]), (HF, CODES[1])]):
        c = Case(qimg, lq, lk, prefix, d=d, page=(16, 32, 64, 256)[i], dtype=dtype, codes=codes, seed=prefix + d,
                 hq=(28, 8, 6, 24)[i], hk=(4, 8, 1, 24)[i])
        got = c.run(qimg, i != 2, with_prefix=True)
        torch.cuda.synchronize()
        _check(got, *c.oracle(i != 2))


@pytest.mark.parametrize("lq,lk,prefix", PREFIXES[1:], ids=lambda x: str(x)[:40])
@pytest.mark.parametrize("d", [64, 128])
def test_prefix_tables_with_room(qimg, lq, lk, prefix, d):
    """Behind a table of that many keys the prefix takes tiles of 128 rows; its length is the device's."""
    for i, (dtype, codes) in enumerate([(BF, CODES[0]), (HF, CODES[1])]):
        page = (32, 256)[i]
        c = Case(qimg, lq, lk, prefix, d=d, page=page, dtype=dtype, codes=codes, seed=prefix + d, hq=(28, 48)[i], hk=(4, 24)[i])
        tiles = -(-sum(lq) * c.q.shape[1] // c.hk // 16)
        wide = torch.full((60001 * 32 // (tiles * c.hk * page) + 2 + c.prefix_table.numel(),), -1, dtype=torch.int32, device=DEV)
        wide[:c.prefix_table.numel()] = c.prefix_table
        c.prefix_table = wide
        got = c.run(qimg, with_prefix=True)
        torch.cuda.synchronize()
        _check(got, *c.oracle())


@pytest.mark.parametrize("prefix,longest", [(0, 30), (0, 3000), (100, 30)])
def test_thousands_of_sequences(qimg, prefix, longest):
    """More sequences than a wave looks over at once, and more tiles than workgroups: some empty, one long."""
    lq = [(1, 0, 2, 1, 3)[i % 5] for i in range(5000)]
    lk = [i % 31 for i in range(5000)]
    lq[4321], lk[4321] = 2, longest
    c = Case(qimg, lq, lk, prefix, hq=2, hk=1, d=64, page=16, codes=CODES[1], seed=21)
    got = c.run(qimg)
    torch.cuda.synchronize()
    _check(got, *c.oracle())


def test_prefix_pages_in_the_tables_instead(qimg):
    """A prefix in front of every sequence's own table gives the same within the bounds."""
    c = Case(qimg, [1] * 9, [3 + i for i in range(9)], prefix=256, page=16, seed=4)
    shared = c.prefix_table[None].expand(9, -1)
    got = qimg.attention_cache(c.q, c.cache, c.cu_q, torch.cat((shared, c.table), 1).contiguous(), c.k_lens + 256)
    _check(got, *c.oracle())


def test_values_of_any_size(qimg):
    """V and K rows of very unlike powers of two, rows of zeros, constant rows."""
    for dtype, top in ((BF, 100), (HF, 8)):
        for codes in CODES:
            c = Case(qimg, [1] * 4 + [3], [100, 1, 300, 64, 700], dtype=dtype, codes=codes, seed=6)
            g = torch.Generator(device=DEV)
            g.manual_seed(7)
            c.cache.v_exp[c.cache.v_exp != 0] = 127
            n, hk, page = c.cache.v_exp.shape
            shift = torch.randint(-top, top, (n, hk, page), generator=g, device=DEV)
            c.cache.v_exp.copy_((127 + shift - (7 if codes == torch.int8 else 9)).to(torch.uint8))
            c.cache.v.view(torch.uint8)[:, :, ::5] = 0
            c.cache.v.view(torch.uint8)[c.cache.v.view(torch.uint8) & 0x7f == 0x7f] = 0
            k64 = []
            for b, x in enumerate(c.lk):
                p = c.table[b, :-(-x // page)].long()
                k64.append(value(c.cache.v[p] if codes == torch.int8 else c.cache.v.view(torch.uint8)[p].view(codes),
                                 c.cache.v_exp[p]).transpose(1, 2).reshape(-1, hk, 128)[:x])
            c.v = torch.cat(k64 + [c.v[:0]])
            got = c.run(qimg)
            torch.cuda.synchronize()
            _check(got, *c.oracle())


def test_constant_values_come_back_exactly(qimg):
    c = Case(qimg, [1, 5], [3000, 77], seed=8, codes=CODES[1])
    c.cache.v.view(torch.uint8).fill_(0x38)  # 1.0
    c.cache.v_exp.fill_(128)
    got = c.run(qimg)
    assert bool((got == 2).all())


@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [100, 2000, 31]), ([150, 60, 3], [200, 60, 2000])], ids=str)
@pytest.mark.parametrize("hq,hk", [(8, 2), (80, 8)])
def test_a_token_that_is_not_finite(qimg, codes, lq, lk, hq, hk):
    """Rows that see it are NaN, in its kv head alone; the others do not change."""
    c = Case(qimg, lq, lk, seed=9, codes=codes, page=32, hq=hq, hk=hk)
    base = c.run(qimg)
    n, hk, page, d = c.cache.k.shape
    key = lk[0] - 1  # the last key of sequence 0: of a piece its last query alone sees it
    slot = int(c.table[0, key // page]) * page + key % page
    rows = torch.ones(1, hk, d, device=DEV)
    rows[0, 1, 5] = float("nan")
    for which in (0, 1):
        cache = qimg.KvCache(*(x.clone() for x in c.cache))
        both = [torch.ones_like(rows), rows] if which else [rows, torch.ones_like(rows)]
        qimg.kv_cache_write(cache, *both, _i32(slot))
        got = qimg.attention_cache(c.q, cache, c.cu_q, c.table, c.k_lens)
        torch.cuda.synchronize()
        seen = torch.arange(hq, device=DEV) // (hq // hk) == 1
        assert bool(got[lq[0] - 1, seen].isnan().all())
        assert not bool(got[lq[0] - 1, ~seen].isnan().any())
        keep = torch.ones(sum(lq), dtype=torch.bool, device=DEV)
        keep[lq[0] - 1] = False
        assert torch.equal(got[keep], base[keep])


@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [300, 3000, 40]), ([100, 40, 3], [300, 200, 90])], ids=str)
@pytest.mark.parametrize("codes", CODES, ids=str)
@pytest.mark.parametrize("hq,hk", [(28, 4), (96, 8)])
def test_pages_outside_the_cache(qimg, lq, lk, codes, hq, hk):
    """Nothing outside the cache is read: rows that see a key there are NaN, the others do not change."""
    for bad in (-1, 2 ** 31 - 1, -2 ** 31, None):
        c = Case(qimg, lq, lk, page=16, seed=10, prefix=64, codes=codes, hq=hq, hk=hk)
        base = c.run(qimg)
        key = 240  # of sequence 0: its last 60 queries' keys reach there
        c.table[0, key // 16] = c.cache.k.shape[0] if bad is None else bad
        got = c.run(qimg)
        torch.cuda.synchronize()
        seen = torch.arange(lq[0], device=DEV) + lk[0] - lq[0] >= key
        assert bool(got[:lq[0]][seen].isnan().all())
        assert torch.equal(got[:lq[0]][~seen], base[:lq[0]][~seen]) and torch.equal(got[lq[0]:], base[lq[0]:])
        c.prefix_table[1] = -1
        assert bool(c.run(qimg).isnan().all())


@pytest.mark.parametrize("lq,lk,prefix", [([1] * 3, [700, 4000, 9], 0), ([130, 20], [130, 300], 0), ([1] * 30, [40] * 30, 800),
                                          ([600, 20], [1300, 300], 0), ([1] * 100, [40] * 100, 12000)])
def test_views_and_rows_of_no_sequence(qimg, lq, lk, prefix):
    c = Case(qimg, lq, lk, prefix, seed=12)
    want = c.run(qimg)
    t = sum(lq)
    proj = torch.full((t + 4, 36, 128), float("nan"), dtype=BF, device=DEV)  # a packed projection, rows behind the last
    proj[:t, :28] = c.q
    room = torch.full((30, t + 4, 136), 7.0, dtype=BF, device=DEV)  # head-major
    c.q = proj[:, :28]
    c.run(qimg, out=room.permute(1, 0, 2)[:, :28, :128])
    torch.cuda.synchronize()
    assert torch.equal(room[:28, :t, :128].permute(1, 0, 2), want)
    assert bool((room[:, t:] == 7).all() and (room[28:] == 7).all() and (room[:, :, 128:] == 7).all())


@pytest.mark.parametrize("m", [1, 100])
def test_offsets_and_lengths_outside_are_clamped(qimg, m):
    c = Case(qimg, [3 * m, 4 * m, 2 * m], [40, 50, 60], prefix=32, page=16, seed=13)
    out = torch.empty_like(c.q)
    for cu in ([0, 5, 3, 20], [-7, 3, 7, 2 ** 31 - 1], [9, 6, 3, 0], [-2 ** 31, 0, 0, 9]):
        cu = [x * m if abs(x) < 100 else x for x in cu]
        for kl in ([2 ** 31 - 1, -5, 1000], [-2 ** 31, 64, 0]):
            for pl in (-1, 10 ** 9):
                qimg.attention_cache(c.q, c.cache, _i32(*cu), c.table, _i32(*kl), prefix_table=c.prefix_table,
                                     prefix_len=_i32(pl), out=out)
    torch.cuda.synchronize()
    # a length past the table is the table's
    full = c.table.shape[1] * 16
    c.table.clamp_(max=c.cache.k.shape[0] - 1)
    c.cache.k_exp.clamp_(max=130), c.cache.v_exp.clamp_(max=130)
    a = qimg.attention_cache(c.q, c.cache, c.cu_q, c.table, _i32(10 ** 9, full, full + 1))
    b = qimg.attention_cache(c.q, c.cache, c.cu_q, c.table, _i32(full, full, full))
    assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))


@pytest.mark.parametrize("lq,lk,prefix", [([1] * 3, [700, 4000, 9], 0), ([130, 20], [1300, 300], 0), ([1] * 30, [40] * 30, 800),
                                          ([600, 20], [1300, 300], 0), ([1] * 100, [40] * 100, 12000)])
def test_replays_other_streams_and_repeats(qimg, lq, lk, prefix):
    """A captured call follows the lists on the device; the same call gives the same bits."""
    c = Case(qimg, lq, lk, prefix, seed=14)
    first = c.run(qimg)
    assert torch.equal(first, c.run(qimg))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = c.run(qimg)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
    need = qimg.attention_cache_scratch_bytes(sum(lq), len(lq), 28, 4, 128, 64, c.table.shape[1],
                                              c.prefix_table.numel() if prefix else 0)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    out, pl = torch.zeros_like(c.q), _i32(prefix)
    more = dict(prefix_table=c.prefix_table, prefix_len=pl) if prefix else {}
    call = lambda o: qimg.attention_cache(c.q, c.cache, c.cu_q, c.table, c.k_lens, out=o, scratch=scratch, **more)  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for n in range(4):
        lens = [max(0, x - 7 * n) for x in lk]
        c.k_lens.copy_(_i32(*lens))
        pl.copy_(_i32(max(0, prefix - 100 * n)))
        scratch.fill_(255 if n % 2 else 127)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = call(torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        c.lk, c.prefix = lens, max(0, prefix - 100 * n)
    # (the rows of the sequences' ends and of the prefix are the first of the same pages)


def test_tables_with_room_for_a_million_keys(qimg):
    """Tiles of many rows make their keys' 16-bit rows a few heads and sequences at a time where the
    tables have room for more than scratch should hold."""
    for prefix in (0, 300):
        c = Case(qimg, [100, 300, 7], [130, 1000, 600], prefix, hq=32, hk=4, page=256, codes=CODES[1], seed=16)
        wide = torch.full((3, 4096), -1, dtype=torch.int32, device=DEV)
        wide[:, :c.table.shape[1]] = c.table
        c.table = wide
        if prefix:
            more = torch.full((9000,), 2 ** 30, dtype=torch.int32, device=DEV)
            more[:c.prefix_table.numel()] = c.prefix_table
            c.prefix_table = more
        need = qimg.attention_cache_scratch_bytes(407, 3, 32, 4, 128, 256, 4096, 9000 if prefix else 0)
        assert 1 << 30 <= need < 5 << 30
        got = c.run(qimg)
        torch.cuda.synchronize()
        _check(got, *c.oracle())


def test_caches_past_32_bits(qimg):
    """Codes of more than 2^32 bytes: pages at their far end."""
    page, hk, d = 256, 8, 128
    n = (1 << 32) // (page * hk * d) + 20
    k, v = (torch.empty(n, hk, page, d, dtype=torch.uint8, device=DEV).view(torch.int8) for _ in range(2))
    ke, ve = (torch.empty(n, hk, page, dtype=torch.uint8, device=DEV) for _ in range(2))
    big = qimg.KvCache(k, v, ke, ve)
    small = Case(qimg, [1, 700], [700, 900], hq=16, hk=hk, d=d, page=page, seed=15, prefix=300)
    m = small.cache.k.shape[0]
    for dst, src in zip(big, small.cache):
        dst[n - m:].copy_(src)
    want = small.run(qimg)
    small.cache = big
    small.table += n - m
    small.prefix_table += n - m
    small.table.clamp_(max=n + 7)
    got = small.run(qimg)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    rows = torch.randn(5, hk, d, device=DEV)
    slots = _i32(*[(n - 1) * page + i for i in range(5)])
    qimg.kv_cache_write(big, rows, rows, slots)
    back = qimg.kv_cache_read(big, _i32(n - 1).view(1, 1), _i32(5), _i32(0, 5), 5, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert float((back[0] - rows).abs().max()) < 0.05 and torch.equal(*back)
