"""The operators around a quantized key/value cache run together, as one layer of a
prompt encoder that writes several variants of a prompt uses them: a template's keys
once in pages of their own, the variants' prompts behind it, then one new token of each
at a time, captured into a graph. Projection, norms and rotation of the heads into the
cache, attention over it, output projection.

Every step is held against its definition in 64 bits on the inputs that the step before
gave. Heads: 16 units of 2^-24 of the magnitudes that are added, and the rounding. Rows in
the cache: half a step of their codes besides, of the exponent that stands there, which has
to be the least one. Attention: 2 u (sum p |v| + |o|) + 2^-20 sum p |v| over the values that
the cache holds. Products: 2 sqrt(K) 2^-24 sum |x w|."""
import math

import pytest
import torch

from cacheutil import BF, CODES, garbage, two_to, value

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HK, D, HID, EPS = 12, 4, 64, 768, 1e-6
PAGE = 32
TEMPLATE, PROMPTS, STEPS = 300, [40, 1, 77, 130, 64], 70


def _i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


class Layer:
    def __init__(self, qimg, codes):
        g = torch.Generator(device=DEV)
        g.manual_seed(3)
        rn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
        self.qimg, self.g, self.codes = qimg, g, codes
        self.wqkv, self.wo = (0.05 * rn((HQ + 2 * HK) * D, HID)).to(BF), (0.04 * rn(HID, HQ * D)).to(BF)
        self.wq, self.wk = (1 + 0.2 * rn(D)).to(BF), (1 + 0.2 * rn(D)).to(BF)
        f = torch.pow(10000.0, -torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
        a = torch.arange(1000, dtype=torch.float64, device=DEV)[:, None] * f
        self.cs = torch.stack((a.cos(), a.sin()), -1).float()
        each = [-(-(n + STEPS) // PAGE) for n in PROMPTS]
        shared = -(-TEMPLATE // PAGE)
        order = torch.randperm(sum(each) + shared + 5, generator=g, device=DEV)
        self.cache = garbage(qimg, len(order), PAGE, HK, D, codes, g)
        self.prefix_table = order[:shared].int()
        self.table = torch.full((len(PROMPTS), max(each)), -1, dtype=torch.int32, device=DEV)
        at = shared
        for b, n in enumerate(each):
            self.table[b, :n] = order[at:at + n]
            at += n

    def slots(self, pages, lo, hi):
        i = torch.arange(lo, hi, device=DEV)
        return pages.long()[i // PAGE] * PAGE + i % PAGE

    def rows(self, pages, n):
        """What the first n keys of some pages stand for: k and v [n, Hk, D], fp64."""
        s = self.slots(pages, 0, n)
        c = self.cache
        return [value(x.view(torch.uint8)[s // PAGE, :, s % PAGE].view(x.dtype), e[s // PAGE, :, s % PAGE])
                for x, e in ((c.k, c.k_exp), (c.v, c.v_exp))]

    def __call__(self, x, slots, pos, cu, k_lens, table, prefix_len=None):
        q = self.qimg
        qkv = q.linear_forward_bf16_fused(x, self.wqkv, out_dtype=torch.float32).view(-1, HQ + 2 * HK, D)
        heads = q.norm_rope_cache(qkv, HQ, self.cache, slots, self.wq, self.wk, EPS, self.cs, pos, out_dtype=BF)
        more = {} if prefix_len is None else dict(prefix_table=self.prefix_table, prefix_len=prefix_len)
        attn = q.attention_cache(heads, self.cache, cu, table, k_lens, **more)
        return qkv, heads, attn, q.linear_forward_bf16_fused(attn.view(-1, HQ * D), self.wo, out_dtype=torch.float32)

    def check(self, x, slots, pos, lq, lens, tables, prefix, qkv, heads, attn, out):
        z, w = x.double(), self.wqkv.double()
        tol = 2 * math.sqrt(HID) * 2.0 ** -24 * (z.abs() @ w.abs().t())
        assert bool(((qkv.view(len(x), -1).double() - z @ w.t()).abs() <= tol).all())

        want = qkv.double()
        for lo, hi, w in ((0, HQ, self.wq), (HQ, HQ + HK, self.wk)):
            y = want[:, lo:hi]
            want[:, lo:hi] = y / ((y ** 2).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
        n, cs = HQ + HK, self.cs.double()[pos.long()][:, None]
        c, s = cs[..., 0], cs[..., 1]
        mag = torch.zeros_like(want)
        a, b = want[:, :n, :D // 2].clone(), want[:, :n, D // 2:].clone()
        want[:, :n, :D // 2], want[:, :n, D // 2:] = a * c - b * s, b * c + a * s
        mag[:, :n, :D // 2], mag[:, :n, D // 2:] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
        err = 16 * 2.0 ** -24 * mag
        u = torch.finfo(BF).eps / 2
        assert bool(((heads.double() - want[:, :HQ]).abs() <= err[:, :HQ] + u * (want[:, :HQ].abs() + err[:, :HQ])).all())
        s = slots.long()
        for codes, exps, lo in ((self.cache.k, self.cache.k_exp, HQ), (self.cache.v, self.cache.v_exp, HQ + HK)):
            e = exps[s // PAGE, :, s % PAGE]
            unit = two_to(e.int() - 127)[..., None]
            y, dy = want[:, lo:lo + HK], err[:, lo:lo + HK]
            half = unit / 2 if self.codes == torch.int8 else torch.maximum((y.abs() + dy) * 2.0 ** -4, unit * 2.0 ** -10)
            got = value(codes.view(torch.uint8)[s // PAGE, :, s % PAGE].view(codes.dtype), e)
            assert bool(((got - y).abs() <= half + dy).all())
            most = unit[..., 0] * (127 if self.codes == torch.int8 else 448)
            top, slack = y.abs().amax(-1), dy.amax(-1)
            assert bool(((top <= most + slack) & (top > most / 2 - slack)).all())

        lead = self.rows(self.prefix_table, prefix) if prefix else None
        at = 0
        for nq, nk, pages in zip(lq, lens, tables):
            k, v = self.rows(pages, nk)
            if lead:
                k, v = torch.cat((lead[0], k)), torch.cat((lead[1], v))
            hide = torch.arange(len(k), device=DEV)[None] > torch.arange(nq, device=DEV)[:, None] + len(k) - nq
            for h in range(HQ):
                sc = (heads[at:at + nq, h].double() @ k[:, h * HK // HQ].t() / math.sqrt(D)).masked_fill(hide, -math.inf)
                p, vv = torch.softmax(sc, -1), v[:, h * HK // HQ]
                o, m = p @ vv, p @ vv.abs()
                assert bool(((attn[at:at + nq, h].double() - o).abs() <= 2 * u * (m + o.abs()) + 2.0 ** -20 * m).all())
            at += nq

        z, w = attn.view(-1, HQ * D).double(), self.wo.double()
        assert bool(((out.double() - z @ w.t()).abs() <= 2 * math.sqrt(HQ * D) * 2.0 ** -24 * (z.abs() @ w.abs().t())).all())


@pytest.mark.parametrize("codes", CODES, ids=str)
def test_template_prompts_and_tokens(qimg, codes):
    m = Layer(qimg, codes)
    rn = lambda t: torch.randn(t, HID, generator=m.g, device=DEV).to(BF)  # noqa: E731

    # the template: its pages are a sequence's own here
    x, pos = rn(TEMPLATE), torch.arange(TEMPLATE, dtype=torch.int32, device=DEV)
    slots = m.slots(m.prefix_table, 0, TEMPLATE).int()
    got = m(x, slots, pos, _i32(0, TEMPLATE), _i32(TEMPLATE), m.prefix_table[None])
    torch.cuda.synchronize()
    m.check(x, slots, pos, [TEMPLATE], [TEMPLATE], [m.prefix_table], 0, *got)

    # the variants' prompts behind it
    cu = _offsets(PROMPTS)
    x = rn(cu[-1])
    pos = torch.cat([torch.arange(TEMPLATE, TEMPLATE + n, dtype=torch.int32, device=DEV) for n in PROMPTS])
    slots = torch.cat([m.slots(m.table[b], 0, n) for b, n in enumerate(PROMPTS)]).int()
    plen = _i32(TEMPLATE)
    got = m(x, slots, pos, _i32(*cu), _i32(*PROMPTS), m.table, plen)
    torch.cuda.synchronize()
    m.check(x, slots, pos, PROMPTS, PROMPTS, m.table, TEMPLATE, *got)

    # what they wrote, read back, is the values that the codes stand for
    back = qimg.kv_cache_read(m.cache, m.table, _i32(*PROMPTS), _i32(*cu), cu[-1], out_dtype=torch.float32)
    for b, n in enumerate(PROMPTS):
        for rows, want in zip(back, m.rows(m.table[b], n)):
            assert torch.equal(rows[cu[b]:cu[b + 1]].double(), want)

    # one token each: captured once, the lists, positions and rows filled in before each replay
    B = len(PROMPTS)
    x, pos, slots, lens = rn(B), torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV), _i32(*PROMPTS)
    ones = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    slots.fill_(-1)  # (the run before the capture writes nothing)
    m(x, slots, pos, ones, lens, m.table, plen)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m(x, slots, pos, ones, lens, m.table, plen)
    for n in range(STEPS):
        now = [p + n + 1 for p in PROMPTS]
        x.copy_(rn(B))
        lens.copy_(_i32(*now))
        pos.copy_(lens - 1 + TEMPLATE)
        slots.copy_(torch.cat([m.slots(m.table[b], now[b] - 1, now[b]) for b in range(B)]))
        graph.replay()
        torch.cuda.synchronize()
        if n % 23 == 0 or n == STEPS - 1:
            m.check(x, slots, pos, [1] * B, now, m.table, TEMPLATE, *got)
            eager = m(x, slots, pos, ones, lens, m.table, plen)
            assert all(torch.equal(a, b) for a, b in zip(eager, got))


def test_two_streams_over_one_cache(qimg):
    """Sequences of their own in one cache, written and attended to on two streams at once."""
    m = Layer(qimg, CODES[1])
    work = []
    for b in (2, 3):
        n = PROMPTS[b]
        x = torch.randn(n, HID, generator=m.g, device=DEV).to(BF)
        work.append((x, m.slots(m.table[b], 0, n).int(), torch.arange(n, dtype=torch.int32, device=DEV), _i32(0, n), _i32(n),
                     m.table[b:b + 1]))
    want = [m(*w) for w in work]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in work], []
    for _ in range(10):
        for s, w in zip(streams, work):
            with torch.cuda.stream(s):
                got.append(m(*w))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))
