"""GPU parity: attention over packed sequences (qimg_attention_varlen) against
the definition in 64 bits on the same bf16 / fp16 inputs.

Tolerance, from the arithmetic: with u = eps / 2 of the type, P is rounded to
the type before the second product (relative u on every p_j, and on the same
rounded values in the row sum), and the result once more. Both roundings are
bounded by u sum_j p_j |v_j - o| + u |o| <= 2 u (sum_j p_j |v_j| + |o|); the
fp32 parts add less: a score's absolute error is at most D 2^-24 max_d-sums
(about sum |q k| D 2^-24) and moves p by that much, covered by a further term
2^-20 sum_j p_j |v_j| (scores here stay below 64 in magnitude)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _cu(lens):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=DEV), c


def _oracle(q, k, v, cq, ck, lk, scale, causal):
    """The definition in 64 bits, and sum_j p_j |v_j| beside it."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    group = q.shape[1] // k.shape[1]
    for b in range(len(cq) - 1):
        n = lk[b]
        nq = cq[b + 1] - cq[b]
        if nq == 0 or n == 0:
            continue
        for h in range(q.shape[1]):
            x = q[cq[b]:cq[b + 1], h].double() @ k[ck[b]:ck[b] + n, h // group].double().t() * scale
            vis = torch.ones(nq, n, dtype=torch.bool, device=q.device)
            if causal:
                vis = torch.arange(n, device=q.device)[None] <= torch.arange(nq, device=q.device)[:, None] + (n - nq)
            x = x.masked_fill(~vis, -math.inf)
            p = torch.softmax(x, dim=-1)
            none = ~vis.any(dim=-1)
            p[none] = 0.0
            vv = v[ck[b]:ck[b] + n, h // group].double()
            out[cq[b]:cq[b + 1], h] = p @ vv
            mag[cq[b]:cq[b + 1], h] = p @ vv.abs()
    return out, mag


def _check(got, want, mag, dtype):
    u = torch.finfo(dtype).eps / 2
    tol = 2 * u * (mag + want.abs()) + 2.0 ** -20 * mag + torch.finfo(dtype).tiny
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"max excess {float((err - tol).max())}, max err {float(err.max())}"


def _make(lq, slots, hq, hk, d, dtype, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    q = torch.randn(sum(lq), hq, d, generator=g, device=DEV).to(dtype)
    k = (torch.randn(sum(slots), hk, d, generator=g, device=DEV) + 0.5).to(dtype)
    v = torch.randn(sum(slots), hk, d, generator=g, device=DEV).to(dtype)
    return q, k, v


def _run(qimg, lq, lk, hq=28, hk=4, d=128, dtype=torch.bfloat16, causal=True, slots=None, seed=0):
    slots = slots or lk
    q, k, v = _make(lq, slots, hq, hk, d, dtype, seed)
    cuq, cq = _cu(lq)
    cuk, ck = _cu(slots)
    kl = torch.tensor(lk, dtype=torch.int32, device=DEV) if slots is not lk else None
    scale = 1.0 / math.sqrt(d)
    got = qimg.attention_varlen(q, k, v, cuq, cuk, scale, causal, k_lens=kl)
    want, mag = _oracle(q, k, v, cq, ck, lk, scale, causal)
    torch.cuda.synchronize()
    _check(got, want, mag, dtype)
    return got


# lengths around the tiles (32 and 128 rows, 32 and 64 keys), of one token, of zero
LENS = [[1], [1, 1, 1], [31], [32], [33], [64], [65, 0, 3], [0, 0, 7], [127, 128, 129], [257, 13, 1, 0, 40]]
DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(qimg, lens, d, causal):
    for dtype in DTYPES:
        _run(qimg, lens, lens, d=d, dtype=dtype, causal=causal, seed=sum(lens) + d)


@pytest.mark.parametrize("hq,hk", [(1, 1), (7, 1), (5, 5), (24, 8), (32, 1)])
@pytest.mark.parametrize("lens", [[70, 9], [300]], ids=str)
def test_head_groups(qimg, hq, hk, lens):
    _run(qimg, lens, lens, hq=hq, hk=hk, seed=hq)


@pytest.mark.parametrize("lens", [[1500, 1], [700, 1301, 64, 257], [2048], [1000], [2600], [130] * 8, [80] * 20],
                         ids=str)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows(qimg, lens, d, causal):
    for dtype in DTYPES:
        _run(qimg, lens, lens, hq=28, hk=4, d=d, dtype=dtype, causal=causal, seed=len(lens))


# launches whose last round of workgroups is cut into key ranges: several tiles and
# one, ranges that a short sequence leaves empty, keys behind a slot's last
TAILS = [([3000], [3000], None, 24, 24, 128, torch.bfloat16), ([3000], [3000], None, 24, 24, 128, torch.float16),
         ([5600], [4000], None, 24, 24, 64, torch.float16), ([3000], [9000], None, 24, 4, 64, torch.bfloat16),
         ([2700, 300, 5], [5000, 40, 0], [7000, 100, 10], 24, 24, 128, torch.bfloat16)]


@pytest.mark.parametrize("lq,lk,slots,hq,hk,d,dtype", TAILS, ids=lambda x: str(x).replace("torch.", ""))
def test_last_tiles_in_key_ranges(qimg, lq, lk, slots, hq, hk, d, dtype):
    slots = slots or lk
    assert qimg.attention_varlen_scratch_bytes(sum(lq), sum(slots), len(lq), hq, hk, d, False) > 0
    q, k, v = _make(lq, slots, hq, hk, d, dtype, 21)
    cuq, cq = _cu(lq)
    cuk, ck = _cu(slots)
    for b, n in enumerate(lk):  # what lies behind a sequence's last key
        k[ck[b] + n:ck[b + 1]] = float("nan")
        v[ck[b] + n:ck[b + 1]] = float("inf")
    v[ck[0] + lk[0] - 1, 0, 3] = float("inf")  # a key that every row sees, in the last range
    kl = torch.tensor(lk, dtype=torch.int32, device=DEV)
    room = torch.full((sum(lq) + 3, hq + 1, d + 8), 7.0, dtype=dtype, device=DEV)  # out as a view, and on its own
    runs = [qimg.attention_varlen(q, k, v, cuq, cuk, 1.0 / math.sqrt(d), False, k_lens=kl,
                                  out=room[:sum(lq), :hq, :d] if i else None) for i in range(2)]
    want, mag = _oracle(q, k, v, cq, ck, lk, 1.0 / math.sqrt(d), False)
    torch.cuda.synchronize()
    assert torch.equal(runs[0], runs[1])
    assert bool((room[sum(lq):] == 7).all() and (room[:, hq:] == 7).all() and (room[:, :, d:] == 7).all())
    seen = torch.isinf(want)
    assert bool(seen[0, 0, 3]) and bool((runs[0].double()[seen] == want[seen]).all())
    want[seen], mag[seen] = 0.0, 0.0
    _check(runs[0].masked_fill(seen, 0.0), want, mag, dtype)


@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [1, 700, 33]), ([1] * 5, [4097, 0, 64, 1, 2000]), ([3, 40], [3000, 41]),
                                   ([200, 300], [1000, 300]), ([1], [20000]), ([900], [1700]), ([2000, 700], [2100, 3000])], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_cached_keys(qimg, lq, lk, d):
    """More keys than queries, a cache with room behind the last key, and few
    rows over many keys (split over workgroups)."""
    for dtype in DTYPES:
        _run(qimg, lq, lk, d=d, dtype=dtype, seed=sum(lk))
        _run(qimg, lq, lk, d=d, dtype=dtype, slots=[n + 37 for n in lk], seed=sum(lk) + 1)


@pytest.mark.parametrize("lq,lk", [([40, 5], [8, 5]), ([600], [100]), ([33], [1]), ([20], [0]), ([1900], [65]), ([2900], [700])], ids=str)
def test_rows_that_see_no_key_are_zero(qimg, lq, lk):
    got = _run(qimg, lq, lk)
    if lq[0] > lk[0]:
        assert bool((got[:lq[0] - lk[0]] == 0).all())


@pytest.mark.parametrize("lens", [[50, 70], [900, 1200]], ids=str)
def test_strided_views_and_rows_of_no_sequence(qimg, lens):
    """q, k and v inside one packed projection, a head-major output, tokens
    behind the last sequence: those rows of out stay as they were."""
    hq, hk, d = 28, 4, 128
    t = sum(lens) + 11
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    x = torch.randn(t, hq + 2 * hk, d, generator=g, device=DEV).bfloat16()
    x[sum(lens):] = float("nan")
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    cu, c = _cu(lens)
    store = torch.full((hq, t, d), 7.0, dtype=torch.bfloat16, device=DEV)
    out = store.permute(1, 0, 2)
    got = qimg.attention_varlen(q, k, v, cu, cu, causal=True, out=out)
    assert got.data_ptr() == store.data_ptr()
    want, mag = _oracle(q, k, v, c, c, lens, 1 / math.sqrt(d), True)
    n = sum(lens)
    torch.cuda.synchronize()
    _check(got[:n], want[:n], mag[:n], torch.bfloat16)
    assert bool((got[n:] == 7.0).all())


@pytest.mark.parametrize("n", [45, 200, 1800, 2600])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_values_in_hidden_places_do_not_reach_a_row(qimg, n, value):
    """Row i sees keys 0 .. i: a NaN or infinite K and V row at key j changes
    no row before j, bit for bit, and rows from j on take the value."""
    hq, hk, d = 28, 4, 128
    for dtype in DTYPES:
        q, k, v = _make([n], [n + 5], hq, hk, d, dtype, n)
        cuq, _ = _cu([n])
        cuk, _ = _cu([n + 5])
        kl = torch.tensor([n], dtype=torch.int32, device=DEV)
        base = qimg.attention_varlen(q, k, v, cuq, cuk, k_lens=kl)
        j = n * 3 // 4
        v2 = v.clone()
        v2[j] = value
        v2[n:] = float("nan")
        k2 = k.clone()
        k2[n:] = value
        got = qimg.attention_varlen(q, k2, v2, cuq, cuk, k_lens=kl)
        torch.cuda.synchronize()
        assert torch.equal(got[:j], base[:j])
        if math.isnan(value):
            assert bool(got[j:].isnan().all())
        else:
            assert bool((got[j:] == value).all())
        k3 = k.clone()
        k3[j] = float("nan")
        got = qimg.attention_varlen(q, k3, v, cuq, cuk, k_lens=kl)
        torch.cuda.synchronize()
        assert torch.equal(got[:j], base[:j]) and bool(got[j:].isnan().all())


def test_infinite_scores(qimg):
    """A row all of whose scores are -inf has no softmax (NaN); -inf scores
    beside finite ones weigh nothing; the type's lowest value is a number."""
    n, d = 40, 64
    for dtype in DTYPES:
        q, k, v = _make([n], [n], 2, 2, d, dtype, 5)
        q = q.abs() + 0.5
        k = k.abs() + 0.5
        k[:20] = -float("inf")
        cu, c = _cu([n])
        got = qimg.attention_varlen(q, k, v, cu, cu, causal=True)
        torch.cuda.synchronize()
        assert bool(got[:20].isnan().all())
        want, mag = _oracle(q[20:], k[20:], v[20:], [0, 20], [0, 20], [20], 1 / math.sqrt(d), True)
        _check(got[20:], want, mag, dtype)
        k[:20] = torch.finfo(dtype).min / 1e3
        got = qimg.attention_varlen(q, k, v, cu, cu, causal=True)
        want, mag = _oracle(q, k, v, c, c, [n], 1 / math.sqrt(d), True)
        torch.cuda.synchronize()
        _check(got[20:], want[20:], mag[20:], dtype)
        assert bool(got.isfinite().all())


@pytest.mark.parametrize("lq,lk", [([90], [90]), ([1, 1], [3000, 900]), ([1000, 900], [1000, 900])], ids=str)
def test_constant_values_come_back_exactly(qimg, lq, lk):
    for dtype in DTYPES:
        q, k, v = _make(lq, lk, 28, 4, 128, dtype, 8)
        v[:] = 0.40625
        got = qimg.attention_varlen(q, k, v, _cu(lq)[0], _cu(lk)[0])
        torch.cuda.synchronize()
        assert bool((got == 0.40625).all())


def test_subnormal_values_are_kept(qimg):
    """fp16 below 2^-14: V of one subnormal value comes back, and K of subnormals
    gives the scores that they are."""
    for lens in ([50], [1500, 700]):
        q, k, v = _make(lens, lens, 28, 4, 64, torch.float16, 3)
        v[:] = 3 * 2.0 ** -22
        k = (k.float() * 2.0 ** -18).half()
        q = (q.float() * 2.0 ** 10).half()
        cu, c = _cu(lens)
        got = qimg.attention_varlen(q, k, v, cu, cu, sm_scale=30.0)
        torch.cuda.synchronize()
        assert bool((got == 3 * 2.0 ** -22).all())
        v = torch.randn(v.shape, device=DEV).half()
        got = qimg.attention_varlen(q, k, v, cu, cu, sm_scale=30.0)
        want, mag = _oracle(q, k, v, c, c, lens, 30.0, True)
        torch.cuda.synchronize()
        _check(got, want, mag, torch.float16)


def test_growing_scores_rescale(qimg):
    """Scores that rise along the keys move the running maximum in every tile."""
    n, d = 700, 128
    for hq in (1, 32):
        q, k, v = _make([n], [n], hq, 1, d, torch.bfloat16, 9)
        k = (k.float() * 0.1 + torch.linspace(-2, 2, n, device=DEV)[:, None, None]).bfloat16()
        q = q.abs()
        cu, c = _cu([n])
        for causal in (True, False):
            got = qimg.attention_varlen(q, k, v, cu, cu, causal=causal)
            want, mag = _oracle(q, k, v, c, c, [n], 1 / math.sqrt(d), causal)
            torch.cuda.synchronize()
            _check(got, want, mag, torch.bfloat16)


def test_many_short_sequences(qimg):
    lens = [(i * 7) % 5 for i in range(150)]
    _run(qimg, lens, lens, hq=8, hk=2, d=64)
    _run(qimg, [1] * 130, [1 + (i * 37) % 90 for i in range(130)], hq=8, hk=2)


def test_broken_offsets_stay_inside(qimg):
    """Offsets that fall or leave the tensors are clamped: no read or write
    outside, and the sequences before them are untouched by it."""
    q, k, v = _make([20, 30], [20, 30], 8, 2, 128, torch.bfloat16, 4)
    good, c = _cu([20, 30])
    want = qimg.attention_varlen(q, k, v, good, good)
    bad = torch.tensor([0, 20, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    got = qimg.attention_varlen(q, k, v, bad, bad)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for cq, ck in (([0, 20, -5], [0, 20, 50]), ([-7, 20, 50], [-7, 20, 50]), ([0, 20, 50], [0, 20, 10 ** 9])):
        out = torch.zeros_like(q)
        qimg.attention_varlen(q, k, v, torch.tensor(cq, dtype=torch.int32, device=DEV),
                              torch.tensor(ck, dtype=torch.int32, device=DEV), out=out)
        torch.cuda.synchronize()
        assert torch.equal(out[:20], want[:20])


def test_graph_replays_follow_lengths_on_the_device(qimg):
    """Lengths are read on the device: one captured call serves other k_lens."""
    for lq, cap, causal in (([1] * 4, 2100, True), ([300, 280], 900, True), ([3000], 3000, False)):
        q, k, v = _make(lq, [cap] * len(lq), 28, 4, 128, torch.bfloat16, 6)
        cuq, cq = _cu(lq)
        cuk, ck = _cu([cap] * len(lq))
        kl = torch.full((len(lq),), cap, dtype=torch.int32, device=DEV)
        out = torch.empty_like(q)
        scratch = torch.empty(max(16, qimg.attention_varlen_scratch_bytes(sum(lq), cap * len(lq), len(lq), 28, 4, 128,
                                                                        causal)), dtype=torch.uint8, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            qimg.attention_varlen(q, k, v, cuq, cuk, causal=causal, k_lens=kl, out=out, scratch=scratch)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qimg.attention_varlen(q, k, v, cuq, cuk, causal=causal, k_lens=kl, out=out, scratch=scratch)
        for n in (cap, 513, 300, cap - 1):
            kl.fill_(n)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            want = qimg.attention_varlen(q, k, v, cuq, cuk, causal=causal, k_lens=kl)
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.parametrize("lq,lk", [([700, 333], [700, 333]), ([1, 1], [5000, 77])], ids=str)
def test_same_bits_twice(qimg, lq, lk):
    q, k, v = _make(lq, lk, 28, 4, 128, torch.bfloat16, 12)
    one = qimg.attention_varlen(q, k, v, _cu(lq)[0], _cu(lk)[0])
    two = qimg.attention_varlen(q, k, v, _cu(lq)[0], _cu(lk)[0])
    torch.cuda.synchronize()
    assert torch.equal(one, two)


def test_long_cache_offsets_past_32_bits(qimg):
    """K and V whose tokens lie 2^20 elements apart: byte offsets of 4 GiB."""
    n, stride, hk, d = 2100, 1 << 20, 1, 128
    store = torch.empty(n * stride, dtype=torch.bfloat16, device=DEV)
    kv = torch.as_strided(store, (n, 2, d), (stride, d, 1))
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    kv.copy_(torch.randn(n, 2, d, generator=g, device=DEV).bfloat16())
    q = torch.randn(3, 4, d, generator=g, device=DEV).bfloat16()
    k, v = kv[:, :1], kv[:, 1:]
    cuq, cq = _cu([3])
    cuk, ck = _cu([n])
    got = qimg.attention_varlen(q, k, v, cuq, cuk)
    want, mag = _oracle(q, k, v, cq, ck, [n], 1 / math.sqrt(d), True)
    torch.cuda.synchronize()
    _check(got, want, mag, torch.bfloat16)
