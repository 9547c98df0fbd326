"""GPU parity of qimg_attention_varlen on values and weights at the ends of the
types' ranges, on each of its kernels: few rows, few rows with the keys in
ranges, many rows with one and with two wave groups, the last tiles in ranges.
Definition and tolerance are those of test_gpu_attention_varlen.py where nothing
else is said."""
import math

import pytest
import torch

from planutil import attn_plan
from test_gpu_attention_varlen import _check, _cu, _make, _oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16

# (queries, keys, heads, kv heads, causal) and the plan: many, groups, in ranges
PATHS = {"few": ([300], [300], 2, 2, True), "few, ranges": ([1, 1], [5000, 900], 28, 4, True),
         "many": ([1500, 1400, 300], [1500, 1400, 300], 28, 4, True), "two groups": ([1024], [1024], 28, 4, True),
         "last tiles": ([3000], [3000], 24, 24, False)}
PLANS = {"few": (False, 0, False), "few, ranges": (False, 0, True), "many": (True, 1, False),
         "two groups": (True, 2, False), "last tiles": (True, 1, True)}


def _path(qimg, name, d=128):
    lq, lk, hq, hk, causal = PATHS[name]
    p = attn_plan(qimg, sum(lq), sum(lk), len(lq), hq, hk, d, causal)
    assert (p.many, p.groups, p.splits > 1) == PLANS[name]
    return lq, lk, hq, hk, causal


@pytest.mark.parametrize("path", PATHS)
def test_largest_values_stay_finite(qimg, path):
    """bf16 reaches as far as fp32, in which P V is summed: the largest V of every
    key, with weights up to 2^8 times that of the running maximum (scores rise by
    just less than what moves it), comes back, and so do both signs mixed."""
    lq, lk, hq, hk, causal = _path(qimg, path)
    q, k, v = _make(lq, lk, hq, hk, 128, BF, 31)
    cuq, cq = _cu(lq)
    cuk, ck = _cu(lk)
    top = torch.finfo(BF).max
    v[:] = top
    for rising in (False, True):
        if rising:
            q.zero_()
            q[:, :, 0] = 1
            k[:, :, 0] = 7.5 * math.log(2)
            k[torch.tensor(ck[:-1], device=DEV), :, 0] = 0
        got = qimg.attention_varlen(q, k, v, cuq, cuk, 1.0 if rising else None, causal)
        torch.cuda.synchronize()
        assert bool((got == top).all())
    v = torch.where(torch.rand(v.shape, device=DEV) < 0.3, -v, v)
    got = qimg.attention_varlen(q, k, v, cuq, cuk, 1.0, causal)
    want, mag = _oracle(q, k, v, cq, ck, lk, 1.0, causal)
    torch.cuda.synchronize()
    assert bool(got.isfinite().all())
    _check(got, want, mag, BF)
    v[:] = 2.0 ** -79  # the least whose products are normal numbers
    got = qimg.attention_varlen(q, k, v, cuq, cuk, 1.0, causal)
    torch.cuda.synchronize()
    assert bool((got == 2.0 ** -79).all())


@pytest.mark.parametrize("path", PATHS)
def test_light_weights_in_fp16(qimg, path):
    """fp16 holds P 2^7 with a step of 2^-24 at least, so a weight below 2^-21 of the
    running maximum is off by up to 2^-32 of it, whatever it is itself: V is zero at
    the heavy key and large at keys of weight 2^-24 to 2^-30. With u = 2^-11 the error is
    at most sum_j (u p_j + 2^-32) |v_j - o|, in fp32 2^-18 of P for its exponent (below 32,
    rounded twice) and 2^-17 of sum p |v| for up to 2^12 terms, and out's own rounding."""
    lq, lk, hq, hk, causal = _path(qimg, path)
    dtype, u = torch.float16, 2.0 ** -11
    q, k, v = _make(lq, lk, hq, hk, 128, dtype, 33)
    cuq, cq = _cu(lq)
    cuk, ck = _cu(lk)
    first = torch.tensor(ck[:-1], device=DEV)
    q.zero_()
    q[:, :, 0] = 1
    k[:, :, 0] = -math.log(2) * (24 + 6 * torch.rand(k.shape[:2], device=DEV))
    k[first, :, 0] = 0
    v = (v.float() * 15000).clamp(-60000, 60000).to(dtype)
    v[first] = 0
    got = qimg.attention_varlen(q, k, v, cuq, cuk, 1.0, causal)
    want, mag = _oracle(q, k, v, cq, ck, lk, 1.0, causal)
    some = torch.zeros_like(want)  # sum of |v_j - o| over the keys that a row sees, at most
    for b, n in enumerate(lk):
        rows = slice(cq[b], cq[b + 1])
        total = v[ck[b]:ck[b] + n].double().abs().cumsum(0).repeat_interleave(hq // hk, 1)
        last = torch.arange(lq[b], device=DEV) + (n - lq[b]) if causal else torch.full((lq[b],), n - 1, device=DEV)
        some[rows] = total[last] + (last + 1)[:, None, None] * want[rows].abs()
    torch.cuda.synchronize()
    tol = u * (mag + want.abs()) + 2.0 ** -32 * some + (2.0 ** -18 + 2.0 ** -17) * mag + u * want.abs() + 2.0 ** -25
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"max excess {float((err - tol).max())}, max err {float(err.max())}"
