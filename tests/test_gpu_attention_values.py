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
