"""GPU parity of qimg_attention_varlen where lengths differ much: tokens over
caches of which one is long, more than 64 sequences on each kernel. Definition
and tolerance are those of test_gpu_attention_varlen.py."""
import pytest
import torch

from planutil import attn_plan
from test_gpu_attention_varlen import DEV, _check, _oracle, _run

pytestmark = pytest.mark.gpu
F16, BF = torch.float16, torch.bfloat16


def _lens(n, top):
    return [top] + [(i * 53) % 70 for i in range(1, n)]


@pytest.mark.parametrize("b,hq,hk,d,dtype", [(6, 24, 24, 128, BF), (17, 16, 8, 64, F16), (32, 28, 4, 128, BF),
                                             (33, 28, 4, 64, BF), (100, 28, 4, 128, F16), (200, 12, 2, 64, BF)])
def test_tokens_over_caches(qimg, b, hq, hk, d, dtype):
    for top, lens in ((8192, _lens(b, 8192)), (3000, [3000 - (i * 211) % 2900 for i in range(b)]), (1200, [1200] * b)):
        p = attn_plan(qimg, b, b * (top + 5), b, hq, hk, d, True)
        assert not p.many and p.splits > 1
        _run(qimg, [1] * b, lens, hq=hq, hk=hk, d=d, dtype=dtype, slots=[top + 5] * b, seed=b)
    lq = [(i % 4) for i in range(b)]  # a few tokens each, none for some
    _run(qimg, lq, [n + 4 for n in _lens(b, 5000)], hq=hq, hk=hk, d=d, dtype=dtype, seed=b + 1)


@pytest.mark.parametrize("causal", [True, False])
def test_many_sequences_of_many_rows(qimg, causal):
    """More sequences than lanes, on the tiles of 128 rows, of 32, and in key ranges."""
    lens = [(i * 37) % 90 for i in range(150)]
    assert attn_plan(qimg, sum(lens), sum(lens), 150, 28, 4, 128, causal).many
    for dtype in (BF, F16):
        _run(qimg, lens, lens, causal=causal, dtype=dtype, seed=3)
    _run(qimg, lens, [n + (i % 7) * 30 for i, n in enumerate(lens)], causal=causal, seed=4)
    few = [i % 2 for i in range(130)]
    keys = [n * (30 + 11 * i) for i, n in enumerate(few)]
    assert attn_plan(qimg, sum(few), sum(keys), 130, 8, 2, 64, causal).splits > 1
    _run(qimg, few, keys, hq=8, hk=2, d=64, causal=causal, seed=5)


def test_one_graph_for_like_and_unlike_lengths(qimg):
    """The ranges follow the lengths on the device: a captured call of 40 tokens serves
    caches that are all alike (whole), of which one is long (in ranges), and empty ones."""
    b, cap = 40, 6000
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    q = torch.randn(b, 28, 128, generator=g, device=DEV).to(BF)
    k, v = (torch.randn(b * cap, 4, 128, generator=g, device=DEV).to(BF) for _ in range(2))
    cuq = torch.arange(b + 1, dtype=torch.int32, device=DEV)
    kl = torch.full((b,), cap, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    scratch = torch.empty(qimg.attention_varlen_scratch_bytes(b, b * cap, b, 28, 4, 128), dtype=torch.uint8, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qimg.attention_varlen(q, k, v, cuq, cuq * cap, k_lens=kl, out=out, scratch=scratch)
    torch.cuda.current_stream().wait_stream(side)
    cuk = cuq * cap
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qimg.attention_varlen(q, k, v, cuq, cuk, k_lens=kl, out=out, scratch=scratch)
    offsets = [i * cap for i in range(b + 1)]
    for lens in ([cap] * b, [cap] + [40] * (b - 1), [0] * b, [i * 149 for i in range(b)], [0, 1] * (b // 2), [700] * b):
        kl.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(7.0)
        scratch.fill_(255)  # NaN in every part
        graph.replay()
        torch.cuda.synchronize()
        want, mag = _oracle(q, k, v, list(range(b + 1)), offsets, lens, 128 ** -0.5, True)
        _check(out, want, mag, BF)
        assert torch.equal(out, qimg.attention_varlen(q, k, v, cuq, cuk, k_lens=kl))
