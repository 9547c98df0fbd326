"""GPU: a captured call of attention over a quantized cache follows the lists on the device.
Every replay is held against the definition in 64 bits on the lists that it found, and
against an eager call; both work on scratch full of noise, of another kind each, so that a
partial result that nobody wrote would show."""
import pytest
import torch

from cacheutil import BF, CODES, HF
from test_gpu_attention_cache import Case, _check, _cu, _i32

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

# ranges of few rows; tiles of 32 rows; shares of 128 rows, whole tiles of them; behind a prefix
# with the sequences' own tiles in one launch, of 32 rows, of 128 beside tokens and beside pieces
CASES = [([1] * 3, [700, 4000, 90], 0, 28, 4), ([13, 20, 1], [1300, 300, 77], 0, 28, 4), ([600, 20], [1300, 300], 0, 28, 4),
         ([400] * 4, [400, 900, 500, 401], 0, 80, 8), ([1] * 30, [40 + i for i in range(30)], 800, 28, 4),
         ([2] * 30, [40] * 30, 9000, 28, 4), ([2] * 30, [40] * 30, 12500, 28, 4), ([300, 70], [500, 300], 3000, 80, 8)]


@pytest.mark.parametrize("lq,lk,prefix,hq,hk", CASES, ids=lambda x: str(x)[:24])
@pytest.mark.parametrize("codes,dtype,d,causal", [(CODES[0], BF, 128, True), (CODES[1], HF, 64, True), (CODES[1], BF, 128, False)],
                         ids=str)
def test_replays_follow_the_lists(qimg, lq, lk, prefix, hq, hk, codes, dtype, d, causal):
    c = Case(qimg, lq, lk, prefix, hq=hq, hk=hk, d=d, dtype=dtype, codes=codes, page=32, seed=41)
    room = torch.full((len(lq), c.table.shape[1] * 3 // 2 + 1), -1, dtype=torch.int32, device=DEV)  # tables with room
    room[:, :c.table.shape[1]] = c.table
    c.table = room
    need = qimg.attention_cache_scratch_bytes(sum(lq), len(lq), hq, hk, d, 32, c.table.shape[1],
                                              c.prefix_table.numel() if prefix else 0)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device=DEV)
    plen = _i32(prefix)
    more = dict(prefix_table=c.prefix_table, prefix_len=plen) if prefix else {}
    out = torch.zeros_like(c.q)

    def call(o):
        return qimg.attention_cache(c.q, c.cache, c.cu_q, c.table, c.k_lens, causal=causal, out=o, scratch=scratch, **more)

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(out)
    total, n = sum(lq), len(lq)
    lists = [(lq, lk, prefix),
             (lq, [max(0, x // 9 - 3) for x in lk], prefix // 10),               # much shorter than the tables
             (lq[::-1], [x if i == 0 else 1 for i, x in enumerate(lk)], prefix),  # one long sequence among short ones
             ([total] + [0] * (n - 1), lk, prefix - 1 if prefix else 0),          # all queries of one
             (lq, [0] * n, 0), (lq, lk, prefix)]
    for i, (q, k, p) in enumerate(lists):
        c.lq, c.lk, c.prefix = q, k, p
        cu, c.cq = _cu(q)
        c.cu_q.copy_(cu)
        c.k_lens.copy_(_i32(*k))
        plen.copy_(_i32(p))
        out.fill_(3)
        scratch.fill_((255, 127, 0)[i % 3])
        graph.replay()
        torch.cuda.synchronize()
        _check(out, *c.oracle(causal))
        scratch.fill_((127, 0, 255)[i % 3])
        eager = call(torch.empty_like(out))
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i
