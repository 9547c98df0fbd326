"""Which kernel the prompt operators' calls take, without a GPU."""
import pytest

from planutil import attn_plan


# (tokens, heads, kv heads, head_dim): the first numbers of sequences whose tiles of 128 rows are
# more than one round of the few-row kernel, and more
@pytest.mark.parametrize("b,hq,hk,d", [(6, 24, 24, 128), (10, 24, 24, 128), (17, 16, 8, 64), (32, 28, 4, 128),
                                       (33, 28, 4, 64), (65, 12, 2, 128), (128, 28, 4, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_tokens_over_caches_may_cut_their_keys(qimg, b, hq, hk, d, causal):
    """One token a sequence over caches of unknown lengths: the keys of a long one
    among short ones can go into ranges, however many sequences there are."""
    for lq in (1, max(1, min(8, 32 * hk // hq))):  # up to 8 queries and 32 rows a sequence
        p = attn_plan(qimg, b * lq, b * 8192, b, hq, hk, d, causal)
        assert not p.many and p.splits >= 8
        assert qimg.attention_varlen_scratch_bytes(b * lq, b * 8192, b, hq, hk, d, causal) <= 160 << 20


def test_prompts_keep_their_tiles(qimg):
    """As many keys as queries, or more rows a sequence than a small tile has."""
    assert attn_plan(qimg, 4096, 4096, 1, 28, 4, 128, True).many
    assert attn_plan(qimg, 400, 400, 20, 24, 24, 128, True).many
    assert attn_plan(qimg, 640, 9000, 20, 28, 4, 128, True).many
    assert attn_plan(qimg, 512 + 31, 32 * 4000, 32, 6, 6, 128, True).many  # a prompt among tokens
    assert not attn_plan(qimg, 90, 90, 2, 28, 4, 128, True).many


@pytest.mark.parametrize("lens,causal,groups", [([300] * 3, True, 1), ([350] * 3, True, 1), ([400] * 2, True, 1),
                                                ([430] * 2, True, 1), ([480] * 2, True, 2), ([700], True, 2),
                                                ([400] * 2, False, 1), ([480] * 2, False, 2), ([1100], True, 2),
                                                ([500] * 4, True, 1), ([2048], True, 2), ([3000], True, 1)], ids=str)
def test_wave_groups_as_measured(qimg, lens, causal, groups):
    """Two wave groups a tile only where they were the faster form of these calls."""
    p = attn_plan(qimg, sum(lens), sum(lens), len(lens), 28, 4, 128, causal)
    assert p.many and p.groups == groups
