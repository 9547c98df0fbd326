"""Calls of the prompt operators that are refused because they could not be
answered in one way, or not within the tensors: without a GPU, on addresses that
are never read."""
import pytest
import torch

from test_prompt_cpu import FAKE, _attn, _err, _rope

# token stride, head stride: of heads of 128 values
OVERLAPS = [(128, 128), (3584, 256), (136, 128), (3576, 128), (128, 256), (256, 136)]
APART = [(4608, 128), (36 * 256, 256), (128, 1280), (136, 136 * 10)]


@pytest.mark.parametrize("t,h", OVERLAPS)
def test_outputs_that_overlap_themselves(qimg, t, h):
    """Tokens and heads each at least head_dim apart, but a head of one token where
    another of the next is: which one stays would be up to chance."""
    assert _attn(qimg, total_q=10, out_stride_t=t, out_stride_h=h) == 1
    assert "tokens and heads apart" in _err(qimg)
    assert _rope(qimg, n_heads=28, n_rotated=28, out_stride_t=t, out_stride_h=h) == 1
    assert "tokens and heads apart" in _err(qimg)


@pytest.mark.parametrize("t,h", APART)
def test_outputs_of_either_order(qimg, t, h):
    """Rows of a longer projection and head-major outputs go on to the next check."""
    assert _attn(qimg, total_q=10, total_k=9000, batch=1, out_stride_t=t, out_stride_h=h) == 3
    assert "scratch" in _err(qimg)


def test_more_sequences_than_the_kernels_count(qimg):
    """The kernels walk the sequences 64 at a time in 32 bits: near 2^31 of them the
    walk would pass the type's end and read in front of the offsets."""
    for batch in (1 << 30, 2 ** 31 - 1):
        assert _attn(qimg, batch=batch) == 1
        assert "2^30" in _err(qimg)


def test_scratch_of_sizes_past_32_bits(qimg):
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        qimg.attention_varlen_scratch_bytes(1 << 32, 100, 1, 1, 1, 64)
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        qimg.linear_bf16_fused_scratch_bytes(torch.bfloat16, 100, 1 << 32, 100)
