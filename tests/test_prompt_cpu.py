"""The operators around a prompt, without a GPU: arguments the C entry points
and the Python wrappers refuse before any HIP call."""
import ctypes

import pytest
import torch

FAKE = 0x10000  # never dereferenced: validation fails first


def _err(qimg):
    return qimg.lib().qimg_last_error().decode()


def _attn(qimg, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, out=FAKE * 2, dtype=qimg.BF16, q_stride_t=3584, q_stride_h=128, k_stride_t=512,
             k_stride_h=128, v_stride_t=512, v_stride_h=128, out_stride_t=3584, out_stride_h=128, cu_seqlens_q=FAKE,
             cu_seqlens_k=FAKE, k_lens=None, batch=2, total_q=100, total_k=100, n_heads=28, n_kv_heads=4,
             head_dim=128, sm_scale=0.1, causal=1)
    a.update(kw)
    return qimg.lib().qimg_attention_varlen(ctypes.byref(qimg._AttnVarlen(**a)), None, 0, None)


@pytest.mark.parametrize("status,text,change", [
    (1, "dtype", dict(dtype=0)), (1, "bad sizes", dict(batch=-1)), (1, "bad sizes", dict(total_k=-1)),
    (1, "multiple", dict(n_heads=27)), (1, "multiple", dict(n_kv_heads=0)), (2, "head_dim", dict(head_dim=96)),
    (1, "sm_scale", dict(sm_scale=0.0)), (1, "sm_scale", dict(sm_scale=float("nan"))),
    (1, "sm_scale", dict(sm_scale=float("inf"))), (1, "2^30", dict(total_q=1 << 28)),
    (1, "strides", dict(k_stride_t=516)), (1, "strides", dict(q_stride_h=-128)),
    (1, "strides", dict(v_stride_t=(1 << 24) + 8)), (1, "null", dict(q=None)), (1, "null", dict(v=None)),
    (1, "null", dict(cu_seqlens_k=None)), (1, "aligned", dict(k=FAKE + 8)), (1, "out must not", dict(out=FAKE)),
    (1, "out strides", dict(out_stride_t=64)), (1, "out strides", dict(out_stride_h=0)),
])
def test_attention_varlen_refuses(qimg, status, text, change):
    assert _attn(qimg, **change) == status
    assert text in _err(qimg)


def test_attention_varlen_empty_calls_and_scratch(qimg):
    assert _attn(qimg, batch=0, q=None, k=None, v=None, out=None, cu_seqlens_q=None) == 0
    assert _attn(qimg, total_q=0, out=None) == 0
    assert qimg.lib().qimg_attention_varlen(None, None, 0, None) == 1
    # one token over a long cache is split over workgroups and needs room for the parts
    need = qimg.attention_varlen_scratch_bytes(1, 8192, 1, 28, 4, 128)
    assert need > 28 * 128 * 4
    assert _attn(qimg, batch=1, total_q=1, total_k=8192) == 3
    assert "scratch" in _err(qimg)
    assert qimg.attention_varlen_scratch_bytes(0, 8192, 1, 28, 4, 128) == 0
    assert qimg.attention_varlen_scratch_bytes(1, 8192, 1, 28, 3, 128) == 0


def test_attention_varlen_wrapper_refuses(qimg):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(qimg.QimgError, match="device tensors"):
        qimg.attention_varlen(x, x, x, cu, cu)
