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
    (1, "sm_scale", dict(sm_scale=float("inf"))), (1, "2^30", dict(total_q=1 << 28)), (1, "2^30", dict(total_k=1 << 30)),
    (1, "sm_scale", dict(sm_scale=3e38)), (1, "at least head_dim", dict(v_stride_t=64)),
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
    # the last tiles of a launch without a causal mask as well
    assert qimg.attention_varlen_scratch_bytes(3000, 3000, 1, 24, 24, 128, False) > 0
    assert qimg.attention_varlen_scratch_bytes(3000, 3000, 1, 24, 24, 128, True) == 0
    assert _attn(qimg, causal=0, total_q=3000, total_k=3000, n_heads=24, n_kv_heads=24, batch=1) == 3


def test_attention_varlen_wrapper_refuses(qimg):
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(qimg.QimgError, match="device tensors"):
        qimg.attention_varlen(x, x, x, cu, cu)


def _linear(qimg, scratch=None, scratch_bytes=0, **kw):
    a = dict(x=FAKE, x_dtype=qimg.BF16, ldx=512, M=100, N=300, K=512, w=FAKE, w_up=None, bias=None, bias_up=None, act=0,
             gate=None, residual=None, residual_dtype=0, ld_residual=0, out=FAKE * 2, out_dtype=qimg.BF16, ldo=300)
    a.update(kw)
    return qimg.lib().qimg_linear_bf16_fused(ctypes.byref(qimg._LinearFused(**a)), scratch, scratch_bytes, None)


@pytest.mark.parametrize("status,text,change", [
    (1, "x_dtype", dict(x_dtype=2)), (1, "out_dtype", dict(out_dtype=2)), (1, "activation", dict(act=3)),
    (1, "activation", dict(act=-1)), (1, "residual_dtype", dict(residual=FAKE, residual_dtype=2, ld_residual=300)),
    (1, "bad sizes", dict(M=-1)), (1, "bad sizes", dict(K=0)), (1, "null", dict(w=None)), (1, "null", dict(out=None)),
    (1, "bias_up", dict(bias_up=FAKE)), (1, "aligned", dict(x=FAKE + 8)), (1, "aligned", dict(w_up=FAKE + 2)),
    (1, "ldx", dict(ldx=511)), (1, "ldx", dict(ldx=1 << 22)), (1, "ldo", dict(ldo=299)),
    (1, "16-byte aligned", dict(ldx=516)), (1, "ld_residual", dict(residual=FAKE * 3, ld_residual=10)),
    (1, "residual's place", dict(residual=FAKE * 2, ld_residual=300, residual_dtype=0)),
    (1, "out must not", dict(out=FAKE)), (1, "out must not", dict(out=FAKE * 3, w_up=FAKE * 3)), (1, "too large", dict(N=1 << 22, ldo=1 << 22)),
    (3, "scratch", dict(K=511, ldx=511)), (3, "scratch", dict(x_dtype=0)),
])
def test_linear_fused_refuses(qimg, status, text, change):
    assert _linear(qimg, **change) == status
    assert text in _err(qimg)


def test_linear_fused_empty_calls_and_scratch(qimg):
    assert _linear(qimg, M=0, x=None, out=None) == 0
    assert _linear(qimg, N=0, w=None) == 0
    assert qimg.lib().qimg_linear_bf16_fused(None, None, 0, None) == 1
    need = qimg.linear_bf16_fused_scratch_bytes
    assert need(torch.bfloat16, 4096, 4096, 4096) == 0          # whole tiles, rows in place
    assert need(torch.float32, 4096, 4096, 4096) == 4096 * 4096 * 2  # x packed to bf16
    assert need(torch.float32, 1, 4096, 4096) == 0              # one row is rounded in registers
    assert need(torch.bfloat16, 1, 4095, 100) == 8192 + 100 * 8192  # odd K: x and w packed
    assert need(torch.bfloat16, 269, 14336, 3584) >= 2 * 269 * 3584 * 4  # K split
    assert need(torch.bfloat16, 0, 64, 64) == 0
    assert _linear(qimg, K=511, ldx=511, scratch=FAKE + 8, scratch_bytes=1 << 40) == 1
    assert "scratch must be 16-byte" in _err(qimg)


def _rope(qimg, **kw):
    a = dict(x=FAKE, x_dtype=qimg.BF16, x_stride_t=4608, x_stride_h=128, out=FAKE * 2, out_dtype=qimg.BF16,
             out_stride_t=4608, out_stride_h=128, tokens=10, n_heads=36, n_rotated=32, head_dim=128, rotary_dim=128,
             interleaved=0, cos_sin=FAKE, table_rows=100, positions=FAKE)
    a.update(kw)
    return qimg.lib().qimg_rope_packed(ctypes.byref(qimg._Rope(**a)), None)


@pytest.mark.parametrize("status,text,change", [
    (1, "dtypes", dict(x_dtype=3)), (1, "dtypes", dict(out_dtype=5)), (1, "bad sizes", dict(tokens=-1)),
    (1, "bad sizes", dict(n_rotated=37)), (1, "bad sizes", dict(table_rows=-1)), (1, "rotary_dim", dict(rotary_dim=136)),
    (1, "rotary_dim", dict(rotary_dim=0)), (2, "multiples of 8", dict(rotary_dim=12)),
    (2, "multiples of 8", dict(head_dim=132, rotary_dim=128)), (1, "strides", dict(x_stride_t=4604)),
    (1, "strides", dict(out_stride_h=-128)), (1, "null", dict(positions=None)), (1, "null", dict(cos_sin=None)),
    (1, "aligned", dict(x=FAKE + 8)), (1, "out strides", dict(out_stride_h=64)),
    (1, "x's place", dict(out=FAKE, out_dtype=0)), (1, "x's place", dict(out=FAKE, out_stride_t=5000)),
])
def test_rope_refuses(qimg, status, text, change):
    assert _rope(qimg, **change) == status
    assert text in _err(qimg)


def test_rope_empty_calls(qimg):
    assert _rope(qimg, tokens=0, x=None) == 0
    assert _rope(qimg, n_heads=0, n_rotated=0, out=None) == 0
    assert qimg.lib().qimg_rope_packed(None, None) == 1


def test_wrappers_refuse_host_tensors(qimg):
    x = torch.zeros(4, 64)
    with pytest.raises(qimg.QimgError, match="device tensors"):
        qimg.linear_forward_bf16_fused(x, x.bfloat16())
    with pytest.raises(qimg.QimgError, match="device tensor"):
        qimg.rope_packed(x.view(4, 1, 64), torch.zeros(8, 32, 2), torch.zeros(4, dtype=torch.int32), 1)
