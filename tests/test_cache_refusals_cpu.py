"""The operators around a quantized key/value cache, without a GPU: arguments that the C
entry points and the Python wrappers refuse before any HIP call, on addresses that are
never read, and empty calls."""
import ctypes

import pytest
import torch

FAKE = 0x10000


def _err(qimg):
    return qimg.lib().qimg_last_error().decode()


def _c(qimg, **kw):
    c = dict(k=FAKE, v=FAKE, k_exp=FAKE, v_exp=FAKE, dtype=qimg.INT8, n_pages=100, page_size=64, n_kv_heads=4, head_dim=128)
    c.update(kw)
    return ctypes.byref(qimg._KvCache(**c))


def _heads(qimg, cache=None, slots=FAKE, **kw):
    a = dict(x=FAKE, x_dtype=qimg.BF16, x_stride_t=4608, x_stride_h=128, out=FAKE * 2, out_dtype=qimg.BF16,
             out_stride_t=4608, out_stride_h=128, tokens=10, n_q_heads=28, n_kv_heads=4, head_dim=128, rotary_dim=128,
             interleaved=0, q_norm=FAKE, k_norm=FAKE, eps=1e-6, cos_sin=FAKE, table_rows=100, positions=FAKE)
    a.update(kw)
    a = ctypes.byref(qimg._NormRope(**a))
    if cache is None:
        return qimg.lib().qimg_norm_rope_packed(a, None)
    return qimg.lib().qimg_norm_rope_cache(a, cache, slots, None)


@pytest.mark.parametrize("status,text,change", [
    (1, "dtypes", dict(x_dtype=3)), (1, "dtypes", dict(out_dtype=5)), (1, "bad sizes", dict(tokens=-1)),
    (1, "bad sizes", dict(n_q_heads=-1)), (1, "bad sizes", dict(n_kv_heads=-4)), (1, "2^30", dict(tokens=1 << 25)),
    (1, "2^30", dict(n_q_heads=1 << 24, tokens=1)), (1, "2^30", dict(n_kv_heads=1 << 30)),
    (2, "head_dim", dict(head_dim=264)), (2, "head_dim", dict(head_dim=0)), (2, "head_dim", dict(head_dim=100)),
    (1, "eps", dict(eps=-1.0)), (1, "eps", dict(eps=float("nan"))), (1, "eps", dict(eps=float("inf"))),
    (1, "table_rows", dict(table_rows=-1)), (1, "rotary_dim", dict(rotary_dim=136)), (1, "rotary_dim", dict(rotary_dim=0)),
    (2, "rotary_dim", dict(rotary_dim=12)), (1, "strides", dict(x_stride_t=4604)), (1, "strides", dict(out_stride_h=-128)),
    (1, "strides", dict(x_stride_t=(1 << 24) + 8)), (1, "null", dict(x=None)), (1, "null", dict(out=None)),
    (1, "null", dict(positions=None)), (1, "aligned", dict(x=FAKE + 8)), (1, "aligned", dict(k_norm=FAKE + 2)),
    (1, "aligned", dict(cos_sin=FAKE + 4)), (1, "out strides", dict(out_stride_h=64)), (1, "out strides", dict(out_stride_t=128)),
    (1, "x's place", dict(out=FAKE, out_dtype=0)), (1, "x's place", dict(out=FAKE, out_stride_t=5000)),
])
def test_norm_rope_refuses(qimg, status, text, change):
    assert _heads(qimg, **change) == status
    assert text in _err(qimg)
    assert _heads(qimg, _c(qimg), **change) == status


CACHES = [(1, "cache dtype", dict(dtype=1)), (1, "bad cache", dict(n_pages=-1)), (1, "bad cache", dict(n_kv_heads=0)),
          (2, "page_size", dict(page_size=8)), (2, "page_size", dict(page_size=48)), (2, "page_size", dict(page_size=512)),
          (2, "head_dim", dict(head_dim=96)), (1, "2^31", dict(n_pages=1 << 25)), (1, "2^31", dict(n_kv_heads=1 << 16)),
          (1, "null", dict(v_exp=None)), (1, "aligned", dict(k=FAKE + 8)), (1, "aligned", dict(k_exp=FAKE + 4))]


def _write(qimg, cache, **kw):
    a = dict(k=FAKE, v=FAKE, dtype=qimg.BF16, kt=512, kh=128, vt=512, vh=128, tokens=10, slots=FAKE)
    a.update(kw)
    return qimg.lib().qimg_kv_cache_write(a["k"], a["v"], a["dtype"], a["kt"], a["kh"], a["vt"], a["vh"], a["tokens"], cache,
                                          a["slots"], None)


def _read(qimg, cache, **kw):
    a = dict(table=FAKE, blocks=4, lens=FAKE, cu=FAKE, batch=2, k=FAKE, v=FAKE * 2, dtype=qimg.BF16, kt=512, kh=128, vt=512,
             vh=128, total=100)
    a.update(kw)
    return qimg.lib().qimg_kv_cache_read(cache, a["table"], a["blocks"], a["lens"], a["cu"], a["batch"], a["k"], a["v"],
                                         a["dtype"], a["kt"], a["kh"], a["vt"], a["vh"], a["total"], None)


def _attn(qimg, cache, scratch=None, scratch_bytes=0, **kw):
    a = dict(q=FAKE, out=FAKE * 2, dtype=qimg.BF16, q_stride_t=3584, q_stride_h=128, out_stride_t=3584, out_stride_h=128,
             cu_seqlens_q=FAKE, block_table=FAKE, k_lens=FAKE, prefix_table=None, prefix_len=None, batch=2, total_q=2,
             n_heads=28, max_blocks=100, prefix_blocks=0, sm_scale=0.1, causal=1)
    a.update(kw)
    return qimg.lib().qimg_attention_cache(ctypes.byref(qimg._AttnCache(**a)), cache, scratch, scratch_bytes, None)


@pytest.mark.parametrize("status,text,change", CACHES)
def test_every_entry_refuses_a_bad_cache(qimg, status, text, change):
    for call in (lambda c: _heads(qimg, c), lambda c: _write(qimg, c), lambda c: _read(qimg, c), lambda c: _attn(qimg, c)):
        assert call(_c(qimg, **change)) == status
        assert text in _err(qimg)


def test_null_arguments_and_other_heads(qimg):
    L = qimg.lib()
    c = _c(qimg)
    assert L.qimg_norm_rope_packed(None, None) == 1 and L.qimg_norm_rope_cache(None, c, FAKE, None) == 1
    assert L.qimg_attention_cache(None, c, None, 0, None) == 1
    assert _write(qimg, None) == 1 and _read(qimg, None) == 1 and _attn(qimg, None) == 1
    assert _heads(qimg, c, slots=None) == 1
    assert _heads(qimg, c, n_kv_heads=2) == 1 and "kv heads" in _err(qimg)
    assert _heads(qimg, c, head_dim=64, rotary_dim=64) == 1 and "kv heads" in _err(qimg)


@pytest.mark.parametrize("text,change", [
    ("dtype", dict(dtype=3)), ("tokens", dict(tokens=-1)), ("tokens", dict(tokens=1 << 28)), ("strides", dict(kt=516)),
    ("strides", dict(vh=-128)), ("null", dict(k=None)), ("null", dict(slots=None)), ("aligned", dict(v=FAKE + 2))])
def test_write_refuses(qimg, text, change):
    assert _write(qimg, _c(qimg), **change) == 1
    assert text in _err(qimg)


@pytest.mark.parametrize("text,change", [
    ("dtype", dict(dtype=3)), ("batch", dict(batch=-1)), ("batch", dict(batch=1 << 30)), ("total_k", dict(total=-1)),
    ("total_k", dict(total=1 << 30)), ("max_blocks", dict(blocks=-1)), ("strides", dict(kt=516)), ("null", dict(k=None)),
    ("null", dict(cu=None)), ("null", dict(lens=None)), ("null", dict(table=None)), ("aligned", dict(v=FAKE + 2)),
    ("same", dict(v=FAKE)), ("apart", dict(kt=128)), ("apart", dict(vh=64))])
def test_read_refuses(qimg, text, change):
    assert _read(qimg, _c(qimg), **change) == 1
    assert text in _err(qimg)


@pytest.mark.parametrize("status,text,change", [
    (1, "dtype", dict(dtype=0)), (1, "bad sizes", dict(batch=-1)), (1, "bad sizes", dict(max_blocks=-1)),
    (1, "bad sizes", dict(prefix_blocks=-1)), (1, "multiple", dict(n_heads=27)), (1, "multiple", dict(n_heads=0)),
    (1, "sm_scale", dict(sm_scale=0.0)), (1, "sm_scale", dict(sm_scale=float("nan"))), (1, "sm_scale", dict(sm_scale=3e38)),
    (1, "2^30", dict(total_q=1 << 28)), (1, "2^30", dict(batch=1 << 30)), (1, "2^30", dict(max_blocks=1 << 24)),
    (1, "2^30", dict(prefix_blocks=1 << 24)), (1, "strides", dict(q_stride_t=3588)), (1, "strides", dict(out_stride_h=-8)),
    (1, "null", dict(q=None)), (1, "null", dict(k_lens=None)), (1, "null", dict(block_table=None)),
    (1, "null", dict(prefix_blocks=3, prefix_len=FAKE)), (1, "null", dict(prefix_blocks=3, prefix_table=FAKE)),
    (1, "aligned", dict(q=FAKE + 8)), (1, "out must not", dict(out=FAKE)), (1, "out strides", dict(out_stride_t=128)),
    (3, "scratch", dict(total_q=2))])
def test_attention_refuses(qimg, status, text, change):
    assert _attn(qimg, _c(qimg), **change) == status
    assert text in _err(qimg)


def test_empty_calls_and_scratch(qimg):
    c = _c(qimg)
    assert _heads(qimg, tokens=0, x=None, out=None) == 0 and _heads(qimg, c, tokens=0, x=None, out=None, slots=None) == 0
    assert _heads(qimg, n_q_heads=0, n_kv_heads=0, x=None) == 0
    assert _write(qimg, c, tokens=0, k=None, v=None, slots=None) == 0
    assert _read(qimg, c, batch=0, table=None) == 0 and _read(qimg, c, total=0, k=None) == 0
    assert _read(qimg, _c(qimg, n_pages=0, k=None, v=None, k_exp=None, v_exp=None), k=None) == 0
    assert _attn(qimg, c, batch=0, q=None) == 0 and _attn(qimg, c, total_q=0, q=None) == 0
    need = qimg.attention_cache_scratch_bytes
    assert need(0, 1, 28, 4, 128, 64, 100) == 0 and need(1, 1, 28, 3, 128, 64, 100) == 0
    # sizes that the call refuses
    top = (1 << 31) - 1
    assert need(top, top, top, 1, 128, 256, top, top) == 0 and need(1, 1, 1 << 30, 1, 128, 64, 2) == 0
    assert need(1, 1, 28, 4, 128, 64, 1 << 24) == 0 and need(1, 1, 28, 4, 96, 64, 100) == 0 and need(1, 1, 28, 4, 128, 8, 100) == 0
    assert need(1, 1 << 30, 28, 4, 128, 64, 100) == 0 and need(1, 1, 28, 4, 128, 64, 1, 1 << 24) == 0
    assert need(16, 16, 28, 4, 128, 64, 2) == 0      # short caches are not cut
    assert need(16, 16, 28, 4, 128, 64, 128) > 16 * 28 * 128 * 4
    assert need(16, 16, 28, 4, 128, 64, 2, 10) > 16 * 28 * 128 * 4  # a prefix is joined with the own keys
    assert _attn(qimg, c, scratch=FAKE + 8, scratch_bytes=1 << 40) == 1 and "16-byte" in _err(qimg)
    with pytest.raises(qimg.QimgError, match="2\\^31"):
        need(1 << 32, 1, 28, 4, 128, 64, 2)


def test_wrappers_refuse(qimg):
    x = torch.zeros(4, 3, 64)
    cache = qimg.kv_cache(2, 16, 1, 64, device="cpu")
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(qimg.QimgError, match="device tensor"):
        qimg.norm_rope_packed(x, 1, 1)
    with pytest.raises(qimg.QimgError, match="device tensor"):
        qimg.norm_rope_cache(x, 1, cache, i)
    with pytest.raises(qimg.QimgError, match="device tensors"):
        qimg.kv_cache_write(cache, x[:, :1], x[:, :1], i)
    with pytest.raises(qimg.QimgError, match="on a device"):
        qimg.kv_cache_read(cache, i.view(4, 1), i, torch.zeros(5, dtype=torch.int32), 4)
    with pytest.raises(qimg.QimgError, match="device tensor"):
        qimg.attention_cache(x.bfloat16(), cache, torch.zeros(5, dtype=torch.int32), i.view(4, 1), i)
    with pytest.raises(qimg.QimgError, match="int8 or float8"):
        qimg.kv_cache(2, 16, 1, 64, dtype=torch.float16, device="cpu")


@pytest.mark.parametrize("page", [0, 8, 15, 16, 24, 32, 48, 96, 128, 255, 256, 512])
@pytest.mark.parametrize("hq,hk", [(28, 4), (28, 3), (1 << 16, 1 << 16), (1 << 17, 1 << 16), ((1 << 16) - 1, (1 << 16) - 1)])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_no_scratch_for_sizes_that_the_call_refuses(qimg, page, hq, hk, d):
    c = _c(qimg, n_pages=100, page_size=page, n_kv_heads=hk, head_dim=d)
    refused = _attn(qimg, c, n_heads=hq, total_q=0, out_stride_t=0, q_stride_t=0) != 0
    assert refused == (page not in (16, 32, 64, 128, 256) or hq % hk != 0 or hk >= 1 << 16 or d == 96)
    need = qimg.attention_cache_scratch_bytes(16, 16, hq, hk, d, page, 2, 4)
    assert (need == 0) == refused  # (a prefix always takes some)
