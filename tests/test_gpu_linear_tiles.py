"""GPU parity of qimg_linear_bf16_fused on the large tiles: the epilogue with a
residual that is loaded ahead of its use (a sum that is not split, rows of whole
groups of four values), in every tile height, type pair and with a gated second
product; and the one tile whose split sum needs sizes of its own. Definition and
bounds are those of test_gpu_linear_fused.py."""
import math

import pytest
import torch

from planutil import LinearPlan, linear_plan
from test_gpu_linear_fused import TILES, _check, _definition, _gen, _ints, _operands

DEV = "cuda:0"
F32, BF = torch.float32, torch.bfloat16

# (M, N, K, gated) and the tile: M odd, M and N end inside a tile, N a multiple of four
RESIDUAL = [((197, 11116, 264, 0), (128, 128)), ((103, 8848, 264, 1), (128, 128)), ((449, 8380, 264, 0), (128, 256)),
            ((129, 11184, 272, 1), (128, 256)), ((661, 11316, 264, 0), (160, 256)), ((263, 11600, 272, 1), (160, 256)),
            ((831, 10960, 264, 0), (192, 256)), ((321, 11160, 280, 1), (192, 256)), ((977, 10792, 264, 0), (224, 256)),
            ((385, 11048, 272, 1), (224, 256)), ((1361, 9328, 264, 0), (256, 256)), ((463, 11348, 264, 1), (256, 256))]
# 128x128 with the sum split: many rows over 33 to 64 gated columns and a very long K. (No other
# sizes plan it: the small tiles or taller ones are estimated faster.)
LONG = (8713, 34, 20792, 1)


def test_every_tile_is_reached(qimg):
    """The shapes of the integer tests, here and in test_gpu_linear_fused.py, run
    every tile, gated or not, with the whole sum and with a split one."""
    large = [(t, 256, False) for t in (256, 224, 192, 160, 128)] + [(128, 128, False)]
    small = [(128, 64, True), (96, 64, True), (64, 128, True), (64, 64, True), (32, 128, True), (32, 64, True)]
    want = {(LinearPlan(*t, split), bool(g)) for t in large + small for split in (False, True) for g in (0, 1)}
    want.remove((LinearPlan(128, 128, False, True), False))  # (only gated sums of LONG's kind)
    got = {(linear_plan(qimg, qimg.BF16, M, N, K, g), bool(g)) for M, N, K, g in TILES + [LONG]}
    assert got == want


@pytest.mark.parametrize("shape,tile", RESIDUAL, ids=str)
def test_residual_shapes_run_unsplit_large_tiles(qimg, shape, tile):
    M, N, K, gated = shape
    assert linear_plan(qimg, qimg.BF16, M, N, K, gated) == LinearPlan(*tile, False, False)
    assert M % tile[0] and N % (tile[1] // (2 if gated else 1)) and N % 4 == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape,tile", RESIDUAL, ids=str)
def test_residual_loaded_ahead(qimg, shape, tile):
    """fp32 and bf16 residual and out, with bias, activation and channel gate; then
    out in residual's place, rows longer than N, what lies between them kept."""
    M, N, K, gated = shape
    o = _operands(M, N, K, BF, M + N)
    wu, bu = (o["wu"], o["bu"]) if gated else (None, None)
    for act, res_dtype, out_dtype in (("gelu", F32, F32), ("silu", BF, F32), ("none", F32, BF), ("gelu", BF, BF)):
        res = o["res"].to(res_dtype)
        got = qimg.linear_forward_bf16_fused(o["x"], o["w"], bias=o["b"], activation=act, weight_up=wu, bias_up=bu,
                                             gate=o["gate"], residual=res, out_dtype=out_dtype)
        want, err = _definition(o["x"], o["w"], o["b"], act, wu, bu, o["gate"], res)
        torch.cuda.synchronize()
        _check(got, want, err)
    for dtype in (F32, BF):
        store = torch.full((M, N + 12), 5.0, dtype=dtype, device=DEV)
        out = store[:, :N]
        out.copy_(o["res"])
        want, err = _definition(o["x"], o["w"], o["b"], "silu", wu, bu, o["gate"], out)
        got = qimg.linear_forward_bf16_fused(o["x"], o["w"], bias=o["b"], activation="silu", weight_up=wu, bias_up=bu,
                                             gate=o["gate"], residual=out, out=out)
        torch.cuda.synchronize()
        assert got.data_ptr() == store.data_ptr()
        _check(got, want, err)
        assert bool((store[:, N:] == 5.0).all())


@pytest.mark.gpu
def test_long_sum_over_128x128_tiles(qimg):
    """Exact, as test_every_tile_with_integers: sums below 2^17, the second factor
    of the gated product kept small."""
    M, N, K, _ = LONG
    g = _gen(7)
    x, w = _ints(g, (M, K), -2, 2), _ints(g, (N, K), -2, 2)
    wu = _ints(g, (N, K), -1, 1) * (torch.arange(K, device=DEV) % 61 == 0)
    xd, res = x.to(BF), _ints(g, (M, N), -16, 16)
    z = (x.double() @ w.double().t()) * (x.double() @ wu.double().t())
    assert float(z.abs().max()) + 16 < 2 ** 24
    got = qimg.linear_forward_bf16_fused(xd, w.to(BF), weight_up=wu.to(BF), residual=res.to(F32), out_dtype=F32)
    torch.cuda.synchronize()
    assert torch.equal(got.double(), res + z)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 8, 64])
def test_activations_to_the_least_normal_value(qimg, M):
    """Far on the negative side SiLU and GELU are products of v and a sigmoid that is
    no normal number any more, while they are. The product with the identity is
    exact; what is left are the argument's roundings (two and those of its constants,
    2^-23 of it each in all) and eight operations' on the result."""
    eye = torch.eye(64, dtype=BF, device=DEV)
    for act, lo, hi in (("silu", -104, -70), ("gelu", -14.5, -9), ("silu", 70, 104), ("gelu", 9, 20)):
        z = torch.linspace(lo, hi, 64 * M, device=DEV).to(BF).reshape(M, 64)
        got = qimg.linear_forward_bf16_fused(z, eye, activation=act, out_dtype=F32)
        zd = z.double()
        s = zd if act == "silu" else 2 * math.sqrt(2 / math.pi) * (zd + 0.044715 * zd ** 3)
        want = zd / (1 + torch.exp(-s))
        torch.cuda.synchronize()
        _check(got, want, want.abs() * 2.0 ** -23 * (8 + 2 * s.abs().clamp(max=150)))
