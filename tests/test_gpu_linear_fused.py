"""GPU parity: the bf16 linear with its epilogue (qimg_linear_bf16_fused)
against its definition in 64 bits.

* Integer operands (products and partial sums exact in fp32 whatever their
  order): out is the exact value, which catches a dropped, repeated or misplaced
  term, also across tiles, splits of K and the two weights of a gated product.
* Random operands: |err| <= tz * (1.2 |rest| ..) + the epilogue's own roundings,
  with tz = 2 sqrt(K) 2^-24 sum_k |x w| + 2^-23 |z| for a product (fp32 sums in
  some order), the activations' slopes below 1.13, six fp32 operations of
  relative error 2^-23 (exp2 and the reciprocal are good to 2 ulp: 8 in all) on the
  result, and half a step of out's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF = torch.float32, torch.bfloat16

# rows up to 16 (weights straight to fragments) and the tiles: sizes about the
# tiles' edges, K of one stage, of a part of one, of several, long enough to be split
SHAPES = [(1, 16, 8), (1, 4608, 3584), (3, 50, 72), (16, 333, 1000), (17, 16, 64), (17, 128, 8), (40, 300, 136),
          (64, 256, 512), (65, 257, 200), (100, 3584, 3584), (129, 130, 64), (200, 1000, 2056), (269, 512, 7000),
          (300, 2048, 64), (500, 777, 320), (781, 4608, 512), (1000, 1000, 128), (1100, 3000, 256), (2047, 2049, 192)]


def _ints(g, shape, lo, hi):
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV)


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("M,N,K", SHAPES, ids=str)
@pytest.mark.parametrize("x_dtype", [F32, BF], ids=["fp32", "bf16"])
def test_integers_are_exact(qimg, M, N, K, x_dtype):
    g = _gen(M + 3 * N + K)
    x, w, wu = _ints(g, (M, K), -2, 2), _ints(g, (N, K), -2, 2), _ints(g, (N, K), -1, 1)
    b, bu = _ints(g, (N,), -8, 8), _ints(g, (N,), -8, 8)
    gate = 2.0 ** _ints(g, (N,), -2, 2).float()
    res = _ints(g, (M, N), -16, 16)
    xd, wd, wud = x.to(x_dtype), w.to(BF), wu.to(BF)
    z = (x.double() @ w.double().t()) + b
    got = qimg.linear_forward_bf16_fused(xd, wd, bias=b.to(BF), out_dtype=F32)
    assert torch.equal(got.double(), z)
    got = qimg.linear_forward_bf16_fused(xd, wd, bias=b.to(BF), gate=gate, residual=res.to(F32), out_dtype=F32)
    assert torch.equal(got.double(), res + gate.double() * z)
    u = x.double() @ wu.double().t() + bu
    if float((z * u).abs().max()) < 2 ** 24:
        got = qimg.linear_forward_bf16_fused(xd, wd, bias=b.to(BF), weight_up=wud, bias_up=bu.to(BF), out_dtype=F32)
        assert torch.equal(got.double(), z * u)
    got = qimg.linear_forward_bf16_fused(xd, wd, residual=res.to(BF), out_dtype=BF)
    assert torch.equal(got, (res.double() + x.double() @ w.double().t()).to(F32).to(BF))


# (M, N, K, gated): each kernel's tiles (256 to 128 rows by 256, 128x128; the small ones of
# 128, 96, 64 and 32 rows), whole K and K split over workgroups; odd sizes, K that ends inside a stage
TILES = [(196, 11191, 264, 0), (104, 8701, 264, 1), (1675, 2329, 264, 0), (198, 8827, 4024, 0), (198, 8314, 264, 1),
         (199, 2094, 7992, 1), (98, 8373, 264, 0), (1775, 65, 3896, 0), (107, 4207, 272, 1), (798, 65, 6968, 1),
         (518, 13478, 272, 0), (137, 10942, 4080, 0), (260, 11553, 280, 1), (130, 2753, 8136, 1), (810, 11318, 264, 0),
         (728, 2701, 5392, 0), (358, 11089, 264, 1), (367, 2738, 5400, 1), (1951, 5953, 264, 0), (212, 10933, 4112, 0),
         (408, 11123, 264, 1), (195, 4098, 5784, 1), (1368, 9810, 264, 0), (233, 10927, 4904, 0), (459, 11623, 272, 1),
         (245, 5473, 5480, 1), (21, 8442, 264, 1), (17, 65, 264, 0), (18, 67, 2472, 0), (19, 65, 264, 1),
         (17, 67, 2640, 1), (129, 8807, 264, 0), (1192, 65, 4640, 0), (33, 8287, 272, 1), (387, 225, 5432, 1),
         (2093, 205, 272, 0), (821, 65, 2768, 0), (1683, 131, 264, 1), (385, 66, 3952, 1), (2086, 453, 272, 0),
         (931, 66, 4104, 0), (2314, 193, 288, 1), (771, 67, 3216, 1), (296, 834, 5352, 0), (289, 417, 6336, 1),
         (2164, 71, 4112, 0), (1396, 65, 4440, 1), (2515, 68, 5240, 0), (215, 531, 5200, 1), (18, 17663, 264, 0),
         (25, 5618, 16288, 0), (17, 2733, 14416, 1)]


@pytest.mark.parametrize("M,N,K,gated", TILES, ids=str)
def test_every_tile_with_integers(qimg, M, N, K, gated):
    """Exact, as above. K <= 16288 products of at most 4 (2): sums below 2^16, the
    gated product below 2^24 because its second factor is kept small."""
    g = _gen(M + N + K)
    x, w = _ints(g, (M, K), -2, 2), _ints(g, (N, K), -2, 2)
    z = x.double() @ w.double().t()
    res = _ints(g, (M, N), -16, 16)
    if gated:
        wu = _ints(g, (N, K), -1, 1) * (torch.arange(K, device=DEV) % 37 == 0)
        z = z * (x.double() @ wu.double().t())
        assert float(z.abs().max()) + 16 < 2 ** 24
    got = qimg.linear_forward_bf16_fused(x.to(BF), w.to(BF), weight_up=wu.to(BF) if gated else None, residual=res.to(F32),
                                         out_dtype=F32)
    assert torch.equal(got.double(), res + z)


def _definition(x, w, b, act, wu, bu, gate, res):
    """The result in 64 bits and the bound on an fp32 evaluation's error."""
    K = x.shape[1]
    xd = x.to(BF).double()

    def product(w, b):
        z = xd @ w.double().t() + (0 if b is None else b.double())
        e = 2 * math.sqrt(K) * 2.0 ** -24 * (xd.abs() @ w.double().abs().t()) + 2.0 ** -23 * z.abs()
        return z, e

    z, e = product(w, b)
    if act == "silu":
        y = z * torch.sigmoid(z)
    elif act == "gelu":
        y = 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    else:
        y = z
    # the argument of exp2 is rounded: its error, |t| 2^-23, times |y| at most (|t| < 60 where y counts)
    e = 1.13 * e + y.abs() * 2.0 ** -23 * (8 + (60 if act != "none" else 0))
    if wu is not None:
        u, eu = product(wu, bu)
        y, e = y * u, e * u.abs() + y.abs() * eu + e * eu
    if gate is not None:
        y, e = y * gate.double(), e * gate.double().abs()
    e = e + 3 * 2.0 ** -23 * y.abs()
    if res is not None:
        y = y + res.double()
    return y, e + 2.0 ** -23 * y.abs()


def _check(got, want, err):
    tol = err + want.abs() * torch.finfo(got.dtype).eps / 2 + torch.finfo(got.dtype).tiny
    bad = (got.double() - want).abs() - tol
    assert float(bad.max()) <= 0, f"max excess {float(bad.max())}"


def _operands(M, N, K, x_dtype, seed):
    g = _gen(seed)
    rn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    return dict(x=rn(M, K).to(x_dtype), w=(0.05 * rn(N, K)).to(BF), b=rn(N).to(BF), wu=(0.05 * rn(N, K)).to(BF),
                bu=rn(N).to(BF), gate=rn(N), res=rn(M, N))


@pytest.mark.parametrize("M,N,K", [(1, 100, 40), (5, 512, 3584), (16, 48, 264), (33, 70, 1000), (150, 520, 3584),
                                   (269, 3584, 1536), (600, 1000, 136)], ids=str)
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("x_dtype,out_dtype", [(F32, BF), (BF, F32), (BF, BF)], ids=["f32-bf16", "bf16-f32", "bf16-bf16"])
def test_epilogues(qimg, M, N, K, act, x_dtype, out_dtype):
    o = _operands(M, N, K, x_dtype, M + N + K)
    for b, wu, bu, gate, res in ((None, None, None, None, None), (o["b"], None, None, None, None),
                                 (o["b"], o["wu"], None, None, None), (None, o["wu"], o["bu"], o["gate"], o["res"]),
                                 (o["b"], None, None, o["gate"], o["res"].to(BF)), (None, None, None, None, o["res"])):
        got = qimg.linear_forward_bf16_fused(o["x"], o["w"], bias=b, activation=act, weight_up=wu, bias_up=bu, gate=gate,
                                             residual=res, out_dtype=out_dtype)
        want, err = _definition(o["x"], o["w"], b, act, wu, bu, gate, res)
        torch.cuda.synchronize()
        _check(got, want, err)


@pytest.mark.parametrize("M,N,K", [(3, 50, 33), (16, 16, 1), (40, 65, 7), (130, 257, 1001), (70, 3, 75)], ids=str)
@pytest.mark.parametrize("x_dtype", [F32, BF], ids=["fp32", "bf16"])
def test_k_of_no_whole_pieces(qimg, M, N, K, x_dtype):
    """K that is no multiple of 8: rows are packed into scratch first."""
    o = _operands(M, N, K, x_dtype, K)
    for wu in (None, o["wu"]):
        got = qimg.linear_forward_bf16_fused(o["x"], o["w"], bias=o["b"], activation="silu", weight_up=wu, residual=o["res"],
                                             out_dtype=F32)
        want, err = _definition(o["x"], o["w"], o["b"], "silu", wu, None, None, o["res"])
        torch.cuda.synchronize()
        _check(got, want, err)


@pytest.mark.parametrize("M,N,K", [(4, 40, 64), (77, 130, 200), (300, 600, 1000)], ids=str)
def test_views_in_place_and_what_lies_between_rows(qimg, M, N, K):
    """x, residual and out with longer rows: NaN between x's rows does not
    reach the result, what lies between out's rows stays; out in residual's place."""
    o = _operands(M, N, K, BF, 7)
    for x_dtype in (F32, BF):
        xs = torch.full((M, K + 24), float("nan"), dtype=x_dtype, device=DEV)
        xs[:, :K] = o["x"]
        for odd in (0, 1):
            store = torch.full((M, N + 12 + odd), 5.0, device=DEV)
            out = store[:, :N]
            out.copy_(o["res"])
            want, err = _definition(o["x"], o["w"], o["b"], "none", None, None, o["gate"], o["res"])
            got = qimg.linear_forward_bf16_fused(xs[:, :K], o["w"], bias=o["b"], gate=o["gate"], residual=out, out=out)
            torch.cuda.synchronize()
            assert got.data_ptr() == store.data_ptr()
            _check(got, want, err)
            assert bool((store[:, N:] == 5.0).all())


@pytest.mark.parametrize("M", [9, 200])
def test_nan_and_infinity_stay_in_their_row_and_column(qimg, M):
    N, K = 200, 136
    o = _operands(M, N, K, BF, 3)
    base = qimg.linear_forward_bf16_fused(o["x"], o["w"], out_dtype=F32)
    x, w = o["x"].clone(), o["w"].clone()
    x[5, 17] = float("nan")
    w[33, 100] = float("inf")
    got = qimg.linear_forward_bf16_fused(x, w, out_dtype=F32)
    torch.cuda.synchronize()
    assert bool(got[5].isnan().all()) and not bool(got[:, 33].isfinite().any())
    keep = torch.ones(M, N, dtype=torch.bool, device=DEV)
    keep[5] = False
    keep[:, 33] = False
    assert torch.equal(got[keep], base[keep])


def test_activations_keep_their_tails(qimg):
    """Far on both sides: z from -80 to 80 through an identity weight."""
    z = torch.linspace(-80, 80, 64 * 40, device=DEV).to(BF).reshape(40, 64)
    eye = torch.eye(64, dtype=BF, device=DEV)
    for act in ("gelu", "silu"):
        got = qimg.linear_forward_bf16_fused(z, eye, activation=act, out_dtype=F32)
        want, err = _definition(z, eye, None, act, None, None, None, None)
        torch.cuda.synchronize()
        _check(got, want, err)


def test_graph_replays_and_same_bits(qimg):
    for M, N, K in ((2, 512, 1024), (269, 512, 7000)):
        o = _operands(M, N, K, BF, 5)
        x = o["x"].clone()
        out = torch.empty(M, N, device=DEV)
        scratch = torch.empty(max(16, qimg.linear_bf16_fused_scratch_bytes(BF, M, K, N)), dtype=torch.uint8, device=DEV)
        call = lambda: qimg.linear_forward_bf16_fused(x, o["w"], bias=o["b"], activation="gelu",  # noqa: E731
                                                      residual=o["res"], out=out, scratch=scratch)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for i in range(3):
            x.copy_(o["x"] * (1 - i))
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            call()
            torch.cuda.synchronize()
            assert torch.equal(got, out)
