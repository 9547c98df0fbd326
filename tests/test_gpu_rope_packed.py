"""GPU parity: rotary positions of packed heads (qimg_rope_packed) against the
definition in 64 bits. A turned value is two products and their difference: off
by at most 2 * 2^-24 (|a cos| + |b sin|) in fp32 and half a step of out's type;
copied values are exact up to that rounding."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _table(rows, r):
    f = torch.pow(10000.0, -torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)
    a = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.stack((a.cos(), a.sin()), -1).float()


def _definition(x, table, pos, n_rot, interleaved):
    x = x.double()
    r = 2 * table.shape[1]
    cs = table.double()[pos.long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    out, mag = x.clone(), torch.zeros_like(x)
    ia = slice(0, r, 2) if interleaved else slice(0, r // 2)
    ib = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[:, :n_rot, ia], x[:, :n_rot, ib]
    out[:, :n_rot, ia], out[:, :n_rot, ib] = a * c - b * s, b * c + a * s
    mag[:, :n_rot, ia], mag[:, :n_rot, ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return out, mag


def _check(got, want, mag):
    i = torch.finfo(got.dtype)
    tol = 2 ** -23 * mag + want.abs() * i.eps / 2 + i.smallest_normal * i.eps / 2
    assert float(((got.double() - want).abs() - tol).max()) <= 0


@pytest.mark.parametrize("t,h,n_rot,d,r", [(1, 36, 32, 128, 128), (7, 3, 3, 64, 64), (33, 5, 0, 64, 32), (100, 9, 4, 80, 40),
                                           (1001, 36, 32, 128, 64), (3, 1, 1, 8, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(qimg, t, h, n_rot, d, r, interleaved):
    g = torch.Generator(device=DEV)
    g.manual_seed(t + h + d)
    table = _table(500, r)
    pos = torch.randint(0, 500, (t,), generator=g, device=DEV, dtype=torch.int32)
    x0 = torch.randn(t, h, d, generator=g, device=DEV)
    for tin in TYPES:
        for tout in TYPES:
            x = x0.to(tin)
            got = qimg.rope_packed(x, table, pos, n_rot, interleaved=interleaved, out_dtype=tout)
            want, mag = _definition(x, table, pos, n_rot, interleaved)
            torch.cuda.synchronize()
            _check(got, want, mag)


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_views_and_tokens_without_a_position(qimg, interleaved):
    """Heads inside longer rows turned in place; what lies between them and
    tokens whose position is outside the table stay as they were."""
    t, h, d = 50, 12, 64
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    store = torch.randn(t, h + 2, d, generator=g, device=DEV).bfloat16()
    before = store.clone()
    table = _table(40, d)
    pos = torch.arange(t, device=DEV, dtype=torch.int32) - 5  # -5 .. 44
    x = store[:, 1:h + 1]
    got = qimg.rope_packed(x, table, pos, 8, interleaved=interleaved, out=x)
    assert got.data_ptr() == x.data_ptr()
    keep = (pos >= 0) & (pos < 40)
    want, mag = _definition(before[keep][:, 1:h + 1], table, pos[keep], 8, interleaved)
    torch.cuda.synchronize()
    _check(store[keep][:, 1:h + 1], want, mag)
    assert torch.equal(store[~keep], before[~keep])
    assert torch.equal(store[:, 0], before[:, 0]) and torch.equal(store[:, h + 1], before[:, h + 1])
    heads = torch.empty(h, t, d, dtype=torch.float16, device=DEV)  # head-major out
    qimg.rope_packed(before[:, 1:h + 1], table, pos.clamp(0, 39), h, interleaved=interleaved, out=heads.permute(1, 0, 2))
    want, mag = _definition(before[:, 1:h + 1], table, pos.clamp(0, 39), h, interleaved)
    torch.cuda.synchronize()
    _check(heads.permute(1, 0, 2), want, mag)


def test_turning_keeps_distances(qimg):
    """q at position p and k at position p + 5 have the same product whatever p is."""
    table = _table(2000, 128)
    q, k = torch.randn(1, 1, 128, device=DEV), torch.randn(1, 1, 128, device=DEV)
    pos = torch.arange(0, 1990, device=DEV, dtype=torch.int32)
    for interleaved in (False, True):
        a = qimg.rope_packed(q.expand(1990, 1, 128).contiguous(), table, pos, 1, interleaved=interleaved)
        b = qimg.rope_packed(k.expand(1990, 1, 128).contiguous(), table, pos + 5, 1, interleaved=interleaved)
        dots = (a.double() * b.double()).sum((1, 2))
        # each factor is off by 2^-22 of its pair's length (table and arithmetic)
        assert float((dots - dots[0]).abs().max()) <= 2 * 2 ** -22 * float(q.norm() * k.norm())
