"""The operators around a prompt run together, as one layer of a prompt
encoder uses them: q, k and v projection with bias, rotary positions, packed
causal attention with grouped heads, output projection onto the fp32 residual
stream, gated MLP, and its way back onto the stream. Two prompts of different
lengths lie one behind the other (a prompt and its negative).

Every step is held against its definition in 64 bits on the inputs that the
step before gave, with the tolerances of the operators' own tests: u = eps / 2
of a type for a rounding to it, 2 sqrt(K) 2^-24 sum |x w| for an fp32 product
sum, 2 u (sum p |v| + |o|) for attention.

The same tokens one at a time over a cache (serving) have to give the whole
prompt's attention within both calls' tolerances."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
HQ, HK, D, MLP = 14, 2, 64, 1000
HID = HQ * D


def _weights(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rn = lambda *s, scale=1.0: (scale * torch.randn(s, generator=g, device=DEV))  # noqa: E731
    return dict(qkv=rn((HQ + 2 * HK) * D, HID, scale=0.04).to(BF), qkv_b=rn((HQ + 2 * HK) * D, scale=0.3).to(BF),
                o=rn(HID, HID, scale=0.03).to(BF), gate=rn(MLP, HID, scale=0.04).to(BF), up=rn(MLP, HID, scale=0.04).to(BF),
                down=rn(HID, MLP, scale=0.03).to(BF), n1=1 + rn(HID, scale=0.1), n2=1 + rn(HID, scale=0.1)), g


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def _table(rows):
    f = torch.pow(10000.0, -torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    a = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.stack((a.cos(), a.sin()), -1).float()


def _close(got, want, err):
    u = torch.finfo(got.dtype).eps / 2
    tol = err + u * want.abs() + torch.finfo(got.dtype).tiny
    excess = float(((got.double() - want).abs() - tol).max())
    assert excess <= 0, excess


def _product(x, w):
    x, w = x.to(BF).double(), w.double()
    return x @ w.t(), 2 * math.sqrt(x.shape[1]) * 2.0 ** -24 * (x.abs() @ w.abs().t())


def _turn(x, table, pos, n):
    x = x.double().clone()
    c, s = (table.double()[pos.long()][:, None][..., i] for i in (0, 1))
    a, b = x[:, :n, :D // 2].clone(), x[:, :n, D // 2:].clone()
    x[:, :n, :D // 2], x[:, :n, D // 2:] = a * c - b * s, b * c + a * s
    return x


def _attend(q, k, v, lens):
    out, mag = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    at = 0
    for n in lens:
        hide = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
        for h in range(HQ):
            s = q[at:at + n, h].double() @ k[at:at + n, h * HK // HQ].double().t() / math.sqrt(D)
            p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
            vv = v[at:at + n, h * HK // HQ].double()
            out[at:at + n, h], mag[at:at + n, h] = p @ vv, p @ vv.abs()
        at += n
    return out, mag


@pytest.mark.parametrize("lens", [[13, 4], [200, 77], [1500, 900]], ids=str)
def test_layer(qimg, lens):
    w, g = _weights(len(lens) + sum(lens))
    t = sum(lens)
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(n, dtype=torch.int32, device=DEV) for n in lens])
    table = _table(max(lens))
    stream = torch.randn(t, HID, generator=g, device=DEV)

    x = _norm(stream, w["n1"])
    qkv = qimg.linear_forward_bf16_fused(x, w["qkv"], bias=w["qkv_b"], out_dtype=torch.float32)
    z, e = _product(x, w["qkv"])
    _close(qkv, z + w["qkv_b"].double(), e + 2.0 ** -23 * z.abs())

    heads = qimg.rope_packed(qkv.view(t, HQ + 2 * HK, D), table, pos, HQ + HK, out_dtype=BF)
    want = _turn(qkv.view(t, HQ + 2 * HK, D), table, pos, HQ + HK)
    _close(heads, want, 2.0 ** -22 * qkv.view(t, HQ + 2 * HK, D).double().abs().amax(-1, keepdim=True))

    q, k, v = heads[:, :HQ], heads[:, HQ:HQ + HK], heads[:, HQ + HK:]
    attn = qimg.attention_varlen(q, k, v, cu, cu)
    want, mag = _attend(q, k, v, lens)
    u = torch.finfo(BF).eps / 2
    bound = 2 * u * (mag + want.abs()) + 2.0 ** -20 * mag
    _close(attn, want, bound)

    before = stream.clone()
    qimg.linear_forward_bf16_fused(attn.view(t, HID), w["o"], residual=stream, out=stream)
    z, e = _product(attn.view(t, HID), w["o"])
    _close(stream, before + z, e + 2.0 ** -23 * (z.abs() + before.abs()))

    x = _norm(stream, w["n2"])
    mid = qimg.linear_forward_bf16_fused(x, w["gate"], activation="silu", weight_up=w["up"])
    (z, e), (y, f) = _product(x, w["gate"]), _product(x, w["up"])
    a = z * torch.sigmoid(z)
    # exp2's argument is rounded: |t| 2^-23 of the result, |t| < 64 here
    _close(mid, a * y, 1.13 * e * y.abs() + a.abs() * f + 2 * e * f + 72 * 2.0 ** -23 * (a * y).abs())

    before = stream.clone()
    qimg.linear_forward_bf16_fused(mid, w["down"], residual=stream, out=stream)
    z, e = _product(mid, w["down"])
    _close(stream, before + z, e + 2.0 ** -23 * (z.abs() + before.abs()))

    # the last tokens again, one query a sequence over caches with room behind their last key
    room = 9
    cap = max(lens) + room
    kc = torch.full((len(lens) * cap, HK, D), float("nan"), dtype=BF, device=DEV)
    vc = kc.clone()
    at = 0
    for i, n in enumerate(lens):
        kc[i * cap:i * cap + n], vc[i * cap:i * cap + n] = k[at:at + n], v[at:at + n]
        at += n
    last = cu[1:].long() - 1
    one = qimg.attention_varlen(q[last], kc, vc, torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV),
                                torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV) * cap,
                                k_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    _close(one, want[last], bound[last])


def test_two_streams_at_once(qimg):
    """Independent calls on two streams, each with scratch of its own."""
    w, g = _weights(5)
    lens = [[300, 41], [1, 1, 1]]
    keys = [[300, 41], [2000, 700, 33]]
    data = []
    for a, b in zip(lens, keys):
        q = torch.randn(sum(a), HQ, D, generator=g, device=DEV).to(BF)
        k = torch.randn(sum(b), HK, D, generator=g, device=DEV).to(BF)
        cq, ck = (torch.tensor([0] + list(torch.tensor(n).cumsum(0)), dtype=torch.int32, device=DEV) for n in (a, b))
        x = torch.randn(sum(a), HID, generator=g, device=DEV).to(BF)
        data.append((q, k, cq, ck, x))

    def go(d):
        q, k, cq, ck, x = d
        return qimg.attention_varlen(q, k, k, cq, ck), qimg.linear_forward_bf16_fused(x, w["down"].t().contiguous())

    want = [go(d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = []
    for _ in range(10):
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(go(d))
    torch.cuda.synchronize()
    for i, pair in enumerate(got):
        for a, b in zip(pair, want[i % 2]):
            assert torch.equal(a, b)
