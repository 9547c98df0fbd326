"""What is timed of the operators around a quantized key/value cache: norms of
the q and k heads with their rotation, the cache as it is written and read
back, attention over its pages, and attention of a batch that shares a prefix.

A case is a dict of plain values; `kind` names the operator:

    heads       per-head RMS norm of q and k, and their rotary positions, of packed rows
    cache       the same with k and v quantized into pages, then the sequences read back
    attention   queries over the pages of their sequences
    prefix      the same behind one prefix that all sequences share

A cache holds codes, int8 or e4m3, of rows (token, kv head) of d values, and a
power of two for each row: the least 2^e, e >= -126, with max|x| <= 127 * 2^e
(int8) or 448 * 2^e (e4m3). A code is x / 2^e, rounded half to even.

With `own` false, `run` computes them in plain torch operations in fp32; with
`own` true it calls the library.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
EPS = 1e-6
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _text(lens):
    """Sequence lengths as a case holds them: numbers in a text."""
    return " ".join(str(n) for n in lens)


def _lens(text):
    return [int(n) for n in text.split()]


def _lib():
    pkg = os.path.join(os.getcwd(), "qwen-image.cu_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import qimg_amd
    return qimg_amd


def listed():
    text = {"hq": 28, "hk": 4, "d": 128, "q": "bf16", "codes": "e4m3", "page": 64, "causal": True}
    heads = {"kind": "heads", "d": 128, "r": 128, "x": "fp32", "out": "bf16", "interleaved": False}
    return [
        # q, k and v of 16 new tokens: the smallest call, all latency.
        dict(heads, name="heads_token", t=16, hq=28, hk=4, x="bf16", table=8192),
        # q, k and v of a batch of prompts, straight from the fp32 projection.
        dict(heads, name="heads_prompt_batch", t=10816, hq=28, hk=4, table=4096),
        # The joint attention's heads of a 1024 x 1024 image and its prompt, interleaved pairs.
        dict(heads, name="heads_joint", t=4352, hq=24, hk=24, out="fp16", interleaved=True, table=4352),
        # One new token for each of 16 sequences, written into their pages.
        dict(text, name="cache_token", kind="cache", r=128, x="bf16", interleaved=False,
             old="512 301 256 129 77 64 33 17 13 8 5 4 3 2 1 0", new="1 " * 15 + "1"),
        # Two long descriptions behind a template, int8, small pages.
        dict(text, name="cache_prompt", kind="cache", codes="int8", page=16, r=128, x="fp32", interleaved=False,
             old="34 34", new="478 235"),
        # A batch of prompts and what they stand behind, read back whole.
        dict(text, name="cache_prompt_batch", kind="cache", page=128, r=128, x="fp32", interleaved=False,
             old="28672 4096 1024 0 0 17 2000 8192 500 1", new="4096 2048 1531 1024 777 512 301 256 129 77"),
        # One new token for each of 16 sequences of every length: the ordinary serving step.
        dict(text, name="attn_token", kind="attention", lq="1 " * 15 + "1",
             lk="8192 7001 6144 5000 4097 4096 3333 2500 2048 1025 777 512 130 64 17 1"),
        # The same for 64 long sequences: the most that is read.
        dict(text, name="attn_token_long", kind="attention", codes="int8", lq="1 " * 63 + "1",
             lk=_text([16384 - 61 * i for i in range(64)])),
        # A few drafted tokens a sequence, other head sizes and type.
        dict(text, name="attn_draft_d64", kind="attention", hq=16, hk=8, d=64, q="fp16", page=16,
             lq="4 5 4 1 8 3 4 2", lk="1157 1424 1029 3000 77 640 2048 4000"),
        # A long description in pieces behind what is cached of it: bound by the products.
        dict(text, name="attn_piece", kind="attention", lq="1024 333", lk="8192 2381"),
        # One new token for each of 32 variants of a prompt behind their common part.
        dict(text, name="prefix_token", kind="prefix", prefix=4096, lq="1 " * 31 + "1",
             lk=_text([1 + 7 * i for i in range(32)])),
        # 128 variants behind a long one, int8.
        dict(text, name="prefix_long", kind="prefix", codes="int8", page=32, prefix=16000, lq="1 " * 127 + "1",
             lk=_text([1 + 4 * i for i in range(128)])),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["heads", "cache", "attention", "attention", "attention", "prefix", "prefix"])
    d = rng.choice([64, 128, 128])
    hq, hk = rng.choice([(28, 4), (28, 4), (24, 24), (16, 8), (8, 1), (12, 2), (6, 6)])
    c = {"kind": kind, "hq": hq, "hk": hk, "d": d}
    if kind in ("heads", "cache"):
        c.update(r=rng.choice([d, d, d // 2]), x=rng.choice(["fp32", "bf16", "fp16"]),
                 interleaved=rng.random() < 0.3)
    if kind == "heads":
        c.update(t=log(1, 10000), out=rng.choice(["bf16", "fp16"]), table=rng.choice([1024, 8192, 100000]))
        return c
    c.update(q=rng.choice(["bf16", "bf16", "fp16"]), codes=rng.choice(["e4m3", "int8"]),
             page=rng.choice([16, 32, 64, 128, 256]))
    if kind == "cache":
        n = rng.randint(1, 16)
        tokens = rng.random() < 0.4
        c["new"] = _text([1 if tokens else log(1, 1500) for _ in range(n)])
        c["old"] = _text([log(1, 6000) - 1 for _ in range(n)])
        return c
    c["causal"] = rng.random() < 0.9
    form = rng.choice(["token", "token", "draft", "piece"]) if kind == "attention" else rng.choice(["token", "draft"])
    if form == "piece":
        lq = [log(16, 1024) for _ in range(rng.randint(1, 4))]
        lk = [n + log(1, 7000) - 1 for n in lq]
    else:
        lq = [1 if form == "token" else rng.randint(1, 9) for _ in range(log(1, 96 if kind == "prefix" else 48))]
        lk = [n + log(1, 1024 if kind == "prefix" else 16384) - 1 for n in lq]
    if kind == "prefix":
        c["prefix"] = log(1, 16384)
    c["lq"], c["lk"] = _text(lq), _text(lk)
    return c


# ---- inputs ----------------------------------------------------------------

def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(rows, r):
    """cos and sin of position * 10000^(-2 i / r), fp32 [rows, r / 2, 2] from angles in 64 bits."""
    freq = torch.pow(10000.0, -torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)
    a = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * freq
    return torch.stack((a.cos(), a.sin()), dim=-1).to(torch.float32)


def _power(e):
    """2^e, e in [-126, 127], fp32, by its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantize(x, codes):
    """Rows [..., d] fp32 -> their codes and biased exponents."""
    m, ex = torch.frexp(x.abs().amax(dim=-1))
    e = ex - 7 + (m > 127 / 128).int() if codes == "int8" else ex - 9 + (m > 0.875).int()
    e = e.clamp(min=-126)
    y = x * _power(-e)[..., None]
    return (y.round() if codes == "int8" else y).to(_CODE[codes]), (e + 127).to(torch.uint8)


def _dequantize(codes, exps):
    return codes.float() * _power(exps.int() - 127)[..., None]


def _pages(s, lens, randn, g):
    """A cache with the sequences' pages in any order, a few that nobody owns among them."""
    hk, d, page = s["hk"], s["d"], s["page"]
    each = [-(-n // page) for n in lens]
    total = sum(each) + 3
    rows = randn(total, hk, page, d)
    for name in ("k", "v"):
        # keys share a mean per channel, as projections with a bias give them
        rows = rows + 0.5 * randn(hk, 1, d) if name == "k" else randn(total, hk, page, d)
        c, e = _quantize(rows, s["codes"])
        s["c" + name], s["e" + name] = c, e
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    tables, at = [], 0
    for n in each:
        tables.append(order[at:at + n])
        at += n
    return tables


def _block_table(tables):
    width = max(1, max(t.numel() for t in tables))
    return torch.stack([torch.nn.functional.pad(t, (0, width - t.numel())) for t in tables]).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    s = dict(case)
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["kind"] in ("heads", "cache"):
        s["wq"], s["wk"] = ((1.0 + 0.2 * randn(d)).to(torch.bfloat16) for _ in range(2))
    if case["kind"] == "heads":
        s["X"] = randn(case["t"], hq + 2 * hk, d).to(_DT[case["x"]])
        s["table_cs"] = _table(case["table"], case["r"])
        s["pos"] = torch.randint(0, case["table"], (case["t"],), generator=g, device=DEV, dtype=torch.int32)
        return s
    if case["kind"] == "cache":
        old, new = _lens(case["old"]), _lens(case["new"])
        both = [a + b for a, b in zip(old, new)]
        tables = _pages(s, both, randn, g)
        s["X"] = randn(sum(new), hq + 2 * hk, d).to(_DT[case["x"]])
        s["table_cs"] = _table(max(both), case["r"])
        pos = [torch.arange(a, a + b, device=DEV) for a, b in zip(old, new)]
        s["pos"] = torch.cat(pos).to(torch.int32)
        page = case["page"]
        s["slots"] = torch.cat([t.long()[p // page] * page + p % page for t, p in zip(tables, pos)]).to(torch.int32)
        s["tables"], s["k_lens"], s["cu_k"], s["total_k"] = _block_table(tables), _i32(both), _i32(_offsets(both)), sum(both)
        every = [torch.arange(n, device=DEV) for n in both]
        s["where"] = torch.cat([t.long()[p // page] * page + p % page for t, p in zip(tables, every)])
        return s
    lq, lk = _lens(case["lq"]), _lens(case["lk"])
    shared = [case["prefix"]] if case["kind"] == "prefix" else []
    tables = _pages(s, lk + shared, randn, g)
    if shared:
        s["prefix_table"], s["prefix_len"] = tables.pop().contiguous(), _i32(shared)
    s["q"] = (randn(sum(lq), hq, d) + 0.3 * randn(hq, d)).to(_DT[case["q"]])
    s["tables"], s["k_lens"], s["cu_q"] = _block_table(tables), _i32(lk), _i32(_offsets(lq))
    s["sm_scale"] = 1.0 / math.sqrt(d)
    # the plain form's padded batch: which query a padded row is, and where each query went
    most, oq = max(lq), _offsets(lq)
    s["most"] = most
    s["pad"] = torch.tensor([[oq[b] + min(i, n - 1) for i in range(most)] for b, n in enumerate(lq)], device=DEV)
    s["unpad"] = torch.tensor([b * most + i for b, n in enumerate(lq) for i in range(n)], device=DEV)
    s["last"] = torch.tensor([[k - n + i if case["causal"] else k - 1 for i in range(most)] for n, k in zip(lq, lk)],
                             device=DEV)
    return s


# ---- one pass ----------------------------------------------------------------

def run(state):
    return {"heads": _run_heads, "cache": _run_cache}.get(state["kind"], _run_attention)(state)


def _cache(s):
    return _lib().KvCache(s["ck"], s["cv"], s["ek"], s["ev"])


def _heads(s):
    """Normed, turned heads of the packed rows, fp32."""
    x = s["X"].float()
    hq, hk, r = s["hq"], s["hk"], s["r"]
    w = torch.cat((s["wq"].float().expand(hq, -1), s["wk"].float().expand(hk, -1)))
    qk = x[:, :hq + hk]
    qk = qk * torch.rsqrt((qk * qk).mean(dim=-1, keepdim=True) + EPS) * w
    cs = s["table_cs"][s["pos"].long()][:, None]
    cos, sin = cs[..., 0], cs[..., 1]
    at, bt = (slice(0, r, 2), slice(1, r, 2)) if s["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    a, b = qk[..., at], qk[..., bt]
    turned = qk.clone()
    turned[..., at] = a * cos - b * sin
    turned[..., bt] = b * cos + a * sin
    return torch.cat((turned, x[:, hq + hk:]), dim=1)


def _run_heads(s):
    if own:
        return _lib().norm_rope_packed(s["X"], s["hq"], s["hk"], s["wq"], s["wk"], EPS, s["table_cs"], s["pos"],
                                       interleaved=s["interleaved"], out_dtype=_DT[s["out"]])
    return _heads(s).to(_DT[s["out"]])


def _run_cache(s):
    hq, hk, d, page = s["hq"], s["hk"], s["d"], s["page"]
    t = _DT[s["q"]]
    if own:
        lib, cache = _lib(), _cache(s)
        q = lib.norm_rope_cache(s["X"], hq, cache, s["slots"], s["wq"], s["wk"], EPS, s["table_cs"], s["pos"],
                                interleaved=s["interleaved"], out_dtype=t)
        k, v = lib.kv_cache_read(cache, s["tables"], s["k_lens"], s["cu_k"], s["total_k"], out_dtype=t)
        return {"q": q, "k": k, "v": v}
    y = _heads(s)
    slots, where, back = s["slots"].long(), s["where"], []
    for name, rows in (("k", y[:, hq:hq + hk]), ("v", y[:, hq + hk:])):
        c, e = _quantize(rows, s["codes"])
        s["c" + name].view(torch.uint8)[slots // page, :, slots % page] = c.view(torch.uint8)
        s["e" + name][slots // page, :, slots % page] = e
        codes = s["c" + name].view(torch.uint8)[where // page, :, where % page].view(_CODE[s["codes"]])
        back.append(_dequantize(codes, s["e" + name][where // page, :, where % page]).to(t))
    return {"q": y[:, :hq].to(t), "k": back[0], "v": back[1]}


def _dense(s, name, tables):
    """The rows of tables [b, n] of pages, fp32 [b, hk, n * page, d]."""
    at = tables.long()
    codes = s["c" + name].view(torch.uint8)[at].view(_CODE[s["codes"]])
    x = _dequantize(codes, s["e" + name][at]).transpose(1, 2)
    return x.reshape(at.shape[0], s["hk"], -1, s["d"])


def _run_attention(s):
    prefix = s["kind"] == "prefix"
    if own:
        more = {"prefix_table": s["prefix_table"], "prefix_len": s["prefix_len"]} if prefix else {}
        return _lib().attention_cache(s["q"], _cache(s), s["cu_q"], s["tables"], s["k_lens"], sm_scale=s["sm_scale"],
                                      causal=s["causal"], **more)
    hq, hk, d, most = s["hq"], s["hk"], s["d"], s["most"]
    batch, group = s["tables"].shape[0], hq // hk
    q = s["q"].float()[s["pad"]].reshape(batch, most, hk, group, d).permute(0, 2, 3, 1, 4)
    q = q.reshape(batch * hk, group * most, d) * s["sm_scale"]
    k = _dense(s, "k", s["tables"]).reshape(batch * hk, -1, d)
    n = k.shape[1]
    p = torch.bmm(q, k.transpose(1, 2).contiguous()).reshape(batch, hk, group, most, n)
    hidden = torch.arange(n, device=DEV) > torch.minimum(s["last"], s["k_lens"][:, None] - 1)[..., None]
    p = p.masked_fill(hidden[:, None, None], float("-inf"))
    top = p.amax(dim=-1, keepdim=True)
    if prefix:
        kp, vp = (_dense(s, name, s["prefix_table"][None])[0, :, :s["prefix"]] for name in ("k", "v"))
        qp = q.reshape(batch, hk, group * most, d).transpose(0, 1).reshape(hk, batch * group * most, d)
        pp = torch.bmm(qp, kp.transpose(1, 2).contiguous())
        pp = pp.reshape(hk, batch, group, most, -1).transpose(0, 1)
        top = torch.maximum(top, pp.amax(dim=-1, keepdim=True))
        pp = torch.exp(pp - top)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(p - top)
    total = p.sum(dim=-1, keepdim=True)
    v = _dense(s, "v", s["tables"]).reshape(batch * hk, -1, d)
    o = torch.bmm(p.reshape(batch * hk, group * most, n), v).reshape(batch, hk, group, most, d)
    if prefix:
        total = total + pp.sum(dim=-1, keepdim=True)
        op = torch.bmm(pp.transpose(0, 1).reshape(hk, batch * group * most, -1), vp.contiguous())
        o = o + op.reshape(hk, batch, group, most, d).transpose(0, 1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(batch * most, hq, d)[s["unpad"]].to(s["q"].dtype)


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["kind"] == "heads":
        t, h = case["t"], hq + 2 * hk
        rows = min(t, case["table"])
        return {"bytes": t * (h * d * (size[case["x"]] + size[case["out"]]) + 4) + rows * case["r"] * 4,
                "flops": t * (hq + hk) * (4 * d + 3 * case["r"])}
    if case["kind"] == "cache":
        old, new = sum(_lens(case["old"])), sum(_lens(case["new"]))
        row = 2 * hk * (d + 1)
        b = new * ((hq + 2 * hk) * d * size[case["x"]] + 2 * hq * d + row + 8 + 4 * case["r"])
        return {"bytes": b + (old + new) * (row + 2 * hk * d * 2), "flops": new * (hq + 2 * hk) * 7 * d}
    lq, lk = _lens(case["lq"]), _lens(case["lk"])
    pairs = sum(n * k - (n * (n - 1) // 2 if case["causal"] else 0) for n, k in zip(lq, lk))
    keys = sum(lk)
    if case["kind"] == "prefix":
        pairs += sum(lq) * case["prefix"]
        keys += case["prefix"]
    return {"bytes": 4 * sum(lq) * hq * d + 2 * keys * hk * (d + 1), "flops": 4 * d * hq * pairs}


# ---- the definitions in 64 bits --------------------------------------------------

def _two_to(n):
    """2^n, fp64."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _value(codes, exps):
    """What codes and biased exponents stand for: e4m3 by its bits."""
    if codes.dtype == torch.int8:
        c = codes.double()
    else:
        u = codes.view(torch.uint8).int()
        ex, m = (u >> 3) & 15, (u & 7).double()
        c = torch.where(ex == 0, m / 8 * 2.0 ** -6, (1 + m / 8) * _two_to(ex - 7))
        c = torch.where(u >= 128, -c, c)
    return c * _two_to(exps.int() - 127)[..., None]


def exact(case, seed):
    s = prepare(case, seed)
    hq, hk = case["hq"], case["hk"]
    if case["kind"] in ("heads", "cache"):
        x, r = s["X"].double(), case["r"]
        for h0, h1, w in ((0, hq, s["wq"]), (hq, hq + hk, s["wk"])):
            x[:, h0:h1] /= (x[:, h0:h1].square().sum(dim=-1, keepdim=True) / case["d"] + EPS).sqrt()
            x[:, h0:h1] *= w.double()
        a = s["table_cs"].double()[s["pos"].long()]
        c = torch.complex(a[..., 0], a[..., 1])[:, None]
        part = x[:, :hq + hk, :r]
        if case["interleaved"]:
            z = torch.view_as_complex(part.reshape(*part.shape[:-1], r // 2, 2).contiguous()) * c
            x[:, :hq + hk, :r] = torch.view_as_real(z).reshape(part.shape)
        else:
            z = torch.complex(part[..., :r // 2].contiguous(), part[..., r // 2:].contiguous()) * c
            x[:, :hq + hk, :r] = torch.cat((z.real, z.imag), dim=-1)
        if case["kind"] == "heads":
            return x
        # Which of two codes a k next to their border takes is up to the last of the 32 bits that it is
        # computed in, so k has no value here; v is quantized as it is.
        page, slots, where = case["page"], s["slots"].long(), s["where"]
        v = _value(s["cv"], s["ev"])
        rows = x[:, hq + hk:]
        most = 127.0 if case["codes"] == "int8" else 448.0
        top = rows.abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -126)
        unit = _two_to(torch.ceil(torch.log2(top / most)))
        unit = torch.where(unit / 2 * most >= top, unit / 2, torch.where(unit * most < top, unit * 2, unit))
        unit = unit.clamp(min=2.0 ** -126)
        y = rows / unit
        # e4m3: steps of 2^-3 of the power of two below, of 2^-9 at least
        step = 1.0 if case["codes"] == "int8" else _two_to(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 4)
        v[slots // page, :, slots % page] = torch.round(y / step) * step * unit
        return {"q": x[:, :hq], "k": None, "v": v[where // page, :, where % page]}
    page, group = case["page"], hq // hk
    lq, lk = _lens(case["lq"]), _lens(case["lk"])
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    shared = case.get("prefix", 0)

    def rows(name, pages, n):
        at = pages[:-(-n // page)].long()
        return _value(s["c" + name][at], s["e" + name][at]).transpose(0, 1).reshape(hk, -1, case["d"])[:, :n]

    kp, vp = (rows(name, s["prefix_table"], shared) for name in ("k", "v")) if shared else (None, None)
    q0 = 0
    for b, (nq, nk) in enumerate(zip(lq, lk)):
        kb, vb = (rows(name, s["tables"][b], nk) for name in ("k", "v"))
        if shared:
            kb, vb = torch.cat((kp, kb), dim=1), torch.cat((vp, vb), dim=1)
        for h in range(hk):
            x = s["q"][q0:q0 + nq, h * group:(h + 1) * group].double().reshape(nq * group, -1) @ kb[h].t() * s["sm_scale"]
            if case["causal"]:
                token = torch.arange(nq * group, device=DEV) // group
                x[torch.arange(shared + nk, device=DEV)[None] > token[:, None] + (shared + nk - nq)] = -math.inf
            out[q0:q0 + nq, h * group:(h + 1) * group] = (torch.softmax(x, dim=-1) @ vb[h]).reshape(nq, group, -1)
        q0 += nq
    return out
