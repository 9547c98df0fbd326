"""What is timed of the operators around a prompt: packed attention, the
bf16 linear with its epilogue, and the rotary positions of packed heads.

A case is a dict of plain values; `kind` names the operator:

    attention   attention over packed sequences of different lengths, grouped
                heads, causal or not, also one query a sequence over a cache
    linear      bf16 product with bias, activation, gated second product,
                channel gate and residual in the epilogue
    rope        rotary positions of the q and k heads of packed rows

With `own` false, `run` computes them in plain torch operations in fp32; with
`own` true it calls the library.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
_DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


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
    text = {"kind": "attention", "dtype": "bf16", "hq": 28, "hk": 4, "d": 128, "causal": True, "cap": 0}
    return [
        # A prompt and its negative prompt, packed: the smallest whole-prompt call.
        dict(text, name="attn_prompt_pair", lq="77 13", lk="77 13"),
        # The two prompts of a long description: the ordinary whole-prompt call.
        dict(text, name="attn_prompt_512", lq="512 269", lk="512 269"),
        # A batch of prompts of every length, one of a single token among them.
        dict(text, name="attn_prompt_batch", lq="4096 2048 1531 1024 777 512 301 256 129 77 64 1",
             lk="4096 2048 1531 1024 777 512 301 256 129 77 64 1"),
        # One new token for each of 16 sequences, over caches with room behind their last key.
        dict(text, name="attn_token", lq="1 " * 15 + "1", cap=8192,
             lk="8192 7001 6144 5000 4097 4096 3333 2500 2048 1025 777 512 130 64 17 1"),
        # New tokens behind a cached prefix, other head sizes and type.
        {"name": "attn_prefix_d64", "kind": "attention", "dtype": "fp16", "hq": 16, "hk": 8, "d": 64, "causal": True,
         "cap": 0, "lq": "133 400 5", "lk": "1157 1424 1029"},
        # Unquantized joint attention of the two guidance branches of a 1024 x 1024 image, whose
        # prompts have 256 and 77 tokens: the largest call.
        {"name": "attn_joint_pair", "kind": "attention", "dtype": "fp16", "hq": 24, "hk": 24, "d": 128,
         "causal": False, "cap": 0, "lq": "4352 4173", "lk": "4352 4173"},
        # The q, k and v projection of one token, with its bias: bound by reading the weight.
        {"name": "linear_token", "kind": "linear", "m": 1, "n": 4608, "k": 3584, "x": "fp32", "out": "bf16",
         "bias": True, "act": "none", "gated": False, "gate": False, "residual": ""},
        # The gated pair of an MLP over a prompt and its negative prompt.
        {"name": "linear_gated_prompt", "kind": "linear", "m": 781, "n": 14336, "k": 3584, "x": "bf16", "out": "bf16",
         "bias": False, "act": "silu", "gated": True, "gate": False, "residual": ""},
        # Its way back onto the residual stream: few output tiles, a long sum.
        {"name": "linear_down_prompt", "kind": "linear", "m": 269, "n": 3584, "k": 14336, "x": "bf16", "out": "fp32",
         "bias": False, "act": "none", "gated": False, "gate": False, "residual": "fp32"},
        # A joint block's second MLP linear kept in bf16, with bias, channel gate and residual.
        {"name": "linear_joint", "kind": "linear", "m": 4352, "n": 3584, "k": 12288, "x": "bf16", "out": "fp32",
         "bias": True, "act": "none", "gated": False, "gate": True, "residual": "fp32"},
        # q, k and v of 16 new tokens.
        {"name": "rope_token", "kind": "rope", "t": 16, "h": 36, "h_rot": 32, "d": 128, "r": 128, "x": "bf16",
         "out": "bf16", "interleaved": False, "table": 8192},
        # q, k and v of a batch of prompts, straight from the fp32 projection.
        {"name": "rope_prompt_batch", "kind": "rope", "t": 10816, "h": 36, "h_rot": 32, "d": 128, "r": 128,
         "x": "fp32", "out": "bf16", "interleaved": False, "table": 4096},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["attention", "attention", "attention", "linear", "linear", "rope"])
    if kind == "attention":
        d = rng.choice([64, 128, 128])
        hq, hk = rng.choice([(28, 4), (28, 4), (24, 24), (16, 8), (8, 1), (12, 2), (6, 6)])
        c = {"kind": kind, "dtype": rng.choice(["bf16", "fp16"]), "hq": hq, "hk": hk, "d": d, "causal": True, "cap": 0}
        form = rng.choice(["prompt", "prompt", "token", "prefix", "joint"])
        if form == "prompt":
            lq = [log(1, 2048) for _ in range(rng.randint(1, 10))]
            lk = lq
        elif form == "token":
            lk = [log(1, 8192) for _ in range(rng.randint(1, 32))]
            lq = [1] * len(lk)
            c["cap"] = max(lk) + rng.randint(0, 100)
        elif form == "prefix":
            lq = [log(1, 512) for _ in range(rng.randint(1, 6))]
            lk = [n + log(1, 4096) for n in lq]
        else:
            c["causal"] = False
            n = log(64, 3500)
            lq = [n + rng.randint(1, 256) for _ in range(rng.randint(1, 2))]
            lk = lq
        c["lq"], c["lk"] = _text(lq), _text(lk)
        return c
    if kind == "linear":
        n, k = rng.choice([(4608, 3584), (3584, 3584), (14336, 3584), (3584, 14336), (12288, 1536), (1000, 2056),
                           (3584, 64), (333, 1000)])
        gated = n == 14336 and rng.random() < 0.7
        residual = "" if gated else rng.choice(["", "fp32", "bf16"])
        return {"kind": kind, "m": log(1, 2048), "n": n, "k": k, "x": rng.choice(["bf16", "bf16", "fp32"]),
                "out": residual or rng.choice(["bf16", "fp32"]), "bias": rng.random() < 0.6,
                "act": "silu" if gated else rng.choice(["none", "none", "gelu", "silu"]), "gated": gated,
                "gate": bool(residual) and rng.random() < 0.5, "residual": residual}
    d = rng.choice([64, 128])
    h_rot = rng.randint(1, 32)
    return {"kind": kind, "t": log(1, 10000), "h": h_rot + rng.randint(0, 8), "h_rot": h_rot, "d": d,
            "r": rng.choice([d, d, d // 2]), "x": rng.choice(["fp32", "bf16"]), "out": rng.choice(["bf16", "fp16"]),
            "interleaved": rng.random() < 0.3, "table": rng.choice([1024, 8192, 100000])}


# ---- inputs ----------------------------------------------------------------

def _offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def _angles(rows, r):
    """Rotary angles [rows, r / 2] in 64 bits: position * 10000^(-2 i / r)."""
    freq = torch.pow(10000.0, -torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)
    return torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * freq


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    s = dict(case)
    if case["kind"] == "attention":
        t = _DT[case["dtype"]]
        d, hk = case["d"], case["hk"]
        lq, lk = _lens(case["lq"]), _lens(case["lk"])
        oq = _offsets(lq)
        slots = [case["cap"]] * len(lk) if case["cap"] else lk
        ok = _offsets(slots)
        # keys share a mean per channel, as projections with a bias give them
        s["q"] = (randn(oq[-1], case["hq"], d) + 0.3 * randn(case["hq"], d)).to(t)
        s["k"] = (randn(ok[-1], hk, d) + 0.5 * randn(hk, d)).to(t)
        s["v"] = randn(ok[-1], hk, d).to(t)
        s["lens"], s["oq"], s["ok"] = list(zip(lq, lk)), oq, ok
        s["cu_q"] = torch.tensor(oq, dtype=torch.int32, device=DEV)
        s["cu_k"] = torch.tensor(ok, dtype=torch.int32, device=DEV)
        s["k_lens"] = torch.tensor(lk, dtype=torch.int32, device=DEV) if case["cap"] else None
        s["sm_scale"] = 1.0 / math.sqrt(d)
        return s
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s["X"] = randn(m, k).to(_DT[case["x"]])
        s["W"] = (0.02 * randn(n, k)).to(torch.bfloat16)
        s["W_up"] = (0.02 * randn(n, k)).to(torch.bfloat16) if case["gated"] else None
        s["B"] = (0.1 * randn(n)).to(torch.bfloat16) if case["bias"] else None
        s["B_up"] = (0.1 * randn(n)).to(torch.bfloat16) if case["bias"] and case["gated"] else None
        s["G"] = 0.5 * randn(n) if case["gate"] else None
        s["R"] = randn(m, n).to(_DT[case["residual"]]) if case["residual"] else None
        return s
    a = _angles(case["table"], case["r"])
    s["X"] = randn(case["t"], case["h"], case["d"]).to(_DT[case["x"]])
    s["table_cs"] = torch.stack((a.cos(), a.sin()), dim=-1).to(torch.float32)
    s["pos"] = torch.randint(0, case["table"], (case["t"],), generator=g, device=DEV, dtype=torch.int32)
    return s


# ---- one pass ----------------------------------------------------------------

def run(state):
    return {"attention": _run_attention, "linear": _run_linear, "rope": _run_rope}[state["kind"]](state)


def _run_attention(s):
    if own:
        return _lib().attention_varlen(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], sm_scale=s["sm_scale"],
                                       causal=s["causal"], k_lens=s["k_lens"])
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    out = torch.empty_like(s["q"])
    group = s["hq"] // s["hk"]
    for i, (lq, lk) in enumerate(s["lens"]):
        q0, k0 = s["oq"][i], s["ok"][i]
        hidden = None
        if s["causal"]:
            last = torch.arange(lq, device=DEV) + (lk - lq)
            hidden = torch.arange(lk, device=DEV)[None, :] > last[:, None]
        step = max(1, (1 << 28) // (group * lq * lk))
        for h in range(0, s["hk"], step):
            e = min(h + step, s["hk"])
            qs = q[q0:q0 + lq, h * group:e * group].reshape(lq, e - h, group, -1).permute(1, 2, 0, 3)
            qs = qs.reshape(e - h, group * lq, -1)
            ks = k[k0:k0 + lk, h:e].permute(1, 2, 0).contiguous()
            vs = v[k0:k0 + lk, h:e].permute(1, 0, 2).contiguous()
            p = (torch.bmm(qs, ks) * s["sm_scale"]).reshape(e - h, group, lq, lk)
            if hidden is not None:
                p = p.masked_fill(hidden, float("-inf"))
            p = torch.exp(p - p.amax(dim=-1, keepdim=True))
            p = p / p.sum(dim=-1, keepdim=True)
            o = torch.bmm(p.reshape(e - h, group * lq, lk), vs).reshape(e - h, group, lq, -1)
            out[q0:q0 + lq, h * group:e * group] = o.permute(2, 0, 1, 3).reshape(lq, (e - h) * group, -1).to(out.dtype)
    return out


def _run_linear(s):
    if own:
        return _lib().linear_forward_bf16_fused(s["X"], s["W"], bias=s["B"], activation=s["act"], weight_up=s["W_up"],
                                                bias_up=s["B_up"], gate=s["G"], residual=s["R"],
                                                out_dtype=_DT[s["out"]])
    x = s["X"].to(torch.bfloat16).float()
    z = x @ s["W"].float().t()
    if s["B"] is not None:
        z = z + s["B"].float()
    if s["act"] == "silu":
        z = z / (1.0 + torch.exp(-z))
    elif s["act"] == "gelu":
        z = z / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if s["W_up"] is not None:
        u = x @ s["W_up"].float().t()
        if s["B_up"] is not None:
            u = u + s["B_up"].float()
        z = z * u
    if s["G"] is not None:
        z = z * s["G"]
    if s["R"] is not None:
        z = z + s["R"].float()
    return z.to(_DT[s["out"]])


def _run_rope(s):
    if own:
        return _lib().rope_packed(s["X"], s["table_cs"], s["pos"], s["h_rot"], interleaved=s["interleaved"],
                                  out_dtype=_DT[s["out"]])
    x = s["X"].float()
    r, hr = s["r"], s["h_rot"]
    cs = s["table_cs"][s["pos"].long()][:, None]
    cos, sin = cs[..., 0], cs[..., 1]
    out = x.clone()
    if s["interleaved"]:
        a, b = x[:, :hr, 0:r:2], x[:, :hr, 1:r:2]
        out[:, :hr, 0:r:2] = a * cos - b * sin
        out[:, :hr, 1:r:2] = b * cos + a * sin
    else:
        a, b = x[:, :hr, :r // 2], x[:, :hr, r // 2:r]
        out[:, :hr, :r // 2] = a * cos - b * sin
        out[:, :hr, r // 2:r] = b * cos + a * sin
    return out.to(_DT[s["out"]])


# ---- what a pass cannot do without ---------------------------------------------

def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    if case["kind"] == "attention":
        pairs = 0
        qs, ks = _lens(case["lq"]), _lens(case["lk"])
        for lq, lk in zip(qs, ks):
            pairs += lq * lk - (lq * (lq - 1) // 2 if case["causal"] else 0)
        rows = 2 * sum(qs) * case["hq"] + 2 * sum(ks) * case["hk"]
        return {"bytes": 2 * case["d"] * rows, "flops": 4 * case["d"] * case["hq"] * pairs}
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        products = 2 if case["gated"] else 1
        b = m * k * size[case["x"]] + products * n * k * 2 + m * n * size[case["out"]]
        if case["residual"]:
            b += m * n * size[case["residual"]]
        b += n * (2 * products * case["bias"] + 4 * case["gate"])
        return {"bytes": b, "flops": 2 * products * m * n * k}
    t, h, d = case["t"], case["h"], case["d"]
    return {"bytes": t * (h * d * (size[case["x"]] + size[case["out"]]) + 4) + min(t, case["table"]) * case["r"] * 4,
            "flops": 3 * t * case["h_rot"] * case["r"]}


# ---- the definitions in 64 bits --------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attention":
        group = case["hq"] // case["hk"]
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        for i, (lq, lk) in enumerate(s["lens"]):
            keys = torch.arange(lk, device=DEV)
            for h in range(case["hq"]):
                kh = s["k"][s["ok"][i]:s["ok"][i] + lk, h // group].double()
                vh = s["v"][s["ok"][i]:s["ok"][i] + lk, h // group].double()
                for r0 in range(0, lq, 8192):
                    r1 = min(r0 + 8192, lq)
                    x = s["q"][s["oq"][i] + r0:s["oq"][i] + r1, h].double() @ kh.t() * s["sm_scale"]
                    if case["causal"]:
                        rows = torch.arange(r0, r1, device=DEV)
                        x[keys[None, :] > rows[:, None] + (lk - lq)] = -math.inf
                    out[s["oq"][i] + r0:s["oq"][i] + r1, h] = torch.softmax(x, dim=-1) @ vh
        return out
    if case["kind"] == "linear":
        x = s["X"].to(torch.bfloat16).double()
        z = x @ s["W"].double().t()
        z = z if s["B"] is None else z + s["B"].double()
        if case["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif case["act"] == "gelu":
            z = 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
        if case["gated"]:
            u = x @ s["W_up"].double().t()
            z = z * (u if s["B_up"] is None else u + s["B_up"].double())
        z = z if s["G"] is None else z * s["G"].double()
        return z if s["R"] is None else z + s["R"].double()
    x, r, hr = s["X"].double(), case["r"], case["h_rot"]
    a = s["table_cs"].double()[s["pos"].long()]
    c = torch.complex(a[..., 0], a[..., 1])[:, None]
    turned = x[:, :hr, :r]
    if case["interleaved"]:
        z = torch.view_as_complex(turned.reshape(*turned.shape[:-1], r // 2, 2).contiguous()) * c
        part = torch.view_as_real(z).reshape(turned.shape)
    else:
        z = torch.complex(turned[..., :r // 2].contiguous(), turned[..., r // 2:].contiguous()) * c
        part = torch.cat((z.real, z.imag), dim=-1)
    x[:, :hr, :r] = part
    return x
