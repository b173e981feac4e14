"""The mixture-of-experts layer and the matrix product with an epilogue, over GGUF-quantised weights: cases, plain forms, exact values.

  moe     y = residual + sum_j weight_j * Down_j (act(Gate_j x) * (Up_j x)), the experts j picked by a router (or given)
  linear  y = act(x W^T + bias) + residual, f32 or bf16

Weights are GGUF blocks (Q4_0, Q8_0, Q4_K, Q5_K, Q6_K; "layout" 1 is the NodeStor element mapping of Q5_K and Q6_K).
"""
import math

import torch

own = False

Q4_0, Q8_0, Q4_K, Q5_K, Q6_K = 2, 8, 12, 13, 14
BLOCK = {Q4_0: (32, 18), Q8_0: (32, 34), Q4_K: (256, 144), Q5_K: (256, 176), Q6_K: (256, 210)}  # weights, bytes


def _row_bytes(t, k):
    return k // BLOCK[t][0] * BLOCK[t][1]


# ---------------------------------------------------------------- cases
def _moe(name, **c):
    base = {"op": "moe", "name": name, "score": "softmax_norm", "sel_bias": False, "scale": 1.0, "residual": False,
            "given": False, "layout": 0, "layout_down": 0, "act": "silu"}
    return {**base, **c}


def _lin(name, **c):
    return {**{"op": "linear", "name": name, "layout": 0, "bias": True, "act": "none", "residual": False}, **c}


def listed():
    return [
        # one token of a model with many small experts: launches and latency count
        _moe("moe_1tok_128e", m=1, e=128, k=8, d=2048, f=768, t_in=Q4_K, t_down=Q6_K),
        # one token, few large experts: two experts' weights stream from memory
        _moe("moe_1tok_8e", m=1, e=8, k=2, d=4096, f=14336, t_in=Q4_K, t_down=Q4_K),
        # a decode batch of 16 that touches every large expert
        _moe("moe_16tok_8e", m=16, e=8, k=2, d=4096, f=14336, t_in=Q4_K, t_down=Q6_K, residual=True),
        # a larger batch, sigmoid scores with a selection bias, 8-bit experts whose width is no multiple of 256
        _moe("moe_32tok_64e", m=32, e=64, k=6, d=2048, f=1408, t_in=Q8_0, t_down=Q8_0, score="sigmoid_norm",
             sel_bias=True, scale=2.5),
        # experts spread over ranks: given picks, unused slots (-1), tokens without any expert here; odd widths
        _moe("moe_given_7tok", m=7, e=32, k=4, d=1056, f=992, t_in=Q4_0, t_down=Q4_0, given=True, residual=True),
        # the smallest call: one token's biased projection
        _lin("linear_1tok_qkv", m=1, n=1152, kk=896, t=Q8_0, dtype="f32"),
        # one token's down projection with the residual stream
        _lin("linear_1tok_down", m=1, n=4096, kk=14336, t=Q6_K, dtype="f32", bias=False, residual=True),
        # a decode batch through a GELU feed-forward input
        _lin("linear_16tok_ff", m=16, n=14336, kk=4096, t=Q4_K, dtype="f32", act="gelu_tanh"),
        # bf16 serving, a few tokens, wide rows
        _lin("linear_3tok_bf16", m=3, n=28672, kk=8192, t=Q5_K, dtype="bf16", act="silu"),
        # an odd prompt against an odd number of rows
        _lin("linear_333_bf16", m=333, n=1003, kk=2816, t=Q8_0, dtype="bf16", act="relu", residual=True),
        # prompts
        _lin("linear_512_bf16", m=512, n=14336, kk=4096, t=Q4_K, dtype="bf16", act="gelu"),
        _lin("linear_2048_bf16", m=2048, n=4096, kk=14336, t=Q6_K, dtype="bf16", residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    t = rng.choice([Q4_0, Q8_0, Q4_K, Q5_K, Q6_K])
    if rng.random() < 0.5:
        td = rng.choice([Q4_0, Q8_0, Q4_K, Q5_K, Q6_K])
        d_unit, f_unit = BLOCK[t][0], BLOCK[td][0]
        d, f = d_unit * max(1, _log(rng, 512, 4096) // d_unit), f_unit * max(1, _log(rng, 256, 8192) // f_unit)
        e = _log(rng, 2, 128)
        while e * d * f > 400_000_000:
            e = max(2, e // 2)
        c = _moe("", m=_log(rng, 1, 48), e=e, k=rng.randint(1, min(8, e)), d=d, f=f, t_in=t, t_down=td,
                 score=rng.choice(["softmax", "softmax_norm", "sigmoid_norm"]), sel_bias=rng.random() < 0.3,
                 scale=rng.choice([1.0, 2.5]), residual=rng.random() < 0.5, given=rng.random() < 0.2,
                 layout=rng.randint(0, 1), layout_down=rng.randint(0, 1), act=rng.choice(["silu", "silu", "gelu_tanh"]))
    elif rng.random() < 0.6:
        unit = BLOCK[t][0]
        c = _lin("", m=_log(rng, 1, 16), n=_log(rng, 100, 20000), kk=unit * max(1, _log(rng, 256, 14336) // unit), t=t,
                 dtype=rng.choice(["f32", "f32", "bf16"]))
    else:
        c = _lin("", m=_log(rng, 17, 2048), n=_log(rng, 100, 14336), kk=256 * rng.randint(1, 16), t=t, dtype="bf16")
    if c["op"] == "linear":
        c.update(bias=rng.random() < 0.7, residual=rng.random() < 0.5, layout=rng.randint(0, 1),
                 act=rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]))
    del c["name"]
    return c


def work(c):
    if c["op"] == "linear":
        b = 2 if c["dtype"] == "bf16" else 4
        return {"bytes": c["n"] * _row_bytes(c["t"], c["kk"]) + b * c["m"] * (c["kk"] + c["n"] * (2 if c["residual"] else 1))
                + 4 * c["n"] * c["bias"], "flops": 2.0 * c["m"] * c["n"] * c["kk"]}
    picks = c["m"] * c["k"] * (0.5 if c["given"] else 1.0)
    seen = c["e"] * (1 - (1 - picks / c["m"] / c["e"]) ** c["m"])  # distinct experts, uniform routing
    one = 2 * c["f"] * _row_bytes(c["t_in"], c["d"]) + c["d"] * _row_bytes(c["t_down"], c["f"])
    route = 0 if c["given"] else 4 * c["e"] * c["d"]
    return {"bytes": seen * one + route + 4 * c["m"] * c["d"] * (3 if c["residual"] else 2),
            "flops": 6.0 * picks * c["d"] * c["f"] + 2.0 * c["m"] * route / 4}


# ---------------------------------------------------------------- inputs
def _half(g, n, lo, hi):
    v = (torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo).to(torch.float16)
    return v.view(torch.uint8).reshape(n, 2)


def _weights(g, t, rows, k, std=0.02):
    """Random GGUF blocks whose weights are about N(0, std)-sized."""
    bw, bb = BLOCK[t]
    n = rows * k // bw
    w = torch.randint(0, 256, (n, bb), generator=g, device="cuda", dtype=torch.uint8)
    if t == Q4_0:
        d = _half(g, n, 0.7 * std / 4.6, 1.3 * std / 4.6)
        d[:, 1] |= w[:, 0] & 0x80  # ggml's Q4_0 scales carry a sign
        w[:, 0:2] = d
    elif t == Q8_0:
        w[:, 0:2] = _half(g, n, 0.7 * std / 74, 1.3 * std / 74)
    elif t == Q6_K:
        w[:, 208:210] = _half(g, n, 0.7 * std / 1360, 1.3 * std / 1360)
    else:
        top = 15 if t == Q4_K else 31
        w[:, 0:2] = _half(g, n, 0.7 * std / (37 * top / 3.3), 1.3 * std / (37 * top / 3.3))
        w[:, 2:4] = _half(g, n, 0.7 * std * 3.3 / 74, 1.3 * std * 3.3 / 74)
    return w.reshape(-1)


def _activations(g, m, k):
    """Normalised hidden states: Gaussian, a few channels far larger than the rest."""
    x = torch.randn(m, k, generator=g, device="cuda")
    big = torch.rand(k, generator=g, device="cuda") < 0.004
    return torch.where(big, 12.0 * x, x)


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    s = {"case": c}
    if c["op"] == "linear":
        dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
        s["w"] = _weights(g, c["t"], c["n"], c["kk"])
        s["x"] = _activations(g, c["m"], c["kk"]).to(dt)
        s["bias"] = torch.randn(c["n"], generator=g, device="cuda") * 0.5 if c["bias"] else None
        s["residual"] = torch.randn(c["m"], c["n"], generator=g, device="cuda").to(dt) if c["residual"] else None
        return s
    e, d, f = c["e"], c["d"], c["f"]
    s["gate"] = _weights(g, c["t_in"], e * f, d)
    s["up"] = _weights(g, c["t_in"], e * f, d)
    s["down"] = _weights(g, c["t_down"], e * d, f)
    s["x"] = _activations(g, c["m"], d)
    s["residual"] = torch.randn(c["m"], d, generator=g, device="cuda") if c["residual"] else None
    if c["given"]:  # picks of a router elsewhere: half of the slots belong to other ranks, one token has none here
        ids = torch.rand(c["m"], e, generator=g, device="cuda").argsort(dim=1)[:, :c["k"]].to(torch.int32)
        away = torch.rand(c["m"], c["k"], generator=g, device="cuda") < 0.5
        away[c["m"] // 2] = True
        s["ids"] = torch.where(away, torch.full_like(ids, -1), ids)
        wts = torch.rand(c["m"], c["k"], generator=g, device="cuda") + 0.1
        s["wts"] = wts / wts.sum(dim=1, keepdim=True)
    else:
        s["router"] = torch.randn(e, d, generator=g, device="cuda") / math.sqrt(d)
        s["sel_bias"] = torch.randn(e, generator=g, device="cuda") * 0.1 if c["sel_bias"] else None
    return s


# ---------------------------------------------------------------- plain forms
def _f16(b):
    return b.contiguous().view(torch.float16).float()


def _k_scales(s):
    """The eight 6-bit scales and mins of a Q4_K / Q5_K super-block, from its 12 bytes."""
    a, b, c = s[:, 0:4].int(), s[:, 4:8].int(), s[:, 8:12].int()
    sc = torch.cat([a & 63, (c & 15) | ((a >> 6) << 4)], 1)
    mn = torch.cat([b & 63, (c >> 4) | ((b >> 6) << 4)], 1)
    return sc.float(), mn.float()


def _dequant(w, t, layout, rows, k):
    """f32 weights [rows, k] of GGUF blocks."""
    b = w.reshape(-1, BLOCK[t][1])
    n = b.shape[0]
    if t == Q8_0:
        return (_f16(b[:, 0:2]) * b[:, 2:].contiguous().view(torch.int8).float()).reshape(rows, k)
    if t == Q4_0:
        q = torch.cat([b[:, 2:] & 15, b[:, 2:] >> 4], 1).float() - 8.0
        return (q * _f16(b[:, 0:2])).reshape(rows, k)
    if t == Q6_K:
        d = _f16(b[:, 208:210])
        if layout == 1:
            lo = torch.stack([b[:, 0:128] & 15, b[:, 0:128] >> 4], 2).reshape(n, 256)
            hi = torch.stack([(b[:, 128:192] >> s) & 3 for s in (0, 2, 4, 6)], 2).reshape(n, 256)
            sc = (b[:, 192:208].float() - 128.0) / 64.0
        else:
            ql, qh = b[:, 0:128].reshape(n, 2, 2, 32), b[:, 128:192].reshape(n, 2, 1, 32)
            lo = torch.cat([ql & 15, ql >> 4], 2).reshape(n, 256)
            hi = torch.cat([(qh >> s) & 3 for s in (0, 2, 4, 6)], 2).reshape(n, 256)
            sc = b[:, 192:208].contiguous().view(torch.int8).float()
        q = (lo | (hi << 4)).float() - 32.0
        return ((d * sc).unsqueeze(2) * q.reshape(n, 16, 16)).reshape(rows, k)
    d, dmin = _f16(b[:, 0:2]), _f16(b[:, 2:4])
    sc, mn = _k_scales(b[:, 4:16])
    qs = b[:, 16:144] if t == Q4_K else b[:, 48:176]
    qs = qs.reshape(n, 4, 1, 32)
    q = torch.cat([qs & 15, qs >> 4], 2).reshape(n, 8, 32)
    if t == Q5_K:
        if layout == 1:
            bits = torch.stack([(b[:, 16:48] >> s) & 1 for s in range(8)], 2).reshape(n, 8, 32)
        else:
            bits = torch.stack([(b[:, 16:48] >> s) & 1 for s in range(8)], 1)
        q = q | (bits << 4)
    return ((d * sc).unsqueeze(2) * q.float() - (dmin * mn).unsqueeze(2)).reshape(rows, k)


def _act(v, act):
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return torch.clamp(v, min=0.0) if act == "relu" else v


def _pick(c, x, router, sel_bias):
    """ids and weights [m, k] of the router's picks; in 64 bits, for scores next to one another."""
    logits = x.double() @ router.double().t()
    s = torch.sigmoid(logits) if c["score"] == "sigmoid_norm" else torch.softmax(logits, dim=1)
    by = s if sel_bias is None else s + sel_bias.double()
    ids = torch.sort(by, dim=1, descending=True, stable=True)[1][:, :c["k"]]
    w = torch.gather(s, 1, ids)
    if c["score"] != "softmax":
        w = w / w.sum(dim=1, keepdim=True)
    return ids, (w * c["scale"])


def _plain_linear(s):
    c = s["case"]
    y = s["x"].float() @ _dequant(s["w"], c["t"], c["layout"], c["n"], c["kk"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    y = _act(y, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_moe(s):
    c = s["case"]
    m, e, k, d, f, x = c["m"], c["e"], c["k"], c["d"], c["f"], s["x"]
    if c["given"]:
        ids, wts = s["ids"].long(), s["wts"]
    else:
        ids, wts = _pick(c, x, s["router"], s["sel_bias"])
        wts = wts.float()
    live = torch.where(ids >= 0, wts, torch.zeros_like(wts))
    at = ids.clamp(min=0)
    if m * k < e:  # fewer picks than experts: the picked experts' matrices alone
        take = at.reshape(-1)
        mats = [w.reshape(e, -1)[take] for w in (s["gate"], s["up"], s["down"])]
        gate = _dequant(mats[0], c["t_in"], c["layout"], m * k * f, d).reshape(m, k, f, d)
        up = _dequant(mats[1], c["t_in"], c["layout"], m * k * f, d).reshape(m, k, f, d)
        h = _act((gate @ x.reshape(m, 1, d, 1)).squeeze(3), c["act"]) * (up @ x.reshape(m, 1, d, 1)).squeeze(3)
        down = _dequant(mats[2], c["t_down"], c["layout_down"], m * k * d, f).reshape(m, k, d, f)
        y = ((down @ h.unsqueeze(3)).squeeze(3) * live.unsqueeze(2)).sum(dim=1)
    else:  # every expert for every token, the others' share zero
        share = torch.zeros(m, e, device=x.device).scatter_add_(1, at, live)
        gate = (x @ _dequant(s["gate"], c["t_in"], c["layout"], e * f, d).t()).reshape(m, e, f)
        up = (x @ _dequant(s["up"], c["t_in"], c["layout"], e * f, d).t()).reshape(m, e, f)
        h = _act(gate, c["act"]) * up * share.unsqueeze(2)
        down = _dequant(s["down"], c["t_down"], c["layout_down"], e * d, f).reshape(e, d, f)
        y = torch.bmm(h.transpose(0, 1), down.transpose(1, 2)).sum(dim=0)
    if s["residual"] is not None:
        y = y + s["residual"]
    return {"y": y} if c["given"] else {"y": y, "ids": ids.to(torch.int32), "weights": wts}


# ---------------------------------------------------------------- the framework's calls
_engine = None


def _own(s):
    """The calls of a user's program, which keeps the engine, the handle of the experts and a workspace."""
    global _engine
    from planejaja_b200.engine import CudaEngine, MoeExperts
    if _engine is None:
        _engine = CudaEngine(0)
    c = s["case"]
    if c["op"] == "linear":
        if "ws" not in s:
            s["ws"] = _engine.linear_workspace(c["m"], c["n"], c["kk"])
        return _engine.linear(s["x"], s["w"], c["t"], c["n"], c["kk"], bias=s["bias"], act=c["act"],
                              residual=s["residual"], q6k_layout=c["layout"], workspace=s["ws"], sync=False)
    if "moe" not in s:
        s["moe"] = MoeExperts(s["gate"], s["up"], s["down"], c["e"], c["d"], c["f"], c["t_in"], c["t_down"],
                              layout_in=c["layout"], layout_down=c["layout_down"], act=c["act"])
        s["ws"] = _engine.moe_workspace(s["moe"], c["m"], c["k"])
    if c["given"]:
        return {"y": _engine.moe_ffn(s["moe"], s["x"], s["ids"], s["wts"], residual=s["residual"], workspace=s["ws"],
                                     sync=False)}
    y, ids, wts = _engine.moe_layer(s["moe"], s["router"], s["x"], c["k"], score=c["score"], sel_bias=s["sel_bias"],
                                    scale=c["scale"], residual=s["residual"], workspace=s["ws"], sync=False)
    return {"y": y, "ids": ids, "weights": wts}


def run(s):
    if own:
        return _own(s)
    return _plain_linear(s) if s["case"]["op"] == "linear" else _plain_moe(s)


# ---------------------------------------------------------------- 64 bits, from the formats' definitions
def _places(t, layout):
    """For each weight i of a block: byte and shift of its low bits, byte and shift of its high bits, number of its scale."""
    low, high, scale = [], [], []
    for i in range(BLOCK[t][0]):
        if t == Q4_0:
            low.append((2 + i % 16, 4 * (i // 16)))
        elif t == Q8_0:
            low.append((2 + i, 0))
        elif t in (Q4_K, Q5_K):
            sub, el = divmod(i, 32)
            low.append(((16 if t == Q4_K else 48) + 32 * (sub // 2) + el, 4 * (sub % 2)))
            high.append((16 + 4 * sub + el // 8, el % 8) if layout else (16 + el, sub))
            scale.append(sub)
        elif layout:
            low.append((i // 2, 4 * (i % 2)))
            high.append((128 + i // 4, 2 * (i % 4)))
            scale.append(i // 16)
        else:
            part, r = divmod(i, 128)
            quarter, el = divmod(r, 32)
            low.append((64 * part + 32 * (quarter % 2) + el, 4 * (quarter // 2)))
            high.append((128 + 32 * part + el, 2 * quarter))
            scale.append(8 * part + 2 * quarter + el // 16)
    return low, high, scale


def _exact_weights(w, t, layout, rows, k):
    b = w.reshape(-1, BLOCK[t][1])
    low, high, scale = _places(t, layout)

    def bits(where, width):
        byte = torch.tensor([p for p, _ in where], device=b.device)
        shift = torch.tensor([s for _, s in where], device=b.device, dtype=torch.uint8)
        return ((b[:, byte] >> shift) & ((1 << width) - 1)).double()

    def half(at):
        return b[:, at:at + 2].contiguous().view(torch.float16).double()

    if t == Q4_0:
        v = (bits(low, 4) - 8) * half(0)
    elif t == Q8_0:
        u = bits(low, 8)
        v = torch.where(u > 127, u - 256, u) * half(0)
    elif t == Q6_K:
        u = b[:, 192:208].double()
        sc = (u - 128) / 64 if layout else torch.where(u > 127, u - 256, u)
        v = half(208) * sc[:, scale] * (bits(low, 4) + 16 * bits(high, 2) - 32)
    else:
        y = b[:, 4:16].long()
        sc = [y[:, j] % 64 if j < 4 else y[:, j + 4] % 16 + y[:, j - 4] // 64 * 16 for j in range(8)]
        mn = [y[:, j + 4] % 64 if j < 4 else y[:, j + 4] // 16 + y[:, j] // 64 * 16 for j in range(8)]
        q = bits(low, 4) + (16 * bits(high, 1) if t == Q5_K else 0)
        v = half(0) * torch.stack(sc, 1).double()[:, scale] * q - half(2) * torch.stack(mn, 1).double()[:, scale]
    return v.reshape(rows, k)


def _exact_act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3))
    return torch.relu(v) if act == "relu" else v


def exact(c, seed):
    s = prepare(c, seed)
    x = s["x"].double()
    if c["op"] == "linear":
        rows = []
        for r in range(0, c["n"], 4096):
            n = min(4096, c["n"] - r)
            rb = _row_bytes(c["t"], c["kk"])
            rows.append(x @ _exact_weights(s["w"][r * rb:(r + n) * rb], c["t"], c["layout"], n, c["kk"]).t())
        y = torch.cat(rows, 1)
        y = _exact_act(y if s["bias"] is None else y + s["bias"].double(), c["act"])
        return y if s["residual"] is None else y + s["residual"].double()
    e, d, f = c["e"], c["d"], c["f"]
    if c["given"]:
        ids, wts = s["ids"].long(), s["wts"].double()
    else:
        logits = (x[:, None, :] * s["router"].double()[None]).sum(2)
        if c["score"] == "sigmoid_norm":
            p = 1 / (1 + torch.exp(-logits))
        else:
            p = torch.exp(logits - logits.amax(1, keepdim=True))
            p = p / p.sum(1, keepdim=True)
        by = (p if s["sel_bias"] is None else p + s["sel_bias"].double()).cpu()
        ids = torch.tensor([sorted(range(e), key=lambda i, row=row: (-row[i], i))[:c["k"]] for row in by.tolist()],
                           device=x.device)
        wts = p.gather(1, ids)
        if c["score"] != "softmax":
            wts = wts / wts.sum(1, keepdim=True)
        wts = wts * c["scale"]
    y = torch.zeros_like(x) if s["residual"] is None else s["residual"].double()
    gate, up, down = (s[n].reshape(e, -1) for n in ("gate", "up", "down"))
    for j in sorted(set(ids[ids >= 0].tolist())):
        tok, slot = torch.nonzero(ids == j, as_tuple=True)
        h = _exact_act(x[tok] @ _exact_weights(gate[j], c["t_in"], c["layout"], f, d).t(), c["act"])
        h = h * (x[tok] @ _exact_weights(up[j], c["t_in"], c["layout"], f, d).t())
        out = h @ _exact_weights(down[j], c["t_down"], c["layout_down"], d, f).t()
        y = y.index_add(0, tok, out * wts[tok, slot][:, None])
    return {"y": y} if c["given"] else {"y": y, "ids": ids.to(torch.int32), "weights": wts}
