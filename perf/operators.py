"""The embedding encoder's operators as measured: 8-bit products, block norms and cross attention.

Each case is one call a serving program makes of ``rag_service_amd.ops``. The sizes are those of the query encoder that
``tools/bench_e2e.py`` runs (hidden 1024, 16 heads of 64, feed-forward 4096, batches of 32, up to 512 tokens) and generic
ones around them: single rows, odd sizes, long states, grouped heads.

``own`` False: the operators in their plain form, elementary torch operations in 32 bits, rounded once at the end.
``own`` True: the framework's calls.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}


# ---- the cases ------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token through the second feed-forward product: what a single short request waits for
        {"name": "linear one token", "op": "linear", "m": 1, "k": 4096, "n": 1024, "type": "bf16", "out": "bf16",
         "act": "none", "bias": True},
        # a served batch of 32 questions, 19 tokens each on average, through the first feed-forward product and its GELU
        {"name": "linear query batch gelu", "op": "linear", "m": 613, "k": 1024, "n": 4096, "type": "bf16", "out": "bf16",
         "act": "gelu", "bias": True},
        # rows already in 8 bits, sizes that fit no tile, exact scales wanted in fp32
        {"name": "linear odd 8-bit rows", "op": "linear", "m": 1031, "k": 1000, "n": 777, "type": "int8", "out": "fp32",
         "act": "none", "bias": False},
        # 32 passages of 512 tokens through the second feed-forward product: building a corpus
        {"name": "linear passages", "op": "linear", "m": 16384, "k": 4096, "n": 1024, "type": "bf16", "out": "bf16",
         "act": "none", "bias": True},
        # one token after its attention block
        {"name": "norm one token", "op": "norm", "rows": 1, "cols": 1024, "type": "bf16", "post": "none",
         "next": "layer", "gate_rows": 0, "residual_scale": 1.0, "stream": False, "rows8": False},
        # a served batch of questions: add, norm, and the 8-bit rows that the next product takes
        {"name": "norm query batch to 8 bits", "op": "norm", "rows": 613, "cols": 1024, "type": "bf16", "post": "none",
         "next": "layer", "gate_rows": 0, "residual_scale": 1.0, "stream": False, "rows8": True},
        # norms on both sides of the block, a gate row for each sequence, a width that fits no vector
        {"name": "norm both sides odd fp32", "op": "norm", "rows": 4097, "cols": 1001, "type": "fp32", "post": "rms",
         "next": "rms", "gate_rows": 17, "residual_scale": 0.5, "stream": True, "rows8": False},
        # a wide encoder over a corpus chunk, both norms, one gate for all rows
        {"name": "norm both sides wide", "op": "norm", "rows": 32768, "cols": 4096, "type": "bf16", "post": "rms",
         "next": "layer", "gate_rows": 1, "residual_scale": 1.0, "stream": True, "rows8": False},
        # one new token of each of 32 sequences against its encoder's states
        {"name": "attention one token", "op": "attention", "b": 32, "lq": 1, "lk": 512, "lo": 40, "h": 16, "hkv": 16, "d": 64,
         "type": "fp16", "form": "lengths"},
        # a served batch of questions, packed, in the encoder's own fp32
        {"name": "attention query batch packed", "op": "attention", "b": 32, "lq": 41, "lk": 40, "lo": 8, "h": 16,
         "hkv": 16, "d": 64, "type": "fp32", "form": "packed"},
        # 32 passages of up to 512 tokens with a padding mask
        {"name": "attention passages masked", "op": "attention", "b": 32, "lq": 512, "lk": 512, "lo": 100, "h": 16, "hkv": 16,
         "d": 64, "type": "bf16", "form": "mask"},
        # one new token each for 4 sequences over very long states, grouped heads of 128
        {"name": "attention one token long", "op": "attention", "b": 4, "lq": 1, "lk": 65536, "lo": 65536, "h": 32, "hkv": 8,
         "d": 128, "type": "bf16", "form": "lengths"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size spread over the logarithm; every other one on a boundary of 64, the rest as they fall."""
    v = _log(rng, lo, hi)
    return max(64, v // 64 * 64) if rng.random() < 0.5 and v >= 64 else v


def draw(rng):
    op = rng.choice(["linear", "norm", "attention"])
    if op == "linear":
        k, n = _size(rng, 48, 4096), _size(rng, 48, 4096)
        m = min(_log(rng, 1, 16384), 16384 * 4096 * 1024 // (k * n))
        kind = rng.choice(["bf16", "fp16", "fp32", "int8"])
        return {"op": op, "m": m, "k": k, "n": n, "type": kind, "out": rng.choice(["bf16", "fp16", "fp32"]),
                "act": rng.choice(["none", "gelu"]), "bias": rng.random() < 0.7}
    if op == "norm":
        cols = _size(rng, 48, 8192)
        rows = min(_log(rng, 1, 32768), 32768 * 4096 // cols)
        kind = rng.choice(["bf16", "fp16", "fp32"])
        nxt = rng.choice(["none", "layer", "rms"])
        return {"op": op, "rows": rows if kind != "fp32" else max(1, rows // 2), "cols": cols, "type": kind,
                "post": rng.choice(["none", "layer", "rms"]), "next": nxt, "gate_rows": rng.choice([0, 1, 7]),
                "residual_scale": rng.choice([1.0, 0.5]), "stream": nxt == "none" or rng.random() < 0.5,
                "rows8": nxt != "none" and kind != "fp32" and rng.random() < 0.5}
    d = rng.choice([32, 64, 80, 128])
    hkv = rng.choice([1, 2, 4, 8, 16])
    h = hkv * rng.choice([1, 2, 4]) if hkv < 16 else 16
    b = _log(rng, 1, 64)
    lk = _log(rng, 1, 16384)
    lq = 1 if rng.random() < 0.4 else _log(rng, 2, 1024)
    most = 32 * 512 * 512 * 16 * 64                                  # the masked passages' products
    lk = max(1, min(lk, 4 * 65536 * 8 * 128 // (b * hkv * d)))        # the long states' bytes
    lq = max(1, min(lq, most // (b * lk * h * d)))
    lo = _log(rng, 1, lk)
    form = rng.choice(["lengths", "packed", "mask"])
    return {"op": op, "b": b, "lq": lq, "lk": lk, "lo": lo, "h": h, "hkv": hkv, "d": d,
            "type": rng.choice(["bf16", "fp16", "fp32"]), "form": form}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _spread(lo, hi, b):
    """b lengths from lo to hi, evenly spread (the same for every seed, in another order)."""
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


def _activations(g, rows, cols):
    """Hidden states as an encoder holds them: a scale per row and a few channels that are far larger than the rest."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= 0.5 + torch.rand(rows, 1, generator=g, device="cuda")
    big = torch.rand(cols, generator=g, device="cuda") < 0.005
    return torch.where(big, x * 8, x)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s = {"case": case, "x_scale": None}
        if case["type"] == "int8":
            s["x"] = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
            s["x_scale"] = 0.01 + 0.05 * torch.rand(m, generator=g, device="cuda")
        else:
            s["x"] = _activations(g, m, k).to(_TYPES[case["type"]])
        w = normal(n, k).mul_(32).round_().clamp_(-127, 127)
        s["w"] = w.to(torch.int8)
        s["w_scale"] = (0.5 + torch.rand(n, generator=g, device="cuda")) / (32 * math.sqrt(k))
        s["bias"] = normal(n) * 0.1 if case["bias"] else None
        return s
    if case["op"] == "norm":
        rows, cols, t = case["rows"], case["cols"], _TYPES[case["type"]]
        s = {"case": case, "y": normal(rows, cols).to(t), "x": _activations(g, rows, cols).to(t), "gate": None}
        if case["gate_rows"]:
            s["gate"] = (0.3 * normal(min(rows, case["gate_rows"]), cols)).to(t)
        for which in ("post", "next"):
            s[which + "_weight"] = (1 + 0.1 * normal(cols)).to(t) if case[which] != "none" else None
            s[which + "_bias"] = (0.1 * normal(cols)).to(t) if case[which] == "layer" else None
        return s
    b, lq, lk, h, hkv, d, t = (case[x] for x in ("b", "lq", "lk", "h", "hkv", "d", "type"))
    t = _TYPES[t]
    perm = torch.randperm(b, generator=g, device="cuda")
    lens = torch.tensor(_spread(case["lo"], lk, b), dtype=torch.int32, device="cuda")[perm]
    s = {"case": case}
    if case["form"] == "packed":
        qlens = torch.tensor(_spread(max(1, min(case["lo"] + 1, lq)), lq, b), dtype=torch.int32, device="cuda")[perm]
        zero = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["q_offsets"] = torch.cat([zero, qlens.cumsum(0, dtype=torch.int32)])
        s["k_offsets"] = torch.cat([zero, lens.cumsum(0, dtype=torch.int32)])
        tq, tk = sum(_spread(max(1, min(case["lo"] + 1, lq)), lq, b)), sum(_spread(case["lo"], lk, b))
        s["q"] = (1.5 * normal(tq, h, d)).to(t)
        s["k"], s["v"] = normal(tk, hkv, d).to(t), normal(tk, hkv, d).to(t)
    else:
        s["q"] = (1.5 * normal(b, lq, h, d)).to(t)
        s["k"], s["v"] = normal(b, lk, hkv, d).to(t), normal(b, lk, hkv, d).to(t)
        if case["form"] == "mask":
            s["mask"] = torch.arange(lk, device="cuda") < lens[:, None]
        else:
            s["lengths"] = lens
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------

def _rows8(x):
    """8-bit values (as floats) and scales of fp32 rows."""
    s = x.abs().amax(dim=1, keepdim=True) / 127
    q = torch.clamp(torch.round(x / torch.where(s > 0, s, 1)), -127, 127)
    return q, s


def _plain_linear(s):
    case = s["case"]
    if s["x_scale"] is None:
        q, sx = _rows8(s["x"].float())
    else:
        q, sx = s["x"].float(), s["x_scale"][:, None]
    y = (q @ s["w"].float().t()) * (sx * s["w_scale"])
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y.to(_TYPES[case["out"]])


def _plain_one_norm(v, kind, w, b):
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + 1e-5) * w.float()
    return v if b is None else v + b.float()


def _plain_norm(s):
    case = s["case"]
    t = _TYPES[case["type"]]
    u = s["y"].float()
    if case["post"] != "none":
        u = _plain_one_norm(u, case["post"], s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        per = -(-case["rows"] // s["gate"].shape[0])
        u = u * s["gate"].float().repeat_interleave(per, dim=0)[: case["rows"]]
    h = s["x"].float() * case["residual_scale"] + u
    out = {}
    if case["stream"]:
        out["stream"] = h.to(t)
    if case["next"] != "none":
        o = _plain_one_norm(h, case["next"], s["next_weight"], s["next_bias"])
        out["normed"] = o.to(t)
        if case["rows8"]:
            q, sc = _rows8(o)
            out["rows8"] = (q * sc).to(t)
    return out


def _padded(x, offsets, length):
    """Packed rows as (b, length, ...) with the rows that are there marked."""
    at = offsets[:-1, None].long() + torch.arange(length, device=x.device)
    there = at < offsets[1:, None]
    return x[at.clamp_(max=x.shape[0] - 1)], there


def _plain_attention(s):
    case = s["case"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, h, hkv, d, lk = case["b"], case["h"], case["hkv"], case["d"], case["lk"]
    if case["form"] == "packed":
        q, q_there = _padded(q, s["q_offsets"], case["lq"])
        k, there = _padded(k, s["k_offsets"], lk)
        v, _ = _padded(v, s["k_offsets"], lk)
    elif case["form"] == "mask":
        there = s["mask"]
    else:
        there = torch.arange(lk, device=q.device) < s["lengths"][:, None]
    lq, group = q.shape[1], h // hkv
    q = q.reshape(b, lq, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * lq, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * (1 / math.sqrt(d))
    x = x.masked_fill_(~there[:, None, None, :], float("-inf"))
    x = torch.exp(x - x.amax(dim=-1, keepdim=True))
    x = x / x.sum(dim=-1, keepdim=True)
    o = torch.matmul(x, v.permute(0, 2, 1, 3).contiguous())
    o = o.reshape(b, hkv, group, lq, d).permute(0, 3, 1, 2, 4).reshape(b, lq, h, d)
    if case["form"] == "packed":
        at = torch.arange(s["q"].shape[0], device=q.device)
        which = torch.searchsorted(s["q_offsets"][1:].long(), at, right=True)
        o = o[which, at - s["q_offsets"].long()[which]]
    return o.to(s["q"].dtype)


def _ops():
    at = os.path.join(os.getcwd(), "rag-serving-system_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from rag_service_amd import ops
    return ops


def _own_linear(s):
    case = s["case"]
    return _ops().linear_int8(s["x"], s["w"], s["w_scale"], x_scale=s["x_scale"], bias=s["bias"], act=case["act"],
                              out_dtype=_TYPES[case["out"]])


def _own_norm(s):
    case = s["case"]
    per = -(-case["rows"] // s["gate"].shape[0]) if s["gate"] is not None else 1
    r = _ops().block_norm(s["y"], s["x"], residual_scale=case["residual_scale"], gate=s["gate"], rows_per_gate=per,
                          post_norm=case["post"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                          next_norm=case["next"], next_weight=s["next_weight"], next_bias=s["next_bias"], eps=1e-5,
                          stream=case["stream"], rows8=case["rows8"])
    out = {}
    if case["stream"]:
        out["stream"] = r.stream
    if case["next"] != "none":
        out["normed"] = r.normed
        if case["rows8"]:
            out["rows8"] = torch.mul(r.rows8, r.scale[:, None], out=torch.empty_like(r.normed))
    return out


def _own_attention(s):
    case = s["case"]
    if case["form"] == "packed":
        return _ops().cross_attention(s["q"], s["k"], s["v"], q_offsets=s["q_offsets"], k_offsets=s["k_offsets"],
                                      max_q=case["lq"], max_k=case["lk"])
    if case["form"] == "mask":
        return _ops().cross_attention(s["q"], s["k"], s["v"], key_mask=s["mask"])
    return _ops().cross_attention(s["q"], s["k"], s["v"], key_lengths=s["lengths"])


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_linear(state) if op == "linear" else _own_norm(state) if op == "norm" else _own_attention(state)
    return _plain_linear(state) if op == "linear" else _plain_norm(state) if op == "norm" else _plain_attention(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * _BYTES[case["type"]] + n * k + m * n * _BYTES[case["out"]] + 4 * n
                + (4 * n if case["bias"] else 0) + (4 * m if case["type"] == "int8" else 0), "flops": 2 * m * n * k}
    if case["op"] == "norm":
        rows, cols, e = case["rows"], case["cols"], _BYTES[case["type"]]
        vectors = min(rows, case["gate_rows"]) + sum({"none": 0, "rms": 1, "layer": 2}[case[x]] for x in ("post", "next"))
        wrote = e * (case["stream"] + (case["next"] != "none")) + case["rows8"]
        return {"bytes": rows * cols * (2 * e + wrote) + vectors * cols * e + 4 * rows * case["rows8"],
                "flops": rows * cols * (4 + 6 * (case["post"] != "none") + 6 * (case["next"] != "none"))}
    b, lq, lk, h, hkv, d, e = case["b"], case["lq"], case["lk"], case["h"], case["hkv"], case["d"], _BYTES[case["type"]]
    ks = _spread(case["lo"], lk, b)
    qs = _spread(max(1, min(case["lo"] + 1, lq)), lq, b) if case["form"] == "packed" else [lq] * b
    extra = {"lengths": 4 * b, "packed": 8 * (b + 1), "mask": b * lk}[case["form"]]
    return {"bytes": e * d * (2 * h * sum(qs) + 2 * hkv * sum(ks)) + extra,
            "flops": 4 * h * d * sum(x * y for x, y in zip(qs, ks))}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------

def _exact_quantised(x):
    """round-half-even of the fp32 quotient x / s, s = the fp32 scale max|x| / 127: both quotients are rounded to 32 bits
    by the operator's definition."""
    scale = (x.abs().max(dim=1).values / 127.0).float().double()
    safe = scale.clone()
    safe[safe == 0] = 1.0
    return (x / safe.unsqueeze(1)).float().double().round().clamp(-127.0, 127.0), scale


def _exact_normalised(v, kind, w, b):
    n = v.shape[1]
    centre = v.sum(1, keepdim=True) / n if kind == "layer" else torch.zeros_like(v[:, :1])
    c = v - centre
    out = c / (c.pow(2).sum(1, keepdim=True) / n + 1e-5).sqrt() * w.double()
    return out + b.double() if b is not None else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        if case["type"] == "int8":
            q, sx = s["x"].double(), s["x_scale"].double()
        else:
            q, sx = _exact_quantised(s["x"].double())
        y = torch.mm(q, s["w"].double().t()).mul_(sx.unsqueeze(1)).mul_(s["w_scale"].double())
        if case["bias"]:
            y += s["bias"].double()
        if case["act"] == "gelu":
            y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2.0))
        return y
    if case["op"] == "norm":
        u = s["y"].double()
        if case["post"] != "none":
            u = _exact_normalised(u, case["post"], s["post_weight"], s["post_bias"])
        if s["gate"] is not None:
            per = -(-case["rows"] // s["gate"].shape[0])
            row = torch.arange(case["rows"], device="cuda") // per
            u = u * s["gate"].double()[row]
        h = u + case["residual_scale"] * s["x"].double()
        out = {}
        if case["stream"]:
            out["stream"] = h
        if case["next"] != "none":
            out["normed"] = _exact_normalised(h, case["next"], s["next_weight"], s["next_bias"])
            if case["rows8"]:
                q, sc = _exact_quantised(out["normed"])
                out["rows8"] = q * sc.unsqueeze(1)
        return out
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["h"] // case["hkv"]
    for i in range(case["b"]):
        if case["form"] == "packed":
            (q0, q1), (k0, k1) = s["q_offsets"][i:i + 2].tolist(), s["k_offsets"][i:i + 2].tolist()
            q, k, v, to = s["q"][q0:q1], s["k"][k0:k1], s["v"][k0:k1], out[q0:q1]
        else:
            n = int(s["mask"][i].sum()) if case["form"] == "mask" else int(s["lengths"][i])
            q, k, v, to = s["q"][i], s["k"][i, :n], s["v"][i, :n], out[i]
        for j in range(case["hkv"]):
            kj, vj = k[:, j].double(), v[:, j].double()
            heads = q[:, j * group:(j + 1) * group].double()
            p = torch.softmax(heads.reshape(-1, case["d"]).mm(kj.t()) * case["d"] ** -0.5, dim=1)
            to[:, j * group:(j + 1) * group] = p.mm(vj).reshape(heads.shape)
    return out
