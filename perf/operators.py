"""Performance cases of the products whose weights every row picks for itself: the expert layer of a
mixture-of-experts model with its router, and low-rank adapters beside shared projections.

An engine keeps the router, the layer and the adapter sets of a model resident (`Backend.router`, `Backend.moe`,
`Backend.adapters`) and calls them once per layer and batch: `route` picks every token's experts and weights, `run_moe`
runs the chosen experts, `apply_adapters` adds the rows' adapters to what the shared projections left in the outputs.

`listed()` holds the cases, `draw()` makes more of the same ranges, `prepare()` builds what a program has in hand before
the call, `run()` is one pass (with `own` through the public entry points, otherwise in plain torch operations), `exact()`
what that pass returns, in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

_BLOCK = {"Q4_0": (32, 18), "Q8_0": (32, 34), "Q4_K": (256, 144), "Q5_K": (256, 176), "Q6_K": (256, 210), "MXFP4": (32, 17)}
_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "f16": torch.float16}
_SIZE = {"bf16": 2, "f32": 4, "f16": 2}
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]
_ALPHA, _LIMIT = 1.702, 7.0        # of the clamped gate


def listed():
    return [
        # The smallest call: one token's choice among 128 experts.  Launch and call overhead count.
        {"name": "route_m1", "kind": "route", "m": 1, "experts": 128, "top_k": 8, "hidden": 2048, "x": "bf16", "w": "f32", "scoring": "softmax"},
        # Reading a prompt in pieces of 512 tokens: the choice among 256 experts by sigmoid scores with a balancing bias.
        {"name": "route_m512", "kind": "route", "m": 512, "experts": 256, "top_k": 8, "hidden": 5120, "x": "bf16", "w": "f32", "scoring": "sigmoid"},
        # One sequence decoding: eight small experts of 128, Q4_K with a Q6_K down projection.
        {"name": "moe_q4km_m1", "kind": "moe", "m": 1, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 768, "type": "Q4_K", "type_down": "Q6_K",
         "x": "bf16", "y": "bf16", "act": "swiglu"},
        # Verifying a draft of three tokens, fp32 activations and results.
        {"name": "moe_q5k_m4", "kind": "moe", "m": 4, "experts": 64, "top_k": 6, "hidden": 4096, "inter": 1536, "type": "Q5_K", "type_down": "Q5_K",
         "x": "f32", "y": "f32", "act": "swiglu"},
        # A few sequences decoding together: router and experts of one layer, one call after the other.
        {"name": "layer_q4km_m8", "kind": "layer", "m": 8, "experts": 128, "top_k": 8, "hidden": 2048, "inter": 768, "type": "Q4_K", "type_down": "Q6_K",
         "x": "bf16", "y": "bf16", "act": "swiglu", "w": "f32", "scoring": "softmax"},
        # Sixteen sequences, experts of odd width in MXFP4 with biases and the clamped gate.
        {"name": "moe_mxfp4_m16", "kind": "moe", "m": 16, "experts": 32, "top_k": 4, "hidden": 2816, "inter": 1440, "type": "MXFP4", "type_down": "MXFP4",
         "x": "bf16", "y": "f32", "act": "clamped"},
        # Sixteen sequences over eight large experts: every one of them is read.
        {"name": "moe_large_q4km_m16", "kind": "moe", "m": 16, "experts": 8, "top_k": 2, "hidden": 4096, "inter": 14336, "type": "Q4_K", "type_down": "Q6_K",
         "x": "bf16", "y": "bf16", "act": "swiglu"},
        # The last piece of a prompt beside decoding sequences: every expert has several tokens.
        {"name": "moe_q8_0_m96", "kind": "moe", "m": 96, "experts": 64, "top_k": 6, "hidden": 2048, "inter": 1408, "type": "Q8_0", "type_down": "Q8_0",
         "x": "bf16", "y": "bf16", "act": "swiglu"},
        # One adapted sequence decoding: the output projection's adapter.
        {"name": "lora_m1", "kind": "lora", "m": 1, "k": 4096, "n": "4096", "ranks": "16", "adapters": 1, "dtype": "bf16", "x": "bf16", "y": "bf16", "rows": "any"},
        # Forty-eight sequences with adapters of their own among 64, some with none: query, key and value projections.
        {"name": "lora_qkv_m48", "kind": "lora", "m": 48, "k": 4096, "n": "4096,1024,1024", "ranks": "8,16,32,64", "adapters": 64, "dtype": "bf16",
         "x": "bf16", "y": "bf16", "rows": "any"},
        # The last, partial pieces of five prompts against a matrix of odd height, fp32 throughout, adapters in fp16.
        {"name": "lora_f32_m333", "kind": "lora", "m": 333, "k": 3328, "n": "11003", "ranks": "24", "adapters": 5, "dtype": "f16", "x": "f32", "y": "f32",
         "rows": "runs"},
        # The largest: 4096 tokens of three prompts beside the gate and up projections of a 32B-class layer.
        {"name": "lora_gate_up_m4096", "kind": "lora", "m": 4096, "k": 5120, "n": "25600,25600", "ranks": "16,32", "adapters": 3, "dtype": "bf16",
         "x": "bf16", "y": "bf16", "rows": "runs"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    """A case of the same ranges: any kind, type and row count, sizes spread over their logarithm, odd ones among them."""
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["route"] * 2 + ["moe"] * 5 + ["layer"] * 2 + ["lora"] * 4)
        case = {"kind": kind, "x": rng.choice(["bf16", "bf16", "f32"])}
        if kind == "lora":
            m = rng.choice([lambda: rng.randint(1, 16), lambda: _log(rng, 17, 256), lambda: _log(rng, 257, 4096)])()
            sets = rng.choice([1, 1, 2, 3])
            k = _log(rng, 512, 16384)
            k = k if rng.random() < 0.3 else max(256, k // 64 * 64)
            ns = [_log(rng, 256, 28672) for _ in range(sets)]
            ns = [n if rng.random() < 0.3 else max(64, n // 64 * 64) for n in ns]
            adapters = rng.choice([1, 2, 5, 16, 64]) if m <= 256 else rng.randint(1, 6)
            ranks = rng.sample([4, 8, 16, 24, 32, 64, 128], rng.randint(1, 3))
            case.update(m=m, k=k, n=",".join(map(str, ns)), ranks=",".join(map(str, ranks)), adapters=adapters, dtype=rng.choice(["bf16", "bf16", "f16"]),
                        y=rng.choice(["bf16", "f32"]), rows=rng.choice(["any", "runs"]) if m <= 256 else "runs")
        else:
            experts, top_k = rng.choice([(8, 2), (16, 2), (32, 4), (60, 4), (64, 6), (64, 8), (128, 8), (160, 6), (256, 8)])
            case.update(experts=experts, top_k=top_k)
            if kind == "route":
                case.update(m=_log(rng, 1, 512), hidden=_log(rng, 512, 8192))
            else:
                case["m"] = rng.choice([lambda: rng.randint(1, 4), lambda: rng.randint(5, 32), lambda: _log(rng, 33, 256)])()
                t = rng.choice(["Q4_K"] * 3 + ["Q6_K"] + ["Q8_0"] * 2 + ["Q5_K", "Q4_0", "MXFP4"])
                td = rng.choice(["Q6_K", t, t]) if t in ("Q4_K", "Q5_K") else t
                block = max(_BLOCK[t][0], _BLOCK[td][0])
                case.update(type=t, type_down=td, hidden=max(512, _log(rng, 768, 6144) // block * block), inter=max(256, _log(rng, 384, 8192) // block * block),
                            y=rng.choice(["bf16", "bf16", "f32"]), act=rng.choice(["swiglu", "swiglu", "clamped"]))
                if experts * 3 * case["hidden"] * case["inter"] > 2.5e9:      # what a card holds next to its unpacked copy in the plain form
                    continue
            if kind != "moe":
                case.update(w=rng.choice(["f32", "f32", "bf16"]), scoring=rng.choice(["softmax", "sigmoid"]))
        if _cost(case) <= limit:
            return case


# ---- what a program has in hand -----------------------------------------------------------------

_BACKEND = None


def _backend():
    """One backend per process, as in an engine."""
    global _BACKEND
    if _BACKEND is None:
        import magnitude_b200 as mb

        _BACKEND = mb.Backend(0)
    return _BACKEND


def _acts(gen, m, k, dtype):
    """N(0, 1) activations with one channel in a hundred twenty times larger, as hidden states have them."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    big = torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 100)]
    x[:, big] *= 20.0
    return x.to(_DTYPES[dtype])


def _bytes_of(v):
    return v.contiguous().view(torch.uint8)


def _packed(gen, t, experts, n, k):
    """Blocks of [experts][n] rows as a quantizer leaves them: levels of normal weights, scales that vary by a factor of two
    around a deviation of 1 / sqrt(k).  uint8 [experts, n, bytes of a row]."""
    elems, size = _BLOCK[t]
    blocks = experts * n * (k // elems)
    dev = "cuda"
    sigma = k ** -0.5
    uniform = lambda shape, lo, hi: torch.rand(shape, generator=gen, device=dev) * (hi - lo) + lo  # noqa: E731
    ints = lambda shape, lo, hi: torch.randint(lo, hi, shape, generator=gen, device=dev, dtype=torch.uint8)  # noqa: E731
    out = torch.empty((blocks, size), dtype=torch.uint8, device=dev)

    def levels(shape, spread, top):       # normal levels in 0 .. top
        v = torch.randn(shape, generator=gen, device=dev, dtype=torch.float16).mul_(spread).add_((top + 1) / 2)
        return v.round_().clamp_(0, top).to(torch.uint8)

    if t == "Q8_0":
        out[:, :2] = _bytes_of((uniform((blocks, 1), 0.7, 1.4) * sigma / 42).half())
        out[:, 2:] = _bytes_of((levels((blocks, 32), 42.0, 255).to(torch.int16) - 128).to(torch.int8))
    elif t == "Q4_0":
        out[:, :2] = _bytes_of((uniform((blocks, 1), 0.7, 1.4) * sigma / 2.8).half())
        q = levels((blocks, 32), 2.8, 15)
        out[:, 2:] = q[:, :16] | q[:, 16:] << 4
    elif t == "MXFP4":
        out[:, 0] = 127 + int(np.floor(np.log2(sigma / 1.7))) + ints((blocks,), 0, 2)
        q = ints((blocks, 32), 0, 16)
        out[:, 1:] = q[:, :16] | q[:, 16:] << 4
    elif t in ("Q4_K", "Q5_K"):
        bits, spread = (4, 2.8) if t == "Q4_K" else (5, 5.6)
        middle = 7.5 if bits == 4 else 15.5
        scale = ints((blocks, 8), 30, 62)
        least = (scale.to(torch.int16) + torch.randint(-4, 3, (blocks, 8), generator=gen, device=dev, dtype=torch.int16)).clamp_(0, 63).to(torch.uint8)
        d = uniform((blocks, 1), 0.7, 1.4) * sigma / spread / 45
        out[:, 0:2] = _bytes_of(d.half())
        out[:, 2:4] = _bytes_of((d * middle).half())
        out[:, 4:8] = scale[:, :4] | scale[:, 4:] >> 4 << 6
        out[:, 8:12] = least[:, :4] | least[:, 4:] >> 4 << 6
        out[:, 12:16] = scale[:, 4:] & 15 | least[:, 4:] << 4
        q = levels((blocks, 8, 32), spread, 2 ** bits - 1)
        low = q & 15
        out[:, size - 128:] = (low[:, 0::2] | low[:, 1::2] << 4).reshape(blocks, 128)
        if t == "Q5_K":
            high = q >> 4
            out[:, 16:48] = (high << torch.arange(8, device=dev, dtype=torch.uint8)[None, :, None]).sum(dim=1, dtype=torch.uint8)
    else:   # Q6_K: two halves of 128 weights, each four runs of 32
        q = levels((blocks, 2, 4, 32), 11.0, 63)
        low, high = q & 15, q >> 4
        out[:, :128] = torch.cat([low[:, :, :2].reshape(blocks, 2, 64) | low[:, :, 2:].reshape(blocks, 2, 64) << 4], dim=2).reshape(blocks, 128)
        out[:, 128:192] = (high[:, :, 0] | high[:, :, 1] << 2 | high[:, :, 2] << 4 | high[:, :, 3] << 6).reshape(blocks, 64)
        out[:, 192:208] = _bytes_of(ints((blocks, 16), 60, 120).to(torch.int8))
        out[:, 208:] = _bytes_of((uniform((blocks, 1), 0.7, 1.4) * sigma / 11 / 90).half())
    return out.reshape(experts, n, k // elems * size)


def _router_parts(gen, c):
    e, k = c["experts"], c["hidden"]
    w = (torch.randn((e, k), generator=gen, device="cuda") * k ** -0.5).to(_DTYPES[c["w"]])
    bias = torch.randn(e, generator=gen, device="cuda") * 0.05 if c["scoring"] == "sigmoid" else None
    return {"router": w, "bias": bias}


def _expert_parts(gen, c):
    e, h, i = c["experts"], c["hidden"], c["inter"]
    p = {"gate": _packed(gen, c["type"], e, i, h), "up": _packed(gen, c["type"], e, i, h), "down": _packed(gen, c["type_down"], e, h, i)}
    if c["act"] == "clamped":
        p.update({b: torch.randn((e, n), generator=gen, device="cuda") * 0.1 for b, n in (("gate_bias", i), ("up_bias", i), ("down_bias", h))})
    return p


def _choice(gen, c):
    """Every token's experts, some experts being favoured, and their weights."""
    logits = torch.randn((c["m"], c["experts"]), generator=gen, device="cuda") + 0.7 * torch.randn(c["experts"], generator=gen, device="cuda")
    best, ids = logits.topk(c["top_k"], dim=1)
    return ids.to(torch.int32), torch.softmax(best, dim=1)


def _adapter_parts(gen, c):
    """Per projection A [adapters, largest rank, k] and B [adapters, largest rank, n] (rows beyond an adapter's rank are zero), and its scales."""
    ranks = [int(r) for r in c["ranks"].split(",")]
    rank = torch.tensor([ranks[i % len(ranks)] for i in range(c["adapters"])])
    top = max(ranks[: c["adapters"]])
    have = (torch.arange(top)[None, :] < rank[:, None]).cuda()[:, :, None]
    sets = []
    for n in (int(v) for v in c["n"].split(",")):
        a = torch.randn((c["adapters"], top, c["k"]), generator=gen, device="cuda") * c["k"] ** -0.5 * have
        b = torch.randn((c["adapters"], top, n), generator=gen, device="cuda") * 0.2 * have
        scale = torch.rand(c["adapters"], generator=gen, device="cuda") + 0.5
        sets.append({"a": a.to(_DTYPES[c["dtype"]]), "b": b.to(_DTYPES[c["dtype"]]), "scale": scale, "n": n})
    return rank.tolist(), sets


def _adapter_rows(gen, c):
    """Every row's adapter, -1 where it has none: rows of many sequences in any order, or whole prompts one after the other."""
    if c["rows"] == "any":
        pick = torch.randint(0, c["adapters"], (c["m"],), generator=gen, device="cuda")
        pick = torch.where(torch.rand(c["m"], generator=gen, device="cuda") < (0.1 if c["m"] > 4 else 0.0), -1, pick)
    else:
        ends = torch.sort(torch.randint(1, c["m"] + 1, (c["adapters"],), generator=gen, device="cuda")).values
        pick = torch.searchsorted(ends, torch.arange(c["m"], device="cuda"), right=True)
        pick = torch.where(pick < c["adapters"], pick, -1)
    return pick.to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c = dict(case)
    m, kind = c["m"], c["kind"]
    s = {"case": c}
    if kind == "lora":
        ranks, sets = _adapter_parts(gen, c)
        s.update(rows=_adapter_rows(gen, c), x=_acts(gen, m, c["k"], c["x"]))
        s["y"] = [torch.randn((m, p["n"]), generator=gen, device="cuda").to(_DTYPES[c["y"]]) for p in sets]
        if own:
            be = _backend()
            s["be"], s["sets"] = be, [be.adapters(p["n"], c["k"], _DTYPES[c["dtype"]], max_adapters=c["adapters"], max_rank=max(ranks)) for p in sets]
            for p, handle in zip(sets, s["sets"]):
                for i, r in enumerate(ranks):
                    handle.load(i, p["a"][i, :r], p["b"][i, :r].T.contiguous(), float(p["scale"][i]))
        else:
            s["sets"] = sets
        return s
    if kind != "moe":
        s.update(_router_parts(gen, c))
    if kind != "route":
        parts = _expert_parts(gen, c)
        s["out"] = torch.empty((m, c["hidden"]), dtype=_DTYPES[c["y"]], device="cuda")
        if not own:
            s.update(parts)
    if kind == "moe":
        s["ids"], s["weights"] = _choice(gen, c)
    s["x"] = _acts(gen, m, c["hidden"], c["x"])
    if own:
        import magnitude_b200 as mb

        s["be"] = be = _backend()
        if kind != "moe":
            s["handle"] = be.router(s["router"], c["top_k"], scoring=mb.SCORING_SIGMOID if c["scoring"] == "sigmoid" else mb.SCORING_SOFTMAX, normalise=True,
                                    scale=_route_scale(c), select_bias=s["bias"], max_rows=m)
            s["ids"] = torch.empty((m, c["top_k"]), dtype=torch.int32, device="cuda")
            s["weights"] = torch.empty((m, c["top_k"]), device="cuda")
        if kind != "route":
            types = {t: getattr(mb, "TYPE_" + t) for t in _BLOCK}
            s["layer"] = be.moe(parts.pop("gate"), parts.pop("up"), parts.pop("down"), gate_up_type=types[c["type"]], down_type=types[c["type_down"]],
                                top_k=c["top_k"], n_embd=c["hidden"], n_ff=c["inter"], max_rows=m,
                                activation=mb.MOE_SWIGLU_CLAMPED if c["act"] == "clamped" else mb.MOE_SWIGLU, alpha=_ALPHA, limit=_LIMIT, **parts)
    return s


def _route_scale(c):
    return 2.5 if c["scoring"] == "sigmoid" else 1.0


# ---- one pass -------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(s, c)
    if c["kind"] == "lora":
        for p, y in zip(s["sets"], s["y"]):
            y.copy_(_plain_adapters(p, s["x"], s["rows"], y))
        return s["y"]
    ids, weights = (s["ids"], s["weights"]) if c["kind"] == "moe" else _plain_route(c, s["router"], s["bias"], s["x"])
    if c["kind"] == "route":
        return ids, weights
    y = s["out"].copy_(_plain_experts(s, c, s["x"], ids, weights))
    return y if c["kind"] == "moe" else (ids, weights, y)


def _run_own(s, c):
    be = s["be"]
    if c["kind"] == "lora":
        return be.apply_adapters(s["sets"], s["x"], s["rows"], s["y"])
    if c["kind"] != "moe":
        be.route(s["handle"], s["x"], s["ids"], s["weights"])
        if c["kind"] == "route":
            return s["ids"], s["weights"]
    y = be.run_moe(s["layer"], s["x"], s["ids"], s["weights"], out=s["out"])
    return y if c["kind"] == "moe" else (s["ids"], s["weights"], y)


# ---- the plain forms ------------------------------------------------------------------------------

def _plain_route(c, w, bias, x):
    """Logits in 64 bits: a choice lies next to a border."""
    logits = x.double() @ w.double().T
    scores = torch.sigmoid(logits) if c["scoring"] == "sigmoid" else torch.softmax(logits, dim=1)
    by = logits if bias is None else scores + bias.double()
    ids = torch.sort(by, dim=1, descending=True, stable=True).indices[:, : c["top_k"]]      # equal ones: the lower index first
    weights = torch.gather(scores, 1, ids)
    weights = weights / weights.sum(dim=1, keepdim=True) * _route_scale(c)
    return ids.to(torch.int32), weights.float()


def _half(b, at):
    return b[..., at:at + 2].contiguous().view(torch.float16).float()


def _unpack(t, packed, k):
    """The weights that rows of blocks stand for, [..., k] in 32 bits."""
    elems, size = _BLOCK[t]
    b = packed.reshape(-1, size)
    if t == "Q8_0":
        v = b[:, 2:].contiguous().view(torch.int8).float().mul_(_half(b, 0))
    elif t == "Q4_0":
        v = torch.cat([b[:, 2:] & 15, b[:, 2:] >> 4], dim=1).float().sub_(8).mul_(_half(b, 0))
    elif t == "MXFP4":
        code = torch.cat([b[:, 1:] & 15, b[:, 1:] >> 4], dim=1)
        step = code & 7
        whole = torch.where(step < 4, step, torch.where(step < 6, 2 * step - 4, 4 * step - 16)).float()       # twice the value
        v = torch.where(code > 7, -whole, whole).mul_(torch.exp2(b[:, :1].float() - 128))
    elif t in ("Q4_K", "Q5_K"):
        s = b[:, 4:16]
        scale = torch.cat([s[:, :4] & 63, s[:, 8:] & 15 | s[:, :4] >> 6 << 4], dim=1).float() * _half(b, 0)
        least = torch.cat([s[:, 4:8] & 63, s[:, 8:] >> 4 | s[:, 4:8] >> 6 << 4], dim=1).float() * _half(b, 2)
        nib = b[:, size - 128:].reshape(-1, 4, 1, 32)
        q = torch.cat([nib & 15, nib >> 4], dim=2).reshape(-1, 8, 32)
        if t == "Q5_K":
            q = q + ((b[:, None, 16:48] >> torch.arange(8, device=b.device, dtype=torch.uint8)[:, None] & 1) << 4)
        v = q.float().mul_(scale[:, :, None]).sub_(least[:, :, None])
    else:
        low = b[:, :128].reshape(-1, 2, 1, 64)
        low = torch.cat([low & 15, low >> 4], dim=2).reshape(-1, 2, 4, 32)
        high = b[:, 128:192].reshape(-1, 2, 1, 32) >> torch.tensor([0, 2, 4, 6], device=b.device, dtype=torch.uint8)[:, None] & 3
        scale = b[:, 192:208].contiguous().view(torch.int8).float() * _half(b, 208)
        v = (low | high << 4).reshape(-1, 16, 16).float().sub_(32).mul_(scale[:, :, None])
    return v.reshape(*packed.shape[:-1], k)


def _plain_experts(s, c, x, ids, weights):
    """Of few tokens the chosen experts alone are unpacked, otherwise all of them; every token is multiplied by those, and the
    share of an expert that it has not chosen is nothing."""
    m, e, k = c["m"], c["experts"], c["top_k"]
    flat = ids.reshape(-1).long()
    if m * k < e:
        which, column = flat, torch.arange(m * k, device="cuda")
    else:
        which, column = torch.arange(e, device="cuda"), flat
    token = torch.arange(m, device="cuda").repeat_interleave(k)
    share = torch.zeros((m, which.numel()), device="cuda").index_put_((token, column), weights.reshape(-1), accumulate=True)
    x = x.float()
    a = torch.matmul(x, _unpack(c["type"], s["gate"][which], c["hidden"]).transpose(1, 2))       # [experts, m, inter]
    b = torch.matmul(x, _unpack(c["type"], s["up"][which], c["hidden"]).transpose(1, 2))
    if c["act"] == "clamped":
        a = (a + s["gate_bias"][which][:, None]).clamp(max=_LIMIT)
        b = (b + s["up_bias"][which][:, None]).clamp(-_LIMIT, _LIMIT)
        h = a * torch.sigmoid(_ALPHA * a) * (b + 1)
    else:
        h = a * torch.sigmoid(a) * b
    y = torch.matmul(h, _unpack(c["type_down"], s["down"][which], c["inter"]).transpose(1, 2))    # [experts, m, hidden]
    if c["act"] == "clamped":
        y = y + s["down_bias"][which][:, None]
    return (y * share.T[:, :, None]).sum(dim=0)


def _plain_adapters(p, x, rows, y):
    a, b = p["a"].float(), p["b"].float()
    adapters, top, k = a.shape
    mine = (rows[:, None] == torch.arange(adapters, device="cuda")).float() * p["scale"]
    t = (x.float() @ a.reshape(-1, k).T).reshape(-1, adapters, top) * mine[:, :, None]
    return y.float() + t.reshape(-1, adapters * top) @ b.reshape(-1, p["n"])


# ---- the same results in 64 bits ---------------------------------------------------------------------

def _values(t, packed, k):
    """The weights of blocks in 64 bits, written down block field by block field."""
    elems, size = _BLOCK[t]
    b = packed.reshape(-1, size)
    bits = lambda v, n: v.to(torch.int32).remainder(1 << n).double()  # noqa: E731
    f16 = lambda at: b[:, at:at + 2].contiguous().view(torch.float16).double()  # noqa: E731
    v = torch.empty((b.shape[0], elems), dtype=torch.float64, device=b.device)
    if t == "Q8_0":
        signed = b[:, 2:].double()
        v[:] = f16(0) * torch.where(signed < 128, signed, signed - 256)
    elif t == "Q4_0":
        v[:, :16], v[:, 16:] = f16(0) * (bits(b[:, 2:], 4) - 8), f16(0) * (bits(b[:, 2:] >> 4, 4) - 8)
    elif t == "MXFP4":
        table = torch.tensor(_E2M1, dtype=torch.float64, device=b.device)
        step = torch.exp2(b[:, :1].double() - 127)
        v[:, :16], v[:, 16:] = step * table[bits(b[:, 1:], 4).long()], step * table[bits(b[:, 1:] >> 4, 4).long()]
    elif t in ("Q4_K", "Q5_K"):
        for j in range(8):
            if j < 4:
                scale, least = bits(b[:, 4 + j], 6), bits(b[:, 8 + j], 6)
            else:
                scale = bits(b[:, 8 + j], 4) + 16 * bits(b[:, j] >> 6, 2)
                least = bits(b[:, 8 + j] >> 4, 4) + 16 * bits(b[:, 4 + j] >> 6, 2)
            q = bits(b[:, size - 128 + 32 * (j // 2):size - 96 + 32 * (j // 2)] >> (4 * (j % 2)), 4)
            if t == "Q5_K":
                q = q + 16 * bits(b[:, 16:48] >> j, 1)
            v[:, 32 * j:32 * j + 32] = f16(0) * scale[:, None] * q - f16(2) * least[:, None]
    else:
        for j in range(8):                       # run j % 4 of half j / 4
            half, at = j // 4, j % 4
            low = bits(b[:, 64 * half + 32 * (at % 2):64 * half + 32 * (at % 2) + 32] >> (4 * (at // 2)), 4)
            q = low + 16 * bits(b[:, 128 + 32 * half:160 + 32 * half] >> (2 * at), 2) - 32
            for part in range(2):
                scale = b[:, 192 + 2 * j + part].double()
                scale = torch.where(scale < 128, scale, scale - 256)
                v[:, 32 * j + 16 * part:32 * j + 16 * part + 16] = f16(208) * scale[:, None] * q[:, 16 * part:16 * part + 16]
    return v.reshape(-1, k)


def _exact_route(c, w, bias, x):
    logits = (x.double()[:, None, :] * w.double()[None]).sum(dim=2) if c["m"] * c["experts"] * c["hidden"] < 2e8 else x.double() @ w.double().T
    if c["scoring"] == "sigmoid":
        scores = 1 / (1 + torch.exp(-logits))
    else:
        scores = torch.exp(logits - logits.max(dim=1, keepdim=True).values)
    by = logits if bias is None else scores + bias.double()
    ids = torch.empty((c["m"], c["top_k"]), dtype=torch.long, device="cuda")
    left = by.clone()
    for j in range(c["top_k"]):
        top = left.max(dim=1, keepdim=True).values
        ids[:, j] = (left == top).to(torch.uint8).argmax(dim=1)      # the first of equal ones
        left.scatter_(1, ids[:, j:j + 1], -torch.inf)
    chosen = scores.gather(1, ids)
    return ids.to(torch.int32), chosen / chosen.sum(dim=1, keepdim=True) * _route_scale(c)


def _exact_experts(p, c, x, ids, weights):
    x = x.double()
    y = torch.zeros((c["m"], c["hidden"]), dtype=torch.float64, device="cuda")
    for e in torch.unique(ids).tolist():
        token, j = torch.nonzero(ids == e, as_tuple=True)
        a = x[token] @ _values(c["type"], p["gate"][e], c["hidden"]).T
        b = x[token] @ _values(c["type"], p["up"][e], c["hidden"]).T
        if c["act"] == "clamped":
            a = torch.minimum(a + p["gate_bias"][e].double(), torch.tensor(_LIMIT, device="cuda", dtype=torch.float64))
            b = torch.maximum(torch.minimum(b + p["up_bias"][e].double(), torch.full_like(b, _LIMIT)), torch.full_like(b, -_LIMIT))
            h = a / (1 + torch.exp(-_ALPHA * a)) * (b + 1)
        else:
            h = a / (1 + torch.exp(-a)) * b
        out = h @ _values(c["type_down"], p["down"][e], c["inter"]).T
        if c["act"] == "clamped":
            out = out + p["down_bias"][e].double()
        y.index_add_(0, token, weights[token, j].double()[:, None] * out)
    return y


def exact(case, seed):
    """What `run` returns on the state of `prepare(case, seed)`, from the same draws, in 64 bits."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    c = dict(case)
    m, kind = c["m"], c["kind"]
    if kind == "lora":
        ranks, sets = _adapter_parts(gen, c)
        rows, x = _adapter_rows(gen, c), _acts(gen, m, c["k"], c["x"]).double()
        out = []
        for p in sets:
            y = torch.randn((m, p["n"]), generator=gen, device="cuda").to(_DTYPES[c["y"]]).double()
            for i, r in enumerate(ranks):
                mine = torch.nonzero(rows == i).flatten()
                inner = x[mine] @ p["a"][i, :r].double().T
                y[mine] += p["scale"][i].double() * (inner @ p["b"][i, :r].double())
            out.append(y)
        return out
    router = _router_parts(gen, c) if kind != "moe" else None
    parts = _expert_parts(gen, c) if kind != "route" else None
    ids, weights = _choice(gen, c) if kind == "moe" else (None, None)
    x = _acts(gen, m, c["hidden"], c["x"])
    if kind != "moe":
        ids, weights = _exact_route(c, router["router"], router["bias"], x)
        if kind == "route":
            return ids, weights
    y = _exact_experts(parts, c, x, ids, weights)
    return y if kind == "moe" else (ids, weights, y)


# ---- what a pass cannot do without ------------------------------------------------------------------

def work(case):
    c = case
    m = c["m"]
    if c["kind"] == "lora":
        ranks = [int(r) for r in c["ranks"].split(",")]
        rank = sum(ranks[i % len(ranks)] for i in range(c["adapters"])) / c["adapters"]
        used = c["adapters"] * (1 - (1 - 1 / c["adapters"]) ** m) if c["rows"] == "any" else min(c["adapters"], m)
        ns = [int(n) for n in c["n"].split(",")]
        nbytes = m * c["k"] * _SIZE[c["x"]] + sum(2 * m * n * _SIZE[c["y"]] + used * rank * (n + c["k"]) * _SIZE[c["dtype"]] for n in ns)
        return {"bytes": nbytes, "flops": sum(2.0 * m * rank * (n + c["k"]) for n in ns)}
    nbytes = m * c["hidden"] * _SIZE[c["x"]] + m * c["top_k"] * 8.0
    flops = 0.0
    if c["kind"] != "moe":
        nbytes += c["experts"] * c["hidden"] * _SIZE[c["w"]]
        flops += 2.0 * m * c["experts"] * c["hidden"]
    if c["kind"] != "route":
        rate = lambda t: _BLOCK[t][1] / _BLOCK[t][0]  # noqa: E731
        used = c["experts"] * (1 - (1 - c["top_k"] / c["experts"]) ** m)      # experts that some token picks, all being equal
        nbytes += used * c["hidden"] * c["inter"] * (2 * rate(c["type"]) + rate(c["type_down"])) + m * c["hidden"] * _SIZE[c["y"]]
        flops += 6.0 * m * c["top_k"] * c["hidden"] * c["inter"]
    return {"bytes": nbytes, "flops": flops}
