"""The operators of products whose weights a row's index chooses, as they are measured: each in its
plain form (`own` false: elementary torch operations, 32 bits, 64 where 32 lose what matters) and
through the library (`own` true).

  route   a router's choice of experts: ids, weights, and the entries sorted by expert
  swiglu  the experts' gate and up projections, silu(gate) * up, over GGUF blocks
  down    the experts' down projection, summed over a row's experts with the router's weights
  lora    low-rank adapters, one to a row, added to shared projections

An entry is a row's j-th expert, number row * top_k + j. `order` lists the entries sorted by
expert (equal ones by entry), those without an expert last; those of expert e are
order[offsets[e]:offsets[e + 1]].

Weights are GGUF blocks ([experts][rows][blocks]); activations are quantized to Q8_0 before a
product with them (blocks of 32: d = amax / 127, codes x / d rounded to even), which is a part of
the operator. Adapters are binary16 or fp32 and meet fp32 activations.
"""
from __future__ import annotations

import math
import random

import torch

own = False

# GGUF types: id, elements and bytes of a block
TYPES = {"Q4_0": (2, 32, 18), "Q5_0": (6, 32, 22), "Q8_0": (8, 32, 34), "Q4_K": (12, 256, 144),
         "Q5_K": (13, 256, 176), "Q6_K": (14, 256, 210)}


# ---- cases ----------------------------------------------------------------------------------

def _route(name, rows, experts, top, sigmoid=False, bias=False, normalise=True, groups=1,
           top_groups=1, scale=1.0):
    c = {"op": "route", "rows": rows, "experts": experts, "top": top, "sigmoid": sigmoid,
         "bias": bias, "normalise": normalise, "groups": groups, "top_groups": top_groups,
         "scale": scale}
    return c if name is None else {"name": name, **c}


def _experts(name, op, rows, experts, top, k, n, typ, skew=0.5):
    c = {"op": op, "rows": rows, "experts": experts, "top": top, "k": k, "n": n, "type": typ,
         "skew": skew}
    return c if name is None else {"name": name, **c}


def _lora(name, rows, adapters, rank, k, outs, half=True, runs=False, none=0.0):
    c = {"op": "lora", "rows": rows, "adapters": adapters, "rank": rank, "k": k, "outs": outs,
         "half": half, "runs": runs, "none": none}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one token of a chat, eight experts: launch and latency bound
        _route("route_1x8_top2", 1, 8, 2),
        # a prompt through a router with selection bias and groups of experts
        _route("route_4099x256_top8", 4099, 256, 8, sigmoid=True, bias=True, groups=8,
               top_groups=4, scale=2.5),
        # one token through two of eight feed-forwards of the 8B model's size
        _experts("swiglu_1_row_q4_k", "swiglu", 1, 8, 2, 4096, 14336, "Q4_K"),
        # a decode batch over many small experts: a few rows to each
        _experts("swiglu_61_rows_q4_k", "swiglu", 61, 128, 8, 2048, 768, "Q4_K"),
        # a prompt of odd length over experts whose rows are no multiple of 256
        _experts("swiglu_509_rows_q8_0", "swiglu", 509, 60, 4, 1408, 1376, "Q8_0"),
        # a long prompt over eight large experts
        _experts("swiglu_2048_rows_q4_k", "swiglu", 2048, 8, 2, 4096, 14336, "Q4_K"),
        # the same three kinds of batch on the way down
        _experts("down_1_row_q6_k", "down", 1, 8, 2, 14336, 4096, "Q6_K"),
        _experts("down_61_rows_q5_k", "down", 61, 128, 8, 768, 2048, "Q5_K"),
        _experts("down_2048_rows_q6_k", "down", 2048, 8, 2, 14336, 4096, "Q6_K"),
        # one token with an adapter on q, k and v of the 8B model
        _lora("lora_1_row_qkv", 1, 4, 16, 4096, "4096,1024,1024"),
        # a decode batch of many tenants on gate and up, some without an adapter
        _lora("lora_64_rows_32_adapters", 64, 32, 64, 4096, "14336,14336", none=0.1),
        # prompts of a few tenants, fp32 adapters
        _lora("lora_2045_rows_q", 2045, 5, 32, 4096, "4096", half=False, runs=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "swiglu", "swiglu", "down", "down", "lora"])
    if op == "route":
        experts = rng.choice([8, 16, 60, 64, 128, 160, 256, 512])
        top = rng.choice([1, 2, 4, 6, 8])
        bias = rng.random() < 0.4
        groups = rng.choice([1, 1, 2, 4])
        top_groups = rng.randint(max(1, -(-top * groups // experts)), groups)
        return _route(None, _log(rng, 1, min(4099, 4099 * 256 // experts)), experts, top,
                      rng.random() < 0.5, bias, rng.random() < 0.7, groups, top_groups,
                      rng.choice([1.0, 2.5]))
    if op == "lora":
        outs = ",".join(str(rng.choice([128, 512, 896, 1000, 1024, 4096, 4864]))
                        for _ in range(rng.randint(1, 3)))
        rows = _log(rng, 1, 2045)
        runs = rows > 100
        return _lora(None, rows, _log(rng, 1, 5 if runs else 64), rng.choice([4, 8, 16, 32, 40, 64]),
                     rng.choice([896, 1000, 2048, 4096, 4864]), outs, rng.random() < 0.7, runs,
                     rng.choice([0.0, 0.2]))
    typ = rng.choice(sorted(TYPES))
    experts = rng.choice([4, 8, 16, 60, 64, 128])
    top = rng.choice([1, 2, 4, 6, 8])
    unit = TYPES[typ][1]
    most = 14336 * 4096 * 8 // experts  # weights of an expert
    k = unit * _log(rng, max(1, 512 // unit), 8192 // unit)
    n = max(32, min(most // k, rng.choice([_log(rng, 100, 8192), 32 * _log(rng, 10, 256)])))
    top = min(top, experts)
    rows = _log(rng, 1, 2048)
    while rows > 1 and rows * top * n * k > 2048 * 2 * 14336 * 4096 // 2:
        rows = rows * 2 // 3
    return _experts(None, op, rows, experts, top, k, n, typ, rng.choice([0.0, 0.5, 1.5]))


def _outs(case):
    return [int(v) for v in case["outs"].split(",")]


# ---- inputs -------------------------------------------------------------------------------------

def _half(x):
    return x.to(torch.float16).view(torch.uint8).view(*x.shape, 2)


def _weights(typ, experts, n, k, gen):
    """Random GGUF blocks [experts, n, row bytes] whose values have about the spread 1 / sqrt(k)."""
    _, unit, size = TYPES[typ]
    blocks = experts * n * (k // unit)
    w = torch.randint(0, 256, (blocks, size), dtype=torch.uint8, device="cuda", generator=gen)
    # spread of codes (and sub-scales) of each type, and where the scale stands
    spread = {"Q4_0": 4.6, "Q5_0": 9.2, "Q8_0": 74.0, "Q4_K": 260.0, "Q5_K": 530.0,
              "Q6_K": 1360.0}[typ]
    d = (torch.randn(blocks, device="cuda", generator=gen) * 0.3).exp() / (spread * math.sqrt(k))
    if typ == "Q6_K":
        w[:, 208:210] = _half(d)
    else:
        w[:, 0:2] = _half(d)
    if typ in ("Q4_K", "Q5_K"):
        w[:, 2:4] = _half(d * (7.5 if typ == "Q4_K" else 15.5))
    return w.view(experts, n, -1)


def _grouped(ids, groups):
    """order and offsets of the entries' ids (int32, those outside [0, groups) last)."""
    flat = ids.reshape(-1)
    flat = torch.where((flat >= 0) & (flat < groups), flat, groups)
    order = torch.sort(flat, stable=True).indices.to(torch.int32)
    counts = (flat[None, :] == torch.arange(groups, device=flat.device)[:, None]).sum(1)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = counts.cumsum(0)
    return order, offsets


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    st = {"case": dict(case)}
    m = case["rows"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["op"] == "route":
        e = case["experts"]
        st["logits"] = randn(m, e) * 1.5 + randn(e)
        st["bias"] = randn(e) * 0.1 if case["bias"] else None
        return st
    if case["op"] == "lora":
        k, rank, slots = case["k"], case["rank"], case["adapters"]
        dt = torch.float16 if case["half"] else torch.float32
        # requests of one row each, or a few prompts
        ids = [rng.randrange(slots) for _ in range(m)]
        if case["runs"]:
            cuts = sorted(rng.randrange(m) for _ in range(slots + 2))
            ids = [(sum(c <= i for c in cuts) * 7) % slots for i in range(m)]
        ids = [-1 if rng.random() < case["none"] else i for i in ids]
        st["ids"] = torch.tensor(ids, dtype=torch.int32, device="cuda")
        st["order"], st["offsets"] = _grouped(st["ids"], slots)
        st["cap"] = max(1, max(ids.count(i) for i in range(slots)))
        ranks = [rank if i % 2 == 0 else max(1, rank - 4 * rng.randint(0, rank // 4)) for i in range(slots)]
        st["ranks"] = torch.tensor(ranks, dtype=torch.int32, device="cuda")
        st["scales"] = torch.rand(slots, device="cuda", generator=gen) + 0.5
        st["x"] = randn(m, k)
        st["a"] = [(randn(slots, rank, k) / math.sqrt(k)).to(dt) for _ in _outs(case)]
        st["b"] = [(randn(slots, n, rank) / math.sqrt(rank)).to(dt) for n in _outs(case)]
        st["base"] = [randn(m, n) for n in _outs(case)]
        return st
    e, top, k, n = case["experts"], case["top"], case["k"], case["n"]
    # popular and unpopular experts
    z = randn(m, e) + randn(e) * case["skew"]
    best = torch.sort(z, dim=1, descending=True, stable=True)
    ids = best.indices[:, :top].to(torch.int32).contiguous()
    st["ids"] = ids
    st["weights"] = torch.softmax(best.values[:, :top], 1)
    st["order"], st["offsets"] = _grouped(ids, e)
    st["cap"] = int((st["offsets"][1:] - st["offsets"][:-1]).max())
    if case["op"] == "swiglu":
        st["w"] = [_weights(case["type"], e, n, k, gen), _weights(case["type"], e, n, k, gen)]
        st["x"] = randn(m, k)
    else:
        st["w"] = [_weights(case["type"], e, n, k, gen)]
        st["x"] = torch.nn.functional.silu(randn(m * top, k)) * randn(m * top, k)
    return st


# ---- the plain forms ------------------------------------------------------------------------------

def _f16(b):
    return b.contiguous().view(torch.float16).to(torch.float32)


def _k_scales(sc):
    """The 6-bit scales and minima of 8 sub-blocks from 12 bytes [..., 12]."""
    sc = sc.to(torch.int32)
    lo, mid, hi = sc[..., 0:4], sc[..., 4:8], sc[..., 8:12]
    s = torch.cat([lo & 63, (hi & 15) | ((lo >> 6) << 4)], -1)
    m = torch.cat([mid & 63, (hi >> 4) | ((mid >> 6) << 4)], -1)
    return s, m


def _dequantize(w, typ, dtype=torch.float32):
    """Blocks [..., row bytes] -> values [..., elements]."""
    _, unit, size = TYPES[typ]
    b = w.reshape(-1, size)
    if typ in ("Q4_K", "Q5_K"):
        s, m = _k_scales(b[:, 4:16])
        d, dm = _f16(b[:, 0:2]).to(dtype), _f16(b[:, 2:4]).to(dtype)
        q = b[:, -128:].view(-1, 4, 1, 32)
        q = torch.cat([q & 15, q >> 4], 2).view(-1, 8, 32)
        if typ == "Q5_K":
            bit = torch.arange(8, device=b.device, dtype=torch.uint8)[None, :, None]
            q = q | (((b[:, None, 16:48] >> bit) & 1) << 4)
        v = (d * s)[..., None] * q.to(dtype) - (dm * m)[..., None]
    elif typ == "Q6_K":
        ql, qh = b[:, :128].view(-1, 2, 2, 32), b[:, 128:192].view(-1, 2, 1, 32)
        low = torch.cat([ql & 15, ql >> 4], 2)  # [.., half, 4, 32]
        two = torch.arange(0, 8, 2, device=b.device, dtype=torch.uint8)[None, None, :, None]
        q = (low | (((qh >> two) & 3) << 4)).to(torch.int32) - 32
        s = b[:, 192:208].contiguous().view(torch.int8).to(dtype).view(-1, 2, 4, 2, 1)
        d = _f16(b[:, 208:210]).to(dtype)
        v = (d[:, :, None, None, None] * s) * q.view(-1, 2, 4, 2, 16).to(dtype)
    else:
        d = _f16(b[:, 0:2]).to(dtype)
        if typ == "Q8_0":
            q = b[:, 2:].contiguous().view(torch.int8).to(dtype)
        else:
            qs = b[:, -16:]
            q = torch.cat([qs & 15, qs >> 4], 1).to(torch.int32)
            if typ == "Q5_0":
                bits = torch.arange(8, device=b.device, dtype=torch.uint8)
                q = q | (((b[:, 2:6, None] >> bits) & 1).view(-1, 32).to(torch.int32) << 4)
            q = (q - (8 if typ == "Q4_0" else 16)).to(dtype)
        v = d * q
    return v.reshape(*w.shape[:-1], -1)


def _quantized(x, dtype=torch.float32):
    """The values of the rows' Q8_0 blocks: scale and codes formed in fp32."""
    b = x.view(*x.shape[:-1], -1, 32)
    d = (b.abs().amax(-1, keepdim=True).double() / 127).float()
    inverse = torch.where(d != 0, (1 / d.double()).float(), 0)
    q = torch.round(b * inverse).clamp(-128, 127)
    return (d.to(dtype) * q.to(dtype)).view(x.shape)


def _places(st):
    """[groups, cap] entries of each group, and whether there is one."""
    offsets, order = st["offsets"].long(), st["order"].long()
    pos = offsets[:-1, None] + torch.arange(st["cap"], device=order.device)
    there = pos < offsets[1:, None]
    return order[pos.clamp(max=order.numel() - 1)], there


def _spread_back(parts, entries, there, n):
    """Rows [groups, cap, width] to their entries [n, width]; entries of no group 0."""
    out = torch.zeros(n + 1, parts.shape[-1], device=parts.device, dtype=parts.dtype)
    at = torch.where(there, entries, n).reshape(-1)
    return out.index_copy_(0, at, parts.reshape(-1, parts.shape[-1]))[:n]


def _product(x, w):
    """x rows [groups, cap, k] times the groups' weights [groups, n, k]."""
    return torch.bmm(x, w.transpose(1, 2).contiguous())


def _choose(z, bias, case, dtype):
    """ids (-1: none) and weights of the chosen experts."""
    e, groups = case["experts"], case["groups"]
    z = z.to(dtype)
    s = torch.sigmoid(z) if case["sigmoid"] else torch.softmax(z, 1)
    key = z if bias is None else s + bias.to(dtype)
    if groups > 1:
        g = key.view(-1, groups, e // groups)
        best = g.amax(-1) if bias is None else torch.sort(g, dim=-1, descending=True).values[..., :2].sum(-1)
        rank = torch.sort(torch.sort(best, dim=1, descending=True, stable=True).indices, dim=1).indices
        key = torch.where((rank < case["top_groups"])[..., None], g, -math.inf).view(-1, e)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["top"]]
    p = s.gather(1, ids)
    if case["normalise"]:
        p = p / p.sum(1, keepdim=True)
    return ids, p * case["scale"]


def _run_plain(st):
    c = st["case"]
    if c["op"] == "route":
        # in 64 bits: scores and biases next to each other decide
        ids, p = _choose(st["logits"], st["bias"], c, torch.float64)
        ids = ids.to(torch.int32)
        order, offsets = _grouped(ids, c["experts"])
        return {"ids": ids, "weights": p.float(), "order": order, "offsets": offsets}
    entries, there = _places(st)
    if c["op"] == "lora":
        r = torch.arange(c["rank"], device="cuda")
        live = (r < st["ranks"][:, None])[:, None, :]
        x = st["x"][entries]

        def add(a, b, base):
            t = _product(x, a.float())
            t = torch.where(live, t, 0) * st["scales"][:, None, None]
            return base + _spread_back(_product(t, b.float()), entries, there, c["rows"])

        return list(map(add, st["a"], st["b"], st["base"]))
    xq = _quantized(st["x"])
    n = c["rows"] * c["top"]
    if c["op"] == "swiglu":
        x = xq[entries // c["top"]]
        g = _product(x, _dequantize(st["w"][0], c["type"]))
        u = _product(x, _dequantize(st["w"][1], c["type"]))
        return _spread_back(g / (1 + torch.exp(-g)) * u, entries, there, n).view(c["rows"], c["top"], -1)
    y = _product(xq[entries], _dequantize(st["w"][0], c["type"]))
    y = _spread_back(y, entries, there, n).view(c["rows"], c["top"], -1)
    return (y * st["weights"][..., None]).sum(1)


# ---- through the library ------------------------------------------------------------------------------

def _run_own(st):
    import cllm_inference_amd as C
    c = st["case"]
    if c["op"] == "route":
        r = C.moe_route_dev(st["logits"], c["top"], bias=st["bias"], sigmoid=c["sigmoid"],
                            normalise=c["normalise"], scale=c["scale"], n_groups=c["groups"],
                            top_groups=c["top_groups"])
        return {"ids": r.ids, "weights": r.weights, "order": r.order, "offsets": r.offsets}
    if c["op"] == "lora":
        groups = C.RowGroups(st["offsets"], st["order"])
        return C.lora_dev(st["x"], st["a"], st["b"], groups, ranks=st["ranks"], scales=st["scales"],
                          base=st["base"])
    route = C.MoeRoute(st["ids"], st["weights"], st["offsets"], st["order"])
    if c["op"] == "swiglu":
        return C.moe_swiglu_dev(st["x"], st["w"][0], st["w"][1], TYPES[c["type"]][0], c["n"], route)
    return C.moe_down_dev(st["x"], st["w"][0], TYPES[c["type"]][0], c["n"], route)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without -------------------------------------------------------------------

def _distinct(slots, rows, each):
    """Expected number of slots that rows of `each` different ones name."""
    return slots * (1 - (1 - each / slots) ** rows)


def work(case):
    m = case["rows"]
    if case["op"] == "route":
        e, top = case["experts"], case["top"]
        return {"bytes": 4 * m * e + 12 * m * top + 4 * (e + 1) + (4 * e if case["bias"] else 0),
                "flops": 4 * m * e}
    if case["op"] == "lora":
        k, rank = case["k"], case["rank"]
        live = m * (1 - case["none"])
        used = min(case["adapters"], live) if case["runs"] else _distinct(case["adapters"], live, 1)
        each = 2 if case["half"] else 4
        w = sum(used * rank * (k + n) * each for n in _outs(case))
        return {"bytes": w + 4 * m * k + sum(8 * m * n for n in _outs(case)),
                "flops": sum(2 * live * rank * (k + n) for n in _outs(case))}
    k, n, top = case["k"], case["n"], case["top"]
    _, unit, size = TYPES[case["type"]]
    mats = 2 if case["op"] == "swiglu" else 1
    w = mats * _distinct(case["experts"], m, top) * n * (k // unit) * size
    rows_in, rows_out = (m, m * top) if mats == 2 else (m * top, m)
    return {"bytes": w + 4 * rows_in * k + 4 * rows_out * n + 12 * m * top,
            "flops": 2 * mats * m * top * n * k}


# ---- the definition in 64 bits -----------------------------------------------------------------------

def _blocks64(w, typ):
    """The values of one expert's blocks [n, row bytes] in 64 bits, from the format's bytes."""
    _, unit, size = TYPES[typ]
    b = w.reshape(-1, size)
    i = torch.arange(unit, device=b.device)

    def half(at):
        return b[:, at:at + 2].contiguous().view(torch.float16).double()

    if typ == "Q8_0":
        return (half(0) * b[:, 2:].contiguous().view(torch.int8).double()).view(w.shape[0], -1)
    if typ in ("Q4_0", "Q5_0"):
        at = 2 if typ == "Q4_0" else 6
        q = (b[:, at + i % 16].long() >> (4 * (i // 16))) & 15
        if typ == "Q5_0":
            q = q + 16 * ((b[:, 2 + i // 8].long() >> (i % 8)) & 1)
        return (half(0) * (q - (8 if typ == "Q4_0" else 16)).double()).view(w.shape[0], -1)
    if typ == "Q6_K":
        h, j, lane = i // 128, (i % 128) // 32, i % 32
        q = (b[:, 64 * h + 32 * (j % 2) + lane].long() >> (4 * (j // 2))) & 15
        q = q + 16 * ((b[:, 128 + 32 * h + lane].long() >> (2 * j)) & 3)
        s = b[:, 192 + i // 16].contiguous().view(torch.int8).double()
        return (half(208) * s * (q - 32).double()).view(w.shape[0], -1)
    sub = i // 32
    low = sub < 4
    at = 4 + sub % 4
    a, c, e = b[:, at].long(), b[:, at + 4].long(), b[:, at + 8].long()
    s = torch.where(low, a & 63, (e & 15) + 16 * (a >> 6))
    m = torch.where(low, c & 63, (e >> 4) + 16 * (c >> 6))
    first = 16 if typ == "Q4_K" else 48
    q = (b[:, first + 32 * (sub // 2) + i % 32].long() >> (4 * (sub % 2))) & 15
    if typ == "Q5_K":
        q = q + 16 * ((b[:, 16 + i % 32].long() >> sub) & 1)
    return (half(0) * (s * q).double() - half(2) * m.double()).view(w.shape[0], -1)


def _rows64(x):
    """The values of the rows' Q8_0 blocks: the scale and its inverse are fp32 numbers, a code is
    the fp32 product with the inverse, rounded to the nearest integer (ties to even)."""
    b = x.view(x.shape[0], -1, 32)
    d = (b.abs().amax(2).double() / 127).float()
    inv = torch.where(d > 0, (1 / d.double()).float(), torch.zeros_like(d))
    code = torch.round((b.double() * inv.double()[..., None]).float().double()).clamp(-128, 127)
    return (code * d.double()[..., None]).view(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "route":
        z = st["logits"].double()
        e, top = case["experts"], case["top"]
        p = z.exp() / z.exp().sum(1, keepdim=True)
        if case["sigmoid"]:
            p = 1 / (1 + (-z).exp())
        key = z if st["bias"] is None else p + st["bias"].double()
        width = e // case["groups"]
        if case["groups"] > 1:
            parts = key.view(-1, case["groups"], width)
            score = parts.max(2).values if st["bias"] is None else parts.topk(min(2, width), 2).values.sum(2)
            keep = score.topk(case["top_groups"], 1).indices
            drop = torch.ones_like(score, dtype=torch.bool).scatter_(1, keep, False)
            key = parts.masked_fill(drop[..., None], -math.inf).view(-1, e)
        w = p.gather(1, key.topk(top, 1).indices)
        if case["normalise"]:
            w = w / w.sum(1, keepdim=True)
        return {"ids": None, "weights": w * case["scale"], "order": None, "offsets": None}
    offsets = st["offsets"].tolist()
    if case["op"] == "lora":
        x, ids = st["x"].double(), st["ids"]
        out = []
        for a, b, base in zip(st["a"], st["b"], st["base"]):
            y = base.double()
            for s in range(case["adapters"]):
                r = int(st["ranks"][s])
                rows = (ids == s).nonzero()[:, 0]
                t = x[rows] @ a[s, :r].double().T
                y[rows] += st["scales"][s].double() * (t @ b[s, :, :r].double().T)
            out.append(y)
        return out
    x = _rows64(st["x"])
    m, top, n = case["rows"], case["top"], case["n"]
    out = torch.zeros(m * top, n, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        at = st["order"][offsets[e]:offsets[e + 1]].long()
        if at.numel() == 0:
            continue
        if case["op"] == "swiglu":
            rows = x[at // top]
            g = rows @ _blocks64(st["w"][0][e], case["type"]).T
            u = rows @ _blocks64(st["w"][1][e], case["type"]).T
            out[at] = g * u / (1 + (-g).exp())
        else:
            out[at] = x[at] @ _blocks64(st["w"][0][e], case["type"]).T
    out = out.view(m, top, n)
    return out if case["op"] == "swiglu" else (out * st["weights"].double()[..., None]).sum(1)
