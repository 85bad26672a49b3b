"""The operators of a decode server over a paged key/value cache held in 4 bits, as they are
measured: each in its plain form (`own` false: elementary torch operations, 32 bits, 64 where 32
lose what matters) and through the library (`own` true).

  attention  grouped-query attention of query rows over the cache (decode, drafts, prompts)
  store      new key and value rows quantized into the cache's pages, and read back
  beam       one beam-search step's page work: the cache forked, extended by a token, partly
             filled pages copied on write
  compact    the pages in use moved to the front of the pool
  logprobs   log probabilities of given tokens, with rank, entropy and top alternatives

The cache
  A page holds page_size positions (a multiple of 32) of every KV head of one layer:
  [n_kv][page_size / 32] tiles of 36 * hd bytes, and the pool is [layers][pages][page bytes].
  Blocks of 32 elements along a head share a scale d, a binary16 number of 8 significant bits; an
  element is d * (c - 8) with a 4-bit code c. A tile (32 positions of one head) is
    key codes     16 hd bytes   [t 2][c][g 4][n 16][w] dwords of 8 codes: position 16 t + n, elements
                                g hd/4 + 8 (c W + w) + e; W = min(4, hd / 32) dwords to a c
    value codes   16 hd bytes   [c hd/64][g 4][n 16][w 4] dwords: element 16 (4 c + w) + n, positions
                                16 (e / 4) + 4 g + e % 4
    key scales     2 hd bytes   [hd / 32][n 16][t 2]: position 16 t + n
    value scales   2 hd bytes   [hd / 32][g 4][e 8]: positions as the value codes'
  with code e of a dword in nibble e / 2 + 4 (e % 2).
  Quantization of a block with largest element mx and smallest mn: a = max(mx, -mn) / 8 rounded to
  bfloat16, at most 8160, then to binary16; d = a if -mn >= mx else -a; c = x / d rounded to the
  nearest integer (ties to even), plus 8, held to 0..15; c = 8 where d is 0.
"""
from __future__ import annotations

import math
import random

import torch

own = False

Q_SCALE = 1.5  # standard deviation of the queries' elements


# ---- cases ----------------------------------------------------------------------------------

def _att(name, seqs, rows, lo, hi, n_head, n_kv, hd, page, mix=0):
    c = {"op": "attention", "seqs": seqs, "rows": rows, "len_lo": lo, "len_hi": hi,
         "n_head": n_head, "n_kv": n_kv, "hd": hd, "page": page, "mix": mix}
    return c if name is None else {"name": name, **c}


def _store(name, seqs, rows, lo, hi, n_kv, hd, page, mix=0):
    c = {"op": "store", "seqs": seqs, "rows": rows, "len_lo": lo, "len_hi": hi, "n_kv": n_kv,
         "hd": hd, "page": page, "mix": mix}
    return c if name is None else {"name": name, **c}


def _beam(name, beams, length, layers, n_kv, hd, page, mix=0):
    c = {"op": "beam", "beams": beams, "length": length, "layers": layers, "n_kv": n_kv, "hd": hd,
         "page": page, "mix": mix}
    return c if name is None else {"name": name, **c}


def _compact(name, pages, fill, layers, n_kv, hd, page, mix=0):
    c = {"op": "compact", "pages": pages, "fill": fill, "layers": layers, "n_kv": n_kv, "hd": hd,
         "page": page, "mix": mix}
    return c if name is None else {"name": name, **c}


def _logp(name, rows, vocab, top, masked=False, ties=False):
    c = {"op": "logprobs", "rows": rows, "vocab": vocab, "top": top, "masked": masked, "ties": ties}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one chat at its start: the 8B model's heads, launch and latency bound
        _att("attention_1_seq_129", 1, 1, 129, 129, 32, 8, 128, 64),
        # a small server of the 0.5B model (heads of 64, seven to a KV head), ragged contexts
        _att("attention_16_seqs_hd64", 16, 1, 1, 2047, 14, 2, 64, 32, mix=1),
        # a full server of the 8B model: 64 sequences of 4096 to 8192 positions, one token each
        _att("attention_64_seqs_8192", 64, 1, 4096, 8192, 32, 8, 128, 64, mix=2),
        # draft tokens to verify: five rows each of 8 sequences, heads of 256
        _att("attention_8_seqs_5_rows", 8, 5, 700, 5000, 16, 4, 256, 64, mix=3),
        # second turns of four chats: up to 509 new tokens after long contexts
        _att("attention_4_seqs_509_rows", 4, 509, 1500, 6000, 32, 8, 128, 128, mix=4),
        # one prompt
        _att("attention_prompt_2048", 1, 2048, 2048, 2048, 32, 8, 128, 64),
        # the new token of 64 sequences
        _store("store_64_tokens", 64, 1, 100, 8000, 8, 128, 64, mix=5),
        # prompts of odd lengths entering the cache together
        _store("store_prompts_4099", 3, 4099, 4099, 6000, 8, 128, 64, mix=6),
        # one step of a beam search with 8 beams after a prompt, every layer of the 8B model
        _beam("beam_8_of_1000", 8, 1000, 32, 8, 128, 64, mix=7),
        # a pool half of whose pages were freed
        _compact("compact_256_pages", 256, 0.5, 32, 8, 128, 64, mix=8),
        # one token of the 8B model's vocabulary
        _logp("logprobs_1x128256_top5", 1, 128256, 5),
        # a prompt scored with its alternatives, an odd vocabulary, some tokens ruled out
        _logp("logprobs_1021x32003_top20", 1021, 32003, 20, masked=True, ties=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "store", "beam", "compact", "logprobs"])
    hd = rng.choice([64, 128, 128, 256])
    n_kv = rng.choice([1, 2, 4, 8])
    page = rng.choice([32, 64, 128, 256])
    mix = rng.randrange(1 << 20)
    if op == "attention":
        group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
        kind = rng.choice(["decode", "decode", "draft", "prompt"])
        rows = {"decode": 1, "draft": rng.randint(2, 9), "prompt": _log(rng, 10, 2048)}[kind]
        seqs = _log(rng, 1, 64 if kind != "prompt" else 6)
        hi = max(rows, _log(rng, 1, 16384))
        # no more work than the largest listed cases: positions read, and scores formed
        while seqs * hi * n_kv * hd > 64 * 6000 * 8 * 128 and seqs > 1:
            seqs -= 1
        while seqs * rows * hi * group * n_kv * hd > 4 * 509 * 3600 * 32 * 128 and rows > 1:
            rows = max(1, rows // 2)
        lo = max(1, rng.choice([hi, hi // 2, hi // 50]))
        return _att(None, seqs, rows, min(lo, hi), hi, n_kv * group, n_kv, hd, page, mix)
    if op == "store":
        rows = rng.choice([1, rng.randint(2, 40), _log(rng, 40, 4096)])
        seqs = _log(rng, 1, 64)
        while seqs * rows * n_kv * hd > 3 * 4099 * 8 * 128 and seqs > 1:
            seqs -= 1
        hi = rows + _log(rng, 1, 4096)
        return _store(None, seqs, rows, max(1, hi // 3), hi, n_kv, hd, page, mix)
    if op == "beam":
        beams = rng.randint(2, 16)
        layers = rng.randint(1, 32)
        length = _log(rng, 1, 3000)
        while (length // page + 5 * beams) * layers * n_kv * page * hd > 32 * 256 * 8 * 64 * 128:
            layers = layers // 2
        return _beam(None, beams, length, layers, n_kv, hd, page, mix)
    if op == "compact":
        layers, pages = rng.randint(1, 32), _log(rng, 5, 4000)
        while layers * pages * n_kv * page * hd > 32 * 256 * 8 * 64 * 128 and pages > 5:
            pages = max(5, pages // 2)
        return _compact(None, pages, rng.choice([0.1, 0.4, 0.7, 0.95]), layers, n_kv, hd, page, mix)
    vocab = rng.choice([32000, 32003, 50257, 128256, 151936, _log(rng, 200, 200000)])
    rows = _log(rng, 1, max(1, min(4000, 1021 * 32003 // vocab)))
    return _logp(None, rows, vocab, min(vocab, rng.choice([0, 1, 5, 20, 64])), rng.random() < 0.5,
                 rng.random() < 0.5)


def _spans(case):
    """The lengths and the new rows of a case's sequences: a part of its description."""
    r = random.Random(case["mix"])
    lens = [r.randint(case["len_lo"], case["len_hi"]) for _ in range(case["seqs"])]
    if case["rows"] == 1:
        return lens, [1] * case["seqs"]
    if case["seqs"] == 1:
        return lens, [min(case["rows"], lens[0])]
    rows = [min(n, r.randint(max(1, case["rows"] // 2), case["rows"])) for n in lens]
    return lens, rows


# ---- the page format, plainly ------------------------------------------------------------------

def _tile_parts(tiles, hd):
    nb = hd // 32
    kc = tiles[:, :16 * hd].contiguous().view(torch.int32)
    vc = tiles[:, 16 * hd:32 * hd].contiguous().view(torch.int32)
    ks = tiles[:, 32 * hd:34 * hd].contiguous().view(torch.float16)
    vs = tiles[:, 34 * hd:].contiguous().view(torch.float16)
    return kc, vc, ks, vs, nb


def _unpack(tiles, hd):
    """tiles [T, 36 hd] bytes -> key codes, value codes [T, 32, hd] (uint8), key scales, value
    scales [T, 32, hd / 32] (binary16)."""
    kc, vc, ks, vs, nb = _tile_parts(tiles, hd)
    n = tiles.shape[0]
    shifts = torch.arange(0, 32, 4, device=tiles.device, dtype=torch.int32)
    w = min(4, hd // 32)
    k = ((kc[..., None] >> shifts) & 15).to(torch.uint8)
    k = k.view(n, 2, nb // w, 4, 16, w, 2, 4).permute(0, 1, 4, 3, 2, 5, 7, 6).reshape(n, 32, hd)
    v = ((vc[..., None] >> shifts) & 15).to(torch.uint8)
    v = v.view(n, hd // 64, 4, 16, 4, 2, 2, 2).permute(0, 6, 2, 7, 5, 1, 4, 3).reshape(n, 32, hd)
    ks = ks.view(n, nb, 16, 2).permute(0, 3, 2, 1).reshape(n, 32, nb)
    vs = vs.view(n, nb, 4, 2, 4).permute(0, 3, 2, 4, 1).reshape(n, 32, nb)
    return k, v, ks, vs


def _pack(k, v, ks, vs, hd):
    """The inverse of _unpack."""
    n, nb, w = k.shape[0], hd // 32, min(4, hd // 32)
    shifts = torch.arange(0, 32, 4, device=k.device, dtype=torch.int64)

    def dwords(x):
        x = (x.to(torch.int64) << shifts).sum(-1)
        return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32).view(n, -1)

    k = k.view(n, 2, 16, 4, nb // w, w, 4, 2).permute(0, 1, 4, 3, 2, 5, 7, 6).reshape(n, -1, 8)
    v = v.view(n, 2, 4, 2, 2, hd // 64, 4, 16).permute(0, 5, 2, 7, 6, 4, 1, 3).reshape(n, -1, 8)
    ks = ks.view(n, 2, 16, nb).permute(0, 3, 2, 1).reshape(n, -1).contiguous()
    vs = vs.view(n, 2, 4, 4, nb).permute(0, 4, 2, 1, 3).reshape(n, -1).contiguous()
    parts = [dwords(k), dwords(v), ks, vs]
    return torch.cat([p.view(torch.uint8).view(n, -1) for p in parts], 1)


def _quantize(x):
    """x [..., hd] fp32 -> codes [..., hd] (uint8), scales [..., hd / 32] (binary16)."""
    b = x.view(*x.shape[:-1], -1, 32)
    mx, mn = b.amax(-1), b.amin(-1)
    a = (torch.maximum(mx, -mn) / 8).to(torch.bfloat16).float().clamp(max=8160.0).to(torch.float16)
    d = torch.where(-mn >= mx, a, -a)
    dd = d.double()[..., None]
    c = torch.where(dd == 0, 8.0, ((b.double() / dd).round() + 8).clamp(0, 15)).to(torch.uint8)
    return c.view(x.shape), d


def _values(codes, scales):
    b = codes.view(*codes.shape[:-1], -1, 32).float() - 8
    return (b * scales.float()[..., None]).view(codes.shape)


def _tiles_of(state, s, t0, t1):
    """Tiles t0..t1 of sequence s as [heads * tiles, 36 hd] bytes, and the pool's view and indexes
    they came from."""
    c = state["case"]
    per = c["page"] // 32
    pool = state["pages"].view(-1, c["n_kv"], per, 36 * c["hd"])
    t = torch.arange(t0, t1, device=pool.device)
    page = state["table"][s][t // per].long()
    return pool, page, t % per


def _cached(state, s, n):
    """Keys and values of the first n positions of sequence s, fp32 [heads, n, hd]."""
    c = state["case"]
    hd, t1 = c["hd"], (n + 31) // 32
    pool, page, sub = _tiles_of(state, s, 0, t1)
    tiles = pool[page, :, sub].transpose(0, 1).reshape(-1, 36 * hd)
    kc, vc, ks, vs = _unpack(tiles, hd)
    k = _values(kc, ks).view(c["n_kv"], t1 * 32, hd)[:, :n]
    v = _values(vc, vs).view(c["n_kv"], t1 * 32, hd)[:, :n]
    return k, v


# ---- inputs -------------------------------------------------------------------------------------

def _random_pool(layers, pages, page, n_kv, hd, gen):
    """A pool whose codes and scales are those of normally distributed rows."""
    pool = torch.empty(layers, pages, n_kv * (page // 32) * 36 * hd, dtype=torch.uint8, device="cuda")
    tiles = pool.view(-1, 36 * hd)
    step = max(1, (1 << 26) // (32 * hd))
    for i in range(0, tiles.shape[0], step):
        t = tiles[i:i + step]
        nib = torch.randn(2, t.shape[0], 32 * hd, device="cuda", generator=gen)
        nib = (nib * 2.7 + 8).round_().clamp_(0, 15).to(torch.uint8)
        t[:, :32 * hd] = nib[0] | (nib[1] << 4)
        d = torch.randn(t.shape[0], 2 * hd, device="cuda", generator=gen)
        sign = torch.randn(t.shape[0], 2 * hd, device="cuda", generator=gen)
        d = ((0.25 * d).exp() * 0.37).to(torch.bfloat16).to(torch.float16)
        t[:, 32 * hd:] = torch.where(sign < 0, -d, d).view(torch.uint8)
    return pool


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _table(lens, page, width, rng):
    """Page ids of sequences of these lengths, from a shuffled pool without gaps."""
    need = [-(-n // page) for n in lens]
    ids = list(range(sum(need)))
    rng.shuffle(ids)
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return table, at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    st = {"case": dict(case)}
    op = case["op"]
    if op == "logprobs":
        n, vocab = case["rows"], case["vocab"]
        x = torch.randn(n, vocab, device="cuda", generator=gen) * 2.5
        # a few likely tokens to a row
        hot = torch.randint(vocab, (n, 8), device="cuda", generator=gen)
        x.scatter_add_(1, hot, 6 + 3 * torch.randn(n, 8, device="cuda", generator=gen))
        if case["ties"]:  # a head computed in bfloat16
            x = x.to(torch.bfloat16).float()
        tok = torch.where(torch.rand(n, device="cuda", generator=gen) < 0.5, hot[:, 0],
                          torch.randint(vocab, (n,), device="cuda", generator=gen))
        if case["masked"]:  # tokens a grammar rules out, never the given one
            out = torch.rand(n, vocab, device="cuda", generator=gen) < 0.1
            x.masked_fill_(out.scatter_(1, tok[:, None], False), -math.inf)
        st["logits"], st["tokens"] = x, tok.to(torch.int32)
        return st
    hd, n_kv, page = case["hd"], case["n_kv"], case["page"]
    if op in ("attention", "store"):
        lens, rows = _spans(case)
        width = max(-(-n // page) for n in lens) + 1
        table, n_pages = _table(lens, page, width, rng)
        st["lens_list"], st["rows_list"] = lens, rows
        starts = [0]
        for r in rows:
            starts.append(starts[-1] + r)
        st["q_start"] = _int32(starts)
        st["pages"] = _random_pool(1, n_pages, page, n_kv, hd, gen)
        refs, lens_now = [1] * n_pages, lens
        total = starts[-1]
        if op == "attention":
            st["q"] = torch.randn(total, case["n_head"] * hd, device="cuda", generator=gen) * Q_SCALE
        else:
            st["k"] = torch.randn(total, n_kv * hd, device="cuda", generator=gen)
            st["v"] = torch.randn(total, n_kv * hd, device="cuda", generator=gen)
            # the large channels that keys have
            big = torch.randint(n_kv * hd, (n_kv * hd // 32,), device="cuda", generator=gen)
            st["k"][:, big] *= 6
    elif op == "beam":
        # every beam has its own last pages and shares the prompt's with the others
        beams, length = case["beams"], case["length"]
        whole = max(0, length // page - 1)
        tail = -(-length // page) - whole
        n_pages = whole + 2 * beams * tail + beams + 1
        ids = list(range(n_pages))
        rng.shuffle(ids)
        table, refs = [], [0] * n_pages
        width = whole + tail + 2
        for b in range(beams):
            t = ids[:whole] + ids[whole + b * tail:whole + (b + 1) * tail]
            for i in t:
                refs[i] += 1
            table.append(t + [-1] * (width - len(t)))
        lens_now = [length] * beams
        st["pages"] = _random_pool(case["layers"], n_pages, page, n_kv, hd, gen)
        st["parents"] = _int32([rng.randrange(beams) for _ in range(beams)])
        st["beams"], st["ones"] = _int32(list(range(beams))), _int32([1] * beams)
    else:
        # sequences of a few pages each; the freed ones left holes
        n_pages, per = case["pages"], 7
        ids = list(range(n_pages))
        rng.shuffle(ids)
        live = ids[:max(1, int(n_pages * case["fill"]))]
        table, refs, lens_now = [], [0] * n_pages, []
        for i in range(0, len(live), per):
            t = live[i:i + per]
            for j in t:
                refs[j] = 1
            table.append(t + [-1] * (per + 1 - len(t)))
            lens_now.append(len(t) * page - rng.randrange(page))
        st["pages"] = _random_pool(case["layers"], n_pages, page, n_kv, hd, gen)
    # table, lengths and reference counts lie together, so one copy restores them
    book = _int32([x for t in table for x in t] + list(lens_now) + refs)
    m, width = len(table), len(table[0])
    st["book"], st["book0"] = book, book.clone()
    st["table"] = book[:m * width].view(m, width)
    st["lens"] = book[m * width:m * width + m]
    st["refs"] = book[m * width + m:]
    if own:
        import cllm_inference_amd as C
        st["cache"] = C.Kv4Cache.from_tensors(st["pages"], st["table"], st["lens"], st["refs"],
                                              page_size=page, n_head_kv=n_kv, head_dim=hd)
        if op == "attention":
            st["max_rows"], st["max_len"] = max(st["rows_list"]), max(st["lens_list"])
    return st


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    return (_run_own if own else _run_plain)(op, state)


def _run_own(op, st):
    import cllm_inference_amd as C
    c = st["case"]
    if op == "logprobs":
        r = C.logprobs_dev(st["logits"], st["tokens"], top_k=c["top"])
        return [r.logprobs, r.ranks, r.entropy, r.top_ids, r.top_logprobs]
    cache = st["cache"]
    if op == "attention":
        return C.kv4_attention_dev(cache, 0, st["q"], st["q_start"], n_head=c["n_head"],
                                   max_rows=st["max_rows"], max_len=st["max_len"])
    if op == "store":
        C.kv4_store_dev(cache, 0, st["k"], st["v"], st["q_start"])
        return list(C.kv4_load_dev(cache, 0, st["q_start"], n_rows=st["k"].shape[0]))
    st["book"].copy_(st["book0"])
    if op == "beam":
        C.kv4_fork_dev(cache, st["parents"], st["beams"])
        status = C.kv4_extend_dev(cache, st["beams"], st["ones"])
        return [st["table"], st["lens"], st["refs"], status, st["pages"]]
    n_live = C.kv4_compact_dev(cache)
    return [st["table"], st["lens"], st["refs"], n_live, st["pages"]]


def _run_plain(op, st):
    return {"attention": _plain_attention, "store": _plain_store, "beam": _plain_beam,
            "compact": _plain_compact, "logprobs": _plain_logprobs}[op](st)


def _plain_attention(st):
    c = st["case"]
    hd, n_kv = c["hd"], c["n_kv"]
    group = c["n_head"] // n_kv
    out = torch.empty_like(st["q"])
    at = 0
    for s, (n, r) in enumerate(zip(st["lens_list"], st["rows_list"])):
        k, v = _cached(st, s, n)
        q = st["q"][at:at + r].view(r, n_kv, group, hd).permute(1, 0, 2, 3).reshape(n_kv, r * group, hd)
        seen = torch.arange(n, device=q.device)[None] <= (n - r + torch.arange(r, device=q.device))[:, None]
        seen = seen.repeat_interleave(group, 0)
        for h in range(n_kv):
            x = q[h] @ k[h].t() / math.sqrt(hd)
            x = torch.where(seen, x, -math.inf)
            p = (x - x.amax(1, keepdim=True)).exp()
            y = (p @ v[h]) / p.sum(1, keepdim=True)
            out[at:at + r].view(r, n_kv, group, hd)[:, h] = y.view(r, group, hd)
        at += r
    return out


def _plain_store(st):
    c = st["case"]
    hd, n_kv = c["hd"], c["n_kv"]
    total = st["k"].shape[0]
    (ck, dk), (cv, dv) = _quantize(st["k"].view(total, n_kv, hd)), _quantize(st["v"].view(total, n_kv, hd))
    back_k, back_v = torch.empty_like(st["k"]), torch.empty_like(st["v"])
    at = 0
    for s, (n, r) in enumerate(zip(st["lens_list"], st["rows_list"])):
        t0, t1 = (n - r) // 32, (n + 31) // 32
        pool, page, sub = _tiles_of(st, s, t0, t1)
        tiles = pool[page, :, sub].transpose(0, 1).reshape(-1, 36 * hd)
        parts = [x.view(n_kv, (t1 - t0) * 32, -1) for x in _unpack(tiles, hd)]
        a = n - r - 32 * t0
        for part, new in zip(parts, (ck, cv, dk, dv)):
            part[:, a:a + r] = new[at:at + r].transpose(0, 1)
        kc, vc, ks, vs = [x.reshape(n_kv * (t1 - t0), 32, -1) for x in parts]
        tiles = _pack(kc, vc, ks, vs, hd).view(n_kv, t1 - t0, 36 * hd)
        pool[page, :, sub] = tiles.transpose(0, 1)
        # read back from the pages
        tiles = pool[page, :, sub].transpose(0, 1).reshape(-1, 36 * hd)
        kc, vc, ks, vs = _unpack(tiles, hd)
        for back, codes, scales in ((back_k, kc, ks), (back_v, vc, vs)):
            x = _values(codes, scales).view(n_kv, (t1 - t0) * 32, hd)[:, a:a + r]
            back[at:at + r] = x.transpose(0, 1).reshape(r, n_kv * hd)
        at += r
    return [back_k, back_v]


def _count(ids, n_pages):
    """How many of the ids (-1: none) name each page."""
    ids = ids.reshape(-1).long()
    return torch.zeros(n_pages + 1, dtype=torch.int32, device=ids.device).scatter_add_(
        0, torch.where(ids < 0, n_pages, ids), torch.ones_like(ids, dtype=torch.int32))[:n_pages]


def _plain_beam(st):
    c = st["case"]
    table, lens, refs, pages = st["table"], st["lens"], st["refs"], st["pages"]
    page = c["page"]
    st["book"].copy_(st["book0"])
    # fork: every beam takes its parent's pages
    par = st["parents"].long()
    lens.copy_(lens[par])
    table.copy_(table[par])
    refs.copy_(_count(table, refs.numel()))
    # extend by one token: a partly filled page that others hold too is copied, by all holders
    # but the last one; a sequence whose pages are full takes a new one
    beams = lens.numel()
    b = torch.arange(beams, device=lens.device)
    last = (lens + page - 1) // page - 1
    part = lens % page != 0
    ids = table[b, last.clamp(min=0).long()]
    same = (ids[:, None] == ids[None]) & part[:, None] & part[None]
    copies = part & (refs[ids.clamp(min=0).long()] - (same & (b[None] < b[:, None])).sum(1) > 1)
    takes = copies | ~part
    free = torch.nonzero(refs == 0)[:, 0]
    fresh = free[(torch.cumsum(takes, 0) - 1).clamp(min=0)].int()
    where = torch.where(part, last, last + 1).long()
    table[b, where] = torch.where(takes, fresh, table[b, where])
    who = torch.nonzero(copies)[:, 0]
    pages[:, fresh[who].long()] = pages[:, ids[who].long()]
    lens += 1
    refs.copy_(_count(table, refs.numel()))
    return [table, lens, refs, torch.zeros(1, dtype=torch.int32, device=lens.device), pages]


def _plain_compact(st):
    table, lens, refs, pages = st["table"], st["lens"], st["refs"], st["pages"]
    st["book"].copy_(st["book0"])
    live = refs > 0
    n = live.sum()
    ids = torch.arange(refs.numel(), device=refs.device)
    src = ids[live & (ids >= n)]
    dst = ids[~live & (ids < n)]
    to = ids.clone()
    to[src] = dst
    table.copy_(torch.where(table < 0, table, to[table.clamp(min=0).long()].int()))
    refs[dst] = refs[src]
    refs[src] = 0
    for layer in pages:
        layer[dst] = layer[src]
    return [table, lens, refs, n.int().view(1), pages]


def _ordered(x):
    """int64 keys in the order of the float32 values, ties to the lowest index first."""
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    return (key << 20) + ((1 << 20) - 1 - torch.arange(x.shape[1], device=x.device))


def _plain_logprobs(st):
    x, tok, top = st["logits"], st["tokens"].long(), st["case"]["top"]
    m = x.amax(1, keepdim=True)
    z = x - m
    e = z.exp()
    s = e.sum(1, dtype=torch.float64)
    lse = s.log()
    # z e, and 0 where the token is ruled out
    t = torch.where(e > 0, z * e, 0.0).sum(1, dtype=torch.float64)
    entropy = (lse - t / s).float()
    lp = (z.gather(1, tok[:, None])[:, 0].double() - lse).float()
    xt = x.gather(1, tok[:, None])
    j = torch.arange(x.shape[1], device=x.device)[None]
    rank = ((x > xt).sum(1) + ((x == xt) & (j < tok[:, None])).sum(1)).int()
    ids = _ordered(x).topk(top, 1).indices
    tops = (z.gather(1, ids).double() - lse[:, None]).float()
    return [lp, rank, entropy, ids.int(), tops]


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case, seed):
    global own
    mine, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mine
    if case["op"] == "attention":
        return _exact_attention(case, st)
    if case["op"] == "store":
        return _exact_store(case, st)
    if case["op"] == "logprobs":
        return _exact_logprobs(case, st)
    return None  # pages are moved, not computed


def _at(case, pos, dim, value):
    """Byte offset in a tile and nibble of element dim at position pos; offset of its scale."""
    hd = case["hd"]
    pos, dim = torch.broadcast_tensors(pos, dim)
    if value:
        r = pos % 16
        e, g, n = pos // 16 * 4 + r % 4, r // 4, dim % 16
        dword = ((dim // 64 * 4 + g) * 16 + n) * 4 + dim // 16 % 4
        code, scale = 16 * hd + 4 * dword, 34 * hd + 2 * ((dim // 32 * 4 + g) * 8 + e)
    else:
        w = min(4, hd // 32)
        g, inner = dim // (hd // 4), dim % (hd // 4)
        e, j = inner % 8, inner // 8
        dword = (((pos // 16 * (hd // 32 // w) + j // w) * 4 + g) * 16 + pos % 16) * w + j % w
        code, scale = 4 * dword, 32 * hd + 2 * ((dim // 32 * 16 + pos % 16) * 2 + pos // 16)
    nib = e // 2 + 4 * (e % 2)
    return code + nib // 2, nib % 2 * 4, scale


def _exact_attention(case, st):
    hd, n_kv, page = case["hd"], case["n_kv"], case["page"]
    group = case["n_head"] // n_kv
    pool = st["pages"].view(-1, n_kv, page // 32, 36 * hd)
    pos, dim = torch.arange(32, device="cuda")[:, None], torch.arange(hd, device="cuda")[None]
    maps = []
    for value in (False, True):
        byte, shift, scale = _at(case, pos, dim, value)
        maps.append((byte.reshape(-1), shift.reshape(-1), scale.reshape(-1)))
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (n, r) in enumerate(zip(*_spans(case))):
        ids = [int(i) for i in st["table"][s].tolist()[:-(-n // page)]]
        for h in range(n_kv):
            tiles = pool[ids, h].reshape(-1, 36 * hd)
            kv = []
            for byte, shift, scale in maps:
                code = (tiles[:, byte].int() >> shift) & 15
                bits = tiles[:, scale].int() | (tiles[:, scale + 1].int() << 8)
                d = bits.to(torch.int16).view(torch.float16).double()
                kv.append((d * (code - 8)).view(-1, hd)[:n])
            k, v = kv
            q = st["q"][at:at + r].view(r, n_kv, group, hd)[:, h].double()
            for i0 in range(0, r, 256):
                i1 = min(r, i0 + 256)
                x = (q[i0:i1].reshape(-1, hd) @ k.t()).view(i1 - i0, group, n) * hd ** -0.5
                limit = n - r + torch.arange(i0, i1, device="cuda")
                x.masked_fill_(torch.arange(n, device="cuda")[None, None] > limit[:, None, None], -math.inf)
                p = torch.softmax(x, -1)
                y = (p.view(-1, n) @ v).view(i1 - i0, group, hd)
                out[at + i0:at + i1].view(i1 - i0, n_kv, group, hd)[:, h] = y
        at += r
    return out


def _exact_store(case, st):
    res = []
    for x in (st["k"], st["v"]):
        b = x.double().view(-1, 32)
        top, low = b.max(1).values, b.min(1).values
        size = torch.maximum(top.abs(), low.abs()) * 0.125
        # eight significant bits: the mantissa of frexp lies in [0.5, 1)
        man = torch.frexp(size).mantissa
        power = torch.where(size > 0, size / man, 0.0)
        size = ((man * 256).round() / 256 * power).clamp(max=8160)
        size = torch.where(size < 2.0 ** -14, (size * 2.0 ** 24).round() * 2.0 ** -24, size)
        d = torch.where(-low >= top, size, -size)[:, None]
        c = torch.where(d == 0, 0.0, (b / torch.where(d == 0, 1.0, d)).round().clamp(-8, 7))
        res.append((c * d).view(x.shape))
    return res


def _exact_logprobs(case, st):
    tok, top = st["tokens"].long(), case["top"]
    outs = [[], [], [], [], []]
    for i in range(0, case["rows"], 64):
        x = st["logits"][i:i + 64].double()
        t = tok[i:i + 64, None]
        lp = torch.log_softmax(x, 1)
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        rank = (order == t).int().argmax(1)
        ids = order[:, :top]
        p = lp.exp()
        h = -torch.where(p > 0, p * lp, 0.0).sum(1)
        for o, y in zip(outs, (lp.gather(1, t)[:, 0], rank.int(), h, ids.int(), lp.gather(1, ids))):
            o.append(y)
    return [torch.cat(o) for o in outs]


# ---- what a pass cannot do without ----------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + case["rows"] * (4 + 12 + 8 * case["top"]), "flops": 4 * n}
    hd, n_kv = case["hd"], case["n_kv"]
    if op in ("attention", "store"):
        lens, rows = _spans(case)
        pos = 2 * n_kv * hd * 9 // 16  # bytes of one position
        if op == "attention":
            pairs = sum(r * n - r * (r - 1) // 2 for n, r in zip(lens, rows))
            return {"bytes": pos * sum(lens) + 8 * sum(rows) * case["n_head"] * hd,
                    "flops": 4 * pairs * case["n_head"] * hd}
        # rows in, codes written, codes read, rows out
        return {"bytes": sum(rows) * (16 * n_kv * hd + 2 * pos), "flops": 8 * sum(rows) * n_kv * hd}
    page_bytes = case["layers"] * n_kv * (case["page"] // 32) * 36 * hd
    if op == "beam":
        whole = case["length"] % case["page"] == 0
        # at the least as many copies as there are beams less one for each parent in use: about
        # 1 - (1 - 1/n)^n of the parents are
        n = case["beams"]
        copies = 0 if whole else max(0, round(n * (1 - 1 / n) ** n))
        width = -(-case["length"] // case["page"]) + 2
        return {"bytes": 2 * copies * page_bytes + 8 * n * width, "flops": 0}
    live = max(1, int(case["pages"] * case["fill"]))
    moved = round(live * (1 - live / case["pages"]))
    return {"bytes": 2 * moved * page_bytes + 8 * (live + case["pages"]), "flops": 0}
