"""The serving operators around a batched KV cache: cases to measure them on, their plain form in
elementary torch operations and their definition in 64 bits.

Five operators, in the order a server runs them (the fifth reads a cache back):
  append   rows of ragged prompt chunks (or single tokens) normed, rotated and stored in a cache
           that is f16 or 4-bit, paged or contiguous; the sequences of a 4-bit cache are read
           back as values
  decode   attention of one token per sequence over a 4-bit cache
  chunk    attention of ragged prompt chunks over a 4-bit, f16 or int8 cache
  logits   penalties, biases and grammar masks on a batch of logits, and the greedy tokens
"""
import math

import numpy as np
import torch

own = False

D = 64
EPS = 1e-5
THETA = 1e6
UNIT = 36  # bytes of one 4-bit (token, kv head) row: 32 of codes, f16 scale, f16 lowest value


# ---- the cases ----------------------------------------------------------------------------------
def listed():
    return [
        # the newest token of one conversation into an f16 cache: latency of the smallest call
        _append("append-one", 1, 1, 777, 32, 8, "f16", 16, True),
        # one prompt chunk behind a cached prefix, stored in 4 bits and read back
        _append("append-chunk-4bit", 1, 509, 1500, 32, 8, "q4", 16, True),
        # a batch of prompts arriving together, f16 pages
        _append("append-prompts", 12, 2048, 0, 32, 8, "f16", 64, True),
        # one conversation of ordinary length, contiguous cache: latency
        _decode("decode-one", 1, 1337, 32, 8, 0),
        # a batch of conversations of very different lengths, small pages
        _decode("decode-batch", 64, 8191, 32, 8, 16),
        # few very long contexts: the cache's bytes count
        _decode("decode-long", 4, 131071, 32, 8, 64),
        # a few tokens a sequence (drafted tokens to verify, tails of prompts) over cached prefixes
        _chunk("chunk-short", 16, 5, 4096, 32, 8, "q4", 16),
        # the usual prefill step: one chunk behind a cached prefix
        _chunk("chunk-prefill", 1, 512, 3583, 32, 8, "q4", 16),
        # whole prompts in one call, f16 pages
        _chunk("chunk-prompts", 4, 4096, 0, 32, 8, "f16", 64),
        # one sequence, a short history: latency
        _logits("logits-one", 1, 65536, "f16", 200, 0, False),
        # a serving batch with every feature
        _logits("logits-batch", 64, 65536, "f16", 2000, 50, True),
        # a large odd vocabulary in f32
        _logits("logits-large", 128, 131071, "f32", 4000, 300, True),
    ]


def _append(name, nseq, rows, past, hq, hkv, fmt, page, norm):
    return {"name": name, "op": "append", "nseq": nseq, "rows": rows, "past": past, "hq": hq,
            "hkv": hkv, "fmt": fmt, "page": page, "norm": norm}


def _decode(name, nseq, past, hq, hkv, page):
    return {"name": name, "op": "decode", "nseq": nseq, "past": past, "hq": hq, "hkv": hkv,
            "fmt": "q4", "page": page}


def _chunk(name, nseq, rows, past, hq, hkv, fmt, page):
    return {"name": name, "op": "chunk", "nseq": nseq, "rows": rows, "past": past, "hq": hq,
            "hkv": hkv, "fmt": fmt, "page": page}


def _logits(name, rows, vocab, dtype, hist, bias, mask):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "dtype": dtype,
            "hist": hist, "bias": bias, "mask": mask}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    heads = rng.choice([(32, 8), (16, 8), (16, 2), (8, 8), (64, 8), (12, 12), (6, 3), (8, 1),
                        (24, 12)])
    page = rng.choice([0, 16, 32, 64, 128])
    op = rng.choice(["append", "decode", "chunk", "logits"])
    if op == "append":
        rows = _log_int(rng, 1, 2048)
        nseq = _log_int(rng, 1, max(1, min(64, 24576 // rows // max(1, heads[0] // 32))))
        past = rng.choice([0, _log_int(rng, 1, 4096)])
        past = min(past, 65536 // nseq)
        c = _append("", nseq, rows, past, *heads, rng.choice(["f16", "q4"]), page,
                    rng.random() < 0.7)
    elif op == "decode":
        past = _log_int(rng, 1, 131071)
        nseq = _log_int(rng, 1, max(1, min(128, 4 * 131072 * 8 // (max(8, heads[1]) * past))))
        c = _decode("", nseq, past, *heads, page)
    elif op == "chunk":
        rows = _log_int(rng, 1, 4096)
        past = rng.choice([0, _log_int(rng, 1, 32768)])
        past = min(past, 4 * 4096 * 4096 // rows)
        cost = rows * max(heads[0], 32) * (past + rows)
        nseq = _log_int(rng, 1, max(1, min(32, 4 * 32 * 4096 * 4096 // cost)))
        while nseq * cost > 4 * 32 * 4096 * 4096:
            past, rows = past // 2, (rows + 1) // 2
            cost = rows * max(heads[0], 32) * (past + rows)
        c = _chunk("", nseq, rows, past, *heads, rng.choice(["q4", "q4", "f16", "i8"]), page)
    else:
        vocab = _log_int(rng, 500, 262144)
        rows = _log_int(rng, 1, max(1, min(256, 128 * 131071 // vocab)))
        c = _logits("", rows, vocab, rng.choice(["f16", "f32"]), _log_int(rng, 1, 4096),
                    rng.choice([0, _log_int(rng, 1, min(300, vocab))]), rng.random() < 0.6)
    del c["name"]
    top = [work(x) for x in listed() if x["op"] == op]
    while any(work(c)[k] > max(w[k] for w in top) for k in ("bytes", "flops")):
        big = max((k for k in ("nseq", "rows", "past", "vocab") if k in c),
                  key=lambda k: c[k])
        c[big] = c[big] * 7 // 10
    return c


# ---- lengths (they belong to the case, not to the inputs' seed) -----------------------------------
def _spread(top, n, low, salt):
    """n whole numbers: `top`, and others spread between low * top and top."""
    u = np.random.RandomState(1000 * n + salt).rand(n - 1)
    return [top] + [int(top * (low + (1 - low) * x)) for x in u]


def _lengths(case):
    """Cached keys and new rows of every sequence."""
    n = case["nseq"]
    past = _spread(case["past"], n, 0.02, 1)
    if case["op"] == "decode":
        return past, [1] * n
    return past, [max(1, r) for r in _spread(case["rows"], n, 0.1, 2)]


def _row_bytes(hkv):
    return (hkv * UNIT + 15) // 16 * 16


def work(case):
    if case["op"] == "logits":
        es = 2 if case["dtype"] == "f16" else 4
        r, v = case["rows"], case["vocab"]
        b = r * (2 * v * es + (v // 8 if case["mask"] else 0))
        b += 4 * sum(_spread(case["hist"], r, 0, 3)) + 8 * sum(_spread(case["bias"], r, 0, 4))
        return {"bytes": float(b), "flops": float(2 * r * v)}
    past, rows = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    per_key = {"q4": 2 * UNIT, "f16": 4 * D, "i8": 2 * D}[case["fmt"]] * hkv
    new, keys = sum(rows), sum(past) + sum(rows)
    if case["op"] == "append":
        b = new * ((hq + 2 * hkv) * D * 2 + hq * D * 2 + per_key + 2 * D)
        if case["fmt"] == "q4":  # the cached sequences read back as f16 values
            b += keys * (per_key + 4 * D * hkv)
        return {"bytes": float(b), "flops": float(new * (hq + hkv) * D * 7)}
    pairs = sum(r * p + r * (r + 1) // 2 for p, r in zip(past, rows))
    return {"bytes": float(keys * per_key + new * hq * D * 4), "flops": float(4 * D * hq * pairs)}


# ---- inputs ---------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _rope(n):
    """f16 [n][cos(32) | sin(32)], angles in 64 bits."""
    i = torch.arange(D // 2, dtype=torch.float64, device="cuda")
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * THETA ** (-i / (D // 2))
    return torch.cat([ang.cos(), ang.sin()], 1).float().half()


def _to_q4(x):
    """f16 [..., hkv, 64] -> uint8 [..., row bytes] of the 4-bit rows."""
    xf = x.float()
    lo, hi = xf.amin(-1, keepdim=True), xf.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15).half()
    sf = scale.float()
    code = torch.where(sf > 0, (xf - lo) / sf, torch.zeros_like(xf)).round().clamp(0, 15)
    code = code.to(torch.uint8)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    unit = torch.cat([packed, scale.view(torch.uint8), lo.half().view(torch.uint8)], -1)
    flat = unit.reshape(*x.shape[:-2], x.shape[-2] * UNIT)
    out = torch.zeros(*flat.shape[:-1], _row_bytes(x.shape[-2]), dtype=torch.uint8, device=x.device)
    out[..., :flat.shape[-1]] = flat
    return out


def _values(rows, fmt, hkv, scale=None):
    """Cache rows [..., row] -> f32 values [..., hkv, 64]."""
    if fmt == "f16":
        return rows.float()
    if fmt == "i8":
        return rows.float() * scale.view(hkv, D)
    unit = rows[..., :hkv * UNIT].reshape(*rows.shape[:-1], hkv, UNIT)
    codes = unit[..., :32]
    code = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], D).float()
    par = unit[..., 32:].contiguous().view(torch.float16).float()
    return code * par[..., 0:1] + par[..., 1:2]


def _cache(case, g, lens, page, fill):
    """Cache pools, block table or offsets and (int8) scales that hold `lens` rows a sequence;
    rows of a sequence are random values where `fill`, else zero."""
    hkv, fmt = case["hkv"], case["fmt"]
    n = case["nseq"]
    st = {}
    if page:
        blocks = [-(-m // page) for m in lens]
        pages = sum(blocks) + 3
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros(n, max(blocks), dtype=torch.int32, device="cuda")
        at = 0
        for i, b in enumerate(blocks):
            table[i, :b] = order[at:at + b]
            at += b
        st["block_table"], st["offsets"] = table, None
        lead = (pages, page)
    else:
        starts = np.concatenate([[0], np.cumsum(lens)])
        st["block_table"], st["offsets"] = None, _i32(starts[:-1].tolist())
        lead = (int(starts[-1]) + 5,)
    st["k_scale"] = st["v_scale"] = None
    pools = []
    for which in range(2):
        if fill:
            x = torch.randn(*lead, hkv, D, generator=g, device="cuda", dtype=torch.float16)
            if which == 0:  # keys have a few large channels in earnest
                x *= 1 + 2 * (torch.rand(hkv, D, generator=g, device="cuda") > 0.9).half()
        else:
            x = torch.zeros(*lead, hkv, D, device="cuda", dtype=torch.float16)
        if fmt == "q4":
            x = _to_q4(x)
        elif fmt == "i8":
            sc = x.reshape(-1, hkv * D).abs().amax(0).float().clamp(min=1e-3) / 127
            x = (x.float() / sc.view(hkv, D)).round().clamp(-128, 127).to(torch.int8)
            st["k_scale" if which == 0 else "v_scale"] = sc.contiguous()
        pools.append(x.contiguous())
    st["k"], st["v"] = pools
    return st


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "logits":
        return _prepare_logits(case, seed, g)
    past, rows = _lengths(case)
    hq, hkv, n = case["hq"], case["hkv"], case["nseq"]
    total = [p + r for p, r in zip(past, rows)]
    st = _cache(case, g, total, case["page"], case["op"] != "append" or case["past"] > 0)
    st["case"] = case
    st["past"], st["max_len"] = _i32(past), max(total)
    st["max_rows"], st["sum_len"] = max(rows), sum(total)
    starts = [0] + np.cumsum(rows).tolist()
    st["row_start"] = _i32(starts)
    st["read_start"] = _i32([0] + np.cumsum(total).tolist())
    st["zero"] = _i32([0] * n)
    new = starts[-1]
    if case["op"] == "append":
        st["qkv"] = torch.randn(new, (hq + 2 * hkv) * D, generator=g, device="cuda",
                                dtype=torch.float16)
        st["norm_w"] = (1 + 0.1 * torch.randn(2 * D, generator=g, device="cuda")).half() \
            if case["norm"] else None
        st["rope"] = _rope(st["max_len"])
        st["q_out"] = torch.zeros(new, hq * D, device="cuda", dtype=torch.float16)
        if case["fmt"] == "q4":
            for k in ("k_read", "v_read"):
                st[k] = torch.zeros(st["sum_len"], hkv, D, device="cuda", dtype=torch.float16)
    else:
        st["q"] = torch.randn(new, hq * D, generator=g, device="cuda", dtype=torch.float16)
        st["out"] = torch.zeros(new, hq * D, device="cuda", dtype=torch.float16)
    return st


def _prepare_logits(case, seed, g):
    rows, vocab, cap = case["rows"], case["vocab"], case["hist"]
    rng = np.random.RandomState(seed % (1 << 31))
    lens = _spread(cap, rows, 0, 3)
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    logits = (3 * torch.randn(rows, vocab, generator=g, device="cuda")).to(dt)
    # text repeats itself: most tokens of the history come from a small part of the vocabulary
    hist = (torch.rand(rows, cap + 1, generator=g, device="cuda") ** 3 * vocab).to(torch.int32)
    st = {"case": case, "logits": logits, "out": torch.zeros_like(logits),
          "tok": torch.zeros(rows, dtype=torch.int32, device="cuda"),
          "hist": hist.clamp(0, vocab - 1), "hist_len": _i32(lens),
          "prompt_len": _i32([m // 3 for m in lens]),
          "repetition": 1 + torch.rand(rows, generator=g, device="cuda"),
          "presence": torch.rand(rows, generator=g, device="cuda"),
          "frequency": torch.rand(rows, generator=g, device="cuda") / 4,
          "bias_start": None, "bias_tok": None, "bias_val": None, "mask": None}
    if case["bias"]:
        nb = _spread(case["bias"], rows, 0, 4)
        st["bias_start"] = _i32([0] + np.cumsum(nb).tolist())
        toks = [rng.permutation(vocab)[:m] for m in nb]
        st["bias_tok"] = _i32(np.concatenate(toks).tolist())
        st["bias_val"] = 4 * torch.randn(sum(nb), generator=g, device="cuda")
    if case["mask"]:
        words = (vocab + 31) // 32
        st["mask"] = torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device="cuda",
                                   dtype=torch.int64).to(torch.int32)
    return st


# ---- the operators --------------------------------------------------------------------------------
_context = None


def _ctx():
    global _context
    if _context is None:
        import p2p_b200
        _context = p2p_b200.Context(torch.cuda.current_device())
    return _context


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _params(case):
    import p2p_b200
    return p2p_b200.Params(case["hq"], case["hkv"])


def _own_append(s):
    ctx, case = _ctx(), s["case"]
    prm = _params(case)
    ctx.kv_append(prm, s["qkv"], s["norm_w"], s["rope"], s["k"], s["v"], s["past"],
                  s["row_start"], max_len=s["max_len"], q_out=s["q_out"], offsets=s["offsets"],
                  block_table=s["block_table"])
    if case["fmt"] != "q4":
        return [s["q_out"], s["k"], s["v"]]
    ctx.kv_read(prm, s["k"], s["v"], s["zero"], s["read_start"], s["k_read"], s["v_read"],
                max_len=s["max_len"], offsets=s["offsets"], block_table=s["block_table"])
    return [s["q_out"], s["k_read"], s["v_read"]]


def _own_decode(s):
    _ctx().attn_decode_kv(_params(s["case"]), s["q"], None, None, s["k"], s["v"], s["past"],
                          s["out"], max_past=s["max_len"] - 1, offsets=s["offsets"],
                          block_table=s["block_table"], fused_prep=False)
    return s["out"]


def _own_chunk(s):
    _ctx().attn_chunk_kv(_params(s["case"]), s["q"], s["k"], s["v"], s["past"], s["row_start"],
                         s["out"], max_len=s["max_len"], offsets=s["offsets"],
                         block_table=s["block_table"], k_scale=s["k_scale"],
                         v_scale=s["v_scale"])
    return s["out"]


def _own_logits(s):
    _ctx().logits_pick(s["logits"], s["tok"], out=s["out"], hist=s["hist"],
                       hist_len=s["hist_len"], prompt_len=s["prompt_len"],
                       repetition=s["repetition"], presence=s["presence"],
                       frequency=s["frequency"], bias_start=s["bias_start"],
                       bias_tok=s["bias_tok"], bias_val=s["bias_val"], mask=s["mask"])
    return [s["out"], s["tok"]]


def _positions(s, count):
    """[nseq][count] cache rows (page, slot) of keys 0 .. count-1 of every sequence."""
    j = torch.arange(count, device="cuda")
    if s["block_table"] is not None:
        page = s["k"].shape[1]
        b = (j // page).clamp(max=s["block_table"].shape[1] - 1)
        return s["block_table"].long()[:, b], (j % page).expand(len(s["past"]), -1)
    rows = s["offsets"].long()[:, None] + j
    return rows.clamp(max=s["k"].shape[0] - 1), None


def _fetch(pool, where):
    return pool[where[0]] if where[1] is None else pool[where[0], where[1]]


def _rotate(x, rope):
    """Rotate-half of f32 [rows][heads][64] by f16 table rows, rounded to f16."""
    cos, sin = rope[:, None, :32].float(), rope[:, None, 32:].float()
    a, b = x[..., :32], x[..., 32:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).half()


def _norm(x, w):
    """RMSNorm of f32 [..., 64] with its sum of squares taken in the cache's documented order
    (pairs 32, 16, ... 1 apart), rounded to f16."""
    t = x * x
    n = 32
    while n:
        t = t[..., :n] + t[..., n:2 * n]
        n //= 2
    inv = 1.0 / torch.sqrt(t / 64.0 + EPS)
    return ((x * inv) * w.float()).half().float()


def _plain_append(s):
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    new = s["qkv"].shape[0]
    r = torch.arange(new, device="cuda")
    seq = (r[:, None] >= s["row_start"].long()[None, 1:]).sum(1)
    pos = s["past"].long()[seq] + r - s["row_start"].long()[seq]
    x = s["qkv"].view(new, hq + 2 * hkv, D).float()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if s["norm_w"] is not None:
        q, k = _norm(q, s["norm_w"][:D]), _norm(k, s["norm_w"][D:])
    rope = s["rope"][pos]
    q, k, v = _rotate(q, rope), _rotate(k, rope), v.half()
    if case["fmt"] == "q4":
        k, v = _to_q4(k), _to_q4(v)
    if s["block_table"] is not None:
        page = s["k"].shape[1]
        at = (s["block_table"].long()[seq, pos // page], pos % page)
    else:
        at = (s["offsets"].long()[seq] + pos,)
    s["k"][at] = k
    s["v"][at] = v
    q = q.reshape(new, hq * D)
    if case["fmt"] != "q4":
        return [q, s["k"], s["v"]]
    r = torch.arange(s["sum_len"], device="cuda")
    seq = (r[:, None] >= s["read_start"].long()[None, 1:]).sum(1)
    pos = r - s["read_start"].long()[seq]
    if s["block_table"] is not None:
        at = (s["block_table"].long()[seq, pos // page], pos % page)
    else:
        at = (s["offsets"].long()[seq] + pos,)
    return [q, _values(s["k"][at], "q4", hkv).half(), _values(s["v"][at], "q4", hkv).half()]


def _plain_attention(s, rows):
    """Attention of `rows` padded query rows per sequence."""
    case = s["case"]
    hq, hkv, n = case["hq"], case["hkv"], case["nseq"]
    grp, keys = hq // hkv, s["max_len"]
    where = _positions(s, keys)
    k = _values(_fetch(s["k"], where), case["fmt"], hkv, s["k_scale"])
    v = _values(_fetch(s["v"], where), case["fmt"], hkv, s["v_scale"])
    start, past = s["row_start"].long(), s["past"].long()
    t = torch.arange(rows, device="cuda")
    row = start[:-1, None] + t  # [n][rows]
    real = row < start[1:, None]
    q = s["q"].float()[row.clamp(max=len(s["q"]) - 1)].view(n, rows, hkv, grp, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, hkv, grp * rows, D)
    sc = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1 / math.sqrt(D))
    see = torch.arange(keys, device="cuda") <= (past[:, None] + t)[..., None]  # [n][rows][keys]
    sc = sc.view(n, hkv, grp, rows, keys).masked_fill_(~see[:, None, None], -math.inf)
    sc -= sc.amax(-1, keepdim=True)
    sc.exp_()
    tot = sc.sum(-1, keepdim=True)
    # keys behind a sequence's end may be other sequences' rows: their weight is 0
    o = torch.matmul(sc.view(n, hkv, grp * rows, keys), v.permute(0, 2, 1, 3))
    o = o.view(n, hkv, grp, rows, D) / tot
    o = o.permute(0, 3, 1, 2, 4).reshape(n, rows, hq * D)
    return o[real].half()


def _plain_decode(s):
    return _plain_attention(s, 1)


def _plain_chunk(s):
    return _plain_attention(s, s["max_rows"])


def _plain_logits(s):
    case = s["case"]
    rows, vocab = case["rows"], case["vocab"]
    x = s["logits"].float()
    t = torch.arange(s["hist"].shape[1], device="cuda")
    inside = t < s["hist_len"][:, None]
    made = inside & (t >= s["prompt_len"][:, None])
    at = s["hist"].long()
    seen = torch.zeros_like(x).scatter_add_(1, at, inside.float()) > 0
    count = torch.zeros_like(x).scatter_add_(1, at, made.float())
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    pen = (x - s["frequency"][:, None] * count) - s["presence"][:, None]
    x = torch.where(count > 0, pen, x)
    if s["bias_start"] is not None:
        e = torch.arange(len(s["bias_tok"]), device="cuda")
        row = (e[:, None] >= s["bias_start"].long()[None, 1:]).sum(1)
        x.index_put_((row, s["bias_tok"].long()), s["bias_val"], accumulate=True)
    if s["mask"] is not None:
        w = torch.arange(vocab, device="cuda")
        bit = (s["mask"][:, w // 32] >> (w % 32)) & 1
        x = x.masked_fill(bit == 0, -math.inf)
    y = x.to(s["logits"].dtype)
    top = y.amax(1, keepdim=True)
    first = torch.where(y == top, torch.arange(vocab, device="cuda"), vocab).amin(1)
    tok = torch.where(top[:, 0] > -math.inf, first, -1).to(torch.int32)
    return [y, tok]


_OWN = {"append": _own_append, "decode": _own_decode, "chunk": _own_chunk, "logits": _own_logits}
_PLAIN = {"append": _plain_append, "decode": _plain_decode, "chunk": _plain_chunk,
          "logits": _plain_logits}


# ---- the definition in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "logits":
        return _exact_logits(case, s)
    return _exact_attention(case, s)


def _rows_of(s, pool, i, count):
    """Keys 0 .. count-1 of sequence i as they lie in the cache."""
    if s["block_table"] is not None:
        page = pool.shape[1]
        pages = s["block_table"][i, :-(-count // page)].long()
        return pool[pages].flatten(0, 1)[:count]
    o = int(s["offsets"][i])
    return pool[o:o + count]


def _doubles(rows, case, scale):
    hkv = case["hkv"]
    if case["fmt"] == "f16":
        return rows.double()
    if case["fmt"] == "i8":
        return rows.double() * scale.double().reshape(1, hkv, D)
    b = rows[:, :hkv * UNIT].reshape(-1, hkv, UNIT)
    par = b[:, :, 32:36].contiguous().view(torch.float16).double()
    out = torch.empty(b.shape[0], hkv, D, dtype=torch.float64, device="cuda")
    out[:, :, 0::2] = (b[:, :, :32] % 16).double()
    out[:, :, 1::2] = (b[:, :, :32] // 16).double()
    return out * par[:, :, :1] + par[:, :, 1:]


def _exact_attention(case, s):
    past, rows = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    if sum(r * (p + r) for p, r in zip(past, rows)) * hq > 4e9:
        return None
    outs, at = [], 0
    for i, (p, r) in enumerate(zip(past, rows)):
        k = _doubles(_rows_of(s, s["k"], i, p + r), case, s["k_scale"])
        v = _doubles(_rows_of(s, s["v"], i, p + r), case, s["v_scale"])
        q = s["q"][at:at + r].double().reshape(r, hq, D)
        at += r
        o = torch.empty(r, hq, D, dtype=torch.float64, device="cuda")
        last = p + torch.arange(r, device="cuda")
        hidden = torch.arange(p + r, device="cuda")[None] > last[:, None]
        for h in range(hq):
            w = (q[:, h] @ k[:, h // (hq // hkv)].T) / 8.0
            w[hidden] = -math.inf
            o[:, h] = torch.softmax(w, -1) @ v[:, h // (hq // hkv)]
        outs.append(o.reshape(r, hq * D))
    return torch.cat(outs)


def _exact_append(case, s):
    past, rows = _lengths(case)
    hq, hkv = case["hq"], case["hkv"]
    x = s["qkv"].double().reshape(-1, hq + 2 * hkv, D)
    pos = torch.cat([p + torch.arange(r) for p, r in zip(past, rows)]).cuda()
    head = x[:, :hq + hkv].clone()
    if s["norm_w"] is not None:
        w = s["norm_w"].double()
        head = head / (head.square().mean(-1, keepdim=True) + EPS).sqrt()
        head[:, :hq] *= w[:D]
        head[:, hq:] *= w[D:]
        head = head.half().double()  # a rounding of the definition
    tab = s["rope"].double()[pos][:, None]
    half = torch.cat([-head[..., 32:], head[..., :32]], -1)
    rot = head * tab[..., :32].repeat(1, 1, 2) + half * tab[..., 32:].repeat(1, 1, 2)
    q = rot[:, :hq].reshape(-1, hq * D)
    if case["fmt"] == "q4":
        return [q, None, None]  # codes next to a border have no one value
    k, v = s["k"].double(), s["v"].double()
    at = 0
    for i, (p, r) in enumerate(zip(past, rows)):
        j = p + torch.arange(r, device="cuda")
        if s["block_table"] is not None:
            page = k.shape[1]
            idx = (s["block_table"][i].long()[j // page], j % page)
        else:
            idx = (int(s["offsets"][i]) + j,)
        k[idx] = rot[at:at + r, hq:]
        v[idx] = x[at:at + r, hq + hkv:]
        at += r
    return [q, k, v]


def _exact_logits(case, s):
    rows, vocab = case["rows"], case["vocab"]
    y = s["logits"].double().cpu().numpy()
    hist, lens, plen = (s[k].cpu().numpy() for k in ("hist", "hist_len", "prompt_len"))
    rep, pres, freq = (s[k].double().cpu().numpy() for k in ("repetition", "presence", "frequency"))
    for i in range(rows):
        line = y[i]
        seen = np.unique(hist[i, :lens[i]])
        line[seen] = np.where(line[seen] > 0, line[seen] / rep[i], line[seen] * rep[i])
        made, count = np.unique(hist[i, plen[i]:lens[i]], return_counts=True)
        line[made] -= freq[i] * count + pres[i]
        if s["bias_start"] is not None:
            a, b = int(s["bias_start"][i]), int(s["bias_start"][i + 1])
            np.add.at(line, s["bias_tok"][a:b].cpu().numpy(),
                      s["bias_val"][a:b].double().cpu().numpy())
        if s["mask"] is not None:
            bits = np.unpackbits(s["mask"][i].cpu().numpy().view(np.uint8), bitorder="little")
            line[bits[:vocab] == 0] = -np.inf
    return [torch.from_numpy(y), None]
