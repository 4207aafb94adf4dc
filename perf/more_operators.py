"""The 8-bit operators of a decoder layer around its attention: cases to measure them on, their
plain form in elementary torch operations and their definition in 64 bits.

Five operators, in the order a model runs them:
  embed  rows of an int8 table, named by tokens, as values
  norm   the residual stream's addition, RMS norm and int8 rows with a scale per token
  quant  rows (activations, or a weight's output channels) as int8 with a scale per row
  gemm   int8 product with scales per token and channel, bias, residual
  gate   both projections of a gated feed-forward block, the activation and the product
The int8 rows of norm and quant are read back as the values they stand for.
"""
import math

import torch

own = False

EPS = 1e-5


# ---- the cases ----------------------------------------------------------------------------------
def listed():
    return [
        # a decode batch's tokens, looked up in the tied embedding: latency
        _embed("embed-batch", 64, 65536, 2048, "f16"),
        # the tokens of whole prompts, an f32 residual stream
        _embed("embed-prompts", 16384, 65536, 2048, "f32"),
        # the newest token of one conversation: latency of the smallest call
        _norm("norm-one", 1, 2048, "f16", True, False),
        # whole prompts of a batch
        _norm("norm-prompts", 8192, 2048, "f16", True, False),
        # attention's outputs in f32, rows of an odd length
        _quant("quant-odd", 777, 1003, "f32"),
        # a matrix's output channels, once where the weights are loaded (the tied embedding)
        _quant("quant-weights", 65536, 1024, "f16"),
        # an output projection of one token, added to the residual stream: latency
        _gemm("gemm-one", 1, 2048, 2048, "f16", False, True),
        # the LM head of a batch, logits in f32
        _gemm("gemm-head", 32, 65536, 2048, "f32", False, False),
        # whole prompts through the down projection
        _gemm("gemm-prompts", 8192, 2048, 8192, "f16", False, True),
        # one token through a feed-forward block's first half: the weights' bytes count
        _gate("gate-one", 1, 8192, 2048, "silu"),
        # an odd batch, a narrower model's block, the other activation
        _gate("gate-batch", 37, 4608, 1024, "gelu"),
        # a prompt chunk
        _gate("gate-prompt", 4096, 8192, 2048, "silu"),
    ]


def _embed(name, tokens, rows, cols, dtype):
    return {"name": name, "op": "embed", "m": tokens, "n": rows, "k": cols, "dtype": dtype}


def _norm(name, rows, cols, dtype, residual, normed):
    return {"name": name, "op": "norm", "m": rows, "k": cols, "dtype": dtype,
            "residual": residual, "normed": normed}


def _quant(name, rows, cols, dtype):
    return {"name": name, "op": "quant", "m": rows, "k": cols, "dtype": dtype}


def _gemm(name, m, n, k, dtype, bias, residual):
    return {"name": name, "op": "gemm", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias,
            "residual": residual}


def _gate(name, m, f, k, act):
    return {"name": name, "op": "gate", "m": m, "n": f, "k": k, "act": act}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _width(rng, lo, hi):
    """Half of the widths are whole multiples of 64, as models have them."""
    w = _log_int(rng, lo, hi)
    return w if rng.random() < 0.5 else max(64, w // 64 * 64)


def draw(rng):
    op = rng.choice(["embed", "norm", "quant", "gemm", "gemm", "gate", "gate"])
    dtype = rng.choice(["f16", "f16", "f32"])
    if op == "embed":
        c = _embed("", _log_int(rng, 1, 16384), _log_int(rng, 100, 131072), _width(rng, 64, 8192),
                   dtype)
    elif op == "norm":
        c = _norm("", _log_int(rng, 1, 8192), _width(rng, 64, 8192), dtype, rng.random() < 0.7,
                  rng.random() < 0.4)
    elif op == "quant":
        c = _quant("", _log_int(rng, 1, 65536), _width(rng, 64, 8192), dtype)
    elif op == "gemm":
        c = _gemm("", _log_int(rng, 1, 8192), _width(rng, 64, 65536), _width(rng, 64, 8192),
                  dtype, rng.random() < 0.3, rng.random() < 0.5)
    else:
        c = _gate("", _log_int(rng, 1, 4096), _width(rng, 64, 8192), _width(rng, 64, 4096),
                  rng.choice(["silu", "silu", "gelu"]))
    del c["name"]
    top = [work(x) for x in listed() if x["op"] == op]
    while any(work(c)[k] > max(w[k] for w in top) for k in ("bytes", "flops")):
        big = max((k for k in ("m", "n", "k") if k in c), key=lambda k: c[k])
        c[big] = c[big] * 7 // 10
    return c


def work(case):
    m, k = case["m"], case["k"]
    es = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "embed":  # every row of the table at most once
        return {"bytes": float(min(m, case["n"]) * (k + 4) + m * (4 + k * es)),
                "flops": float(2 * m * k)}
    if case["op"] in ("norm", "quant"):  # rows made (1 byte), read back (1) as f16 (2)
        per = es + 4
        if case["op"] == "norm":
            per += es * (2 * case["residual"] + case["normed"])
        return {"bytes": float(m * k * per + 2 * k * (case["op"] == "norm") + 8 * m),
                "flops": float(7 * m * k)}
    n = case["n"]
    if case["op"] == "gemm":
        b = m * k + n * k + 4 * (m + n) + m * n * es * (1 + case["residual"]) + 4 * n * case["bias"]
        return {"bytes": float(b), "flops": float(2 * m * n * k)}
    return {"bytes": float(m * k + 2 * n * k + 4 * (m + 2 * n) + 2 * m * n),
            "flops": float(4 * m * n * k)}


# ---- inputs ---------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _type(case):
    return torch.float32 if case["dtype"] == "f32" else torch.float16


def _codes(g, rows, cols):
    """int8 [rows][cols] with rows on 16-byte boundaries, and a scale per row: normal values whose
    rows reach their largest code."""
    pitch = (cols + 15) // 16 * 16
    q = torch.zeros(rows, pitch, dtype=torch.int8, device="cuda")[:, :cols]
    q.copy_((34 * torch.randn(rows, cols, generator=g, device="cuda", dtype=torch.float16))
            .round_().clamp_(-127, 127))
    q[:, 0] = 127
    return q, (0.5 + torch.rand(rows, generator=g, device="cuda")) / 50


def _empty_codes(rows, cols):
    pitch = (cols + 15) // 16 * 16
    return (torch.zeros(rows, pitch, dtype=torch.int8, device="cuda")[:, :cols],
            torch.zeros(rows, device="cuda"))


def prepare(case, seed):
    g = _gen(seed)
    m, k = case["m"], case["k"]
    st = {"case": case}
    if case["op"] in ("norm", "quant"):
        dt = _type(case)
        x = torch.randn(m, k, generator=g, device="cuda", dtype=dt)
        # tokens of different sizes, and a few channels that are large in every token
        x *= (0.3 + 2 * torch.rand(m, 1, generator=g, device="cuda")).to(dt)
        x *= (1 + 5 * (torch.rand(k, generator=g, device="cuda") > 0.99)).to(dt)
        st["x"] = x
        st["q"], st["scale"] = _empty_codes(m, k)
        st["values"] = torch.zeros(m, k, device="cuda", dtype=torch.float16)
        if case["op"] == "norm":
            st["w"] = (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).half()
            st["r"] = torch.randn(m, k, generator=g, device="cuda", dtype=dt) \
                if case["residual"] else None
            st["sum"] = torch.zeros_like(x) if case["residual"] else None
            st["y"] = torch.zeros_like(x) if case["normed"] else None
        return st
    n = case["n"]
    if case["op"] == "embed":
        st["q"], st["scale"] = _codes(g, n, k)
        st["tok"] = torch.randint(0, n, (m,), generator=g, device="cuda", dtype=torch.int32)
        st["out"] = torch.zeros(m, k, device="cuda", dtype=_type(case))
        return st
    st["xq"], st["xs"] = _codes(g, m, k)
    if case["op"] == "gemm":
        dt = _type(case)
        st["wq"], st["ws"] = _codes(g, n, k)
        st["ws"] = st["ws"] / math.sqrt(k)
        st["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        st["res"] = torch.randn(m, n, generator=g, device="cuda", dtype=dt) \
            if case["residual"] else None
        st["y"] = torch.zeros(m, n, device="cuda", dtype=dt)
        return st
    st["gq"], gs = _codes(g, n, k)
    st["uq"], us = _codes(g, n, k)
    st["gs"], st["us"] = gs * (3 / math.sqrt(k)), us / math.sqrt(k)
    st["h"] = torch.zeros(m, n, device="cuda", dtype=torch.float16)
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


def _own_embed(s):
    _ctx().read_rows_q8(s["q"], s["scale"], s["out"], index=s["tok"])
    return s["out"]


def _own_norm(s):
    _ctx().add_norm_q8(s["x"], s["w"], s["q"], s["scale"], residual=s["r"], sum_out=s["sum"],
                       y=s["y"], eps=EPS)
    _ctx().read_rows_q8(s["q"], s["scale"], s["values"])
    return [s["sum"], s["y"], s["scale"], s["values"]]


def _own_quant(s):
    _ctx().quantize_rows_q8(s["x"], s["q"], s["scale"])
    _ctx().read_rows_q8(s["q"], s["scale"], s["values"])
    return [s["scale"], s["values"]]


def _own_gemm(s):
    _ctx().gemm_q8((s["wq"], s["ws"]), s["xq"], s["xs"], s["y"], bias=s["bias"],
                   residual=s["res"])
    return s["y"]


def _own_gate(s):
    _ctx().gate_q8((s["gq"], s["gs"]), (s["uq"], s["us"]), s["xq"], s["xs"], s["h"],
                   act=s["case"]["act"])
    return s["h"]


def _rows_q8(v):
    """f32 rows -> codes and scales."""
    a = v.abs().amax(1)
    code = (v * torch.where(a > 0, 127 / a, 0.0)[:, None]).round().to(torch.int8)
    return code, a / 127


def _plain_embed(s):
    at = s["tok"].long()
    return (s["q"][at].float() * s["scale"][at][:, None]).to(s["out"].dtype)


def _plain_norm(s):
    x, dt = s["x"], s["x"].dtype
    if s["r"] is not None:
        x = (x.float() + s["r"].float()).to(dt)
    v = x.float()
    rstd = 1 / torch.sqrt(v.square().mean(1, keepdim=True) + EPS)
    y = (v * s["w"].float()) * rstd
    code, scale = _rows_q8(y)
    return [x if s["r"] is not None else None, y.to(dt) if s["y"] is not None else None, scale,
            (code.float() * scale[:, None]).half()]


def _plain_quant(s):
    code, scale = _rows_q8(s["x"].float())
    return [scale, (code.float() * scale[:, None]).half()]


def _product(x, w):
    """Integer sums over k of int8 rows, as f32: whole in parts of at most 1024 (2^24 holds 1024 *
    127 * 127), whole numbers beyond."""
    k = x.shape[1]
    if k <= 1024:
        return x.float() @ w.float().T
    parts = -(-k // 1024)
    part = -(-k // parts)
    x = torch.nn.functional.pad(x.float(), (0, parts * part - k)).view(-1, parts, part)
    w = torch.nn.functional.pad(w.float(), (0, parts * part - k)).view(-1, parts, part)
    return torch.bmm(x.transpose(0, 1), w.permute(1, 2, 0)).to(torch.int32).sum(
        0, dtype=torch.int32).float()


def _plain_gemm(s):
    y = (_product(s["xq"], s["wq"]) * s["xs"][:, None]) * s["ws"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(s["y"].dtype)


def _plain_gate(s):
    g = (_product(s["xq"], s["gq"]) * s["xs"][:, None]) * s["gs"]
    u = (_product(s["xq"], s["uq"]) * s["xs"][:, None]) * s["us"]
    t = g
    if s["case"]["act"] == "gelu":
        t = (2 * math.sqrt(2 / math.pi)) * (g + 0.044715 * g * g * g)
    return (g / (1 + torch.exp(-t)) * u).half()


_OWN = {"embed": _own_embed, "norm": _own_norm, "quant": _own_quant, "gemm": _own_gemm,
        "gate": _own_gate}
_PLAIN = {"embed": _plain_embed, "norm": _plain_norm, "quant": _plain_quant, "gemm": _plain_gemm,
          "gate": _plain_gate}


# ---- the definition in 64 bits ----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        at = s["tok"].long()
        return s["q"].double()[at] * s["scale"].double()[at, None]
    if case["op"] in ("norm", "quant"):
        v = s["x"].double()
        if case["op"] == "norm":
            if s["r"] is not None:
                v = v + s["r"].double()
            total = v
            # what is normed is the stream as it is stored
            v = v.to(s["x"].dtype).double()
            v = v * s["w"].double() / torch.sqrt(
                (v * v).sum(1, keepdim=True) / case["k"] + EPS)
        scale = v.abs().max(1).values / 127
        values = torch.round(v / scale[:, None]) * scale[:, None]
        if case["op"] == "quant":
            return [scale, values]
        return [total if s["r"] is not None else None, v if s["y"] is not None else None, scale,
                values]
    x = s["xq"].double() * s["xs"].double()[:, None]
    if case["op"] == "gemm":
        y = torch.matmul(x, (s["wq"].double() * s["ws"].double()[:, None]).T)
        y += s["bias"].double() if s["bias"] is not None else 0
        y += s["res"].double() if s["res"] is not None else 0
        return y
    g = torch.matmul(x, (s["gq"].double() * s["gs"].double()[:, None]).T)
    u = torch.matmul(x, (s["uq"].double() * s["us"].double()[:, None]).T)
    if case["act"] == "silu":
        return g * torch.sigmoid(g) * u
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
