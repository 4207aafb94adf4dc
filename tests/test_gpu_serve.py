"""The batched serving operators on a B200 against plain implementations in 64 bits: ragged
appends into f16 / int8 / 4-bit, contiguous and paged caches, reading them back, attention of
single tokens over 4-bit caches and of prompt chunks over every format, the tokens of a batch of
logits -- and all of them in the order a server runs them, captured and replayed."""
import itertools
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

D, UNIT = 64, 36
FMTS = ("f16", "i8", "q4")


@pytest.fixture(scope="module")
def ctx():
    import p2p_b200
    c = p2p_b200.Context(0)
    yield c
    c.close()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def randh(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float16)


def row_bytes(hkv):
    return (hkv * UNIT + 15) // 16 * 16


# ---- plain 4-bit rows ---------------------------------------------------------------------------
def quant4(x):
    """f16 [..., hkv, 64] -> uint8 [..., row bytes], the rule of the header in torch."""
    xf = x.float()
    lo, hi = xf.amin(-1, keepdim=True), xf.amax(-1, keepdim=True)
    sc = ((hi - lo) / 15).half()
    s = sc.float()
    code = torch.where(s > 0, (xf - lo) / s, torch.zeros_like(xf)).round().clamp(0, 15)
    code = code.to(torch.uint8)
    unit = torch.cat([code[..., 0::2] | (code[..., 1::2] << 4), sc.view(torch.uint8),
                      lo.half().view(torch.uint8)], -1)
    flat = unit.reshape(*x.shape[:-2], -1)
    out = torch.zeros(*flat.shape[:-1], row_bytes(x.shape[-2]), dtype=torch.uint8, device="cuda")
    out[..., :flat.shape[-1]] = flat
    return out


def quant8(x, scale, hkv):
    s = scale.view(hkv, D) if scale.numel() > 1 else scale
    return (x.float() / s).round().clamp(-128, 127).to(torch.int8)


def values64(rows, fmt, hkv, scale):
    """Cache rows -> their values in f64 [..., hkv, 64]."""
    if fmt == "f16":
        return rows.double()
    if fmt == "i8":
        return rows.double() * (scale.double().view(hkv, D) if scale.numel() > 1
                                else scale.double())
    u = rows[..., :hkv * UNIT].reshape(*rows.shape[:-1], hkv, UNIT)
    code = torch.stack([u[..., :32] & 15, u[..., :32] >> 4], -1).flatten(-2).double()
    par = u[..., 32:].contiguous().view(torch.float16).double()
    return code * par[..., :1] + par[..., 1:]


class Cache:
    """A cache of any layout with `lens` rows reserved per sequence, filled with random rows (so
    that what lies behind a sequence is not zero)."""

    def __init__(self, seed, fmt, page, hq, hkv, lens, spare=3, per_channel=True, amp=1.0):
        import p2p_b200
        g = gen(seed)
        self.fmt, self.page, self.hkv, self.hq = fmt, page, hkv, hq
        self.prm = p2p_b200.Params(hq, hkv)
        n = len(lens)
        self.table = self.offsets = None
        if page:
            need = [max(1, -(-m // page)) for m in lens]
            pages = sum(need) + spare
            order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
            self.table = torch.full((n, max(need)), 10**6, dtype=torch.int32, device="cuda")
            at = 0
            for i, b in enumerate(need):
                self.table[i, :b] = order[at:at + b]
                at += b
            lead = (pages, page)
        else:
            starts = np.concatenate([[1], 1 + np.cumsum([m + 2 for m in lens])])
            self.offsets = i32(starts[:-1])
            lead = (int(starts[-1]) + spare,)
        self.ks = self.vs = None
        if fmt == "i8":
            m = hkv * D if per_channel else 1
            self.ks, self.vs = (0.01 + 0.02 * torch.rand(m, generator=g, device="cuda")
                                for _ in range(2))
        k, v = (amp * randh(g, *lead, hkv, D) for _ in range(2))
        self.k, self.v = self.stored(k, self.ks), self.stored(v, self.vs)

    def stored(self, x, scale):
        return {"f16": lambda: x.clone(), "i8": lambda: quant8(x, scale, self.hkv),
                "q4": lambda: quant4(x)}[self.fmt]()

    def kw(self):
        d = {"offsets": self.offsets, "block_table": self.table}
        if self.fmt == "i8":
            d |= {"k_scale": self.ks, "v_scale": self.vs}
        return d

    def at(self, i, pos):
        pos = torch.as_tensor(pos, device="cuda")
        if self.table is not None:
            return self.table[i].long()[pos // self.page], pos % self.page
        return (self.offsets[i].long() + pos,)

    def keys64(self, i, n):
        at = self.at(i, torch.arange(n, device="cuda"))
        return (values64(self.k[at], self.fmt, self.hkv, self.ks),
                values64(self.v[at], self.fmt, self.hkv, self.vs))


def rope_table(n, theta=1e6):
    i = torch.arange(32, dtype=torch.float64, device="cuda")
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * theta ** (-i / 32)
    return torch.cat([a.cos(), a.sin()], 1).float().half()


def starts_of(lens):
    return i32(np.concatenate([[0], np.cumsum(lens)]))


# ---- append and read back -------------------------------------------------------------------------
def prep(ctx, prm, qkv, nw, rope, pos0):
    """QK_PREP of one sequence's rows by the framework's own operator (pinned to the shader)."""
    m = qkv.shape[0]
    q = torch.zeros(m, prm.num_heads * D, dtype=torch.float16, device="cuda")
    k = torch.zeros(pos0 + m, prm.num_kv_heads, D, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    ctx.qk_prep(prm, qkv.contiguous(), nw, rope, q, k, v, pos0=pos0)
    return q, k[pos0:], v[pos0:]


APPENDS = [
    # heads, page, chunk rows, past
    ((32, 8), 16, [1], [0]),
    ((32, 8), 16, [1], [777]),
    ((16, 8), 0, [33, 1, 0, 7], [0, 15, 9, 100]),
    ((16, 2), 64, [130, 3, 64], [0, 63, 1]),
    ((12, 12), 32, [5, 32, 31, 33], [0, 32, 31, 33]),
    ((6, 3), 16, [17, 2], [14, 31]),
    ((8, 1), 0, [40], [3]),
    ((64, 8), 128, [9], [1000]),
    ((8, 8), 16, [1] * 70, list(range(0, 700, 10))),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"{c[0]}-{c[1]}-{len(c[2])}")
def test_append_is_qk_prep_into_any_cache(ctx, fmt, case):
    (hq, hkv), page, rows, past = case
    total = [p + r for p, r in zip(past, rows)]
    c = Cache(11, fmt, page, hq, hkv, total)
    g = gen(12)
    new, pad = sum(rows), 5
    wide = randh(g, new + pad, (hq + 2 * hkv) * D + 24)  # rows with a stride, rows behind the last
    qkv = wide[:, :(hq + 2 * hkv) * D]
    nw = (1 + 0.1 * torch.randn(2 * D, generator=g, device="cuda")).half()
    rope = rope_table(max(total) + 1)
    q_wide = torch.full((new + pad, hq * D + 8), 7.0, dtype=torch.float16, device="cuda")
    want_k, want_v = c.k.clone(), c.v.clone()
    want_q = q_wide.clone()
    at = 0
    for i, (p, r) in enumerate(zip(past, rows)):
        if r:
            q, k, v = prep(ctx, c.prm, qkv[at:at + r], nw, rope, p)
            want_q[at:at + r, :hq * D] = q
            idx = c.at(i, p + torch.arange(r, device="cuda"))
            for pool, x, s in ((want_k, k, c.ks), (want_v, v, c.vs)):
                used = hkv * UNIT if fmt == "q4" else hkv
                pool[(*idx, slice(0, used))] = c.stored(x, s)[:, :used]
        at += r
    ctx.kv_append(c.prm, qkv, nw, rope, c.k, c.v, i32(past), starts_of(rows),
                  max_len=max(total), q_out=q_wide[:, :hq * D], **c.kw())
    ctx.sync()
    assert torch.equal(q_wide, want_q)
    assert torch.equal(c.k, want_k) and torch.equal(c.v, want_v)


@pytest.mark.parametrize("fmt", FMTS)
def test_append_without_norm_or_q(ctx, fmt):
    c = Cache(1, fmt, 16, 8, 2, [40], per_channel=False)
    qkv, rope = randh(gen(2), 40, 12 * D), rope_table(40)
    _, k, v = prep(ctx, c.prm, qkv, None, rope, 0)
    ctx.kv_append(c.prm, qkv, None, rope, c.k, c.v, i32([0]), i32([0, 40]), max_len=40, **c.kw())
    ctx.sync()
    used = slice(0, 2 * UNIT if fmt == "q4" else 2)
    at = c.at(0, torch.arange(40, device="cuda"))
    assert torch.equal(c.k[(*at, used)], c.stored(k, c.ks)[:, used])
    assert torch.equal(c.v[(*at, used)], c.stored(v, c.vs)[:, used])


@pytest.mark.parametrize("rows", [[3, 40], [1500, 700]])
def test_append_with_q_in_place(ctx, rows):
    past = [5, 0]
    c = Cache(15, "f16", 16, 32, 8, [p + r for p, r in zip(past, rows)])
    qkv, rope = randh(gen(16), sum(rows), 48 * D), rope_table(2000)
    nw = randh(gen(17), 2 * D)
    q = torch.zeros(sum(rows), 32 * D, dtype=torch.float16, device="cuda")
    args = (i32(past), starts_of(rows))
    ctx.kv_append(c.prm, qkv, nw, rope, c.k, c.v, *args, max_len=2000, q_out=q, **c.kw())
    ctx.sync()
    k, v = c.k.clone(), c.v.clone()
    same = qkv.clone()
    ctx.kv_append(c.prm, same, nw, rope, c.k, c.v, *args, max_len=2000, q_out=same[:, :32 * D],
                  **c.kw())
    ctx.sync()
    assert torch.equal(same[:, :32 * D], q) and torch.equal(same[:, 32 * D:], qkv[:, 32 * D:])
    assert torch.equal(c.k, k) and torch.equal(c.v, v)


@pytest.mark.parametrize("fmt,page", list(itertools.product(FMTS, (0, 16, 64))))
@pytest.mark.parametrize("heads", [(32, 8), (6, 3), (8, 1), (12, 12)])
def test_read_back(ctx, fmt, page, heads):
    hq, hkv = heads
    first, rows = [0, 3, 17, 40], [1, 0, 50, 33]
    c = Cache(3, fmt, page, hq, hkv, [f + r for f, r in zip(first, rows)])
    n = sum(rows)
    k = torch.full((n + 2, hkv, D), 7.0, dtype=torch.float16, device="cuda")
    v = k.clone()
    ctx.kv_read(c.prm, c.k, c.v, i32(first), starts_of(rows), k, v, max_len=100, **c.kw())
    only = torch.full_like(k, 7.0)
    ctx.kv_read(c.prm, c.k, c.v, i32(first), starts_of(rows), None, only, max_len=100, **c.kw())
    ctx.sync()
    at = 0
    for i, (f, r) in enumerate(zip(first, rows)):
        wk, wv = c.keys64(i, f + r)
        # the product of a code (or int8 value) and the scale and the sum with lo round to f32 once
        # (2^-24) before f16: equal but for ties of f16, which f64 sees the same way
        assert torch.equal(k[at:at + r], wk[f:].float().half())
        assert torch.equal(v[at:at + r], wv[f:].float().half())
        at += r
    assert (k[n:] == 7).all() and (v[n:] == 7).all()
    assert torch.equal(only, v)


@pytest.mark.parametrize("hkv", [1, 2, 3, 5, 8, 16])
def test_quantize_q4(ctx, hkv):
    x = randh(gen(5), 41, hkv, D)
    x[0] = 0
    x[1] = 3.25            # a constant row: scale 0
    x[2, :, ::2] = 65504.0
    x[2, :, 1::2] = -65504.0
    x[3] *= 2.0 ** -20     # subnormal values
    x[4, :, 0] = -0.0
    x[5, :, 1:] = 1.0
    x[5, :, 0] = 1.0 + 2.0 ** -10
    got = ctx.kv_quantize_q4(x)
    ctx.sync()
    assert torch.equal(got, quant4(x))
    # half a step (plus the scale's own rounding over 15 steps) of every value
    val = values64(got, "q4", hkv, None)
    step = got[:, :hkv * UNIT].view(41, hkv, UNIT)[..., 32:34].contiguous().view(
        torch.float16).double()
    err = (val - x.double()).abs()
    span = (x.double().amax(-1, keepdim=True) - x.double().amin(-1, keepdim=True))
    assert (err <= step * 0.5 + span * 2.0 ** -11 + 15 * 2.0 ** -25).all()


# ---- attention ------------------------------------------------------------------------------------
def attention64(c, q, past, rows, chunk):
    """out and how far a kernel may be from it, [rows][hq][64] in f64 on the GPU.

    The bound counts roundings of half a step: the weights to f16 after an exp2 of 2^-10 relative
    error (2^-11 + 2^-10) and, for chunks, the cached values to f16 (2^-11 each: a key's shifts its
    score by up to 2^-11 sum |q k| / 8 and so its weight by that share), and out to f16.  An error
    e of the weights' own shares moves out by at most sum p |v - out| e.  f32 sums of the scores
    (64 products, 2^-24 each, twice for the scale and offset of a 4-bit row) and of the weights
    are below 2^-18 of the magnitudes.

    A 4-bit value is lo + s c.  The decode sums (p s) c with p s rounded to f16 and p lo with p in
    f32, apart from each other: the rounding of a weight by up to 2^-11 then moves out by
    2^-11 w s c = 2^-11 w (v - lo), which |v| does not bound (v may be near 0 with lo far below):
    sum w 2^-11 (v - lo) is added for single tokens over 4-bit caches."""
    outs, tols = [], []
    at = 0
    for i, (p, r) in enumerate(zip(past, rows)):
        if r == 0:
            continue
        k, v = c.keys64(i, p + r)
        grp = c.hq // c.hkv
        k, v = (t.repeat_interleave(grp, 1).permute(1, 0, 2) for t in (k, v))  # [hq][keys][64]
        qi = q[at:at + r].double().view(r, c.hq, D).permute(1, 0, 2)
        at += r
        s = qi @ k.transpose(1, 2) / 8
        mag = qi.abs() @ k.abs().transpose(1, 2) / 8
        hidden = torch.arange(p + r, device="cuda")[None] > \
            (p + torch.arange(r, device="cuda"))[:, None]
        w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
        o = w @ v
        e = 2.0 ** -11 + 2.0 ** -10 + mag * ((2.0 ** -11 if chunk else 0) + 2.0 ** -18)
        # sum w e |v - o| <= sum w e |v| + |o| sum w e
        t = (w * e) @ v.abs() + o.abs() * (w * e).sum(-1, keepdim=True)
        t = t + (w @ v.abs()) * ((2.0 ** -11 if chunk else 0) + 2.0 ** -16)
        t = t + o.abs() * 2.0 ** -11 + 2.0 ** -24
        if c.fmt == "q4" and not chunk:
            lo = v.amin(-1, keepdim=True)  # a row's smallest value has code 0
            t = t + 2.0 ** -11 * (w @ (v - lo))
        outs.append(o.permute(1, 0, 2))
        tols.append(t.permute(1, 0, 2))
    return torch.cat(outs).flatten(1), torch.cat(tols).flatten(1)


def assert_within(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst "
                           f"{float(err.max()):.3e}, {float((err / tol).max()):.2f} of the bound")


DECODES = [
    # heads, page, past
    ((32, 8), 0, [0]),
    ((32, 8), 16, [0, 1, 15, 16, 17, 30, 31, 32, 63, 64, 65]),
    ((32, 8), 0, [1337]),
    ((32, 8), 16, [4099, 5, 700, 0, 2048]),
    ((16, 8), 64, [255, 256, 257]),
    ((16, 2), 16, [333, 40]),
    ((8, 8), 32, [100, 1000]),
    ((64, 8), 16, [513, 3]),
    ((12, 12), 16, [200, 31]),
    ((6, 3), 0, [77, 500]),
    ((8, 1), 128, [1500]),
    ((24, 12), 16, [129]),
    ((32, 32), 64, [300, 64]),
    ((40, 20), 0, [90, 21]),
    ((32, 8), 4096, [9000]),
    ((32, 8), 16, [20000]),
    ((16, 8), 16, [(37 * i) % 400 for i in range(200)]),
]


@pytest.mark.parametrize("case", DECODES, ids=lambda c: f"{c[0]}-{c[1]}-{len(c[2])}x{max(c[2])}")
def test_decode_q4(ctx, case):
    (hq, hkv), page, past = case
    n = len(past)
    c = Cache(21, "q4", page, hq, hkv, [p + 1 for p in past])
    q = randh(gen(22), n, hq * D + 8)[:, :hq * D]
    out = torch.full((n + 1, hq * D + 16), 7.0, dtype=torch.float16, device="cuda")
    ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32(past), out[:, :hq * D],
                       max_past=max(past), fused_prep=False, **c.kw())
    ctx.sync()
    want, tol = attention64(c, q, past, [1] * n, False)
    assert_within(out[:n, :hq * D], want, tol)
    assert (out[n:] == 7).all() and (out[:, hq * D:] == 7).all()


@pytest.mark.parametrize("amp", [1e-4, 30.0, 2000.0])
def test_decode_q4_ranges(ctx, amp):
    """Caches of tiny and of large values: the scales' range."""
    c = Cache(23, "q4", 16, 16, 4, [600, 50], amp=amp)
    q = randh(gen(24), 2, 16 * D) * (0.05 if amp > 1 else 1.0)
    out = torch.zeros_like(q)
    ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32([599, 49]), out, max_past=599,
                       fused_prep=False, **c.kw())
    ctx.sync()
    want, tol = attention64(c, q, [599, 49], [1, 1], False)
    # f16 weights times the rows' scales have an absolute floor of 2^-27 in a code's weight: 15
    # codes of 2^-27 for each key whose weight counts
    assert_within(out, want, tol + 15 * 2.0 ** -27 * 600 ** 0.5)


@pytest.mark.parametrize("case", [c for c in DECODES if len(c[2]) < 20],
                         ids=lambda c: f"{c[0]}-{c[1]}-{len(c[2])}x{max(c[2])}")
def test_decode_q4_fused_is_append_then_attend(ctx, case):
    (hq, hkv), page, past = case
    n = len(past)
    a = Cache(25, "q4", page, hq, hkv, [p + 1 for p in past])
    b = Cache(25, "q4", page, hq, hkv, [p + 1 for p in past])
    g = gen(26)
    qkv = randh(g, n, (hq + 2 * hkv) * D)
    nw = (1 + 0.1 * torch.randn(2 * D, generator=g, device="cuda")).half()
    rope = rope_table(max(past) + 1)
    q, out, out2 = (torch.zeros(n, hq * D, dtype=torch.float16, device="cuda") for _ in range(3))
    ctx.kv_append(a.prm, qkv, nw, rope, a.k, a.v, i32(past), i32(range(n + 1)),
                  max_len=max(past) + 1, q_out=q, **a.kw())
    ctx.attn_decode_kv(a.prm, q, None, None, a.k, a.v, i32(past), out, max_past=max(past),
                       fused_prep=False, **a.kw())
    ctx.attn_decode_kv(b.prm, qkv, nw, rope, b.k, b.v, i32(past), out2, max_past=max(past),
                       fused_prep=True, **b.kw())
    ctx.sync()
    assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    assert torch.equal(out, out2)
    want, tol = attention64(a, q, past, [1] * n, False)
    assert_within(out2, want, tol)


CHUNKS = [
    # heads, page, rows, past
    ((32, 8), 16, [1], [0]),
    ((32, 8), 16, [5, 1, 0, 2, 33], [40, 0, 7, 1000, 64]),
    ((32, 8), 64, [129], [0]),
    ((32, 8), 16, [128, 127, 31, 32], [0, 1, 97, 128]),
    ((32, 8), 16, [300], [777]),
    ((16, 8), 0, [64, 63, 65, 200], [0, 65, 63, 10]),
    ((16, 2), 32, [40, 3], [500, 2000]),
    ((8, 8), 16, [150, 6], [33, 128]),
    ((12, 12), 64, [257], [0]),
    ((6, 3), 0, [77], [130]),
    ((8, 1), 128, [50, 16], [0, 300]),
    ((64, 8), 16, [17, 48], [100, 15]),
    ((32, 8), 16, [3], [9000]),
    ((16, 8), 16, [4] * 40, [(53 * i) % 300 for i in range(40)]),
    ((24, 12), 16, [1024], [100]),
    # more items than the equal parts are for: a CTA each
    ((64, 8), 64, [2400, 5, 77], [3, 0, 500]),
    ((16, 16), 16, [5] * 48, [(31 * i) % 500 for i in range(48)]),
]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: f"{c[0]}-{c[1]}-{len(c[2])}x{max(c[2])}")
def test_chunk(ctx, fmt, case):
    (hq, hkv), page, rows, past = case
    total = [p + r for p, r in zip(past, rows)]
    c = Cache(31, fmt, page, hq, hkv, total, per_channel=page != 64)
    n = sum(rows)
    q = randh(gen(32), n + 3, hq * D + 16)[:, :hq * D]
    out = torch.full((n + 3, hq * D + 8), 7.0, dtype=torch.float16, device="cuda")
    ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32(past), starts_of(rows), out[:, :hq * D],
                      max_len=max(total), **c.kw())
    ctx.sync()
    want, tol = attention64(c, q, past, rows, True)
    assert_within(out[:n, :hq * D], want, tol)
    assert (out[n:] == 7).all() and (out[:, hq * D:] == 7).all()


def test_rows_behind_a_sequence_do_not_reach_it(ctx):
    """NaN and infinities behind the sequences' ends (f16 caches) and in their pages' tails."""
    for page in (0, 64):
        c = Cache(33, "f16", page, 8, 4, [70, 5])
        wipe_k, wipe_v = torch.full_like(c.k, math.nan), torch.full_like(c.v, math.inf)
        for i, m in enumerate([70, 5]):
            at = c.at(i, torch.arange(m, device="cuda"))
            wipe_k[at], wipe_v[at] = c.k[at], c.v[at]
        c.k, c.v = wipe_k, wipe_v
        q = randh(gen(34), 12, 8 * D)
        out = torch.zeros_like(q)
        ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32([60, 3]), i32([0, 10, 12]), out, max_len=70,
                          **c.kw())
        ctx.sync()
        want, tol = attention64(c, q, [60, 3], [10, 2], True)
        assert_within(out, want, tol)


@pytest.mark.parametrize("fmt", ["f16", "q4"])
@pytest.mark.parametrize("page", [0, 16, 256])
@pytest.mark.parametrize("case", [
    # heads, past, rows, the tokens whose V overflowed (sequence, row of the chunk)
    ((32, 8), [0, 130, 40], [70, 5, 300], [(0, 69), (1, 3), (2, 100), (2, 101), (2, 270)]),
    ((16, 16), [500], [400], [(0, 0), (0, 255), (0, 256), (0, 399)]),
    ((8, 1), [5000], [33], [(0, 17)]),
    # more items than the equal parts are for: a CTA each
    ((64, 8), [3, 0], [2400, 77], [(0, 1200), (0, 2399), (1, 40)]),
], ids=lambda c: f"{c[0]}-{len(c[2])}x{max(c[2])}")
def test_values_that_overflowed_reach_no_earlier_token(ctx, fmt, page, case):
    """A token's infinite or NaN K and V: the rows in front of it are as without (within the bound
    of a chunk), those that see an infinity of V get it in its dims (f16: dim 3 inf, dim 10 NaN,
    the rest as without; 4 bits: the whole head), and those that see a NaN K are NaN."""
    (hq, hkv), past, rows, odd = case
    c = Cache(35, fmt, page, hq, hkv, [p + r for p, r in zip(past, rows)])
    n = sum(rows)
    q, first = randh(gen(36), n, hq * D), [sum(rows[:i]) for i in range(len(rows))]

    want, tol = (t.view(n, hq, D) for t in attention64(c, q, past, rows, True))

    def check(what):
        out = torch.full_like(q, math.nan)
        ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32(past), starts_of(rows), out, max_len=6000,
                          **c.kw())
        ctx.sync()
        got = out.view(n, hq, D)
        live = want.isfinite()
        assert same_bits(got.double()[~live], want[~live]), what
        assert_within(got[live], want[live], tol[live], what)
    check("clean")
    grp, last = hq // hkv, hkv - 1
    for i, r in odd:
        at = tuple(x if torch.is_tensor(x) and x.dim() == 0 else torch.as_tensor(x, device="cuda")
                   for x in c.at(i, past[i] + r))
        sees = want[first[i] + r:first[i] + rows[i]]
        if fmt == "f16":
            c.v[(*at, 0, 3)], c.v[(*at, 0, 10)] = math.inf, math.nan
            sees[:, :grp, 3], sees[:, :grp, 10] = math.inf, math.nan
            c.v[(*at, last, 63)] = -math.inf
            sees[:, last * grp:, 63] = -math.inf
        else:
            unit = c.v[at]
            unit[34:36] = torch.tensor([math.inf], dtype=torch.float16,
                                       device="cuda").view(torch.uint8)
            c.v[at] = unit
            sees[:, :grp] = math.inf
    check("V")
    i, r = odd[-1]
    at = tuple(torch.as_tensor(x, device="cuda") for x in c.at(i, past[i] + r))
    row = c.k[at]
    if fmt == "f16":
        row[0] = math.nan
    else:
        row[32:34] = torch.tensor([math.nan], dtype=torch.float16, device="cuda").view(torch.uint8)
    c.k[at] = row
    want[first[i] + r:first[i] + rows[i], :grp] = math.nan
    check("K")


# ---- refusals on the device -------------------------------------------------------------------------
@pytest.mark.parametrize("op", ["append", "read", "chunk", "decode", "fused"])
@pytest.mark.parametrize("page", [0, 16])
def test_bad_sequences_are_skipped(ctx, op, page):
    """Sequence 1 does not fit (too long, then a bad page or offset): it is left alone and
    reported; its neighbours are computed."""
    import p2p_b200
    hq, hkv = 8, 2
    rows = [1, 1, 1] if op in ("decode", "fused") else [20, 9, 3]
    past = [5, 40, 33]
    total = [p + r for p, r in zip(past, rows)]
    for fault in ("length", "place"):
        c = Cache(41, "q4", page, hq, hkv, total)
        good_k, good_v = c.k.clone(), c.v.clone()
        p = list(past)
        if fault == "length":
            p[1] = 60 if op != "read" else -1
        elif page:
            c.table[1, 2] = len(c.k)  # the page behind the pool
        else:
            c.offsets[1] = len(c.k) - 10
        max_len = 59
        g = gen(42)
        n = sum(rows)
        qkv = randh(g, n, (hq + 2 * hkv) * D)
        rope = rope_table(max_len)
        out = torch.full((n, hq * D), 7.0, dtype=torch.float16, device="cuda")
        with pytest.raises(p2p_b200.KvFullError):
            if op == "append":
                ctx.kv_append(c.prm, qkv, None, rope, c.k, c.v, i32(p), starts_of(rows),
                              max_len=max_len, q_out=out, **c.kw())
            elif op == "read":
                k = torch.full((n, hkv, D), 7.0, dtype=torch.float16, device="cuda")
                ctx.kv_read(c.prm, c.k, c.v, i32(p), starts_of(rows), k, None, max_len=max_len,
                            **c.kw())
            elif op == "chunk":
                ctx.attn_chunk_kv(c.prm, qkv[:, :hq * D].contiguous(), c.k, c.v, i32(p),
                                  starts_of(rows), out, max_len=max_len, **c.kw())
            else:
                ctx.attn_decode_kv(c.prm, qkv, None, rope, c.k, c.v, i32(p), out,
                                   max_past=47, fused_prep=op == "fused", **c.kw())
            ctx.sync()
        ctx.sync()  # reported once
        a, b = rows[0], rows[0] + rows[1]
        if op == "read":
            assert torch.equal(k[:a], c.keys64(0, total[0])[0][p[0]:].float().half())
            assert torch.equal(k[b:], c.keys64(2, total[2])[0][p[2]:].float().half())
            # paged: rows 40 .. 47 of the bad page are skipped, row 48 is in the next page
            if fault == "length" or not page:
                assert (k[a:b] == 7).all()
            else:
                assert (k[a:b - 1] == 7).all()
            continue
        if op in ("append", "fused"):
            for i in (0, 2):
                at = c.at(i, p[i] + torch.arange(rows[i], device="cuda"))
                assert not torch.equal(c.k[at], good_k[at])
                c.k[at], c.v[at] = good_k[at], good_v[at]
            if op == "append" and page and fault == "place":
                at = c.at(1, torch.tensor([48], device="cuda"))  # its last row is in a good page
                c.k[at], c.v[at] = good_k[at], good_v[at]
            assert torch.equal(c.k, good_k) and torch.equal(c.v, good_v)
        if op == "append":
            assert not (out[:a] == 7).any() and not (out[b:] == 7).any()
            assert (out[a:b - 1] == 7).all()
            continue
        assert (out[a:b] == 7).all()
        if op != "fused":
            q = qkv[:, :hq * D]
            for i, s in ((0, slice(0, a)), (2, slice(b, n))):
                one = Cache(41, "q4", page, hq, hkv, total)
                one.k, one.v = c.k, c.v
                if page:
                    one.table = c.table[i:i + 1]
                else:
                    one.offsets = c.offsets[i:i + 1]
                want, tol = attention64(one, q[s], [p[i]], [rows[i]], True)
                assert_within(out[s], want, tol, f"sequence {i}")


def test_host_refusals(ctx):
    import p2p_b200
    c = Cache(43, "q4", 16, 8, 2, [40])
    q = randh(gen(44), 4, 12 * D)
    out = torch.zeros(4, 8 * D, dtype=torch.float16, device="cuda")
    rope = rope_table(40)
    E = p2p_b200.P2PError
    ok = dict(max_len=40, **c.kw())
    rs, z = i32([0, 4]), i32([0])

    def refused(fn, *a, **k):
        with pytest.raises(E) as e:
            fn(*a, **k)
        assert e.value.status in (1, 7), e.value
    refused(ctx.attn_chunk_kv, c.prm, q.float(), c.k, c.v, z, rs, out, **ok)
    refused(ctx.attn_chunk_kv, c.prm, q[:, :64], c.k, c.v, z, rs, out, **ok)
    refused(ctx.attn_chunk_kv, c.prm, q, c.k, c.v[1:], z, rs, out, **ok)
    refused(ctx.attn_chunk_kv, c.prm, q, c.k, c.v, z.long(), rs, out, **ok)
    refused(ctx.attn_chunk_kv, c.prm, q, c.k, c.v, z, z, out, **ok)             # row_start short
    refused(ctx.attn_chunk_kv, c.prm, q, c.k, c.v, z, rs, out[:2], **ok)
    refused(ctx.attn_chunk_kv, c.prm, q, c.k, c.v, z, rs, out, max_len=-1, **c.kw())
    refused(ctx.attn_chunk_kv, c.prm, q, c.k, c.v, z, rs, out, max_len=40, offsets=z)
    shifted = torch.zeros(4 * 12 * D + 8, dtype=torch.float16, device="cuda")[1:]
    refused(ctx.attn_chunk_kv, c.prm, shifted[:4 * 12 * D].view(4, 12 * D), c.k, c.v, z, rs, out,
            **ok)
    refused(ctx.attn_chunk_kv, p2p_b200.Params(6, 2), q, c.k, c.v, z, rs, out, **ok)  # group 3
    refused(ctx.attn_chunk_kv, p2p_b200.Params(8, 2, dtype=torch.float32), q, c.k, c.v, z, rs, out,
            **ok)
    refused(ctx.kv_append, c.prm, q, None, rope[:20], c.k, c.v, z, rs, **ok)    # rope too short
    refused(ctx.kv_append, c.prm, q, None, ctx.rope_table(39), c.k, c.v, z, rs, **ok)
    refused(ctx.kv_append, c.prm, q, rope[0], rope, c.k, c.v, z, rs, **ok)      # 64 norm weights
    refused(ctx.kv_read, c.prm, c.k, c.v, z, rs, None, None, **ok)
    refused(ctx.attn_decode_kv, c.prm, q, None, rope, c.k, c.v, z, out, max_past=40 + 16, **c.kw())
    refused(ctx.kv_quantize_q4, q)
    p = Cache(43, "q4", 0, 8, 2, [40])
    refused(ctx.attn_chunk_kv, p.prm, q, p.k, p.v, z, rs, out, max_len=40)      # no offsets
    t8 = Cache(43, "i8", 16, 8, 2, [40])
    refused(ctx.attn_chunk_kv, t8.prm, q, t8.k, t8.v, z, rs, out, max_len=40, block_table=t8.table)


def test_empty_calls(ctx):
    c = Cache(45, "q4", 16, 8, 2, [40])
    none = torch.zeros(0, 12 * D, dtype=torch.float16, device="cuda")
    q = randh(gen(1), 3, 12 * D)
    out = torch.full((3, 8 * D), 7.0, dtype=torch.float16, device="cuda")
    empty, rope = i32([]), rope_table(40)
    ctx.attn_chunk_kv(c.prm, none, c.k, c.v, i32([0]), i32([0, 0]), out, max_len=40, **c.kw())
    ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32([0]), i32([0, 0]), out, max_len=40, **c.kw())
    ctx.attn_chunk_kv(c.prm, q, c.k, c.v, empty, i32([0]), out, max_len=40, **c.kw())
    ctx.kv_append(c.prm, q, None, rope, c.k, c.v, i32([0]), i32([0, 0]), max_len=40, q_out=out,
                  **c.kw())
    ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, empty, out, max_past=39, fused_prep=False,
                       **c.kw())
    ctx.sync()
    assert (out == 7).all()


# ---- logits -----------------------------------------------------------------------------------------
def plain_logits(x, hist, hist_len, prompt_len, rep, pres, freq, bias, mask, dt):
    """One rounding per operation in f32 (numpy), as the header states it."""
    y = x.float().cpu().numpy().copy()
    n, vocab = y.shape
    for i in range(n):
        h = hist[i][:hist_len[i]] if hist is not None else np.zeros(0, np.int64)
        made = h[min(max(prompt_len[i], 0), len(h)):] if prompt_len is not None else h
        inside = h[(h >= 0) & (h < vocab)]
        made = made[(made >= 0) & (made < vocab)]
        line = y[i]
        s = np.unique(inside)
        if rep is not None:
            line[s] = np.where(line[s] > 0, line[s] / rep[i], line[s] * rep[i])
        m, c = np.unique(made, return_counts=True)
        f = np.float32(freq[i]) if freq is not None else np.float32(0)
        p = np.float32(pres[i]) if pres is not None else np.float32(0)
        line[m] = (line[m] - f * c.astype(np.float32)) - p
        if bias is not None:
            for t, b in bias[i]:
                if 0 <= t < vocab:
                    line[t] = line[t] + np.float32(b)
        if mask is not None:
            line[~mask[i]] = -np.inf
    out = torch.from_numpy(y).to(dt).cuda()
    toks = []
    for i in range(n):
        line = out[i].float().cpu().numpy()
        live = np.where(np.isnan(line), -np.inf, line)
        toks.append(int(np.argmax(live)) if live.max() > -np.inf else -1)
    return out, toks


def same_bits(a, b):
    """Equal values, NaN where NaN."""
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


LOGITS = [
    # rows, vocab, history, biases, mask
    (1, 1, 3, 1, True), (1, 7, 0, 0, False), (2, 31, 5, 3, True), (3, 33, 60, 5, True),
    (1, 1000, 100, 0, False), (5, 1025, 300, 20, True), (4, 4099, 1000, 300, True),
    (3, 65536, 2000, 50, True), (2, 131071, 4000, 10, True), (1, 262144, 50, 0, True),
    (70, 513, 40, 4, True), (1, 400000, 10, 5, True),
    # long histories; more biases than threads
    (2, 900, 4097, 2000, True), (3, 65536, 9000, 700, True), (2, 131071, 20000, 5000, False),
    (1, 262144, 5000, 0, False), (1, 400000, 4097, 1, True), (2, 30, 6000, 600, False),
]


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
@pytest.mark.parametrize("case", LOGITS, ids=lambda c: f"{c[0]}x{c[1]}")
def test_logits_pick(ctx, dt, case):
    n, vocab, cap, nb, with_mask = case
    rng = np.random.default_rng(n * vocab)
    g = gen(vocab)
    for strided in (False, True):
        wide = (3 * torch.randn(n, vocab + (5 if strided else 0), generator=g,
                                device="cuda")).to(dt)
        x = wide[:, :vocab]
        x[0, vocab // 2] = math.nan
        x[-1, vocab // 3] = math.inf if vocab > 100 else 1.0
        out = torch.full((n, vocab + 3), 7.0, dtype=dt, device="cuda")
        hist = rng.integers(0, vocab, (n, cap + 2))
        hist[:, ::3] = hist[:, :1]           # one token many times
        hist[:, 1::7] = -1                   # not a token
        hist[:, 2::7] = vocab
        lens = np.minimum(rng.integers(0, cap + 1, n) + cap // 2, cap)
        lens[-1] = 0
        plen = lens // 2
        rep, pres, freq = (1 + rng.random(n), rng.random(n), rng.random(n) / 3)
        rep, pres, freq = (a.astype(np.float32) for a in (rep, pres, freq))
        rep[0] = 0.5
        bias = [[(int(t), float(b)) for t, b in zip(rng.integers(-1, vocab + 1, nb),
                                                    rng.standard_normal(nb) * 4)]
                for _ in range(n)]
        if nb > 2:
            bias[0][2] = (bias[0][0][0], 1.25)  # the same token twice
        mask = rng.random((n, vocab)) < 0.5 if with_mask else None
        kw = {}
        if nb:
            kw["bias_start"] = starts_of([len(b) for b in bias])
            kw["bias_tok"] = i32(t for b in bias for t, _ in b)
            kw["bias_val"] = torch.tensor([v for b in bias for _, v in b], device="cuda")
        if mask is not None:
            words = (vocab + 31) // 32
            bits = np.zeros((n, words * 32), bool)
            bits[:, :vocab] = mask
            packed = np.packbits(bits, axis=1, bitorder="little").view(np.int32)
            kw["mask"] = torch.from_numpy(packed.copy()).cuda()
        tok = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        want, toks = plain_logits(x, hist, lens, plen, rep, pres, freq, bias if nb else None, mask,
                                  dt)
        h = dev(hist.astype(np.int32))
        kw |= dict(hist=h, hist_len=i32(lens), prompt_len=i32(plen), repetition=dev(rep),
                   presence=dev(pres), frequency=dev(freq))
        ctx.logits_pick(x, tok, out=out[:, :vocab], **kw)
        ctx.sync()
        assert tok.tolist() == toks + [-7]
        assert same_bits(out[:, :vocab], want)
        assert (out[:, vocab:] == 7).all()
        tok2 = torch.zeros_like(tok)
        ctx.logits_pick(x, tok2, **kw)       # without an output, and in place
        keep = wide.clone()
        ctx.logits_pick(x, tok2, out=x, **kw)
        ctx.sync()
        assert tok2.tolist()[:n] == toks and same_bits(x, want)
        assert torch.equal(wide[:, vocab:], keep[:, vocab:])


def test_logits_empty_lists(ctx):
    x, tok = randh(gen(8), 2, 300), torch.zeros(2, dtype=torch.int32, device="cuda")
    none, f = i32([]), torch.zeros(0, device="cuda")
    out = torch.zeros_like(x)
    ctx.logits_pick(x, tok, out=out, bias_start=i32([0, 0, 0]), bias_tok=none, bias_val=f)
    ctx.logits_pick(x[:0], tok)
    ctx.sync()
    assert torch.equal(out, x)
    assert tok.tolist() == [int(np.argmax(r)) for r in x.float().cpu().numpy()]


def test_logits_without_anything_is_argmax(ctx):
    x = randh(gen(3), 9, 5000)
    x[0, 77] = x[0, 4000] = 9.0     # a tie: the lowest index
    x[1] = -math.inf                # nothing left
    x[2] = math.nan
    x[3, 1:] = -math.inf
    x[4] = 0.0
    x[4, 6] = -0.0                  # equal to +0: index 0
    tok = torch.zeros(9, dtype=torch.int32, device="cuda")
    ctx.logits_pick(x, tok)
    ctx.sync()
    got = tok.tolist()
    assert got[:5] == [77, -1, -1, 0, 0]
    for i in range(5, 9):
        assert got[i] == int(np.argmax(x[i].float().cpu().numpy()))


def test_logits_masks_that_leave_one_or_none(ctx):
    n, vocab = 3, 70000
    x = randh(gen(4), n, vocab)
    mask = torch.zeros(n, (vocab + 31) // 32, dtype=torch.int32, device="cuda")
    mask[1, 69999 // 32] = 1 << (69999 % 32)
    mask[2] = -1
    tok = torch.zeros(n, dtype=torch.int32, device="cuda")
    hist = torch.zeros(n, 4, dtype=torch.int32, device="cuda")
    hist_len, past = i32([1, 1, 4]), i32([10, 20, 30])
    import p2p_b200
    ctx.logits_pick(x, tok, mask=mask, hist=hist, hist_len=hist_len, past=past, advance=True)
    with pytest.raises(p2p_b200.P2PError) as e:  # row 2's history is full
        ctx.sync()
    assert e.value.status == 1
    best = int(np.argmax(x[2].float().cpu().numpy()))
    assert tok.tolist() == [-1, 69999, best]
    assert hist_len.tolist() == [1, 2, 4] and past.tolist() == [10, 21, 30]
    assert hist.tolist() == [[0] * 4, [0, 69999, 0, 0], [0] * 4]


def test_logits_advance_replays(ctx):
    """A captured pick that feeds on its own history: each replay picks the next token."""
    vocab, steps = 3001, 12
    x = randh(gen(6), 2, vocab)
    hist = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    hist_len, past = i32([0, 3]), i32([0, 100])
    hist[1, :3] = torch.tensor([1, 2, 2], dtype=torch.int32)
    start_hist = hist.cpu().numpy().copy()
    pres = torch.tensor([100.0, 100.0], device="cuda")  # a picked token never comes again
    tok = torch.zeros(2, dtype=torch.int32, device="cuda")
    kw = dict(hist=hist, hist_len=hist_len, past=past, presence=pres, advance=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.logits_pick(x, tok, **kw)
    for _ in range(steps):
        graph.replay()
    ctx.sync()
    assert hist_len.tolist() == [steps, 3 + steps] and past.tolist() == [steps, 100 + steps]
    h, lens = start_hist, [0, 3]
    for _ in range(steps):
        _, toks = plain_logits(x, h, lens, None, None, [100.0] * 2, None, None, None, x.dtype)
        for i, t in enumerate(toks):
            h[i, lens[i]] = t
            lens[i] += 1
    assert np.array_equal(h, hist.cpu().numpy())


def test_logits_refusals(ctx):
    import p2p_b200
    x = randh(gen(7), 2, 100)
    tok = torch.zeros(2, dtype=torch.int32, device="cuda")
    f = torch.ones(2, device="cuda")
    h = torch.zeros(2, 5, dtype=torch.int32, device="cuda")

    def refused(*a, **k):
        with pytest.raises(p2p_b200.P2PError) as e:
            ctx.logits_pick(*a, **k)
        assert e.value.status in (1, 7)
    refused(x.double(), tok)
    refused(x[0], tok)
    refused(x, tok[:1])
    refused(x, tok.long())
    refused(x, tok, out=x[:, :50])
    refused(x, tok, out=x.float())
    refused(x, tok, hist=h)
    refused(x, tok, hist_len=tok)
    refused(x, tok, hist=h[:, :0], hist_len=tok)
    refused(x, tok, prompt_len=tok)
    refused(x, tok, repetition=f.half())
    refused(x, tok, presence=f[:1])
    refused(x, tok, bias_start=tok, bias_tok=tok, bias_val=f)        # needs rows + 1 starts
    refused(x, tok, bias_start=h[0], bias_tok=tok)
    refused(x, tok, mask=h[:, :3])
    refused(torch.zeros(1, 400001, dtype=torch.float16, device="cuda"), tok)


# ---- together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FMTS)
def test_a_server_run(ctx, fmt):
    """Prompts of a batch appended and attended in chunks, then captured decode steps (append,
    attention, logits, token), replayed: every row agrees with the 64-bit attention over the
    cache, and the tokens with the plain picks."""
    hq, hkv, vocab, steps = 16, 4, 999, 6
    prompts = [37, 1, 130]
    n = len(prompts)
    total = [p + steps + 1 for p in prompts]
    c = Cache(51, fmt, 16, hq, hkv, total, amp=0.0)
    prm, g = c.prm, gen(52)
    nw = (1 + 0.1 * torch.randn(2 * D, generator=g, device="cuda")).half()
    rope = rope_table(max(total))
    emb = randh(g, vocab, (hq + 2 * hkv) * D)      # a token's qkv row
    head = randh(g, hq * D, vocab) * 0.05
    toks = torch.randint(0, vocab, (sum(prompts),), generator=g, device="cuda")
    ml = max(total)
    # prompts in two ragged chunks
    cut = [p // 2 for p in prompts]
    rows_of = np.concatenate([[0], np.cumsum(prompts)])
    for part in range(2):
        past = [0] * n if part == 0 else cut
        rows = cut if part == 0 else [p - h for p, h in zip(prompts, cut)]
        idx = np.concatenate([np.arange(rows_of[i] + past[i], rows_of[i] + past[i] + rows[i])
                              for i in range(n)]).astype(np.int64)
        qkv = emb[toks[torch.from_numpy(idx).cuda()]]
        q, out = (torch.zeros(len(idx), hq * D, dtype=torch.float16, device="cuda")
                  for _ in range(2))
        rs, pt = starts_of(rows), i32(past)
        ctx.kv_append(prm, qkv, nw, rope, c.k, c.v, pt, rs, max_len=ml, q_out=q, **c.kw())
        ctx.attn_chunk_kv(prm, q, c.k, c.v, pt, rs, out, max_len=ml, **c.kw())
        ctx.sync()
        want, tol = attention64(c, q, past, rows, True)
        assert_within(out, want, tol)
    last = out[torch.tensor(np.cumsum(rows) - 1).cuda()]
    hist = torch.full((n, max(prompts) + steps + 2), -1, dtype=torch.int32, device="cuda")
    for i in range(n):
        hist[i, :prompts[i]] = toks[rows_of[i]:rows_of[i + 1]].int()
    hist_len, plen, past = i32(prompts), i32(prompts), i32([p - 1 for p in prompts])
    kw = dict(hist=hist, hist_len=hist_len, prompt_len=plen,
              repetition=torch.full((n,), 1.3, device="cuda"),
              presence=torch.full((n,), 0.5, device="cuda"),
              frequency=torch.full((n,), 0.25, device="cuda"), past=past, advance=True)
    tok = torch.zeros(n, dtype=torch.int32, device="cuda")
    logits = last @ head
    first = plain_logits(logits, hist.cpu().numpy(), prompts, prompts, [np.float32(1.3)] * n,
                         [0.5] * n, [0.25] * n, None, None, torch.float16)[1]
    ctx.logits_pick(logits, tok, **kw)
    ctx.sync()
    assert tok.tolist() == first
    # decode: past now points at the picked token's position
    q, out = (torch.zeros(n, hq * D, dtype=torch.float16, device="cuda") for _ in range(2))
    one = i32(range(n + 1))

    def step():
        qkv = emb[tok.long()]
        if fmt == "q4":
            ctx.attn_decode_kv(prm, qkv, nw, rope, c.k, c.v, past, out, max_past=ml - 1, **c.kw())
        else:
            ctx.kv_append(prm, qkv, nw, rope, c.k, c.v, past, one, max_len=ml, q_out=q, **c.kw())
            ctx.attn_chunk_kv(prm, q, c.k, c.v, past, one, out, max_len=ml, **c.kw())
        ctx.logits_pick(out @ head, tok, **kw)

    keep = [t.clone() for t in (c.k, c.v, hist, hist_len, past, tok)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # a warm-up outside the capture: workspaces are made here
    torch.cuda.current_stream().wait_stream(side)
    for t, k in zip((c.k, c.v, hist, hist_len, past, tok), keep):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    state = (hist.cpu().numpy().copy(), list(prompts))
    state[0][range(n), prompts] = first
    lens = [p + 1 for p in prompts]
    for s in range(steps - 1):
        before = tok.clone()
        graph.replay()
        ctx.sync()
        pos = [p + s for p in prompts]
        qs = []
        for i in range(n):
            qs.append(prep(ctx, prm, emb[before[i].long()][None], nw, rope, pos[i])[0])
        want, tol = attention64(c, torch.cat(qs), pos, [1] * n, fmt != "q4")
        assert_within(out, want, tol, f"step {s}")
        ref = plain_logits(out @ head, state[0], lens, prompts, [np.float32(1.3)] * n, [0.5] * n,
                           [0.25] * n, None, None, torch.float16)[1]
        assert tok.tolist() == ref
        for i, t in enumerate(ref):
            state[0][i, lens[i]] = t
            lens[i] += 1
    assert np.array_equal(state[0], hist.cpu().numpy())
    assert past.tolist() == [p + steps - 1 for p in prompts]
    del graph


@pytest.mark.parametrize("op", ["decode", "chunk"])
def test_two_graphs_of_different_sizes_share_a_context(ctx, op):
    """A small call captured, a larger one captured and run, the small one replayed."""
    graphs, checks = [], []
    for seed, past in ((61, [300, 20]), (62, [5000, 100, 2000, 77])):
        c = Cache(seed, "q4", 16, 32, 8, [p + 1 for p in past])
        n = len(past)
        q = randh(gen(seed), n, 32 * D)
        out = torch.zeros_like(q)
        p, rs = i32(past), i32(range(n + 1))

        def call(c=c, q=q, out=out, p=p, rs=rs, top=max(past)):
            if op == "decode":
                ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, p, out, max_past=top,
                                   fused_prep=False, **c.kw())
            else:
                ctx.attn_chunk_kv(c.prm, q, c.k, c.v, p, rs, out, max_len=top + 1, **c.kw())
        call()
        ctx.sync()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        graphs.append((g, call))
        checks.append((c, q, out, past, p, rs))
    for order in ((0, 1), (1, 0), (0, 0)):
        for k in order:
            checks[k][2].zero_()
            graphs[k][0].replay()
        ctx.sync()
        for k in order:
            c, q, out, past, _, _ = checks[k]
            want, tol = attention64(c, q, past, [1] * len(past), op == "chunk")
            assert_within(out, want, tol)
    graphs.clear()


@pytest.mark.parametrize("op", ["decode", "chunk"])
def test_the_workspace_is_made_outside_captures_and_may_not_fit(op):
    import p2p_b200
    past = [300, 20]
    c = Cache(63, "q4", 16, 16, 4, [p + 1 for p in past])
    q = randh(gen(64), 2, 16 * D)
    out = torch.full_like(q, 7.0)
    p, rs = i32(past), i32([0, 1, 2])
    fresh = p2p_b200.Context(0)
    try:
        def call():
            if op == "decode":
                fresh.attn_decode_kv(c.prm, q, None, None, c.k, c.v, p, out, max_past=300,
                                     fused_prep=False, **c.kw())
            else:
                fresh.attn_chunk_kv(c.prm, q, c.k, c.v, p, rs, out, max_len=301, **c.kw())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.fill_(7.0)
            with pytest.raises(p2p_b200.P2PError) as e:
                call()
        assert e.value.status == p2p_b200.P2P_ERR_INVALID_ARG
        g.replay()
        torch.cuda.synchronize()
        assert (out == 7).all()
        try:
            p2p_b200.lib.p2p_debug_set_alloc_limit(0)
            with pytest.raises(p2p_b200.P2PError) as e:
                call()
            assert e.value.status == p2p_b200.P2P_ERR_OOM
        finally:
            p2p_b200.lib.p2p_debug_set_alloc_limit(-1)
        call()
        fresh.sync()
        want, tol = attention64(c, q, past, [1, 1], op == "chunk")
        assert_within(out, want, tol)
    finally:
        fresh.close()


@pytest.mark.parametrize("op", ["decode", "chunk"])
def test_same_bits_every_time(ctx, op):
    past = [3000, 5, 1200, 64, 900, 2500]
    c = Cache(71, "q4", 16, 32, 8, [p + 1 for p in past])
    q = randh(gen(72), len(past), 32 * D)
    outs = []
    for _ in range(6):
        out = torch.zeros_like(q)
        if op == "decode":
            ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32(past), out, max_past=3000,
                               fused_prep=False, **c.kw())
        else:
            ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32(past), i32(range(len(past) + 1)), out,
                              max_len=3001, **c.kw())
        outs.append(out)
    ctx.sync()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_another_stream_than_the_current_one(ctx):
    c = Cache(73, "q4", 16, 16, 8, [513])
    qkv, rope = randh(gen(74), 513, 32 * D), rope_table(513)
    q, out, out2 = (torch.zeros(513, 16 * D, dtype=torch.float16, device="cuda")
                    for _ in range(3))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    kw = dict(max_len=513, stream=s, **c.kw())
    z, rs = i32([0]), i32([0, 513])
    torch.cuda.synchronize()
    ctx.kv_append(c.prm, qkv, None, rope, c.k, c.v, z, rs, q_out=q, **kw)
    ctx.attn_chunk_kv(c.prm, q, c.k, c.v, z, rs, out, **kw)
    with torch.cuda.stream(s):
        ctx.attn_chunk_kv(c.prm, q, c.k, c.v, z, rs, out2, max_len=513, **c.kw())
    ctx.sync(s)
    want, tol = attention64(c, q, [0], [513], True)
    assert_within(out, want, tol)
    assert torch.equal(out, out2)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows", [[70, 3], [4900, 100]])
def test_chunk_wait_runs_out(ctx, fmt, rows):
    import p2p_b200
    past = [900, 40]
    c = Cache(77, fmt, 16, 32, 8, [p + r for p, r in zip(past, rows)])
    q = randh(gen(78), sum(rows), 32 * D)
    out = torch.full_like(q, 7.0)
    args = (c.prm, q, c.k, c.v, i32(past), starts_of(rows), out)
    kw = dict(max_len=6000, **c.kw())
    ctx.attn_chunk_kv(*args, **kw)
    ctx.sync()
    good = out.clone()
    out.fill_(7.0)
    try:
        p2p_b200.lib.p2p_debug_set_wait_deficit(16)
        ctx.attn_chunk_kv(*args, **kw)
        with pytest.raises(p2p_b200.P2PError) as e:
            ctx.sync()
    finally:
        p2p_b200.lib.p2p_debug_set_wait_deficit(0)
    assert e.value.status == p2p_b200.P2P_ERR_TIMEOUT
    assert (out == 7).all()
    ctx.attn_chunk_kv(*args, **kw)
    ctx.sync()
    assert torch.equal(out, good)


@pytest.mark.parametrize("heads", [(32, 8), (16, 2)])
def test_decode_wait_runs_out(ctx, heads):
    """A copy that never completes (more bytes expected than come): the kernel gives up after its
    limit, writes nothing and reports it; the next call works, so no counter was left behind."""
    import p2p_b200
    hq, hkv = heads
    past = [3000, 40, 700]
    c = Cache(75, "q4", 16, hq, hkv, [p + 1 for p in past])
    q = randh(gen(76), 3, hq * D)
    out = torch.full_like(q, 7.0)
    args = (c.prm, q, None, None, c.k, c.v, i32(past), out)
    kw = dict(max_past=3000, fused_prep=False, **c.kw())
    ctx.attn_decode_kv(*args, **kw)
    ctx.sync()
    good = out.clone()
    out.fill_(7.0)
    try:
        p2p_b200.lib.p2p_debug_set_wait_deficit(16)
        ctx.attn_decode_kv(*args, **kw)
        with pytest.raises(p2p_b200.P2PError) as e:
            ctx.sync()
    finally:
        p2p_b200.lib.p2p_debug_set_wait_deficit(0)
    assert e.value.status == p2p_b200.P2P_ERR_TIMEOUT
    assert (out == 7).all()
    ctx.attn_decode_kv(*args, **kw)
    ctx.sync()
    assert torch.equal(out, good)


# ---- the weights' range of the 4-bit decode ---------------------------------------------------------
def decode_of_constant_keys(c, q, n):
    """One token over the n keys of a 4-bit cache whose K rows are constant (codes of 0, so that a
    score is lo * sum(q) / 8 in plain f32): out [hq][64] in f64 and how far a kernel may be from it.

    Weights.  A score in log2 units is a sum of 64 f16 values, a product and two additions: 24
    roundings of 2^-24 of its size, of the reference's (kept 12 below the largest score + log2 of the
    scale or of 2^-14) and of the differences; exp2 is off by 2^-22.  An error e of a
    weight moves out by w e |v - out|.
    A weight times the scale goes into the product sum in two f16 parts (2^-22) or, for 8 query heads
    per kv head, in one (2^-11), which moves out by that share of w (v - lo); below f16's normal numbers
    by 2^-25 with the largest product at 2^12 or more: 2^-37 of it in each code's weight.
    The product sums of 64 keys are four MMAs, each of up to 17 addends cut off at 2^-22 of the
    largest, which is below 2^-14 (a subnormal code) times the largest weight, or the sum so far; the
    result counts 2^22.  The other sums are f32: a lane's 8 keys of a block, its blocks, of 64 keys each,
    and the joins, below 64 + n / 64 roundings of 2^-24."""
    grp = c.hq // c.hkv
    at = c.at(0, torch.arange(n, device="cuda"))
    lo_k = c.k[at][:, :c.hkv * UNIT].reshape(n, c.hkv, UNIT)
    assert not lo_k[..., :34].any()  # codes and scale
    lo_k = lo_k[..., 34:].contiguous().view(torch.float16).double()[..., 0]    # [n][hkv]
    u = c.v[at][:, :c.hkv * UNIT].reshape(n, c.hkv, UNIT)
    par = u[..., 32:].contiguous().view(torch.float16).double()
    scale, lo = par[..., 0], par[..., 1]
    outs, tols = [], []
    for h in range(c.hkv):
        qs = q.view(c.hq, D)[h * grp:(h + 1) * grp].double()
        s = qs.sum(-1, keepdim=True) * lo_k[None, :, h] / 8                       # [grp][n]
        w = torch.softmax(s, -1)
        code = torch.stack([u[:, h, :32] & 15, u[:, h, :32] >> 4], -1).flatten(-2).double()
        above = code * scale[:, h, None]                                          # v - lo
        v = above + lo[:, h, None]
        o = w @ v
        e = 2.0 ** -21 + 2.0 ** -24 * 24 * (s.abs().amax() / math.log(2) + 40)
        t = e * (w @ v.abs() + o.abs())
        t = t + (2.0 ** -11 if grp == 8 else 2.0 ** -22) * (w @ above)
        t = t + 2.0 ** -37 * (w * scale[:, h].clamp(min=2.0 ** -14)).amax(-1, keepdim=True) * code.sum(0)
        ws = torch.nn.functional.pad(w * scale[:, h], (0, -n % 64)).view(grp, -1, 64)
        t = t + 68 * 2.0 ** -14 * ws.amax(-1).sum(-1, keepdim=True)
        t = t + (68 * 2.0 ** -22 + (64 + n / 64) * 2.0 ** -24) * (w @ above + w @ lo[:, h].abs()[:, None])
        t = t + o.abs() * 2.0 ** -11 + 2.0 ** -25
        outs.append(o)
        tols.append(t)
    return torch.cat(outs), torch.cat(tols)


def decode_constant_keys(ctx, hq, hkv, page, k, v, copies=1):
    """One token of each of `copies` sequences over the same n keys: k [n][hkv] (the rows' only value),
    v f16 [n][hkv][64].  (One sequence's keys are spread over all SMs; of hundreds, each is one CTA's.)"""
    n = len(k)
    c = Cache(91, "q4", page, hq, hkv, [n])
    at = c.at(0, torch.arange(n, device="cuda"))
    c.k[at] = quant4(k.half()[..., None].expand(n, hkv, D).contiguous())
    c.v[at] = quant4(v)
    q = torch.ones(copies, hq * D, dtype=torch.float16, device="cuda")
    out = torch.zeros_like(q)
    if page:
        c.table = c.table.repeat(copies, 1)
    else:
        c.offsets = c.offsets.repeat(copies)
    ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32([n - 1] * copies), out, max_past=n - 1,
                       fused_prep=False, **c.kw())
    ctx.sync()
    want, tol = decode_of_constant_keys(c, q[0], n)
    return out.view(copies, hq, D), want, tol


@pytest.mark.parametrize("amp", [1.0, 0.1, 0.03, 0.01, 1e-4])
@pytest.mark.parametrize("heads,n,gap", [((8, 8), 8192, 14), ((16, 8), 8192, 13), ((32, 8), 8192, 14),
                                         ((64, 8), 8192, 14), ((8, 1), 8192, 12), ((4, 1), 32768, 13),
                                         ((32, 8), 131071, 14), ((8, 1), 131071, 14)],
                         ids=lambda x: str(x).replace(" ", ""))
def test_decode_q4_strong_first_key(ctx, heads, n, gap, amp):
    """A key far above a long tail, whose weights times small scales are tiny: the tail counts."""
    hq, hkv = heads
    k = torch.zeros(n, hkv, device="cuda")
    k[0] = gap / 8
    v = amp * randh(gen(92), n, hkv, D)
    for copies in (1, 600 if n < 30000 else 300):
        got, want, tol = decode_constant_keys(ctx, hq, hkv, 64, k, v, copies)
        assert_within(got, want, tol, f"{copies} sequences")
        assert float(((got.double() - want).norm(dim=(1, 2)) / want.norm()).max()) < 1e-3


@pytest.mark.parametrize("heads", [(8, 8), (32, 8), (64, 8), (8, 1), (12, 12)])
@pytest.mark.parametrize("kind", ["mixed scales", "a loud key of no weight", "rising scores"])
def test_decode_q4_scales_of_all_sizes(ctx, heads, kind):
    hq, hkv = heads
    n, g = 9000, gen(93)
    v = torch.randn(n, hkv, D, generator=g, device="cuda")
    k = torch.randn(n, hkv, generator=g, device="cuda") / 2
    if kind == "mixed scales":
        v = v * 2.0 ** (22 * torch.rand(n, hkv, 1, generator=g, device="cuda") - 12)
        v[::7] = v[::7, :, :1]  # constant rows: a scale of 0
    elif kind == "rising scores":
        k = (k / 4 + torch.arange(n, device="cuda")[:, None] * (8 / n))
        v = v * 0.01
    else:
        k, v = k / 4, v * 0.01
        k[0] = 14 / 8 + 0.5
        k[n // 2], v[n // 2] = -4, 2000 * v[0]
    for copies in (1, 600):
        got, want, tol = decode_constant_keys(ctx, hq, hkv, 16, k, v.half(), copies)
        assert_within(got, want, tol, f"{copies} sequences")


@pytest.mark.parametrize("gap", [3.0, 3.125, 3.25, 3.375])
@pytest.mark.parametrize("heads", [(8, 8), (16, 8), (32, 8), (4, 1)])
def test_decode_q4_weights_in_two_parts(ctx, heads, gap):
    """Equal weights whose product with the scale is no f16: up to four query heads per kv head keep
    22 bits of them, which shows where the values' mean is near 0 and their lowest value is not."""
    hq, hkv = heads
    n = 8192
    k = torch.zeros(n, hkv, device="cuda")
    k[0] = gap / 8
    v = torch.full((n, hkv, D), -1 + 7 * 2 / 15, device="cuda")
    v[1::2] = -1 + 8 * 2 / 15
    v[..., 0], v[..., 1] = -1, 1
    got, want, tol = decode_constant_keys(ctx, hq, hkv, 0, k, v.half())
    assert_within(got, want, tol)
    assert (tol[:, 2:] < 2.0 ** -13).all()  # one f16 would be off by up to 2^-11


@pytest.mark.parametrize("amp", [1e-4, 0.01, 30.0, 2000.0])
@pytest.mark.parametrize("heads", [(8, 8), (8, 4), (16, 4), (64, 8), (8, 1)])
def test_decode_q4_ranges_of_every_group(ctx, heads, amp):
    """Tiny and large caches, with the bound of ordinary ones."""
    hq, hkv = heads
    c = Cache(94, "q4", 16, hq, hkv, [600, 50, 2000], amp=amp)
    q = randh(gen(95), 3, hq * D) * (0.05 if amp > 1 else 1.0)
    out = torch.zeros_like(q)
    past = [599, 49, 1999]
    ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32(past), out, max_past=1999,
                       fused_prep=False, **c.kw())
    ctx.sync()
    want, tol = attention64(c, q, past, [1] * 3, False)
    assert_within(out, want, tol)


# ---- infinite scores in prompt chunks ----------------------------------------------------------------
def chunk_with_infinite_keys(ctx, case, page, keys, sign):
    """One sequence whose keys `keys` have a K of sign * inf in dim 5 of kv head 0: out and the 64-bit
    one [rows][hq][64], with the bound of attention64 (the infinite products left out of its sizes: a
    score of -inf has weight 0, one of +inf makes the row NaN)."""
    (hq, hkv), past, rows = case
    n, grp = past + rows, hq // hkv
    c = Cache(96, "f16", page, hq, hkv, [n])
    q = randh(gen(97), rows, hq * D)
    k, v = c.keys64(0, n)
    at = c.at(0, torch.as_tensor(keys, device="cuda"))
    c.k[(*at, 0, 5)] = sign * math.inf
    out = torch.full_like(q, 7.0)
    ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32([past]), i32([0, rows]), out, max_len=n, **c.kw())
    ctx.sync()
    k, v = (t.repeat_interleave(grp, 1).permute(1, 0, 2) for t in (k, v))
    qi = q.double().view(rows, hq, D).permute(1, 0, 2)
    s, mag = qi @ k.transpose(1, 2) / 8, qi.abs() @ k.abs().transpose(1, 2) / 8
    s[:grp, :, keys] = sign * math.inf * qi[:grp, :, 5].sign()[..., None]
    hidden = torch.arange(n, device="cuda")[None] > \
        (past + torch.arange(rows, device="cuda"))[:, None]
    w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    o = w @ v
    e = 2.0 ** -11 + 2.0 ** -10 + mag * (2.0 ** -11 + 2.0 ** -18)
    t = (w * e) @ v.abs() + o.abs() * (w * e).sum(-1, keepdim=True)
    t = t + (w @ v.abs()) * (2.0 ** -11 + 2.0 ** -16) + o.abs() * 2.0 ** -11 + 2.0 ** -24
    return out.view(rows, hq, D), o.permute(1, 0, 2), t.permute(1, 0, 2)


def assert_nan_or_within(got, want, tol, what):
    odd = want.isnan()
    assert torch.equal(got.isnan(), odd), (what, int((got.isnan() != odd).sum()))
    assert_within(got[~odd], want[~odd], tol[~odd], what)


INFINITE = [
    # heads, past, rows: items that one CTA works on alone, and items split over several
    ((32, 8), 0, 40), ((32, 8), 130, 70), ((32, 8), 3000, 33), ((8, 1), 9000, 5), ((16, 16), 700, 257),
]


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("case", INFINITE, ids=str)
def test_an_infinite_key_at_any_place(ctx, case, sign):
    (hq, hkv), past, rows = case
    n = past + rows
    for j in range(8):
        for key in {j, n - 17 + j, n // 2 // 8 * 8 + j}:
            got, want, tol = chunk_with_infinite_keys(ctx, case, 16, [key], sign)
            assert_nan_or_within(got, want, tol, f"key {key}")
            # the other kv heads do not see it
            assert hkv == 1 or not want[:, hq // hkv:].isnan().any()


@pytest.mark.parametrize("page", [0, 64])
@pytest.mark.parametrize("case", INFINITE, ids=str)
def test_rows_of_infinite_scores(ctx, case, page):
    """All of a kv head's keys infinite, its first ones, its last ones, all but one."""
    _, past, rows = case
    n = past + rows
    for keys in (range(n), range(min(n - 1, 200)), range(n // 2, n), range(1, n)):
        for sign in (1, -1):
            got, want, tol = chunk_with_infinite_keys(ctx, case, page, list(keys), sign)
            assert_nan_or_within(got, want, tol, f"{sign} * inf at {keys}")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("case", INFINITE, ids=str)
def test_an_infinite_query_is_its_rows_alone(ctx, fmt, case):
    (hq, hkv), past, rows = case
    c = Cache(98, fmt, 16, hq, hkv, [past + rows])
    q = randh(gen(99), rows, hq * D)
    want, tol = (t.view(rows, hq, D) for t in attention64(c, q, [past], [rows], True))
    for r, h, d, x in ((0, 1, 3, math.inf), (rows - 1, hq - 1, 60, -math.inf), (rows // 2, 0, 0, math.nan)):
        q[r, h * D + d] = x
        want[r, h] = math.nan
    out = torch.zeros_like(q)
    ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32([past]), i32([0, rows]), out, max_len=past + rows, **c.kw())
    ctx.sync()
    got = out.view(rows, hq, D)
    # (the first row of the first case sees one key: a score of -inf or +inf, NaN either way)
    assert_nan_or_within(got, want, tol, "q")


@pytest.mark.parametrize("op", ["append", "read"])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("starts,done", [
    ([0, 4, 8, 12], [(0, 0, 4), (1, 4, 8)]),   # of 8 rows: the last sequence's all lie behind them
    ([0, 4, 8, 8], [(0, 0, 4), (1, 4, 8)]),    # nothing wrong
    ([0, 6, 2, 4], [(0, 0, 2)]),               # falling: sequence 1 has -4 rows
], ids=str)
def test_rows_without_a_sequence_are_left_alone_and_reported(ctx, op, page, starts, done):
    import p2p_b200
    hq, hkv, past, n = 8, 2, [5, 40, 33], 8
    c = Cache(47, "q4", page, hq, hkv, [60, 60, 60])
    good_k, good_v = c.k.clone(), c.v.clone()
    qkv, rope = randh(gen(48), n, 12 * D), rope_table(60)
    out = torch.full((n, hq * D), 7.0, dtype=torch.float16, device="cuda")
    back = torch.full((n, hkv, D), 7.0, dtype=torch.float16, device="cuda")
    if op == "append":
        ctx.kv_append(c.prm, qkv, None, rope, c.k, c.v, i32(past), i32(starts), max_len=60,
                      q_out=out, **c.kw())
    else:
        ctx.kv_read(c.prm, c.k, c.v, i32(past), i32(starts), back, None, max_len=60, **c.kw())
    if starts[-1] == n:
        ctx.sync()
    else:
        with pytest.raises(p2p_b200.KvFullError):
            ctx.sync()
    ctx.sync()
    left = torch.ones(n, dtype=torch.bool, device="cuda")
    for i, a, b in done:
        left[a:b] = False
        if op == "read":
            assert torch.equal(back[a:b], c.keys64(i, 60)[0][past[i]:past[i] + b - a].float().half())
            continue
        assert not (out[a:b] == 7).any()
        at = c.at(i, past[i] + torch.arange(b - a, device="cuda"))
        _, k, v = prep(ctx, c.prm, qkv[a:b], None, rope, past[i])
        used = slice(0, hkv * UNIT)
        assert torch.equal(c.k[(*at, used)], quant4(k)[:, used])
        assert torch.equal(c.v[(*at, used)], quant4(v)[:, used])
        c.k[at], c.v[at] = good_k[at], good_v[at]
    assert (out[left] == 7).all() and (back[left] == 7).all()
    assert torch.equal(c.k, good_k) and torch.equal(c.v, good_v)


def test_append_refuses_a_q_that_overlaps_qkv(ctx):
    import p2p_b200
    c = Cache(49, "f16", 16, 8, 2, [40])
    buf = randh(gen(50), 4, 24 * D)
    qkv, rope = buf[:, :12 * D], rope_table(40)
    keep, k, v = buf.clone(), c.k.clone(), c.v.clone()
    args, kw = (c.k, c.v, i32([3]), i32([0, 4])), dict(max_len=40, **c.kw())
    flat = buf.view(-1)
    for bad in (flat[:4 * 8 * D].view(4, 8 * D),              # in place with its own pitch
                buf[:, 4 * D:12 * D],                         # shifted by heads
                flat[24 * D:24 * D * 4 + 8 * D].as_strided((3, 8 * D), (24 * D, 1)),
                flat[8 * D:].as_strided((4, 8 * D), (16 * D, 1))):
        with pytest.raises(p2p_b200.P2PError) as e:
            ctx.kv_append(c.prm, qkv[:len(bad)], None, rope, *args, q_out=bad, **kw)
        assert e.value.status == p2p_b200.P2P_ERR_INVALID_ARG
    ctx.sync()
    assert torch.equal(buf, keep) and torch.equal(c.k, k) and torch.equal(c.v, v)
    # beside it, in place with its pitch, and one row in place are fine
    q = torch.zeros(4, 8 * D, dtype=torch.float16, device="cuda")
    ctx.kv_append(c.prm, qkv, None, rope, *args, q_out=q, **kw)
    ctx.kv_append(c.prm, qkv, None, rope, *args, q_out=buf[:, 12 * D:20 * D], **kw)
    one = buf[:1, :12 * D].clone()
    ctx.kv_append(c.prm, one, None, rope, c.k, c.v, i32([3]), i32([0, 1]), q_out=one[:, :8 * D], **kw)
    ctx.kv_append(c.prm, qkv, None, rope, *args, q_out=buf[:, :8 * D], **kw)
    ctx.sync()
    assert torch.equal(buf[:, 12 * D:20 * D], q) and torch.equal(buf[:, :8 * D], q)
    assert torch.equal(one[:, :8 * D], q[:1])


def test_chunk_refuses_an_out_that_overlaps_q(ctx):
    import p2p_b200
    c = Cache(51, "q4", 16, 8, 2, [40])
    buf = randh(gen(52), 9, 24 * D)
    keep = buf.clone()
    q = buf[:4, :8 * D]
    args, kw = (c.k, c.v, i32([3]), i32([0, 4])), dict(max_len=40, **c.kw())
    for bad in (q, buf[1:5, :8 * D], buf[:4, 4 * D:12 * D], buf[3:7, 7 * D:15 * D],
                buf.view(-1)[16 * D:].as_strided((4, 8 * D), (16 * D, 1))):
        with pytest.raises(p2p_b200.P2PError) as e:
            ctx.attn_chunk_kv(c.prm, q, *args, bad, **kw)
        assert e.value.status == p2p_b200.P2P_ERR_INVALID_ARG
    ctx.sync()
    assert torch.equal(buf, keep)
    out = torch.zeros(4, 8 * D, dtype=torch.float16, device="cuda")
    ctx.attn_chunk_kv(c.prm, q, *args, out, **kw)
    for beside in (buf[:4, 8 * D:16 * D], buf[4:8, :8 * D], buf[2:6, 16 * D:]):
        ctx.attn_chunk_kv(c.prm, q, *args, beside, **kw)
        ctx.sync()
        assert torch.equal(beside, out) and torch.equal(q, keep[:4, :8 * D])


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_logits_refuse_an_out_that_overlaps_them(ctx, dt):
    import p2p_b200
    buf = randh(gen(53), 7, 1500).to(dt)
    keep = buf.clone()
    x, tok = buf[:4, :500], torch.full((4,), -7, dtype=torch.int32, device="cuda")
    for bad in (buf[:4, 1:501], buf[1:5, :500], buf[:4, 499:999],
                buf.view(-1)[1000:].as_strided((4, 500), (1000, 1))):
        with pytest.raises(p2p_b200.P2PError) as e:
            ctx.logits_pick(x, tok, out=bad)
        assert e.value.status == p2p_b200.P2P_ERR_INVALID_ARG
    ctx.sync()
    assert torch.equal(buf, keep) and tok.tolist() == [-7] * 4
    want = [int(np.argmax(r)) for r in x.float().cpu().numpy()]
    for fine in (buf[:4, 500:1000], buf[3:7, 1000:], x):
        ctx.logits_pick(x, tok, out=fine)
        ctx.sync()
        assert torch.equal(fine, keep[:4, :500]) and tok.tolist() == want


@pytest.mark.parametrize("amp", [1e-5, 1e-4, 1e-3, 3e3])
@pytest.mark.parametrize("heads", [(8, 8), (16, 4), (64, 8), (8, 1)])
def test_decode_q4_queries_of_any_size(ctx, heads, amp):
    """Queries down to f16's subnormal numbers over keys that make up for it: scores of the usual size
    and the bound of attention64, with the MMAs' share of a score's error for 4-bit codes: four of them,
    each of up to 17 addends cut off at 2^-22 of the largest, which is below 2^-14 (a subnormal code)
    times the head's largest query value and counts 2^24 times the key's scale."""
    import p2p_b200
    hq, hkv = heads
    past = [11, 40, 0, 333]
    k_amp = min(1e4, 1.0 / amp)
    c = Cache(54, "q4", 16, hq, hkv, [p + 1 for p in past])
    c.k = quant4((k_amp * randh(gen(55), *c.k.shape[:2], hkv, D).float()).clamp(-6e4, 6e4).half())
    scale = 0.8 / (amp * k_amp)
    c.prm = p2p_b200.Params(hq, hkv, scale=scale)
    q = (amp * randh(gen(56), 4, hq * D).float()).half()
    q[0, :D] = 0
    q[3, D:D + 40] = 0
    out = torch.zeros_like(q)
    ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32(past), out, max_past=333,
                       fused_prep=False, **c.kw())
    ctx.sync()
    grp = hq // hkv
    for i, p in enumerate(past):
        k, v = (t.repeat_interleave(grp, 1).permute(1, 0, 2) for t in c.keys64(i, p + 1))
        qi = q[i].double().view(hq, 1, D)
        s = scale * qi @ k.transpose(1, 2)                                 # [hq][1][keys]
        w = torch.softmax(s, -1)
        o = w @ v
        lo = v.amin(-1, keepdim=True)
        step = (k.amax(-1) - k.amin(-1))[:, None] / 14                     # the scale or more
        e = 2.0 ** -11 + 2.0 ** -10 + scale * (qi.abs() @ k.abs().transpose(1, 2)) * 2.0 ** -18
        e = e + 68 * 2.0 ** -12 * scale * qi.abs().amax(-1, keepdim=True) * step
        t = (w * e) @ v.abs() + o.abs() * (w * e).sum(-1, keepdim=True)
        t = t + (w @ v.abs()) * 2.0 ** -16 + 2.0 ** -11 * (w @ (v - lo)) + o.abs() * 2.0 ** -11 + 2.0 ** -24
        assert_within(out[i].view(hq, D), o[:, 0], t[:, 0], f"sequence {i}")


def test_decode_q4_infinite_queries_are_their_rows_alone(ctx):
    past, hq, hkv = [300, 5, 0], 16, 4
    c = Cache(57, "q4", 16, hq, hkv, [p + 1 for p in past])
    q = randh(gen(58), 3, hq * D)
    want, tol = (t.view(3, hq, D) for t in attention64(c, q, past, [1] * 3, False))
    for r, h, d, x in ((0, 1, 3, math.inf), (1, 15, 60, -math.inf), (2, 0, 0, math.nan)):
        q[r, h * D + d] = x
        want[r, h] = math.nan
    out = torch.zeros_like(q)
    ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32(past), out, max_past=300,
                       fused_prep=False, **c.kw())
    ctx.sync()
    assert_nan_or_within(out.view(3, hq, D), want, tol, "q")


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("gap", [13, 15, 17, 18])
@pytest.mark.parametrize("heads,n,rows,copies", [((32, 8), 8192, 2, 60), ((32, 8), 32768, 2, 24),
                                                 ((8, 1), 32768, 40, 150)], ids=str)
def test_chunk_behind_a_strong_first_key(ctx, fmt, gap, heads, n, rows, copies):
    """A first key of no value far above a long tail: the rows are what the tail's small weights make
    of it.  (Hundreds of items over the same keys: each is one CTA's or two.)"""
    (hq, hkv), g = heads, gen(60)
    c = Cache(59, fmt, 64, hq, hkv, [n], per_channel=False)
    at = c.at(0, torch.arange(n, device="cuda"))
    v = 1 + 0.5 * randh(g, n, hkv, D)
    v[0] = 0
    k = torch.zeros(n, hkv, D, dtype=torch.float16, device="cuda")
    k[0] = gap / 8
    if fmt == "i8":
        c.ks.fill_(1 / 64)
        c.vs.fill_(1 / 32)
    c.k[at], c.v[at] = c.stored(k, c.ks), c.stored(v, c.vs)
    q = torch.ones(copies * rows, hq * D, dtype=torch.float16, device="cuda")
    out = torch.zeros_like(q)
    kw = c.kw() | {"block_table": c.table.repeat(copies, 1)}
    ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32([n - rows] * copies), i32(range(0, len(q) + 1, rows)), out,
                      max_len=n, **kw)
    ctx.sync()
    want, tol = attention64(c, q[:rows], [n - rows], [rows], True)
    assert_within(out.view(copies, rows, hq * D), want, tol)


@pytest.mark.parametrize("fmt,op", [("f16", "chunk"), ("i8", "chunk"), ("q4", "chunk"), ("q4", "decode")])
def test_sequences_near_the_end_of_32_bits_are_refused(ctx, fmt, op):
    """A table whose entries repeat one page of 4096 tokens: from 2^31 - 4096 keys on, a sequence is
    skipped and reported, and its neighbour is computed."""
    import p2p_b200
    c = Cache(61, fmt, 4096, 8, 1, [4096])
    n, top = 2**31 // 4096, 2**31 - 4096
    c.table = c.table.expand(2, 1).repeat(1, n).contiguous()
    q = randh(gen(62), 2, 8 * D)
    for past in (top - 1, 2**31 - 2):
        out = torch.full_like(q, 7.0)
        if op == "chunk":
            ctx.attn_chunk_kv(c.prm, q, c.k, c.v, i32([past, 600]), i32([0, 1, 2]), out,
                              max_len=2**31 - 1, **c.kw())
        else:
            ctx.attn_decode_kv(c.prm, q, None, None, c.k, c.v, i32([past, 600]), out,
                               max_past=2**31 - 2, fused_prep=False, **c.kw())
        with pytest.raises(p2p_b200.KvFullError):
            ctx.sync()
        want, tol = attention64(c, q[1:], [600], [1], op == "chunk")
        assert (out[0] == 7).all()
        assert_within(out[1:], want, tol)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("heads", [(32, 8), (8, 1), (72, 9)])
def test_decode_q4_in_place_or_apart(ctx, heads, fused):
    """out over the q columns gives what it gives apart; any other overlap with qkv is refused."""
    import p2p_b200
    (hq, hkv), past = heads, [700, 3, 64, 20, 5000]
    n, w = len(past), hq * D
    g = gen(63)
    wide = (hq + 2 * hkv) * D
    buf = randh(g, n + 1, wide + 24)
    rope = rope_table(5001)

    def call(c, x, out):
        ctx.attn_decode_kv(c.prm, x[:, :wide], None, rope, c.k, c.v, i32(past), out, max_past=5000,
                           fused_prep=fused, **c.kw())
        ctx.sync()
    a, b = (Cache(64, "q4", 16, hq, hkv, [p + 1 for p in past]) for _ in range(2))
    keep, out = buf.clone(), torch.zeros(n, w, dtype=torch.float16, device="cuda")
    call(a, buf[:n], out)
    k = a.k.clone()
    for bad in (buf[:n, 16:16 + w], buf[1:, :w], buf.view(-1)[:n * w].view(n, w)):
        with pytest.raises(p2p_b200.P2PError) as e:
            call(a, buf[:n], bad)
        assert e.value.status == p2p_b200.P2P_ERR_INVALID_ARG
    assert torch.equal(buf, keep) and torch.equal(a.k, k)
    call(b, buf[:n], buf[:n, :w])
    assert torch.equal(buf[:n, :w], out) and torch.equal(b.k, a.k) and torch.equal(b.v, a.v)
    assert torch.equal(buf[:, w:], keep[:, w:]) and torch.equal(buf[n], keep[n])
