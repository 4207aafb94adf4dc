"""The 8-bit layer operators on a B200 against their definition in 64 bits: rows quantised, read back
and looked up, the residual addition with the RMS norm, products with scales, the gated projections
-- and all of them in the order a model runs them, captured and replayed.

Tolerances: an f32 operation is off by 2^-24 of its result, a rounding to f16 by 2^-11 (or 2^-25, half
of the smallest f16 number); each test counts the ones on its way."""
import itertools
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0**-24
HALF = {torch.float16: 2.0**-11, torch.float32: U}
F16, F32 = torch.float16, torch.float32
F16_ZERO = torch.zeros((), dtype=F16)


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


def rows_in(g, m, k, dt, pad=0, off=0, amp=1.0):
    """Random rows with `pad` values between two and the first `off` values behind an aligned start."""
    buf = torch.randn(m * (k + pad) + off, generator=g, device="cuda", dtype=F32).mul_(amp).to(dt)
    return buf[off:].view(m, k + pad)[:, :k]


def empty_q8(m, k, gap=0, fill=77):
    ld = (k + 15) // 16 * 16 + gap
    whole = torch.full((m, ld), fill, dtype=torch.int8, device="cuda")
    return whole, whole[:, :k], torch.full((m,), -5.0, device="cuda")


def codes(g, m, k, gap=0, full=False):
    whole, q, s = empty_q8(m, k, gap)
    q.copy_(torch.randint(-128 if full else -127, 128, (m, k), generator=g, device="cuda",
                          dtype=torch.int64).to(torch.int8))
    return q, (0.5 + torch.rand(m, generator=g, device="cuda")) / 100


def close(x, want, tol, what=""):
    """|x - want| <= tol everywhere, all in 64 bits."""
    off = (x.double() - want).abs() - tol
    assert not torch.isnan(off).any(), what
    assert off.max().item() <= 0, (what, off.max().item())


# ---- rows -> codes --------------------------------------------------------------------------------
def check_codes(q, scale, v, err):
    """Codes and scales of rows whose exact values are v, known to a relative `err`."""
    a = v.abs().amax(1, keepdim=True)
    # a code is a rounding (1/2) of v * inv, inv = 127 / a: both factors' errors and two roundings
    close(q, v * (127 / a), 0.5 + 127 * (2 * err + 3 * U), "codes")
    close(scale, a[:, 0] / 127, a[:, 0] / 127 * (err + 2 * U), "scales")
    assert (q.abs().amax(1) == 127).all()  # the largest value has the largest code


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("m,k,pad,off", [
    (1, 1, 0, 0), (3, 7, 2, 1), (5, 64, 0, 0), (300, 1003, 0, 0), (2, 1024, 8, 8), (1, 2048, 0, 0),
    (7, 2048, 0, 1), (4000, 520, 0, 0), (3, 5000, 0, 0), (5, 8192, 0, 0), (3, 8193, 7, 0),
    (2, 20000, 0, 0), (1, 65536, 0, 0)])
def test_quantize(ctx, dt, m, k, pad, off):
    x = rows_in(gen(m + k), m, k, dt, pad, off)
    whole, q, s = empty_q8(m, k, 16)
    ctx.quantize_rows_q8(x, q, s)
    check_codes(q, s, x.double(), 0)
    # one division, rounded once (torch divides f32 by a plain number as a product with its inverse,
    # rounded twice; 64 bits are more than twice 24, so the second rounding here changes nothing)
    assert torch.equal(s, (x.double().abs().amax(1) / 127).float())
    assert (whole[:, k:] == 77).all()
    q2, s2 = ctx.quantize_rows_q8(x)
    assert torch.equal(q2, q) and torch.equal(s2, s)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("k", [9, 1000, 9001])
def test_quantize_rows_of_every_kind(ctx, dt, k):
    x = rows_in(gen(k), 9, k, dt)
    x[0] = 0
    x[1, k // 2] = math.inf
    x[2, k - 1] = -math.inf
    x[3, 0] = math.nan
    x[4] = 0
    x[4, 1] = 2.0**-24 if dt is F16 else 2.0**-101
    x[5] = 65504 if dt is F16 else 3e38
    x[6] = -0.0
    x[7] = 0
    x[7, 3] = -2.0**-14 if dt is F16 else -2.0**-99
    q, s = ctx.quantize_rows_q8(x)
    for i in (0, 6):
        assert s[i] == 0 and (q[i] == 0).all()
    for i in (1, 2, 3):
        assert torch.isnan(s[i]) and (q[i] == 0).all()
    if dt is F32:  # below 2^-100: zeros
        assert s[4] == 0 and (q[4] == 0).all()
    else:
        check_codes(q[4:5], s[4:5], x[4:5].double(), 0)
    check_codes(q[[5, 7, 8]], s[[5, 7, 8]], x[[5, 7, 8]].double(), 0)


@pytest.mark.parametrize("at_once,pad", [(300, 0), (4096, 0), (4096, 7), (16384, 0)])
@pytest.mark.parametrize("top", ["subnormal", 2.0**-14, 1.0, 2.0**15])
def test_quantize_ties_of_f16(ctx, top, at_once, pad):
    """Every f16 significand as a row's largest value, against every f16 value up to it, of both signs: the
    codes are 127 v / a rounded to even, ties too.  (In 64 bits the quotient is exact at a tie, and no other
    one lies within 2^-20 of a half.)"""
    low = 0 if top == "subnormal" else torch.tensor(top, dtype=F16).view(torch.int16).item()
    largest = torch.arange(low, low + 1024, device="cuda", dtype=torch.int16).view(F16)
    largest = largest[largest > 0] if low == 0 else largest  # a row of zeros is another test's
    ties = 0
    for first in range(0, low + 1024, at_once):
        v = torch.arange(first, min(first + at_once, low + 1024), device="cuda",
                         dtype=torch.int16).view(F16)
        a = largest[:, None]
        v = torch.where(v <= a, v, F16_ZERO.to("cuda"))
        whole = torch.zeros(len(largest), 1 + 2 * v.shape[1] + pad, device="cuda", dtype=F16)
        x = whole[:, :1 + 2 * v.shape[1]]
        x[:, :1], x[:, 1::2], x[:, 2::2] = a, v, -v
        q, s = ctx.quantize_rows_q8(x)
        want = 127 * x.double() / a.double()
        ties += ((want - want.floor()) == 0.5).sum().item()
        assert torch.equal(q.double(), torch.round(want))
    assert ties > 0


# ---- codes -> values ------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("n,k,m,pad,off", [(1, 1, 1, 0, 0), (5, 7, 9, 1, 0), (50, 64, 33, 0, 0),
                                           (300, 1003, 300, 0, 0), (9, 2048, 1000, 8, 8),
                                           (11, 2500, 40, 0, 3), (3, 65536, 2, 0, 0)])
def test_read(ctx, dt, n, k, m, pad, off):
    g = gen(n + k)
    q, s = codes(g, n, k, 16, full=True)
    index = torch.randint(0, n, (m,), generator=g, device="cuda", dtype=torch.int32)
    index[m // 2] = -1
    out = rows_in(g, m, k, dt, pad, off)
    before = out.clone()
    ctx.read_rows_q8(q, s, out, index=index, factor=3.5)
    at = index.long().clamp(min=0)
    # one product each with the scale and the factor, then out's rounding
    want = q.double()[at] * s.double()[at, None] * 3.5
    want[m // 2] = 0
    close(out, want, want.abs() * (2 * U + HALF[dt]) + 2.0**-25)
    few = min(n, m)
    ctx.read_rows_q8(q, s, out[:few])
    want = q.double()[:few] * s.double()[:few, None]
    close(out[:few], want, want.abs() * (2 * U + HALF[dt]) + 2.0**-25)
    ctx.sync()
    assert before.shape == out.shape


def test_read_outside_the_table(ctx):
    import p2p_b200
    g = gen(3)
    q, s = codes(g, 10, 100)
    index = torch.tensor([3, 10, -2, 2**31 - 1, 0, -1], dtype=torch.int32, device="cuda")
    out = torch.full((6, 100), 9.0, device="cuda")
    ctx.read_rows_q8(q, s, out, index=index)
    with pytest.raises(p2p_b200.P2PError, match="outside the table"):
        ctx.sync()
    ctx.sync()  # reported once
    want = q.float()[[3, 0]] * s[[3, 0], None]
    assert torch.equal(out[[0, 4]], want) and (out[[1, 2, 3, 5]] == 0).all()
    # a NaN scale is the row's values, whatever the codes
    s[3] = math.nan
    ctx.read_rows_q8(q, s, out[:2])
    assert not torch.isnan(out[:2]).any()
    ctx.read_rows_q8(q, s, out[:4], index=index[:1].expand(4).contiguous())
    assert torch.isnan(out[:4]).all()


# ---- norm -----------------------------------------------------------------------------------------
def norm_error(k):
    """Relative error of y: half of the sum of squares' (each thread adds at most 32 values, or
    k / 256 of a long row, then 5 + 4 sums; a square, the mean with eps: 16 in all with some to
    spare), an inverse root (2^-22.9, 2.2 units), two products."""
    return ((max(32, k / 256 + 16) + 16) / 2 + 5) * U


def check_norm(x, r, w, eps, dt, q=None, s=None, total=None, y=None):
    k = x.shape[1]
    v = x.float() + (r.float() if r is not None else 0)
    v = v.to(dt)
    if total is not None:
        assert torch.equal(total, v)
    v = v.double()
    want = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    if w is not None:
        want = want * w.double()
    e = norm_error(k)
    if y is not None:
        close(y, want, want.abs() * (e + HALF[dt]) + (2.0**-25 if dt is F16 else 0), "y")
    if q is not None:
        check_codes(q, s, want, e)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("m,k,pad,off", [
    (1, 1, 0, 0), (3, 7, 1, 1), (1, 2048, 0, 0), (300, 1003, 0, 0), (2000, 1024, 0, 0),
    (9, 1024, 8, 8), (700, 2048, 0, 0), (3, 6000, 0, 0), (5, 8192, 0, 0), (2, 8200, 3, 1),
    (2, 30000, 0, 0)])
@pytest.mark.parametrize("weighted,residual", [(True, True), (True, False), (False, True)])
def test_norm(ctx, dt, m, k, pad, off, weighted, residual):
    g = gen(m * 7 + k)
    x = rows_in(g, m, k, dt, pad, off)
    r = rows_in(g, m, k, dt, pad, 0, 2.0) if residual else None
    w = (1 + 0.3 * torch.randn(k, generator=g, device="cuda")).half() if weighted else None
    total, y = rows_in(g, m, k, dt, pad, off), rows_in(g, m, k, dt, pad + 1, off)
    whole, q, s = empty_q8(m, k, 32)
    ctx.add_norm_q8(x, w, q, s, residual=r, sum_out=total, y=y, eps=1e-5)
    check_norm(x, r, w, 1e-5, dt, q, s, total, y)
    assert (whole[:, k:] == 77).all()
    # without the other outputs the codes are the same
    q2, s2 = ctx.add_norm_q8(x, w, residual=r)
    assert torch.equal(q2, q) and torch.equal(s2, s)
    # in place: the sum over x, y over the residual; then the sum over the residual
    x2 = x.clone()
    r2 = r.clone() if residual else None
    ctx.add_norm_q8(x2, w, q2, s2, residual=r2, sum_out=x2, y=r2)
    assert torch.equal(q2, q) and torch.equal(s2, s) and torch.equal(x2, total)
    if residual:
        assert torch.equal(r2, y)
        r2 = r.clone()
        ctx.add_norm_q8(x, w, q2, s2, residual=r2, sum_out=r2)
        assert torch.equal(q2, q) and torch.equal(r2, total)


@pytest.mark.parametrize("m,k,pad", [(3, 1, 0), (200, 64, 0), (500, 1003, 0), (300, 2048, 0), (40, 2048, 1),
                                     (9, 8192, 0), (4, 20000, 0)])
def test_norm_is_f32_operations(ctx, m, k, pad):
    """Of whole numbers, whose squares add up exactly in any order, y and the scales are those of the formula
    in f32 operations, each rounded: a mean, a root, a quotient, two products; the largest |y| over 127."""
    g = gen(m + k)
    x = rows_in(g, m, k, F32, pad)
    x.copy_(torch.randint(-15, 16, (m, k), generator=g, device="cuda"))
    x[:, 0] = 13
    w = (1 + 0.3 * torch.randn(k, generator=g, device="cuda")).half()
    y = torch.zeros(m, k, device="cuda")
    q, s = ctx.add_norm_q8(x, w, y=y, eps=0.001953125)
    f = lambda v: v.float().double()  # noqa: E731  (64 bits are more than twice 24: rounded as once)
    d = x.double()
    mean = f(f((d * d).sum(1, keepdim=True) / k) + 0.001953125)
    rstd = f(1 / f(torch.sqrt(mean)))
    want = f(f(d * w.double()) * rstd)
    assert torch.equal(y.double(), want)
    assert torch.equal(s.double(), f(want.abs().amax(1) / 127))


@pytest.mark.parametrize("k", [512, 1003])
def test_norm_weights_anywhere(ctx, k):
    """Weights that start between two 16-byte boundaries, and no codes' neighbours touched."""
    g = gen(k)
    x, r = rows_in(g, 50, k, F16), rows_in(g, 50, k, F16)
    w = (1 + 0.3 * torch.randn(k + 1, generator=g, device="cuda")).half()[1:]
    q, s = ctx.add_norm_q8(x, w, residual=r)
    check_norm(x, r, w, 1e-5, F16, q, s)
    q2, s2 = ctx.add_norm_q8(x, w.clone(), residual=r)
    assert torch.equal(q, q2) and torch.equal(s, s2)


def test_norm_without_codes(ctx):
    from p2p_b200 import _lib, lib
    import ctypes as C
    g = gen(1)
    x, w = rows_in(g, 6, 500, F16), torch.ones(500, device="cuda", dtype=F16)
    y = torch.zeros_like(x)
    a = _lib.AddNorm(x.data_ptr(), None, w.data_ptr(), None, y.data_ptr(), 500, 0, 0, 500,
                     _lib.Q8Rows(None, None, 0, 6, 500), 0, 0.5)
    assert lib.p2p_add_norm_q8(ctx.h, C.byref(a), None) == 0
    torch.cuda.synchronize()
    check_norm(x, None, w, 0.5, F16, y=y)


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("k", [64, 1500, 9000])
def test_norm_rows_of_every_kind(ctx, dt, k):
    g = gen(k)
    x, r = rows_in(g, 8, k, dt), rows_in(g, 8, k, dt)
    w = (1 + 0.3 * torch.randn(k, generator=g, device="cuda")).half()
    x[0], r[0] = 0, 0
    x[1, 5] = math.nan
    x[2, 6] = math.inf
    x[3, 7], r[3, 7] = math.inf, -math.inf
    x[4], r[4] = 1e-4, 1e-4                                     # far below eps
    x[5], r[5] = (60000, 0) if dt is F16 else (1e15, 1e15)      # large
    if dt is F16:
        x[6], r[6] = 60000, 60000                               # the sum is infinite
    else:
        x[6] = 1e25                                             # its square is
    y, total = torch.zeros_like(x), torch.zeros_like(x)
    q, s = ctx.add_norm_q8(x, w, residual=r, sum_out=total, y=y)
    assert s[0] == 0 and (q[0] == 0).all() and (y[0] == 0).all()
    for i in (1, 2, 3, 6):
        assert torch.isnan(s[i]) and (q[i] == 0).all() and torch.isnan(y[i]).all()
    good = [4, 5, 7]
    check_norm(x[good], r[good], w, 1e-5, dt, q[good], s[good], total[good], y[good])


# ---- what lies around the rows ------------------------------------------------------------------------
def framed(m, k, dt, pad, off):
    """Rows of nines inside a buffer of nines: `off` values in front, `pad` between two rows, some behind."""
    buf = torch.full((off + m * (k + pad) + 40,), 9.0, device="cuda", dtype=dt)
    return buf, buf[off:off + m * (k + pad)].view(m, k + pad)[:, :k]


def only_rows_written(buf, rows):
    outside = buf.clone()
    outside.as_strided(rows.shape, rows.stride(), rows.storage_offset()).fill_(9.0)
    return bool((outside == 9).all())


@pytest.mark.parametrize("dt", [F16, F32])
@pytest.mark.parametrize("pad,off", [(0, 0), (1, 1), (8, 8), (3, 0)])
@pytest.mark.parametrize("m,k", [(1, 1), (5, 7), (9, 128), (33, 250), (7, 257), (40, 512), (6, 520), (11, 1003),
                                 (5, 2048), (3, 5001), (3, 20001)])
def test_nothing_around_the_rows_is_written(ctx, dt, m, k, pad, off):
    """Outputs of any pitch and start: their rows, the same as of rows on 16-byte boundaries, and nothing in
    front of, between and behind them."""
    g = gen(m + k)
    x, r, w = rows_in(g, m, k, dt), rows_in(g, m, k, dt), torch.ones(k, device="cuda", dtype=F16)
    (sums, total), (ys, y) = framed(m, k, dt, pad, off), framed(m, k, dt, pad, off)
    q, s = ctx.add_norm_q8(x, w, residual=r, sum_out=total, y=y)
    check_norm(x, r, w, 1e-5, dt, q, s, total, y)
    assert only_rows_written(sums, total) and only_rows_written(ys, y)
    outs, out = framed(m, k, dt, pad, off)
    straight = torch.zeros(m, (k + 7) // 8 * 8, device="cuda", dtype=dt)[:, :k]
    ctx.read_rows_q8(q, s, out)
    ctx.read_rows_q8(q, s, straight)
    assert only_rows_written(outs, out) and torch.equal(out, straight)
    outs.fill_(9)
    ctx.read_rows_q8(q, s, out, index=torch.arange(m, device="cuda", dtype=torch.int32).flip(0))
    assert only_rows_written(outs, out) and torch.equal(out, straight.flip(0))


# ---- products -------------------------------------------------------------------------------------
def product(x, xs, w, ws):
    return (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()


def check_gemm(y, x, xs, w, ws, bias, res, dt):
    p = product(x, xs, w, ws)
    want, tol = p, p.abs() * 3 * U  # the sum as f32, two products
    if bias is not None:
        want = want + bias.double()
        tol = tol + (want.abs() + tol) * U
    if res is not None:
        want = want + res.double()
        tol = tol + (want.abs() + tol) * U
    close(y, want, tol + (want.abs() + tol) * HALF[dt] + 2.0**-25)


SIZES = [(1, 1, 1), (1, 64, 64), (1, 2048, 2048), (2, 100, 33), (3, 257, 1003), (7, 130, 4096),
         (8, 64, 128), (9, 1000, 700), (16, 512, 2048), (17, 384, 160), (31, 128, 65), (32, 4100, 256),
         (33, 129, 129), (48, 640, 8192), (64, 256, 1024), (65, 127, 512), (100, 300, 200),
         (128, 128, 128), (129, 257, 300), (200, 2048, 1024), (255, 512, 96), (256, 1024, 512),
         (257, 2331, 1531), (400, 96, 2048), (513, 768, 768), (1000, 1333, 640), (2050, 1024, 256), (2100, 2331, 300), (2300, 130, 1003),
         (2304, 768, 512)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dt,bias,residual", [(F16, False, False), (F32, True, False),
                                              (F16, True, True), (F32, False, True)])
def test_gemm(ctx, m, n, k, dt, bias, residual):
    g = gen(m + 3 * n + 5 * k)
    x, xs = codes(g, m, k, 16)
    w, ws = codes(g, n, k, 32)
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    r = rows_in(g, m, n, dt, 3) if residual else None
    whole = torch.full((m + 1, n + 8), 7.0, device="cuda", dtype=dt)
    y = whole[:m, :n]
    ctx.gemm_q8((w, ws), x, xs, y, bias=b, residual=r)
    check_gemm(y, x, xs, w, ws, b, r, dt)
    assert (whole[m:] == 7).all() and (whole[:, n:] == 7).all()
    if residual:  # in place, rows that start anywhere
        y2 = rows_in(g, m, n, dt, 1, 1)
        y2.copy_(r)
        ctx.gemm_q8((w, ws), x, xs, y2, bias=b, residual=y2)
        assert torch.equal(y2, y)


# Calls whose CTAs (or pairs of them) take several tiles each: a ring and two accumulators that run on across
# tiles, tokens' scales that change with the tile, MMAs of 128 rows (tests/test_q8_host.py holds which sizes
# reach what).
MANY_TILES = [(1, 32001, 256), (7, 65536, 130), (8, 65536, 128), (16, 40001, 700), (20, 20000, 512),
              (24, 65536, 256), (24, 65536, 2048), (32, 50000, 2048), (32, 40007, 333), (100, 20000, 256),
              (128, 20001, 257), (300, 20000, 128), (260, 50000, 64), (2304, 5000, 256), (2500, 5003, 128)]
MANY_GATED = [(1, 30000, 256), (8, 50000, 300), (17, 20003, 128), (33, 20000, 2048), (40, 20000, 512),
              (128, 20007, 256), (600, 9000, 256), (2300, 3000, 200)]


@pytest.mark.parametrize("m,n,k", MANY_TILES)
@pytest.mark.parametrize("dt,bias,residual", [(F32, False, False), (F16, True, True)])
def test_gemm_of_many_tiles(ctx, m, n, k, dt, bias, residual):
    g = gen(m + 3 * n + 5 * k)
    x, xs = codes(g, m, k, 16)
    w, ws = codes(g, n, k, 32)
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    r = rows_in(g, m, n, dt, 3) if residual else None
    whole = torch.full((m + 1, n + 8), 7.0, device="cuda", dtype=dt)
    y = whole[:m, :n]
    ctx.gemm_q8((w, ws), x, xs, y, bias=b, residual=r)
    check_gemm(y, x, xs, w, ws, b, r, dt)
    assert (whole[m:] == 7).all() and (whole[:, n:] == 7).all()


@pytest.mark.parametrize("m,n,k", MANY_GATED)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gate_of_many_tiles(ctx, m, n, k, act):
    g = gen(m + 3 * n + 5 * k)
    x, xs = codes(g, m, k, 16)
    (wg, gs), (wu, us) = codes(g, n, k, 32), codes(g, n, k)
    amp = 40 / (74 * 74 * math.sqrt(k) / 10000)  # outputs of both signs, from far below to far above 1
    gs, us = gs * amp * torch.rand(n, generator=g, device="cuda"), us * amp / 20
    whole = torch.full((m + 1, n + 8), 7.0, device="cuda", dtype=F16)
    h = whole[:m, :n]
    ctx.gate_q8((wg, gs), (wu, us), x, xs, h, act=act)
    check_gate(h, x, xs, wg, gs, wu, us, act)
    assert (whole[m:] == 7).all() and (whole[:, n:] == 7).all()


@pytest.mark.parametrize("m", [1, 20, 130, 600])
def test_gemm_sums_are_whole_numbers(ctx, m):
    """The longest rows of the largest codes: sums of 2^30, which f32 sums would round on the way."""
    k, n = 65536, 70
    g = gen(m)
    x, xs = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    ws = torch.ones(n, device="cuda")
    w[:, ::7] = 127
    x[:, -1] = torch.randint(-128, 128, (m,), generator=g, device="cuda").to(torch.int8)
    w[1] = torch.randint(-128, 128, (k,), generator=g, device="cuda").to(torch.int8)
    y = torch.zeros(m, n, device="cuda")
    ctx.gemm_q8((w, ws), x, xs, y)
    assert torch.equal(y, (x.double() @ w.double().T).float())


def test_gemm_rows_without_numbers(ctx):
    """A token or channel without a scale touches its own outputs only."""
    g = gen(4)
    for m in (1, 40, 300):
        x, xs = codes(g, m, 200)
        w, ws = codes(g, 150, 200)
        y0, y = torch.zeros(m, 150, device="cuda"), torch.zeros(m, 150, device="cuda")
        ctx.gemm_q8((w, ws), x, xs, y0)
        xs[m // 2], ws[77] = math.nan, math.nan
        ctx.gemm_q8((w, ws), x, xs, y)
        bad = torch.zeros_like(y, dtype=torch.bool)
        bad[m // 2], bad[:, 77] = True, True
        assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], y0[~bad])


def check_gate(h, x, xs, g, gs, u, us, act):
    p, q = product(x, xs, g, gs), product(x, xs, u, us)
    if act == "silu":
        t = p
        want = p * torch.sigmoid(p) * q
    else:
        t = 2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p**3)
        want = 0.5 * p * (1 + torch.tanh(math.sqrt(2 / math.pi) * (p + 0.044715 * p**3))) * q
    # p and q: three roundings each.  t is off by 12 of its own (three of them cubed, five operations);
    # exp turns that, and what its own argument loses, into 16 |t|; the exponential, the sum, the
    # quotient and the product lose 10 more
    close(h, want, want.abs() * (2.0**-11 + U * (16 + 16 * t.abs())) + 2.0**-25 * 1.01)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gate(ctx, m, n, k, act):
    g = gen(m + 3 * n + 5 * k)
    x, xs = codes(g, m, k, 16)
    (wg, gs), (wu, us) = codes(g, n, k, 32), codes(g, n, k)
    # outputs of both signs, from far below to far above 1
    amp = 40 / (74 * 74 * math.sqrt(k) / 10000)
    gs = gs * amp * torch.rand(n, generator=g, device="cuda")
    us = us * amp / 20
    whole = torch.full((m + 1, n + 8), 7.0, device="cuda", dtype=F16)
    h = whole[:m, :n]
    ctx.gate_q8((wg, gs), (wu, us), x, xs, h, act=act)
    check_gate(h, x, xs, wg, gs, wu, us, act)
    assert (whole[m:] == 7).all() and (whole[:, n:] == 7).all()
    h2 = rows_in(g, m, n, F16, 1, 1)
    ctx.gate_q8((wg, gs), (wu, us), x, xs, h2, act=act)
    assert torch.equal(h2, h)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m", [1, 150])
def test_gate_ends_of_the_activation(ctx, act, m):
    """Gate values out to +-1e6, where the exponential leaves f32: h is g u, or 0."""
    x = torch.full((m, 16), 0, dtype=torch.int8, device="cuda")
    x[:, 0] = 1
    w = torch.zeros(64, 16, dtype=torch.int8, device="cuda")
    w[:, 0] = torch.tensor([1, -1] * 32, device="cuda").to(torch.int8)
    xs = torch.ones(m, device="cuda")
    gs = torch.logspace(-6, 6, 64, device="cuda")
    us = 1 / gs.clamp(min=1e-2)
    h = torch.zeros(m, 64, device="cuda", dtype=F16)
    ctx.gate_q8((w, gs), (w, us), x, xs, h, act=act)
    check_gate(h, x, xs, w, gs, w, us, act)
    xs[m // 2], gs[9] = math.nan, math.nan
    ctx.gate_q8((w, gs), (w, us), x, xs, h, act=act)
    bad = torch.zeros(m, 64, dtype=torch.bool, device="cuda")
    bad[m // 2], bad[:, 9] = True, True
    assert torch.isnan(h[bad]).all() and not torch.isnan(h[~bad]).any()


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m", [1, 150, 2100])
def test_gate_of_a_large_up_value(ctx, act, m):
    """Gate values down to where exp(-t) still is an f32 number: 1 / (1 + exp(-t)) is below f32's normal
    numbers there, and a large up value brings the product back."""
    x = torch.zeros(m, 16, dtype=torch.int8, device="cuda")
    x[:, 0] = 1
    w = torch.zeros(64, 16, dtype=torch.int8, device="cuda")
    w[:, 0] = 1
    xs = torch.ones(m, device="cuda")
    t = torch.linspace(-88.6, -80, 64, device="cuda", dtype=torch.float64)
    g = t.clone()
    if act == "gelu":  # t = 2c (g + 0.044715 g^3), solved for g
        for _ in range(60):
            f = 2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g**3) - t
            g -= f / (2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g**2))
    gs, us = g.float(), torch.exp(-t).float()
    h = torch.zeros(m, 64, device="cuda", dtype=F16)
    ctx.gate_q8((w, gs), (w, us), x, xs, h, act=act)
    # (check_gate's 16 |t| roundings stay; its bound on h itself is 2^-11 and no less: nothing here is small)
    p, u = gs.double(), us.double()
    t = p if act == "silu" else 2 * math.sqrt(2 / math.pi) * (p + 0.044715 * p**3)
    want = (p / (1 + torch.exp(-t)) * u).expand(m, 64)
    assert want.abs().min() > 1
    # the quotient below 2^-126 keeps 2^-21 or more of itself
    close(h, want, want.abs() * (2.0**-11 + U * (16 + 16 * t.abs()) + 2.0**-21))


@pytest.mark.parametrize("m", [3, 200, 2100])
def test_the_same_rows_on_every_side(ctx, m):
    """One matrix as gate, up and tokens."""
    q, s = codes(gen(m), m, 256)
    s = s / 16
    h = torch.zeros(m, m, device="cuda", dtype=F16)
    ctx.gate_q8((q, s), (q, s), q, s, h)
    check_gate(h, q, s, q, s, q, s, "silu")


def test_empty_calls(ctx):
    e = torch.empty
    q, s = e((0, 64), dtype=torch.int8, device="cuda"), e(0, device="cuda")
    w, ws = codes(gen(0), 5, 64)
    ctx.gemm_q8((w, ws), q, s, e((0, 5), device="cuda"))
    ctx.gate_q8((w, ws), (w, ws), q, s, e((0, 5), device="cuda", dtype=F16))
    ctx.gemm_q8((q, s), w, ws, e((5, 0), device="cuda"))
    ctx.quantize_rows_q8(e((0, 64), device="cuda"))
    ctx.add_norm_q8(e((0, 64), device="cuda", dtype=F16), None)
    ctx.read_rows_q8(w, ws, e((0, 64), device="cuda"))
    ctx.sync()


def test_refusals(ctx):
    import p2p_b200
    w, ws = codes(gen(0), 5, 64)
    x, xs = codes(gen(1), 3, 64)
    y, f = torch.zeros(3, 5, device="cuda"), torch.zeros(3, 64, device="cuda", dtype=F16)
    odd = torch.zeros(3, 72, dtype=torch.int8, device="cuda")[:, :64]
    for call in (lambda: ctx.gemm_q8((w, ws), x[:, :32], xs, y),
                 lambda: ctx.gemm_q8((w, ws), odd, xs, y),
                 lambda: ctx.gemm_q8((w, ws), x, xs[:2], y),
                 lambda: ctx.gemm_q8((w, ws), x, xs, y[:, :4]),
                 lambda: ctx.gemm_q8((w, ws), x, xs, y.double()),
                 lambda: ctx.gemm_q8((w, ws), x, xs, y, residual=y.half()),
                 lambda: ctx.gemm_q8((w, ws), x, xs, y, bias=ws[:4]),
                 lambda: ctx.gate_q8((w, ws), (w, ws), x, xs, y),
                 lambda: ctx.gate_q8((w, ws), (w, ws), x, xs, y.half(), act="relu"),
                 lambda: ctx.add_norm_q8(f, ws),
                 lambda: ctx.add_norm_q8(f, None, y=f.float()),
                 lambda: ctx.add_norm_q8(f, None, residual=f[:2]),
                 lambda: ctx.quantize_rows_q8(f, odd),
                 lambda: ctx.quantize_rows_q8(f.T),
                 lambda: ctx.quantize_rows_q8(f.bfloat16()),
                 lambda: ctx.read_rows_q8(x, xs, f[:, :32]),
                 lambda: ctx.read_rows_q8(x, xs, f, index=xs),
                 lambda: ctx.read_rows_q8(x[:2], xs[:2], f)):
        with pytest.raises(p2p_b200.P2PError):
            call()
    ctx.sync()


def test_long_offsets(ctx):
    """Rows that start behind 2^31 bytes, and rows far apart."""
    k, n = 128, 20
    big = torch.zeros(1200000, 2048, dtype=torch.int8, device="cuda")
    table, rowsum = big[:, :k], torch.ones(1200000, device="cuda")
    g = gen(8)
    at = torch.tensor([0, 1048575, 1048577, 1199999], dtype=torch.int32, device="cuda")
    table[at.long()] = torch.randint(-127, 128, (4, k), generator=g, device="cuda").to(torch.int8)
    out = torch.zeros(4, k, device="cuda")
    ctx.read_rows_q8(table, rowsum, out, index=at)
    assert torch.equal(out, table[at.long()].float())
    # a product whose rows are all that far apart: the last n rows of the table, pitch 2^20
    far = big.view(-1)[:1048576 * n].view(n, 1048576)[:, :k]
    far.copy_(torch.randint(-127, 128, (n, k), generator=g, device="cuda").to(torch.int8))
    x, xs = codes(g, 5, k)
    for a, b in (((far, rowsum[:n]), (x, xs)), ((x, xs), (far, rowsum[:n]))):
        y = torch.zeros(len(b[0]), len(a[0]), device="cuda")
        ctx.gemm_q8(a, *b, y)
        check_gemm(y, *b, *a, None, None, F32)
    f = torch.zeros(1048577, 2048, device="cuda", dtype=F16)  # values behind 2^32 bytes
    f[-1] = torch.randn(2048, generator=g, device="cuda")
    q, s = ctx.quantize_rows_q8(f)
    check_codes(q[-1:], s[-1:], f[-1:].double(), 0)


# ---- streams, captures, a whole model ---------------------------------------------------------------
def test_two_streams_at_once(ctx):
    g = gen(5)
    w, ws = codes(g, 1000, 2048)
    xs_ = [codes(g, m, 2048) for m in (300, 8)]
    want = []
    for x, s in xs_:
        y = torch.zeros(len(x), 1000, device="cuda")
        ctx.gemm_q8((w, ws), x, s, y)
        want.append(y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs_]
    got = [torch.zeros_like(y) for y in want]
    for _ in range(20):
        for st, (x, s), y in zip(streams, xs_, got):
            ctx.gemm_q8((w, ws), x, s, y, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("norm", [False, True])
def test_outputs_that_a_call_makes_belong_to_its_stream(ctx, norm):
    """Memory that the current stream still reads is not what a call on another stream writes."""
    x = rows_in(gen(9), 300, 4096, F16)
    want = ctx.add_norm_q8(x, None) if norm else ctx.quantize_rows_q8(x)
    side = torch.cuda.Stream()
    old, sums = torch.ones(300, 4096, dtype=torch.int8, device="cuda"), torch.ones(300, device="cuda")
    torch.cuda.synchronize()
    at = {t.untyped_storage().data_ptr() for t in (old, sums)}
    torch.cuda._sleep(20000000)
    copies = old.clone(), sums.clone()
    del old, sums  # the allocator may give them away on this stream, whose copies have yet to run
    q, s = ctx.add_norm_q8(x, None, stream=side) if norm else ctx.quantize_rows_q8(x, stream=side)
    assert not at & {t.untyped_storage().data_ptr() for t in (q, s)}
    torch.cuda.synchronize()
    assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    assert all((c == 1).all() for c in copies)


@pytest.mark.parametrize("m,n,k", [(8, 64, 1024), (8, 4000, 256), (2100, 700, 1000)])
def test_a_wait_that_runs_out_is_a_status(ctx, m, n, k):
    """The first stage of every ring waits for bytes that never come: the call ends, nothing is stored,
    p2p_sync says so, and the next call is as ever.  (k split over clusters, one CTA a tile, pairs.)"""
    import p2p_b200
    g = gen(7)
    x, xs = codes(g, m, k)
    w, ws = codes(g, n, k)
    y = torch.full((m, n), 3.0, device="cuda")
    p2p_b200.lib.p2p_debug_set_wait_deficit(16)
    try:
        ctx.gemm_q8((w, ws), x, xs, y)
    finally:
        p2p_b200.lib.p2p_debug_set_wait_deficit(0)
    with pytest.raises(p2p_b200.P2PError) as e:
        ctx.sync()
    assert e.value.status == p2p_b200.P2P_ERR_TIMEOUT
    assert (y == 3).all()
    ctx.gemm_q8((w, ws), x, xs, y)
    check_gemm(y, x, xs, w, ws, None, None, F32)
    ctx.sync()


FIRST = """
import sys
sys.path.insert(0, {root!r})
import torch, p2p_b200
ctx = p2p_b200.Context(0)
w = torch.randint(-127, 128, (700, 1024), device="cuda").to(torch.int8)
s = torch.rand(700, device="cuda")
xs = [torch.randint(-127, 128, (m, 1024), device="cuda").to(torch.int8) for m in (1, 100, 2100)]
t = torch.rand(2100, device="cuda")
ys = [torch.zeros(len(x), 700, device="cuda") for x in xs]
hs = [torch.zeros(len(x), 700, device="cuda", dtype=torch.float16) for x in xs]
f = torch.randn(2100, 1024, device="cuda", dtype=torch.float16)
q, c = torch.zeros(2100, 1024, device="cuda", dtype=torch.int8), torch.zeros(2100, device="cuda")
v = torch.zeros_like(f)
def calls():
    for x, y, h in zip(xs, ys, hs):
        ctx.gemm_q8((w, s), x, t[:len(x)], y)
        ctx.gate_q8((w, s), (w, s), x, t[:len(x)], h)
    ctx.add_norm_q8(f, None, q, c)
    ctx.quantize_rows_q8(f, q, c)
    ctx.read_rows_q8(q, c, v)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    calls()
g.replay()
torch.cuda.synchronize()
outs = ys + hs + [q, c, v]
got = [y.clone() for y in outs]
calls()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, outs))
assert all((a == a).all() and a.abs().max() > 0 for a in got[:3])
print("same")
"""


def test_first_calls_of_a_process_captured():
    """Nothing has to be called before a capture: no workspace, no first call that sets anything up on a
    stream."""
    import subprocess
    import sys
    from conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST.format(root=str(ROOT))], capture_output=True,
                       text=True, timeout=120)
    assert r.stdout.strip() == "same", r.stderr[-2000:]


class Model:
    """A decoder layer of 4 query heads and 2 kv heads with an embedding that is the LM head too,
    every product in 8 bits."""

    def __init__(self, ctx, seed=0, hidden=320, ffn=500, vocab=1000, hq=4, hkv=2):
        import p2p_b200
        g = gen(seed)
        self.ctx, self.prm, self.hidden, self.vocab = ctx, p2p_b200.Params(hq, hkv), hidden, vocab

        def matrix(n, k):
            return ctx.quantize_rows_q8(torch.randn(n, k, generator=g, device="cuda", dtype=F16)
                                        / math.sqrt(k))
        self.table = ctx.quantize_rows_q8(torch.randn(vocab, hidden, generator=g, device="cuda"))
        self.qkv, self.o = matrix(self.prm.qkv_width, hidden), matrix(hidden, hq * 64)
        self.gate, self.up, self.down = matrix(ffn, hidden), matrix(ffn, hidden), matrix(hidden, ffn)
        self.norms = [(1 + 0.2 * torch.randn(hidden, generator=g, device="cuda")).half()
                      for _ in range(3)]
        self.rope = ctx.rope_table(64)
        self.ffn = ffn

    def buffers(self, m):
        z = lambda *s, dt=F16: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
        p = self.prm
        return {"x": z(m, self.hidden), "res": z(m, self.hidden), "qkv": z(m, p.qkv_width),
                "rot": z(m, p.num_heads * 64), "att": z(m, p.num_heads * 64),
                "h": z(m, self.ffn), "logits": z(m, self.vocab, dt=F32),
                "tok": z(m, dt=torch.int32),
                "k": z(200, p.num_kv_heads, 64), "v": z(200, p.num_kv_heads, 64),
                **{n: empty_q8(m, w)[1:] for n, w in (
                    ("a", self.hidden), ("b", p.num_heads * 64), ("c", self.hidden),
                    ("d", self.ffn), ("e", self.hidden))}}

    def step(self, b, tokens, past, start, check=False):
        c = self.ctx
        off = torch.arange(len(past), device="cuda", dtype=torch.int32) * 64
        c.read_rows_q8(*self.table, b["x"], index=tokens)
        c.add_norm_q8(b["x"], self.norms[0], *b["a"])
        c.gemm_q8(self.qkv, *b["a"], b["qkv"])
        c.kv_append(self.prm, b["qkv"], None, self.rope, b["k"], b["v"], past, start, max_len=64,
                    q_out=b["rot"], offsets=off)
        c.attn_chunk_kv(self.prm, b["rot"], b["k"], b["v"], past, start, b["att"], max_len=64,
                        offsets=off)
        c.quantize_rows_q8(b["att"], *b["b"])
        c.gemm_q8(self.o, *b["b"], b["res"], residual=b["x"])
        if check:
            check_norm(b["x"], None, self.norms[0], 1e-5, F16, *b["a"])
            check_gemm(b["qkv"], *b["a"], *self.qkv, None, None, F16)
            check_codes(*b["b"], b["att"].double(), 0)
            check_gemm(b["res"], *b["b"], *self.o, None, b["x"], F16)
        c.add_norm_q8(b["res"], self.norms[1], *b["c"])
        c.gate_q8(self.gate, self.up, *b["c"], b["h"])
        c.quantize_rows_q8(b["h"], *b["d"])
        c.gemm_q8(self.down, *b["d"], b["res"], residual=b["res"])
        c.add_norm_q8(b["res"], self.norms[2], *b["e"])
        c.gemm_q8(self.table, *b["e"], b["logits"])
        c.logits_pick(b["logits"], b["tok"])
        if check:
            check_gate(b["h"], *b["c"], *self.gate, *self.up, "silu")
            check_codes(*b["d"], b["h"].double(), 0)
            check_norm(b["res"], None, self.norms[2], 1e-5, F16, *b["e"])
            check_gemm(b["logits"], *b["e"], *self.table, None, None, F32)
            assert torch.equal(b["tok"].long(), b["logits"].argmax(1))


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("lens", [(1,), (5, 1, 30), (40, 41, 60)])
def test_a_model_in_8_bits(ctx, lens):
    """A prompt chunk of every sequence, then steps of a token each whose tokens stay on the device:
    eager, and captured once and replayed."""
    mdl = Model(ctx)
    n, m = len(lens), sum(lens)
    g = gen(sum(lens))
    tokens = torch.randint(0, mdl.vocab, (m,), generator=g, device="cuda", dtype=torch.int32)
    start = i32(itertools.accumulate((0, *lens)))
    b = mdl.buffers(m)
    mdl.step(b, tokens, i32([0] * n), start, check=True)
    last = (start[1:] - 1).long()

    def steps(captured):
        d = mdl.buffers(n)
        d["k"].copy_(b["k"])
        d["v"].copy_(b["v"])
        d["tok"].copy_(b["tok"][last])
        past, one = i32(lens), i32(range(n + 1))
        mdl.step(d, d["tok"], past, one, check=not captured)
        made = [d["tok"].clone()]
        graph = None
        if captured:
            past += 1
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                mdl.step(d, d["tok"], past, one)
            past -= 1
        for _ in range(3):
            past += 1
            graph.replay() if graph else mdl.step(d, d["tok"], past, one)
            made.append(d["tok"].clone())
        return made, d["res"].clone(), d["k"].clone()
    eager, graph = steps(False), steps(True)
    assert all(torch.equal(x, y) for x, y in zip(eager[0], graph[0]))
    assert torch.equal(eager[1], graph[1]) and torch.equal(eager[2], graph[2])
    ctx.sync()
