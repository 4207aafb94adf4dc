"""The 8-bit layer operators without a GPU: what their host side refuses, with made-up addresses and
launchers that only count, and what the Python layer refuses before it."""
import ctypes as C
import subprocess

import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")

BAD, UNSUPPORTED = 1, 7
MB = 1 << 20


@pytest.fixture(scope="module")
def api(tmp_path_factory):
    import importlib.util
    from p2p_b200._lib import PROTOTYPES
    spec = importlib.util.spec_from_file_location("p2p_build", ROOT / "p2p_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    so = tmp_path_factory.mktemp("q8_api") / "q8_api_host.so"
    subprocess.run([build.nvcc(), *build.ARCH, *build.NVCC_FLAGS, "-shared", "-cudart", "static",
                    str(ROOT / "tests" / "q8_api_host.cu"), "-o", str(so)], check=True,
                   capture_output=True)
    lib = C.CDLL(str(so))
    for name in ("p2p_quantize_rows_q8", "p2p_read_rows_q8", "p2p_add_norm_q8", "p2p_gemm_q8",
                 "p2p_gate_q8"):
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = PROTOTYPES[name]
    lib.host_message.restype = C.c_char_p
    return lib


def rows(at, n=4, k=64, ld=None, scale=None):
    """int8 rows at a made-up address, their scales 2^16 bytes behind them unless given."""
    from p2p_b200._lib import Q8Rows
    return Q8Rows(at, at + 65536 if scale is None else scale, (k + 15) // 16 * 16 if ld is None
                  else ld, n, k)


def said(api, status, want, text=None):
    assert status == want, api.host_message()
    if text:
        assert text in api.host_message().decode(), api.host_message()


CTX = 1  # not NULL


def test_null_context_is_a_status():
    from p2p_b200 import _lib, lib
    g = _lib.AddNorm()
    assert lib.p2p_quantize_rows_q8(None, C.byref(_lib.QuantizeRows()), None) == BAD
    assert lib.p2p_read_rows_q8(None, C.byref(_lib.ReadRows()), None) == BAD
    assert lib.p2p_add_norm_q8(None, C.byref(g), None) == BAD
    assert lib.p2p_gemm_q8(None, C.byref(_lib.Product()), None) == BAD
    assert lib.p2p_gate_q8(None, C.byref(_lib.Gated()), None) == BAD


def test_packed_structures_are_the_c_ones():
    """The Python layer packs the argument structures itself: sizes and offsets have to be the C ones."""
    from p2p_b200 import _lib, attention as A

    def flat(t, at=0):
        for name, kind in t._fields_:
            off = at + getattr(t, name).offset
            if issubclass(kind, C.Structure):
                yield from flat(kind, off)
            else:
                yield off, kind
    for pack, t in ((A._QUANTIZE_ROWS, _lib.QuantizeRows), (A._READ_ROWS, _lib.ReadRows),
                    (A._ADD_NORM, _lib.AddNorm), (A._PRODUCT, _lib.Product),
                    (A._GATED, _lib.Gated)):
        fields = list(flat(t))
        values = [float(i + 1) if kind is C.c_float else i + 1 for i, (_, kind) in enumerate(fields)]
        data = pack(*values)
        assert len(data) == C.sizeof(t)
        for (off, kind), v in zip(fields, values):
            assert kind.from_buffer_copy(data, off).value == v, (t, off)


def quantize(api, dst, src=MB, ld=64, dtype=0):
    from p2p_b200._lib import QuantizeRows
    a = QuantizeRows(src, ld, dst, dtype) if dst else None
    return api.p2p_quantize_rows_q8(CTX, C.byref(a) if a else None, None)


def test_quantize_refusals(api):
    before = api.host_launches()
    good = rows(4 * MB)
    said(api, quantize(api, good), 0)
    assert api.host_launches() == before + 1
    said(api, quantize(api, rows(4 * MB, n=0), src=None), 0)  # nothing to do
    said(api, quantize(api, None), BAD, "NULL")
    said(api, quantize(api, good, dtype=2), UNSUPPORTED)
    said(api, quantize(api, good, src=None), BAD)
    said(api, quantize(api, good, src=MB + 1), BAD)
    said(api, quantize(api, good, src=MB + 2, dtype=1), BAD)
    said(api, quantize(api, good, ld=63), BAD)
    for bad in (rows(4 * MB, n=-1), rows(4 * MB, n=2**30 + 1), rows(4 * MB, k=0), rows(4 * MB, k=65537), rows(4 * MB + 8),
                rows(4 * MB, ld=72), rows(4 * MB, ld=48), rows(4 * MB, scale=5 * MB + 2),
                rows(0, scale=MB)):
        said(api, quantize(api, bad), BAD)
    bad = rows(4 * MB)
    bad.scale = None
    said(api, quantize(api, bad), BAD)
    # overlaps: codes in the source, scales in the source, scales in the codes
    said(api, quantize(api, rows(MB + 128)), BAD, "overlaps")
    said(api, quantize(api, rows(4 * MB, scale=MB + 64)), BAD, "overlaps")
    said(api, quantize(api, rows(4 * MB, scale=4 * MB + 192)), BAD, "overlaps")
    # columns of one buffer beside each other are apart
    said(api, quantize(api, rows(MB + 128, ld=256), ld=128), 0)
    assert api.host_launches() == before + 2


def read(api, src, n=4, index=None, out=MB, ld=64, dtype=0, factor=1.0):
    from p2p_b200._lib import ReadRows
    a = ReadRows(src, index, out, ld, n, dtype, factor) if src else None
    return api.p2p_read_rows_q8(CTX, C.byref(a) if a else None, None)


def test_read_refusals(api):
    before = api.host_launches()
    good = rows(4 * MB)
    said(api, read(api, good), 0)
    said(api, read(api, good, n=9, index=8 * MB), 0)
    said(api, read(api, good, n=0, out=None), 0)
    assert api.host_launches() == before + 2
    said(api, read(api, None), BAD)
    said(api, read(api, good, n=5), BAD)  # more rows than there are, in order
    said(api, read(api, good, n=-1, index=8 * MB), BAD)
    said(api, read(api, good, n=2**30 + 1, index=2**45), BAD)
    said(api, read(api, good, index=8 * MB + 2), BAD)
    said(api, read(api, good, dtype=5), UNSUPPORTED)
    said(api, read(api, good, out=None), BAD)
    said(api, read(api, good, ld=63), BAD)
    said(api, read(api, good, out=4 * MB + 64), BAD, "overlaps")
    said(api, read(api, good, out=4 * MB + 65536), BAD, "overlaps")
    said(api, read(api, good, n=9, index=MB + 8), BAD, "overlaps")
    assert api.host_launches() == before + 2


def norm(api, **kw):
    from p2p_b200._lib import AddNorm
    g = AddNorm()
    g.x, g.residual, g.weight, g.sum, g.y = MB, 2 * MB, 3 * MB, 5 * MB, 6 * MB
    g.ld_x = g.ld_r = g.ld_sum = g.ld_y = 64
    g.out = rows(4 * MB)
    for k, v in kw.items():
        setattr(g, k, v)
    return api.p2p_add_norm_q8(CTX, C.byref(g), None)


def test_norm_refusals(api):
    from p2p_b200._lib import Q8Rows
    before = api.host_launches()
    said(api, norm(api), 0)
    said(api, norm(api, residual=None, weight=None, sum=None, y=None), 0)
    said(api, norm(api, out=Q8Rows(None, None, 0, 4, 64)), 0)  # no codes wanted
    said(api, norm(api, sum=MB), 0)                            # in place
    said(api, norm(api, sum=2 * MB, y=MB), 0)
    assert api.host_launches() == before + 5
    said(api, norm(api, out=rows(4 * MB, n=0), x=None), 0)
    said(api, api.p2p_add_norm_q8(CTX, None, None), BAD)
    said(api, norm(api, out=Q8Rows(None, None, 0, 4, 64), sum=None, y=None), BAD, "all NULL")
    said(api, norm(api, out=Q8Rows(None, None, 0, 4, 0)), BAD)
    said(api, norm(api, out=Q8Rows(None, None, 0, -1, 64)), BAD)
    said(api, norm(api, out=Q8Rows(None, None, 0, 2**30 + 1, 64)), BAD)
    said(api, norm(api, out=rows(4 * MB, ld=72)), BAD)
    said(api, norm(api, dtype=3), UNSUPPORTED)
    for eps in (-1.0, float("nan"), float("inf")):
        said(api, norm(api, eps=eps), BAD, "eps")
    for bad in ({"x": None}, {"x": MB + 1}, {"ld_x": 63}, {"ld_r": 63}, {"ld_sum": 63},
                {"ld_y": 63}, {"weight": 3 * MB + 1}, {"y": 6 * MB + 1}):
        said(api, norm(api, **bad), BAD)
    for bad in ({"sum": MB, "ld_sum": 80}, {"sum": MB + 2}, {"y": 2 * MB + 128}, {"y": 5 * MB},
                {"sum": 3 * MB}, {"sum": 4 * MB}, {"y": 4 * MB + 65536}, {"out": rows(MB)},
                {"out": rows(3 * MB)}, {"out": rows(4 * MB, scale=MB + 4)}):
        said(api, norm(api, **bad), BAD, "overlaps")
    assert api.host_launches() == before + 5


def gemm(api, w=None, x=None, bias=None, res=None, ld_r=0, y=MB, ld_y=32, dtype=0):
    w = w or rows(4 * MB, n=32)
    x = x or rows(8 * MB)
    from p2p_b200._lib import Product
    return api.p2p_gemm_q8(CTX, C.byref(Product(w, x, bias, res, y, ld_r, ld_y, dtype)), None)


def test_gemm_refusals(api):
    before = api.host_launches()
    said(api, gemm(api), 0)
    said(api, gemm(api, bias=2 * MB, res=3 * MB, ld_r=40, dtype=1), 0)
    said(api, gemm(api, res=MB, ld_r=32), 0)  # in place
    said(api, gemm(api, x=rows(8 * MB, n=1), res=MB, ld_r=99), 0)
    assert api.host_launches() == before + 4
    said(api, api.p2p_gemm_q8(CTX, None, None), BAD)
    said(api, gemm(api, x=rows(8 * MB, n=0), y=None), 0)
    said(api, gemm(api, w=rows(8 * MB, n=0), y=None), 0)
    said(api, gemm(api, x=rows(8 * MB, k=65)), BAD, "64 and 65")
    said(api, gemm(api, dtype=2), UNSUPPORTED)
    for bad in ({"y": None}, {"ld_y": 31}, {"y": MB + 1}, {"y": MB + 2, "dtype": 1},
                {"res": 3 * MB, "ld_r": 31}, {"res": 3 * MB + 1, "ld_r": 32}, {"bias": 2 * MB + 2},
                {"w": rows(4 * MB + 4, n=32)}, {"x": rows(8 * MB, ld=80 + 8)}):
        said(api, gemm(api, **bad), BAD)
    for bad in ({"res": MB, "ld_r": 48}, {"res": MB + 64, "ld_r": 32}, {"y": 4 * MB},
                {"y": 8 * MB}, {"y": 8 * MB + 65536}, {"bias": MB + 64}):
        said(api, gemm(api, **bad), BAD, "overlaps")
    assert api.host_launches() == before + 4


def gate(api, g=None, u=None, x=None, act=0, h=MB, ld_h=32):
    g = g or rows(4 * MB, n=32)
    u = u or rows(6 * MB, n=32)
    x = x or rows(8 * MB)
    from p2p_b200._lib import Gated
    return api.p2p_gate_q8(CTX, C.byref(Gated(g, u, x, h, ld_h, act)), None)


def test_gate_refusals(api):
    before = api.host_launches()
    said(api, gate(api), 0)
    said(api, gate(api, act=1), 0)
    said(api, gate(api, u=rows(4 * MB, n=32)), 0)  # the same weights twice
    assert api.host_launches() == before + 3
    said(api, api.p2p_gate_q8(CTX, None, None), BAD)
    said(api, gate(api, x=rows(8 * MB, n=0), h=None), 0)
    for bad in ({"act": 2}, {"act": -1}, {"u": rows(6 * MB, n=31)}, {"u": rows(6 * MB, n=32, k=63)},
                {"x": rows(8 * MB, k=63)}, {"h": None}, {"h": MB + 1}, {"ld_h": 31},
                {"g": rows(4 * MB + 1, n=32)}):
        said(api, gate(api, **bad), BAD)
    for bad in ({"h": 4 * MB}, {"h": 6 * MB + 64}, {"h": 8 * MB}):
        said(api, gate(api, **bad), BAD, "overlaps")
    assert api.host_launches() == before + 3


def test_python_refusals():
    import p2p_b200
    ctx = object.__new__(p2p_b200.Context)
    ctx.h, ctx.device = None, 0
    f = torch.zeros(3, 64, dtype=torch.float16)
    q, s = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3)
    for call in (lambda: ctx.quantize_rows_q8(f), lambda: ctx.read_rows_q8(q, s, f),
                 lambda: ctx.add_norm_q8(f, None), lambda: ctx.gemm_q8((q, s), q, s, f),
                 lambda: ctx.gate_q8((q, s), (q, s), q, s, f)):
        with pytest.raises(p2p_b200.P2PError):  # nothing of this is on a device
            call()


class Streams:
    """Stands for the library and torch's streams: which stream was the allocator's at each torch.empty, and
    the handle that each call got."""

    def __init__(self, monkeypatch):
        import contextlib
        from p2p_b200 import attention as A
        self.current, self.made, self.calls = None, [], []
        empty = torch.empty

        @contextlib.contextmanager
        def stream(s):
            before, self.current = self.current, s
            yield
            self.current = before

        def recorded(*a, **kw):
            self.made.append(self.current)
            return empty(*a, **kw)
        monkeypatch.setattr(torch.cuda, "stream", stream)
        monkeypatch.setattr(torch, "empty", recorded)
        monkeypatch.setattr(A, "lib", self)

    def __getattr__(self, name):
        def call(*a):
            self.calls.append((name, a))
            return 0
        return call


class Side:
    cuda_stream = 77


def host_context():
    """A context whose device is that of CPU tensors."""
    import p2p_b200
    ctx = object.__new__(p2p_b200.Context)
    ctx.h, ctx.device = None, -1
    return ctx


def test_outputs_are_made_on_the_stream_of_the_call(monkeypatch):
    ctx, f, side = host_context(), torch.zeros(3, 64, dtype=torch.float16), Side()
    q, s = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3)
    seen = Streams(monkeypatch)
    for call, made in ((lambda: ctx.quantize_rows_q8(f, stream=side), 2),
                       (lambda: ctx.quantize_rows_q8(f, q, stream=side), 1),
                       (lambda: ctx.add_norm_q8(f, None, stream=side), 2),
                       (lambda: ctx.add_norm_q8(f, None, scale=s, stream=side), 1),
                       (lambda: ctx.quantize_rows_q8(f, q, s, stream=side), 0)):
        seen.made.clear()
        out = call()
        assert seen.made == [side] * made and seen.calls[-1][1][-1] == 77
        assert out[0].shape == (3, 64) and out[1].shape == (3,)


def test_copies_in_other_formats_are_made_on_the_stream_of_the_call(monkeypatch):
    ctx, side = host_context(), Side()
    rows = torch.zeros(5, 2, 64, dtype=torch.float16)
    w = (torch.zeros(8, 8, dtype=torch.int32), torch.zeros(8, 2, dtype=torch.float16),
         torch.zeros(2, dtype=torch.int32))
    seen = Streams(monkeypatch)
    monkeypatch.setattr("p2p_b200.attention.kv_q4_row_bytes", lambda hkv: 72 * hkv)
    for call, shape in ((lambda: ctx.kv_quantize_q4(rows, stream=side), (5, 144)),
                        (lambda: ctx.kv_quantize_q8(rows, torch.ones(1), stream=side), (5, 2, 64)),
                        (lambda: ctx.q4_to_f16(w, stream=side), (8, 64))):
        seen.made.clear()
        out = call()
        assert seen.made == [side] and tuple(out.shape) == shape
        handle = seen.calls[-1][1][-1]
        assert getattr(handle, "value", handle) == 77


def test_no_eps_is_taken_for_another_one(monkeypatch):
    """0 and what rounds to it select 1e-5 in the C structure: never what a caller of the Python layer means."""
    import p2p_b200
    ctx, f = host_context(), torch.zeros(3, 64, dtype=torch.float16)
    seen = Streams(monkeypatch)
    for eps in (0.0, -0.0, 0, 1e-50, 1e-39, -1e-5, 1e39, 1e400, float("nan")):
        with pytest.raises(p2p_b200.P2PError, match="eps"):
            ctx.add_norm_q8(f, None, eps=eps, stream=Side())
    assert not seen.calls
    for eps in (1e-37, 1e-6, 1, 1e38):
        ctx.add_norm_q8(f, None, eps=eps, stream=Side())
    assert len(seen.calls) == 4


def test_no_factor_is_taken_for_another_one(api, monkeypatch):
    """0 and what rounds to it select 1 in the C structure; an infinity would make NaN of the rows of zeros
    that an index of -1 gives."""
    import p2p_b200
    before, good = api.host_launches(), rows(4 * MB)
    for factor in (float("inf"), float("-inf"), float("nan")):
        said(api, read(api, good, factor=factor), BAD, "factor")
    for factor in (0.0, -2.0, 3.4028234663852886e38):
        said(api, read(api, good, factor=factor), 0)
    assert api.host_launches() == before + 3
    ctx, f = host_context(), torch.zeros(3, 64, dtype=torch.float16)
    q, s = torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3)
    seen = Streams(monkeypatch)
    for factor in (0.0, 1e-50, -1e-50, 1e39, -1e400, float("nan")):
        with pytest.raises(p2p_b200.P2PError, match="factor"):
            ctx.read_rows_q8(q, s, f, factor=factor, stream=Side())
    assert not seen.calls
    for factor in (1e-37, -1, 1e38):
        ctx.read_rows_q8(q, s, f, factor=factor, stream=Side())
    assert len(seen.calls) == 3


def test_sizes_beyond_32_bits_are_refused(monkeypatch):
    """As any other argument, not by an error of the packing."""
    import p2p_b200
    ctx, many = host_context(), 2**31
    ctx.device = torch.empty(1, device="meta").get_device()
    z = lambda *s, dt=torch.int8: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
    f16, f32 = torch.float16, torch.float32
    tall, wide, one = (z(many, 16), z(many, dt=f32)), (z(1, many), z(1, dt=f32)), (z(1, 16), z(1, dt=f32))
    seen = Streams(monkeypatch)
    for call in (lambda: ctx.read_rows_q8(*one, z(many, 16, dt=f16), stream=Side()),
                 lambda: ctx.read_rows_q8(*tall, z(1, 16, dt=f16), stream=Side()),
                 lambda: ctx.quantize_rows_q8(z(many, 16, dt=f16), *tall, stream=Side()),
                 lambda: ctx.quantize_rows_q8(z(1, many, dt=f16), *wide, stream=Side()),
                 lambda: ctx.add_norm_q8(z(many, 16, dt=f16), None, *tall, stream=Side()),
                 lambda: ctx.gemm_q8(tall, *one, z(1, many, dt=f16), stream=Side()),
                 lambda: ctx.gate_q8(one, one, *tall, z(many, 1, dt=f16), stream=Side())):
        with pytest.raises(p2p_b200.P2PError):
            call()
    assert not seen.calls


# ---- how products are cut up --------------------------------------------------------------------------
@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """plan(m, n, k, gate): what gemm_q8.cu makes of a call on 148 SMs that run 74, 35 and 15 clusters of 2, 4
    and 8 CTAs at once (or those of `room`)."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("p2p_build", ROOT / "p2p_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    so = tmp_path_factory.mktemp("q8_plan") / "q8_plan_host.so"
    subprocess.run([build.nvcc(), *build.ARCH, *build.NVCC_FLAGS, "-shared", "-cudart", "static",
                    str(ROOT / "tests" / "q8_plan_host.cu"), "-o", str(so)], check=True,
                   capture_output=True)
    lib = C.CDLL(str(so))

    def call(m, n, k, gate=False, room=(74, 35, 15)):
        o = (C.c_int64 * 10)()
        lib.host_plan(m, n, k, int(gate), 148, sum(r << (8 * i) for i, r in enumerate(room)), o)
        if o[0]:
            return {"kernel": "wide", "whole": o[1], "items": o[2]}
        names = ("rows", "tokens", "split", "chunks", "steps", "tiles", "stages", "smem", "cols")
        return {"kernel": "narrow", **dict(zip(names, o[1:]))}
    return call


def shapes(count):
    import random
    rng = random.Random(1)
    for _ in range(count):
        yield (int(2**rng.uniform(0, 11.1)), int(2**rng.uniform(0, 17)), int(2**rng.uniform(0, 16)),
               rng.random() < 0.5, rng.choice([(74, 35, 15), (74, 36, 16), (60, 20, 7), (1, 1, 1)]))


def test_split_ctas_find_their_tensor_memory(plan):
    """CTAs of a cluster wait for one another: whatever of them fits on an SM by its 228 KB of shared memory
    (1 KB of it kept of each) has to fit into its 512 columns too."""
    seen = set()
    for m, n, k, gate, room in ((128, 512, 512, True, (74, 35, 15)), (64, 256, 512, False, (74, 35, 15)),
                                *shapes(4000)):
        p = plan(m, n, k, gate, room)
        if p["kernel"] == "wide":
            continue
        assert 1 <= p["stages"] <= 24 and p["smem"] <= 227 * 1024 and p["cols"] <= 512
        if p["split"] > 1:
            seen.add(p["cols"])
            assert (p["smem"] + 1024) * 512 >= p["cols"] * 228 * 1024, (m, n, k, gate, p)
            assert p["smem"] >= 48 * 1024  # none beside a pair form's CTA
    assert seen == {32, 64, 128, 256}


def test_products_take_known_instruction_shapes(plan):
    """Integer MMAs of 8 columns or a multiple of 16 (of 64 rows, 24 too), over whole swizzle atoms of rows."""
    for m in range(1, 131):
        for n, k, gate in ((65536, 2048, False), (20000, 512, False), (2048, 2048, False),
                           (30000, 300, True), (8192, 2048, True), (100, 77, True)):
            p = plan(m, n, k, gate)
            if p["kernel"] == "narrow":
                t = p["tokens"]
                assert t == 8 or t % 16 == 0 or (t == 24 and p["rows"] <= 64), (m, n, k, gate, p)
                assert min(m, 128) <= t <= 128
                assert p["rows"] % 8 == 0 and 8 <= p["rows"] <= 128


def test_sizes_of_the_gpu_tests_reach_every_walk(plan):
    """A CTA's second tile (other accumulator), its third (the first accumulator handed back), a ring that goes
    round, MMAs of 64 and 128 rows, tiles of few and of many tokens, pairs of CTAs with three items, and
    clusters: among the sizes that are compared on a GPU."""
    import test_gpu_q8 as T
    for gate, many in ((False, T.MANY_TILES), (True, T.MANY_GATED)):
        plans = [plan(*c, gate) for c in many]
        walks = [p for p in plans if p["kernel"] == "narrow" and p["split"] == 1 and p["tiles"] > 148]
        assert any(p["tiles"] > 2 * 148 for p in walks)
        assert any(p["stages"] < p["steps"] * (p["tiles"] // 148) for p in walks)
        assert {8, 32, 128} <= {p["tokens"] for p in walks}
        assert any(p["rows"] > 64 and p["tokens"] == 8 for p in walks)
        assert any(p["items"] > 2 * 74 for p in plans if p["kernel"] == "wide")
    assert any(p["rows"] <= 64 for p in (plan(*c) for c in T.MANY_TILES) if p.get("tiles", 0) > 2 * 148)
    for gate in (False, True):
        few = [plan(*c, gate) for c in T.SIZES]
        assert {2, 4, 8} <= {p["split"] for p in few if p["kernel"] == "narrow"}
        assert any(p["items"] < 74 for p in few if p["kernel"] == "wide")
