"""The batched serving operators without a GPU: refusals of their host-side checks, and the
address arithmetic of ragged chunks over paged and contiguous caches (bad pages, negative
lengths, ends of the pool) compiled for the host."""
import ctypes as C
import subprocess

import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")

I32_MAX = 2**31 - 1


def test_null_context_is_a_status():
    from p2p_b200 import _lib, lib
    lay, prm, lg = _lib.KvLayout(), _lib.AttnParams(32, 8, 64, 0, 0, 0), _lib.Logits()
    assert lib.p2p_kv_append(None, C.byref(prm), C.byref(lay), None, 0, None, None, None, None, 0,
                             None, None, None, 0, 0, 0, None, 0, None) == 1
    assert lib.p2p_kv_read(None, C.byref(lay), 8, None, None, 0, None, None, None, 0, 0, 0, None,
                           None, None) == 1
    assert lib.p2p_attn_chunk_kv(None, C.byref(prm), C.byref(lay), None, 0, None, None, 0, None,
                                 None, None, 0, 0, 0, None, 0, None) == 1
    assert lib.p2p_logits_pick(None, C.byref(lg), None) == 1
    assert lib.p2p_kv_quantize_q4(None, None, None, 0, 8, None) == 1


@pytest.mark.parametrize("hkv,want", [(0, 0), (-3, 0), (1, 48), (2, 80), (3, 112), (4, 144),
                                      (8, 288), (12, 432), (32, 1152)])
def test_row_bytes(hkv, want):
    from p2p_b200 import kv_q4_row_bytes
    assert kv_q4_row_bytes(hkv) == want


def test_python_refusals():
    import p2p_b200
    ctx = object.__new__(p2p_b200.Context)
    ctx.h, ctx.device = None, 0
    prm = p2p_b200.Params(4, 2)
    ints = torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(3, 8 * 64, dtype=torch.float16)
    cache = torch.zeros(16, 2, 64, dtype=torch.float16)
    with pytest.raises(p2p_b200.P2PError):  # nothing of this is on a device
        ctx.kv_append(prm, f, None, f, cache, cache, ints, ints, max_len=4, offsets=ints)
    with pytest.raises(p2p_b200.P2PError):
        ctx.attn_chunk_kv(prm, f, cache, cache, ints, ints, f, max_len=4, offsets=ints)
    with pytest.raises(p2p_b200.P2PError):
        ctx.kv_read(prm, cache, cache, ints, ints, cache, cache, max_len=4, offsets=ints)
    with pytest.raises(p2p_b200.P2PError):
        ctx.kv_quantize_q4(cache)
    with pytest.raises(p2p_b200.P2PError):
        ctx.logits_pick(f, ints)
    u8 = torch.zeros(16, 80, dtype=torch.uint8)
    with pytest.raises(p2p_b200.P2PError):
        ctx.attn_decode_kv(prm, f, None, None, u8, u8, ints, f, max_past=3, offsets=ints,
                           fused_prep=False)


@pytest.fixture(scope="module")
def host_rows(tmp_path_factory):
    import importlib.util
    spec = importlib.util.spec_from_file_location("p2p_build", ROOT / "p2p_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    exe = tmp_path_factory.mktemp("kv_view") / "kv_view_host"
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr", "-I",
                    str(build.CSRC), str(ROOT / "tests" / "kv_view_host.cu"), "-o", str(exe)],
                   check=True, capture_output=True)

    def ask(paged, kv_rows, past, r0, r1, n_rows, max_len, shift=4, offset=0, table=()):
        line = " ".join(str(x) for x in (int(paged), kv_rows, shift, len(table), past, r0, r1,
                                         n_rows, max_len, offset, *table))
        out = subprocess.run([str(exe)], input=line + "\n", capture_output=True, text=True,
                             check=True).stdout.split()
        return bool(int(out[0])), [int(x) for x in out[1:]]
    return ask


def test_contiguous_rows(host_rows):
    assert host_rows(False, 10, 3, 0, 4, 4, 10, offset=2) == (True, [5, 6, 7, 8])
    assert host_rows(False, 9, 3, 0, 4, 4, 10, offset=2) == (True, [5, 6, 7, 8])
    assert not host_rows(False, 8, 3, 0, 4, 4, 10, offset=2)[0]  # one row behind the cache
    assert not host_rows(False, 100, 3, 0, 4, 4, 6)[0]           # longer than max_len
    assert not host_rows(False, 100, -1, 0, 4, 4, 60)[0]
    assert not host_rows(False, 100, 3, 0, 4, 4, 60, offset=-1)[0]
    assert not host_rows(False, 100, 3, 0, 5, 4, 60)[0]          # rows behind n_rows
    assert not host_rows(False, 100, 3, 4, 2, 4, 60)[0]          # a negative length
    assert not host_rows(False, 100, 3, -2, 2, 4, 60)[0]
    assert host_rows(False, 100, 3, 2, 2, 4, 60) == (True, [])   # an empty chunk


def test_sums_near_the_end_of_32_bits(host_rows):
    assert not host_rows(False, 100, I32_MAX, 0, 4, 4, I32_MAX)[0]
    assert not host_rows(False, 100, 3, I32_MAX - 1, I32_MAX, 4, 60)[0]
    big = 2**33
    assert host_rows(False, big, 2**30, 0, 2, 2, I32_MAX, offset=2**31 - 1) == \
        (True, [2**31 - 1 + 2**30, 2**31 + 2**30])
    # a page far behind 2^31 rows
    assert host_rows(True, 2**28, 17, 0, 1, 1, 64, table=[0, 2**28 - 1]) == \
        (True, [(2**28 - 1) * 16 + 1])


def test_paged_rows(host_rows):
    t = [7, 2, 9]
    assert host_rows(True, 10, 14, 0, 4, 4, 60, table=t) == \
        (True, [7 * 16 + 14, 7 * 16 + 15, 2 * 16, 2 * 16 + 1])
    assert host_rows(True, 10, 46, 0, 2, 4, 60, table=t)[0]
    assert not host_rows(True, 10, 46, 0, 3, 4, 60, table=t)[0]  # a fourth page
    # pages outside the pool: the rows in them are -1, the others stand
    assert host_rows(True, 9, 30, 0, 4, 4, 60, table=t) == \
        (True, [2 * 16 + 14, 2 * 16 + 15, -1, -1])
    assert host_rows(True, 10, 15, 0, 2, 4, 60, table=[7, -1, 9]) == (True, [7 * 16 + 15, -1])


@pytest.fixture(scope="module")
def find_seq(tmp_path_factory):
    import importlib.util
    spec = importlib.util.spec_from_file_location("p2p_build", ROOT / "p2p_b200" / "build.py")
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    exe = tmp_path_factory.mktemp("find_seq") / "find_seq_host"
    subprocess.run([build.nvcc(), *build.ARCH, "-std=c++17", "--expt-relaxed-constexpr",
                    "--extended-lambda", "-I", str(build.CSRC),
                    str(ROOT / "tests" / "find_seq_host.cu"), "-o", str(exe)],
                   check=True, capture_output=True)

    def ask(cases):
        """cases: (row_start, rows) pairs -> the sequences of the rows."""
        lines = [" ".join(map(str, [len(s) - 1, *s, len(r), *r])) for s, r in cases]
        out = subprocess.run([str(exe)], input="\n".join(lines) + "\n", capture_output=True,
                             text=True, check=True).stdout.splitlines()
        return [[int(x) for x in line.split()] for line in out]
    return ask


def test_a_rows_sequence(find_seq):
    """Every row of rising starts is found, empty sequences are passed over."""
    import random
    rng = random.Random(3)
    cases = []
    for n in (1, 2, 31, 32, 33, 64, 65, 1000, 1025, 3000):
        for top in (0, 1, 3):
            lens = [rng.randint(0, top) for _ in range(n)]
            start = [rng.randint(0, 2)]
            for x in lens:
                start.append(start[-1] + x)
            cases.append((start, range(0, start[-1] + 3)))
    for (start, rows), got in zip(cases, find_seq(cases)):
        want = {r: i for i in range(len(start) - 1) for r in range(start[i], start[i + 1])}
        assert got == [want.get(r, -1) for r in rows]


def test_falling_starts_never_give_a_row_to_a_sequence_that_ends_before_it(find_seq):
    """Whatever row_start holds, the sequence that a row is given has it among its rows (a position
    behind a sequence's checked end would lie outside its pages)."""
    import random
    rng = random.Random(4)
    cases = [([0, 100, 2, 4], range(105))]
    for n in (3, 5, 32, 40, 100, 700, 2000):
        for _ in range(60):
            start = [rng.randint(-3, 2 * n) for _ in range(n + 1)]
            if rng.random() < 0.5:  # nearly rising
                start.sort()
                for _ in range(rng.randint(1, 4)):
                    start[rng.randrange(n + 1)] = rng.randint(-3, 2 * n)
            cases.append((start, [rng.randint(0, 2 * n) for _ in range(60)]))
    for (start, rows), got in zip(cases, find_seq(cases)):
        for r, i in zip(rows, got):
            assert i == -1 or start[i] <= r < start[i + 1], (start, r, i)


def test_parameters_stay_plain_values():
    """Parameters that were used in a call can be copied, sent and changed like others."""
    import copy
    import pickle
    import p2p_b200
    prm = p2p_b200.Params(8, 2, scale=0.5)
    c = prm.ref()._obj
    assert (c.num_heads, c.num_kv_heads, c.head_dim, c.scale, c.dtype) == (8, 2, 64, 0.5, 0)
    assert copy.deepcopy(prm) == prm and pickle.loads(pickle.dumps(prm)) == prm
    assert vars(prm) == vars(p2p_b200.Params(8, 2, scale=0.5))
    prm.num_heads, prm.dtype = 16, torch.float32
    c = prm.ref()._obj
    assert (c.num_heads, c.scale, c.dtype) == (16, 0.5, 1)


def test_rows_overlap(tmp_path):
    """Strided rows against the sets of their bytes: shifted, interleaved, of other pitches."""
    import random
    exe = tmp_path / "rows_host"
    subprocess.run(["g++", "-std=c++17", "-I", str(ROOT / "p2p_b200" / "csrc"),
                    str(ROOT / "tests" / "rows_host.cpp"), "-o", str(exe)], check=True,
                   capture_output=True)
    rng = random.Random(5)
    cases = []
    for _ in range(6000):
        n, pa = rng.randint(1, 6), rng.randint(1, 12)
        pb = pa if rng.random() < 0.6 else rng.randint(1, 12)
        cases.append((rng.randint(100, 160), pa, rng.randint(1, pa), rng.randint(100, 160), pb,
                      rng.randint(1, pb), n))
        if n == 1:  # a single row may be wider than its pitch
            cases.append((*cases[-1][:2], 9, *cases[-1][3:5], 7, 1))
    big = 2**40
    cases += [(big, 2**20, 2**19, big + 2**19, 2**20, 2**19, 2**31 - 1),      # side by side
              (big, 2**20, 2**19 + 1, big + 2**19, 2**20, 2**19, 2**31 - 1)]  # one byte shared
    out = subprocess.run([str(exe)], input="\n".join(" ".join(map(str, c)) for c in cases) + "\n",
                         capture_output=True, text=True, check=True).stdout.split()
    for (a, pa, wa, b, pb, wb, n), got in zip(cases[:-2], out):
        one, two = ({at + i * p + j for i in range(n) for j in range(w)}
                    for at, p, w in ((a, pa, wa), (b, pb, wb)))
        assert bool(int(got)) == bool(one & two), (a, pa, wa, b, pb, wb, n)
    assert out[-2:] == ["0", "1"]
