"""Host side of the serving operators, without a GPU.

* hc_b200/csrc/kernels/kv_params.h compiled for the host: whatever lengths,
  starts and tables hold, positions and rows lie inside the buffers, and the
  equal shares of the attention cover every tile once;
* the C-ABI on a driver stand-in that records launches
  (oracle/recording_cuda.c): refusals, kernel choice, grids, streams;
* the oracle's 8-bit float against torch's.
"""

import ctypes as C
import os
import random
import subprocess
import sys
import textwrap
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import serving as oracle

REPO = Path(__file__).resolve().parent.parent


def test_e4m3_rounding_is_torchs():
    x = np.concatenate([np.random.default_rng(0).normal(size=4096) * 10.0 ** e
                        for e in range(-4, 3)])
    x = np.clip(x, -448, 448)
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn)
    assert np.array_equal(oracle.to_e4m3(x.astype(np.float32)), want.view(torch.uint8).numpy())
    assert np.array_equal(oracle.e4m3_values()[oracle.to_e4m3(x.astype(np.float32))],
                          want.double().numpy())


def test_oracle_unpacks_the_low_half_first():
    w = np.array([[0x21, 0x43]], np.uint8)
    assert oracle.unpack_w4(w, np.ones((1, 1)), np.zeros((1, 1)), 3, 32).tolist() == [[1, 2, 3]]


@pytest.fixture(scope="module")
def params(tmp_path_factory):
    out = tmp_path_factory.mktemp("kv") / "kv.so"
    src = out.with_suffix(".cpp")
    src.write_text(textwrap.dedent("""
        #include "kv_params.h"
        extern "C" void span(int seqs, int width, int tokens, int maxNew, int block, int length,
                             int begin, int end, int *r) {
          HcKvPlaceDev p{};
          p.seqs = seqs, p.width = width, p.tokens = tokens, p.maxNew = maxNew;
          HcKvSpan s = hcKvSpanOf(p, block, length, begin, end);
          r[0] = s.row, r[1] = s.count, r[2] = s.first, r[3] = s.allRow, r[4] = s.allCount;
        }
        extern "C" int page(int e, int pages) { return hcKvPageOf(e, pages); }
        extern "C" int touched(int n, int block) { return hcKvTouchedBlocks(n, block); }
        extern "C" unsigned begin(unsigned c, unsigned t, unsigned n) {
          return hcKvShareBegin(hcKvSharesOf(t, n), c); }
        extern "C" unsigned share(unsigned x, unsigned t, unsigned n) {
          return hcKvShareOf(hcKvSharesOf(t, n), x); }
        extern "C" unsigned unit_begin(unsigned c, unsigned t, unsigned n) {
          return hcKvShareBegin(hcKvSharesOfUnits(t, n), c); }
        extern "C" unsigned unit_share(unsigned x, unsigned t, unsigned n) {
          return hcKvShareOf(hcKvSharesOfUnits(t, n), x); }
        """))
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-fsanitize=undefined",
                    "-fno-sanitize-recover", "-static-libubsan", "-I",
                    str(REPO / "hc_b200" / "csrc" / "kernels"), "-o", str(out), str(src)],
                   check=True)
    lib = C.CDLL(str(out))
    for fn in (lib.begin, lib.share, lib.unit_begin, lib.unit_share):
        fn.restype, fn.argtypes = C.c_uint, [C.c_uint] * 3
    return lib


def _span(lib, *args):
    r = (C.c_int * 5)()
    lib.span(*args, r)
    return list(r)


def test_spans_stay_inside_whatever_the_arrays_hold(params):
    rng = random.Random(0)
    wild = [-2 ** 31, -7, -1, 0, 1, 2, 15, 16, 17, 100, 2 ** 30, 2 ** 31 - 1]
    for _ in range(20000):
        block = rng.choice([16, 32, 256])
        width, tokens = rng.choice([0, 1, 3, 1000]), rng.choice([0, 1, 5, 40, 2 ** 31 - 1])
        max_new = rng.choice([0, 1, 4, 40])
        length, begin, end = (rng.choice(wild) for _ in range(3))
        row, count, first, all_row, all_count = _span(params, 4, width, tokens, max_new, block,
                                                      length, begin, end)
        assert 0 <= all_row and 0 <= all_count and all_row + all_count <= tokens
        assert 0 <= count <= max(max_new, 0) and all_row <= row
        assert row + count <= all_row + all_count
        assert 0 <= first and first + count <= width * block
        if count and length >= 0:  # the position belongs to the row
            assert first - row == length - (all_row + all_count)


def test_spans_are_the_oracles(params):
    rng = random.Random(1)
    for _ in range(3000):
        block, width, max_new = 16, rng.randint(1, 4), rng.randint(1, 20)
        n = rng.randint(0, 25)
        length = rng.randint(0, 90)
        want = oracle.place([length], [3, 3 + n], 40, width, block, max_new)[0]
        row, count, first, _, _ = _span(params, 1, width, 40, max_new, block, length, 3, 3 + n)
        assert count == want[2]
        if count:
            assert (row, first) == want[:2]


def test_pages_and_touched_blocks(params):
    assert [params.page(e, 5) for e in (-2 ** 31, -1, 0, 4, 5, 2 ** 31 - 1)] == [-1, -1, 0, 4, -1,
                                                                                -1]
    for block in (16, 64):
        for n in range(0, 200):
            most = max([0] + [(first + n - 1) // block - first // block + 1
                              for first in range(block)] if n else [0])
            assert params.touched(n, block) == most


def test_shares_cover_every_tile_once(params):
    for total in (1, 2, 7, 295, 296, 297, 1000, 99991, 2 ** 31 - 1):
        for shares in (1, 2, 3, 148, 296):
            n = min(shares, total)
            bounds = [params.begin(c, total, n) for c in range(n + 1)]
            assert bounds[0] == 0 and bounds[-1] == total
            assert all(a < b for a, b in zip(bounds, bounds[1:]))
            for c in range(0, n, max(1, n // 7)):
                for x in (bounds[c], bounds[c + 1] - 1):
                    assert params.share(x, total, n) == c


def test_shares_of_like_units_end_with_them(params):
    for tiles in (1, 2, 7, 94, 297, 99991, 2 ** 27 - 1):
        for per in (1, 2, 3, 12, 37, 296):
            n = min(per, tiles)
            units = min(16, (2 ** 31 - 1) // tiles)
            bounds = [params.unit_begin(c, tiles, n) for c in range(units * n + 1)]
            assert bounds[::n] == [u * tiles for u in range(units + 1)]
            assert all(a < b for a, b in zip(bounds, bounds[1:]))
            for c in range(0, units * n, max(1, n // 7)):
                for x in (bounds[c], bounds[c + 1] - 1):
                    assert params.unit_share(x, tiles, n) == c


def test_a_part_that_gave_up_shows_in_its_rows(tmp_path):
    """The parts of a divided unit, joined as the kernel does: one that was given up makes
    sum, logarithm and outputs NaN, whatever the others hold and its place held before;
    one that saw nothing adds nothing."""
    src = tmp_path / "join.cpp"
    src.write_text(textwrap.dedent("""
        #include "kv_params.h"
        extern "C" float join(int n, const float *tops, const float *sums, const int *lost,
                              float *weights) {
          float top = -INFINITY, sum = 0.0f;
          for (int i = 0; i < n; ++i) {
            const HcKvPart p = lost[i] ? hcKvLostPart() : HcKvPart{tops[i], sums[i]};
            top = fmaxf(top, p.top);
          }
          for (int i = 0; i < n; ++i) {
            const HcKvPart p = lost[i] ? hcKvLostPart() : HcKvPart{tops[i], sums[i]};
            const float power = exp2f(p.top - top);
            sum += hcKvPartSum(p, power);
            weights[i] = hcKvPartWeight(p, power);
          }
          return sum;
        }
        """))
    out = tmp_path / "join.so"
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I",
                    str(REPO / "hc_b200" / "csrc" / "kernels"), "-o", str(out), str(src)],
                   check=True)
    lib = C.CDLL(str(out))
    lib.join.restype = C.c_float

    def join(tops, sums, lost):
        n = len(tops)
        weights = (C.c_float * n)()
        return lib.join(n, (C.c_float * n)(*tops), (C.c_float * n)(*sums), (C.c_int * n)(*lost),
                        weights), list(weights)

    inf, nan = float("inf"), float("nan")
    assert join([3, 1, -inf], [2, 4, 0], [0, 0, 0]) == (3, [1, 0.25, 0])
    for at in range(3):
        total, weights = join([3, 1, 0], [2, 4, 1], [i == at for i in range(3)])
        assert np.isnan(total) and weights[at] == 0 and not np.isnan(weights).any()
    total, weights = join([-inf, -inf], [0, 0], [0, 1])
    assert np.isnan(total) and weights == [0, 0]
    total, weights = join([-inf, 2], [nan, 1], [0, 0])  # scores that are NaN
    assert np.isnan(total) and weights == [0, 1]


def test_inputs_that_require_gradients_are_refused():
    """There is no backward pass; under no_grad the call goes on (to the refusal of CPU
    tensors, here)."""
    from types import SimpleNamespace

    from hc_b200 import serving

    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    gain, rows = torch.zeros(64, dtype=torch.bfloat16), torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    w = torch.zeros(16, 32, dtype=torch.uint8)
    scale, pages = torch.zeros(16, 2), torch.zeros(1, 1, 16, 64, dtype=torch.int8)
    ints = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    cache = SimpleNamespace(_native=None, _root=1.0)
    grad = lambda t: t.clone().requires_grad_()  # noqa: E731
    calls = [lambda: serving.add_rms_norm(grad(x), gain),
             lambda: serving.add_rms_norm(x, grad(gain)),
             lambda: serving.add_rms_norm(x, gain, grad(x)),
             lambda: serving.gemm_w4(grad(x), w, scale, group=32),
             lambda: serving.gemm_w4(x, w, grad(scale), group=32),
             lambda: serving.kv_append(cache, grad(rows), rows, *ints),
             lambda: serving.kv_append(cache, rows, grad(rows), *ints),
             lambda: serving.kv_attention(cache, grad(rows), *ints),
             lambda: serving.KvCache(pages, pages, grad(scale), scale)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA tensors"):
            call()


def test_a_capture_on_another_device_than_the_current_one(monkeypatch):
    """The attention's workspace is a captured call's own where the stream of its device is
    being captured, whichever device is the current one."""
    from types import SimpleNamespace

    from hc_b200 import serving

    state = dict(current=0, capturing={0: False, 1: False})

    class On:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, state["current"] = state["current"], self.index

        def __exit__(self, *_):
            state["current"] = self.before

    empty = torch.empty
    monkeypatch.setattr(torch.cuda, "current_device", lambda: state["current"])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing",
                        lambda: state["capturing"][state["current"]])
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    monkeypatch.setattr(serving, "_scratch", {})
    native = SimpleNamespace(kv_attention_workspace_bytes=lambda ctx: 8192)
    get = lambda i: serving._attention_workspace(  # noqa: E731
        native, None, SimpleNamespace(index=i), 7)
    kept = [get(0), get(1)]
    assert get(0) is kept[0] and get(1) is kept[1] and kept[0] is not kept[1]
    state["capturing"][1] = True
    assert get(1) is not kept[1] and get(0) is kept[0]
    state["capturing"] = {0: True, 1: False}
    assert get(1) is kept[1] and get(0) is not kept[0]
    assert state["current"] == 0


# ---- the C-ABI on a recording driver --------------------------------------------------------
SCRIPT = """
import ctypes as C
import sys
sys.path.insert(0, {repo!r})
from hc_b200 import capi
fake = C.CDLL("libcuda.so.1")
class Launch(C.Structure):
    _fields_ = [("name", C.c_char * 96), ("grid", C.c_uint * 3), ("block", C.c_uint),
                ("smem", C.c_uint), ("stream", C.c_ulonglong)]
fake.recorded_launch.restype = C.POINTER(Launch)
def launches():
    got = [fake.recorded_launch(i).contents for i in range(fake.recorded_launches())]
    got = [(l.name.decode(), tuple(l.grid), l.block, l.smem, l.stream) for l in got]
    fake.recorded_clear()
    return got
def refused(match, call, *args, **kw):
    try:
        call(*args, **kw)
    except capi.HcError as e:
        assert match in str(e), (match, str(e))
        assert not launches()
        return
    raise AssertionError("not refused: " + match)
hc = capi.Context("cuda:0")
P = 0x700000000  # an address that nothing dereferences
launches()
"""


@pytest.fixture(scope="module")
def recording(tmp_path_factory):
    out = tmp_path_factory.mktemp("fake")
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-Wl,-soname,libcuda.so.1", "-o",
                    str(out / "libcuda.so.1"), str(REPO / "oracle" / "recording_cuda.c")],
                   check=True)

    def run(body):
        env = dict(os.environ, LD_LIBRARY_PATH=str(out))
        script = SCRIPT.format(repo=str(REPO)) + textwrap.dedent(body)
        done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True,
                              env=env, timeout=300)
        assert done.returncode == 0, done.stdout + done.stderr

    return run


def test_norm_refusals_and_choice(recording):
    recording("""
    def norm(rows=4, cols=64, x=P, residual=P, summed=P, gain=P, out=P, scale=P, xp=None, rp=None,
             sp=None, op=None, cp=8, group=0, eps=1e-5, dtype=capi.HC_BF16, out_dtype=capi.HC_I8):
        hc.add_rms_norm(x, residual, summed, gain, out, scale, rows, cols, *(
            cols if v is None else v for v in (xp, rp, sp, op)), cp, group, eps, dtype, out_dtype)
    refused("unsupported dtype", norm, dtype=capi.HC_F64)
    refused("unsupported output", norm, out_dtype=capi.HC_F32)
    refused("invalid shape", norm, rows=-1)
    refused("invalid shape", norm, xp=63)
    refused("invalid shape", norm, rp=63)
    refused("invalid group", norm, group=-2)
    refused("invalid group", norm, group=32, out_dtype=capi.HC_BF16)
    refused("scale pitch", norm, cols=1024, group=64)
    refused("eps", norm, eps=float("nan"))
    refused("null buffer", norm, scale=None)
    refused("null buffer", norm, gain=None)
    refused("no residual", norm, residual=None)
    norm(rows=0); norm(cols=0)
    assert not launches()
    for cols, rows, kernel in ((64, 4, "bf16_i8_t64_v1"), (4096, 1, "bf16_i8_t512_v1"),
                               (4096, 4000, "bf16_i8_t256_v2"), (8192, 4000, "bf16_i8_t256_v4"),
                               (16384, 1, "bf16_i8_t512_v4"), (16392, 1, "bf16_i8_generic"),
                               (100, 1, "bf16_i8_generic")):
        norm(rows=rows, cols=cols)
        (name, grid, block, smem, _), = launches()
        assert name == "hc_add_rms_norm_" + kernel and grid == (rows, 1, 1), name
    norm(cols=1024, x=P + 2); norm(cols=1024, op=1028); norm(cols=1024, group=96, cp=11)
    assert all(l[0].endswith("generic") for l in launches())
    norm(cols=60000)
    assert launches()[0][3] == 0  # longer than shared memory: the row is computed again
    """)


def test_w4_refusals_and_choice(recording):
    recording("""
    def w4(m=1, n=4096, k=4096, group=128, a_group=0, a=P, a_scale=None, w=P, scale=P, zero=None,
           out=P, ws=P, ws_bytes=1 << 40, lda=None, ldas=64, ldw=None, lds=1024, ldz=1024,
           ldc=None, a_dtype=capi.HC_BF16, scale_dtype=capi.HC_BF16):
        pick = lambda v, d: d if v is None else v
        hc.gemm_w4(a, a_scale, w, scale, zero, out, ws, ws_bytes, m, n, k, group, a_group,
                   pick(lda, k), ldas, pick(ldw, k // 2), lds, ldz, pick(ldc, n), a_dtype,
                   scale_dtype)
    refused("activation dtype", w4, a_dtype=capi.HC_F32)
    refused("scale dtype", w4, scale_dtype=capi.HC_I8)
    refused("invalid shape", w4, m=-1)
    refused("invalid shape", w4, ldw=2047)
    refused("invalid shape", w4, ldc=4095)
    refused("multiple of 32", w4, group=33)
    refused("multiple of 32", w4, group=0)
    refused("pitch", w4, lds=31)
    refused("pitch", w4, zero=P, ldz=31)
    refused("activations' group", w4, a_dtype=capi.HC_I8, a_scale=P, a_group=100)
    refused("null buffer", w4, a_dtype=capi.HC_I8)
    refused("null buffer", w4, out=None)
    refused("null buffer", w4, scale=None)
    refused("workspace", w4, m=1025, ws=None)
    refused("workspace", w4, m=1025, ws_bytes=4096 * 4096 * 2 - 1)
    refused("workspace", w4, m=9, a_dtype=capi.HC_I8, a_scale=P, ws=None)
    refused("workspace", w4, m=9, lda=4097, ws_bytes=9 * 8192 - 1)
    refused("workspace", w4, m=9, w=P + 8, ws_bytes=4096 * 2048 - 1)
    refused("workspace", w4, m=1025, ws=P + 8)
    w4(m=0); w4(n=0)
    assert not launches()
    need = lambda m, n, k, lda, ldw, t=capi.HC_BF16: hc.lib.hcGemmW4WorkspaceBytes(m, n, k, lda, ldw, t)
    up = lambda x, to: -(-x // to) * to
    assert need(1024, 4096, 4096, 4096, 2048) == 0
    assert need(64, 4090, 4097, 4097, 2064) == up(64 * 4104 * 2, 256)
    assert need(64, 4090, 4097, 4104, 2049) == 4090 * 2064
    assert need(64, 4096, 4096, 4096, 2048, capi.HC_I8) == 64 * 4096 * 2
    assert need(1025, 4090, 4096, 4096, 2048) == 4096 * 4096 * 2
    assert need(1025, 4096, 4096, 4096, 2048, capi.HC_I8) == (1025 + 4096) * 4096 * 2
    # Few rows: one launch.
    for kw, kernel in ((dict(), "bf16_coarse"), (dict(m=8), "bf16_coarse"),
                       (dict(m=3, group=64), "bf16_fine"),
                       (dict(m=5, group=1 << 20), "bf16_coarse"),
                       (dict(a_dtype=capi.HC_I8, a_scale=P), "i8_coarse"),
                       (dict(w=P + 1), "bf16_coarse_any"),
                       (dict(k=4098, ldw=2064), "bf16_coarse_any")):
        w4(**kw)
        (name, grid, block, smem, _), = launches()
        assert name == "hc_gemm_w4_" + kernel, name
        assert grid == (148, 1, 1) and block == 512 and smem <= 227 << 10
    # More rows: the tcgen05 kernel, the K axis divided where there are few tiles.
    for kw, names, grid in (
            (dict(m=9), ["narrow_coarse_bf16"], (32, 8, 1)),
            (dict(m=64, group=32, lds=128, scale_dtype=capi.HC_F32), ["narrow_fine_f32"], (32, 8, 1)),
            (dict(m=65), ["wide_coarse_bf16"], (32, 4, 1)),
            (dict(m=1024), ["wide_coarse_bf16"], (128, 1, 1)),
            (dict(m=16, n=130, k=100, lda=104, ldw=64), ["narrow_coarse_bf16"], (2, 1, 1)),
            (dict(m=16, w=P + 4), ["copy", "narrow_coarse_bf16"], (32, 8, 1)),
            (dict(m=16, lda=4097), ["hc_repack_a16_bf16", "narrow_coarse_bf16"], (32, 8, 1)),
            (dict(m=16, a_dtype=capi.HC_I8, a_scale=P), ["hc_repack_a8_bf16", "narrow_coarse_bf16"],
             (32, 8, 1))):
        w4(**kw)
        got = launches()
        assert len(got) == len(names), got
        for (name, *_), want in zip(got, names):
            assert want in name, (name, want)
        name, shape, block, smem, _ = got[-1]
        assert shape == grid, (kw, shape)
        assert block == (384 if "narrow" in name else 640)
        assert smem <= (113 if "narrow" in name else 227) << 10
    # Whatever the sizes: shared memory within a CTA's limit, a cluster of at most eight.
    import random
    rng = random.Random(0)
    for _ in range(500):
        k = rng.choice([1, 31, 128, 4096, 30000, 1 << 20])
        group = 32 * rng.choice([1, 2, 3, 4, 8, 1000])
        w4(m=rng.randint(1, 1024), n=rng.choice([1, 500, 100000]), k=k, group=group,
           lda=k + 7 & ~7, ldw=((k + 1) // 2) + 15 & ~15, lds=1 << 16, ldz=1 << 16,
           zero=rng.choice([None, P]), a_dtype=rng.choice([capi.HC_BF16, capi.HC_I8]), a_scale=P)
        name, grid, block, smem, _ = launches()[-1]
        assert smem <= 227 << 10, (name, smem, k, group)
        assert "umma" not in name or grid[1] <= 8
    w4(m=1025)
    assert [l[0] for l in launches()] == ["hc_dequant_w4_bf16", "hc_gemm_bf16_umma_pair"]
    w4(m=1025, a_dtype=capi.HC_I8, a_scale=P)
    assert [l[0] for l in launches()] == ["hc_repack_a8_bf16", "hc_dequant_w4_bf16",
                                          "hc_gemm_bf16_umma_pair"]
    # The choice can be made by hand.
    hc.set_option("w4_variant", 2)
    w4()
    assert launches()[0][0] == "hc_gemm_w4_umma_narrow_coarse_bf16"
    hc.set_option("w4_variant", 1)
    refused("few rows", w4, m=9)
    """)


def test_w4_workspace_of_a_call(recording):
    """The kernel for few rows takes none, whatever the layout; others what the size that
    knows the layout alone says."""
    recording("""
    from hc_b200._native import _dispatcher as d
    def call(m, k, group, ws, lda, ldw, t):
        hc.gemm_w4(P, P if t == capi.HC_I8 else None, P, P, None, P, P if ws else None, ws, m, 100,
                   k, group, 0, lda, 1, ldw, 1 << 16, 0, 100, t)
        return [l[0] for l in launches()]
    layout = hc.lib.hcGemmW4WorkspaceBytes
    need = hc.lib.hcGemmW4CallWorkspaceBytes
    ctx = d.Context("cuda:0")
    launches()
    for t in (capi.HC_I8, capi.HC_BF16):
        for m in (1, 3, 7, 8, 9, 40, 1100):
            for k in (100, 4096, 4098, 8192, 30000):
                for group in (32, 64, 128):
                    for lda, ldw in ((k, (k + 1) // 2), (k + 7 & ~7, (k + 31) // 32 * 16)):
                        ws = need(hc.handle, m, 100, k, group, lda, ldw, t)
                        assert ws == d.w4_workspace_bytes(ctx, m, 100, k, group, lda, ldw,
                                                          t == capi.HC_I8)
                        names = call(m, k, group, ws, lda, ldw, t)
                        few = "umma" not in names[-1]
                        assert ws == (0 if few else layout(m, 100, k, lda, ldw, t)), (m, k, group)
                        assert not few or m <= 8 and len(names) == 1
                        if ws:
                            refused("workspace", call, m, k, group, ws - 1, lda, ldw, t)
    assert need(hc.handle, 3, 100, 4096, 128, 4096, 2048, capi.HC_I8) == 0
    hc.set_option("w4_variant", 2)
    assert need(hc.handle, 3, 100, 4096, 128, 4096, 2048, capi.HC_I8) == 3 * 8192
    """)


def test_cache_refusals_and_choice(recording):
    recording("""
    def cache(**kw):
        c = capi.HcKvCache(P, P, P, P, 4 * 16 * 128, 16 * 128, 128, 4, 100, 16, 4, 128, capi.HC_I8)
        for name, v in kw.items():
            setattr(c, name, v)
        return c
    def place(**kw):
        p = capi.HcKvPlace(P, P, P, 320, 8, 320, 8, 1)
        for name, v in kw.items():
            setattr(p, name, v)
        return p
    WS = hc.kv_attention_workspace_bytes()
    def append(c=None, p=None, k=P, v=P, strides=(512, 128, 512, 128)):
        hc.kv_append(c or cache(), p or place(), k, v, *strides)
    def attend(c=None, p=None, q=P, out=P, lse=P, share=4, scale=1.0, window=0,
               strides=(2048, 128, 2048, 128, 16), ws=P, ws_bytes=WS):
        hc.kv_attention(c or cache(), p or place(), q, out, lse, share, scale, window, *strides, ws,
                        ws_bytes)
    for call in (append, attend):
        refused("cache dtype", call, cache(dtype=capi.HC_BF16))
        for block in (0, 8, 24, 272):
            refused("block of", call, cache(block=block))
        for dim in (0, 8, 120, 272):
            refused("head dimension", call, cache(dim=dim))
        refused("pages of", call, cache(pages=-1))
        refused("pages of", call, cache(heads=0))
        refused("16-byte aligned", call, cache(tokenStride=136))
        refused("16-byte aligned", call, cache(tokenStride=112))
        refused("16-byte aligned", call, cache(pageStride=8))
        refused("16-byte aligned", call, cache(v=P + 8))
        refused("scale pitch", call, cache(scalePitch=3))
        refused("spans 2^31", call, cache(tokenStride=1 << 27))
        refused("below 2^31", call, cache(pageStride=1 << 31))
        refused("below 2^31", call, cache(scalePitch=1 << 31))
        refused("pages of", call, cache(heads=1 << 15, scalePitch=1 << 15))
        refused("null cache buffer", call, cache(kScale=None))
        refused("invalid place", call, p=place(seqs=-1))
        refused("invalid place", call, p=place(maxNew=-1))
        refused("invalid place", call, p=place(tablePitch=31))
        refused("invalid place", call, p=place(width=1 << 30, tablePitch=1 << 30))
        refused("rows for", call, p=place(starts=None, tokens=7))
        refused("null lengths", call, p=place(lengths=None))
        refused("null lengths", call, p=place(table=None))
        call(p=place(seqs=0)); call(p=place(tokens=0))
        assert not launches()
    refused("negative strides", append, strides=(-1, 128, 512, 128))
    refused("null buffer", append, k=None)
    append(p=place(maxNew=0)); append(cache(pages=0))
    assert not launches()
    append()
    assert launches()[0][:3] == ("hc_kv_append_i8_warp", (8, 2, 1), 128)
    append(cache(dtype=capi.HC_E4M3), place(maxNew=40, tokens=300))
    assert launches()[0][:3] == ("hc_kv_append_e4m3_cta", (8 * 4, 8, 1), 256)
    append(p=place(maxNew=40, tokens=300, starts=None))  # one row per sequence
    assert launches()[0][1] == (8, 2, 1)
    refused("too many", append, p=place(seqs=1 << 30, maxNew=100, tokens=1 << 30))

    refused("query heads", attend, share=0)
    refused("query heads", attend, window=-1)
    refused("query heads", attend, scale=float("inf"))
    refused("invalid strides", attend, strides=(-1, 1, 1, 1, 16))
    refused("invalid strides", attend, strides=(2048, 128, 2048, 128, 15))
    refused("null buffer", attend, q=None)
    refused("8-byte aligned", attend, out=P + 2)
    refused("8-byte aligned", attend, strides=(2048, 128, 2050, 128, 16))
    refused("workspace", attend, ws=None)
    refused("workspace", attend, ws=P + 64)
    refused("workspace", attend, ws_bytes=WS - 1)
    for kw, kernel, ctas in (
            (dict(), "i8_d128_r1", 296), (dict(share=9, lse=None), "i8_d128_r2", 148),
            (dict(c=cache(dim=64, dtype=capi.HC_E4M3)), "e4m3_d64_r1", 296),
            (dict(c=cache(dim=256, tokenStride=256), share=16, lse=None), "i8_d256_r1", 148),
            (dict(p=place(seqs=1, width=1, tokens=1)), "i8_d128_r1", 1)):
        attend(**kw)
        (name, grid, block, smem, _), = launches()
        assert name == "hc_kv_attention_" + kernel and grid == (ctas, 1, 1), (name, grid)
        assert smem <= 227 << 10
    """)


def test_arrays_that_are_written_to_have_memory_of_their_own(recording):
    """Expanded caches and outputs: every layout without shared elements is taken."""
    recording("""
    from hc_b200._native import _dispatcher as d

    class Dev:  # what the dispatcher reads of a device array
        is_cuda = True
        device = type("D", (), dict(index=0))
        def __init__(self, dtype, shape, strides, size):
            self.dtype, self.shape, self.strides, self.size = "torch." + dtype, shape, strides, size
        def data_ptr(self): return P
        def element_size(self): return self.size
        def stride(self): return self.strides
    def dense(dtype, size, *shape, order=None):
        strides, at = [0] * len(shape), 1
        for axis in reversed(order or range(len(shape))):
            strides[axis], at = at, at * shape[axis]
        return Dev(dtype, shape, tuple(strides), size)

    ctx = d.Context("cuda:0")
    scale = dense("float32", 4, 5, 2)
    table, lengths = dense("int32", 4, 3, 2), dense("int32", 4, 3)
    rows = dense("bfloat16", 2, 3, 2, 64)
    ws = Dev("uint8", (d.kv_attention_workspace_bytes(ctx),), (1,), 1)
    launches()
    def append(pages):
        d.kv_append(ctx, d.KvCache(ctx, pages, pages, scale, scale), rows, rows, table, lengths)
        return len(launches())
    def attend(pages, out):
        cache = d.KvCache(ctx, pages, pages, scale, scale)
        d.kv_attention(ctx, cache, dense("bfloat16", 2, 3, 4, 64), out, None, table, lengths, None,
                       -1, 0.125, 0, ws)
        return len(launches())
    def no(match, call, *args):
        try:
            call(*args)
        except ValueError as e:
            assert match in str(e) and not launches(), str(e)
            return
        raise AssertionError("not refused")
    out = dense("bfloat16", 2, 3, 4, 64)
    for order in (None, (0, 2, 1, 3), (1, 0, 2, 3), (2, 0, 1, 3)):
        pages = dense("int8", 1, 5, 2, 16, 64, order=order)
        assert append(pages) == 1 and attend(pages, out) == 1
    wide = Dev("int8", (5, 2, 16, 64), (2 * 2 * 16 * 80, 16 * 80, 80, 1), 1)
    assert append(wide) == 1
    one = Dev("int8", (5, 1, 16, 64), (16 * 64, 0, 64, 1), 1)  # an axis of one: any stride
    single = dense("float32", 4, 5, 1)
    d.kv_append(ctx, d.KvCache(ctx, one, one, single, single), dense("bfloat16", 2, 3, 1, 64),
                dense("bfloat16", 2, 3, 1, 64), table, lengths)
    assert len(launches()) == 1
    for strides in ((0, 1024, 64, 1), (2048, 0, 64, 1), (1024, 1024, 64, 1), (2048, 512, 64, 1)):
        pages = Dev("int8", (5, 2, 16, 64), strides, 1)
        no("share memory", append, pages)
        assert attend(pages, out) == 1
    pages = dense("int8", 1, 5, 2, 16, 64)
    assert attend(pages, dense("bfloat16", 2, 3, 4, 64, order=(1, 0, 2))) == 1
    for strides in ((0, 64, 1), (256, 0, 1), (128, 64, 1), (64, 128, 1)):
        no("share memory", attend, pages, Dev("bfloat16", (3, 4, 64), strides, 2))
    """)


def test_launches_go_to_the_stream_in_use(recording):
    recording("""
    def go():
        hc.softmax_rows(P, P + (1 << 20), 4, 64, 64, 64)
        return launches()[0][4]
    own = go()
    assert own == hc.stream
    hc.use_stream(0x1234000)
    assert go() == 0x1234000 and hc.stream == own
    hc.use_stream(0)
    assert go() == 0
    hc.use_own_stream()
    assert go() == own
    hc.close()
    """)


def test_pushed_streams_nest_and_are_the_threads_own(recording):
    recording("""
    import threading
    def go():
        hc.softmax_rows(P, P + (1 << 20), 4, 64, 64, 64)
        return launches()[0][4]
    own = hc.stream
    hc.push_stream(0x1000)
    hc.push_stream(0x2000)
    assert go() == 0x2000
    seen = []
    t = threading.Thread(target=lambda: seen.append(go()))
    t.start(); t.join()
    assert seen == [own]
    hc.pop_stream()
    assert go() == 0x1000
    hc.use_stream(0x3000)  # the context's choice waits behind the thread's
    assert go() == 0x1000
    hc.pop_stream()
    assert go() == 0x3000
    hc.use_own_stream()
    refused("pushed none", hc.pop_stream)
    assert go() == own
    hc.close()
    """)


def test_errors_and_pushed_streams_are_a_contexts_own(recording):
    """Two contexts' last errors side by side; a context opened where one with a pushed
    stream was released starts on its own."""
    recording("""
    other = capi.Context("cuda:0")
    last = hc.lib.hcLastError
    last.restype = C.c_void_p
    assert hc.lib.hcSetOption(hc.handle, b"no such option", 1)
    assert other.lib.hcReportError(other.handle, b"of the other")
    a, b = last(hc.handle), last(other.handle)
    assert b"no such option" in C.string_at(a) and C.string_at(b) == b"of the other"
    for _ in range(20):
        c = capi.Context("cuda:0")
        c.softmax_rows(P, P + (1 << 20), 4, 64, 64, 64)
        assert launches()[0][4] == c.stream
        c.push_stream(0x5000)
        c.push_stream(0x6000)
        c.close()
    """)


def test_serving_calls_beside_a_host_buffer_call(recording):
    """Two threads of one process, one context: the host-buffer call, which runs without
    the interpreter lock, keeps its kernels on the context's stream, and the serving
    calls go to theirs."""
    recording("""
    import threading
    import time
    import numpy as np
    from hc_b200._native import _dispatcher as d

    class Dev:  # what the dispatcher reads of a device array
        is_cuda = True
        device = type("D", (), dict(index=0))
        def __init__(self, *shape, dtype="torch.bfloat16"):
            self.shape, self.dtype = shape, dtype
        def data_ptr(self): return P
        def element_size(self): return 2
        def stride(self): return (64, 1)[-len(self.shape):]

    ctx = d.Context("cuda:0")
    x, gain, out = Dev(4, 64), Dev(64), Dev(4, 64)
    big = np.empty((1 << 18, 1024), np.float32)  # 64 chunks
    res = np.empty_like(big)
    launches()
    sys.setswitchinterval(1e-4)
    calls = [0, 0]
    def host():
        while calls[0] < 20 or calls[1] < 1000:
            d.softmax_rows_host(ctx, big, res)
            calls[0] += 1
            seen = calls[1]
            while calls[0] < 20 and calls[1] == seen:  # (a single core runs them in turn)
                time.sleep(0)
    t = threading.Thread(target=host)
    t.start()
    while calls[0] < 20 or calls[1] < 1000:
        d.add_rms_norm(ctx, x, gain, None, None, out, None, stream=0x1234000)
        calls[1] += 1
    t.join()
    got = launches()
    names = ["softmax" in l[0] for l in got]
    assert len(got) == 64 * calls[0] + calls[1], (len(got), calls)
    switches = sum(a != b for a, b in zip(names, names[1:]))
    assert switches > 10, (switches, calls)  # beside each other
    for soft, l in zip(names, got):
        assert l[4] == (ctx.stream if soft else 0x1234000), l
    """)


def test_host_buffer_calls_of_two_threads_take_turns(recording):
    """They share the context's device slots: a call's chunks are its own from the first
    to the last."""
    recording("""
    import threading
    import numpy as np
    from hc_b200._native import _dispatcher as d
    fake.recorded_upload.restype = C.c_ulong
    ctx = d.Context("cuda:0")
    big = [np.empty((1 << 18, 1024), np.float32) for _ in range(2)]  # 64 chunks
    start = threading.Barrier(2)
    def host(x):
        start.wait()
        for _ in range(20):
            d.reduce_rows_host(ctx, x, np.empty(1 << 18, np.float32), None)
    threads = [threading.Thread(target=host, args=(x,)) for x in big]
    for t in threads: t.start()
    for t in threads: t.join()
    who = [fake.recorded_upload(i) for i in range(fake.recorded_uploads())]
    assert len(who) == 2 * 20 * 64 and len(set(who)) == 2
    for i in range(0, len(who), 64):
        assert len(set(who[i:i + 64])) == 1, i
    """)


def test_every_serving_kernel_is_found_by_its_name():
    """The families that the launch code names lie in the images it says."""
    from hc_b200 import capi
    from tests.test_abi_cpu import _elf_symbols

    lib = capi.load_kernels()
    for image, count in (("add_rms_norm", 60), ("gemm_w4", 11), ("gemm_w4_umma", 8),
                         ("kv_append", 4), ("kv_attention", 20),
                         ("kv_attention_umma", 6)):
        blob = (REPO / "hc_b200" / "_native" / f"{image}.cubin").read_bytes()
        names = [s for s in _elf_symbols(blob) if s.startswith("hc_")]
        assert len(names) == count, (image, len(names))
        for name in names:
            assert lib.hcImageName(lib.hcImageOfKernel(name.encode())).decode() == image
