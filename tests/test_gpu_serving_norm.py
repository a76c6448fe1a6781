"""Root-mean-square norm with the residual's addition and 8-bit outputs
(hcAddRmsNorm, hc_b200.serving.add_rms_norm) against its formula in 64 bits.

Tolerances.  The kernel computes y in float32: the sum of squares adds at most
a few hundred rounded partial sums per row on top of exact-to-2^-24 products
(shuffle tree of depth 9 above chains of at most 32), the square root, the
reciprocal and two products round once each: below 64 * 2^-24 = 2^-18 of |y|.
On top of that an output rounds once: half a step, 2^-8 |y| in bfloat16, 2^-24
in float32, 2^-4 |y| (or half of the smallest step, 2^-10 scale) in e4m3, half
a scale in int8."""

import numpy as np
import pytest
import torch

from hc_b200 import serving
from oracle import serving as oracle

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -18


def _inputs(rows, cols, dtype, seed=0, pad=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def wide(r):
        t = torch.randn(r, cols + pad, device="cuda", generator=gen).to(dtype)
        return t[:, :cols]

    gain = (1 + 0.3 * torch.randn(cols, device="cuda", generator=gen)).to(dtype)
    return wide(rows), wide(rows) * 2 if pad == 0 else wide(rows), gain


def _f64(t):
    return t.double().cpu().numpy()


def _check(x, residual, gain, out, scale, summed, group, eps=1e-5):
    y, s = oracle.add_rms_norm(_f64(x), None if residual is None else _f64(residual), _f64(gain),
                               eps)
    if residual is not None:
        assert torch.equal(summed, (x.float() + residual.float()).to(x.dtype))
    if scale is None:
        step = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
        assert np.all(np.abs(_f64(out) - y) <= (step + F32) * np.abs(y) + 1e-37)
        return
    store = "int8" if out.dtype == torch.int8 else "e4m3"
    want = oracle.group_scales(y, group, store)
    assert np.all(np.abs(_f64(scale) - want) <= 2 * F32 * want)
    wide = oracle.widen(_f64(scale), group, x.shape[1])
    got = oracle.stored_values(out.view(torch.uint8).cpu().numpy(), store) * wide
    if store == "int8":
        room = wide * (0.5 + 128 * 2 * F32)
    else:
        room = (2.0 ** -4 + 2 * F32) * np.abs(y) + wide * 2.0 ** -10
    assert np.all(np.abs(got - y) <= room)


SHAPES = [(1, 8), (3, 64), (1, 512), (5, 520), (2, 1024), (300, 2048), (7, 4096), (301, 4096),
          (129, 5120), (2, 8192), (400, 8192), (3, 16384), (2, 16392), (2, 45000)]
ODD = [(1, 1), (2, 3), (3, 1001), (2, 4097), (1, 50001)]


@pytest.mark.parametrize("store", [None, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES + ODD)
def test_against_the_formula(shape, dtype, store):
    x, residual, gain = _inputs(*shape, dtype)
    out, scale, summed = serving.add_rms_norm(x, gain, residual, out_dtype=store)
    _check(x, residual, gain, out, scale, summed, 0)


@pytest.mark.parametrize("store", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape,group", [((3, 256), 8), ((5, 1000), 32), ((2, 4096), 64),
                                         ((131, 5120), 128), ((2, 1032), 256), ((2, 1000), 100),
                                         ((3, 999), 128), ((2, 45000), 384), ((2, 128), 4096)])
def test_groups(shape, group, store):
    x, residual, gain = _inputs(*shape, torch.bfloat16)
    out, scale, summed = serving.add_rms_norm(x, gain, residual, out_dtype=store, group=group)
    _check(x, residual, gain, out, scale, summed, group)


def test_without_residual_and_pitched_rows():
    x, residual, gain = _inputs(5, 1024, torch.bfloat16, pad=24)
    assert not x.is_contiguous()
    out, scale, summed = serving.add_rms_norm(x, gain)
    assert scale is None and summed is None
    _check(x, None, gain, out, None, None, 0)
    out, scale, summed = serving.add_rms_norm(x, gain, residual, out_dtype=torch.int8)
    _check(x, residual, gain, out, scale, summed, 0)
    # A pitch that 16-byte loads cannot use.
    x, residual, gain = _inputs(5, 1024, torch.bfloat16, pad=3)
    out, scale, summed = serving.add_rms_norm(x, gain, residual)
    _check(x, residual, gain, out, None, summed, 0)


@pytest.mark.parametrize("cols", [4096, 45000, 1001])
def test_in_place(cols):
    """The sum over the residual, the output over the input."""
    x, residual, gain = _inputs(9, cols, torch.bfloat16)
    want, _, total = serving.add_rms_norm(x, gain, residual)
    x2, r2 = x.clone(), residual.clone()
    out, _, summed = serving.add_rms_norm(x2, gain, r2, out=x2, summed=r2)
    assert out is x2 and summed is r2
    assert torch.equal(x2, want) and torch.equal(r2, total)


def test_zero_rows_and_values_that_are_not_finite():
    x, _, gain = _inputs(6, 1024, torch.bfloat16)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    x[4] = torch.finfo(torch.bfloat16).tiny
    for store in (torch.int8, torch.float8_e4m3fn):
        out, scale, _ = serving.add_rms_norm(x, gain, out_dtype=store, eps=1e-5)
        value = out.float() * scale
        assert scale[1].item() == 0 and torch.equal(value[1], torch.zeros_like(value[1]))
        assert not torch.isfinite(scale[2:4]).any()
        assert not torch.isfinite(value[2]).any() and torch.isnan(value[3]).any()
        keep = torch.tensor([0, 4, 5], device="cuda")
        _check(x[keep], None, gain, out[keep], scale[keep], None, 0)
    # The largest finite rows: squares overflow float32, as they do in the formula there.
    out, _, _ = serving.add_rms_norm(x[:1] * 0, gain, eps=0.0)
    assert torch.isnan(out).all()  # 0 / 0


def test_other_stream_and_graph():
    x, residual, gain = _inputs(33, 4096, torch.bfloat16)
    want, scale, total = serving.add_rms_norm(x, gain, residual, out_dtype=torch.int8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        xs = x.clone()
        got, s2, t2 = serving.add_rms_norm(xs, gain, residual, out_dtype=torch.int8)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(s2, scale) and torch.equal(t2, total)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, s2, t2 = serving.add_rms_norm(x, gain, residual, out_dtype=torch.int8)
    fresh = torch.randn_like(x)
    x.copy_(fresh)
    graph.replay()
    want, scale, total = serving.add_rms_norm(x, gain, residual, out_dtype=torch.int8)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(s2, scale) and torch.equal(t2, total)


def test_refusals():
    x, residual, gain = _inputs(4, 64, torch.bfloat16)
    with pytest.raises(TypeError, match="gain"):
        serving.add_rms_norm(x, gain.float())
    with pytest.raises(ValueError, match="gain"):
        serving.add_rms_norm(x, gain[:-1])
    with pytest.raises(ValueError, match="differ in shape"):
        serving.add_rms_norm(x, gain, residual[:3])
    with pytest.raises(TypeError, match="residual"):
        serving.add_rms_norm(x, gain, residual.float())
    with pytest.raises(TypeError, match="int8 or float8_e4m3fn"):
        serving.add_rms_norm(x, gain, out_dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensors"):
        serving.add_rms_norm(x.cpu(), gain)
    with pytest.raises(RuntimeError, match="invalid group"):
        serving.add_rms_norm(x, gain, out_dtype=torch.int8, group=-1)
    with pytest.raises(RuntimeError, match="eps"):
        serving.add_rms_norm(x, gain, eps=-1.0)
    assert serving.add_rms_norm(x[:0], gain)[0].shape == (0, 64)


@pytest.mark.parametrize("store", [None, torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols,group", [(512, 0), (8192, 128), (1001, 0), (45000, 0),
                                        (45000, 384)])
@pytest.mark.parametrize("power", [-90, -70, 66, 120])
def test_rows_whose_squares_leave_float32(power, cols, group, dtype, store):
    """Finite rows whose squares overflow, or (eps = 0) vanish: y is what it is for others.
    Rows of either kind among ordinary ones, and zeros."""
    x, residual, gain = _inputs(5, cols, dtype, seed=power + 100)
    by = torch.tensor([1.0, 2.0 ** power, 0.0, 2.0 ** power, 2.0 ** 30], device="cuda")[:, None]
    x, residual = (x.float() * by).to(dtype), (residual.float() * by).to(dtype)
    group = group if store is not None else 0
    eps = 0.0 if power < 0 else 1e-5
    out, scale, summed = serving.add_rms_norm(x, gain, residual, out_dtype=store, eps=eps,
                                              group=group)
    keep = [0, 1, 3, 4]
    _check(x[keep], residual[keep], gain, out[keep], None if scale is None else scale[keep],
           summed[keep], group, eps)
    assert power < 0 or not out[2].float().any()
