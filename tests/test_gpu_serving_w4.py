"""Products with 4-bit weights (hcGemmW4, hc_b200.serving.gemm_w4) against the
formula in 64 bits.

Tolerances, with P = sum_k |a| |u - z| s and Q = sum_k |a| s.  Up to 8 rows
weights enter exactly.  A group's sum is an fp32 sum in the tensor cores, which
add in blocks of 16 and may drop bits below 2^-23 of the largest term of a
block; it is formed per segment of 128 or 32 k: off by at most (128 / 16 + 8) *
2^-22 of the terms' sum, the terms being a u (of 15 Q), and z sum(a) comes off
with two roundings of 2^-24 of 15 Q.  Activations below 2^-24 of their segment's
largest lose up to half of 2^-24 of a sixteenth of 2^-14 of it, 2^-35 each.  int8
sums are exact.  Adding the segments costs (K / 32 + 8) * 2^-24 of P + 30 Q, the
result rounds to bf16 once: 2^-8 of it.  More rows: every weight is rounded to bf16 first, 2^-8 P in
the worst case, int8 activations with several scales per row likewise; the
fp32 sum over K is off by (K / 16 + 8) * 2^-22 P."""

import numpy as np
import pytest
import torch

from hc_b200 import serving
from hc_b200.hckernel.kernel import get_context
from oracle import serving as oracle

pytestmark = pytest.mark.gpu


def _case(m, n, k, group, zeros, seed=0, a8=False, scale_dtype=torch.bfloat16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    groups = -(-k // group)
    dev = dict(device="cuda", generator=gen)
    c = dict(w=torch.randint(0, 256, (n, (k + 1) // 2), dtype=torch.uint8, **dev),
             scale=(torch.rand(n, groups, **dev) * 0.02 + 0.001).to(scale_dtype),
             zero=torch.randint(0, 16, (n, groups), dtype=torch.uint8, **dev) if zeros else None,
             group=group)
    if a8:
        c["a"] = torch.randint(-127, 128, (m, k), dtype=torch.int8, **dev)
        c["a_scale"] = torch.rand(m, 1, **dev) * 0.1 + 0.01
    else:
        c["a"] = torch.randn(m, k, **dev).bfloat16()
    return c


def _weights(c):
    """The weights in float64, on the GPU (oracle.serving.unpack_w4 on the host says
    the same: test_exact_on_small_integers)."""
    n, k, group = c["w"].shape[0], c["a"].shape[1], c["group"]
    u = torch.stack((c["w"] & 15, c["w"] >> 4), dim=2).view(n, -1)[:, :k].double()
    at = torch.arange(k, device="cuda") // group
    z = 8.0 if c["zero"] is None else c["zero"].double()[:, at]
    return (u - z) * c["scale"].double()[:, at]


def _check(c, out, a_group=0):
    k = c["a"].shape[1]
    a = c["a"].double()
    if "a_scale" in c:
        width = a_group if 0 < a_group < k else k
        a = a * c["a_scale"].double()[:, torch.arange(k, device="cuda") // width]
    w = _weights(c)
    want, most = a @ w.T, a.abs() @ w.abs().T
    got = out.double()
    assert got.shape == want.shape and not torch.isnan(got).any()
    if a.shape[0] <= 8 and k <= 8192:
        s = c["scale"].double()[:, torch.arange(k, device="cuda") // c["group"]]
        q = a.abs() @ s.T
        room = (k / 32 + 8) * 2.0 ** -24 * (most + 30 * q)
        if "a_scale" not in c:
            room += 17 * 2.0 ** -22 * 15 * q
            room += 2.0 ** -35 * 15 * a.abs().amax(1, keepdim=True) @ s.sum(1)[None]
    else:
        room = ((k / 16 + 8) * 2.0 ** -22 + 2.0 ** -8 * (2 if "a_scale" in c else 1)) * most
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + room).all()


SHAPES = [(1, 16, 128), (1, 128, 128), (1, 4096, 4096), (2, 130, 256), (5, 1000, 8160),
          (8, 64, 1024), (9, 333, 640), (16, 256, 4096), (17, 500, 1152), (32, 1024, 2048),
          (33, 200, 512), (64, 384, 8192), (65, 384, 1024), (130, 300, 1088), (300, 520, 256), (256, 384, 2048),
          (250, 130, 4224), (48, 1030, 4096), (1100, 200, 512)]


@pytest.mark.parametrize("a8", [False, True])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256, 1 << 20])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(shape, group, zeros, a8):
    c = _case(*shape, group, zeros, a8=a8)
    _check(c, serving.gemm_w4(**c))


@pytest.mark.parametrize("a8", [False, True])
@pytest.mark.parametrize("m", [1, 7, 40, 100])
@pytest.mark.parametrize("k", [1, 2, 31, 33, 100, 127, 129, 1000, 1001])
def test_odd_depths(k, m, a8):
    for group in (32, 128):
        c = _case(m, 77, k, group, True, a8=a8)
        _check(c, serving.gemm_w4(**c))


def test_depth_of_zero_and_no_rows():
    c = _case(3, 50, 64, 32, False)
    c.update(a=c["a"][:, :0], w=c["w"][:, :0], scale=c["scale"][:, :0])
    assert torch.equal(serving.gemm_w4(**c), torch.zeros(3, 50, dtype=torch.bfloat16,
                                                         device="cuda"))
    c = _case(3, 50, 64, 32, False)
    c["a"] = c["a"][:0]
    assert serving.gemm_w4(**c).shape == (0, 50)


@pytest.mark.parametrize("m", [1, 5, 8, 12, 64])
def test_depths_and_widths_that_share_the_work_differently(m):
    """Depths that give the warps 1 to 16 ways to divide, tiles fewer and more than the
    SMs; rows that do not fit in shared memory; twice alike."""
    for n, k in ((40, 128), (200, 256), (5000, 384), (200, 1000), (3000, 1152), (77, 4224),
                 (4800, 2048), (33, 14336), (20, 40960)):
        c = _case(m, n, k, 64, True)
        first = serving.gemm_w4(**c)
        _check(c, first)
        assert torch.equal(first, serving.gemm_w4(**c))  # the order of the sums is fixed


@pytest.mark.parametrize("m", [3, 70])
def test_pitches_scales_and_activation_groups(m):
    c = _case(m, 96, 640, 64, True, scale_dtype=torch.float32)
    wide = torch.zeros(96, 352, dtype=torch.uint8, device="cuda")
    wide[:, :320] = c["w"]
    c["w"] = wide[:, :320]
    _check(c, serving.gemm_w4(**c))
    odd = torch.zeros(96, 321, dtype=torch.uint8, device="cuda")  # rows that are not aligned
    odd[:, 1:] = c["w"]
    c["w"] = odd[:, 1:]
    a = torch.zeros(m, 643, dtype=torch.bfloat16, device="cuda")
    a[:, :640] = c["a"]
    c["a"] = a[:, :640]
    out = torch.full((m, 100), 7.0, dtype=torch.bfloat16, device="cuda")
    _check(c, serving.gemm_w4(**c, out=out[:, :96]))
    assert torch.equal(out[:, 96:], torch.full_like(out[:, 96:], 7.0))
    c = _case(m, 96, 700, 64, True, a8=True)
    c["a_scale"] = torch.rand(m, 6, device="cuda") * 0.1 + 0.01
    _check(c, serving.gemm_w4(**c, a_group=128), a_group=128)


def test_exact_on_small_integers():
    """Integers that bf16 holds: the product has one right answer."""
    for m in (1, 20, 100):
        c = _case(m, 100, 96, 32, True)
        c["a"] = torch.randint(-2, 3, (m, 96), device="cuda").bfloat16()
        c["scale"] = torch.ones(100, 3, dtype=torch.bfloat16, device="cuda")
        w = torch.from_numpy(oracle.unpack_w4(c["w"].cpu().numpy(), np.ones((100, 3)),
                                              c["zero"].cpu().numpy(), 96, 32)).cuda()
        assert torch.equal(serving.gemm_w4(**c), (c["a"].double() @ w.T).bfloat16())


def test_values_that_are_not_finite_stay_in_their_rows():
    for m in (4, 80):
        c = _case(m, 64, 256, 128, False)
        want = serving.gemm_w4(**c)
        c["a"][1, 5] = float("inf")
        c["a"][2, 200] = float("nan")
        out = serving.gemm_w4(**c)
        assert torch.isnan(out[2]).all() and not torch.isfinite(out[1]).any()
        keep = [0] + list(range(3, m))
        assert torch.equal(out[keep], want[keep])


def test_norm_feeds_the_product():
    x = torch.randn(6, 1024, device="cuda").bfloat16()
    gain = torch.rand(1024, device="cuda").bfloat16() + 0.5
    for group in (0, 128):
        c = _case(6, 320, 1024, 128, True)
        q, scale, _ = serving.add_rms_norm(x, gain, out_dtype=torch.int8, group=group)
        c.update(a=q, a_scale=scale)
        _check(c, serving.gemm_w4(**c, a_group=group), a_group=group)


def test_other_stream_and_graph():
    for m in (2, 96):
        c = _case(m, 512, 1024, 128, True)
        want = serving.gemm_w4(**c)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = serving.gemm_w4(**c)
        side.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = serving.gemm_w4(**c)
        c["a"].copy_(torch.randn_like(c["a"]))
        graph.replay()
        want = serving.gemm_w4(**c)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_refusals():
    c = _case(2, 64, 256, 128, True)
    for change, match, error in (
            (dict(group=48), "multiple of 32", ValueError),
            (dict(w=c["w"][:, :-1]), "shapes", ValueError),
            (dict(w=c["w"].to(torch.int8)), "uint8", TypeError),
            (dict(scale=c["scale"].half()), "scale", TypeError),
            (dict(scale=c["scale"][:, :1]), "scale must be", ValueError),
            (dict(zero=c["zero"][:, :1]), "differ in shape", ValueError),
            (dict(a=c["a"].float()), "bfloat16 or int8", TypeError),
            (dict(a=c["a"].to(torch.int8)), "need their scales", ValueError),
            (dict(a_scale=torch.ones(2, 1, device="cuda")), "belongs to int8", ValueError),
            (dict(out=torch.empty(2, 64, device="cuda")), "out must be", TypeError)):
        with pytest.raises(error, match=match):
            serving.gemm_w4(**{**c, **change})
    a8 = _case(2, 64, 256, 128, True, a8=True)
    a8["a_scale"] = torch.ones(2, 3, device="cuda")
    with pytest.raises(RuntimeError, match="activations' group"):
        serving.gemm_w4(**a8, a_group=100)


def test_single_rows_of_any_stride():
    """A single row may report any stride, too deep for the kernel for few rows or not."""
    for k in (4098, 120002):
        c = _case(1, 48, k, 64, True, seed=k)
        want = serving.gemm_w4(**c)
        _check(c, want)
        a = torch.zeros(k + 16, dtype=torch.bfloat16, device="cuda")
        a[:k] = c["a"][0]
        got = serving.gemm_w4(**{**c, "a": a.as_strided((1, k), (8, 1))})
        assert torch.equal(got, want)
        w = c["w"][:1].clone().as_strided((1, (k + 1) // 2), (16, 1))
        one = {**c, "w": w, "scale": c["scale"][:1], "zero": c["zero"][:1]}
        assert torch.equal(serving.gemm_w4(**one), want[:, :1])


@pytest.mark.parametrize("m", [1, 8, 40])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("power", [-100, -60, 100, 112, 118, 120])
def test_activations_of_any_size(power, zeros, group, m):
    """Far from 1 in either direction: the bounds are relative, nothing overflows or
    vanishes on the way to a result that bfloat16 holds."""
    c = _case(m, 130, 640, group, zeros)
    c["a"] = (c["a"].float() * 2.0 ** power).bfloat16()
    _check(c, serving.gemm_w4(**c))


@pytest.mark.parametrize("m", [1, 8])
@pytest.mark.parametrize("group", [32, 128])
def test_the_largest_activations(group, m):
    """Every activation of a segment at bfloat16's end: their sum is beyond float32, the
    product with small weights is not."""
    c = _case(m, 64, 256, group, True)
    most = torch.finfo(torch.bfloat16).max
    c["a"] = torch.full_like(c["a"], most)
    c["a"][:, 1::2] = -most
    c["scale"] = (c["scale"].float() * 2.0 ** -8).bfloat16()
    _check(c, serving.gemm_w4(**c))
    c["a"] = torch.full_like(c["a"], most)
    c["scale"] = (c["scale"].float() * 2.0 ** -8).bfloat16()
    _check(c, serving.gemm_w4(**c))


@pytest.mark.parametrize("m", [3, 8, 40, 1000, 1024, 1025, 1300])
def test_int8_rows_with_one_scale_enter_exactly(m):
    """Integer sums below 2^24 that cancel to little: exact, then one product with the row's
    scale in float32 and one rounding.  (Scaled activations rounded to bfloat16 would leave
    an error of the size of the terms.)"""
    gen = torch.Generator(device="cuda").manual_seed(m)
    dev = dict(device="cuda", generator=gen)
    n, k = 72, 384
    a = torch.randint(-40, 41, (m, k // 3, 3), dtype=torch.int8, **dev)
    a[:, :, 2] = a[:, :, 0] + a[:, :, 1]
    u = torch.tensor([9, 9, 7], dtype=torch.uint8, device="cuda").repeat(n, k // 3)
    u[:, 0] = torch.randint(0, 16, (n,), dtype=torch.uint8, **dev)
    w = u[:, 0::2] | u[:, 1::2] << 4
    a, a_scale = a.view(m, k), torch.rand(m, 1, **dev) * 0.1 + 0.01
    out = serving.gemm_w4(a, w, torch.ones(n, k // 32, device="cuda"), group=32, a_scale=a_scale)
    want = a.double() @ (u.double() - 8).T
    assert torch.equal(out, (want.float() * a_scale).bfloat16())


@pytest.mark.parametrize("m", [2, 20, 1100])
def test_row_scales_of_any_pitch_and_the_cuda_core_product(m):
    c = _case(m, 96, 256, 64, True, a8=True)
    want = serving.gemm_w4(**c)
    wide = torch.full((m, 5), float("nan"), device="cuda")
    wide[:, 2:3] = c["a_scale"]
    assert torch.equal(serving.gemm_w4(**{**c, "a_scale": wide[:, 2:3]}), want)
    ctx = get_context("cuda:0")
    ctx.set_option("gemm_variant", 3)  # (has no place for a row's scale)
    try:
        _check(c, serving.gemm_w4(**c))
        torch.cuda.synchronize()
    finally:
        ctx.set_option("gemm_variant", 0)


@pytest.mark.parametrize("group,m", [(32, 7), (32, 8), (64, 7), (64, 8), (128, 8)])
def test_eight_rows_of_the_deepest_that_fit(group, m):
    """8 rows of K = 8192: in groups of 128 they fit in shared memory and weights enter
    exactly; in finer groups fewer rows do, and the others take weights rounded to bf16
    (worst case 2^-8 of the terms' sum)."""
    c = _case(m, 96, 8192, group, True, seed=group)
    out = serving.gemm_w4(**c).double()
    w, a = _weights(c), c["a"].double()
    room = ((8192 / 16 + 8) * 2.0 ** -22 + 2.0 ** -8) * (a.abs() @ w.abs().T)
    assert ((out - a @ w.T).abs() <= 2.0 ** -8 * (a @ w.T).abs() + room).all()
    if group == 128 or (group, m) == (64, 7):
        _check(c, serving.gemm_w4(**c))


@pytest.mark.parametrize("group", [65537 * 32, 65536 * 32 * 4])
def test_groups_of_millions(group):
    """The group of a column is found for every depth: the last 32 columns of the group
    before a boundary belong to it."""
    m, n, groups = 9, 16, 7
    k = groups * group if group < 1 << 22 else 6 * group
    groups = k // group
    scale = torch.ones(n, groups, dtype=torch.bfloat16, device="cuda")
    scale *= 2.0 ** torch.arange(groups, device="cuda")
    w = torch.full((n, k // 2), 0x99, dtype=torch.uint8, device="cuda")
    for g in range(1, groups):
        a = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
        a[:, g * group - 32:g * group] = 1
        out = serving.gemm_w4(a, w, scale, group=group)
        assert torch.equal(out, torch.full_like(out, 32 * 2.0 ** (g - 1)))
        a[:, g * group - 32:g * group] = 0
        a[:, g * group:g * group + 32] = 1
        out = serving.gemm_w4(a, w, scale, group=group)
        assert torch.equal(out, torch.full_like(out, 32 * 2.0 ** g))
