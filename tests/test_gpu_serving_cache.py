"""The paged 8-bit cache: appending (hcKvAppend) and attention (hcKvAttention),
through hc_b200.serving, against oracle/serving.py.

Appending is determined byte by byte (each step is one correctly rounded
float32 operation), so it is compared exactly.  Attention, per output element:
keys, values and probabilities' signs enter exactly; scores are fp32 sums of
`dim` products of f16-exact factors (2^-22 of sum |q||k| each, times the scale,
as an absolute error of the exponent: a relative error of the probability);
probabilities round to f16 (2^-11 with the exponential's own 2^-21), and the
output once to bf16 (2^-8):
    |out - o| <= 2^-8 |o| + (2^-11 + 2 * dE) * sum_j p_j |v_j|,
    dE = (dim / 16 + 4) * 2^-22 * scale * sum |q||k| at its largest + 2^-20.
Probabilities are held as 2^11 p / (at most 2^4 times the largest so far) in
f16, whose smallest step is 2^-24: one below 2^-25 of the largest contribution
may lose up to half of that, 2^-36 of it: (number of tokens) * 2^-36 * max |v|
on top."""

import numpy as np
import pytest
import torch

from hc_b200 import serving
from oracle import serving as oracle

pytestmark = pytest.mark.gpu

TORCH = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


class Setup:
    """A cache with earlier tokens, new tokens, and the oracle's view of both."""

    def __init__(self, store, lengths, fresh, block=16, heads=2, share=2, dim=64, seed=0,
                 spare=2, one_each=False, layout="phbd", width=None):
        rng = np.random.default_rng(seed)
        self.store, self.block, self.heads, self.share, self.dim = store, block, heads, share, dim
        self.lengths, self.fresh = list(lengths), list(fresh)
        need = [-(-max(n, 0) // block) for n in lengths]
        self.width = max(need + [1]) if width is None else width
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).tolist()
        self.table = np.full((len(lengths), self.width), -1, np.int32)
        for s, n in enumerate(need):
            for b in range(min(n, self.width)):
                self.table[s, b] = order.pop()
        self.starts = np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
        tokens = int(self.starts[-1])
        shape = (self.pages, heads, block, dim)
        if store == "int8":
            self.raw = [rng.integers(-127, 128, shape).astype(np.int8).view(np.uint8)
                        for _ in range(2)]
            self.scale = [(rng.random((self.pages, heads)) * 0.02 + 0.001).astype(np.float32)
                          for _ in range(2)]
        else:
            self.raw = [oracle.to_e4m3(rng.normal(size=shape) * 60) for _ in range(2)]
            self.scale = [np.float32(2.0) ** rng.integers(-9, -4, (self.pages, heads))
                          for _ in range(2)]
        bf16 = lambda a: torch.from_numpy(a).float().cuda().bfloat16()  # noqa: E731
        spread = np.exp(rng.normal(size=(tokens, heads, 1)))
        self.k = bf16(rng.normal(size=(tokens, heads, dim)) * spread)
        self.v = bf16(rng.normal(size=(tokens, heads, dim)) * spread)
        self.q = bf16(rng.normal(size=(tokens, heads * share, dim)) * 1.5)
        self.max_new = max(list(fresh) + [1])
        self.one_each = one_each
        self.layout = layout
        self.upload()

    def upload(self):
        dev = []
        for raw in self.raw:
            t = torch.from_numpy(raw.copy()).cuda()
            if self.layout == "pbhd":  # tokens outside heads
                t = t.transpose(1, 2).contiguous().transpose(1, 2)
            dev.append(t.view(TORCH[self.store]))
        scales = [torch.from_numpy(s.astype(np.float32).copy()).cuda() for s in self.scale]
        self.cache = serving.KvCache(dev[0], dev[1], scales[0], scales[1])
        self.d_table = torch.from_numpy(self.table).cuda()
        self.d_lengths = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.d_starts = None if self.one_each else torch.from_numpy(self.starts).cuda()

    def place(self):
        return (self.d_table, self.d_lengths, self.d_starts)

    def spans(self):
        return oracle.place(self.lengths, self.starts, int(self.k.shape[0]), self.width,
                            self.block, self.max_new)

    def bytes(self):
        return [t.view(torch.uint8).cpu().numpy() for t in (self.cache.k, self.cache.v)]

    def append(self):
        serving.kv_append(self.cache, self.k, self.v, *self.place(), max_new=self.max_new)

    def check_append(self):
        got, scales = self.bytes(), (self.cache.k_scale, self.cache.v_scale)
        for i, new in enumerate((self.k, self.v)):
            raw, scale = oracle.kv_append(self.raw[i], self.scale[i], new.double().cpu().numpy(),
                                          self.table.tolist(), self.spans(), self.store)
            assert np.array_equal(scales[i].cpu().numpy(), scale.astype(np.float32))
            assert np.array_equal(got[i], raw)

    def attend(self, window=0, **more):
        return serving.kv_attention(self.cache, self.q, *self.place(), max_new=self.max_new,
                                    window=window, return_lse=True, **more)

    def check_attention(self, out, lse, window=0, scale=None, q=None):
        scale = self.dim ** -0.5 if scale is None else scale
        q = (self.q if q is None else q).double().cpu().numpy()
        values = [oracle.stored_values(b, self.store) for b in self.bytes()]
        scales = [s.double().cpu().numpy() for s in (self.cache.k_scale, self.cache.v_scale)]
        args = (q, self.table.tolist(), self.spans(), self.share, scale, window)
        want, want_lse = oracle.kv_attention(values, scales, *args)
        with np.errstate(all="ignore"):
            most, _ = oracle.kv_attention((values[0], np.abs(values[1])), scales, *args)
        top = max(np.abs(values[0] * scales[0][:, :, None, None]).max(initial=0), 0)
        d_e = (self.dim / 16 + 4) * 2.0 ** -22 * scale * np.abs(q).max(initial=0) * top * self.dim
        tail = max(self.lengths + [1]) * 2.0 ** -36 * np.abs(
            values[1] * scales[1][:, :, None, None]).max(initial=0)
        got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        room = 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2 * (d_e + 2.0 ** -20)) * most + tail
        assert not np.isnan(got).any()
        assert np.all(np.abs(got - want) <= room)
        dead = np.isneginf(want_lse)
        assert np.array_equal(dead, np.isneginf(got_lse))
        live = ~dead
        assert np.all(np.abs(got_lse[live] - want_lse[live]) <=
                      d_e + 2.0 ** -20 + 2.0 ** -22 * np.abs(want_lse[live]))


STORES = ["int8", "e4m3"]


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("block", [16, 32, 64, 256])
def test_append_one_token_each(store, block):
    lengths = [1, 2, block, block + 1, 3 * block - 1, 3 * block, 77]
    s = Setup(store, lengths, [1] * len(lengths), block=block, one_each=True)
    s.append()
    s.check_append()


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 128, 256])
def test_append_ragged(store, dim):
    s = Setup(store, [40, 5, 1, 64, 100, 33], [40, 3, 1, 17, 0, 33], block=32, heads=3, dim=dim)
    s.append()
    s.check_append()


@pytest.mark.parametrize("store", STORES)
def test_append_token_by_token_grows_scales(store):
    """Sixteen calls of one token: what a decoding loop does.  Each is exact."""
    s = Setup(store, [1], [1], one_each=True)
    rng = np.random.default_rng(5)
    for n in range(1, 20):
        s.lengths = [n]
        s.d_lengths.fill_(n)
        if n > 16:
            s.table = np.array([[s.table[0, 0], 1 - s.table[0, 0] if s.table[0, 0] < 2 else 0]],
                               np.int32)
            s.width = 2
            s.d_table = torch.from_numpy(s.table).cuda()
        size = np.exp(rng.normal() * 2)
        s.k = (torch.randn(1, 2, 64, device="cuda") * size).bfloat16()
        s.v = (torch.randn(1, 2, 64, device="cuda") * size).bfloat16()
        s.append()
        s.check_append()
        s.raw = s.bytes()
        s.scale = [t.cpu().numpy() for t in (s.cache.k_scale, s.cache.v_scale)]


@pytest.mark.parametrize("store", STORES)
def test_append_what_is_not_finite(store):
    s = Setup(store, [20, 20, 3], [4, 2, 3], block=16)
    s.k[0, 0, 3], s.k[1, 1, 5], s.k[2, 0, 1] = float("nan"), float("inf"), -float("inf")
    s.v[5] = 0
    s.v[6:] = 0
    s.append()
    s.check_append()


@pytest.mark.parametrize("store", STORES)
def test_append_layout_and_strides(store):
    s = Setup(store, [40, 9], [7, 9], layout="pbhd", heads=4, dim=128)
    wide = torch.zeros(16, 4, 264, dtype=torch.bfloat16, device="cuda")
    wide[:, :, :128], wide[:, :, 129:257] = s.k, s.v
    s.k, s.v = wide[:, :, :128], wide[:, :, 129:257]  # v's rows are not 16-byte aligned
    s.append()
    s.check_append()


def test_append_leaves_the_rest_alone():
    """Bad pages, lengths that leave no room, rows behind the last sequence."""
    s = Setup("int8", [40, 20, 2, 0, 33], [5, 4, 6, 1, 2], width=2)
    s.table[1, 1] = s.pages  # the block of sequence 1's new tokens: no such page
    s.table[0, 1] = -7
    s.upload()
    before = s.bytes()
    s.append()
    s.check_append()
    written = [p for p in range(s.pages) if not np.array_equal(before[0][p], s.bytes()[0][p])]
    # Sequence 2's newest tokens, and of sequence 4's two the one before the table's end.
    assert written == sorted([s.table[2, 0], s.table[4, 1]])


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("share", [1, 4, 5, 8, 12, 16])
def test_attention_one_token(store, dim, share):
    lengths = [1, 15, 16, 17, 130, 300, 47]
    s = Setup(store, lengths, [1] * len(lengths), share=share, dim=dim, one_each=True)
    s.append()
    s.check_attention(*s.attend())


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("block", [16, 32, 128, 256])
@pytest.mark.parametrize("window", [0, 1, 16, 50, 5000])
def test_attention_drafts_and_windows(store, block, window):
    s = Setup(store, [200, 9, 64, 300, 1], [5, 9, 1, 3, 1], block=block, share=3, dim=64)
    s.append()
    s.check_attention(*s.attend(window), window=window)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim,share", [(64, 1), (128, 4), (256, 2), (96, 7)])
def test_attention_chunks(store, dim, share):
    """Prompts in chunks: many rows per sequence, some whole, some behind others."""
    s = Setup(store, [150, 70, 33], [100, 70, 20], block=32, share=share, dim=dim)
    s.append()
    s.check_attention(*s.attend())
    s.check_attention(*s.attend(40), window=40)


@pytest.mark.parametrize("store", STORES)
def test_attention_splits_one_long_sequence(store):
    """One head over a long cache: every share of the GPU holds a piece, joined twice
    alike; and many short sequences, more than one pass over their lengths takes."""
    s = Setup(store, [20000], [2], block=64, heads=1, share=1, dim=128)
    s.append()
    out, lse = s.attend()
    s.check_attention(out, lse)
    again, lse2 = s.attend()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    rng = np.random.default_rng(3)
    lengths = rng.integers(0, 40, 600).tolist()
    s = Setup(store, lengths, [1] * 600, heads=1, share=2, dim=32, one_each=True)
    s.append()
    s.check_attention(*s.attend())


def test_attention_shares_pages_between_sequences():
    """A common prefix: two tables that name the same pages."""
    s = Setup("int8", [40, 40], [1, 1], one_each=True)
    s.table[1, :2] = s.table[0, :2]
    s.upload()
    s.append()
    s.check_attention(*s.attend())


def test_attention_rows_that_see_nothing():
    """Lengths of zero, pages that do not exist, rows without a position."""
    s = Setup("e4m3", [0, 40, 3, 17, 90], [1, 1, 6, 2, 1], share=2, width=3)
    s.table[1] = -1
    s.table[3, 0] = s.pages + 5
    s.upload()
    out, lse = s.attend()
    s.check_attention(out, lse)
    dead = torch.isneginf(lse[:, 0])
    # The sequence of length 0, the one without pages, three rows before position 0, the
    # last token of a block that is not there, and the row whose position lies behind
    # the table.
    assert dead.tolist() == [True, True, True, True, True, False, False, False, True, False, True]
    assert torch.equal(out[dead], torch.zeros_like(out[dead]))


def test_attention_rows_behind_the_last_sequence_stay():
    s = Setup("int8", [40, 9], [2, 3])
    padded = torch.randn(9, 4, 64, device="cuda").bfloat16()
    padded[:5] = s.q
    out = torch.full_like(padded, 3.0)
    got = serving.kv_attention(s.cache, padded, *s.place(), max_new=5, out=out)
    assert got is out and torch.equal(out[5:], torch.full_like(out[5:], 3.0))
    want, _ = s.attend()
    assert torch.equal(out[:5], want)


def test_attention_masks_what_is_not_finite():
    """NaN in places that a row does not see: behind a sequence's end, later tokens of
    a draft, outside the window, other sequences' pages."""
    s = Setup("e4m3", [37, 80], [4, 3], share=2, dim=64)
    s.append()
    clean, clean_lse = s.attend(20)
    raw = s.bytes()
    page, at = s.table[0, 2], 37 % 16
    for which in (s.cache.k, s.cache.v):
        view = which.view(torch.uint8)
        view[page, :, at:] = 0x7F                # behind the end
        view[s.table[0, 0]] = 0xFF               # positions 0..15
        view[s.table[0, 2], 1, at - 1, 5] = 0x7F  # the newest token: seen by the last row alone
    s.cache.k.view(torch.uint8)[page, 1, at - 1, 5] = int(raw[0][page, 1, at - 1, 5])
    out, lse = s.attend(20)
    # Rows 0 and 1 (positions 33 and 34) see 14 or 15 first: NaN keys and values.
    assert torch.isnan(out[:2]).all() and torch.isnan(lse[:2]).all()
    # Rows 2 and 3 do not; row 3 alone sees its own value, of key/value head 1.
    assert torch.isnan(out[3, 2:, 5]).all()
    out[3, 2:, 5] = clean[3, 2:, 5]
    assert torch.equal(out[2:], clean[2:]) and torch.equal(lse[2:], clean_lse[2:])


@pytest.mark.parametrize("store", STORES)
def test_attention_scales_from_tiny_to_large(store):
    """Block scales that differ by many orders, zeros among them."""
    s = Setup(store, [200, 120], [1, 1], one_each=True, dim=64)
    s.append()
    for i, p in enumerate(s.table[0, :12]):
        s.cache.v_scale[p] = [0.0, 1e-30, 1e-6, 1.0, 100.0, 2.0 ** -14][i % 6]
    s.cache.k_scale[s.table[0, 3]] = 0.0
    s.check_attention(*s.attend())
    s.cache.v_scale.fill_(2.0 ** -40)
    s.check_attention(*s.attend())
    s.cache.v_scale.zero_()
    out, lse = s.attend()
    assert torch.equal(out, torch.zeros_like(out)) and torch.isfinite(lse).all()


def test_attention_query_rows_of_any_size():
    s = Setup("int8", [50, 50, 50, 50], [1, 1, 1, 1], one_each=True, dim=64)
    s.append()
    s.cache.k_scale.mul_(2.0 ** -20)
    s.q[0] *= 2.0 ** 30  # beyond f16
    s.q[1] *= 2.0 ** -30
    s.q[2] = 0
    s.q[3, 0, 0] = float("inf")
    s.q[3, 1, 0] = float("nan")
    out, lse = s.attend(scale=2.0 ** -6)
    assert not torch.isfinite(out[3, :2]).any()
    assert torch.isfinite(out[3, 2:]).all()
    q = s.q.clone()
    q[3] = 0
    out[3], lse[3] = s.attend(scale=2.0 ** -6)[0][2], lse[2]
    values = [oracle.stored_values(b, "int8") for b in s.bytes()]
    scales = [x.double().cpu().numpy() for x in (s.cache.k_scale, s.cache.v_scale)]
    want, want_lse = oracle.kv_attention(values, scales, q.double().cpu().numpy(),
                                         s.table.tolist(), s.spans(), 2, 2.0 ** -6, 0)
    got = out.double().cpu().numpy()
    # Row 0's probabilities sit on one or two tokens; the scores' error is relative to
    # the scores (up to 2^13): 2^-22 * 8 * 2^13 of exponent.
    most = np.abs(values[1] * scales[1][:, :, None, None]).max()
    assert np.all(np.abs(got - want)[:3] <= 2.0 ** -8 * np.abs(want[:3]) + 2.0 ** -5 * most)
    assert np.all(np.abs(got - want)[1:3] <= 2.0 ** -8 * np.abs(want[1:3]) + 2.0 ** -10 * most)


@pytest.mark.parametrize("store", STORES)
def test_attention_layouts_and_strides(store):
    s = Setup(store, [100, 33], [3, 2], layout="pbhd", heads=4, share=2, dim=128)
    wide = torch.zeros(5, 3, 8, 136, dtype=torch.bfloat16, device="cuda")
    wide[:, 1, :, :128] = s.q
    s.append()
    base, base_lse = s.attend()
    s.check_attention(base, base_lse)
    out = torch.full((5, 3, 8, 136), 2.0, dtype=torch.bfloat16, device="cuda")
    got = serving.kv_attention(s.cache, wide[:, 1, :, :128], *s.place(), max_new=3,
                               out=out[:, 2, :, :128])
    assert torch.equal(got, base)
    assert torch.equal(out[:, :2], torch.full_like(out[:, :2], 2.0))
    assert torch.equal(out[:, 2, :, 128:], torch.full_like(out[:, 2, :, 128:], 2.0))


def test_step_on_another_stream_and_in_graphs():
    """A decoding step captured twice; both graphs replayed beside each other."""
    s = Setup("int8", [200, 3000], [1, 1], one_each=True, dim=128, heads=4)
    s.append()
    want, want_lse = s.attend()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s.append()
        out, lse = s.attend()
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    graphs, outs, qs = [], [], [s.q.clone(), torch.randn_like(s.q)]
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(serving.kv_attention(s.cache, q, *s.place()))
        graphs.append(graph)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want)
    assert torch.equal(outs[1], serving.kv_attention(s.cache, qs[1], *s.place()))


def test_a_decoding_loop():
    """The operators in a run, as a model's layer uses them, against the same steps in
    float64 on what the cache holds: norm, product, append, attention, product."""
    torch.manual_seed(0)
    seqs, heads, share, dim, hidden = 3, 2, 4, 64, 512
    cache = serving.KvCache.empty(12, heads, 16, dim)
    table = torch.randperm(12, device="cuda").int().view(3, 4)
    lengths = torch.zeros(3, dtype=torch.int32, device="cuda")

    def weights(n, k):
        return dict(w=torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda"),
                    scale=(torch.rand(n, k // 128, device="cuda") * 0.02).bfloat16(), group=128)

    qkv, back = weights((share + 2) * heads * dim, hidden), weights(hidden, share * heads * dim)
    gain = torch.rand(hidden, device="cuda").bfloat16() + 0.5
    residual = torch.randn(seqs, hidden, device="cuda").bfloat16()
    update = torch.zeros_like(residual)
    for step in range(20):
        q8, scale, residual = serving.add_rms_norm(update, gain, residual, out_dtype=torch.int8)
        x = serving.gemm_w4(q8, a_scale=scale, **qkv).view(seqs, -1, dim)
        q, k, v = x.split([share * heads, heads, heads], dim=1)
        lengths += 1
        serving.kv_append(cache, k, v, table, lengths)
        out, lse = serving.kv_attention(cache, q, table, lengths, return_lse=True)
        values = [oracle.stored_values(t.view(torch.uint8).cpu().numpy(), "e4m3")
                  for t in (cache.k, cache.v)]
        scales = [t.double().cpu().numpy() for t in (cache.k_scale, cache.v_scale)]
        spans = [(i, step, 1) for i in range(seqs)]
        want, _ = oracle.kv_attention(values, scales, q.double().cpu().numpy(), table.tolist(),
                                      spans, share, dim ** -0.5, 0)
        room = 2.0 ** -8 * np.abs(want) + 2.0 ** -9 * np.abs(want).max()
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= room)
        update = serving.gemm_w4(out.view(seqs, -1), **back)
        assert torch.isfinite(update).all()


def test_refusals():
    s = Setup("int8", [20, 9], [2, 1])
    q, (table, lengths, starts) = s.q, s.place()
    call = lambda **kw: serving.kv_attention(  # noqa: E731
        kw.get("cache", s.cache), kw.get("q", q), kw.get("table", table),
        kw.get("lengths", lengths), kw.get("starts", starts), max_new=kw.get("max_new", 2),
        window=kw.get("window", 0), scale=kw.get("scale"))
    for kw, match, error in (
            (dict(q=q.float()), "bfloat16", TypeError),
            (dict(q=q[:, :3]), "multiple", ValueError),
            (dict(q=q[:, :, :32]), "expected", ValueError),
            (dict(table=table.long()), "int32", TypeError),
            (dict(lengths=lengths[:1]), "lengths", ValueError),
            (dict(starts=starts[:2]), "starts", ValueError),
            (dict(max_new=None), "max_new", ValueError),
            (dict(starts=None, q=q[:1]), "one row per sequence", ValueError),
            (dict(window=-1), "window", RuntimeError),
            (dict(scale=float("nan")), "scale", RuntimeError)):
        with pytest.raises(error, match=match):
            call(**kw)
    with pytest.raises(TypeError, match="bfloat16"):
        serving.kv_append(s.cache, s.k.float(), s.v, *s.place(), max_new=2)
    with pytest.raises(ValueError, match="v: expected"):
        serving.kv_append(s.cache, s.k, s.v[:2], *s.place(), max_new=2)
    k, ks = s.cache.k, s.cache.k_scale
    with pytest.raises(TypeError, match="int8 or float8_e4m3fn"):
        serving.KvCache(k.float(), k.float(), ks, ks)
    with pytest.raises(ValueError, match="k_scale"):
        serving.KvCache(k, k, ks[:1], ks[:1])
    odd = torch.zeros(4, 2, 24, 64, dtype=torch.int8, device="cuda")
    bad = serving.KvCache(odd, odd, ks[:4].contiguous(), ks[:4].contiguous())
    with pytest.raises(RuntimeError, match="multiple of 16"):
        call(cache=bad)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("tiny", [-16, -30, -60])
def test_attention_zeros_outweigh_small_values(store, tiny):
    """Blocks of zeros that hold nearly all of the probability beside blocks of small
    values: what little the output is has its full precision.  (More tiles than warps.)"""
    lengths = [12000, 11000, 12000, 10000, 9000, 12000]
    s = Setup(store, lengths, [1] * 6, one_each=True, dim=64, heads=2, share=2)
    s.append()
    # Keys along the query in the blocks of zeros alone: a score of 8 more, e^8 of the weight.
    s.q = torch.zeros(6, 4, 64, dtype=torch.bfloat16, device="cuda")
    s.q[:, :, 0] = 8
    raw = 64 if store == "int8" else int(oracle.to_e4m3(np.array([64.0]))[0])
    zeros = torch.zeros(s.pages, dtype=torch.bool, device="cuda")
    for row in s.d_table:
        zeros[row[row >= 0][::2].long()] = True
    k = s.cache.k.view(torch.uint8)
    k.zero_()
    k[zeros, :, :, 0] = raw
    s.cache.k_scale.fill_(2.0 ** -3)
    s.cache.v_scale.fill_(2.0 ** tiny)
    s.cache.v_scale[zeros] = 0
    out, lse = s.attend()
    values = [oracle.stored_values(b, store) for b in s.bytes()]
    scales = [t.double().cpu().numpy() for t in (s.cache.k_scale, s.cache.v_scale)]
    args = (s.q.double().cpu().numpy(), s.table.tolist(), s.spans(), 2, 64 ** -0.5, 0)
    want, want_lse = oracle.kv_attention(values, scales, *args)
    most, _ = oracle.kv_attention((values[0], np.abs(values[1])), scales, *args)
    assert (most > 0).all() and most.max() < 448 * 2.0 ** (tiny - 10)
    # The scores, 0 and 8, are exact in f16 and float32; the sums have up to 2^7 rounded
    # partial sums per lane, 2^-17; probabilities round to f16.
    room = 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2.0 ** -16) * most
    assert np.all(np.abs(out.double().cpu().numpy() - want) <= room)
    assert np.all(np.abs(lse.double().cpu().numpy() - want_lse) <= 2.0 ** -16)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-6])
def test_attention_scales_of_any_sign(store, scale):
    s = Setup(store, [300, 17, 90], [1, 3, 2], block=32, share=3, dim=64)
    s.append()
    for window in (0, 20):
        out, lse = s.attend(window, scale=scale)
        want, want_lse = oracle.kv_attention(
            [oracle.stored_values(b, store) for b in s.bytes()],
            [t.double().cpu().numpy() for t in (s.cache.k_scale, s.cache.v_scale)],
            s.q.double().cpu().numpy(), s.table.tolist(), s.spans(), 3, scale, window)
        top = np.abs(want).max() * 4
        # |scale| up to the default's, so the default's bound on the scores' error (2^-9 at these
        # magnitudes, as in check_attention) holds.
        assert np.all(np.abs(out.double().cpu().numpy() - want) <=
                      2.0 ** -8 * np.abs(want) + 2.0 ** -9 * top)
        assert np.all(np.abs(lse.double().cpu().numpy() - want_lse) <= 2.0 ** -9)


def test_threads_with_a_stream_each():
    """A step in each of three threads at once: streams and workspaces are each one's own."""
    import threading

    setups = [Setup(store, lengths, fresh, share=share, dim=64, seed=i)
              for i, (store, lengths, fresh, share) in enumerate((
                  ("int8", [2000, 40], [1, 1], 2), ("e4m3", [700], [60], 4),
                  ("int8", [300, 9, 64], [5, 9, 1], 3)))]
    w = torch.randint(0, 256, (128, 32), dtype=torch.uint8, device="cuda")
    scale, gain = torch.rand(128, 2, device="cuda"), torch.rand(64, device="cuda").bfloat16()

    def step(s):
        out, lse = s.attend()
        h, a_scale, _ = serving.add_rms_norm(out.view(-1, 64), gain, out_dtype=torch.int8)
        return out, lse, serving.gemm_w4(h, w, scale, group=32, a_scale=a_scale)

    for s in setups:
        s.append()
    want = [step(s) for s in setups]
    torch.cuda.synchronize()
    got = [[] for _ in setups]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got[i] = [step(setups[i]) for _ in range(50)]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(3):
        assert len(got[i]) == 50
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


@pytest.mark.parametrize("store", STORES)
def test_caches_beyond_four_gigabytes(store):
    """The same step in a small cache and in one whose pages lie beyond 2^32 bytes (and at
    both ends of it): the same bytes and outputs."""
    pages, heads, block, dim = 70000, 8, 64, 128
    small = serving.KvCache.empty(40, heads, block, dim, TORCH[store])
    large = serving.KvCache.empty(pages, heads, block, dim, TORCH[store])
    gen = torch.Generator(device="cuda").manual_seed(1)
    rows = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).bfloat16()  # noqa: E731
    lengths = torch.tensor([600, 900, 130], dtype=torch.int32, device="cuda")
    table = torch.full((3, 15), -1, dtype=torch.int32, device="cuda")
    order = torch.randperm(40, device="cuda", generator=gen).int()
    table[0, :10], table[1], table[2, :3] = order[:10], order[10:25], order[25:28]
    far = torch.where(table < 0, table, torch.where(table % 2 == 0, table, pages - 1 - table))
    starts = torch.tensor([0, 600, 1500, 1630], dtype=torch.int32, device="cuda")
    k, v, q = rows(1630, heads, dim), rows(1630, heads, dim), rows(1630, 2 * heads, dim)
    for cache, at in ((small, table), (large, far)):
        serving.kv_append(cache, k, v, at, lengths, starts, max_new=900)
    for a, b, sa, sb in ((small.k, large.k, small.k_scale, large.k_scale),
                         (small.v, large.v, small.v_scale, large.v_scale)):
        used, there = table[table >= 0].long(), far[table >= 0].long()
        assert torch.equal(a.view(torch.uint8)[used], b.view(torch.uint8)[there])
        assert torch.equal(sa[used], sb[there])
    few = torch.tensor([0, 1, 3, 8], dtype=torch.int32, device="cuda")
    for new, at in ((starts, 900), (few, 5)):
        tokens = int(new[-1])
        outs = [serving.kv_attention(c, q[:tokens], t, lengths, new, max_new=at, return_lse=True)
                for c, t in ((small, table), (large, far))]
        assert torch.isfinite(outs[0][1]).all()
        assert all(torch.equal(a, b) for a, b in zip(*outs))
