"""Attention over the paged 8-bit cache for many query rows per head (the tcgen05
kernel of hcKvAttention), against oracle/serving.py.  The roundings are those of the
kernel for few rows, so are the bounds (tests/test_gpu_serving_cache.py): every
attention test of that file runs here again with this kernel whatever the number of
rows, and more at the sizes that are its own."""

import numpy as np
import pytest
import torch

from hc_b200 import serving
from hc_b200.hckernel.kernel import get_context
from tests import test_gpu_serving_cache as few
from tests.test_gpu_serving_cache import STORES, Setup

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def rows_kernel():
    ctx = get_context("cuda:0")
    ctx.set_option("attention_variant", 2)
    yield ctx
    ctx.set_option("attention_variant", 0)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("share", [1, 5, 16])
def test_rows_one_token(store, dim, share):
    few.test_attention_one_token(store, dim, share)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("block", [16, 32, 256])
@pytest.mark.parametrize("window", [0, 1, 50, 5000])
def test_rows_drafts_and_windows(store, block, window):
    few.test_attention_drafts_and_windows(store, block, window)


@pytest.mark.parametrize("name", [
    "test_attention_shares_pages_between_sequences", "test_attention_rows_that_see_nothing",
    "test_attention_rows_behind_the_last_sequence_stay",
    "test_attention_masks_what_is_not_finite", "test_attention_query_rows_of_any_size",
    "test_step_on_another_stream_and_in_graphs", "test_a_decoding_loop"])
def test_rows_what_holds_for_few(name):
    getattr(few, name)()


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("name", [
    "test_attention_splits_one_long_sequence", "test_attention_scales_from_tiny_to_large",
    "test_attention_layouts_and_strides"])
def test_rows_what_holds_for_few_of_each_type(name, store):
    getattr(few, name)(store)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim,share,block", [(64, 4, 16), (128, 4, 64), (128, 1, 128),
                                             (256, 3, 32), (80, 9, 48), (192, 2, 256)])
@pytest.mark.parametrize("window", [0, 130])
def test_rows_chunks(store, dim, share, block, window):
    """Whole prompts, chunks behind earlier tokens, single rows among them."""
    s = Setup(store, [310, 700, 1, 129, 260], [310, 150, 1, 1, 33], block=block, share=share,
              dim=dim, heads=2)
    s.append()
    s.check_attention(*s.attend(window), window=window)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_divide_a_long_sequence(store, dim):
    """A few row tiles over a long cache: parts joined, twice alike, and other calls of
    other sizes in the same workspace between."""
    s = Setup(store, [9000], [20], block=64, heads=2, share=8, dim=dim)
    s.append()
    out, lse = s.attend()
    s.check_attention(out, lse)
    other = Setup(store, [2500, 40], [3, 40], block=16, heads=3, share=3, dim=dim, seed=5)
    other.append()
    other.check_attention(*other.attend())
    again, lse2 = s.attend()
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("seqs", [3, 40, 1100])
def test_rows_one_prompt_among_single_tokens(store, seqs):
    """A prompt beside sequences of one token, of none and without a place: the units
    that there are, found over more than one pass of a CTA's threads."""
    rng = np.random.default_rng(seqs)
    lengths = rng.integers(0, 60, seqs)
    fresh = np.minimum(rng.integers(0, 2, seqs), lengths)
    lengths[seqs // 2], fresh[seqs // 2] = 400, 390
    fresh[1] = lengths[1] + 2  # more new tokens than the sequence is long
    s = Setup(store, lengths.tolist(), fresh.tolist(), block=16, share=3, dim=64, heads=2)
    s.append()
    s.check_attention(*s.attend())


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_again_and_again(store, dim):
    """Sequences of few tiles, many times over: nothing is read before it is complete, and
    every row is written (the outputs are NaN before each call)."""
    s = Setup(store, [310, 700, 1, 129, 260], [310, 150, 1, 1, 33], block=32, share=3, dim=dim)
    s.append()
    first, first_lse = s.attend()
    s.check_attention(first, first_lse)
    out = torch.empty_like(first)
    for _ in range(300):
        out.fill_(float("nan"))
        _, lse = s.attend(out=out)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)


@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("dim,share", [(64, 3), (128, 1), (256, 3)])
def test_workspace_holds_nothing_but_counters(rows_kernel, store, dim, share, variant):
    """Whatever the workspace holds behind its counters, it is written before it is read."""
    rows_kernel.set_option("attention_variant", variant)
    for lengths, fresh in (([310, 700, 1, 129, 260], [310, 150, 1, 1, 33]), ([9000], [5]),
                           ([3000, 17, 900], [1, 1, 1])):
        s = Setup(store, lengths, fresh, block=32, share=share, dim=dim)
        s.append()
        want, want_lse = s.attend()
        s.check_attention(want, want_lse)
        for _ in range(5):
            for buf in serving._scratch.values():
                buf[4096:].fill_(0xFF)
            out = torch.full_like(s.q, float("nan"))
            _, lse = s.attend(out=out)
            assert torch.equal(out, want) and torch.equal(lse, want_lse)


def test_rows_missing_pages():
    """Blocks that are not there among those that are, whole tiles of them too."""
    s = Setup("int8", [900, 300], [60, 300], block=16, share=4, dim=128)
    s.append()
    for b in [0, 3, 4, *range(8, 25), 50]:
        s.table[0, b] = -1
    s.table[1, :10] = s.pages + 7
    s.upload()
    out, lse = s.attend()
    s.check_attention(out, lse)


@pytest.mark.parametrize("window", [0, 60])
def test_rows_nan_values(window):
    """A NaN among the values reaches the rows that see its token, in its place alone."""
    s = Setup("e4m3", [400, 200], [150, 200], block=16, share=2, dim=64, heads=2)
    s.append()
    clean, clean_lse = s.attend(window)
    marks = [(0, 260, 0, 3), (0, 399, 1, 63), (0, 120, 1, 9), (1, 0, 0, 5), (1, 70, 1, 17),
             (1, 199, 0, 40)]
    view = s.cache.v.view(torch.uint8)
    want = torch.zeros(clean.shape, dtype=torch.bool)
    for seq, pos, head, d in marks:
        view[s.table[seq, pos // 16], head, pos % 16, d] = 0xFF if d % 2 else 0x7F
        first, n, row = ((250, 150, 0), (0, 200, 150))[seq]
        for i in range(n):
            at = first + i
            if pos <= at and (window == 0 or at - pos < window):
                want[row + i, 2 * head:2 * head + 2, d] = True
    out, lse = s.attend(window)
    assert torch.equal(torch.isnan(out).cpu(), want)
    assert torch.equal(out[~want.cuda()], clean[~want.cuda()]) and torch.equal(lse, clean_lse)


def test_rows_is_the_choice_for_many(rows_kernel):
    """Either kernel, and the choice between them, within the bounds on the same rows."""
    s = Setup("int8", [500, 90], [40, 90], block=32, share=4, dim=128)
    s.append()
    outs = []
    for variant in (0, 1, 2):
        rows_kernel.set_option("attention_variant", variant)
        out, lse = s.attend()
        s.check_attention(out, lse)
        outs.append(out)
    assert torch.equal(outs[0], outs[2]) and not torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("fresh,share", [(45, 1), (61, 3), (130, 1), (7, 5)])
def test_rows_nan_values_where_rows_end_inside_a_warp(dim, fresh, share):
    """The last warp of a unit has rows in some of its lanes only, and each of them passes
    over another number of the tokens that are mended: again and again the same."""
    s = Setup("e4m3", [400], [fresh], block=16, share=share, dim=dim, heads=2)
    s.append()
    clean, clean_lse = s.attend()
    want = torch.zeros(clean.shape, dtype=torch.bool)
    view, first = s.cache.v.view(torch.uint8), 400 - fresh
    for i, back in enumerate(range(0, fresh, 3)):
        head, d = i % 2, (7 * i) % dim
        view[s.table[0, (399 - back) // 16], head, (399 - back) % 16, d] = 0x7F
        want[399 - back - first:, share * head:share * (head + 1), d] = True
    for _ in range(30):
        out, lse = s.attend(out=torch.full_like(clean, 3.0))
        assert torch.equal(torch.isnan(out).cpu(), want)
        assert torch.equal(out[~want.cuda()], clean[~want.cuda()]) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("tiny", [-16, -30, -60])
def test_rows_zeros_outweigh_small_values(store, tiny):
    few.test_attention_zeros_outweigh_small_values(store, tiny)


@pytest.mark.parametrize("store", STORES)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-6])
def test_rows_scales_of_any_sign(store, scale):
    few.test_attention_scales_of_any_sign(store, scale)


def test_rows_threads_with_a_stream_each():
    few.test_threads_with_a_stream_each()
