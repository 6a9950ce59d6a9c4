"""Beam selection against a 64-bit log-softmax and a stable sort.

Tolerance of a score v: its rounding to fp32, 2^-24 |v|, and the error of log sum exp.  A term exp(x - r) has the roundings of x - r
and of its product with log2 e and that constant's (each 2^-24 of up to 104, where exp ends in fp32) and 2^-22 of the
exponential itself; a thread adds at most vocab / 256 + 32 terms one after the other.  So the sum, all of whose terms are positive, is off
by at most (3 * 104 + 4 + vocab / 256 + 32) 2^-24 of itself, and its logarithm by as much.  The lists must be equal wherever the
values are further apart than that on both sides; where beams or tokens tie exactly, always."""
import ctypes

import numpy as np
import pytest
import torch

import wuda_b200 as wuda
from step_oracle import beam_select
from wuda_b200._lib import BeamSelectArgs, lib

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def likely(groups, width, vocab, kind, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(groups, width, vocab, generator=g) * spread
    return x.to(TYPES[kind]).cuda(), (-torch.rand(groups, width, generator=g) * 9 - 5).cuda()


def check(got, logits, scores, k, finished=None, eos=None, exact=False):
    torch.cuda.synchronize()
    values, parents, tokens, done = beam_select(logits.double().cpu().numpy(), scores.cpu().numpy(), k,
                                                None if finished is None else finished.cpu().numpy(), -5 if eos is None else eos)
    vocab = logits.size(2)
    s, p, t, d = (x.cpu().numpy() for x in got)
    assert s.dtype == np.float32 and p.dtype == t.dtype == np.int32 and d.dtype == bool
    there = np.isfinite(values)
    assert np.array_equal(s == -np.inf, ~there)
    tol = np.where(there, 2.0 ** -24 * np.abs(np.where(there, values, 0)) + (348 + vocab / 256) * 2.0 ** -24, 0)
    assert np.all(np.abs(np.where(there, s, 0).astype(np.float64) - np.where(there, values, 0)) <= tol)
    clear = np.ones_like(there)          # further than the tolerance from both neighbours (padding is)
    with np.errstate(invalid="ignore"):
        gap = np.where(there[:, 1:], values[:, :-1] - values[:, 1:], np.inf) if k > 1 else np.zeros((len(values), 0))
    for g in range(len(values)):
        for j in range(k - 1):
            if there[g, j + 1] and 0 < gap[g, j] <= 2 * (tol[g, j] + tol[g, j + 1]) and not exact:
                clear[g, j] = clear[g, j + 1] = False
    if not exact and k:
        clear[:, -1] &= ~there[:, -1] | (vocab * logits.size(1) == k)      # (its lower neighbour is not in the list)
    assert clear.mean() > 0.5 or k <= 2
    for a, b, name in ((p, parents, "parents"), (t, tokens, "tokens"), (d, done, "finished")):
        assert np.array_equal(np.where(clear, a, 0), np.where(clear, b, 0)), name


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("groups, width, vocab, k", [
    (1, 1, 1, 1), (1, 1, 2, 3), (2, 3, 7, 30), (3, 2, 255, 4), (1, 4, 256, 8), (2, 5, 1000, 10), (1, 8, 2047, 16), (1, 1, 2048, 64),
    (4, 3, 2049, 6), (1, 4, 4096, 1), (2, 4, 4097, 8), (1, 32, 8192, 64), (3, 2, 8193, 4), (1, 4, 32000, 8), (2, 3, 50001, 6),
    (1, 2, 131072, 64), (1, 1, 262147, 5), (40, 4, 3001, 4), (256, 1, 513, 2)])
def test_against_64_bits(groups, width, vocab, k, kind):
    logits, scores = likely(groups, width, vocab, kind, seed=vocab + k)
    check(wuda.beam_select(logits, scores, k), logits, scores, k)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad", [0, 1, 3, 8])
def test_rows_that_start_anywhere_and_ties(kind, pad):
    """Beams with the same logits and scores tie exactly whatever their rows' alignment, and so do tokens with the same logit: lower
    beam first, then lower token."""
    vocab, width = 20003, 5
    held = torch.zeros(2, width, vocab + pad, dtype=TYPES[kind], device="cuda")
    logits = held[:, :, :vocab]
    one, _ = likely(2, 1, vocab, kind, seed=4)
    logits.copy_(torch.round(one * 4) / 4)         # many equal logits
    scores = torch.full((2, width), -3.25, device="cuda")
    got = wuda.beam_select(logits, scores, 23)
    check(got, logits, scores, 23, exact=True)
    assert len(set(got[0][0].tolist())) < 23       # (there are ties in the list)
    # on a storage that starts off the grid, too
    flat = torch.zeros(2 * width * vocab + 3, dtype=TYPES[kind], device="cuda")
    moved = flat[3:].view(2, width, vocab)
    moved.copy_(logits)
    for a, b in zip(got, wuda.beam_select(moved, scores, 23)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [100, 5000, 40000])
def test_rows_of_one_value_and_sorted_rows(kind, vocab):
    """All logits equal (zero, the type's lowest, its largest), ascending and descending ones: what fills and refills every list on
    the way."""
    lowest, largest = torch.finfo(TYPES[kind]).min, torch.finfo(TYPES[kind]).max
    rows = [torch.zeros(vocab), torch.full((vocab,), lowest), torch.full((vocab,), largest),
            torch.linspace(-30, 30, vocab), torch.linspace(30, -30, vocab)]
    for row in rows:
        logits = row.to(TYPES[kind]).cuda().view(1, 1, vocab).expand(2, 3, vocab)       # (stride 0)
        scores = torch.tensor([[-1.0, -1.0, -1.5], [-2.0, -1.0, -1.0]], device="cuda")
        k = 40
        check(wuda.beam_select(logits, scores, k), logits, scores, k, exact=True)


@pytest.mark.parametrize("kind", list(TYPES))
def test_masked_tokens(kind):
    """-inf, NaN, +inf and the type's lowest value in most places, rows with nothing left, one token left, all but the last ones
    masked; the rest is as if the masked tokens were not there."""
    vocab, width, k = 9001, 6, 7
    logits, scores = likely(3, width, vocab, kind, seed=8)
    nan, inf, lowest = float("nan"), float("inf"), torch.finfo(TYPES[kind]).min
    logits[0, 0] = -inf
    logits[0, 1] = nan
    logits[0, 2, ::2], logits[0, 2, 1::3] = -inf, inf
    logits[0, 3] = -inf
    logits[0, 3, 8999] = 1.5
    logits[0, 4, :8990] = lowest
    logits[0, 5, 5:] = nan
    logits[1] = -inf
    logits[2, :, 100:] = -inf
    logits[2, 1], logits[2, 2, :50] = nan, inf
    got = wuda.beam_select(logits, scores, k)
    check(got, logits, scores, k)
    assert got[1][1].tolist() == [-1] * k and got[2][1].tolist() == [-1] * k
    only = logits[:1, 3:4].contiguous()
    got = wuda.beam_select(only, scores[:1, 3:4].contiguous(), 3)
    assert got[2].tolist() == [[8999, -1, -1]] and float(got[0][0, 0]) == float(scores[0, 3])


def test_large_and_small_magnitudes():
    vocab = 5003
    logits, scores = likely(1, 4, vocab, "fp32", seed=3)
    logits[0, 0] *= 1e37
    logits[0, 1] = logits[0, 1] * 1e-30
    logits[0, 2] += 3e4
    logits[0, 3, 17] = 3.4e38
    got = wuda.beam_select(logits, scores, 12)
    assert got[1].tolist()[0].count(3) == 1
    check(got, logits, scores, 12, exact=False)


@pytest.mark.parametrize("kind", list(TYPES))
def test_dead_and_finished_beams(kind):
    vocab, width, k, eos = 3001, 6, 12, 2
    logits, scores = likely(4, width, vocab, kind, seed=6)
    scores[0, 1:] = float("-inf")                       # a prompt's first step: one beam
    scores[1, 2], scores[1, 3] = float("nan"), float("inf")
    scores[2] = float("-inf")                           # nothing is left
    finished = torch.zeros(4, width, dtype=torch.bool, device="cuda")
    finished[1, 0] = finished[1, 2] = finished[3, :5] = True
    logits[1, 0] = float("nan")                         # (not read)
    scores[3, 0] = scores[3, 1]                         # finished beams tie: lower beam first
    logits[3, 5, 2] += 40                               # and the last beam's best token finishes it
    got = wuda.beam_select(logits, scores, k, finished=finished, eos_token=eos)
    check(got, logits, scores, k, finished, eos)
    assert got[3][3].tolist()[:1] == [True]
    got = wuda.beam_select(logits, scores, k, eos_token=eos)      # no beam is finished yet
    check(got, logits, scores, k, None, eos)
    all_done = torch.ones(4, width, dtype=torch.bool, device="cuda")
    got = wuda.beam_select(logits, scores, k, finished=all_done, eos_token=eos)
    check(got, logits, scores, k, all_done, eos)
    # fewer than k continuations
    few = logits[:, :, :1].contiguous()
    check(wuda.beam_select(few, scores, k), few, scores, k)


def test_default_k_strided_beams_and_the_same_again():
    logits, scores = likely(3, 8, 4099, "bf16", seed=1)
    got = wuda.beam_select(logits, scores)
    assert got[0].shape == (3, 8)
    turned = logits.transpose(0, 1).contiguous().transpose(0, 1)
    for _ in range(20):
        for a, b in zip(got, wuda.beam_select(turned, scores)):
            assert torch.equal(a, b)
    every_other = logits[:, ::2]
    check(wuda.beam_select(every_other, scores[:, ::2].contiguous(), 5), every_other, scores[:, ::2], 5)


def test_captured_graphs_and_streams():
    """Two graphs replayed by turns and at the same time on streams of their own, eager calls of other sizes between them."""
    cases = [likely(2, 4, 30011, "bf16", 5), likely(5, 3, 9973, "fp16", 6)]
    held = [(x.clone(), s.clone()) for x, s in cases]
    graphs = []
    for x, s in held:
        wuda.beam_select(x, s, 6)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            out = wuda.beam_select(x, s, 6)
        graphs.append((graph, out, stream))
    for round_ in range(6):
        for (x, s), (a, b) in zip(held, cases):
            x.copy_(a.roll(round_, 2))
            s.copy_(b.roll(round_, 1))
        torch.cuda.synchronize()
        for graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        check(wuda.beam_select(cases[0][0], cases[0][1], 9), *cases[0], 9)
        torch.cuda.synchronize()
        for (x, s), (_, out, _) in zip(held, graphs):
            check(out, x, s, 6)


def test_refused_arguments():
    logits, scores = likely(2, 3, 50, "fp32", seed=0)
    done = torch.zeros(2, 3, dtype=torch.bool, device="cuda")
    for bad in (lambda: wuda.beam_select(logits.double(), scores), lambda: wuda.beam_select(logits.cpu(), scores.cpu()),
                lambda: wuda.beam_select(logits[0], scores), lambda: wuda.beam_select(logits.transpose(1, 2), scores),
                lambda: wuda.beam_select(logits, scores.double()), lambda: wuda.beam_select(logits, scores[:, :2]),
                lambda: wuda.beam_select(logits, scores, 0), lambda: wuda.beam_select(logits, scores, 65),
                lambda: wuda.beam_select(logits, scores, finished=done), lambda: wuda.beam_select(logits, scores, finished=done.int(), eos_token=1),
                lambda: wuda.beam_select(logits, scores, eos_token=50), lambda: wuda.beam_select(logits, scores, eos_token=-2),
                lambda: wuda.beam_select(logits, scores, finished=done[:1], eos_token=1),
                lambda: wuda.beam_select(logits.expand(2, 3, 50)[:, :1].expand(2, 33, 50), torch.zeros(2, 33, device="cuda")),
                lambda: wuda.beam_select(logits[:1].expand(257, 3, 50), torch.zeros(257, 3, device="cuda"))):
        with pytest.raises(wuda.WudaError):
            bad()
    empty = wuda.beam_select(logits[:0], scores[:0], 4)
    assert [tuple(t.shape) for t in empty] == [(0, 4)] * 4


def test_numbers_are_not_cut():
    logits, scores = likely(2, 3, 50, "fp32", seed=0)
    for bad in (dict(k=(1 << 32) + 4), dict(k=-(1 << 32) + 4), dict(eos_token=(1 << 32) + 4)):
        with pytest.raises(wuda.WudaError):
            wuda.beam_select(logits, scores, **bad)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("vocab", [50, 9001, 70001])
def test_zeros_of_both_signs_are_equal(kind, vocab):
    """The best logits are zeros, signs by turns: the lower token first; scores of both signs: the lower beam."""
    logits = torch.full((2, 3, vocab), -4.0, dtype=TYPES[kind], device="cuda")
    logits[:, :, 5::3] = -0.0
    logits[:, :, 7::6] = 0.0
    logits[1, :, 40:] = logits[1, :, 40:].flip(-1)
    scores = torch.tensor([[-0.0, 0.0, -0.0], [-0.0, 0.0, 0.0]], device="cuda")
    for k in (1, 11, 40):
        check(wuda.beam_select(logits, scores, k), logits, scores, k, exact=True)
    ended = torch.ones(2, 3, dtype=torch.bool, device="cuda")
    check(wuda.beam_select(logits, scores, 3, finished=ended, eos_token=4), logits, scores, 3, ended, 4, exact=True)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("groups, width, vocab, k", [(5, 32, 9001, 64), (9, 31, 20011, 62), (6, 32, 33000, 32), (13, 31, 8300, 33), (14, 30, 8300, 34)])
def test_wide_groups_with_long_lists(groups, width, vocab, k, kind):
    """One or two chunks to a row because the merge holds no more lists, on both sides of the rule for the size of the CTAs."""
    logits, scores = likely(groups, width, vocab, kind, seed=groups * k)
    check(wuda.beam_select(logits, scores, k), logits, scores, k)


COUNTS = (383, 385, 1023, 1024, 1025, 1200, 1366, 1536, 1537, 2050)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("pad", [0, 3])
@pytest.mark.parametrize("groups, vocab", [(10, 131072), (10, 8192), (2, 131072)])
def test_as_many_candidates_as_a_list_holds_and_more(groups, vocab, pad, kind):
    """One group each with so many equal maxima in one chunk, and with so many tokens in front that are not masked: what is ranked as
    it is, trimmed, and selected exactly, in CTAs of 512 threads (10 rows of 131072) and of 128."""
    for first in range(0, len(COUNTS), groups):
        counts = COUNTS[first:first + groups]
        held = torch.full((groups, 1, vocab + pad), -3.0, dtype=TYPES[kind], device="cuda")
        logits = held[:, :, :vocab]
        scores = torch.full((groups, 1), -2.5, device="cuda")
        for g, n in enumerate(counts):       # spread over as many threads of a tile as there are
            logits[g, 0, :min(vocab, 8192) // n * n:min(vocab, 8192) // n] = 2.0
        for k in (4, 64):
            got = wuda.beam_select(logits, scores, k)
            check(got, logits, scores, k, exact=True)
            for a, b in zip(got, wuda.beam_select(logits, scores, k)):
                assert torch.equal(a, b)
        logits.copy_(torch.round(likely(groups, 1, vocab, kind, seed=first)[0] * 4) / 4)
        for g, n in enumerate(counts):
            logits[g, 0, n:] = float("-inf")
        for k in (4, 64):
            check(wuda.beam_select(logits, scores, k), logits, scores, k, exact=True)


@pytest.mark.parametrize("kind", list(TYPES))
def test_full_lists_of_several_beams(kind):
    """Every sixth of the first tokens at one maximum, in all beams of all groups; few tokens of many allowed, in wide groups."""
    logits = torch.full((16, 4, 131072), -3.0, dtype=TYPES[kind], device="cuda")
    logits[:, :, 0:8191:6] = 2.0
    scores = torch.full((16, 4), -1.25, device="cuda")
    check(wuda.beam_select(logits, scores, 4), logits, scores, 4, exact=True)
    for allowed in (1100, 1500):
        logits, scores = likely(1, 32, 131072, kind, seed=allowed)
        logits[:, :, allowed:] = float("-inf")
        check(wuda.beam_select(logits, scores, 64), logits, scores, 64)


@pytest.mark.parametrize("kind", list(TYPES))
def test_rows_of_one_value_and_sorted_rows_in_large_blocks(kind):
    vocab = 131072
    up = torch.linspace(-30, 30, vocab)
    rows = torch.stack([torch.zeros(vocab), torch.full((vocab,), torch.finfo(TYPES[kind]).min), torch.full((vocab,), torch.finfo(TYPES[kind]).max),
                        up, up.flip(0), up.abs(), -up.abs()])
    logits = rows.to(TYPES[kind]).cuda().view(7, 1, vocab)
    scores = torch.full((7, 1), -0.75, device="cuda")
    for k in (5, 40):
        check(wuda.beam_select(logits, scores, k), logits, scores, k, exact=True)


def test_scores_and_finished_in_place():
    """Through the C ABI, with k = width: the beams' scores and flags are those after the selection."""
    logits, scores = likely(5, 6, 20011, "bf16", seed=12)
    finished = torch.zeros(5, 6, dtype=torch.bool, device="cuda")
    finished[1, 2] = finished[4] = True
    want = wuda.beam_select(logits, scores, finished=finished, eos_token=7)
    parents, tokens = torch.empty(5, 6, dtype=torch.int32, device="cuda"), torch.empty(5, 6, dtype=torch.int32, device="cuda")
    nbytes = lib.wuda_beam_select_workspace_bytes(5, 6, 20011, 6, 0)
    workspace, counters = torch.empty(nbytes, dtype=torch.uint8, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    a = BeamSelectArgs(logits.data_ptr(), logits.stride(0), logits.stride(1), scores.data_ptr(), finished.data_ptr(), scores.data_ptr(),
                       parents.data_ptr(), tokens.data_ptr(), finished.data_ptr(), workspace.data_ptr(), nbytes, counters.data_ptr(),
                       5, 6, 20011, 6, 7, 0)
    assert lib.wuda_beam_select(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    for got, ref in zip((scores, parents, tokens, finished), want):
        assert torch.equal(got, ref)
