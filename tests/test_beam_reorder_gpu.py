"""Beam reordering against the definition, entry by entry.  Bytes have to be equal, those that no fork touches included."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import wuda_b200 as wuda
from step_oracle import beam_slots

pytestmark = pytest.mark.gpu
# (entries per page, segments, tokens per entry, ring, extra bytes of a page)
FP8_INDEX, FP4_INDEX = (64, (128, 4), 4, 0, 0), (64, (64, 4), 4, 0, 0)
RECORDS, WINDOW = (64, (576, 8), 4, 0, 64), (256, (576, 8), 1, 128, 512)
ODD = (12, (20, 4), 3, 0, 32)
ONE = (4, (4,), 1, 0, 0)
RING = (3, (16, 12), 2, 7, 12)


def world(rng, groups, width, pools, states, length, shared, spare=3):
    """length / shared: token counts of each group."""
    capacity = groups * width + spare
    w = dict(slots=rng.permutation(capacity)[:groups * width].astype(np.int32).reshape(groups, width),
             lengths=rng.integers(0, 50, capacity).astype(np.int32), shared=np.zeros(capacity, np.int32), capacity=capacity)
    for g in range(groups):
        w["lengths"][w["slots"][g]], w["shared"][w["slots"][g]] = length[g], shared[g]
    w["states"] = [rng.integers(0, 256, (capacity, n), dtype=np.uint8) for n in states]
    w["pools"] = []
    for epb, segments, tpe, ring, extra in pools:
        entries = [min(n // tpe, ring) if ring else n // tpe for n in w["lengths"]]
        pages = max(1, max(-(-e // epb) for e in entries))
        table = rng.permutation(capacity * pages).astype(np.int32).reshape(capacity, pages)
        for g in range(groups):       # a group's shared pages are the same ones
            common = 0 if ring else shared[g] // tpe // epb
            table[w["slots"][g], :common] = table[w["slots"][g, 0], :common]
        stride = -(-(epb * sum(segments) + extra) // 16) * 16
        w["pools"].append((rng.integers(0, 256, (capacity * pages, stride), dtype=np.uint8), table, epb, segments, tpe, ring))
    return w


def plan_of(w, status=None, shared=True):
    d = lambda a: torch.from_numpy(a.copy()).cuda()
    pools = [wuda.PagedState(d(data), d(table), epb, segments, tpe, ring) for data, table, epb, segments, tpe, ring in w["pools"]]
    return wuda.BeamReorder(d(w["lengths"]), w["slots"].shape[1], shared_lengths=d(w["shared"]) if shared else None,
                            states=[d(s) for s in w["states"]], pools=pools, status_word=status)


def want_of(w, parents):
    out, moves = beam_slots(parents, w["slots"], w["capacity"])
    states, pools = [s.copy() for s in w["states"]], [p[0].copy() for p in w["pools"]]
    for g, j, src, dst in moves:
        length = w["lengths"][src]
        if length < 0 or w["lengths"][dst] != length or w["shared"][dst] != w["shared"][src] or any(
                -(-(min(length // tpe, ring) if ring else length // tpe) // epb) > table.shape[1] for _, table, epb, _, tpe, ring in w["pools"]):
            out[g, j] = -1
            continue
        for new, old in zip(states, w["states"]):
            new[dst] = old[src]
        for new, (old, table, epb, segments, tpe, ring) in zip(pools, w["pools"]):
            entries = min(length // tpe, ring) if ring else length // tpe
            for e in range(0 if ring else w["shared"][src] // tpe // epb * epb, entries):
                a, b, offset = table[src, e // epb], table[dst, e // epb], 0
                if not (0 <= a < len(old) and 0 <= b < len(old)):
                    continue
                for size in segments:
                    at = offset + e % epb * size
                    new[b, at:at + size] = old[a, at:at + size]
                    offset += epb * size
    return out, states, pools


def run(plan, w, parents):
    out = torch.full((len(parents), parents.shape[1]), -9, dtype=torch.int32, device="cuda")
    plan.run(torch.from_numpy(parents).cuda(), torch.from_numpy(w["slots"]).cuda(), out)
    return out


def check(plan, w, parents, out):
    torch.cuda.synchronize()
    want, states, pools = want_of(w, parents)
    assert np.array_equal(out.cpu().numpy(), want)
    for got, ref in zip(plan.states, states):
        assert np.array_equal(got.cpu().numpy(), ref)
    for i, (got, ref) in enumerate(zip(plan.pools, pools)):
        assert np.array_equal(got.data.cpu().numpy(), ref), i


LAYER = [FP8_INDEX, RECORDS, WINDOW]


@pytest.mark.parametrize("groups, width, pools, states, longest", [
    (1, 1, LAYER, [64], 300), (1, 2, LAYER, [65536, 16384, 2052], 40), (1, 4, LAYER, [65536, 16384, 36], 700), (3, 5, [FP4_INDEX, RECORDS, WINDOW], [4, 65540], 1100),
    (2, 32, [FP8_INDEX, ODD], [20], 900), (7, 3, [ODD, ONE, RING, WINDOW], [16388, 12, 48, 4, 8, 16, 32, 64], 400), (2, 8, [], [100], 10),
    (4, 4, [RECORDS], [], 257), (40, 31, [ONE], [8], 30)])
@pytest.mark.parametrize("seed", [0, 1])
def test_forks(groups, width, pools, states, longest, seed):
    rng = np.random.default_rng(seed * 100 + groups * width)
    length = rng.integers(0, longest + 1, groups)
    length[0] = longest
    shared = (length * rng.random(groups) * rng.integers(0, 2, groups)).astype(int)
    if groups > 2:
        shared[1] = length[1]                # nothing generated yet
    w = world(rng, groups, width, pools, states, length, shared)
    parents = rng.integers(0, width, (groups, width)).astype(np.int32)
    parents[-1] = np.arange(width)[::-1] if seed else 0       # everyone goes on, or all continue one beam
    status = wuda.device_status_word()
    plan = plan_of(w, status, shared=True)
    check(plan, w, parents, run(plan, w, parents))
    assert int(status) == 0
    if not shared.any():
        plan = plan_of(w, status, shared=False)
        check(plan, w, parents, run(plan, w, parents))


def test_lengths_around_pages_and_rings():
    """Every length around the borders of an entry, a page and the window, nothing shared or all but the last tokens."""
    rng = np.random.default_rng(1)
    lengths = [0, 1, 3, 4, 7, 8, 127, 128, 129, 252, 255, 256, 257, 259, 260, 511, 512, 516]
    for back in (0, 1, 5, 260, 10 ** 6):
        shared = [max(0, n - back) for n in lengths]
        w = world(rng, len(lengths), 3, LAYER + [RING], [40], lengths, shared)
        parents = rng.integers(0, 3, (len(lengths), 3)).astype(np.int32)
        plan = plan_of(w)
        check(plan, w, parents, run(plan, w, parents))


def test_beams_without_parents_and_padded_groups():
    rng = np.random.default_rng(2)
    w = world(rng, 5, 4, LAYER, [16], [300] * 5, [100] * 5)
    w["slots"][3] = -1                                   # a padded group
    w["slots"][4, 2] = -1
    parents = np.array([[2, -1, -1, 2], [-1, -1, -1, -1], [1, 1, 1, -1], [0, 1, 0, -1], [0, 2, 1, 1]], np.int32)
    status = wuda.device_status_word()
    plan = plan_of(w, status)
    check(plan, w, parents, run(plan, w, parents))
    assert int(status) == 0


@pytest.mark.parametrize("code, change", [
    (161, lambda w, p: w["slots"].__setitem__((1, 2), 1000)), (161, lambda w, p: w["slots"].__setitem__((1, 2), w["slots"][0, 1])),
    (161, lambda w, p: w["slots"].__setitem__((1, 2), w["slots"][1, 0])), (161, lambda w, p: w["slots"].__setitem__((0, 0), -2 ** 31)),
    (164, lambda w, p: p.__setitem__((0, 1), 4)), (164, lambda w, p: p.__setitem__((2, 3), -2)),
    (163, lambda w, p: w["lengths"].__setitem__(w["slots"][0, 3], 299)), (163, lambda w, p: w["shared"].__setitem__(w["slots"][0, 3], 0)),
    (163, lambda w, p: w["lengths"].__setitem__(w["slots"][0], -1)), (163, lambda w, p: w["lengths"].__setitem__(w["slots"][0], 5000)),
    (163, lambda w, p: w["lengths"].__setitem__(w["slots"][0], 2 ** 31 - 1)),
    (110, lambda w, p: w["pools"][0][1].__setitem__((w["slots"][0, 3], 1), 10 ** 6)), (110, lambda w, p: w["pools"][1][1].__setitem__((w["slots"][0, 0], 1), -1))])
def test_what_is_reported_and_left_out(code, change):
    rng = np.random.default_rng(4)
    w = world(rng, 3, 4, LAYER, [32], [300] * 3, [64] * 3)
    parents = np.array([[0, 1, 0, 2], [1, 1, 2, 2], [3, 0, 0, 0]], np.int32)
    change(w, parents)
    status = wuda.device_status_word()
    plan = plan_of(w, status)
    check(plan, w, parents, run(plan, w, parents))
    assert int(status) == code


def test_captured_on_another_stream():
    rng = np.random.default_rng(6)
    w = world(rng, 4, 8, LAYER, [65536, 40], [500, 260, 90, 3], [200, 256, 0, 0])
    parents = [rng.integers(0, 8, (4, 8)).astype(np.int32) for _ in range(4)]
    plan = plan_of(w)
    dev, slots = torch.from_numpy(parents[0]).cuda(), torch.from_numpy(w["slots"]).cuda()
    out = torch.empty_like(slots)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        plan.run(dev, slots, out)
        slots.copy_(out)
    for p in parents:                        # each step starts from what the last one left
        with torch.cuda.stream(side):
            dev.copy_(torch.from_numpy(p))
            graph.replay()
        side.synchronize()
        check(plan, w, p, slots)
        want, states, pools = want_of(w, p)
        w["slots"], w["states"] = want, states
        w["pools"] = [(data, *old[1:]) for data, old in zip(pools, w["pools"])]


def test_refused_arguments():
    rng = np.random.default_rng(7)
    w = world(rng, 2, 4, LAYER, [32], [300] * 2, [64] * 2)
    plan = plan_of(w)
    parents = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    slots, out = torch.from_numpy(w["slots"]).cuda(), torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    for args in ((parents.long(), slots, out), (parents, slots, slots), (parents, slots, parents), (parents, slots[:1], out), (parents, slots, out.cpu()),
                 (parents[:, :3], slots, out), (parents.t(), slots, out)):
        with pytest.raises(wuda.WudaError):
            plan.run(*args)
    plan.run(parents[:0], slots[:0], out[:0])
    lengths = plan.lengths
    pool = plan.pools[0]
    made = lambda **c: wuda.BeamReorder(c.pop("lengths", lengths), c.pop("width", 4), **c)
    paged = lambda **c: [wuda.PagedState(**dict(dict(data=pool.data, table=pool.table, entries_per_block=64, segments=(128, 4), tokens_per_entry=4), **c))]
    made(pools=paged())
    for change in (dict(width=0), dict(width=33), dict(lengths=lengths.long()), dict(lengths=lengths.cpu()), dict(shared_lengths=lengths[:3]),
                   dict(states=[torch.zeros(5, 4, device="cuda")]), dict(states=[torch.zeros(lengths.numel(), 3, dtype=torch.uint8, device="cuda")]),
                   dict(states=[plan.states[0]] * 9), dict(states=[plan.states[0].cpu()]), dict(pools=paged() * 5),
                   dict(pools=paged(segments=(130, 4))), dict(pools=paged(segments=(0, 4))), dict(pools=paged(segments=(128, 4, 4))),
                   dict(pools=paged(entries_per_block=65)), dict(pools=paged(entries_per_block=0)), dict(pools=paged(tokens_per_entry=0)),
                   dict(pools=paged(ring=-1)), dict(pools=paged(table=pool.table[:2])), dict(pools=paged(table=pool.table.long())),
                   dict(pools=paged(data=pool.data.view(torch.int8))), dict(pools=paged(data=pool.data[:, 4:])),
                   dict(pools=paged(data=pool.data.view(-1)[:8444 * 4].view(4, 8444))), dict(status_word=lengths.long())):
        with pytest.raises(wuda.WudaError):
            made(**change)


def test_numbers_are_not_cut():
    w = world(np.random.default_rng(7), 2, 4, LAYER, [32], [300] * 2, [64] * 2)
    lengths, pool = plan_of(w).lengths, plan_of(w).pools[0]
    paged = lambda **c: [wuda.PagedState(**dict(dict(data=pool.data, table=pool.table, entries_per_block=64, segments=(128, 4), tokens_per_entry=4), **c))]
    wuda.BeamReorder(lengths, 4, pools=paged())
    for width, pools in (((1 << 32) + 4, paged()), (4, paged(entries_per_block=(1 << 32) + 64)), (4, paged(segments=((1 << 32) + 128, 4))),
                         (4, paged(tokens_per_entry=(1 << 32) + 4)), (4, paged(ring=1 << 32))):
        with pytest.raises(wuda.WudaError):
            wuda.BeamReorder(lengths, width, pools=pools)


WHERE_SHARED_MEMORY_PASSES_48_KB = """
import torch
import wuda_b200 as wuda

# (8 x beams + capacity) x 4 bytes for the plan beside what a CTA has in any case: the first call of each size in a process that has
# made no larger one
for groups, width, capacity in ((1, 4, 11700), (1, 4, 11836), (1, 4, 11837), (128, 8, 3690), (128, 8, 3800), (1, 4, 11900), (100, 10, 4032),
                                (1, 4, 12000), (1, 4, 12001), (128, 8, 3841), (128, 32, 16384)):
    beams = groups * width
    state = torch.arange(capacity * 3, dtype=torch.int32, device="cuda").view(capacity, 3)
    want = state.clone()
    lengths = torch.full((capacity,), 5, dtype=torch.int32, device="cuda")
    slots = torch.randperm(capacity, device="cuda")[:beams].int().view(groups, width)
    parents = torch.zeros(groups, width, dtype=torch.int32, device="cuda")
    out = torch.empty_like(slots)
    wuda.BeamReorder(lengths, width, states=[state]).run(parents, slots, out)
    want[slots.view(-1).long()] = want[slots[:, :1].expand(groups, width).reshape(-1).long()]
    assert torch.equal(out, slots) and torch.equal(state, want), (groups, width, capacity)
print("all sizes")
"""


def test_sizes_around_the_shared_memory_of_a_plain_launch():
    """In a process of its own: a larger call before would have asked for more shared memory for good."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", WHERE_SHARED_MEMORY_PASSES_48_KB], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "all sizes" in run.stdout, run.stderr[-2000:]
