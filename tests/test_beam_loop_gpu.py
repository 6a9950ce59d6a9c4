"""The operators together, as a server uses them around a layer: the next beams from the logits, their caches, the next step."""
import numpy as np
import pytest
import torch

import wuda_b200 as wuda
from wuda_b200.layer_setup import build_random_layer
from wuda_b200.step_tables import CacheTables

pytestmark = pytest.mark.gpu
SMALL = dict(topk=512, experts=32, inter=512, moe_topk=4)
HIDDEN = 7168


def pools_of(cache):
    return [cache.swa_pool, cache.cmp_pool, cache.idx_pool, cache.main_state, cache.idx_state]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("fp4", [False, True])
def test_steps_prepared_on_the_device_give_the_host_prepared_bits(native, fp4):
    """Ten steps: prepared by the cache manager on the host; on the device step by step; and as ten replays of one graph that
    prepares its own step.  Outputs, pools, rings and page tables are the same, across a page border and a padded row."""
    runs = []
    for how in ("host", "device", "graph"):
        layer, slots, x = build_random_layer(5, 250, seed=23, native=native, indexer_fp4=fp4, **SMALL)
        cache, outs = layer.attn.cache, []
        if how == "host":
            slots = slots[:4]
            x = x[:4].contiguous()
        else:
            dev = torch.tensor(slots[:2] + [-1] + slots[2:4], dtype=torch.int32, device="cuda")
            x = x[[0, 1, 4, 2, 3]].contiguous()
            layer.device_tables()
            with pytest.raises(RuntimeError):
                layer.prepare(slots)
            if how == "graph":
                layer.capture(x, 5, slots=dev)
        for step in range(10):
            if how == "host":
                layer.prepare(slots)
                out = layer.launch(x, 4)
            elif how == "device":
                layer.prepare_on_device(dev)
                out = layer.launch(x, 5)[[0, 1, 3, 4]]
            else:
                out = layer.replay()[[0, 1, 3, 4]]
            outs.append(out.clone())
        torch.cuda.synchronize()
        layer.check_status()
        if how != "host":
            layer.device_tables().pull()
        runs.append((outs, [p.clone() for p in pools_of(cache)], [(cache.reqs[s]["pos"], cache.reqs[s]["cmp"], cache.reqs[s]["idx"]) for s in slots[:4]],
                     [cache._pools[n]._free for n in ("idx", "cmp")]))
        del layer
    for other in runs[1:]:
        assert other[2] == runs[0][2] and other[3] == runs[0][3]
        for a, b in zip(runs[0][0], other[0]):
            assert torch.equal(a, b)
        for a, b in zip(runs[0][1], other[1]):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_graphs_of_both_ways_of_preparing_live_side_by_side():
    """A graph captured before the layer had tables on the device replays the host's steps and, later, the device's: the same
    buffers.  One that prepares its own steps is refused while the cache manager has the state, and with too few slots."""
    layer, slots, x = build_random_layer(3, 250, seed=31, **SMALL)
    twin, twin_slots, _ = build_random_layer(3, 250, seed=31, **SMALL)
    layer.prepare(slots)
    graph = layer.capture(x, 3)
    outs = []

    def compare(out):
        twin.prepare(twin_slots)
        outs.append(out)
        assert torch.equal(out, twin.launch(x, 3))

    compare(layer.replay().clone())
    dev = torch.tensor(slots, dtype=torch.int32, device="cuda")
    tables = layer.device_tables()
    for _ in range(3):
        layer.prepare_on_device(dev)
        graph.replay()
        compare(layer._graph_out.clone())
    with pytest.raises(ValueError):
        layer.capture(x, 3, slots=dev[:2])
    layer.capture(x, 3, slots=dev)
    compare(layer.replay().clone())
    tables.pull()
    with pytest.raises(RuntimeError):
        layer.replay()
    layer.prepare(slots)
    graph.replay()
    compare(layer.out[:3].clone())
    tables.push()
    compare(layer.replay().clone())
    layer.check_status()
    assert len({tuple(o.view(torch.int16).flatten()[:4096].tolist()) for o in outs}) == len(outs)
    for a, b in zip(pools_of(layer.attn.cache), pools_of(twin.attn.cache)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


class Head:
    """A stand-in for what lies around the one layer: an embedding and an output projection over a small vocabulary."""

    def __init__(self, vocab):
        g = torch.Generator(device="cuda").manual_seed(77)
        self.embed = torch.randn(vocab, 4, HIDDEN, generator=g, device="cuda").bfloat16()
        self.out = (torch.randn(HIDDEN, vocab, generator=g, device="cuda") * 0.05).bfloat16()

    def logits(self, streams):
        return torch.mm(streams.float().mean(1).bfloat16(), self.out)


@pytest.mark.parametrize("captured", [False, True])
def test_a_beam_search_moves_whole_requests(captured):
    """Two prompts with four beams each over twelve steps, a layer with shared prompt pages and forks in place.  Beside it the same
    search in which every beam is a request of its own and a new beam gets a copy of everything its parent has (all pages, by
    torch): the same beams, tokens and scores, bit for bit."""
    groups, width, vocab, steps, context = 2, 4, 1009, 12, 251
    rows = groups * width
    head = Head(vocab)
    start = torch.randn(groups, width, vocab, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 3
    start_scores = torch.full((groups, width), float("-inf"), device="cuda")
    start_scores[:, 0] = 0

    def fresh():
        layer, slots, _ = build_random_layer(rows, context, seed=29, **SMALL)
        return layer, layer.attn.cache, slots

    # ---- shared pages, forks on the device
    layer, cache, slots = fresh()
    for s in slots[groups:]:
        cache.free_request(s)
    beams = [[s] + cache.fork_request(s, width - 1) for s in slots[:groups]]
    status = wuda.device_status_word()
    tables = layer.device_tables()
    history = torch.zeros(cache.capacity, steps, dtype=torch.int32, device="cuda")
    reorder = tables.beam_reorder(width, states=[history], status_word=status)
    now = torch.tensor(beams, dtype=torch.int32, device="cuda")
    then = torch.empty_like(now)
    logits, scores = start.bfloat16(), start_scores.clone()
    finished = torch.zeros(groups, width, dtype=torch.bool, device="cuda")
    x = torch.zeros(rows, 4, HIDDEN, dtype=torch.bfloat16, device="cuda")
    at = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        s, p, t, f = wuda.beam_select(logits, scores, finished=finished, eos_token=3)
        reorder.run(p, now, then)
        now.copy_(then), scores.copy_(s), finished.copy_(f)
        history[now.view(-1).long(), at] = t.view(-1)
        at.add_(1)
        x.copy_(head.embed[t.view(-1).long()])
        layer.prepare_on_device(now.view(-1))
        logits.copy_(head.logits(layer.launch(x, rows)).view(groups, width, vocab))

    if captured:
        held = [t.clone() for t in (now, scores, finished, logits, at, history, tables.lengths, tables.free_counts, *pools_of(cache))]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for t, was in zip((now, scores, finished, logits, at, history, tables.lengths, tables.free_counts, *pools_of(cache)), held):
            t.copy_(was)
    for _ in range(steps):
        graph.replay() if captured else step()
    torch.cuda.synchronize()
    layer.check_status()
    assert int(status) == 0
    got = scores.clone(), history[now.view(-1).long()].clone(), logits.clone(), finished.clone()
    order = now.view(-1).tolist()
    tables.pull()
    pos = {cache.reqs[s]["pos"] for s in order}
    for s in order:
        cache.free_request(s)
    for name in ("swa", "cmp", "idx"):        # every page comes back once
        assert sorted(cache._pools[name]._free) == list(range(cache._pools[name].data.size(0)))
    del layer, tables, reorder

    # ---- every beam a request of its own, copied whole
    layer, cache, slots = fresh()

    def copied(src, dst, pool_from, state_from):
        for i, state in enumerate((cache.main_state, cache.idx_state)):
            state[dst] = state_from[i][src]
        for i, name in enumerate(("swa", "cmp", "idx")):
            for a, b in zip(cache.reqs[src][name], cache.reqs[dst][name]):
                cache._pools[name].data[b] = pool_from[i][a]

    for g in range(groups):                   # the prompts of the other run, in every beam
        for w in range(width):
            src, dst = slots[g], slots[groups + g * (width - 1) + w - 1] if w else slots[g]
            if src != dst:
                copied(src, dst, [cache._pools[n].data.clone() for n in ("swa", "cmp", "idx")], [cache.main_state.clone(), cache.idx_state.clone()])
    mine = [[slots[g]] + slots[groups + g * (width - 1):groups + (g + 1) * (width - 1)] for g in range(groups)]
    tokens = [[[] for _ in range(width)] for _ in range(groups)]
    logits, scores, finished = start.bfloat16(), start_scores.clone(), torch.zeros_like(finished)
    for _ in range(steps):
        value = scores.double()[:, :, None] + torch.log_softmax(logits.double(), 2)
        ended = finished[:, :, None].expand(-1, -1, vocab)
        value = torch.where(ended, float("-inf"), value)
        value[:, :, 3] = torch.where(finished, scores.double(), value[:, :, 3])
        best, flat = value.view(groups, -1).sort(dim=1, descending=True, stable=True)
        p, t = flat[:, :width] // vocab, flat[:, :width] % vocab
        finished = torch.gather(finished, 1, p) | (t == 3)
        pools, states = [cache._pools[n].data.clone() for n in ("swa", "cmp", "idx")], [cache.main_state.clone(), cache.idx_state.clone()]
        for g in range(groups):
            for w in range(width):
                copied(mine[g][int(p[g, w])], mine[g][w], pools, states)
        tokens = [[tokens[g][int(p[g, w])] + [int(t[g, w])] for w in range(width)] for g in range(groups)]
        scores = wuda.beam_select(logits, scores, finished=ended[:, :, 0].contiguous(), eos_token=3)[0]
        assert torch.allclose(scores.double(), best[:, :width], rtol=1e-5, atol=1e-4)
        layer.prepare([s for g in mine for s in g])
        logits = head.logits(layer.launch(head.embed[t.reshape(-1)].contiguous(), rows)).view(groups, width, vocab)
    torch.cuda.synchronize()
    layer.check_status()
    assert pos == {cache.reqs[s]["pos"] for g in mine for s in g}
    assert got[1].view(groups, width, steps).tolist() == tokens
    assert torch.equal(got[0], scores) and torch.equal(got[2], logits) and torch.equal(got[3], finished)


@pytest.mark.parametrize("native", [True, False])
def test_a_capture_that_fails_leaves_the_requests_where_they_were(native):
    layer, slots, x = build_random_layer(3, 250, seed=37, native=native, **SMALL)
    dev = torch.tensor(slots, dtype=torch.int32, device="cuda")
    tables = layer.device_tables()
    before = tables.lengths.tolist(), tables.free_counts.tolist()
    for bad in (x[:, :2], x.float(), x.transpose(0, 1)):
        with pytest.raises((ValueError, RuntimeError)):
            layer.capture(bad, 3, slots=dev)
        assert (tables.lengths.tolist(), tables.free_counts.tolist()) == before
    layer.capture(x, 3, slots=dev)
    layer.replay()
    torch.cuda.synchronize()
    layer.check_status()
    assert tables.lengths.tolist() == [n + 1 for n in before[0]]


def test_a_graph_steps_only_from_the_state_of_its_own_tables():
    """Two tables over one cache: while the other ones have its state, a graph of the layer's would step from an old one."""
    layer, slots, x = build_random_layer(2, 250, seed=41, **SMALL)
    dev = torch.tensor(slots, dtype=torch.int32, device="cuda")
    tables = layer.device_tables()
    layer.capture(x, 2, slots=dev)
    layer.replay()
    tables.pull()
    other = CacheTables(layer.attn.cache, 2)
    other.step(dev)
    with pytest.raises(RuntimeError):
        layer.replay()
    other.pull()
    tables.push()
    layer.replay()
    torch.cuda.synchronize()
    layer.check_status()
    assert tables.lengths.tolist() == [252, 252]
