"""Step tables made on the device: against the definition row by row, and against the host's cache manager over steps with
requests that come, fork and go.  Everything is whole numbers and has to be equal."""
import numpy as np
import pytest
import torch

import wuda_b200 as wuda
from step_oracle import pages_of, step_tables
from wuda_b200.kv_cache import KVCacheManager
from wuda_b200.step_tables import CacheTables

pytestmark = pytest.mark.gpu
TOKEN = ("pos", "q_pos", "state_row", "idx_dst", "cmp_dst", "swa_dst")
ROW = ("n_compressed", "cmp_lengths", "swa_lengths", "swa_indices", "idx_block_table", "cmp_block_table")
GEOMETRY = dict(idx_epb=64, cmp_epb=64, swa_epb=256, ratio=4, ring=8, window=128, topk=512)


def state(rng, capacity, width, lengths, geometry, free):
    """Distinct pages for what the slots hold, and `free` more on each stack."""
    s = dict(lengths=np.asarray(lengths, np.int32), free_counts=np.array([free, free], np.int32))
    for name in ("idx", "cmp"):
        held = [min(pages_of(max(int(n), 0), geometry["ratio"], geometry[name + "_epb"]), width) for n in lengths]
        pages = rng.permutation(sum(held) + free + 3).astype(np.int32)
        table, at = np.zeros((capacity, width), np.int32), 0
        for slot, n in enumerate(held):
            table[slot, :n], at = pages[at:at + n], at + n
        s[name + "_table"], s[name + "_free"] = table, pages[at:]
    wp = -(-geometry["window"] // geometry["swa_epb"])
    s["swa_table"] = rng.permutation(capacity * wp).astype(np.int32).reshape(capacity, wp)
    return s


def plan_of(s, max_rows, max_tokens, geometry, in_place, status=None):
    d = {k: torch.from_numpy(v.copy()).cuda() for k, v in s.items()}
    more = {} if in_place else dict(lengths_out=torch.full_like(d["lengths"], -7), free_counts_out=torch.full_like(d["free_counts"], -7))
    plan = wuda.StepTables(d["lengths"], d["idx_table"], d["cmp_table"], d["swa_table"], d["idx_free"], d["cmp_free"], d["free_counts"],
                           max_rows=max_rows, max_tokens=max_tokens, idx_entries_per_block=geometry["idx_epb"],
                           cmp_entries_per_block=geometry["cmp_epb"], swa_entries_per_block=geometry["swa_epb"], ratio=geometry["ratio"],
                           ring_entries=geometry["ring"], window=geometry["window"], topk=geometry["topk"], status_word=status, **more)
    for t in plan.out.values():
        t.fill_(-99)
    return plan


def check(plan, want, rows, untouched=True):
    torch.cuda.synchronize()
    tokens = len(want["pos"])
    for name in TOKEN:
        got = plan.out[name].cpu().numpy()
        assert np.array_equal(got[:tokens], want[name]), name
        assert not untouched or (got[tokens:] == -99).all(), name
    for name in ROW:
        got = plan.out[name].cpu().numpy()
        assert np.array_equal(got[:rows], want[name]), name
        assert not untouched or (got[rows:] == -99).all(), name
    got = plan.out["token_starts"].cpu().numpy()
    assert np.array_equal(got[:rows + 1], want["token_starts"]) and (not untouched or (got[rows + 1:] == -99).all())
    for got, name in ((plan.lengths_out, "lengths"), (plan.free_counts_out, "counts"), (plan.idx_table, "idx_table"), (plan.cmp_table, "cmp_table")):
        assert np.array_equal(got.cpu().numpy(), want[name]), name


def oracle(s, slots, new, max_tokens, geometry):
    return step_tables(slots, new, s["lengths"], s["idx_table"], s["cmp_table"], s["swa_table"], s["idx_free"], s["cmp_free"], s["free_counts"],
                       max_tokens, **geometry)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows, capacity, longest, spare", [(1, 1, 0, 0), (1, 1, 255, 2), (2, 5, 256, 1), (31, 31, 5000, 0), (64, 70, 33000, 5),
                                                           (129, 200, 70001, 0), (513, 600, 2000, 3), (1500, 1600, 300, 0)])
def test_one_token_each(rows, capacity, longest, spare, in_place):
    rng = np.random.default_rng(rows * 7 + longest)
    lengths = rng.integers(0, longest + 1, capacity)
    lengths[:min(capacity, 4)] = np.array([longest, 3, 255, 0])[:min(capacity, 4)]      # a full page, its border, nothing
    width = pages_of(longest + 1, 4, 64) + 1
    s = state(rng, capacity, width, lengths, GEOMETRY, free=rows + spare)
    slots = rng.permutation(capacity)[:rows].astype(np.int32)
    if rows > 8:
        slots[rng.permutation(rows)[:3]] = -1
    status = wuda.device_status_word()
    plan = plan_of(s, rows + spare, rows + spare, GEOMETRY, in_place, status)
    want = oracle(s, slots, None, rows + spare, GEOMETRY)
    plan.step(torch.from_numpy(slots).cuda())
    check(plan, want, rows)
    assert int(status) == 0


GEOMETRIES = [GEOMETRY, dict(GEOMETRY, idx_epb=32, cmp_epb=64), dict(idx_epb=1, cmp_epb=7, swa_epb=3, ratio=1, ring=9, window=5, topk=4),
              dict(idx_epb=5, cmp_epb=2, swa_epb=64, ratio=3, ring=11, window=130, topk=1)]


@pytest.mark.parametrize("geometry", GEOMETRIES)
@pytest.mark.parametrize("seed", range(6))
def test_ragged_chunks_with_rows_that_cannot_be_served(geometry, seed):
    """Chunks of none to hundreds of tokens; padded rows, slots outside or twice, negative lengths and counts, tables and
    token buffers that are too short, a pool that runs out in the middle: what is left out and what is still served."""
    rng = np.random.default_rng(seed)
    rows, capacity = int(rng.integers(1, 60)), 64
    new = rng.integers(0, 300, rows) * rng.integers(0, 2, rows)
    new = np.where(rng.random(rows) < 0.3, 1, new).astype(np.int32)
    lengths = rng.integers(0, 400, capacity)
    width = max(pages_of(800, geometry["ratio"], min(geometry["idx_epb"], geometry["cmp_epb"])), 1)
    slots = rng.permutation(capacity)[:rows].astype(np.int32)
    max_tokens = int(new.sum()) + 5
    if seed >= 2:       # troubled batches
        for value in (-1, capacity, -3, 2 ** 31 - 1, slots[0], slots[rows // 2]):
            slots[int(rng.integers(0, rows))] = value
        lengths[rng.permutation(capacity)[:4]] = (-1, -2 ** 31, 2 ** 31 - 1, 100000)
        new[int(rng.integers(0, rows))] = -1
        new[int(rng.integers(0, rows))] = 2 ** 31 - 1 if seed % 2 else 1200
    if seed == 3:
        max_tokens = max(1, int(new[:rows // 2].clip(0, 1000).sum()) - 3)
    s = state(rng, capacity, width, lengths, geometry, free=2000 if seed != 4 else 0)
    if seed in (4, 5):
        s = state(rng, capacity, width, lengths, geometry, free=int(rng.integers(0, 12)))
        s["free_counts"][1] = max(0, s["free_counts"][0] - 2)
    status = wuda.device_status_word()
    plan = plan_of(s, rows + 2, max_tokens, geometry, in_place=bool(seed % 2), status=status)
    want = oracle(s, slots, new.astype(np.int64), max_tokens, geometry)
    plan.step(torch.from_numpy(slots).cuda(), torch.from_numpy(new).cuda())
    check(plan, want, rows)
    assert int(status) in ((161, 162, 163) if want["left_out"] else (0,))


@pytest.mark.parametrize("code, change", [
    (161, lambda s, slots: slots.__setitem__(2, slots[1])), (161, lambda s, slots: slots.__setitem__(2, 40)),
    (161, lambda s, slots: slots.__setitem__(2, -2)), (162, lambda s, slots: s["free_counts"].__setitem__(0, 0)),
    (163, lambda s, slots: s["lengths"].__setitem__(slots[2], -5)), (163, lambda s, slots: s["lengths"].__setitem__(slots[2], 2 ** 31 - 1)),
    (163, lambda s, slots: s["free_counts"].__setitem__(1, 5000)), (163, lambda s, slots: s["free_counts"].__setitem__(1, -1))])
def test_what_is_reported(code, change):
    rng = np.random.default_rng(5)
    s = state(rng, 40, 8, rng.integers(0, 255, 40) // 4 * 4 + 3, GEOMETRY, free=50)      # every row completes an entry
    s["lengths"][:] = np.where(np.arange(40) % 3 == 0, 255 + 0 * s["lengths"], s["lengths"])   # a third of them needs a page
    s = dict(state(rng, 40, 8, s["lengths"], GEOMETRY, free=50))
    slots = np.arange(20, dtype=np.int32)
    change(s, slots)
    status = wuda.device_status_word()
    plan = plan_of(s, 20, 20, GEOMETRY, False, status)
    plan.step(torch.from_numpy(slots).cuda())
    torch.cuda.synchronize()
    assert int(status) == code
    if code != 163 or s["free_counts"].max() <= 53 and s["free_counts"].min() >= 0:
        check(plan, oracle(s, slots, None, 20, GEOMETRY), 20)


def test_long_tables_and_far_positions():
    """Rows of more pages than one piece of work takes, positions beyond 2^24, a table whose rows start anywhere."""
    rng = np.random.default_rng(9)
    geometry = dict(GEOMETRY, idx_epb=4096)
    lengths = np.array([4 * 64 * 5001, 4 * 64 * 257 + 255, 3, 4 * 64 * 256 - 1, 4 * 64 * 4096 - 1])
    s = state(rng, 5, 5003, lengths, geometry, free=9)
    slots = np.array([4, 0, 3, 1, 2], np.int32)
    plan = plan_of(s, 5, 5, geometry, True)
    want = oracle(s, slots, None, 5, geometry)
    plan.step(torch.from_numpy(slots).cuda())
    check(plan, want, 5)


def test_no_token_and_no_row():
    rng = np.random.default_rng(1)
    s = state(rng, 3, 2, [5, 300, 0], GEOMETRY, free=2)
    plan = plan_of(s, 3, 0, GEOMETRY, True)
    slots, new = np.array([1, 0, 2], np.int32), np.zeros(3, np.int32)
    want = oracle(s, slots, new, 0, GEOMETRY)
    plan.step(torch.from_numpy(slots).cuda(), torch.from_numpy(new).cuda())
    check(plan, want, 3)
    plan = plan_of(s, 3, 3, GEOMETRY, True)
    plan.step(torch.zeros(0, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert all((t.cpu().numpy() == -99).all() for t in plan.out.values())


def test_steps_in_place_captured_and_replayed_on_another_stream():
    """Forty steps of a captured plan are forty steps of the definition: lengths, tables and stacks go on from each other."""
    rng = np.random.default_rng(3)
    s = state(rng, 9, 4, rng.integers(0, 300, 9), GEOMETRY, free=20)
    slots = np.array([3, 8, -1, 0, 5, 1], np.int32)
    plan = plan_of(s, 6, 6, GEOMETRY, True)
    dev = torch.from_numpy(slots).cuda()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        plan.step(dev)
    for _ in range(300):
        want = oracle(s, slots, None, 6, GEOMETRY)
        s.update(lengths=want["lengths"], free_counts=want["counts"], idx_table=want["idx_table"], cmp_table=want["cmp_table"])
    with torch.cuda.stream(side):
        for _ in range(300):
            graph.replay()
    side.synchronize()
    check(plan, want, 6)


def test_many_plans_on_streams_of_their_own():
    rng = np.random.default_rng(8)
    jobs = []
    for i in range(6):
        s = state(rng, 300, 40, rng.integers(0, 9000, 300), GEOMETRY, free=300)
        slots = rng.permutation(300)[:256].astype(np.int32)
        jobs.append((s, slots, plan_of(s, 256, 256, GEOMETRY, True), torch.from_numpy(slots).cuda(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, slots, plan, dev, stream in jobs:
            with torch.cuda.stream(stream):
                plan.step(dev)
    torch.cuda.synchronize()
    for s, slots, plan, dev, stream in jobs:
        for _ in range(5):
            want = oracle(s, slots, None, 256, GEOMETRY)
            s.update(lengths=want["lengths"], free_counts=want["counts"], idx_table=want["idx_table"], cmp_table=want["cmp_table"])
        check(plan, want, 256)


def compare_with_manager(tables, twin, slots, step):
    """tables' last step against the host manager's step on its own copy of the requests."""
    st = twin.step_begin(slots)
    m, out = len(slots), tables.out
    torch.cuda.synchronize()
    for name, key in (("pos", "pos"), ("q_pos", "q_pos"), ("state_row", "main_state_row"), ("idx_dst", "idx_dst"), ("cmp_dst", "cmp_dst"),
                      ("swa_dst", "swa_dst")):
        assert out[name][:m].tolist() == st[key].tolist(), (step, name)
    pos = st["pos"].tolist()
    for name in ("idx", "cmp"):
        assert torch.equal(out[name + "_block_table"][:m].cpu(), twin.block_table(name, slots)), (step, name)
    assert out["n_compressed"][:m].tolist() == twin.n_compressed(slots, pos).tolist()
    idx, lens = twin.swa_indices(slots, pos, 128)
    assert torch.equal(out["swa_indices"][:m].cpu(), idx.view(m, 128)) and out["swa_lengths"][:m].tolist() == lens.tolist()


@pytest.mark.parametrize("geometry", [{}, dict(idx_entries_per_block=32, cmp_entries_per_block=16, swa_entries_per_block=64),
                                      dict(indexer_fp8=False, state_ring_entries=12)])
def test_the_same_pages_as_the_cache_manager(geometry):
    """600 steps with requests that come, fork and go on the host in between, in a manager on the device and in its twin."""
    rng = np.random.default_rng(11)
    cache, twin = (KVCacheManager(12, 60, 12, device=d, **geometry) for d in ("cuda", "cpu"))
    live = []
    for m in (cache, twin):
        live = [m.alloc_request() for _ in range(5)]
        m.advance(live[1], 700)
        m.advance(live[2], 63)
    status = wuda.device_status_word()
    tables = CacheTables(cache, 12, status_word=status)
    for step in range(600):
        if step % 40 == 17:
            tables.pull()
            for slot in live:
                for name in ("idx", "cmp", "swa"):
                    assert cache.reqs[slot][name] == twin.reqs[slot][name], (step, name)
            if len(live) > 3:
                gone = live.pop(int(rng.integers(0, len(live))))
                cache.free_request(gone), twin.free_request(gone)
            if step % 80 == 17:
                new = [m.alloc_request() for m in (cache, twin)]
                assert new[0] == new[1]
                live.append(new[0])
            if step == 337:
                plain = next(s for s in live if not cache.reqs[s].get("shared"))
                forks = [m.fork_request(plain, 2) for m in (cache, twin)]
                assert forks[0] == forks[1]
                live += forks[0]
            tables.push()
            assert tables.shared_lengths.tolist() == [cache.reqs.get(s, {}).get("shared", 0) for s in range(12)]
        order = rng.permutation(live)[:max(1, len(live) - step % 3)].tolist()
        tables.step(torch.tensor(order, dtype=torch.int32, device="cuda"))
        compare_with_manager(tables, twin, order, step)
    tables.pull()
    for slot in list(live):
        cache.free_request(slot), twin.free_request(slot)
    for name in ("idx", "cmp", "swa"):
        assert cache._pools[name]._free == twin._pools[name]._free and sorted(cache._pools[name]._free) == list(range(60))
    assert int(status) == 0


def test_a_slot_without_a_request_is_refused_and_the_state_has_one_owner():
    cache = KVCacheManager(3, 8, 4)
    a = cache.alloc_request()
    status = wuda.device_status_word()
    tables = CacheTables(cache, 2, status_word=status)
    tables.step(torch.tensor([a, 2], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert int(status) == 163 and tables.lengths.tolist()[a] == 1 and tables.out["state_row"].tolist()[1] == -1
    with pytest.raises(wuda.WudaError):
        tables.push()
    for change in (cache.alloc_request, lambda: cache.free_request(a), lambda: cache.step_begin([a]), lambda: cache.advance(a, 1),
                   lambda: cache.fork_request(a, 0), lambda: CacheTables(cache, 2)):
        with pytest.raises(RuntimeError):
            change()
    tables.pull()
    assert cache.reqs[a]["pos"] == 0
    for call in (tables.pull, lambda: tables.step(torch.zeros(1, dtype=torch.int32, device="cuda"))):
        with pytest.raises(wuda.WudaError):
            call()


def test_refused_arguments():
    rng = np.random.default_rng(2)
    s = state(rng, 4, 3, [1, 2, 3, 4], GEOMETRY, free=2)
    plan = plan_of(s, 4, 4, GEOMETRY, True)
    good = torch.zeros(2, dtype=torch.int32, device="cuda")
    for slots, new in ((good.long(), None), (good.cpu(), None), (torch.zeros(5, dtype=torch.int32, device="cuda"), None),
                       (torch.zeros(4, dtype=torch.int32, device="cuda")[::2], None), (good, good[:1]), (good, good.cpu()), (good, good.long())):
        with pytest.raises(wuda.WudaError):
            plan.step(slots, new)
    d = {k: torch.from_numpy(v.copy()).cuda() for k, v in s.items()}
    names = ("lengths", "idx_table", "cmp_table", "swa_table", "idx_free", "cmp_free", "free_counts")

    def made(**change):
        more = {k: change.pop(k) for k in list(change) if k not in names}
        return wuda.StepTables(*[change.get(n, d[n]) for n in names], **dict(dict(max_rows=2), **more))

    made()
    for change in (dict(lengths=d["lengths"].cpu()), dict(lengths=d["lengths"].long()), dict(idx_table=d["idx_table"][:, :2]),
                   dict(cmp_table=d["idx_table"]), dict(cmp_table=d["cmp_table"][:3]), dict(swa_table=d["idx_table"]),
                   dict(free_counts=d["free_counts"][:1]), dict(max_rows=0), dict(max_rows=5000, max_tokens=-1), dict(ratio=0), dict(ring_entries=0),
                   dict(window=0), dict(max_tokens=300000), dict(out=dict(pos=d["lengths"])), dict(out=dict(nothing=d["lengths"])),
                   dict(lengths_out=d["lengths"][:2]), dict(status_word=d["lengths"].long()), dict(idx_entries_per_block=0)):
        with pytest.raises((wuda.WudaError, ZeroDivisionError)):
            made(**change)


def test_what_a_step_writes_overlaps_nothing_and_numbers_are_not_cut():
    s = state(np.random.default_rng(3), 4, 3, [1, 2, 3, 4], GEOMETRY, free=2)
    d = {k: torch.from_numpy(v.copy()).cuda() for k, v in s.items()}
    names = ("lengths", "idx_table", "cmp_table", "swa_table", "idx_free", "cmp_free", "free_counts")

    def made(change={}, **more):
        return wuda.StepTables(*[change.get(n, d[n]) for n in names], max_rows=2, **more)

    block = torch.zeros(64, dtype=torch.int32, device="cuda")
    made(dict(idx_free=block[:8], cmp_free=block[4:12]))                                  # only read: may overlap
    made(lengths_out=d["lengths"], free_counts_out=block[:2])
    made(lengths_out=block[4:8], free_counts_out=block[8:10], out=dict(n_compressed=block[:2], swa_lengths=block[2:4]))
    for change, more in ((dict(lengths=block[:4]), dict(lengths_out=block[2:6])), (dict(), dict(free_counts_out=d["lengths"][:2])),
                         (dict(), dict(out=dict(idx_block_table=d["idx_table"]))), (dict(), dict(out=dict(cmp_block_table=d["idx_table"]))),
                         (dict(), dict(out=dict(n_compressed=block[:2], cmp_lengths=block[1:3]))),
                         (dict(idx_free=block[:8]), dict(out=dict(n_compressed=block[6:8]))), (dict(idx_free=block), dict(lengths_out=block[60:])),
                         (dict(), dict(topk=1 << 32)), (dict(), dict(window=(1 << 32) + 128)), (dict(), dict(max_tokens=1 << 32)),
                         (dict(), dict(ring_entries=(1 << 32) + 8))):
        with pytest.raises(wuda.WudaError):
            made(change, **more)


@pytest.mark.parametrize("in_place", [False, True])
def test_a_step_of_no_rows_carries_the_state_over(in_place):
    s = state(np.random.default_rng(5), 9, 3, [1, 2, 3, 4, 5, 6, 7, 8, 300], GEOMETRY, free=2)
    plan = plan_of(s, 4, 4, GEOMETRY, in_place)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    want = oracle(s, np.zeros(0, np.int32), None, 4, GEOMETRY)
    for new in (None, none):
        plan.lengths_out.fill_(-7) if not in_place else None
        plan.step(none, new)
        torch.cuda.synchronize()
        assert np.array_equal(plan.lengths_out.cpu().numpy(), want["lengths"]) and np.array_equal(plan.free_counts_out.cpu().numpy(), want["counts"])
        assert plan.out["token_starts"][1:].eq(-99).all() and (in_place or int(plan.out["token_starts"][0]) == 0)
        assert all(plan.out[name].eq(-99).all() for name in TOKEN + ROW)
    assert int(plan._counter) == 0


def test_making_a_plan_launches_nothing():
    """A plan whose next state is not in place: what the caller holds there is written by its steps alone, on their stream."""
    s = state(np.random.default_rng(6), 9, 3, [1, 2, 3, 4, 5, 6, 7, 8, 300], GEOMETRY, free=4)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    plan_of(s, 4, 4, GEOMETRY, False)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        plan = plan_of(s, 4, 4, GEOMETRY, False)
    torch.cuda.synchronize()
    assert plan.lengths_out.eq(-7).all() and plan.free_counts_out.eq(-7).all()
    slots = np.array([3, 8, 0], np.int32)
    dev, want = torch.from_numpy(slots).cuda(), oracle(s, slots, None, 4, GEOMETRY)
    d = {k: torch.from_numpy(v.copy()).cuda() for k, v in s.items()}
    after = torch.full_like(d["lengths"], -7), torch.full_like(d["free_counts"], -7)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):            # made while a graph is captured, too
        plan = wuda.StepTables(d["lengths"], d["idx_table"], d["cmp_table"], d["swa_table"], d["idx_free"], d["cmp_free"], d["free_counts"],
                               max_rows=4, topk=GEOMETRY["topk"], lengths_out=after[0], free_counts_out=after[1])
        plan.step(dev)
    graph.replay()
    check(plan, want, 3, untouched=False)


def test_beams_move_only_while_the_tables_have_the_state():
    """Between a pull() and the next push() the pages in the tables may be other requests' already."""
    cache = KVCacheManager(4, 12, 4)
    a = cache.alloc_request()
    cache.advance(a, 300)
    tables = CacheTables(cache, 4)
    reorder = tables.beam_reorder(2)
    pair = lambda *v: torch.tensor([v], dtype=torch.int32, device="cuda")
    out = pair(-5, -5)
    tables.pull()
    (b,) = cache.fork_request(a, 1)
    with pytest.raises(wuda.WudaError):
        reorder.run(pair(0, 0), pair(a, b), out)
    torch.cuda.synchronize()
    assert out.tolist() == [[-5, -5]]
    tables.push()
    cache.main_state[a] = 3.0
    reorder.run(pair(0, 0), pair(a, b), out)
    assert out.tolist() == [[a, b]] and torch.all(cache.main_state[b] == 3.0)
