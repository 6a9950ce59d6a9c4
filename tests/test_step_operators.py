"""Step tables, beam selection and beam reordering without a GPU: what the C ABI refuses before it looks for a device, the layouts of
the argument structs, the cache manager's forks."""
import ctypes
import os
import subprocess

import pytest
import torch

import wuda_b200._lib as L
from wuda_b200.kv_cache import KVCacheManager
from wuda_b200.step_tables import StepTables

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "wuda_b200.h")
FAKE = 0x10000          # refused calls never read it
INVALID, NO_DEVICE = 1, 4


def message():
    return L.lib.wuda_last_error().decode()


def tables(**change):
    pointers = {n: FAKE for n, t in L.StepTablesArgs._fields_ if t is ctypes.c_void_p}
    pointers["cmp_table"] = 2 * FAKE
    numbers = dict(table_stride=8, block_table_stride=8, capacity=16, table_width=8, idx_free_capacity=4, cmp_free_capacity=4, max_tokens=4,
                   idx_entries_per_block=64, cmp_entries_per_block=64, swa_entries_per_block=256, ratio=4, ring_entries=8, window=128, topk=512)
    return L.StepTablesArgs(**{**pointers, **numbers, **change})


@pytest.mark.parametrize("change, rows, word", [
    (dict(), -1, "rows"), (dict(), 4097, "rows"), (dict(), 5, "max_tokens"), (dict(capacity=0), 1, "capacity"), (dict(capacity=16385), 1, "capacity"),
    (dict(table_width=0), 1, "table_width"), (dict(table_width=262145, table_stride=1 << 20, block_table_stride=1 << 20), 1, "table_width"),
    (dict(max_tokens=-1), 0, "max_tokens"), (dict(max_tokens=262145), 1, "max_tokens"), (dict(table_stride=7), 1, "shorter"),
    (dict(block_table_stride=7), 1, "shorter"), (dict(idx_free_capacity=-1), 1, "negative"), (dict(cmp_entries_per_block=0), 1, "entries"),
    (dict(swa_entries_per_block=-1), 1, "entries"), (dict(ratio=0), 1, "ratio"), (dict(window=65537), 1, "window"), (dict(topk=-1), 1, "topk"),
    (dict(lengths=None), 1, "NULL"), (dict(counter=None), 0, "NULL"), (dict(pos=None), 1, "token outputs"), (dict(idx_free=None), 1, "free stacks"),
    (dict(cmp_table=FAKE), 1, "share")])
def test_step_tables_refusals(change, rows, word):
    st = L.lib.wuda_step_tables(ctypes.byref(tables(**change)), FAKE, None, rows, None, None)
    assert st == INVALID and word in message(), message()


def test_step_tables_other_refusals():
    assert L.lib.wuda_step_tables(None, FAKE, None, 1, None, None) == INVALID
    assert L.lib.wuda_step_tables(ctypes.byref(tables()), None, None, 1, None, None) == INVALID and "slots" in message()
    assert L.lib.wuda_step_tables(ctypes.byref(tables()), None, None, 0, None, None) == 0
    assert L.lib.wuda_step_tables(ctypes.byref(tables(max_tokens=0, pos=None, idx_free=None, idx_free_capacity=0)), None, FAKE, 0, None, None) == 0


def select(**change):
    given = {n: FAKE for n, t in L.BeamSelectArgs._fields_ if t is ctypes.c_void_p and n != "finished"}
    given.update(group_stride=400, beam_stride=100, workspace_bytes=1 << 30, groups=2, width=4, vocab=100, k=8, eos_token=-1, logits_type=0)
    return L.BeamSelectArgs(**{**given, **change})


@pytest.mark.parametrize("change, word", [
    (dict(groups=-1), "groups"), (dict(groups=257), "groups"), (dict(width=0), "width"), (dict(width=33), "width"), (dict(k=0), "k must"),
    (dict(k=65), "k must"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 24) + 1), "vocab"), (dict(logits_type=3), "logits_type"),
    (dict(logits=None), "NULL"), (dict(counters=None), "NULL"), (dict(beam_stride=-1), "strides"), (dict(logits=FAKE + 1), "aligned"),
    (dict(logits=FAKE + 2, logits_type=2), "aligned"), (dict(eos_token=100), "eos_token"), (dict(eos_token=-2), "eos_token"),
    (dict(finished=FAKE), "eos_token"), (dict(workspace_bytes=8), "workspace"), (dict(workspace=FAKE + 8), "workspace")])
def test_beam_select_refusals(change, word):
    assert L.lib.wuda_beam_select(ctypes.byref(select(**change)), None) == INVALID and word in message(), message()


def test_beam_select_sizes():
    size = L.lib.wuda_beam_select_workspace_bytes
    assert L.lib.wuda_beam_select(None, None) == INVALID
    assert L.lib.wuda_beam_select(ctypes.byref(select(groups=0, logits=None)), None) == 0
    for bad in ((257, 4, 100, 8, 0), (1, 33, 100, 8, 0), (1, 4, 0, 8, 0), (1, 4, 100, 65, 0), (1, 4, 100, 8, 3), (-1, 4, 100, 8, 0)):
        assert size(*bad) == -1
    for kind in (0, 1, 2):
        for groups, width, vocab, k in ((1, 1, 1, 1), (1, 4, 32000, 8), (256, 32, 1 << 24, 64), (3, 5, 100003, 10)):
            assert 0 < size(groups, width, vocab, k, kind) < 1 << 28
    assert size(0, 4, 100, 8, 0) == 0


def reorder(states=((FAKE, 64),), pools=({},), **change):
    a = L.BeamReorderArgs(**dict(dict(lengths=FAKE, num_states=len(states), num_pools=len(pools), capacity=16, width=4), **change))
    for i, (data, row_bytes) in enumerate(states[:8]):
        a.states[i].data, a.states[i].row_bytes = data, row_bytes
    for i, c in enumerate(pools[:4]):
        c = dict(dict(data=FAKE, table=FAKE, stride_bytes=8448, num_blocks=8, table_width=4, entries_per_block=64, tokens_per_entry=4, ring=0,
                      segment_bytes=(128, 4)), **c)
        for name, value in c.items():
            setattr(a.pools[i], name, (ctypes.c_int32 * 2)(*value) if name == "segment_bytes" else value)
    return a


@pytest.mark.parametrize("args, groups, word", [
    (dict(width=0), 1, "width"), (dict(width=33), 1, "width"), (dict(), -1, "groups"), (dict(), 1025, "groups"), (dict(capacity=0), 1, "capacity"),
    (dict(capacity=16385), 1, "capacity"), (dict(num_states=9), 0, "num_states"), (dict(num_pools=5), 0, "num_pools"), (dict(lengths=None), 0, "lengths"),
    (dict(states=((None, 64),)), 0, "state 0"), (dict(states=((FAKE, 64), (FAKE, 6))), 0, "state 1"), (dict(states=((FAKE + 2, 64),)), 0, "state 0"),
    (dict(states=((FAKE, 0),)), 0, "state 0"), (dict(pools=(dict(data=FAKE + 8),)), 0, "pool 0"), (dict(pools=({}, dict(stride_bytes=8456))), 0, "pool 1"),
    (dict(pools=(dict(table=None),)), 0, "pool 0"), (dict(pools=(dict(num_blocks=0),)), 0, "positive"), (dict(pools=(dict(ring=-1),)), 0, "positive"),
    (dict(pools=(dict(tokens_per_entry=0),)), 0, "positive"), (dict(pools=(dict(segment_bytes=(126, 4)),)), 0, "multiples"),
    (dict(pools=(dict(segment_bytes=(0, 4)),)), 0, "multiples"), (dict(pools=(dict(segment_bytes=(4, 4), entries_per_block=3),)), 0, "16 bytes"),
    (dict(pools=(dict(stride_bytes=8432),)), 0, "hold"), (dict(states=((FAKE, 1 << 40),)), 100, "pieces")])
def test_beam_reorder_refusals(args, groups, word):
    st = L.lib.wuda_beam_reorder(ctypes.byref(reorder(**args)), FAKE, 2 * FAKE, 3 * FAKE, groups, None, None)
    assert st == INVALID and word in message(), message()


@pytest.mark.parametrize("pool, word", [
    (dict(entries_per_block=4, segment_bytes=(1 << 30, 1 << 30), stride_bytes=1 << 33), "16 MB"),
    (dict(entries_per_block=1 << 30, table_width=1 << 30, segment_bytes=(16, 0), stride_bytes=1 << 34), "pieces")])
def test_beam_reorder_refuses_what_does_not_fit_its_numbers(pool, word):
    st = L.lib.wuda_beam_reorder(ctypes.byref(reorder(pools=(pool,) * 4)), FAKE, 2 * FAKE, 3 * FAKE, 1024, None, None)
    assert st == INVALID and word in message(), message()


def test_beam_reorder_other_refusals():
    ok = ctypes.byref(reorder())
    assert L.lib.wuda_beam_reorder(None, FAKE, FAKE, FAKE, 1, None, None) == INVALID
    assert L.lib.wuda_beam_reorder(ok, None, None, None, 0, None, None) == 0
    assert L.lib.wuda_beam_reorder(ok, FAKE, None, 3 * FAKE, 1, None, None) == INVALID
    assert L.lib.wuda_beam_reorder(ok, FAKE, 2 * FAKE, 2 * FAKE, 1, None, None) == INVALID and "its own" in message()
    assert L.lib.wuda_beam_reorder(ok, FAKE, 2 * FAKE, FAKE, 1, None, None) == INVALID and "its own" in message()
    assert L.lib.wuda_beam_reorder(ok, FAKE, 2 * FAKE, 2 * FAKE + 12, 1, None, None) == INVALID and "its own" in message()


def test_struct_layouts_match_the_header(tmp_path):
    structs = {"wuda_step_tables_args": L.StepTablesArgs, "wuda_beam_select_args": L.BeamSelectArgs, "wuda_beam_state": L.BeamState,
               "wuda_beam_pool": L.BeamPool, "wuda_beam_reorder_args": L.BeamReorderArgs}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "%s"' % HEADER, 'int main(void) {']
    for cname, cls in structs.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in cls._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ['return 0; }']))
    subprocess.check_call(["gcc", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")])
    out = dict(line.split() for line in subprocess.check_output([str(tmp_path / "layout")], text=True).splitlines())
    for cname, cls in structs.items():
        assert int(out[cname]) == ctypes.sizeof(cls), cname
        for field, _ in cls._fields_:
            assert int(out["%s.%s" % (cname, field)]) == getattr(cls, field).offset, "%s.%s" % (cname, field)


def test_forked_requests_share_filled_pages_and_give_each_back_once():
    m = KVCacheManager(6, 20, 8, device="cpu")
    a = m.alloc_request()
    m.advance(a, 4 * (2 * 64 + 10))                      # two filled pages and one of ten entries
    m.main_state[a] = 5.0
    m.cmp_pool.copy_(torch.arange(20, dtype=torch.uint8)[:, None].expand(20, m.cmp_pool.size(1)))
    m.swa_pool[m.reqs[a]["swa"][0]] = 77
    before = {n: len(m._pools[n]._free) for n in ("swa", "cmp", "idx")}
    b, c = m.fork_request(a, 2)
    for s in (b, c):
        assert m.reqs[s]["pos"] == m.reqs[a]["pos"] and m.reqs[s]["shared"] == 4 * 138 == m.reqs[a]["shared"]
        for name in ("cmp", "idx"):
            assert m.reqs[s][name][:2] == m.reqs[a][name][:2] and m.reqs[s][name][2] != m.reqs[a][name][2]
        assert torch.all(m.main_state[s] == 5.0) and torch.all(m.swa_pool[m.reqs[s]["swa"][0]] == 77)
        assert torch.equal(m.cmp_pool[m.reqs[s]["cmp"][2]], m.cmp_pool[m.reqs[a]["cmp"][2]])
    assert {n: before[n] - len(m._pools[n]._free) for n in before} == dict(swa=2, cmp=2, idx=2)
    with pytest.raises(ValueError):
        m.fork_request(b, 1)
    for _ in range(4 * 60):                              # on their own from here
        m.step_begin([a, b, c])
    assert len(set(m.reqs[a]["cmp"][2:] + m.reqs[b]["cmp"][2:] + m.reqs[c]["cmp"][2:])) == 6
    for s in (b, a, c):
        m.free_request(s)
        held = [p for r in m.reqs.values() for p in r["cmp"]]
        assert not set(held) & set(m._pools["cmp"]._free) and len(set(m._pools["cmp"]._free)) == len(m._pools["cmp"]._free)
    assert not m._owners["cmp"] and not m._owners["idx"]
    for name in ("swa", "cmp", "idx"):
        assert sorted(m._pools[name]._free) == list(range(20))


def test_a_fork_without_room_takes_nothing():
    m = KVCacheManager(4, 3, 8, device="cpu")
    a = m.alloc_request()
    m.advance(a, 300)                                    # two pages of three
    with pytest.raises(ValueError):
        m.fork_request(a, 2)
    with pytest.raises(ValueError):
        m.fork_request(a, 4)
    assert len(m._pools["cmp"]._free) == 1 and len(m._pools["swa"]._free) == 2 and not m.reqs[a].get("shared") and len(m._free_slots) == 3
    assert m.fork_request(a, 0) == [] and not m.reqs[a].get("shared")
    (b,) = m.fork_request(a, 1)
    assert m.reqs[b]["cmp"][0] == m.reqs[a]["cmp"][0]


@pytest.mark.parametrize("tokens", [0, 100, 1000])
def test_what_is_left_of_a_fork_is_forked_again(tokens):
    """The winner of a search goes on alone and starts the next one; until then no member of the fork starts one of its own."""
    m = KVCacheManager(5, 30, 30, device="cpu")
    a = m.alloc_request()
    m.advance(a, tokens)
    b, c = m.fork_request(a, 2)
    for freed in (a, c):
        with pytest.raises(ValueError):
            m.fork_request(b, 1)
        m.free_request(freed)
    for _ in range(300):
        m.step_begin([b])
    d, e = m.fork_request(b, 2)
    filled = (tokens + 300) // 4 // 64
    for s in (d, e):
        assert m.reqs[s]["shared"] == m.reqs[b]["shared"] == tokens + 300 and m.reqs[s]["cmp"][:filled] == m.reqs[b]["cmp"][:filled]
        assert not set(m.reqs[s]["cmp"][filled:]) & set(m.reqs[b]["cmp"])
    for s in (d, b, e):
        m.free_request(s)
    assert not m._owners["cmp"] and not m._owners["idx"]
    for name in ("swa", "cmp", "idx"):
        assert sorted(m._pools[name]._free) == list(range(30))


def test_page_tables_are_not_answered_while_they_grow_on_the_device():
    m = KVCacheManager(2, 4, 4, device="cpu")
    a = m.alloc_request()
    m.advance(a, 300)
    pages = m.block_table("idx", [a])
    m.on_device = True
    with pytest.raises(RuntimeError):
        m.block_table("idx", [a])
    m.on_device = False
    assert torch.equal(m.block_table("idx", [a]), pages)


@pytest.mark.parametrize("rows", [0, -1, 4097, 5000])
def test_a_plan_of_more_rows_than_a_step_takes_is_refused(rows):
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(L.WudaError, match="max_rows"):
        StepTables(i32(4), i32(4, 3), i32(4, 3), i32(4, 1), i32(2), i32(2), i32(2), max_rows=rows, max_tokens=8)


@pytest.mark.parametrize("change", [dict(scores_out=FAKE), dict(scores_out=FAKE + 124), dict(scores_out=FAKE - 60, k=4), dict(scores_out=FAKE - 252),
                                    dict(finished=FAKE, finished_out=FAKE, eos_token=1), dict(finished=FAKE, finished_out=FAKE + 31, eos_token=1),
                                    dict(finished=FAKE, finished_out=FAKE - 63, eos_token=1)])
def test_beam_select_outputs_that_overlap_what_other_groups_still_read(change):
    """scores float [8, 4] from FAKE to FAKE + 128, finished [8, 4] to FAKE + 32; outputs [8, k], k = 8 if not 4."""
    a = select(**{**dict(groups=8, scores_out=2 * FAKE, finished_out=2 * FAKE), **change})
    assert L.lib.wuda_beam_select(ctypes.byref(a), None) == INVALID and "overlap" in message(), message()
