"""The bookkeeping of decode steps on the GPU.

KVCacheManager (kv_cache.py) hands out slots and pages on the host and copies thirteen small arrays to the device for every
step.  StepTables keeps what it needs for a step - lengths, page tables by slot, free pages - on the device and makes the step's
arrays there in one launch, from the request slots alone: a step can be prepared inside a CUDA graph, and a server whose next tokens
are chosen on the GPU needs no host between two steps.  The counterpart in the reference is the host code of
dsv4_megakernel/megakernel/test/kv_cache_manager.py:53-257; one token per request gives the same numbers and the same pages.
"""
import ctypes
import math

import torch

from . import _lib
from ._lib import check, lib
from . import ops as _ops
from .beams import BeamReorder, PagedState
from .kv_cache import M1_BODY, RATIO, WIN
from .ops import _int32, _on_current_device, _require, _stream

_TOKEN_OUTPUTS = (("pos", torch.int64), ("q_pos", torch.int32), ("state_row", torch.int64), ("idx_dst", torch.int64),
                  ("cmp_dst", torch.int64), ("swa_dst", torch.int64))
_MOST_ROWS = 4096       # of a step (wuda_step_tables)


class StepTables:
    """lengths int32 [capacity]: tokens that the caches of each request slot hold; idx_table / cmp_table int32
    [capacity, pages]: its pages in the two compressed pools (grown in place); swa_table int32 [capacity,
    ceil(window / swa_entries_per_block)]: its pages of the window ring; idx_free / cmp_free int32: free pages, the next
    one last; free_counts int32 [2]: how many of them there are.  All are the caller's, contiguous, on the current device.

    step() writes the state after the step to lengths_out / free_counts_out, by default in place, and the step's arrays to
    `out`: given tensors (a subset by name, e.g. a CsaDecodeStage's buffers) or ones allocated here.

    A plan belongs to one stream at a time: its outputs, like the caches, are those of the last step."""

    def __init__(self, lengths, idx_table, cmp_table, swa_table, idx_free, cmp_free, free_counts, *, max_rows, max_tokens=None,
                 idx_entries_per_block=64, cmp_entries_per_block=64, swa_entries_per_block=256, ratio=4, ring_entries=8,
                 window=128, topk=2048, lengths_out=None, free_counts_out=None, out=None, status_word=None):
        max_tokens = max_rows if max_tokens is None else max_tokens
        for value, name in ((max_rows, "max_rows"), (max_tokens, "max_tokens"), (idx_entries_per_block, "idx_entries_per_block"),
                            (cmp_entries_per_block, "cmp_entries_per_block"), (swa_entries_per_block, "swa_entries_per_block"),
                            (ratio, "ratio"), (ring_entries, "ring_entries"), (window, "window"), (topk, "topk")):
            _int32(value, name)
        _require(1 <= max_rows <= _MOST_ROWS and max_tokens >= 0, "max_rows must be in [1, %d], max_tokens not negative" % _MOST_ROWS)
        _require(_on_current_device(lengths), "the state must be on the current CUDA device")
        dev = lengths.device

        def state(t, name, *shape):
            _require(t.device == dev and t.dtype == torch.int32 and t.is_contiguous() and
                     t.dim() == len(shape) and all(n is None or n == m for n, m in zip(shape, t.shape)),
                     "%s must be contiguous int32 %s on the lengths' device" % (name, list(shape)))
            return t

        state(lengths, "lengths", None)
        capacity = lengths.size(0)
        state(idx_table, "idx_table", capacity, None)
        width = idx_table.size(1)
        state(cmp_table, "cmp_table", capacity, width)
        state(swa_table, "swa_table", capacity, -(-window // max(swa_entries_per_block, 1)))
        state(idx_free, "idx_free", None)
        state(cmp_free, "cmp_free", None)
        state(free_counts, "free_counts", 2)
        self.lengths_out = state(lengths if lengths_out is None else lengths_out, "lengths_out", capacity)
        self.free_counts_out = state(free_counts if free_counts_out is None else free_counts_out, "free_counts_out", 2)
        self.lengths, self.idx_table, self.cmp_table, self.swa_table = lengths, idx_table, cmp_table, swa_table
        self.idx_free, self.cmp_free, self.free_counts = idx_free, cmp_free, free_counts
        self.max_rows, self.max_tokens = int(max_rows), int(max_tokens)
        shapes = {name: ((self.max_tokens,), dtype) for name, dtype in _TOKEN_OUTPUTS}
        shapes.update({name: ((self.max_rows,), torch.int32) for name in ("n_compressed", "cmp_lengths", "swa_lengths")})
        shapes.update(token_starts=((self.max_rows + 1,), torch.int32), swa_indices=((self.max_rows, window), torch.int32),
                      idx_block_table=((self.max_rows, width), torch.int32), cmp_block_table=((self.max_rows, width), torch.int32))
        given = dict(out or {})
        _require(set(given) <= set(shapes), "no output named %s" % sorted(set(given) - set(shapes)))
        # the counter and the outputs that are not given, in one block of zeros, each on 16 bytes
        places, size = {}, 16
        for name, (shape, dtype) in shapes.items():
            if given.get(name) is None:
                places[name] = size, size + math.prod(shape) * dtype.itemsize
                size = (places[name][1] + 15) // 16 * 16
        block = torch.zeros(size, dtype=torch.uint8, device=dev)
        self._counter = block[:4].view(torch.int32)
        self.out = {}
        for name, (shape, dtype) in shapes.items():
            t = given.get(name)
            if t is None:
                t = block[slice(*places[name])].view(dtype).view(shape)
            _require(t.device == dev and t.dtype == dtype and t.is_contiguous() and t.dim() == len(shape) and
                     t.size(0) >= shape[0] and tuple(t.shape[1:]) == shape[1:],
                     "%s must be contiguous %s of at least %s on the lengths' device" % (name, dtype, list(shape)))
            self.out[name] = t
        _require(status_word is None or (status_word.device == dev and status_word.dtype == torch.int32 and status_word.numel() >= 1),
                 "status_word must be int32 on the lengths' device")
        # what a step writes overlaps nothing else (rows are written while others are read), but the state may be its own successor
        written = [idx_table, cmp_table, self.lengths_out, self.free_counts_out, *self.out.values()]
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * 4 * (1 + (t.dtype is torch.int64)), i < len(written))
                       for i, t in enumerate(written + [swa_table, idx_free, cmp_free] +
                                             [t for t, after in ((lengths, self.lengths_out), (free_counts, self.free_counts_out))
                                              if t.data_ptr() != after.data_ptr()]) if t.numel())
        end, end_written = 0, 0
        for begin, stop, writes in spans:
            _require(begin >= (end if writes else end_written), "what a step writes must not overlap its other tensors")
            end, end_written = max(end, stop), max(end_written, stop) if writes else end_written
        self.status_word = status_word
        self._device = dev.index
        p = lambda t: t.data_ptr()
        self._args = _lib.StepTablesArgs(
            lengths=p(lengths), lengths_out=p(self.lengths_out), idx_table=p(idx_table), cmp_table=p(cmp_table), swa_table=p(swa_table),
            idx_free=p(idx_free), cmp_free=p(cmp_free), free_counts=p(free_counts), free_counts_out=p(self.free_counts_out),
            counter=p(self._counter), table_stride=width, block_table_stride=width, capacity=capacity, table_width=width,
            idx_free_capacity=idx_free.size(0), cmp_free_capacity=cmp_free.size(0), max_tokens=self.max_tokens,
            idx_entries_per_block=idx_entries_per_block, cmp_entries_per_block=cmp_entries_per_block,
            swa_entries_per_block=swa_entries_per_block, ratio=ratio, ring_entries=ring_entries, window=window, topk=topk,
            **{name: p(t) for name, t in self.out.items()})
        self._args_ref, self._address = ctypes.byref(self._args), ctypes.addressof(self._args)
        self._status = None if status_word is None else status_word.data_ptr()
        # the library's checks: a call of no rows launches nothing where the state is in place
        checked = _lib.StepTablesArgs.from_buffer_copy(self._args)
        checked.lengths_out, checked.free_counts_out = checked.lengths, checked.free_counts
        check(lib.wuda_step_tables(ctypes.byref(checked), None, None, 0, None, None))

    def step(self, slots, new_tokens=None):
        """slots int32 [rows]: the request slot of each row, -1 for a padded row, each slot once; new_tokens int32 [rows]: its
        tokens in this step (None: one each).  Fills and returns self.out:
          pos, state_row, idx_dst, cmp_dst, swa_dst int64 and q_pos int32 [max_tokens] by token, row after row
          token_starts int32 [rows + 1]; n_compressed, cmp_lengths, swa_lengths int32 [rows]
          swa_indices int32 [rows, window]; idx_block_table, cmp_block_table int32 [rows, pages]
        What lies behind the last token and the last row is left as it was.  A row that cannot be served (a slot given twice,
        no free page, a context beyond the tables) is reported in status_word and left out: positions 0, destinations -1,
        lengths 0; its state stays.
        More than one token to a request is for a caller's own prefill: only a request's last tokens get a ring row, and the cache
        writers of this package skip those without one."""
        if _ops._fast.step_tables(self._address, slots, new_tokens, self.max_rows, self._device, self._status):
            return self.out
        rows = slots.numel()
        if not (slots.dtype is torch.int32 and slots.is_contiguous() and rows <= self.max_rows and slots.is_cuda and
                slots.get_device() == self._device == torch._C._cuda_getDevice()):
            _require(False, "slots must be contiguous int32, at most max_rows = %d of them, on the plan's device, which must be the "
                            "current one" % self.max_rows)
        if new_tokens is not None and not (new_tokens.dtype is torch.int32 and new_tokens.is_contiguous() and new_tokens.numel() == rows
                                           and new_tokens.is_cuda and new_tokens.get_device() == self._device):
            _require(False, "new_tokens must be contiguous int32, one for each slot, on the plan's device")
        status = lib.wuda_step_tables(self._args_ref, slots.data_ptr(), None if new_tokens is None else new_tokens.data_ptr(), rows,
                                      self._status, _stream())
        if status:
            check(status)
        return self.out


class CacheTables(StepTables):
    """The step tables of a KVCacheManager.  push() brings the manager's requests, page tables and free pages to the device;
    steps then run there, and the manager knows nothing of them until pull() brings its state up to date.  So requests come, fork and go
    on the host between a pull() and a push(), at whatever pace they do; steps need neither."""

    def __init__(self, cache, max_rows, *, max_tokens=None, topk=2048, out=None, status_word=None):
        self.cache = cache
        dev = cache.main_state.device
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=dev)
        epb = cache.entries_per_block
        pages = {name: cache._pools[name].data.size(0) for name in ("idx", "cmp")}
        self.shared_lengths = i32(cache.capacity)
        self.has_state = False      # these tables have the state, from a push() to the next pull(); else the manager has it, or other tables
        super().__init__(i32(cache.capacity), i32(cache.capacity, cache.max_pages), i32(cache.capacity, cache.max_pages),
                         i32(cache.capacity, -(-WIN // epb["swa"])), i32(pages["idx"]), i32(pages["cmp"]), i32(2),
                         max_rows=max_rows, max_tokens=max_tokens, idx_entries_per_block=epb["idx"],
                         cmp_entries_per_block=epb["cmp"], swa_entries_per_block=epb["swa"], ratio=RATIO,
                         ring_entries=cache.state_ring_entries, window=WIN, topk=topk, out=out, status_word=status_word)
        self.push()

    def push(self):
        """The manager's state to the device, on the current stream."""
        cache = self.cache
        if cache.on_device:
            raise _lib.WudaError(1, "the state is on the device: pull() it before the manager changes anything")
        lengths, shared = [-1] * cache.capacity, [0] * cache.capacity      # (a slot without a request is refused)
        tables = {name: torch.zeros(tuple(t.shape), dtype=torch.int32)
                  for name, t in (("idx", self.idx_table), ("cmp", self.cmp_table), ("swa", self.swa_table))}
        for slot, req in cache.reqs.items():
            lengths[slot], shared[slot] = req["pos"] + 1, req.get("shared", 0)
            for name, table in tables.items():
                if len(req[name]) > table.size(1):
                    raise ValueError("request %d holds more pages than max_pages_per_req" % slot)
                table[slot, :len(req[name])] = torch.tensor(req[name], dtype=torch.int32)
        for name, device in (("idx", self.idx_table), ("cmp", self.cmp_table), ("swa", self.swa_table)):
            device.copy_(tables[name])
        for name, device in (("idx", self.idx_free), ("cmp", self.cmp_free)):
            free = cache._pools[name]._free
            device[:len(free)].copy_(torch.tensor(free, dtype=torch.int32))
        self.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.shared_lengths.copy_(torch.tensor(shared, dtype=torch.int32))
        self.free_counts.copy_(torch.tensor([len(cache._pools[name]._free) for name in ("idx", "cmp")], dtype=torch.int32))
        cache.on_device = self.has_state = True

    def pull(self):
        """The device's state back into the manager; waits for the current stream.  Captured steps are not replayed until the
        next push()."""
        if not self.has_state:
            raise _lib.WudaError(1, "the manager has the state already")
        cache = self.cache
        lengths, counts = self.lengths.tolist(), self.free_counts.tolist()
        for i, (name, table, free) in enumerate((("idx", self.idx_table, self.idx_free), ("cmp", self.cmp_table, self.cmp_free))):
            epb, rows = cache.entries_per_block[name], table.cpu()
            cache._pools[name]._free = free[:counts[i]].tolist()
            for slot, req in cache.reqs.items():
                req[name] = rows[slot, :-(-(lengths[slot] // RATIO) // epb)].tolist()
        for slot, req in cache.reqs.items():
            req["pos"] = lengths[slot] - 1
        cache.on_device = self.has_state = False

    def step(self, slots, new_tokens=None):
        if not self.has_state:
            raise _lib.WudaError(1, "the cache manager has the state: push() it first")
        return super().step(slots, new_tokens)

    def beam_reorder(self, width, states=(), status_word=None):
        """A BeamReorder over the cache's state rings and pools, and `states` beside them ([capacity, ...] by slot).  Like a step, it
        runs from a push() to the next pull()."""
        cache = self.cache
        epb, key = cache.entries_per_block, cache.idx_entry_bytes - 4
        pools = [PagedState(cache.idx_pool, self.idx_table, epb["idx"], (key, 4), tokens_per_entry=RATIO),
                 PagedState(cache.cmp_pool, self.cmp_table, epb["cmp"], (M1_BODY, 8), tokens_per_entry=RATIO),
                 PagedState(cache.swa_pool, self.swa_table, epb["swa"], (M1_BODY, 8), ring=WIN)]
        return _CacheReorder(self, width, states=[cache.main_state, cache.idx_state, *states], pools=pools,
                             status_word=self.status_word if status_word is None else status_word)


class _CacheReorder(BeamReorder):
    """The beams of a KVCacheManager's requests.  While the manager has their state, the pages in the tables may be others'."""

    def __init__(self, tables, width, **more):
        super().__init__(tables.lengths, width, shared_lengths=tables.shared_lengths, **more)
        self._tables = tables

    def run(self, parents, slots, slots_out):
        if not self._tables.has_state:
            raise _lib.WudaError(1, "the cache manager has the state: push() it first")
        return super().run(parents, slots, slots_out)
