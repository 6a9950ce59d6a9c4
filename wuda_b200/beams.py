"""Beam search over paged caches: what a beam's request slot holds moves to the slots of its children, on the GPU.

beam_select (ops.py) gives each new beam its parent and token; BeamReorder gives it a slot and copies what forks take over;
StepTables (step_tables.py) then prepares the next step of the new slots.  Neither of the three needs the host, so that the loop around
a captured layer can be captured with it.  The reference decodes without beams; its per-request caches are those of
dsv4_megakernel/megakernel/test/kv_cache_manager.py:13-50.
"""
import ctypes
from dataclasses import dataclass
from typing import Tuple

import torch

from . import _lib
from . import ops as _ops
from ._lib import check, lib
from .ops import _int32, _on_current_device, _require, _stream


@dataclass
class PagedState:
    """A paged byte pool: data uint8 [pages, stride], a page holding entries_per_block x segments[0] bytes, then
    entries_per_block x segments[1] (keys, then scales); table int32 [capacity, pages] the pages of each slot.  A slot holds
    length / tokens_per_entry entries, or the last min(length, ring) of them in a ring."""
    data: torch.Tensor
    table: torch.Tensor
    entries_per_block: int
    segments: Tuple[int, ...]
    tokens_per_entry: int = 1
    ring: int = 0


class BeamReorder:
    """lengths int32 [capacity]: tokens that each slot holds; shared_lengths int32 [capacity] (or None): how many of them lie in
    pages that the slots of a group share (whole pages only; what lies behind is each slot's own).  states: contiguous
    tensors [capacity, ...] whose rows move whole (a state ring, a token history), pools: PagedState.  All are the
    caller's, on the current device; run() copies within them."""

    def __init__(self, lengths, width, *, shared_lengths=None, states=(), pools=(), status_word=None):
        _require(_on_current_device(lengths) and lengths.dtype == torch.int32 and lengths.is_contiguous() and lengths.dim() == 1,
                 "lengths must be contiguous int32 [capacity] on the current CUDA device")
        dev, capacity = lengths.device, lengths.size(0)
        _require(shared_lengths is None or (shared_lengths.device == dev and shared_lengths.dtype == torch.int32 and
                                            shared_lengths.is_contiguous() and tuple(shared_lengths.shape) == (capacity,)),
                 "shared_lengths must be contiguous int32 [capacity] on the lengths' device")
        _require(len(states) <= 8 and len(pools) <= 4, "at most 8 states and 4 pools")
        _require(status_word is None or (status_word.device == dev and status_word.dtype == torch.int32 and status_word.numel() >= 1),
                 "status_word must be int32 on the lengths' device")
        a = _lib.BeamReorderArgs(lengths=lengths.data_ptr(), num_states=len(states), num_pools=len(pools), capacity=capacity,
                                 width=_int32(width, "width"), shared_lengths=None if shared_lengths is None else shared_lengths.data_ptr())
        for i, t in enumerate(states):
            _require(t.device == dev and t.is_contiguous() and t.dim() >= 1 and t.size(0) == capacity and t.numel() > 0,
                     "state %d must be contiguous [capacity, ...] on the lengths' device" % i)
            a.states[i].data, a.states[i].row_bytes = t.data_ptr(), t.numel() // capacity * t.element_size()
        for i, q in enumerate(pools):
            _require(q.data.device == dev and q.data.dtype == torch.uint8 and q.data.dim() == 2 and q.data.is_contiguous(),
                     "pool %d must be contiguous uint8 [pages, stride] on the lengths' device" % i)
            _require(q.table.device == dev and q.table.dtype == torch.int32 and q.table.dim() == 2 and q.table.is_contiguous() and
                     q.table.size(0) == capacity, "the table of pool %d must be contiguous int32 [capacity, pages] on the lengths' device" % i)
            _require(1 <= len(q.segments) <= 2, "a page has one or two segments")
            b = a.pools[i]
            b.data, b.table, b.stride_bytes = q.data.data_ptr(), q.table.data_ptr(), q.data.size(1)
            b.num_blocks, b.table_width, b.entries_per_block = q.data.size(0), q.table.size(1), _int32(q.entries_per_block, "entries_per_block")
            for k, size in enumerate(q.segments):
                b.segment_bytes[k] = _int32(size, "a segment")
            b.tokens_per_entry, b.ring = _int32(q.tokens_per_entry, "tokens_per_entry"), _int32(q.ring, "ring")
        self.lengths, self.shared_lengths, self.states, self.pools = lengths, shared_lengths, list(states), list(pools)
        self.width, self.status_word = int(width), status_word
        self._device, self._args = dev.index, a
        self._args_ref, self._address = ctypes.byref(a), ctypes.addressof(a)
        self._status = None if status_word is None else status_word.data_ptr()
        check(lib.wuda_beam_reorder(self._args_ref, None, None, None, 0, None, None))

    def run(self, parents, slots, slots_out):
        """parents int32 [groups, width]: the beam that new beam j of a group continues (-1: none); slots int32 [groups, width]: the
        beams' request slots (-1: none).  Fills and returns slots_out int32 [groups, width], a tensor of its own: the first child
        of a beam keeps its slot, the others take the slots of beams without children, with a copy of their parent's contents.
        Lengths and page tables stay as they are (the slots of a group hold equally many tokens)."""
        if _ops._fast.beam_reorder(self._address, parents, slots, slots_out, self.width, self._device, self._status):
            return slots_out
        groups = parents.numel() // self.width
        for t, name in ((parents, "parents"), (slots, "slots"), (slots_out, "slots_out")):
            if not (t.dtype is torch.int32 and t.is_contiguous() and t.numel() == groups * self.width and t.is_cuda and
                    t.get_device() == self._device == torch._C._cuda_getDevice()):
                _require(False, "%s must be contiguous int32 [groups, %d] on the plan's device, which must be the current one" %
                         (name, self.width))
        status = lib.wuda_beam_reorder(self._args_ref, parents.data_ptr(), slots.data_ptr(), slots_out.data_ptr(), groups, self._status,
                                       _stream())
        if status:
            check(status)
        return slots_out
