"""Slot maps of a batch's new tokens, built on the device from its lengths (C
ABI ``akv_map_slots``).

The reference's scheduler allocates the slots of a forward's new tokens and
writes them into ``req_to_token`` from Python
(akv/system/sglang.patch:3133-3180).  ``SlotMapper.run`` does it in one launch
for device-resident lengths and a device free list (``FreeSlotRing``, the one
the Drop pushes its freed slots on): the slot and the position of every new
token, the row entries, and, where asked, block tables for a paged reader and
the ancestor masks of drafted token trees for ``context_tree.TreeAttention``.

A verification step lends its pages (``commit=False``): the ring keeps them,
and the next call gives them out again, so rejected tokens cost nothing.  A
prompt chunk or a plain decode step takes them (``commit=True``).  To take
what a verification accepted, call again with the accepted counts and
``commit=True`` and move the accepted tokens' K/V from the slots that were lent
to the ones given now, all reads of a pool before its writes: they differ
where a tree's path skips nodes, and for every request behind one that accepted
fewer tokens than it drafted.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _native

TREE_NODES = 64  # new tokens per request with a tree: one 64-bit mask word each


@dataclass
class SlotMap:
    """Device views of one call (the mapper's buffers: the next call
    overwrites them).  New tokens lie in request order, request b's in
    [new_offsets[b], new_offsets[b + 1])."""

    new_offsets: torch.Tensor   # int32 [batch + 1]
    slots: torch.Tensor         # int32 [max_new_tokens]; -1: none given out, or behind the last token
    positions: torch.Tensor     # int32 [max_new_tokens]; 0 behind the last token
    tree_mask: torch.Tensor | None  # int64 [max_new_tokens], with parents; not written behind them
    block_table: torch.Tensor | None
    totals: torch.Tensor        # int32 [2]: new tokens, pages taken or lent
    status: torch.Tensor        # int32 [1]: AKV_SLOTS_* bits

    ERRORS = {
        _native.SLOTS_RING_UNDERFLOW: "not enough free pages in the ring",
        _native.SLOTS_CAPACITY: "more new tokens than max_new_tokens",
        _native.SLOTS_BAD_REQUEST: "a request's row or lengths are out of range",
        _native.SLOTS_BAD_PAGE: "a row's last slot is not at its offset of a page",
        _native.SLOTS_BAD_PARENT: "a draft token's parent is not an earlier token",
    }

    def check(self):
        """Raise RuntimeError if the call set a status bit (synchronises)."""
        bits = int(self.status.item())
        if bits:
            why = "; ".join(msg for bit, msg in self.ERRORS.items() if bits & bit)
            raise RuntimeError(f"slot map: {why}")


_fields, _INT32, _INT64 = _native.fields, _native.INT32, _native.INT64


class SlotMapper:
    """Outputs are allocated once, for up to ``max_batch`` requests with
    ``max_new_tokens`` new tokens in all; a call allocates nothing, so it can
    be captured in a CUDA graph.  Calls of one mapper, replays of its graphs
    among them, share its buffers and must not overlap on the device."""

    def __init__(self, max_batch, max_new_tokens, device, *, page_size=1):
        if page_size != 1 and (page_size < 4 or page_size > 128 or page_size & (page_size - 1)):
            raise ValueError("page_size must be 1 or a power of two from 4 to 128")
        if not 0 < max_batch <= 65535 or not 0 <= max_new_tokens < 2**31:
            raise ValueError("slot maps hold 1 to 65535 requests and fewer than 2^31 new tokens")
        device = torch.device(device)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device, self._index = device, device.index
        self.max_batch, self.max_new_tokens = int(max_batch), int(max_new_tokens)
        self.page_size = int(page_size)

        def vector(n, dtype=torch.int32):
            return torch.zeros(n, dtype=dtype, device=device)

        self._offsets = vector(self.max_batch + 1)
        self._slots, self._positions = vector(self.max_new_tokens), vector(self.max_new_tokens)
        self._slots.fill_(-1)
        self._mask = vector(self.max_new_tokens, torch.int64)
        self._totals, self._status, self._work = vector(2), vector(1), vector(2)
        self._outputs = tuple(t.data_ptr() for t in (self._offsets, self._slots, self._positions,
                                                     self._mask))
        self._words = tuple(t.data_ptr() for t in (self._totals, self._status, self._work))

    def run(self, req_to_token, row_ids, raw_lens, new_lens, ring, *, next_positions=None,
            parents=None, block_table=None, commit=True, keep_offsets=False) -> SlotMap:
        """``req_to_token`` int32 [rows, columns]; ``row_ids``, ``raw_lens`` (columns
        in use) and ``new_lens`` int32 or int64 [batch]; ``ring`` a
        ``FreeSlotRing`` of page ids (slots at page_size 1).
        ``next_positions``: the position of each request's first new token,
        the Drop's ``next_position`` (default ``raw_lens``).  ``parents``:
        int32 [>= max_new_tokens], for each new token the parent's number in the
        request or -1 (at most 64 new tokens per request); positions then follow
        the depth.  A row whose last page a Drop has freed (all of its tokens
        dropped) is passed with ``raw_lens`` rounded up to whole pages, or the
        new tokens would go on in that page.  ``block_table``: int32 [>= batch, columns], filled with the
        page ids of whole rows.  A request whose row or lengths are out of range (one that no longer
        fits its row, say) counts as one without new tokens, and the entries of those behind it
        move up; with ``keep_offsets`` it keeps its entries, without slots, which is what tokens
        need that are laid out by the caller's own lengths (a length that is itself out of range
        then refuses the call).  Two requests of one call must not share a
        row, unless at most one of them has new tokens and the other's columns end before them.
        Failures that only the device sees are bits of ``status`` (``SlotMap.check``)."""
        index = self._index
        (rows_ptr, rows_dev, rows_dt, batch, rows_step, raw_ptr, raw_dev, raw_dt, n_raw, raw_step,
         new_ptr, new_dev, new_dt, n_new, new_step, free_ptr, free_dev, free_dt, free_n, free_step,
         state_ptr, state_dev, state_dt, state_n, state_step) = _fields(
             1, row_ids, raw_lens, new_lens, ring.ring, ring.state)
        if batch > self.max_batch:
            raise ValueError("batch exceeds max_batch")
        if n_raw != batch or n_new != batch or not rows_dev == raw_dev == new_dev == index or \
                (batch > 1 and not rows_step == raw_step == new_step == 1):
            raise ValueError("row_ids, raw_lens and new_lens must be contiguous vectors of one "
                             "entry per request, on the mapper's device")
        for dt in (rows_dt, raw_dt, new_dt):
            if dt != _INT32 and dt != _INT64:
                raise ValueError("row_ids, raw_lens and new_lens must be int32 or int64")
        if free_dev != index or state_dev != index or free_n < ring.capacity or state_n < 2 or \
                free_dt != _INT32 or state_dt != _INT64 or state_step != 1 or \
                (free_step != 1 and free_n > 1):
            raise ValueError("the free ring must be contiguous int32 entries, with an int64 state, "
                             "on the mapper's device")
        table, dev, dt, rows, columns, row_stride, unit = _fields(2, req_to_token)
        if dt != _INT32 or unit != 1 or dev != index:
            raise ValueError("req_to_token must be int32 [rows, columns] with unit last stride, "
                             "on the mapper's device")
        next_ptr = next64 = parents_ptr = table_ptr = table_stride = table_columns = 0
        if next_positions is not None:
            next_ptr, dev, dt, n, step = _fields(1, next_positions)
            if n != batch or dev != index or (step != 1 and n > 1) or \
                    (dt != _INT32 and dt != _INT64):
                raise ValueError("next_positions must be a contiguous int32 or int64 vector of "
                                 "one entry per request, on the mapper's device")
            next64 = 1 if dt == _INT64 else 0
        if parents is not None:
            parents_ptr, dev, dt, n, step = _fields(1, parents)
            if dt != _INT32 or dev != index or n < self.max_new_tokens or (step != 1 and n > 1):
                raise ValueError("parents must be a contiguous int32 vector of max_new_tokens "
                                 "entries on the mapper's device")
        if block_table is not None:
            table_ptr, dev, dt, n, table_columns, table_stride, unit = _fields(2, block_table)
            if dt != _INT32 or unit != 1 or n < batch or dev != index:
                raise ValueError("block_table must be int32 [>= batch, columns] with unit last "
                                 "stride, on the mapper's device")
        offsets = self._offsets if batch == self.max_batch else self._offsets[: batch + 1]
        result = SlotMap(offsets, self._slots, self._positions,
                         self._mask if parents is not None else None, block_table, self._totals,
                         self._status)
        if batch == 0:
            self._slots.fill_(-1)
            for t in (self._positions, result.new_offsets, result.totals, result.status):
                t.zero_()
            return result
        status = _native.launch(index, _native.lib.akv_map_slots, _native.MAP_SLOTS.pack(
            table, row_stride, rows, columns, rows_ptr, 1 if rows_dt == _INT64 else 0, raw_ptr,
            1 if raw_dt == _INT64 else 0, new_ptr, 1 if new_dt == _INT64 else 0, batch,
            self.page_size, free_ptr, state_ptr, ring.capacity, next_ptr, next64, parents_ptr,
            self.max_new_tokens, *self._outputs, table_ptr, table_stride, table_columns,
            *self._words,
            (1 if commit else 0) + (_native.SLOTS_KEEP_OFFSETS if keep_offsets else 0)))
        _native.check(status, "map_slots")
        return result
