"""Attention of drafted token trees over the paged cache (C ABI
``akv_tree_attention``).

Speculative decoding verifies, in one forward, a tree of drafted tokens per
request: each sees the request's cached keys and, among the drafted tokens,
itself and its ancestors.  The reference's runtime hands such a step to its
native backends with a dense mask over all keys; ``TreeAttention`` takes the
same paged inputs as ``DecodeAttention`` plus the drafted tokens' slots and one
64-bit mask word per token (``context_slots.SlotMapper`` makes both).

Like ``DecodeAttention``, ``plan`` cuts the batch into a work list on the host
(one pinned copy to the device) and ``run`` launches on the current stream
without host synchronisation: one kernel, and a second one that joins the
pieces of requests that were cut.  A captured run follows later plans.
"""

from __future__ import annotations

import math

import numpy as np
import torch

from . import _native

MAX_DRAFT = 64      # drafted tokens per request: bits of a mask word
TILE_ROWS = 128     # rows (drafted token x query head of the group) per tile
TILE_KEYS = 128
UNITS = int(_native.lib.akv_tree_attention_units())
MIN_TILES = 1       # key tiles per CTA, if the batch has as many


def tree_work_list(kv_indptr, draft_indptr, group, num_kv_heads, pair_heads, ctas,
                   min_tiles=MIN_TILES):
    """(items int32 [n, 12], cta_items int32 [ctas + 1], merges int32 [m, 8],
    partials) of a batch, as ``akv_tree_attention`` reads them.

    A CTA has two units.  A pair of (KV head, row tile)s over the same key
    tiles is one group: two heads of a request whose rows fill one tile (with
    ``pair_heads``), or two row tiles of one head; what is left over is a
    single, whose key tiles the units share out, at half the cost per tile.
    The key tiles of all groups, one after another, are cut into runs of equal
    cost, one per CTA; a group whose tiles fall to several CTAs gets a partial
    result for each and one merge."""
    kv, dr = np.asarray(kv_indptr, np.int64), np.asarray(draft_indptr, np.int64)
    if kv.ndim != 1 or kv.shape != dr.shape or len(kv) < 1 or kv[0] < 0 or dr[0] < 0:
        raise ValueError("kv_indptr and draft_indptr must be CSR offsets of one batch")
    prefix, n = np.diff(kv), np.diff(dr)
    if np.any(prefix < 0) or np.any(n < 0):
        raise ValueError("kv_indptr and draft_indptr must not decrease")
    # Numbers of keys and tokens, the end of a request's last tile included, are 32 bits.
    if kv[-1] + MAX_DRAFT + TILE_KEYS >= 2**31 or dr[-1] + MAX_DRAFT >= 2**31:
        raise ValueError("the batch has 2^31 keys or more, or a request's last tile passes them")
    if n.size and n.max() > MAX_DRAFT:
        raise ValueError(f"a request has more than {MAX_DRAFT} drafted tokens")
    row_tiles = -(-n * group // TILE_ROWS)
    by_head = (row_tiles == 1) & bool(pair_heads)
    # Groups of a request: over its heads in pairs, or per head over its row tiles in pairs.
    per_head = np.where(by_head, 1, -(-row_tiles // 2))
    groups = np.where(by_head, -(-num_kv_heads // 2), num_kv_heads * per_head)
    req = np.repeat(np.arange(len(n)), groups)
    local = np.arange(len(req)) - np.repeat(np.cumsum(groups) - groups, groups)
    heads = by_head[req]
    head = np.where(heads, 2 * local, local // per_head[req].clip(1))
    tile = np.where(heads, 0, 2 * (local % per_head[req].clip(1)))
    pair = np.where(heads, head + 1 < num_kv_heads, tile + 1 < row_tiles[req])
    tiles = -(-(prefix + n) // TILE_KEYS)[req]
    tile_end, weight = np.cumsum(tiles), 1 + pair
    cost_end = np.cumsum(tiles * weight)
    total, cost = (int(tile_end[-1]), int(cost_end[-1])) if len(req) else (0, 0)
    ctas = min(int(ctas), -(-total // max(1, min_tiles)))
    bounds = (np.arange(ctas + 1) * cost) // max(1, ctas)
    if ctas:
        g = np.minimum(np.searchsorted(cost_end, bounds, side="right"), len(req) - 1)
        at = (bounds - (cost_end[g] - tiles[g] * weight[g])) // weight[g]
        # A cut one tile off a group's end moves there: a piece of one tile
        # costs more (its own start, a partial result, a merge) than it evens.
        at = np.where((at == 1) & (tiles[g] > 1), 0, at)
        at = np.where((at == tiles[g] - 1) & (tiles[g] > 2), tiles[g], at)
        bounds = tile_end[g] - tiles[g] + at
    cuts = np.unique(np.concatenate((bounds, tile_end, [0])))
    first, last = cuts[:-1], cuts[1:]
    g = np.searchsorted(tile_end, first, side="right")
    r = req[g]
    begin = first - (tile_end[g] - tiles[g])
    items = np.zeros((len(g), 12), np.int64)
    items[:, 0], items[:, 1], items[:, 2], items[:, 3] = dr[r], n[r], kv[r], prefix[r]
    items[:, 4] = begin * TILE_KEYS
    items[:, 5] = np.minimum((begin + last - first) * TILE_KEYS, prefix[r] + n[r])
    items[:, 6], items[:, 7] = head[g], tile[g]
    items[:, 8], items[:, 9] = pair[g] & heads[g], pair[g] & ~heads[g]
    items[:, 10] = weight[g]
    pieces = np.bincount(g, minlength=len(req))
    cut = pieces[g] > 1
    items[:, 11] = np.where(cut, (np.cumsum(cut) - 1) * UNITS, -1)
    lead = cut & np.concatenate(([True], g[1:] != g[:-1])) if len(g) else cut
    m = items[lead]
    merges = np.zeros((len(m), 8), np.int64)
    merges[:, :4] = m[:, [0, 1, 6, 7]]
    merges[:, 4] = m[:, 8] | m[:, 9] << 1 | m[:, 10] << 2
    merges[:, 5], merges[:, 6] = m[:, 11], pieces[g[lead]]
    cta_items = np.searchsorted(first, bounds).astype(np.int32)
    return items.astype(np.int32), cta_items, merges.astype(np.int32), int(cut.sum()) * UNITS


_fields, _INT32, _INT64 = _native.fields, _native.INT32, _native.INT64


class TreeAttention:
    """Plans and partial results live in the instance: runs of one instance,
    replays of its graphs among them, must not overlap on the device.

    A captured run launches the instance's largest grid and takes everything
    else from the plan that the device holds when it replays, so a graph
    serves any later ``plan`` (on the replaying stream) whose tokens and keys fit in the
    tensors that were passed to it: pass vectors with room for a cache that
    grows, and ``out``.  A plan that does not fit is reported by ``check``."""

    def __init__(self, num_q_heads, num_kv_heads, head_dim, max_batch, device, *,
                 dtype=torch.bfloat16, sm_scale=None, ctas=None):
        if num_kv_heads <= 0 or num_q_heads <= 0 or num_q_heads % num_kv_heads:
            raise ValueError("tree attention needs num_q_heads a multiple of num_kv_heads")
        if head_dim not in (64, 128):
            raise ValueError("tree attention supports head_dim 64 and 128")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("tree attention runs on bf16 or fp16")
        if max_batch <= 0 or (ctas is not None and ctas <= 0):
            raise ValueError("max_batch and ctas must be positive")
        if sm_scale is not None and not 1e-30 < sm_scale < 1e30:
            raise ValueError("sm_scale must be positive and an ordinary fp32 number")
        device = torch.device(device)
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device, self._index, self.dtype = device, device.index, dtype
        self.hq, self.hkv, self.d = num_q_heads, num_kv_heads, head_dim
        self.group = num_q_heads // num_kv_heads
        self.sm_scale = 1.0 / math.sqrt(head_dim) if sm_scale is None else float(sm_scale)
        self.max_batch = int(max_batch)
        # Two heads' rows of head_dim 64 are 256 bytes a key, as one head's of 128.
        self.pair_heads = head_dim == 64
        if ctas is None:
            ctas = torch.cuda.get_device_properties(device).multi_processor_count
        self.ctas = int(ctas)
        # Every CTA boundary cuts at most one group.
        row_tiles = -(-MAX_DRAFT * self.group // TILE_ROWS)
        groups = self.hkv * -(-row_tiles // 2)
        self.max_items = self.max_batch * groups + self.ctas
        self.max_merges = min(self.max_batch * groups, self.ctas)
        partials = 2 * self.ctas * UNITS
        # The device's plan: cta_items, merges and items, so that one copy of a
        # prefix brings it.  Entries past a plan's CTAs hold no item and those past its
        # merges join nothing: what a run launches beyond them has no work.
        self._at = (self.ctas + 1, self.ctas + 1 + 8 * self.max_merges)
        size = self._at[1] + 12 * self.max_items
        self._host = torch.zeros(size, dtype=torch.int32, pin_memory=True)
        self._host_np = self._host.numpy()
        self._dev = torch.zeros(size, dtype=torch.int32, device=device)
        self._acc = torch.empty((partials, TILE_ROWS, head_dim), dtype=torch.float32, device=device)
        self._ml = torch.empty((partials, TILE_ROWS, 2), dtype=torch.float32, device=device)
        # Error bits, kept until check().
        self.error_flag = torch.zeros(1, dtype=torch.int32, device=device)
        self._plan_ptr, self._flag_ptr = self._dev.data_ptr(), self.error_flag.data_ptr()
        self._partial_ptrs = self._acc.data_ptr(), self._ml.data_ptr()
        self._code = _native.DTYPE_CODE[dtype]
        self._copied = torch.cuda.Event()
        self._copied.record(torch.cuda.current_stream(device))
        self.tokens = self.keys = self.n_ctas = self.n_merges = 0

    def plan(self, kv_indptr_host, draft_indptr_host):
        """Work list from the host-known CSR offsets of the cached keys and of
        the drafted tokens (at most ``MAX_DRAFT`` per request), copied on the
        current stream: runs and replays follow it there."""
        if len(kv_indptr_host) - 1 > self.max_batch:
            raise ValueError("batch exceeds max_batch")
        items, cta_items, merges, partials = tree_work_list(
            kv_indptr_host, draft_indptr_host, self.group, self.hkv, self.pair_heads, self.ctas)
        assert len(items) <= self.max_items and len(merges) <= self.max_merges and \
            partials <= len(self._acc)
        self._copied.synchronize()
        host, (m, i) = self._host_np, self._at
        used = i + items.size
        host[: len(cta_items)], host[len(cta_items): m] = cta_items, cta_items[-1]
        host[m: m + merges.size], host[m + merges.size: i] = merges.reshape(-1), 0
        host[i: used] = items.reshape(-1)
        stream = torch.cuda.current_stream(self.device)
        with torch.cuda.stream(stream):
            self._dev[:used].copy_(self._host[:used], non_blocking=True)
            self._copied.record(stream)
        self.tokens, self.keys = int(draft_indptr_host[-1]), int(kv_indptr_host[-1])
        self.n_ctas, self.n_merges = len(cta_items) - 1, len(merges)
        return self

    def run(self, q, k_pool, v_pool, kv_indices, draft_slots, tree_mask, sinks=None, window=None,
            q_positions=None, kv_positions=None, out=None, return_lse=False):
        """``q`` [drafted tokens, Hq, D]; pools [slots, Hkv, D]; ``kv_indices`` int32
        [cached keys] and ``draft_slots`` int32 [drafted tokens], a negative
        draft slot for a padding token (read as zeros); ``tree_mask`` int64
        [drafted tokens]: bit j set for a visible drafted token j of the
        request.  A token that sees no key gets zeros (and lse -inf, or the
        sink).  ``window`` (None or negative: none) hides keys with
        q_position - kv_position > window and needs both position vectors
        (int32; those of the drafted keys are ``q_positions``).  Rows of
        ``out`` past the planned tokens are left as they were; ``out`` may be ``q``.

        The head's maximum, sum and accumulator are fp32; P is rounded to the
        pools' type for P.V.  Returns out, or (out, lse fp32 [tokens, Hq])."""
        index, tokens, keys, hq, hkv, d = (self._index, self.tokens, self.keys, self.hq, self.hkv,
                                           self.d)
        (q_ptr, q_dev, q_dt, n, heads, dim, q_token, q_head, q_unit, k_ptr, k_dev, k_dt, k_slots,
         k_heads, k_dim, k_slot, k_head, k_unit, v_ptr, v_dev, v_dt, v_slots, v_heads, v_dim,
         v_slot, v_head, v_unit) = _fields(3, q, k_pool, v_pool)
        code = _native.FIELD_CODE.get(q_dt)
        if code != self._code or n < tokens or heads != hq or dim != d or q_unit != 1 or \
                q_dev != index:
            raise ValueError("q must be [>= tokens, num_q_heads, head_dim] of the planned type "
                             "with unit last stride, on the plan's device")
        if k_dt != q_dt or v_dt != q_dt or k_heads != hkv or v_heads != hkv or k_dim != d or \
                v_dim != d or k_unit != 1 or v_unit != 1 or k_dev != index or v_dev != index:
            raise ValueError("KV pools must be [slots, num_kv_heads, head_dim] of the planned type "
                             "with unit last stride, on the plan's device")
        (kv_ptr, kv_dev, kv_dt, kv_n, kv_step, draft_ptr, draft_dev, draft_dt, draft_n, draft_step,
         mask_ptr, mask_dev, mask_dt, mask_n, mask_step) = _fields(1, kv_indices, draft_slots,
                                                                   tree_mask)
        if kv_n < keys or draft_n < tokens or mask_n < tokens or kv_dt != _INT32 or \
                draft_dt != _INT32 or mask_dt != _INT64 or \
                not kv_dev == draft_dev == mask_dev == index or (kv_step != 1 and kv_n > 1) or \
                (draft_step != 1 and draft_n > 1) or (mask_step != 1 and mask_n > 1):
            raise ValueError("kv_indices (int32), draft_slots (int32) and tree_mask (int64) must "
                             "be contiguous vectors of the plan's lengths, on its device")
        if draft_n < n:
            n = draft_n
        if mask_n < n:
            n = mask_n  # tokens that the vectors hold
        window = -1 if window is None or window < 0 else int(window)
        dev = self._plan_ptr
        q_pos = kv_pos = sinks_ptr = lse_ptr = 0
        if window >= 0:
            if q_positions is None or kv_positions is None:
                raise ValueError("a window needs q_positions and kv_positions")
            (q_pos, dev0, dt0, n0, step0, kv_pos, dev1, dt1, n1,
             step1) = _fields(1, q_positions, kv_positions)
            if n0 < tokens or n1 < keys or not dt0 == dt1 == _INT32 or \
                    not dev0 == dev1 == index or (step0 != 1 and n0 > 1) or (step1 != 1 and n1 > 1):
                raise ValueError("q_positions and kv_positions must be contiguous int32 vectors "
                                 "of the plan's lengths, on its device")
            kv_pos = kv_pos or dev
            if n1 < kv_n:
                kv_n = n1
            if n0 < n:
                n = n0
        if sinks is not None:
            sinks_ptr, dev0, dt0, n0, step0 = _fields(1, sinks)
            if n0 != hq or _native.FIELD_CODE.get(dt0) != _native.AKV_F32 or dev0 != index or \
                    (step0 != 1 and n0 > 1):
                raise ValueError("sinks must be fp32 [num_q_heads] on the plan's device")
        if out is None:
            out = torch.empty((tokens, hq, d), dtype=self.dtype, device=self.device)
        o_ptr, o_dev, o_dt, o_n, heads, dim, o_token, o_head, unit = _fields(3, out)
        if o_n < tokens or heads != hq or dim != d or unit != 1 or o_dev != index or o_dt != q_dt:
            raise ValueError("out must be [>= tokens, num_q_heads, head_dim] of the planned type "
                             "with unit last stride, on the plan's device")
        lse = None
        if return_lse:
            lse = torch.empty((tokens, self.hq), dtype=torch.float32, device=self.device)
            lse_ptr, n = lse.data_ptr(), tokens
        if o_n < n:
            n = o_n
        n_ctas, n_merges = self.n_ctas, self.n_merges
        if n and _native.capturing(index):
            n_ctas, n_merges = self.ctas, self.max_merges
        status = _native.launch(index, _native.lib.akv_tree_attention, _native.TREE_ATTENTION.pack(
            q_ptr, q_token, q_head, k_ptr, v_ptr, k_slot, k_head, v_slot, v_head,
            k_slots if k_slots < v_slots else v_slots, code, n, kv_n, kv_ptr or dev,
            draft_ptr, mask_ptr, q_pos, kv_pos, window, sinks_ptr, self.sm_scale, hq, hkv, d,
            dev + 4 * self._at[1], dev, n_ctas, dev + 4 * self._at[0], n_merges,
            *self._partial_ptrs, o_ptr, o_token, o_head, lse_ptr, self._flag_ptr))
        _native.check(status, "tree_attention")
        return (out, lse) if return_lse else out

    ERRORS = {1: "a key slot outside the KV pools was read as slot 0",
              2: "a wait inside the kernel ran out; the output of that launch is invalid",
              4: "a captured run was replayed on a plan of more tokens or keys than its "
                 "tensors hold"}

    def check(self):
        """Raise RuntimeError if a launch since the last check reported an
        error, and clear the error bits (synchronises)."""
        bits = int(self.error_flag[0].item())
        if bits:
            self.error_flag[0].zero_()
            why = "; ".join(msg for bit, msg in self.ERRORS.items() if bits & bit)
            raise RuntimeError(f"tree attention: {why}")
