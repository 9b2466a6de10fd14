"""The packed serving step: new tokens of many sequences in one tensor, over the paged KV cache.

Prism's executor gives every sequence of a call the same number of new tokens (engine/executor.py:77-130 prefills
one sequence, :320-396 decodes one token each).  A server that batches continuously mixes them: some sequences
bring a prompt chunk, the others the token they decode, all in one [tokens, ...] tensor without padding.  Per step:

    kv.prepare_append(seq_ids, num_new)
    batch = kv.build_packed_batch(seq_ids, num_new, n_heads)           # lengths, slots, work list: one upload
    for each layer:
        qkv = F.linear(rms_norm(hidden, w), qkv_w, qkv_b)              # [tokens, (n_heads + 2 n_kv) * head_dim]
        q = packed_rope_append(qkv, kv.k_caches[l], kv.v_caches[l], batch, cos, sin)
        attn = packed_attention(q, kv.k_caches[l], kv.v_caches[l], batch)
    kv.update_seqlens(seq_ids, num_new)

Calls are asynchronous on the current stream, keep nothing between them, and can be captured in a HIP graph (whose
replays then work on that very batch: its lengths are in the work list).
"""
from __future__ import annotations

import contextlib
from typing import Sequence

import numpy as np
import torch

from . import _lib
from .attention import _raw_stream, _require_gpu, status_tensor

_MAX_KEYS = 1 << 27
_captured: list[torch.Tensor] = []   # work lists that a captured graph reads (PackedBatch.release takes them out)


_here = contextlib.nullcontext()


def _on(device: torch.device):
    """Makes `device` current where it is not: kernels are launched on the current device."""
    return _here if device.type != "cuda" or device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _host_ints(x, name: str, ndim: int) -> np.ndarray:
    if isinstance(x, torch.Tensor):
        if x.device.type != "cpu":
            raise RuntimeError(f"{name} must be on the host: the step's work is laid out there")
        x = x.numpy()
    a = np.asarray(x)
    if a.size and a.dtype.kind not in "iu" or a.ndim != ndim:
        raise RuntimeError(f"{name} must be {ndim}-dimensional integers, got {a.dtype} {a.shape}")
    if a.dtype != np.int32:
        if a.size and (a.min() < -1 << 31 or a.max() > (1 << 31) - 1):
            raise RuntimeError(f"{name} must fit int32")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


class PackedBatch:
    """One step's sequences: ``new_lens[b]`` new tokens each behind ``cache_lens[b]`` cached ones, on the pages that
    row b of ``block_table`` lists (all three on the host).  Zero new tokens are allowed.

    Holds on the device, from one upload on the current stream: ``positions`` and ``slots`` (int32 [tokens]: each
    token's position and place in the cache, page * page_size + row), ``block_table`` (int32 [batch, max_blocks])
    and, for each of ``windows`` (None: every key; w: the last w keys), the attention's work list.  On another
    stream, use it behind this one, as any tensor made here; calls there keep its memory until they have run, and a
    call that a graph captures keeps it (a replay reads it, whether the batch lives or not) until ``release``.

    ``evicted[b]`` tokens of the sequence are not in the cache any more (evict_keys): its positions go on behind them.
    ``weight_rows`` other than 0 lays the batch out for packed_key_weights too: None, every new token's weights count;
    n, those of each sequence's last n.  ``weighed[b]`` of the cached keys have weights already (all, where it is not
    given).  The sequences of such a batch share no page.

    A page that a new token is written to must belong to one sequence alone, and every page that a token is written
    to or sees must be one of the pool's; columns behind them, or out of every window, may hold anything."""

    def __init__(self, new_lens, cache_lens, block_table, *, page_size: int, num_pages: int, n_heads: int, n_kv: int,
                 head_dim: int, windows: Sequence[int | None] = (None,), weight_rows: int | None = 0,
                 weighed=None, evicted=None, device: torch.device | str = "cuda"):
        device = torch.device(device)
        if device.type == "cuda":
            if device.index is None:
                device = torch.device("cuda", torch.cuda.current_device())
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a PackedBatch is uploaded from the host: build it before the capture")
        new, ctx = _host_ints(new_lens, "new_lens", 1), _host_ints(cache_lens, "cache_lens", 1)
        bt = _host_ints(block_table, "block_table", 2)
        if len(new) != len(ctx) or len(new) != bt.shape[0]:
            raise RuntimeError(f"{len(new)} new lengths, {len(ctx)} cached lengths and {bt.shape[0]} block-table rows")
        if not 0 < page_size <= _MAX_KEYS or not 0 < num_pages < 1 << 31:
            raise RuntimeError(f"{num_pages} pages of {page_size} tokens: no pool of that size")
        if head_dim not in (64, 128):
            raise RuntimeError(f"head_dim {head_dim} unsupported (64 or 128)")
        if n_kv <= 0 or n_heads <= 0 or n_heads % n_kv or n_heads > 1 << 20:
            raise RuntimeError(f"n_heads {n_heads} must be a multiple of n_kv {n_kv}")
        if not windows:
            raise RuntimeError("windows must name at least one window (None: every key)")
        for w in windows:
            if w is not None and (isinstance(w, bool) or not isinstance(w, (int, np.integer)) or not 1 <= w <= _MAX_KEYS):
                raise RuntimeError(f"window {w!r} must be None or 1 to 2^27 keys")
        if weight_rows is not None and (isinstance(weight_rows, bool) or not isinstance(weight_rows, (int, np.integer))
                                        or not 0 <= weight_rows <= _MAX_KEYS):
            raise RuntimeError(f"weight_rows {weight_rows!r} must be None (every new token) or 0 to 2^27 tokens")
        had, gone = (None if x is None else _host_ints(x, name, 1) for x, name in ((weighed, "weighed"), (evicted, "evicted")))
        for x, name in ((had, "weighed"), (gone, "evicted")):
            if x is not None and (len(x) != len(new) or (len(x) and x.min() < 0)):
                raise RuntimeError(f"{name} must have one number, not negative, for each of the {len(new)} sequences")
        self.batch, self.total_tokens = len(new), int(new.sum(dtype=np.int64))
        self.page_size, self.num_pages = page_size, num_pages
        self.n_heads, self.n_kv, self.head_dim, self.device = n_heads, n_kv, head_dim, device
        self.max_blocks = max(bt.shape[1], 1)
        lib, total = _lib.load(), self.total_tokens
        lengths = (new.ctypes.data, ctx.ctypes.data, self.batch)
        if total * n_heads > 1 << 30:
            raise RuntimeError(f"{total} tokens of {n_heads} heads: more than 2^30 query rows")
        where = np.empty((2, max(total, 0)), np.int32)
        widest = 0 if any(w is None for w in windows) else max(windows)
        _lib.check(lib.pkv_packed_layout(*lengths, bt.ctypes.data, bt.shape[1], bt.shape[1], page_size, num_pages, widest,
                                         where[0].ctypes.data, where[1].ctypes.data), "pkv_packed_layout")
        if gone is not None and total > 0:
            if any(w is not None for w in windows) and (gone[new > 0] > 0).any():
                raise RuntimeError("a window counts positions, which an evicted sequence's cached keys do not have any more")
            if int((ctx.astype(np.int64) + new + gone).max()) > _MAX_KEYS:
                raise RuntimeError("cached, new and evicted tokens of a sequence: at most 2^27 together")
            where[0] += np.repeat(gone, new)
        cus = torch.cuda.get_device_properties(device).multi_processor_count if device.type == "cuda" else 256
        plans = {w: self._plan(lengths, w, cus) for w in dict.fromkeys(windows)}
        weight_plans = {}
        if weight_rows != 0:
            self._check_apart(new, ctx, had, bt, widest, int(weight_rows or 0))
            weight_plans = {w: self._weight_plan(lengths, had, w, int(weight_rows or 0), cus) for w in plans}
        parts = [where[0], where[1], bt.ravel()] + [a.ravel() for items, merges, _ in plans.values() for a in (items, merges)]
        after = len(parts)
        parts += [items.ravel() for items, _ in weight_plans.values()]
        starts = np.cumsum([0] + [-(-p.size // 4) * 4 for p in parts])     # 16-byte aligned
        staged = torch.empty(int(starts[-1]) + 4, dtype=torch.int32, pin_memory=device.type == "cuda")
        host = staged.numpy()
        for p, at in zip(parts, starts):
            host[at:at + p.size] = p
        self._stream = _raw_stream(device.index) if device.type == "cuda" else 0
        with _on(device):
            self._buf = staged.to(device, non_blocking=True)
        view = [self._buf[at:at + p.size] for p, at in zip(parts, starts)]
        self.positions, self.slots = view[0], view[1]
        self.block_table = view[2].view(self.batch, bt.shape[1])
        # per window: the kernels' arguments (window, items, their number, merges, their number, partials, merge rows)
        base = self._buf.data_ptr()
        self._plans = {w: (int(w or 0), base + 4 * int(starts[3 + 2 * i]), len(items), base + 4 * int(starts[4 + 2 * i]),
                           len(merges), int(counts[2]), int(counts[3]))
                       for i, (w, (items, merges, counts)) in enumerate(plans.items())}
        # the same for the weights: window, items, the number of each of their lists, partials
        self._weight_plans = {w: (int(w or 0), base + 4 * int(starts[after + i]), *map(int, counts))
                              for i, (w, (_, counts)) in enumerate(weight_plans.items())}
        self._captured = False
        self._native = _lib.fast().new_batch(self._buf, total, self.batch, n_heads, n_kv, head_dim, page_size, num_pages,
                                             self.max_blocks, self.positions.data_ptr(), self.slots.data_ptr(),
                                             base + 4 * int(starts[2]))

    def _used_on(self, stream: int) -> None:
        """A call on `stream` will read the batch's memory."""
        if torch._C._cuda_isCurrentStreamCapturing():
            if not self._captured:
                _captured.append(self._buf)
                self._captured = True
        elif stream != self._stream:
            self._buf.record_stream(torch.cuda.current_stream(self.device))

    def release(self) -> None:
        """Lets go of the memory that captured calls kept, which then lives as long as the batch.  For a batch whose
        graphs are gone, or were captured again with another: none of their replays may run now or later."""
        _captured[:] = [buf for buf in _captured if buf is not self._buf]
        self._captured = False

    def _plan(self, lengths, window, cus):
        lib = _lib.load()
        counts = np.zeros(4, np.int32)
        sizes = (*lengths, self.n_heads, self.n_kv, self.head_dim, int(window or 0), cus)
        # enough for a block per 128 query rows and sequence and two ranges per workgroup; asked for where it is not
        g = self.n_heads // self.n_kv
        room = self.total_tokens * g // 128 + self.batch + 4 * max(2 * cus // self.n_kv, 1)
        while True:
            items, merges = np.empty((room, 12), np.int32), np.empty((room, 8), np.int32)
            rc = lib.pkv_packed_plan(*sizes, items.ctypes.data, room, merges.ctypes.data, room, counts.ctypes.data)
            if rc != _lib.PKV_ENOSPC:
                break
            room = int(counts[:2].max())
        _lib.check(rc, "pkv_packed_plan")
        return items[:counts[0]], merges[:counts[1]], counts


    def _weight_plan(self, lengths, weighed, window, rows, cus):
        lib = _lib.load()
        counts = np.zeros(4, np.int32)
        sizes = (*lengths[:2], 0 if weighed is None else weighed.ctypes.data, self.batch, self.n_heads, self.n_kv,
                 int(window or 0), rows, cus)
        _lib.check(lib.pkv_key_weights_plan(*sizes, 0, 0, counts.ctypes.data), "pkv_key_weights_plan")
        items = np.empty((int(counts[:3].sum()), 12), np.int32)
        if len(items):
            _lib.check(lib.pkv_key_weights_plan(*sizes, items.ctypes.data, len(items), counts.ctypes.data),
                       "pkv_key_weights_plan")
        return items, counts

    def _check_apart(self, new, ctx, weighed, bt, widest, rows):
        """The pages whose keys get weights belong to one sequence each: a key's sum is nobody else's."""
        end = ctx.astype(np.int64) + new
        first = np.zeros_like(end)
        if widest > 0:
            count = np.minimum(new, rows) if rows > 0 else new
            first = np.minimum(np.maximum(end - count - widest + 1, 0), ctx if weighed is None else np.minimum(weighed, ctx))
        col = np.arange(bt.shape[1])[None]
        used = bt[(new > 0)[:, None] & (col >= (first // self.page_size)[:, None]) & (col < (-(-end // self.page_size))[:, None])]
        used = used[used >= 0]
        if len(np.unique(used)) < len(used):
            raise RuntimeError("two sequences of the batch share a page (or one is in it twice): their keys' weights "
                               "cannot be taken in one step")


def packed_rope_append(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, batch: PackedBatch,
                       cos: torch.Tensor, sin: torch.Tensor, *, interleaved: bool = False,
                       q_norm_w: torch.Tensor | None = None, k_norm_w: torch.Tensor | None = None, eps: float = 1e-6,
                       positions: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                       status: torch.Tensor | None = None) -> torch.Tensor:
    """QKV split, optional RMSNorm of every query and key head, rotation and paged append of a packed batch, in one
    launch: ``qkv`` [tokens, (n_heads + 2 n_kv) * head_dim] bf16 -> the rotated queries [tokens, n_heads,
    head_dim]; the rotated keys and the values go to the batch's slots of the cache.

    ``cos`` / ``sin`` are fp32 [n_pos, rotary_dim / 2] (rotary_tables); rotary_dim, a multiple of 16, may be less
    than the head.  A token turns by its place in its sequence, or by ``positions`` (int32 [tokens]) where they
    differ.  Rows of ``qkv`` and ``q_out`` behind the batch's tokens are not touched (zero in a result made here)."""
    dev = batch.device
    _require_gpu(qkv, "qkv")
    stream = _raw_stream(dev.index)
    with _on(dev):
        batch._used_on(stream)
        return _lib.fast().packed_rope_append(qkv, k_cache, v_cache, batch._native, cos, sin, interleaved, q_norm_w,
                                              k_norm_w, eps, positions, q_out,
                                              status if status is not None else status_tensor(dev), stream)


def packed_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, batch: PackedBatch, *,
                     window: int | None = None, sinks: torch.Tensor | None = None, softmax_scale: float | None = None,
                     return_lse: bool = False, out: torch.Tensor | None = None, status: torch.Tensor | None = None):
    """Causal attention of a packed batch's tokens over their sequences' pages (the new keys and values are in the
    cache already: packed_rope_append): ``q`` [tokens, n_heads, head_dim] bf16 -> out of its shape.

    A token sees its sequence up to itself, with ``window`` the last that many keys (one of the windows the batch
    was laid out for).  ``sinks`` (fp32 [n_heads]) adds exp(sinks[h]) to each row's softmax denominator.
    ``softmax_scale`` defaults to 1/sqrt(head_dim).  With ``return_lse`` also the natural logarithm of the
    denominators, fp32 [tokens, n_heads].  Rows of ``q`` and ``out`` behind the batch's tokens are not touched
    (zero in results made here)."""
    dev = batch.device
    _require_gpu(q, "q")
    plan = batch._plans.get(window)
    if plan is None:
        raise RuntimeError(f"the batch was laid out for the windows {list(batch._plans)}, not {window}")
    stream = _raw_stream(dev.index)
    with _on(dev):
        batch._used_on(stream)
        return _lib.fast().packed_attention(q, k_cache, v_cache, batch._native, plan, sinks, softmax_scale, return_lse,
                                            out, status if status is not None else status_tensor(dev), stream)


def packed_key_weights(q: torch.Tensor, k_cache: torch.Tensor, lse: torch.Tensor, key_weights: torch.Tensor,
                       batch: PackedBatch, *, window: int | None = None, softmax_scale: float | None = None,
                       status: torch.Tensor | None = None) -> torch.Tensor:
    """Adds to ``key_weights`` (fp32 [num_pages, n_kv, page_size], the cache's pages) the attention weight that every
    cached key got from the batch's new tokens, summed over them and over the query heads of each KV head, and
    returns it: what evict_keys goes by.

    ``q``, ``window`` and ``softmax_scale`` are packed_attention's, and ``lse`` (fp32 [tokens, n_heads]) what it
    returned with ``return_lse``.  Which tokens count, and which keys start from nothing (this step's own), the batch
    knows: it was laid out with ``weight_rows``.  A row whose lse is infinite weighs nothing
    (its scores being finite)."""
    dev = batch.device
    _require_gpu(q, "q")
    plan = batch._weight_plans.get(window)
    if plan is None:
        raise RuntimeError("the batch was laid out without weight_rows" if not batch._weight_plans else
                           f"the batch was laid out for the windows {list(batch._weight_plans)}, not {window}")
    stream = _raw_stream(dev.index)
    with _on(dev):
        batch._used_on(stream)
        return _lib.fast().packed_key_weights(q, k_cache, lse, key_weights, batch._native, plan, softmax_scale,
                                              status if status is not None else status_tensor(dev), stream)
