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
import math
from typing import Sequence

import numpy as np
import torch

from . import _lib
from .attention import _BF16, _check_cache, _raw_stream, _require_gpu, status_tensor

_MAX_KEYS = 1 << 27


def _on(device: torch.device):
    """Makes `device` current where it is not: kernels are launched on the current device."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _host_ints(x, name: str, ndim: int) -> np.ndarray:
    if isinstance(x, torch.Tensor):
        if x.device.type != "cpu":
            raise RuntimeError(f"{name} must be on the host: the step's work is laid out there")
        x = x.numpy()
    a = np.asarray(x)
    if a.size == 0:
        a = a.astype(np.int64)
    if a.ndim != ndim or a.dtype.kind not in "iu":
        raise RuntimeError(f"{name} must be {ndim}-dimensional integers, got {a.dtype} {a.shape}")
    return a.astype(np.int64)


class PackedBatch:
    """One step's sequences: ``new_lens[b]`` new tokens each behind ``cache_lens[b]`` cached ones, on the pages that
    row b of ``block_table`` lists (all three on the host).  Zero new tokens are allowed.

    Holds on the device, from one upload on the current stream: ``positions`` and ``slots`` (int32 [tokens]: each
    token's position and place in the cache, page * page_size + row), ``block_table`` (int32 [batch, max_blocks])
    and, for each of ``windows`` (None: every key; w: the last w keys), the attention's work list.  Use it on
    other streams, and free it while they run, as any tensor made on the current one.

    A page that a new token is written to must belong to one sequence alone, and every page that a token is written
    to or sees must be one of the pool's; columns behind them, or out of every window, may hold anything."""

    def __init__(self, new_lens, cache_lens, block_table, *, page_size: int, num_pages: int, n_heads: int, n_kv: int,
                 head_dim: int, windows: Sequence[int | None] = (None,), device: torch.device | str = "cuda"):
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
        if page_size < 16 or page_size & (page_size - 1):
            raise RuntimeError(f"page_size {page_size} must be a power of two >= 16")
        if num_pages <= 0 or num_pages * page_size > 0x7FFFFFFF:
            raise RuntimeError(f"{num_pages} pages of {page_size} tokens: the pool must have 1 to 2^31 - 1 slots")
        if head_dim not in (64, 128):
            raise RuntimeError(f"head_dim {head_dim} unsupported (64 or 128)")
        if n_kv <= 0 or n_heads <= 0 or n_heads % n_kv:
            raise RuntimeError(f"n_heads {n_heads} must be a multiple of n_kv {n_kv}")
        if not windows:
            raise RuntimeError("windows must name at least one window (None: every key)")
        for w in windows:
            if w is not None and (isinstance(w, bool) or not isinstance(w, (int, np.integer)) or not 1 <= w <= _MAX_KEYS):
                raise RuntimeError(f"window {w!r} must be None or 1 to 2^27 keys")
        if (new < 0).any() or (ctx < 0).any() or (new + ctx > _MAX_KEYS).any():
            raise RuntimeError("lengths must not be negative, nor 2^27 keys be passed")
        total = int(new.sum())
        if total * n_heads > 1 << 30:
            raise RuntimeError(f"{total} tokens of {n_heads} heads: more than 2^30 query rows")
        self.batch, self.total_tokens = len(new), total
        self.page_size, self.num_pages = page_size, num_pages
        self.n_heads, self.n_kv, self.head_dim, self.device = n_heads, n_kv, head_dim, device
        self._page_shape = (page_size, n_kv, head_dim)
        self._page_strides = (n_kv * head_dim, head_dim, 1)
        self.max_blocks = max(bt.shape[1], 1)
        widest = _MAX_KEYS if any(w is None for w in windows) else max(windows)
        self._check_pages(new, ctx, bt, widest)
        seq = np.repeat(np.arange(self.batch), new)
        pos = np.arange(total) - np.repeat(np.cumsum(new) - new, new) + ctx[seq]
        slots = bt[seq, pos // page_size] * page_size + pos % page_size if total else pos

        cus = torch.cuda.get_device_properties(device).multi_processor_count if device.type == "cuda" else 256
        plans = {w: self._plan(new, ctx, w, cus) for w in dict.fromkeys(windows)}
        parts = [pos, slots, bt.ravel()] + [a.ravel() for items, merges, _ in plans.values() for a in (items, merges)]
        starts = np.cumsum([0] + [-(-p.size // 4) * 4 for p in parts])     # 16-byte aligned
        staged = torch.empty(int(starts[-1]) + 4, dtype=torch.int32, pin_memory=device.type == "cuda")
        host = staged.numpy()
        for p, at in zip(parts, starts):
            host[at:at + p.size] = p
        with _on(device) if device.type == "cuda" else contextlib.nullcontext():
            self._buf = staged.to(device, non_blocking=True)
        view = [self._buf[at:at + p.size] for p, at in zip(parts, starts)]
        self.positions, self.slots = view[0], view[1]
        self.block_table = view[2].view(self.batch, bt.shape[1])
        self._plans = {}
        for i, (w, (items, merges, counts)) in enumerate(plans.items()):
            self._plans[w] = (view[3 + 2 * i], len(items), view[4 + 2 * i], len(merges), int(counts[2]), int(counts[3]))

    def _check_pages(self, new, ctx, bt, widest) -> None:
        P, busy = self.page_size, new > 0
        end = -(-(ctx + new) // P)
        if (end[busy] > bt.shape[1]).any():
            raise RuntimeError(f"a sequence needs {int(end[busy].max())} pages, the block table has {bt.shape[1]} columns")
        cols = np.arange(bt.shape[1])[None]
        first = np.maximum(ctx - widest + 1, 0) // P
        used = busy[:, None] & (cols >= first[:, None]) & (cols < end[:, None])
        if ((bt < 0) | (bt >= self.num_pages))[used].any():
            raise RuntimeError(f"the block table lists a page outside [0, {self.num_pages}) that a sequence needs")
        written = bt[busy[:, None] & (cols >= (ctx // P)[:, None]) & (cols < end[:, None])]
        if np.unique(written).size != written.size:
            raise RuntimeError("two places of the batch write to one page (the same sequence twice, or a shared page "
                               "that was not copied before the write)")
        if np.abs(bt).max(initial=0) > 0x7FFFFFFF:
            raise RuntimeError("block_table must fit int32")

    def _plan(self, new, ctx, window, cus):
        lib = _lib.load()
        n32, c32 = np.ascontiguousarray(new, np.int32), np.ascontiguousarray(ctx, np.int32)
        counts = np.zeros(4, np.int32)
        sizes = (n32.ctypes.data, c32.ctypes.data, self.batch, self.n_heads, self.n_kv, self.head_dim, int(window or 0), cus)
        # enough for a block per 128 query rows and sequence and two ranges per workgroup; asked for where it is not
        g = self.n_heads // self.n_kv
        room = self.total_tokens * g // 128 + self.batch + 4 * max(2 * cus // self.n_kv, 1)
        while True:
            items, merges = np.empty((room, 8), np.int32), np.empty((room, 8), np.int32)
            rc = lib.pkv_packed_plan(*sizes, items.ctypes.data, room, merges.ctypes.data, room, counts.ctypes.data)
            if rc != _lib.PKV_ENOSPC:
                break
            room = int(counts[:2].max())
        _lib.check(rc, "pkv_packed_plan")
        return items[:counts[0]], merges[:counts[1]], counts

    def _check_cache(self, k_cache, v_cache) -> int:
        """The caches' page stride."""
        shape, strides = k_cache.shape, k_cache.stride()
        if k_cache.dtype is _BF16 and v_cache.dtype is _BF16 and shape == v_cache.shape and strides == v_cache.stride() \
                and len(shape) == 4 and shape[0] >= self.num_pages and shape[1:] == self._page_shape and \
                strides[1:] == self._page_strides and k_cache.device == self.device and v_cache.device == self.device:
            return strides[0]
        num_pages, page_size, n_kv, hd = _check_cache(k_cache, v_cache)   # says what is wrong, where it is the cache's own
        if (page_size, n_kv, hd) != self._page_shape or num_pages < self.num_pages:
            raise RuntimeError(f"cache of {num_pages} pages x {page_size} x {n_kv} heads x {hd} does not fit a batch laid "
                               f"out for {self.num_pages} x {self.page_size} x {self.n_kv} x {self.head_dim}")
        raise RuntimeError(f"the cache must be on the batch's device {self.device}")


def _rows3(t: torch.Tensor, name: str, batch: PackedBatch) -> tuple[int, int]:
    shape, strides = t.shape, t.stride()
    if t.dtype is not _BF16:
        raise RuntimeError(f"{name} must be {_BF16}, got {t.dtype}")
    if len(shape) != 3 or shape[0] < batch.total_tokens or shape[1] != batch.n_heads or shape[2] != batch.head_dim:
        raise RuntimeError(f"{name} has shape {tuple(shape)}, expected [>= {batch.total_tokens}, {batch.n_heads}, "
                           f"{batch.head_dim}]")
    if strides[2] != 1:
        raise RuntimeError(f"{name} must be contiguous in head_dim")
    if t.device != batch.device:
        raise RuntimeError(f"{name} must be on the batch's device {batch.device}")
    return strides[0], strides[1]


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
    from .epilogue import _check_norms, _check_rotary_tables
    _require_gpu(qkv, "qkv")
    page_stride = batch._check_cache(k_cache, v_cache)
    nh, nk, hd, total, dev = batch.n_heads, batch.n_kv, batch.head_dim, batch.total_tokens, batch.device
    shape, strides = qkv.shape, qkv.stride()
    if qkv.dtype is not _BF16 or len(shape) != 2 or shape[0] < total or shape[1] != (nh + 2 * nk) * hd or strides[1] != 1:
        raise RuntimeError(f"qkv must be bfloat16 [>= {total}, {(nh + 2 * nk) * hd}], contiguous in its last dimension, "
                           f"got {qkv.dtype} {tuple(shape)}")
    if qkv.device != dev:
        raise RuntimeError(f"qkv must be on the batch's device {dev}")
    rotary = _check_rotary_tables(cos, sin, hd, dev)
    if q_norm_w is not None or k_norm_w is not None:
        _check_norms(q_norm_w, k_norm_w, hd, _BF16, dev)
    if positions is None:
        positions = batch.positions
    elif positions.dtype != torch.int32 or positions.dim() != 1 or positions.shape[0] < total or \
            positions.device != dev or (total > 1 and positions.stride(0) != 1):
        raise RuntimeError(f"positions must be contiguous int32 [>= {total}] on the batch's device")
    if q_out is None:
        q_out = torch.empty((shape[0], nh, hd), dtype=_BF16, device=dev)
        if shape[0] > total:
            q_out[total:].zero_()
        qo = nh * hd, hd
    else:
        qo = _rows3(q_out, "q_out", batch)
    if total == 0:
        return q_out
    st = status if status is not None else status_tensor(dev)
    with _on(dev):
        rc = _lib.fast().pkv_packed_rope_append(
            qkv.data_ptr(), strides[0], positions.data_ptr(), batch.slots.data_ptr(), cos.data_ptr(), sin.data_ptr(),
            cos.shape[0], q_norm_w.data_ptr() if q_norm_w is not None else 0,
            k_norm_w.data_ptr() if k_norm_w is not None else 0, float(eps), q_out.data_ptr(), qo[0], qo[1],
            k_cache.data_ptr(), v_cache.data_ptr(), page_stride, total, nh, nk, hd, rotary, int(interleaved),
            batch.page_size, batch.num_pages, st.data_ptr(), _raw_stream(dev.index))
    if rc:
        _lib.check(rc, "pkv_packed_rope_append")
    return q_out


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
    _require_gpu(q, "q")
    qs = _rows3(q, "q", batch)
    page_stride = batch._check_cache(k_cache, v_cache)
    plan = batch._plans.get(window)
    if plan is None:
        raise RuntimeError(f"the batch was laid out for the windows {list(batch._plans)}, not {window}")
    dev, total, nh, hd = batch.device, batch.total_tokens, batch.n_heads, batch.head_dim
    if sinks is not None and (sinks.dtype != torch.float32 or tuple(sinks.shape) != (nh,) or sinks.stride(0) != 1 or
                              sinks.device != dev):
        raise RuntimeError(f"sinks must be a contiguous float32 [{nh}] vector on the batch's device")
    scale = 1.0 / math.sqrt(hd) if softmax_scale is None else float(softmax_scale)
    items, n_items, merges, n_merges, partials, merge_rows = plan
    with _on(dev):
        if out is None:
            rows = q.shape[0]
            out = torch.empty((rows, nh, hd), dtype=_BF16, device=dev)
            if rows > total:
                out[total:].zero_()
            os_ = nh * hd, hd
        else:
            os_ = _rows3(out, "out", batch)
        lse = None
        if return_lse:
            lse = torch.empty((q.shape[0], nh), dtype=torch.float32, device=dev)
            if q.shape[0] > total:
                lse[total:].zero_()
        if total == 0:
            return (out, lse) if return_lse else out
        # the partials of this call alone, from torch's allocator: of the current stream, or of the graph it captures
        nbytes, ws = 0, None
        if partials:
            nbytes = _lib.load().pkv_packed_workspace_bytes(partials, batch.n_kv, hd)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        st = status if status is not None else status_tensor(dev)
        rc = _lib.fast().pkv_packed_attn(
            q.data_ptr(), qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), page_stride,
            batch.block_table.data_ptr(), batch.max_blocks, out.data_ptr(), os_[0], os_[1],
            lse.data_ptr() if lse is not None else 0, sinks.data_ptr() if sinks is not None else 0,
            items.data_ptr(), n_items, merges.data_ptr() if n_merges else 0, n_merges, partials, merge_rows,
            ws.data_ptr() if ws is not None else 0, nbytes, total, batch.batch, nh, batch.n_kv, hd, batch.page_size,
            batch.num_pages, batch.max_blocks, int(window or 0), scale, st.data_ptr(), _raw_stream(dev.index))
    if rc:
        _lib.check(rc, "pkv_packed_attn")
    return (out, lse) if return_lse else out
