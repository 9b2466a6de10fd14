"""Eviction from the paged cache by accumulated attention weight.

Prism frees pages by whole sequences alone (engine/kv_cache.py:87-104), so a pool that long conversations fill ends in
KVCacheOutOfPages.  packed_key_weights keeps, for every cached key and KV head, the attention weight it has had;
evict_keys drops the keys that had least, in every layer and KV head on their own, and closes the gaps.
FlashAttnKVCache.evict makes the call for whole sequences and takes their pages back.
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _raw_stream, _require_gpu, status_tensor
from .packed import _on


def _pool_strides(t: torch.Tensor, name: str) -> tuple[int, int]:
    _require_gpu(t, name)
    if t.dtype != torch.bfloat16 or t.dim() != 5:
        raise RuntimeError(f"{name} must be bfloat16 [layers, num_pages, page_size, n_kv, head_dim], got {t.dtype} {tuple(t.shape)}")
    inner = t.shape[3] * t.shape[4]
    if t.stride()[2:] != (inner, t.shape[4], 1):
        raise RuntimeError(f"{name} must be contiguous within a page")
    return t.stride(0), t.stride(1)


def _ints(t: torch.Tensor, name: str, shape, dev: torch.device) -> int:
    if t.dtype != torch.int32 or t.device != dev or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous int32 {list(shape)} on {dev}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def evict_keys(k_pool: torch.Tensor, v_pool: torch.Tensor, key_weights: torch.Tensor, block_table: torch.Tensor,
               seq_lens: torch.Tensor, keep_lens: torch.Tensor, max_keep: int, *, first: int = 4, recent: int = 64,
               status: torch.Tensor | None = None) -> torch.Tensor:
    """Cuts sequences down to ``keep_lens[b]`` of their ``seq_lens[b]`` tokens, in every layer and KV head: the first
    ``first`` stay, the last ``recent``, and of the others those with the largest ``key_weights`` (of equal ones the
    earlier).  K, V and weights of those that stay move, in their order, to the front of the pages that
    ``block_table`` lists; what lies behind them is left as it is.  A sequence of at most ``keep_lens[b]`` tokens
    does not change.  first + recent past keep_lens[b]: the first ones stay, and of the last as many as fit.

    Pools are [layers, num_pages, page_size, n_kv, head_dim], bf16, weights fp32 [layers, num_pages, n_kv, page_size],
    the table and the lengths int32 on their device; ``max_keep`` bounds what stays of any sequence.  Returns the kept
    positions, int32 [layers, batch, n_kv, max_keep], ascending, -1 behind them.  A page that kept tokens move into must not
    be listed anywhere else in the call."""
    ks, vs = _pool_strides(k_pool, "k_pool"), _pool_strides(v_pool, "v_pool")
    dev = k_pool.device
    if v_pool.shape != k_pool.shape or vs != ks or v_pool.device != dev:
        raise RuntimeError("k_pool and v_pool must have the same shape, strides and device")
    layers, pages, P, nk, hd = k_pool.shape
    _require_gpu(key_weights, "key_weights")
    if key_weights.dtype != torch.float32 or key_weights.device != dev or tuple(key_weights.shape) != (layers, pages, nk, P) \
            or key_weights.stride()[2:] != (P, 1):
        raise RuntimeError(f"key_weights must be float32 {[layers, pages, nk, P]} on {dev}, contiguous within a page, got "
                           f"{key_weights.dtype} {list(key_weights.shape)} on {key_weights.device}")
    if block_table.dim() != 2:
        raise RuntimeError(f"block_table must be [batch, max_blocks], got {list(block_table.shape)}")
    batch, blocks = block_table.shape
    for x, name in ((max_keep, "max_keep"), (first, "first"), (recent, "recent")):
        if isinstance(x, bool) or not isinstance(x, int) or not 0 <= x <= 1 << 27:
            raise RuntimeError(f"{name} must be 0 to 2^27 tokens, got {x!r}")
    bt = _ints(block_table, "block_table", (batch, blocks), dev)
    lens, keeps = _ints(seq_lens, "seq_lens", (batch,), dev), _ints(keep_lens, "keep_lens", (batch,), dev)
    if status is None:
        status = status_tensor(dev)
    elif status.dtype != torch.int32 or status.numel() < 1 or status.device != dev:
        raise RuntimeError(f"status must be an int32 word on {dev}")
    with _on(dev):
        kept = torch.empty((layers, batch, nk, max_keep), dtype=torch.int32, device=dev)
        if kept.numel() == 0 or blocks == 0:
            return kept.fill_(-1)
        lib = _lib.load()
        # of this call alone, from torch's allocator: of the current stream, or of the graph it captures
        ws = torch.empty(lib.pkv_evict_workspace_bytes(layers, batch, nk, hd, max_keep), dtype=torch.uint8, device=dev)
        rc = lib.pkv_evict(k_pool.data_ptr(), v_pool.data_ptr(), *ks, key_weights.data_ptr(),
                           *key_weights.stride()[:2], bt, blocks, lens, keeps, kept.data_ptr(), layers, batch, nk, hd,
                           P, pages, blocks, max_keep, first, recent, ws.data_ptr(), ws.numel(), status.data_ptr(),
                           _raw_stream(dev.index))
        _lib.check(rc, "pkv_evict")
    return kept
