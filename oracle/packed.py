"""fp64 restatement of the packed step's operators (test-only): rotation, rotating append, ragged attention.

The rotation is engine/executor.py:45-57 and :108-118 (``_build_rope``, ``_apply_rope``) in general form: part of
the head, either layout, any frequencies, an optional norm of each head.  The attention is flash_attn's over a
paged cache (engine/executor.py:119-120) with a number of new tokens of its own for every sequence.
"""
from __future__ import annotations

import math

import torch


def rotate64(x, positions, inv_freq, *, gain=1.0, interleaved=False, norm_w=None, eps=1e-6):
    """x [tokens, heads, head_dim] -> (rotated fp64, the sum of the magnitudes that each element is made of)."""
    y = x.double()
    if norm_w is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * norm_w.double()
    half = inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq.double()[None]
    c, s = (torch.cos(angle) * gain)[:, None], (torch.sin(angle) * gain)[:, None]
    out, mag = y.clone(), y.abs()
    for i in range(half):
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = y[..., ia], y[..., ib]
        out[..., ia], out[..., ib] = a * c[..., i] - b * s[..., i], b * c[..., i] + a * s[..., i]
        mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * gain
    return out, mag


def packed_attention64(q, k_cache, v_cache, new_lens, ctx_lens, block_table, *, window=None, sinks=None, scale=None):
    """q [tokens, n_heads, hd] over caches [pages, P, n_kv, hd] -> (out, lse, sum_t p_t |v_t|), all fp64."""
    P, nk, hd = k_cache.shape[1:]
    nh = q.shape[1]
    g = nh // nk
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag = torch.zeros_like(out)
    lse = torch.zeros(q.shape[:2], dtype=torch.float64)
    t0 = 0
    for b, (n, c) in enumerate(zip(new_lens, ctx_lens)):
        n, c = int(n), int(c)
        first = max(c - window + 1, 0) if window else 0
        at = torch.arange(first, c + n)
        pages = block_table[b].long()[at // P]
        for h in range(nk):
            k, v = k_cache[pages, at % P, h].double(), v_cache[pages, at % P, h].double()
            for hq in range(h * g, (h + 1) * g):
                s = q[t0:t0 + n, hq].double() @ k.T * scale
                behind = torch.arange(c, c + n)[:, None] - at[None]
                s[(behind < 0) | (behind >= (window or 1 << 40))] = -math.inf
                z = torch.logsumexp(s, -1)
                if sinks is not None:
                    z = torch.logaddexp(z, sinks[hq].double().expand_as(z))
                p = torch.exp(s - z[:, None])
                out[t0:t0 + n, hq], mag[t0:t0 + n, hq], lse[t0:t0 + n, hq] = p @ v, p @ v.abs(), z
        t0 += n
    return out, lse, mag
