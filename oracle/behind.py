"""fp64 restatement of what follows the packed step's attention (test-only): key weights, eviction, sampling."""
from __future__ import annotations

import math

import numpy as np
import torch


def key_weights64(q, k_cache, lse, weights, new_lens, ctx_lens, block_table, *, window=None, rows=None, weighed=None,
                  scale=None):
    """weights [pages, n_kv, P] after a step, fp64, and what each key gained (the sum of its terms)."""
    P, nk, hd = k_cache.shape[1:]
    g = q.shape[1] // nk
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    out = weights.double().clone()
    gain = torch.zeros_like(out)
    t0 = 0
    for b, (n, c) in enumerate(zip(new_lens, ctx_lens)):
        n, c = int(n), int(c)
        if n == 0:
            continue
        had = min(int(weighed[b]), c) if weighed is not None else c
        lo = n - min(rows or n, n)
        at = torch.arange(c + n)
        behind = torch.arange(c + lo, c + n)[:, None] - at[None]
        see = (behind >= 0) & (behind < (window or 1 << 40))
        cols = at // P
        pages = block_table[b].long()[cols]
        use = see.any(0) | (at >= had)
        at, pages, see = at[use], pages[use], see[:, use]
        for h in range(nk):
            k = k_cache[pages, at % P, h].double()
            got = torch.zeros(len(at), dtype=torch.float64)
            for i in range(h * g, (h + 1) * g):
                z = lse[t0 + lo:t0 + n, i].double()[:, None]
                x = q[t0 + lo:t0 + n, i].double() @ k.T * scale - z
                got += torch.where(see & ~torch.isinf(z), x.exp(), 0.0).sum(0)
            old = torch.where(at < had, out[pages, h, at % P], 0.0)
            out[pages, h, at % P] = old + got
            gain[pages, h, at % P] = got
        t0 += n
    return out, gain


def evict_np(k_pool, v_pool, weights, block_table, lens, keeps, first, recent, max_keep):
    """The pools after an eviction and the kept positions: numpy arrays (k and v as bits), copied."""
    k, v, w = k_pool.copy(), v_pool.copy(), weights.copy()
    L, _, P, nk, _ = k.shape
    kept = np.full((L, len(lens), nk, max_keep), -1, np.int32)
    for b, (n, keep) in enumerate(zip(lens, keeps)):
        n, keep = int(n), int(min(keep, n))
        t = np.arange(n)
        pg, row = block_table[b][t // P], t % P
        f = min(first, keep)
        r = min(recent, keep - f)
        for l in range(L):
            for h in range(nk):
                x = weights[l, pg, h, row].astype(np.float64)
                middle = t[f:n - r]
                x = np.where(np.isnan(x), np.inf, x), np.isnan(x)
                # NaN first, then the largest, then the earliest
                order = np.lexsort((middle, -x[0][f:n - r], ~x[1][f:n - r]))[:keep - f - r]
                idx = np.sort(np.concatenate([t[:f], middle[order], t[n - r:] if r else t[:0]])).astype(np.int64)
                kept[l, b, h, :keep] = idx
                if keep == n:
                    continue
                to = np.arange(keep)
                k[l, pg[to], row[to], h] = k_pool[l, pg[idx], row[idx], h]
                v[l, pg[to], row[to], h] = v_pool[l, pg[idx], row[idx], h]
                w[l, pg[to], h, row[to]] = weights[l, pg[idx], h, row[idx]]
    return k, v, w, kept


def kept64(x, temperature, top_k, top_p, min_p):
    """One row: the tokens that stay, ascending, their weights, and how far the nearest border of a rule lies."""
    x = np.asarray(x, np.float64)
    can = ~(np.isnan(x) | np.isneginf(x))
    at = np.flatnonzero(can)
    order = at[np.lexsort((at, -x[at]))]
    if len(order) == 0 or not temperature > 0 or top_p <= 0:
        return order[:1], np.ones(len(order[:1])), 1.0
    top = x[order[0]]
    if 0 < top_k < len(order):
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, 0.0 if np.isinf(top) else np.exp((x[order] - top) / temperature))
    near = 1.0
    if top_p < 1:
        before = np.cumsum(w) - w
        share = top_p * w.sum()
        near = min(near, np.abs(before[1:] - share).min(initial=1.0) / w.sum())
        stay = (before < share) | (np.arange(len(w)) == 0)
        order, w = order[stay], w[stay]
    if min_p > 0:
        stay = w >= min(min_p, 1.0)
        near = min(near, np.abs(w[1:] / min(min_p, 1.0) - 1.0)[w[1:] < 1.0].min(initial=1.0))
        order, w = order[stay], w[stay]
    by = np.argsort(order)
    return order[by], w[by], near


def sample64(x, u, temperature, top_k, top_p, min_p):
    """One row: (token, log-probability, how far u lies from the nearest border of a decision, in shares of the sum)."""
    order, w, near = kept64(x, temperature, top_k, top_p, min_p)
    if len(order) == 0:
        return -1, -math.inf, 1.0
    if not temperature > 0 or top_p <= 0:
        return int(order[0]), 0.0, 1.0
    run = np.cumsum(w)
    near = min(near, np.abs(run[:-1] / run[-1] - u).min(initial=1.0))
    j = int(np.searchsorted(run, min(max(u, 0.0), 1.0) * run[-1], side="right"))
    j = min(j, int(np.flatnonzero(w > 0)[-1]))
    return int(order[j]), math.log(w[j] / run[-1]), near
