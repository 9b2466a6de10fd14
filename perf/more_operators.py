"""Operators behind the packed step's attention: a cache held to a budget, and the next tokens.

A server whose conversations outgrow the page pool keeps, per layer and KV head, the keys that the attention has
weighed most, and draws the next tokens on the device, so that a decode loop never waits for the host:

  weigh    packed_key_weights: adds up, for every cached key and KV head, the attention weight that the step's new
           tokens gave it (their queries, the keys and the softmax denominators' logarithms are in hand)
  evict    evict_keys: per layer, sequence and KV head the heaviest keys stay, beside the first and the latest ones,
           and K, V and weights of those that stay move to the front of the sequence's pages, in order
  sample   sample_tokens: temperature, top-k, top-p, min-p and the draw itself, from given uniform numbers

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what the program
holds before the call, ``run`` makes one pass (``own`` false: the formulas in elementary torch operations; true:
this package's entry points), ``work`` says what a pass cannot do without, ``exact`` recomputes it in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

# decoder shapes of this repository's workloads
SHAPES = {
    "0.5B": dict(n_heads=14, n_kv=2, head_dim=64, layers=24),
    "7B": dict(n_heads=28, n_kv=4, head_dim=128, layers=28),
    "14B": dict(n_heads=40, n_kv=8, head_dim=128, layers=48),
    "7B-tp4": dict(n_heads=7, n_kv=1, head_dim=128, layers=28),
}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MAX_KEYS = 131072          # the longest context
MAX_FLOPS = 1.8e11         # of one pass
MAX_BYTES = 1.2e9
MAX_POOL = 1.8e9           # K and V of an evicting call's sequences, all layers


def listed() -> list[dict]:
    return [
        # one token of one conversation on a draft model: the smallest call of the step
        dict(name="weigh_one", op="weigh", shape="0.5B", page=256, ones=1, chunks=0, chunk=0, ctx=700, rows=0,
             window=0, lengths=0),
        # a decode step of a loaded server
        dict(name="weigh_decode", op="weigh", shape="7B", page=256, ones=48, chunks=0, chunk=0, ctx=2500, rows=0,
             window=0, lengths=1),
        # long documents being answered from on one GPU's share of the heads, small pages
        dict(name="weigh_long", op="weigh", shape="7B-tp4", page=64, ones=7, chunks=0, chunk=0, ctx=50000, rows=0,
             window=0, lengths=2),
        # decode tokens beside prompt chunks that every new token weighs, tiny pages, normal load of the larger model
        dict(name="weigh_mixed", op="weigh", shape="14B", page=16, ones=37, chunks=3, chunk=601, ctx=1800, rows=0,
             window=0, lengths=3),
        # whole prompts, every token's weights: all of it matrix products and exponentials
        dict(name="weigh_prompts", op="weigh", shape="7B", page=256, ones=0, chunks=4, chunk=3500, ctx=0, rows=0,
             window=0, lengths=4),
        # one chat on the draft model over its budget: the smallest eviction
        dict(name="evict_chat", op="evict", shape="0.5B", page=256, seqs=1, length=1500, keep=0.6, first=4, recent=64,
             lengths=5),
        # the conversations that a decode step found over their budget
        dict(name="evict_batch", op="evict", shape="7B", page=256, seqs=6, length=2800, keep=0.5, first=4, recent=256,
             lengths=6),
        # a long document cut to an eighth
        dict(name="evict_long", op="evict", shape="7B-tp4", page=64, seqs=1, length=100000, keep=0.125, first=4,
             recent=1024, lengths=7),
        # one answer's next token, small vocabulary
        dict(name="sample_one", op="sample", rows=1, vocab=32000, dtype="bf16", temperature=0.8, top_k=50, top_p=0.9,
             min_p=0.0, mixed=False, logprobs=False),
        # the usual step: a batch of chats with a nucleus, no top-k
        dict(name="sample_nucleus", op="sample", rows=32, vocab=151003, dtype="bf16", temperature=0.7, top_k=0,
             top_p=0.9, min_p=0.0, mixed=False, logprobs=False),
        # requests with settings of their own, greedy ones among them, and the drawn tokens' log-probabilities
        dict(name="sample_mixed", op="sample", rows=60, vocab=128000, dtype="fp32", temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0, mixed=True, logprobs=True),
        # a large rollout batch, the distribution as it is
        dict(name="sample_rollout", op="sample", rows=256, vocab=131072, dtype="fp32", temperature=1.0, top_k=0,
             top_p=1.0, min_p=0.0, mixed=False, logprobs=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        c = dict(op=rng.choice(["weigh", "weigh", "evict", "sample", "sample"]))
        if c["op"] == "sample":
            c.update(rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 1000, 200000),
                     dtype=rng.choice(["bf16", "fp16", "fp32", "fp32"]), temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.3]),
                     top_k=rng.choice([0, 0, 1, 20, 50, 400]), top_p=rng.choice([1.0, 0.95, 0.9, 0.5]),
                     min_p=rng.choice([0.0, 0.0, 0.05]), mixed=rng.random() < 0.4, logprobs=rng.random() < 0.5)
        elif c["op"] == "evict":
            c.update(shape=rng.choice(list(SHAPES)), page=rng.choice([16, 64, 256, 256]), seqs=_log_int(rng, 1, 12),
                     length=_log_int(rng, 40, 100000), keep=rng.choice([0.05, 0.125, 0.25, 0.5, 0.6, 0.9]),
                     first=rng.choice([0, 4, 16]), recent=_log_int(rng, 1, 1024), lengths=rng.randrange(1 << 20))
            s = SHAPES[c["shape"]]
            if int(_evict_lengths(c)[0].sum()) * s["layers"] * s["n_kv"] * s["head_dim"] * 4 > MAX_POOL:
                continue
        else:
            c.update(shape=rng.choice(list(SHAPES)), page=rng.choice([16, 64, 256, 256]),
                     ones=rng.choice([0, _log_int(rng, 1, 200)]), chunks=rng.choice([0, 0, _log_int(rng, 1, 10)]),
                     chunk=_log_int(rng, 2, 3500), ctx=rng.choice([0, _log_int(rng, 16, 50000)]),
                     rows=rng.choice([0, 0, _log_int(rng, 1, 256)]), window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]),
                     lengths=rng.randrange(1 << 20))
            if c["ones"] + c["chunks"] == 0:
                continue
            new, ctx = _lengths(c)
            s = SHAPES[c["shape"]]
            # scores of the plain form's widest (chunk, KV head) product, and the pool
            if int((new * ctx + new * new).max()) * s["n_heads"] // s["n_kv"] > 6e8:
                continue
            if int((new + ctx).sum()) * s["n_kv"] * s["head_dim"] * 2 > 3e9:
                continue
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


# ---------------------------------------------------------------------------------- lengths and inputs
def _lengths(case: dict) -> tuple[np.ndarray, np.ndarray]:
    """(new tokens, cached tokens) of each sequence, chunks and decode tokens mixed as they arrive."""
    rng = np.random.default_rng(case["lengths"])
    n1, nc, ctx = case["ones"], case["chunks"], case["ctx"]
    new = np.concatenate([np.ones(n1, np.int64),
                          rng.integers(max(case["chunk"] // 2, 1), case["chunk"] + 1, size=nc)])
    if ctx:
        c = np.concatenate([np.clip(np.round(rng.lognormal(math.log(ctx), 0.5, size=n1)), 1, MAX_KEYS),
                            rng.integers(0, ctx + 1, size=nc)])
    else:
        c = np.zeros(n1 + nc)
    order = rng.permutation(n1 + nc)
    new, c = new[order], c[order].astype(np.int64)
    return new, np.minimum(c, MAX_KEYS - new)


def _evict_lengths(case: dict) -> tuple[np.ndarray, np.ndarray]:
    """(cached tokens, how many of them stay) of each sequence; now and then one is within its budget already."""
    rng = np.random.default_rng(case["lengths"])
    n = np.clip(np.round(case["length"] * rng.uniform(0.8, 1.2, size=case["seqs"])), 1, MAX_KEYS).astype(np.int64)
    keep = np.maximum(np.round(n * case["keep"] * rng.uniform(0.9, 1.1, size=case["seqs"])), 1).astype(np.int64)
    return n, keep


def _block_table(tokens: np.ndarray, page: int, rng) -> tuple[np.ndarray, int]:
    """The sequences' pages scattered over a pool (its size too); columns a sequence does not have are -1."""
    need = -(-tokens // page)
    pool = int(need.sum()) + 3
    ids = rng.permutation(pool)
    bt = np.full((len(need), int(need.max())), -1, np.int32)
    off = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[off:off + n]
        off += n
    return bt, pool


def _randn(shape, g, dev, dtype=torch.bfloat16, scale=1.0) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=dev).normal_(0.0, scale, generator=g)


def _past_weights(shape, g, dev) -> torch.Tensor:
    """Accumulated weights: a heavy tail, and keys that no token has looked at."""
    w = torch.empty(shape, dtype=torch.float32, device=dev).exponential_(1.0, generator=g)
    return (w ** 3 * 0.05) * (w > 0.1)


def _sample_settings(case: dict, seed: int, dev) -> dict:
    """temperature, top_k, top_p, min_p (32 bits): numbers for the whole batch, or a tensor with one for each row."""
    if not case["mixed"]:
        return {k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}
    rng, n = np.random.default_rng(seed + 77), case["rows"]
    pick = lambda *of: torch.from_numpy(np.stack([np.asarray(o).repeat(n) if np.ndim(o) == 0 else o for o in of])
                                        [rng.integers(0, len(of), size=n), np.arange(n)])
    return dict(temperature=pick(0.0, 1.0, rng.uniform(0.3, 1.5, n), rng.uniform(0.3, 1.5, n)).float().to(dev),
                top_k=pick(0, 50, rng.integers(1, 1000, n)).int().to(dev),
                top_p=pick(1.0, rng.uniform(0.5, 0.99, n), rng.uniform(0.5, 0.99, n)).float().to(dev),
                min_p=pick(0.0, 0.0, rng.uniform(0.01, 0.2, n)).float().to(dev))


def _inputs(case: dict, seed: int) -> dict:
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    st = dict(case=case)
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        # a broad ground, and a few dozen tokens that the context calls for, more or less clearly
        x = _randn((n, v), g, dev, torch.float32, 2.0)
        lift = torch.empty((n, 40), device=dev).exponential_(1.0, generator=g)
        apart = torch.empty((n, 40), dtype=torch.float64, device=dev).uniform_(0.0, 1.0, generator=g)
        at = ((torch.arange(40, device=dev) + apart) * (v / 40)).long().clamp(max=v - 1)
        sharp = torch.empty((n, 1), device=dev).uniform_(1.0, 5.0, generator=g)
        x.scatter_(1, at, 4.0 + sharp * lift)
        st["logits"] = x.to(DTYPES[case["dtype"]])
        st["uniforms"] = torch.empty((n,), device=dev).uniform_(0.0, 1.0, generator=g)
        st["settings"] = _sample_settings(case, seed, dev)
        return st
    s = SHAPES[case["shape"]]
    nh, nk, hd, P = s["n_heads"], s["n_kv"], s["head_dim"], case["page"]
    if case["op"] == "evict":
        n, keep = _evict_lengths(case)
        bt, pool = _block_table(n, P, rng)
        st.update(n=n, keep=keep, bt=bt, k_pool=_randn((s["layers"], pool, P, nk, hd), g, dev),
                  v_pool=_randn((s["layers"], pool, P, nk, hd), g, dev),
                  weights=_past_weights((s["layers"], pool, nk, P), g, dev))
        return st
    new, ctx = _lengths(case)
    bt, pool = _block_table(new + ctx, P, rng)
    total = int(new.sum())
    st.update(new=new, ctx=ctx, bt=bt, k_cache=_randn((pool, P, nk, hd), g, dev), q=_randn((total, nh, hd), g, dev),
              weights=_past_weights((pool, nk, P), g, dev))
    # the denominators' logarithms as the attention returns them, near enough: what such keys give on the average
    seen = np.concatenate([np.minimum(np.arange(c, c + n) + 1, case["window"] or MAX_KEYS + 1) for n, c in zip(new, ctx)])
    seen = torch.from_numpy(seen.astype(np.float32)).to(dev)
    st["lse"] = torch.log(seen)[:, None] + st["q"].float().square().sum(-1) / (2.0 * hd)
    return st


def prepare(case: dict, seed: int) -> dict:
    st = _inputs(case, seed)
    if case["op"] == "sample":
        return st
    s, dev = SHAPES[case["shape"]], torch.device("cuda:0")
    if case["op"] == "evict":
        if own:
            # the call's lengths and pages on the device
            st["args"] = [torch.from_numpy(np.asarray(a, np.int32)).to(dev) for a in (st["bt"], st["n"], st["keep"])]
            st["most"] = int(np.minimum(st["keep"], st["n"]).max())
        return st
    if own:
        import prism_amd
        # the step's batch: lengths, positions, cache slots and work lists, uploaded once per step
        st["batch"] = prism_amd.PackedBatch(st["new"], st["ctx"], st["bt"], page_size=case["page"],
                                            num_pages=st["k_cache"].shape[0], n_heads=s["n_heads"], n_kv=s["n_kv"],
                                            head_dim=s["head_dim"], windows=(case["window"] or None,),
                                            weight_rows=case["rows"] or None, device=dev)
        return st
    st["pages"] = [torch.from_numpy(st["bt"][b, :n].astype(np.int64)).to(dev)
                   for b, n in enumerate(-(-(st["new"] + st["ctx"]) // case["page"]))]
    return st


# ---------------------------------------------------------------------------------- the plain forms
def _weigh_plain(st: dict):
    case, s = st["case"], SHAPES[st["case"]["shape"]]
    nk, hd, dev = s["n_kv"], s["head_dim"], st["q"].device
    g = s["n_heads"] // nk
    first = 0
    for b, (n, c) in enumerate(zip(st["new"].tolist(), st["ctx"].tolist())):
        rows = min(case["rows"] or n, n)               # the last so many new tokens count
        lo = first + n - rows
        keys = st["k_cache"][st["pages"][b]].reshape(-1, nk, hd)[:c + n]
        old = st["weights"][st["pages"][b]]            # [pages, n_kv, page]
        t = torch.arange(c + n, device=dev)
        p = torch.arange(c + n - rows, c + n, device=dev)[:, None]
        seen = t <= p
        if case["window"]:
            seen = seen & (t > p - case["window"])
        flat = old.transpose(0, 1).reshape(nk, -1).clone()
        for h in range(nk):
            qh = st["q"][lo:first + n, h * g:(h + 1) * g].float().reshape(rows * g, hd)
            sc = (qh @ keys[:, h].float().t()) / math.sqrt(hd)
            lse = st["lse"][lo:first + n, h * g:(h + 1) * g].reshape(rows * g, 1)
            weight = torch.exp(sc - lse).view(rows, g, c + n) * seen[:, None]
            got = weight.sum((0, 1), dtype=torch.float64).float()
            flat[h, :c] += got[:c]                     # a key that this step appended starts from nothing
            flat[h, c:c + n] = got[c:]
        st["weights"][st["pages"][b]] = flat.view(nk, -1, case["page"]).transpose(0, 1)
        first += n
    return [st["weights"]]


def _evict_plain(st: dict):
    case, s = st["case"], SHAPES[st["case"]["shape"]]
    L, nk, hd, P, dev = s["layers"], s["n_kv"], s["head_dim"], case["page"], st["k_pool"].device
    most = int(np.minimum(st["keep"], st["n"]).max())
    kept = torch.full((L, len(st["n"]), nk, most), -1, dtype=torch.int32, device=dev)
    for b, (n, keep) in enumerate(zip(st["n"].tolist(), st["keep"].tolist())):
        if n <= keep:
            kept[:, b, :, :n] = torch.arange(n, device=dev, dtype=torch.int32)
            continue
        slots = torch.from_numpy(st["bt"][b].astype(np.int64)).to(dev)[torch.arange(n, device=dev) // P] * P \
            + torch.arange(n, device=dev) % P
        first = min(case["first"], keep)
        recent = min(case["recent"], keep - first)
        w = st["weights"][:, slots // P, :, slots % P].permute(1, 2, 0)      # [L, n_kv, n]
        middle = w[..., first:n - recent]
        order = torch.sort(middle, dim=-1, descending=True, stable=True).indices[..., :keep - first - recent] + first
        ends = torch.cat([torch.arange(first, device=dev), torch.arange(n - recent, n, device=dev)])
        idx = torch.cat([order, ends.expand(L, nk, -1)], -1).sort(-1).values  # [L, n_kv, keep]
        kept[:, b, :, :keep] = idx.int()
        to = slots[:keep]
        wide = idx.transpose(1, 2)[..., None].expand(-1, -1, -1, hd)
        for pool in (st["k_pool"], st["v_pool"]):
            flat = pool.view(L, -1, nk, hd)
            flat[:, to] = flat[:, slots].gather(1, wide)
        st["weights"][:, to // P, :, to % P] = w.gather(2, idx).permute(2, 0, 1)
    return [st["k_pool"], st["v_pool"], st["weights"], kept]


def _sample_plain(st: dict):
    x, u, dev = st["logits"].double(), st["uniforms"].double(), st["logits"].device
    n, v = x.shape
    per_row = lambda a: (a if torch.is_tensor(a) else torch.full((n,), a, dtype=torch.float32, device=dev)).double()[:, None]
    t, k, p, m = (per_row(st["settings"][a]) for a in ("temperature", "top_k", "top_p", "min_p"))
    greedy = t <= 0
    top = x.amax(1, keepdim=True)
    # a border can lie as near as the next token's weight, 1e-6 of the sum: 64 bits
    w = torch.exp((x - top) / torch.where(greedy, 1.0, t))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    rank = torch.arange(v, device=dev)
    ws = w.gather(1, order)
    ws = torch.where((rank < torch.where(k > 0, k, v)) & (~greedy | (rank == 0)), ws, 0.0)
    before = ws.cumsum(1) - ws
    stays = ((before < p * ws.sum(1, keepdim=True)) | (p >= 1) | (rank == 0)) & ((ws >= m.clamp(max=1.0)) | (rank == 0))
    ws = torch.where(stays, ws, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, ws)
    run_sum = w.cumsum(1)
    total = run_sum[:, -1:]
    token = (run_sum <= u[:, None] * total).sum(1)
    # u * total rounded up to the total: the last token that stays
    token = torch.minimum(token, v - 1 - (w > 0).flip(1).int().argmax(1))
    out = [token]
    if st["case"]["logprobs"]:
        out.append(torch.log(w.gather(1, token[:, None]) / total)[:, 0].float())
    return out


# ---------------------------------------------------------------------------------- one pass
def run(state: dict):
    case = state["case"]
    if not own:
        return {"weigh": _weigh_plain, "evict": _evict_plain, "sample": _sample_plain}[case["op"]](state)
    import prism_amd
    if case["op"] == "weigh":
        return [prism_amd.packed_key_weights(state["q"], state["k_cache"], state["lse"], state["weights"],
                                             state["batch"], window=case["window"] or None)]
    if case["op"] == "evict":
        bt, n, keep = state["args"]
        kept = prism_amd.evict_keys(state["k_pool"], state["v_pool"], state["weights"], bt, n, keep, state["most"],
                                    first=case["first"], recent=case["recent"])
        return [state["k_pool"], state["v_pool"], state["weights"], kept]
    r = prism_amd.sample_tokens(state["logits"], state["uniforms"], **state["settings"],
                                return_logprobs=case["logprobs"])
    return list(r) if case["logprobs"] else [r]


# ---------------------------------------------------------------------------------- what a pass needs
def work(case: dict) -> dict:
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        # the logits, once; settings, uniforms and tokens
        return dict(bytes=float(n * v * DTYPES[case["dtype"]].itemsize + n * (12 + (16 if case["mixed"] else 0)
                                                                              + (4 if case["logprobs"] else 0))),
                    flops=float(n * v * 4))
    s = SHAPES[case["shape"]]
    nh, nk, hd, L = s["n_heads"], s["n_kv"], s["head_dim"], s.get("layers", 1)
    if case["op"] == "evict":
        n, keep = _evict_lengths(case)
        over = keep < n
        n, keep = n[over].astype(np.float64), keep[over].astype(np.float64)
        # every weight that is compared, then the kept keys' K, V and weights read and written, but for the first ones
        # which lie where they have to; the kept positions
        moved = np.maximum(keep - case["first"], 0)
        return dict(bytes=float(L * nk * (4 * n.sum() + moved.sum() * (2 * hd * 2 * 2 + 4) + 4 * keep.sum())) + 8 * len(n),
                    flops=float(L * nk * n.sum()))
    new, ctx = (a.astype(np.float64) for a in _lengths(case))
    rows = np.minimum(new, case["rows"]) if case["rows"] else new
    w = float(case["window"] or 1 << 40)
    at = ctx + new - rows                                   # keys before the first row that counts
    keys = np.minimum(at, w - 1) + rows
    short = np.clip(w - at, 0, rows)                        # rows whose window reaches the first key
    pairs = short * at + short * (short + 1) / 2 + (rows - short) * w if case["window"] else \
        rows * at + rows * (rows + 1) / 2
    nbytes = float(keys.sum()) * nk * hd * 2 + float(rows.sum()) * nh * (hd * 2 + 4) \
        + float(keys.sum() * 2 - np.minimum(rows, keys).sum()) * nk * 4 + 4 * float(np.ceil(keys / case["page"]).sum())
    return dict(bytes=nbytes, flops=2.0 * nh * (hd + 1) * float(pairs.sum()))


# ---------------------------------------------------------------------------------- 64 bits
def _weigh64(st: dict) -> list:
    case, s, dev = st["case"], SHAPES[st["case"]["shape"]], st["q"].device
    P, g = case["page"], s["n_heads"] // s["n_kv"]
    out = st["weights"].double()
    row = 0
    for b, (n, c) in enumerate(zip(st["new"].tolist(), st["ctx"].tolist())):
        at = torch.arange(c + n)
        pages, places = torch.from_numpy(st["bt"][b].astype(np.int64))[at // P].to(dev), (at % P).to(dev)
        behind = torch.arange(c, c + n, device=dev)[:, None] - at.to(dev)      # how far each key lies back
        seen = (behind >= 0) & (behind < (case["window"] or MAX_KEYS + 1))
        if case["rows"]:
            seen[:max(n - case["rows"], 0)] = False
        out[pages[c:, None], torch.arange(s["n_kv"], device=dev), places[c:, None]] = 0.0
        for h in range(s["n_heads"]):
            k = st["k_cache"][pages, places, h // g].double()
            sc = st["q"][row:row + n, h].double() @ k.t() * s["head_dim"] ** -0.5 - st["lse"][row:row + n, h:h + 1].double()
            out[pages, h // g, places] += torch.where(seen, sc, -math.inf).exp().sum(0)
        row += n
    return [out]


def _evict64(st: dict) -> list:
    case, s = st["case"], SHAPES[st["case"]["shape"]]
    P = case["page"]
    K, V, W = st["k_pool"], st["v_pool"], st["weights"].cpu().numpy()
    W2 = W.copy()
    most = int(np.minimum(st["keep"], st["n"]).max())
    kept = np.full((s["layers"], len(st["n"]), s["n_kv"], most), -1, np.int32)
    K2, V2 = K.clone(), V.clone()
    for b, (n, keep) in enumerate(zip(st["n"].tolist(), st["keep"].tolist())):
        at = np.arange(n)
        page, place = st["bt"][b][at // P].astype(np.int64), at % P
        f = min(case["first"], keep)
        r = min(case["recent"], keep - f)
        tier = np.where((at < f) | (at >= n - r), 0, 1)     # what stays whatever it weighs, then by weight, then by age
        for layer in range(s["layers"]):
            for h in range(s["n_kv"]):
                w = W[layer, page, h, place]
                idx = np.sort(np.lexsort((at, -w, tier))[:keep])
                kept[layer, b, h, :len(idx)] = idx
                if n <= keep:
                    continue
                to = np.arange(keep)
                W2[layer, page[to], h, place[to]] = w[idx]
                src, dst = (torch.from_numpy(page[i] * P + place[i]).to(K.device) for i in (idx, to))
                for new, old in ((K2, K), (V2, V)):
                    new[layer].flatten(0, 1)[dst, h] = old[layer].flatten(0, 1)[src, h]
    return [K2, V2, torch.from_numpy(W2).to(K.device), torch.from_numpy(kept).to(K.device)]


def _sample64(st: dict) -> list:
    case, v = st["case"], st["case"]["vocab"]
    tokens, logs = [], []
    at = np.arange(v)
    for i in range(case["rows"]):
        x = st["logits"][i].double().cpu().numpy()
        t, k, p, m = (float(a[i]) if torch.is_tensor(a) else float(np.float32(a)) for a in
                      (st["settings"][n] for n in ("temperature", "top_k", "top_p", "min_p")))
        order = np.lexsort((at, -x))                        # the largest first, of equal ones the lowest token
        if t <= 0:
            order, t = order[:1], 1.0
        elif k > 0:
            order = order[:int(k)]
        w = np.exp((x[order] - x[order[0]]) / t)
        if p < 1:
            sums = np.cumsum(w)
            order = order[:1 + int(np.searchsorted(sums, p * sums[-1], side="left"))]
            w = w[:len(order)]
        order, w = order[w >= min(m, 1.0)], w[w >= min(m, 1.0)]
        by_token = np.argsort(order)
        order, w = order[by_token], w[by_token]
        sums = np.cumsum(w)
        j = min(int(np.searchsorted(sums, float(st["uniforms"][i]) * sums[-1], side="right")), len(order) - 1)
        tokens.append(int(order[j]))
        logs.append(math.log(w[j] / sums[-1]))
    dev = st["logits"].device
    out = [torch.tensor(tokens, device=dev)]
    return out + [torch.tensor(logs, dtype=torch.float64, device=dev)] if case["logprobs"] else out


def exact(case: dict, seed: int):
    return {"weigh": _weigh64, "evict": _evict64, "sample": _sample64}[case["op"]](_inputs(case, seed))
