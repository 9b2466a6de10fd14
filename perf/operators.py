"""Operators of the packed serving step: tokens of many sequences in one tensor, no padding between them.

A server that batches continuously hands the model one packed tensor per step: a few sequences bring a prompt
chunk, most bring the one token they decode.  Three operators carry such a step through a decoder layer's
attention:

  rotate     rotate_qk: RMSNorm of every query and key head (optional) and the position rotation, in one pass;
             half or interleaved layout, all or part of the head, frequencies scaled for long contexts
  append     packed_rope_append: the same from the fused QKV projection's output, with the rotated keys and the
             values written to their pages of the KV cache
  attention  packed_attention: every new token over its own sequence's pages, causal, with an optional sliding
             window, attention sinks and the rows' log-sum-exp

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what the program
holds before the call, ``run`` makes one pass (``own`` false: the formulas in elementary torch operations and 32
bits; true: this package's entry points), ``work`` says what a pass cannot do without, ``exact`` recomputes it
in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

# decoder shapes of this repository's workloads
SHAPES = {
    "0.5B": dict(n_heads=14, n_kv=2, head_dim=64),
    "7B": dict(n_heads=28, n_kv=4, head_dim=128),
    "14B": dict(n_heads=40, n_kv=8, head_dim=128),
    "7B-tp4": dict(n_heads=7, n_kv=1, head_dim=128),
}
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 1e6
EPS = 1e-6
MAX_KEYS = 131072          # the longest context
MAX_FLOPS = 2.2e11         # of one pass
MAX_BYTES = 5.0e8
# contexts past what the model was trained on: every frequency's period against the original length decides how
# much of it is stretched by the factor
SCALING = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)


def listed() -> list[dict]:
    return [
        # one token of one conversation on a draft model: the smallest call of the step
        dict(name="rotate_one", op="rotate", shape="0.5B", tokens=1, layout="half", rotary=64, dtype="bf16",
             norm=False, scaled=False, far=4096),
        # a prompt chunk of a model that normalises its query and key heads
        dict(name="rotate_chunk_norm", op="rotate", shape="14B", tokens=2048, layout="half", rotary=128,
             dtype="bf16", norm=True, scaled=False, far=32768),
        # a quarter of every head rotated, pairs side by side, in 32 bits, at positions far past the trained ones
        dict(name="rotate_partial_fp32", op="rotate", shape="7B", tokens=5003, layout="interleaved", rotary=32,
             dtype="fp32", norm=False, scaled=True, far=MAX_KEYS),
        # a decode step of 32 ragged sequences
        dict(name="append_decode", op="append", shape="7B", page=256, ones=32, chunks=0, chunk=0, ctx=1500,
             layout="half", rotary=128, norm=False, scaled=False, lengths=0),
        # decode tokens beside three prompt chunks, normalised heads, small pages
        dict(name="append_mixed", op="append", shape="14B", page=16, ones=61, chunks=3, chunk=701, ctx=3000,
             layout="half", rotary=128, norm=True, scaled=False, lengths=1),
        # whole prompts and long documents at once, scaled frequencies
        dict(name="append_prompts", op="append", shape="7B", page=256, ones=0, chunks=9, chunk=2000, ctx=20000,
             layout="half", rotary=128, norm=False, scaled=True, lengths=2),
        # one token onto a short conversation on the draft model: the smallest attention call
        dict(name="attend_one", op="attention", shape="0.5B", page=256, ones=1, chunks=0, chunk=0, ctx=400,
             window=0, sinks=False, lse=False, lengths=3),
        # the usual step of a loaded server: 47 decode tokens and two prompt chunks
        dict(name="attend_mixed", op="attention", shape="7B", page=256, ones=47, chunks=2, chunk=512, ctx=1500,
             window=0, sinks=False, lse=False, lengths=4),
        # long documents being answered from, and two being read on: few rows, many keys
        dict(name="attend_long", op="attention", shape="7B", page=64, ones=6, chunks=2, chunk=100, ctx=40000,
             window=0, sinks=False, lse=True, lengths=5),
        # a sliding-window layer with sinks on the larger model, small pages
        dict(name="attend_window", op="attention", shape="14B", page=16, ones=24, chunks=4, chunk=900, ctx=6000,
             window=1024, sinks=True, lse=False, lengths=6),
        # many short chats on the draft model
        dict(name="attend_chats", op="attention", shape="0.5B", page=256, ones=200, chunks=8, chunk=120, ctx=600,
             window=0, sinks=False, lse=False, lengths=7),
        # whole prompts: all of it matrix products
        dict(name="attend_prompts", op="attention", shape="7B", page=256, ones=0, chunks=4, chunk=3500, ctx=0,
             window=0, sinks=False, lse=False, lengths=8),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    while True:
        c = dict(op=rng.choice(["rotate", "append", "append", "attention", "attention", "attention"]),
                 shape=rng.choice(list(SHAPES)))
        hd = SHAPES[c["shape"]]["head_dim"]
        if c["op"] == "rotate":
            c.update(tokens=_log_int(rng, 1, 9000), layout=rng.choice(["half", "interleaved"]),
                     rotary=rng.choice([hd, hd, hd // 2, hd // 4]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                     norm=rng.random() < 0.5, scaled=rng.random() < 0.5, far=_log_int(rng, 2048, MAX_KEYS))
        else:
            c.update(page=rng.choice([16, 64, 256, 256]), ones=rng.choice([0, _log_int(rng, 1, 200)]),
                     chunks=rng.choice([0, _log_int(rng, 1, 10)]), chunk=_log_int(rng, 2, 3500),
                     ctx=rng.choice([0, _log_int(rng, 16, 40000)]), lengths=rng.randrange(1 << 20))
            if c["ones"] + c["chunks"] == 0:
                continue
            if c["op"] == "append":
                c.update(layout=rng.choice(["half", "half", "interleaved"]), rotary=rng.choice([hd, hd, hd // 2]),
                         norm=rng.random() < 0.5, scaled=rng.random() < 0.5)
            else:
                c.update(window=rng.choice([0, 0, _log_int(rng, 1, 4096)]), sinks=rng.random() < 0.3,
                         lse=rng.random() < 0.3)
            new, ctx = _lengths(c)
            s = SHAPES[c["shape"]]
            # scores of the plain form's widest (chunk, KV head) product, and the pools
            if int((new * ctx + new * new).max()) * s["n_heads"] // s["n_kv"] > 6e8:
                continue
            if int((new + ctx).sum()) * s["n_kv"] * hd * 4 > 4e9:
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
        # decode tokens sit on ragged conversations, chunks on anything from nothing to that
        c = np.concatenate([np.clip(np.round(rng.lognormal(math.log(ctx), 0.7, size=n1)), 1, MAX_KEYS),
                            rng.integers(0, ctx + 1, size=nc)])
    else:
        c = np.zeros(n1 + nc)
    order = rng.permutation(n1 + nc)
    new, c = new[order], c[order].astype(np.int64)
    return new, np.minimum(c, MAX_KEYS - new)


def _pages(case: dict) -> np.ndarray:
    new, ctx = _lengths(case)
    return -(-(new + ctx) // case["page"])


def _block_table(case: dict, rng) -> np.ndarray:
    """The batch's pages scattered over the pool; columns a sequence does not have are -1."""
    need = _pages(case)
    ids = rng.permutation(int(need.sum()) + 3)
    bt = np.full((len(need), int(need.max())), -1, np.int32)
    off = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[off:off + n]
        off += n
    return bt


def _frequencies(rotary: int, scaled: bool) -> tuple[np.ndarray, float]:
    """Angle per position of each pair, and what cos and sin are multiplied by."""
    i = np.arange(0, rotary, 2, dtype=np.float64)
    freq = THETA ** (-i / rotary)
    if not scaled:
        return freq, 1.0
    f, orig = SCALING["factor"], SCALING["original_max_position_embeddings"]

    def pair_of(turns):  # the pair that turns so often over the original length
        return rotary * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(THETA))

    lo, hi = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), rotary - 1)
    stretch = np.clip((i / 2 - lo) / max(hi - lo, 1e-3), 0.0, 1.0)
    return freq * (1.0 - stretch) + freq / f * stretch, 0.1 * math.log(f) + 1.0


def _tables(rotary: int, n_pos: int, scaled: bool, dev) -> tuple[torch.Tensor, torch.Tensor]:
    if own:
        import prism_amd
        return prism_amd.rotary_tables(rotary, n_pos, THETA, scaling=SCALING if scaled else None, device=dev)
    freq, gain = _frequencies(rotary, scaled)
    angle = torch.outer(torch.arange(n_pos, dtype=torch.float64, device=dev), torch.from_numpy(freq).to(dev))
    return (angle.cos() * gain).float(), (angle.sin() * gain).float()


def _randn(shape, g, dev, dtype=torch.bfloat16, scale=1.0, mean=0.0) -> torch.Tensor:
    return torch.empty(shape, dtype=dtype, device=dev).normal_(mean, scale, generator=g)


def _inputs(case: dict, seed: int) -> dict:
    s, dev = SHAPES[case["shape"]], torch.device("cuda:0")
    nh, nk, hd = s["n_heads"], s["n_kv"], s["head_dim"]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    st = dict(case=case)
    if case["op"] != "attention" and case["norm"]:
        dt = DTYPES[case.get("dtype", "bf16")]
        st["wq"], st["wk"] = (_randn((hd,), g, dev, dt, 0.1, 1.0) for _ in range(2))
    if case["op"] == "rotate":
        dt = DTYPES[case["dtype"]]
        # the fused projection's output: q and k are views of its rows
        qkv = _randn((case["tokens"], (nh + 2 * nk) * hd), g, dev, dt)
        st["q"] = qkv[:, :nh * hd].unflatten(1, (nh, hd))
        st["k"] = qkv[:, nh * hd:(nh + nk) * hd].unflatten(1, (nk, hd))
        st["pos"] = torch.from_numpy(rng.integers(0, case["far"], size=case["tokens"]).astype(np.int32)).to(dev)
        return st
    new, ctx = _lengths(case)
    st.update(new=new, ctx=ctx, bt=_block_table(case, rng))
    pool = (int(_pages(case).sum()) + 3, case["page"], nk, hd)
    st["k_cache"], st["v_cache"] = _randn(pool, g, dev), _randn(pool, g, dev)
    total = int(new.sum())
    if case["op"] == "append":
        st["qkv"] = _randn((total, (nh + 2 * nk) * hd), g, dev)
        return st
    st["q"] = _randn((total, nh, hd), g, dev)
    if case["sinks"]:
        st["sinks"] = _randn((nh,), g, dev, torch.float32, 2.0)
    return st


def prepare(case: dict, seed: int) -> dict:
    st = _inputs(case, seed)
    s, dev = SHAPES[case["shape"]], torch.device("cuda:0")
    if case["op"] != "attention":
        far = case["far"] if case["op"] == "rotate" else int((st["new"] + st["ctx"]).max())
        st["cos"], st["sin"] = _tables(case["rotary"], far, case["scaled"], dev)
    if case["op"] == "rotate":
        return st
    if own:
        import prism_amd
        # the step's batch: lengths, positions, cache slots and the attention's work list, uploaded once per step
        st["batch"] = prism_amd.PackedBatch(st["new"], st["ctx"], st["bt"], page_size=case["page"],
                                            num_pages=st["k_cache"].shape[0], n_heads=s["n_heads"], n_kv=s["n_kv"],
                                            head_dim=s["head_dim"], windows=(case.get("window") or None,), device=dev)
        return st
    # what the plain form indexes with: each token's position and cache slot, each sequence's pages
    pos = np.concatenate([np.arange(c, c + n) for n, c in zip(st["new"], st["ctx"])])
    seq = np.repeat(np.arange(len(st["new"])), st["new"])
    slot = st["bt"][seq, pos // case["page"]].astype(np.int64) * case["page"] + pos % case["page"]
    st["pos"], st["slot"] = torch.from_numpy(pos).to(dev), torch.from_numpy(slot).to(dev)
    st["pages"] = [torch.from_numpy(st["bt"][b, :n].astype(np.int64)).to(dev) for b, n in enumerate(_pages(case))]
    return st


# ---------------------------------------------------------------------------------- the plain forms
def _rotate_plain(x, pos, cos, sin, layout, weight):
    x32 = x.float()
    if weight is not None:
        x32 = x32 * torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS) * weight.float()
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    half = c.shape[-1]
    out = x32.clone()
    if layout == "half":
        a, b = x32[..., :half], x32[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = a * c - b * s, b * c + a * s
    else:
        a, b = x32[..., 0:2 * half:2], x32[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    return out.to(x.dtype)


def _attention_plain(st: dict):
    case, s = st["case"], SHAPES[st["case"]["shape"]]
    nh, nk, hd = s["n_heads"], s["n_kv"], s["head_dim"]
    g, q, dev = nh // nk, st["q"], st["q"].device
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
    first = 0
    for b, (n, c) in enumerate(zip(st["new"].tolist(), st["ctx"].tolist())):
        keys = st["k_cache"][st["pages"][b]].reshape(-1, nk, hd)[:c + n]
        vals = st["v_cache"][st["pages"][b]].reshape(-1, nk, hd)[:c + n]
        t = torch.arange(c + n, device=dev)
        p = torch.arange(c, c + n, device=dev)[:, None]
        hidden = t > p
        if case["window"]:
            hidden = hidden | (t <= p - case["window"])
        for h in range(nk):
            qh = q[first:first + n, h * g:(h + 1) * g].float().transpose(0, 1).reshape(g * n, hd)
            sc = (qh @ keys[:, h].float().t()) / math.sqrt(hd)
            sc = sc.view(g, n, c + n).masked_fill(hidden, -math.inf)
            m = sc.amax(-1, keepdim=True)
            if case["sinks"]:
                m = torch.maximum(m, st["sinks"][h * g:(h + 1) * g, None, None])
            e = torch.exp(sc - m)
            l = e.sum(-1, keepdim=True)
            if case["sinks"]:
                l = l + torch.exp(st["sinks"][h * g:(h + 1) * g, None, None] - m)
            o = (e.view(g * n, -1) @ vals[:, h].float()).view(g, n, hd) / l
            out[first:first + n, h * g:(h + 1) * g] = o.transpose(0, 1).to(out.dtype)
            lse[first:first + n, h * g:(h + 1) * g] = (m + torch.log(l))[..., 0].t()
        first += n
    return [out, lse] if case["lse"] else [out]


def _run_plain(st: dict):
    case, s = st["case"], SHAPES[st["case"]["shape"]]
    nh, nk, hd = s["n_heads"], s["n_kv"], s["head_dim"]
    if case["op"] == "attention":
        return _attention_plain(st)
    rot = (st["pos"], st["cos"], st["sin"], case["layout"])
    if case["op"] == "rotate":
        return [_rotate_plain(st["q"], *rot, st.get("wq")), _rotate_plain(st["k"], *rot, st.get("wk"))]
    qkv = st["qkv"]
    q = _rotate_plain(qkv[:, :nh * hd].unflatten(1, (nh, hd)), *rot, st.get("wq"))
    k = _rotate_plain(qkv[:, nh * hd:(nh + nk) * hd].unflatten(1, (nk, hd)), *rot, st.get("wk"))
    st["k_cache"].view(-1, nk, hd)[st["slot"]] = k
    st["v_cache"].view(-1, nk, hd)[st["slot"]] = qkv[:, (nh + nk) * hd:].unflatten(1, (nk, hd))
    return [q, st["k_cache"], st["v_cache"]]


# ---------------------------------------------------------------------------------- one pass
def _run_own(st: dict):
    import prism_amd
    case = st["case"]
    if case["op"] == "attention":
        r = prism_amd.packed_attention(st["q"], st["k_cache"], st["v_cache"], st["batch"],
                                       window=case["window"] or None, sinks=st.get("sinks"), return_lse=case["lse"])
        return list(r) if case["lse"] else [r]
    how = dict(interleaved=case["layout"] == "interleaved", q_norm_w=st.get("wq"), k_norm_w=st.get("wk"), eps=EPS)
    if case["op"] == "rotate":
        return list(prism_amd.rotate_qk(st["q"], st["k"], st["pos"], st["cos"], st["sin"], **how))
    q = prism_amd.packed_rope_append(st["qkv"], st["k_cache"], st["v_cache"], st["batch"], st["cos"], st["sin"], **how)
    return [q, st["k_cache"], st["v_cache"]]


def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------- what a pass needs
def work(case: dict) -> dict:
    s = SHAPES[case["shape"]]
    nh, nk, hd = s["n_heads"], s["n_kv"], s["head_dim"]
    if case["op"] != "attention":
        size = DTYPES[case.get("dtype", "bf16")].itemsize
        if case["op"] == "rotate":
            tokens, moved = case["tokens"], (nh + nk) * hd * 2
            rows = min(tokens, case["far"])
            index = 4
        else:
            new, ctx = _lengths(case)
            tokens, moved = int(new.sum()), (nh + 2 * nk) * hd * 2
            rows = min(tokens, int((new + ctx).max()))
            index = 8
        # activations in and out, one row of cos and of sin per position, the positions and slots
        nbytes = tokens * (moved * size + index) + rows * case["rotary"] * 4 + (2 * hd * size if case["norm"] else 0)
        return dict(bytes=float(nbytes),
                    flops=float(tokens * (nh + nk) * (case["rotary"] * 3 + (hd * 4 if case["norm"] else 0))))
    new, ctx = (a.astype(np.float64) for a in _lengths(case))
    w = float(case["window"] or 1 << 40)
    # keys that some row sees: all, or those from the first row's window on; and the pairs (row, key) it sees
    keys = np.minimum(ctx, w - 1) + new
    short = np.clip(w - ctx, 0, new)  # rows whose window reaches the first key: they see ctx + 1, ctx + 2, ...
    pairs = short * ctx + short * (short + 1) / 2 + (new - short) * w if case["window"] else \
        new * ctx + new * (new + 1) / 2
    tokens = float(new.sum())
    nbytes = float(keys.sum()) * nk * hd * 4 + tokens * nh * (hd * 4 + (4 if case["lse"] else 0)) \
        + 4 * float(np.ceil(keys / case["page"]).sum()) + 8 * len(new)
    return dict(bytes=nbytes, flops=4.0 * nh * hd * float(pairs.sum()))


# ---------------------------------------------------------------------------------- 64 bits
def _angles64(case: dict, pos: torch.Tensor) -> tuple[torch.Tensor, float]:
    freq, gain = _frequencies(case["rotary"], case["scaled"])
    return pos.double()[:, None] * torch.from_numpy(freq).to(pos.device)[None], gain


def _rotated64(case: dict, x: torch.Tensor, pos: torch.Tensor, weight) -> torch.Tensor:
    """Each pair as a complex number, turned by its angle."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS) * weight.double()
    angle, gain = _angles64(case, pos)
    turn = torch.polar(torch.full_like(angle, gain), angle)[:, None]
    rd = case["rotary"]
    part = y[..., :rd]
    pairs = part.unflatten(-1, (2, rd // 2)).transpose(-1, -2) if case["layout"] == "half" else \
        part.unflatten(-1, (rd // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else z.flatten(-2)
    return torch.cat([z, y[..., rd:]], -1)


def _attention64(st: dict) -> list:
    case, s, dev = st["case"], SHAPES[st["case"]["shape"]], st["q"].device
    g = s["n_heads"] // s["n_kv"]
    outs, lses = [], []
    first = 0
    for b, (n, c) in enumerate(zip(st["new"].tolist(), st["ctx"].tolist())):
        at = torch.arange(c + n)
        pages = torch.from_numpy(st["bt"][b].astype(np.int64))[at // case["page"]].to(dev)
        rows = (at % case["page"]).to(dev)
        behind = torch.arange(c, c + n, device=dev)[:, None] - at.to(dev)   # how far each key lies back
        seen = (behind >= 0) & (behind < (case["window"] or MAX_KEYS + 1))
        o, z = [], []
        for h in range(s["n_heads"]):
            if h % g == 0:
                k, v = (st[x][pages, rows, h // g].double() for x in ("k_cache", "v_cache"))
            sc = st["q"][first:first + n, h].double() @ k.t() * s["head_dim"] ** -0.5
            sc = torch.where(seen, sc, -math.inf)
            norm = torch.logsumexp(sc, -1, keepdim=True)
            if case["sinks"]:
                norm = torch.logaddexp(norm, st["sinks"][h].double())
            o.append(torch.exp(sc - norm) @ v)
            z.append(norm[:, 0])
        outs.append(torch.stack(o, 1))
        lses.append(torch.stack(z, 1))
        first += n
    return [torch.cat(outs), torch.cat(lses)] if case["lse"] else [torch.cat(outs)]


def exact(case: dict, seed: int):
    st = _inputs(case, seed)
    if case["op"] == "attention":
        return _attention64(st)
    if case["op"] == "rotate":
        return [_rotated64(case, st["q"], st["pos"], st.get("wq")), _rotated64(case, st["k"], st["pos"], st.get("wk"))]
    s = SHAPES[case["shape"]]
    nh, nk, hd = s["n_heads"], s["n_kv"], s["head_dim"]
    dev = st["qkv"].device
    q, k, v = st["qkv"].split([nh * hd, nk * hd, nk * hd], 1)
    pos = torch.cat([torch.arange(c, c + n) for n, c in zip(st["new"].tolist(), st["ctx"].tolist())]).to(dev)
    kc, vc = st["k_cache"].double(), st["v_cache"].double()
    k64 = _rotated64(case, k.unflatten(1, (nk, hd)), pos, st.get("wk"))
    first = 0
    for b, (n, c) in enumerate(zip(st["new"].tolist(), st["ctx"].tolist())):
        at = torch.arange(c, c + n)
        page = torch.from_numpy(st["bt"][b].astype(np.int64))[at // case["page"]].to(dev)
        row = (at % case["page"]).to(dev)
        kc[page, row] = k64[first:first + n]
        vc[page, row] = v[first:first + n].unflatten(1, (nk, hd)).double()
        first += n
    return [_rotated64(case, q.unflatten(1, (nh, hd)), pos, st.get("wq")), kc, vc]
