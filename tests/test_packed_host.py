"""The packed step without a GPU: work lists, slots, tables, refusals."""
import math

import numpy as np
import pytest
import torch

import prism_amd
from oracle import epilogue
from oracle import packed as op
from oracle import paged_attention as pa
from pkv_testutil import PAIR_CASES, pair_tolerance
from prism_amd import _lib
from prism_amd.kv_cache import FlashAttnKVCache

A16 = 1 << 20


def _plan(new, ctx, nh, nk, hd, window=0, cus=256):
    lib = _lib.load()
    new, ctx = np.asarray(new, np.int32), np.asarray(ctx, np.int32)
    counts = np.zeros(4, np.int32)
    args = (new.ctypes.data, ctx.ctypes.data, len(new), nh, nk, hd, window, cus)
    assert lib.pkv_packed_plan(*args, 0, 0, 0, 0, counts.ctypes.data) == 0
    items, merges = np.zeros((counts[0], 12), np.int32), np.zeros((max(counts[1], 1), 8), np.int32)
    assert lib.pkv_packed_plan(*args, items.ctypes.data, counts[0], merges.ctypes.data, counts[1], counts.ctypes.data) == 0
    return items, merges[:counts[1]], counts


@pytest.mark.parametrize("nh,nk,hd", [(28, 4, 128), (14, 2, 64), (7, 1, 128), (40, 8, 128), (300, 2, 64), (64, 64, 128)])
@pytest.mark.parametrize("window", [0, 1, 33, 1000])
@pytest.mark.parametrize("cus", [256, 8, 1])
def test_plan_covers_every_visible_key_once(nh, nk, hd, window, cus):
    rng = np.random.default_rng(nh + window + cus)
    for trial in range(6):
        n = int(rng.integers(0, 40))
        new = np.where(rng.random(n) < 0.6, 1, rng.integers(0, 700, n)) * (rng.random(n) < 0.9)
        ctx = rng.integers(0, [1, 50, 3000, 60000][trial % 4], n) if n else new
        items, merges, counts = _plan(new, ctx, nh, nk, hd, window, cus)
        g, tok = nh // nk, 32 if hd == 128 else 64
        tok0 = np.cumsum(new) - new
        stages, slots = {}, []
        marks = {}
        for t0, s, c, b, row0, st0, ns, slot, first, count, *_ in items.tolist():
            marks.setdefault((b, row0), set()).add((first, count))
            assert (t0, s, c) == (tok0[b], new[b], ctx[b]) and s > 0 and ns > 0 and row0 % 128 == 0 and row0 < s * g
            stages.setdefault((b, row0), []).append((st0, ns, slot))
            if slot >= 0:
                slots.append(slot)
        assert sorted(slots) == list(range(counts[2]))
        assert set(stages) == {(b, r) for b in range(n) for r in range(0, int(new[b]) * g, 128)}
        for (b, row0), parts in stages.items():
            last = ctx[b] + (min(row0 + 128, new[b] * g) - 1) // g
            first = max(ctx[b] + row0 // g - window + 1, 0) if window else 0
            parts.sort()
            at = first // tok
            for st0, ns, slot in parts:
                assert st0 == at and (slot >= 0) == (len(parts) > 1)
                at += ns
            assert at == last // tok + 1
        split = {}
        for (b, row0), parts in stages.items():
            rows = min(128, new[b] * g - row0)
            if len(parts) == 1:
                assert marks[b, row0] == {(0, 0)}
            elif rows <= 32 and len(parts) <= 64:   # merged by the last range to end
                ((first, count),) = marks[b, row0]
                assert sorted(p[2] for p in parts) == list(range(first, first + count))
            else:
                assert marks[b, row0] == {(0, 0)}
                split[b, row0] = parts
        assert len(merges) == len(split)
        for t0, s, row0, slot, count, *_ in merges.tolist():
            (b,) = [b for b in range(n) if tok0[b] == t0 and new[b] == s and (b, row0) in split]
            assert sorted(p[2] for p in split[b, row0]) == list(range(slot, slot + count))
            assert counts[3] >= min(128, s * g - row0)
        assert counts[3] <= 128


def _ends(new, ctx, nh, nk, hd, window=0, cus=256):
    """The planner's schedule, replayed: when its list ends, when the blocks would end whole, an even share of the work,
    and blocks per slot.  A range costs its stages and five, a piece of a block up to eight more, by its rows."""
    import heapq
    g, tok, slots = nh // nk, 32 if hd == 128 else 64, max(2 * cus // nk, 1)
    blocks = {}
    for b, (n, c) in enumerate(zip(new, ctx)):
        for r0 in range(0, n * g, 128):
            rows = min(128, n * g - r0)
            first = max(c + r0 // g - window + 1, 0) if window else 0
            blocks[b, r0] = ((c + (r0 + rows - 1) // g) // tok + 1 - first // tok, rows)

    def end(costs):
        load = [0] * slots
        for cost in costs:
            heapq.heapreplace(load, load[0] + cost)
        return max(load)
    listed = []
    for it in _plan(new, ctx, nh, nk, hd, window, cus)[0].tolist():
        stages, rows = blocks[it[3], it[4]]
        listed.append(it[6] + 5 + (-(-8 * rows // 128) if it[6] < stages else 0))
    whole = [stages + 5 for stages, _ in sorted(blocks.values(), key=lambda x: -x[0])]
    return end(listed), end(whole), sum(whole) / slots, len(blocks) / slots


SHAPES = [(28, 4, 128), (14, 2, 64), (40, 8, 128), (7, 1, 128)]


def test_plan_is_not_worse_than_whole_blocks():
    """Where the blocks are more than the slots, cutting them never ends later than leaving them whole."""
    seen = 0
    for chunks, n, c, w, s in [(6, 1000, 4000, 512, 0), (4, 2048, 8000, 2048, 1), (4, 700, 4000, 1024, 2), (3, 3500, 0, 2048, 3),
                               (2, 2048, 1000, 1024, 0), (8, 500, 4000, 1024, 0), (5, 500, 1000, 0, 2), (2, 1500, 1000, 0, 0)]:
        listed, whole, _, per_slot = _ends([n] * chunks, [c] * chunks, *SHAPES[s], w)
        assert per_slot > 1 and listed <= whole, (chunks, n, c, w, s)
    rng = np.random.default_rng(5)
    for trial in range(300):
        n = int(rng.integers(1, 300))
        new = np.where(rng.random(n) < rng.random(), 1, rng.integers(1, 900, n)).tolist()
        ctx = rng.integers(0, int(rng.choice([1, 600, 5000, 30000])), n).tolist()
        listed, whole, _, per_slot = _ends(new, ctx, *SHAPES[trial % 4], int(rng.choice([0, 0, 100, 1024])))
        if per_slot > 1:
            seen += 1
            assert listed <= whole, trial
    assert seen > 100


def test_plan_cuts_a_long_block_among_many():
    """Rounds of short blocks even out by themselves, one long block beside them does not: a document of 100,000 keys
    among 1100 chats, a chunk on 30,000 keys among them, one document among 9000 sequences."""
    for new, ctx, s in [([1] * 1101, [400] * 1100 + [100000], 0), ([1] * 1100 + [600], [400] * 1100 + [30000], 0),
                        ([1] * 9001, [16] * 4500 + [120000] + [16] * 4500, 2)]:
        listed, whole, share, per_slot = _ends(new, ctx, *SHAPES[s])
        assert per_slot > 8 and whole > 2 * share
        assert listed <= 1.1 * share + 20, (listed, whole, share)     # 20: a piece's start, cut and end
    # and equal blocks stay whole, however many
    items, merges, counts = _plan([1] * 9000, [100] * 9000, *SHAPES[2])
    assert counts[0] == 9000 and counts[2] == 0


def test_layout_refusals():
    lib = _lib.load()
    one, bt, out = np.array([1], np.int32), np.array([[3]], np.int32), np.zeros(4, np.int32)

    def call(new=one, ctx=one, batch=1, bt=bt, bts=1, mb=1, page=16, pages=4, window=0, pos=out.ctypes.data):
        return lib.pkv_packed_layout(new.ctypes.data, ctx.ctypes.data, batch, bt.ctypes.data, bts, mb, page, pages, window,
                                     pos, out.ctypes.data)
    assert call() == 0 and out[0] == 3 * 16 + 1
    for bad in [dict(page=8), dict(page=24), dict(pages=3), dict(pages=0), dict(pages=1 << 30), dict(mb=2), dict(batch=-1),
                dict(window=-1), dict(pos=0), dict(new=np.array([16], np.int32)), dict(bt=np.array([[-1]], np.int32)),
                dict(ctx=np.array([-1], np.int32)), dict(ctx=np.array([1 << 27], np.int32))]:
        assert call(**bad) == _lib.PKV_EINVAL, bad
        assert "pkv_packed_layout" in lib.pkv_last_error().decode()


def test_plan_refusals():
    lib = _lib.load()
    c = np.zeros(4, np.int32)
    one, neg, big = np.array([1], np.int32), np.array([-1], np.int32), np.array([1 << 27], np.int32)

    def call(new=one, ctx=one, batch=1, nh=4, nk=2, hd=128, window=0, cus=256, counts=c.ctypes.data, mi=0, items=0):
        return lib.pkv_packed_plan(new.ctypes.data if new is not None else 0, ctx.ctypes.data, batch, nh, nk, hd, window,
                                   cus, items, mi, 0, 0, counts)
    assert call() == 0
    for bad in [dict(new=neg), dict(ctx=neg), dict(ctx=big), dict(nh=3), dict(nk=0), dict(hd=96), dict(window=-1),
                dict(cus=0), dict(batch=-1), dict(counts=0), dict(new=None), dict(new=big, ctx=np.zeros(1, np.int32), nh=64)]:
        assert call(**bad) == _lib.PKV_EINVAL, bad
        assert "pkv_packed_plan" in lib.pkv_last_error().decode()
    room = np.zeros(12, np.int32)
    assert call(items=room.ctypes.data, mi=0) == _lib.PKV_ENOSPC


def _batch(**over):
    a = dict(new_lens=[1, 0, 300], cache_lens=[500, 3, 7], block_table=[[1, 2], [-1, -1], [4, 5]], page_size=256, num_pages=9,
             n_heads=28, n_kv=4, head_dim=128, device="cpu")
    a.update(over)
    return prism_amd.PackedBatch(a.pop("new_lens"), a.pop("cache_lens"), a.pop("block_table"), **a)


def test_batch_positions_and_slots():
    b = _batch(windows=(None, 64, None))
    assert b.total_tokens == 301 and list(b._plans) == [None, 64]
    assert b.positions.tolist() == [500] + list(range(7, 307))
    assert b.slots.tolist() == [2 * 256 + 244] + [(4 if t < 256 else 5) * 256 + t % 256 for t in range(7, 307)]
    assert b.block_table.tolist() == [[1, 2], [-1, -1], [4, 5]]
    empty = _batch(new_lens=[], cache_lens=[], block_table=np.zeros((0, 1), np.int32))
    assert empty.total_tokens == 0 and empty.positions.numel() == 0
    none = _batch(new_lens=[0, 0, 0])
    assert none.total_tokens == 0 and none._plans[None][2] == 0
    # pages wholly before the window may be gone
    _batch(new_lens=[1, 0, 0], block_table=[[-1, 2], [-1, -1], [-1, -1]], windows=(100,))


@pytest.mark.parametrize("over,msg", [
    (dict(new_lens=[1, 0]), "block-table rows"),
    (dict(new_lens=[1, 0, -3]), "negative"),
    (dict(cache_lens=[500, 3, 1 << 27]), "2\\^27"),
    (dict(new_lens=[1.0, 0.0, 3.0]), "integers"),
    (dict(block_table=[[1, 2, 3, 4, 5, 6]]), "block-table rows"),
    (dict(new_lens=[1, 0, 600]), "columns"),
    (dict(block_table=[[1, 9], [-1, -1], [4, 5]]), "outside"),
    (dict(block_table=[[-1, 2], [-1, -1], [4, 5]]), "outside"),
    (dict(block_table=[[1, 2], [-1, -1], [4, 2]]), "one page"),
    (dict(block_table=[[1, 2], [-1, -1], [4, 4]]), "one page"),
    (dict(page_size=48), "power of two"),
    (dict(page_size=8), "power of two"),
    (dict(num_pages=0), "pool"),
    (dict(num_pages=1 << 24), "pool"),
    (dict(num_pages=1 << 32), "pool"),
    (dict(page_size=(1 << 32) + 16), "pool"),
    (dict(new_lens=[1 << 26, 0, 1]), "2\\^30"),
    (dict(new_lens=[1 << 33, 0, 1]), "int32"),
    (dict(new_lens=[-(1 << 30), 1 << 20, 1]), "negative"),
    (dict(head_dim=96), "head_dim"),
    (dict(n_heads=30), "multiple"),
    (dict(windows=()), "at least one"),
    (dict(windows=(0,)), "window"),
    (dict(windows=(2.5,)), "window"),
    (dict(windows=(True,)), "window"),
])
def test_batch_refusals(over, msg):
    with pytest.raises(RuntimeError, match=msg):
        _batch(**over)


def test_ops_need_the_device():
    b = _batch()
    x = torch.zeros(301, 36 * 128, dtype=torch.bfloat16)
    cache = torch.zeros(9, 256, 4, 128, dtype=torch.bfloat16)
    cos, sin = prism_amd.rotary_tables(128, 4, device="cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        prism_amd.packed_rope_append(x, cache, cache, b, cos, sin)
    with pytest.raises(RuntimeError, match="no CPU path"):
        prism_amd.packed_attention(x[:, :3584].view(301, 28, 128), cache, cache, b)
    with pytest.raises(RuntimeError, match="no CPU path"):
        prism_amd.rotate_qk(x.view(301, 36, 128), None, torch.zeros(301, dtype=torch.int32), cos, sin)


def test_cache_builds_the_batch():
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    kv.new_sequence(1)
    kv.new_sequence(2)
    kv.prepare_append([1, 2], [20, 1])
    kv.update_seqlens([1, 2], [20, 1])
    with pytest.raises(RuntimeError, match="prepare_append"):
        kv.build_packed_batch([1, 2], [40, 1], 14)
    with pytest.raises(ValueError, match="twice"):
        kv.build_packed_batch([1, 1], 1, 14)
    with pytest.raises(ValueError, match="counts"):
        kv.build_packed_batch([1, 2], [1], 14)
    kv.prepare_append([1, 2], [40, 1])
    b = kv.build_packed_batch([2, 1], [1, 40], 14, windows=(None, 8))
    pages = kv.seq_pages
    assert b.positions.tolist() == [1] + list(range(20, 60))
    assert b.slots.tolist() == [pages[2][0] * 16 + 1] + [pages[1][t // 16] * 16 + t % 16 for t in range(20, 60)]
    kv.fork_sequence(2, 3)
    with pytest.raises(RuntimeError, match="shared"):
        kv.build_packed_batch([3], 1, 14)
    assert kv.build_packed_batch([], [], 14).total_tokens == 0


# ---------------------------------------------------------------------------------- tables
def _yarn(rd, theta, f, orig, fast=32.0, slow=1.0):
    """Pair by pair: turns over the original length decide between the plain and the stretched frequency."""
    out = []
    number = lambda turns: rd * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
    lo, hi = max(math.floor(number(fast)), 0), min(math.ceil(number(slow)), rd - 1)
    for i in range(rd // 2):
        plain = theta ** (-2 * i / rd)
        r = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
        out.append(plain * (1 - r) + plain / f * r)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("rd,theta,n_pos,scaling", [
    (128, 1e6, 70000, None), (64, 1e4, 3, None), (2, 1e4, 5, None),
    (64, 1e4, 900, dict(rope_type="linear", factor=8.0)),
    (64, 1e4, 900, dict(rope_type="default")),
    (32, 1e4, 9000, dict(type="dynamic", factor=2.0, original_max_position_embeddings=2048)),
    (32, 1e4, 900, dict(type="dynamic", factor=2.0, original_max_position_embeddings=2048)),
    (128, 1e6, 131072, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)),
    (64, 1e4, 500, dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=2048, beta_fast=20, beta_slow=2,
                        attention_factor=1.0)),
])
def test_rotary_tables(rd, theta, n_pos, scaling):
    cos, sin = prism_amd.rotary_tables(rd, n_pos, theta, scaling=scaling, device="cpu")
    assert cos.shape == sin.shape == (n_pos, rd // 2) and cos.dtype == torch.float32
    kind = (scaling or {}).get("rope_type", (scaling or {}).get("type"))
    freq, gain = theta ** (-torch.arange(rd // 2, dtype=torch.float64) * 2 / rd), 1.0
    if kind == "linear":
        freq = freq / scaling["factor"]
    elif kind == "dynamic":
        orig, f = 2048, 2.0
        base = theta * max(f * max(n_pos, orig) / orig - f + 1, 1.0) ** (rd / (rd - 2))
        freq = base ** (-torch.arange(rd // 2, dtype=torch.float64) * 2 / rd)
    elif kind == "yarn":
        freq = _yarn(rd, theta, scaling["factor"], scaling["original_max_position_embeddings"],
                     scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0))
        gain = scaling.get("attention_factor", 0.1 * math.log(scaling["factor"]) + 1)
    pos = torch.unique(torch.tensor([0, 1, n_pos // 2, n_pos - 1]).clamp(max=n_pos - 1))
    angle = pos.double()[:, None] * freq
    # the fp64 angle is off by a few 2^-53 of up to n_pos radians; then one rounding to 24 bits
    tol = gain * (2.0 ** -24 + 8 * n_pos * 2.0 ** -53)
    assert (cos[pos].double() - angle.cos() * gain).abs().max() <= tol
    assert (sin[pos].double() - angle.sin() * gain).abs().max() <= tol


def test_rotary_tables_frequencies_and_refusals():
    f = torch.tensor([0.5, 0.25])
    cos, sin = prism_amd.rotary_tables(4, 3, inv_freq=f, gain=2.0, device="cpu")
    assert torch.allclose(cos[2], 2 * torch.cos(2 * f)) and torch.allclose(sin[1], 2 * torch.sin(f))
    for kw in [dict(rotary_dim=3), dict(rotary_dim=0), dict(n_pos=0), dict(theta=1.0), dict(inv_freq=torch.ones(3)),
               dict(inv_freq=torch.ones(2), scaling=dict(rope_type="linear", factor=2.0)),
               dict(scaling=dict(rope_type="linear", factor=0.5)), dict(scaling=dict(rope_type="ntk", factor=2.0)),
               dict(rotary_dim=2, scaling=dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=8)),
               dict(scaling=dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=8, beta_fast=1, beta_slow=2)),
               dict(scaling=dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=0))]:
        a = dict(rotary_dim=4, n_pos=3, device="cpu")
        a.update(kw)
        with pytest.raises(ValueError):
            prism_amd.rotary_tables(a.pop("rotary_dim"), a.pop("n_pos"), **a)


def _yarn_dict(**over):
    return dict(rope_type="yarn", factor=32.0, original_max_position_embeddings=4096, **over)


def _yarn_ends(rd, theta, orig, fast=32.0, slow=1.0):
    """The pairs that turn `fast` and `slow` times over the original length, not rounded to whole pairs."""
    return [rd * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (fast, slow)]


@pytest.mark.parametrize("rd,theta", [(64, 150000.0), (128, 1e6), (32, 1e4)])
def test_yarn_ramp_not_rounded(rd, theta):
    """truncate: false keeps the ramp's ends where they fall between two pairs."""
    lo, hi = _yarn_ends(rd, theta, 4096)
    if rd == 64:
        assert abs(lo - 8.09) < 0.01 and abs(hi - 17.40) < 0.01
    freq, gain = prism_amd.epilogue._scaled_frequencies(rd, 9, theta, _yarn_dict(truncate=False))
    for i in range(rd // 2):
        plain, r = theta ** (-2 * i / rd), min(max((i - lo) / (hi - lo), 0.0), 1.0)
        want = plain * (1 - r) + plain / 32.0 * r
        assert abs(float(freq[i]) - want) <= 1e-12 * plain, i      # a few 2^-53 per power, quotient and product
    assert abs(gain - (0.1 * math.log(32.0) + 1)) < 1e-15
    whole, _ = prism_amd.epilogue._scaled_frequencies(rd, 9, theta, _yarn_dict())
    same, _ = prism_amd.epilogue._scaled_frequencies(rd, 9, theta, _yarn_dict(truncate=True))
    assert torch.equal(whole, same) and not torch.equal(whole, freq)


@pytest.mark.parametrize("a,b", [(1.0, 1.0), (0.707, 0.707), (1.0, 0.5), (0.5, 2)])
def test_yarn_gain_of_two_scales(a, b):
    """mscale and mscale_all_dim: cos and sin take the ratio of their two gains, the attention's scale the rest."""
    _, gain = prism_amd.epilogue._scaled_frequencies(64, 9, 1e4, _yarn_dict(mscale=a, mscale_all_dim=b))
    assert abs(gain - (0.1 * a * math.log(32.0) + 1) / (0.1 * b * math.log(32.0) + 1)) < 1e-15
    _, gain = prism_amd.epilogue._scaled_frequencies(64, 9, 1e4, _yarn_dict(mscale=a, mscale_all_dim=b, attention_factor=1.25))
    assert gain == 1.25


def test_scaling_none_is_absent():
    full = _yarn_dict(beta_fast=None, beta_slow=None, attention_factor=None, truncate=None, mscale=None, mscale_all_dim=None,
                      type="yarn", low_freq_factor=None)
    a, b = (prism_amd.epilogue._scaled_frequencies(64, 9, 1e4, s) for s in (full, _yarn_dict()))
    assert torch.equal(a[0], b[0]) and a[1] == b[1]
    for s in ({}, dict(rope_type=None), dict(rope_type="default", factor=None)):
        f, gain = prism_amd.epilogue._scaled_frequencies(8, 9, 1e4, s)
        assert torch.equal(f, 1e4 ** (-torch.arange(0, 8, 2, dtype=torch.float64) / 8)) and gain == 1.0


@pytest.mark.parametrize("scaling", [
    dict(factor=4.0), dict(rope_type="default", factor=4.0), dict(type="linear", factor=4.0, original=8),
    dict(rope_type="yarn", type="linear", factor=4.0, original_max_position_embeddings=8),
    dict(rope_type="linear", factor=4.0, beta_fast=32.0), dict(rope_type="linear", factor=None),
    dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=8, attention_factor=1.0),
    _yarn_dict(mscale=1.0), _yarn_dict(mscale_all_dim=1.0), _yarn_dict(mscale=0.0, mscale_all_dim=1.0),
    _yarn_dict(mscale=1.0, mscale_all_dim=-1.0), _yarn_dict(mscale=1.0, mscale_all_dim=math.nan), _yarn_dict(truncate=0.5), _yarn_dict(short_factor=[1.0]),
    _yarn_dict(rope_theta=1e4), _yarn_dict(partial_rotary_factor=0.5), _yarn_dict(finetuned=True),
    _yarn_dict(beta_fast=float("nan")), dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192),
])
def test_scaling_keys_that_are_not_understood(scaling):
    """Nothing that would change the tables is passed over."""
    with pytest.raises(ValueError):
        prism_amd.rotary_tables(64, 3, scaling=scaling, device="cpu")


def test_tables_argument_errors():
    lib = _lib.load()
    f = np.ones(4)
    ok = dict(freq=f.ctypes.data, half=3, n_pos=3, cos=A16, sin=A16)
    for bad in [dict(freq=0), dict(half=0), dict(n_pos=0), dict(n_pos=1 << 31), dict(cos=0), dict(sin=A16 + 2)]:
        assert lib.pkv_rotary_tables(*{**ok, **bad}.values(), None) == _lib.PKV_EINVAL, bad
        assert "pkv_rotary_tables" in lib.pkv_last_error().decode()


def test_oracle_rotation_is_the_others():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 3, 64, generator=g, dtype=torch.float64)
    pos = torch.tensor([0, 1, 77, 4095, 100000])
    f = 1e4 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    half, mag = op.rotate64(x, pos, f)
    want = epilogue.rope_f64(x.numpy(), pos.numpy()[:, None], 64)
    assert np.abs(half.numpy() - want).max() < 1e-9      # the angles of 100000 agree to 2^-53 of it
    assert (mag >= half.abs() - 1e-12).all()
    order = torch.arange(64).view(2, 32).t().flatten()   # pairs side by side
    inter, _ = op.rotate64(x[..., order], pos, f, interleaved=True)
    assert torch.equal(inter, half[..., order])
    w = torch.rand(64, generator=g, dtype=torch.float64)
    norm, _ = op.rotate64(x, torch.zeros(5), f, norm_w=w, eps=1e-3)
    assert (norm - torch.nn.functional.rms_norm(x, (64,), w, 1e-3)).abs().max() < 1e-12
    part, _ = op.rotate64(x, pos, f[:8])
    assert torch.equal(part[..., 16:], x[..., 16:])


def test_oracle_attention_is_the_other():
    g = torch.Generator().manual_seed(4)
    kc, vc = (torch.randn(9, 16, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(3, 4, 6, 64, generator=g).to(torch.bfloat16)
    ctx, bt = [20, 0, 33], torch.tensor([[3, 1, 8], [5, 0, 0], [2, 7, 4]])
    out, lse, mag = op.packed_attention64(q.flatten(0, 1), kc, vc, [4] * 3, ctx, bt)
    want = pa.attention_fp64(pa.bf16_bits(q), pa.bf16_bits(kc), pa.bf16_bits(vc), bt.numpy(), np.array(ctx) + 4, True)
    assert np.abs(out.view(3, 4, 6, 64).numpy() - want).max() < 1e-12 and (mag >= out.abs() - 1e-12).all()
    # row by row, with a window and sinks
    sinks = torch.tensor([-1e30, 0.0, 3.0, 50.0, -2.0, 1.0])
    out, lse, _ = op.packed_attention64(q.flatten(0, 1)[:7], kc, vc, [2, 0, 5], ctx, bt, window=6, sinks=sinks, scale=0.2)
    for row, (b, p) in enumerate([(0, 20), (0, 21), (2, 33), (2, 34), (2, 35), (2, 36), (2, 37)]):
        for h in range(6):
            e, num = math.exp(sinks[h].double()), torch.zeros(64, dtype=torch.float64)
            for t in range(max(p - 5, 0), p + 1):
                page, r = int(bt[b, t // 16]), t % 16
                x = math.exp(0.2 * float(q.flatten(0, 1)[row, h].double() @ kc[page, r, h // 3].double()))
                e, num = e + x, num + x * vc[page, r, h // 3].double()
            assert (out[row, h] - num / e).abs().max() < 1e-12 and abs(float(lse[row, h]) - math.log(e)) < 1e-12


def test_oracle_rotation_gradient():
    """The rotation is linear in the head: its gradient is the rotation by the opposite angle."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 2, 16, generator=g, dtype=torch.float64)
    w = torch.randn(3, 2, 16, generator=g, dtype=torch.float64)
    pos, f = torch.tensor([0, 5, 9]), torch.rand(4, generator=g, dtype=torch.float64)
    for inter in (False, True):
        back, _ = op.rotate64(w, -pos, f, interleaved=inter, gain=1.5)
        for k in range(5):
            d = torch.zeros_like(x)
            d.view(-1)[k * 17] = 1.0
            diff = ((op.rotate64(x + d, pos, f, interleaved=inter, gain=1.5)[0] -
                     op.rotate64(x - d, pos, f, interleaved=inter, gain=1.5)[0]) / 2 * w).sum()
            want = back.clone()
            want[..., 8:] = w[..., 8:]
            assert abs(diff - want.view(-1)[k * 17]) < 1e-12


# ---------------------------------------------------------------------------------- the C entries' refusals
def _rotate(lib, **over):
    a = dict(q=A16, q_st=512, q_sh=128, k=A16, k_st=512, k_sh=128, pos=A16, cos=A16, sin=A16, n_pos=5, qw=0, kw=0, eps=1e-6,
             qo=A16, qo_st=512, qo_sh=128, ko=A16, ko_st=512, ko_sh=128, tokens=3, nh=4, nk=4, hd=128, rd=128, inter=0, dtype=0)
    a.update(over)
    return lib.pkv_rotate_qk(*a.values(), None, None)


@pytest.mark.parametrize("over,msg", [
    (dict(tokens=-1), "bad sizes"), (dict(nh=0), "bad sizes"), (dict(n_pos=0), "bad sizes"), (dict(nk=-1), "bad sizes"),
    (dict(hd=0), "head_dim"), (dict(hd=1025), "head_dim"), (dict(rd=0), "rotary_dim"), (dict(rd=130), "rotary_dim"),
    (dict(rd=63), "rotary_dim"), (dict(cos=0), "null"), (dict(sin=A16 + 2), "aligned"), (dict(eps=-1.0), "eps"),
    (dict(eps=math.nan), "eps"), (dict(dtype=3), "dtype"), (dict(q=0), "null"), (dict(k=0), "null"), (dict(ko=0), "null"),
    (dict(pos=0), "null"), (dict(qo=A16 + 1), "aligned"), (dict(kw=A16 + 1), "aligned"), (dict(q=A16 + 2, dtype=2), "aligned"),
    (dict(nh=70000), "heads"),
])
def test_rotate_argument_errors(over, msg):
    lib = _lib.load()
    assert _rotate(lib, **over) == _lib.PKV_EINVAL
    err = lib.pkv_last_error().decode()
    assert "pkv_rotate_qk" in err and msg in err, err


def test_rotate_nothing_to_do():
    assert _rotate(_lib.load(), tokens=0, q=0, k=0) == 0


def _append(lib, **over):
    a = dict(qkv=A16, st=36 * 128, pos=A16, slots=A16, cos=A16, sin=A16, n_pos=5, qw=0, kw=0, eps=1e-6, qo=A16, qo_st=28 * 128,
             qo_sh=128, kc=A16, vc=A16, ps=256 * 512, tokens=3, nh=28, nk=4, hd=128, rd=128, inter=0, page=256, pages=9)
    a.update(over)
    return lib.pkv_packed_rope_append(*a.values(), None, None)


@pytest.mark.parametrize("over,msg", [
    (dict(hd=96, rd=96), "head_dim"), (dict(rd=24), "rotary_dim"), (dict(nk=0), "bad sizes"), (dict(pages=0), "bad sizes"),
    (dict(page=24), "page_size"), (dict(page=8), "page_size"), (dict(pages=1 << 23), "slots"), (dict(slots=0), "null"),
    (dict(kc=0), "null"), (dict(ps=100), "page stride"), (dict(ps=256 * 512 + 4), "page stride"), (dict(qkv=A16 + 8), "aligned"),
    (dict(st=36 * 128 + 4), "aligned"), (dict(vc=A16 + 8), "aligned"), (dict(cos=A16 + 4), "aligned"),
    (dict(qw=A16 + 4), "aligned"), (dict(qo=A16 + 4), "aligned"), (dict(qo_sh=132), "multiples of 8"), (dict(tokens=-1), "bad sizes"),
])
def test_append_argument_errors(over, msg):
    lib = _lib.load()
    assert _append(lib, **over) == _lib.PKV_EINVAL
    err = lib.pkv_last_error().decode()
    assert "pkv_packed_rope_append" in err and msg in err, err


def _attn(lib, **over):
    a = dict(q=A16, q_st=28 * 128, q_sh=128, kc=A16, vc=A16, ps=256 * 512, bt=A16, bts=4, out=A16, o_st=28 * 128, o_sh=128, lse=0,
             sinks=0, items=A16, n_items=3, merges=A16, n_merges=1, partials=2, merge_rows=7, ws=A16, wsb=1 << 30, tokens=3,
             batch=3, nh=28, nk=4, hd=128, page=256, pages=9, mb=4, window=0, scale=0.1)
    a.update(over)
    return lib.pkv_packed_attn(*a.values(), None, None)


@pytest.mark.parametrize("over,msg", [
    (dict(tokens=-1), "bad sizes"), (dict(n_items=-1), "bad sizes"), (dict(window=-1), "bad sizes"), (dict(hd=96), "head_dim"),
    (dict(page=24), "page_size"), (dict(bts=3), "bt_stride"), (dict(nh=30), "multiple of n_kv"), (dict(q=A16 + 8), "aligned"),
    (dict(o_st=28 * 128 + 4), "multiples of 8"), (dict(lse=A16 + 2), "aligned"), (dict(sinks=A16 + 1), "aligned"),
    (dict(items=0), "null"), (dict(merges=0), "null"), (dict(items=A16 + 4), "aligned"), (dict(n_merges=65536), "too many"),
    (dict(ws=0), "workspace"), (dict(ws=A16 + 8), "workspace"), (dict(scale=math.inf), "softmax_scale"), (dict(kc=0), "null"),
    (dict(n_items=1 << 30), "too many"),
])
def test_attention_argument_errors(over, msg):
    lib = _lib.load()
    assert _attn(lib, **over) == _lib.PKV_EINVAL
    err = lib.pkv_last_error().decode()
    assert "pkv_packed_attn" in err and msg in err, err


def test_attention_workspace():
    lib = _lib.load()
    need = lib.pkv_packed_workspace_bytes(2, 4, 128)
    assert need == 2 * 4 * (128 * 132 * 4 + 8)
    assert lib.pkv_packed_workspace_bytes(0, 4, 128) == 0
    assert _attn(lib, wsb=need - 1) == _lib.PKV_ENOSPC
    assert _attn(lib, n_items=0, items=0, ws=0) == 0


# ---------------------------------------------------------------------------------- the binding
def _in_a_process(code):
    import subprocess
    import sys

    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=str(_lib.FASTCALL_PATH.parents[1]))
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_only_the_packed_step_needs_the_binding():
    """Without _fastcall.so the library loads and its calls go through ctypes, as they do where that module was built
    against another torch; a packed call names what is missing."""
    out = _in_a_process("""
import pathlib
from prism_amd import _lib
_lib.FASTCALL_PATH = pathlib.Path("/nowhere/_fastcall.so")
print(_lib.load().pkv_abi_version())
import prism_amd
kv = prism_amd.FlashAttnKVCache(1, 2, 64, 4, 16, "cpu")
kv.new_sequence(1)
kv.prepare_append([1], 3)
try:
    kv.build_packed_batch([1], 3, 14)
except _lib.PrismKVError as e:
    print(e)
""")
    assert "_fastcall.so is not built" in out and out.startswith("1\n")


def test_the_binding_follows_the_library_in_use():
    """_lib.use after the first packed call: the binding's calls go to the library that is loaded then."""
    stamps = _lib.LIB_PATH.with_name("libprism_kv_stamps.so")
    out = _in_a_process(f"""
import pathlib
from prism_amd import _lib
seen = []
class Fake:
    attach = staticmethod(lambda handle, error: seen.append(handle))
first = _lib.load()
_lib.fast()
_lib._fast = Fake
second = _lib.use(pathlib.Path({str(stamps)!r}))
assert _lib.fast() is Fake
print(seen == [second._handle] and second._handle != first._handle)
""")
    assert out == "True\n"


def test_a_released_batch_keeps_nothing(monkeypatch):
    """A captured call keeps the batch's memory, once; release gives it up, and a later capture keeps it again."""
    import gc
    import weakref

    from prism_amd import packed

    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: True)
    a, b = _batch(), _batch()
    held = len(packed._captured)
    for _ in range(2):
        for x in (a, b, a):
            x._used_on(0)
        assert len(packed._captured) == held + 2
        a.release()
        a.release()
        assert len(packed._captured) == held + 1 and any(t is b._buf for t in packed._captured)
    gone, kept = weakref.ref(a._buf), weakref.ref(b._buf)
    del a, b, x
    gc.collect()
    assert gone() is None and kept() is not None
    packed._captured[:] = [t for t in packed._captured if t is not kept()]


@pytest.mark.parametrize("new,ctx", PAIR_CASES)
@pytest.mark.parametrize("nh,nk,hd", [(7, 1, 128), (14, 2, 64), (8, 8, 128)])
def test_the_pair_tolerance_tells_a_pair_from_one_rounding(new, ctx, nh, nk, hd):
    """Probabilities rounded once to bf16 are outside it, as a pair inside."""
    g, bf = torch.Generator().manual_seed(21), torch.bfloat16
    need = [-(-(n + c) // 64) for n, c in zip(new, ctx)]
    bt = torch.full((len(new), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        bt[b, :n] = torch.arange(sum(need[:b]), sum(need[:b]) + n)
    kc, vc = (torch.randn(sum(need), 64, nk, hd, generator=g).to(bf) for _ in range(2))
    q = torch.randn(sum(new), nh, hd, generator=g).to(bf)
    ref, lse, mag = op.packed_attention64(q, kc, vc, new, ctx, bt)
    got, row = {1: torch.empty_like(ref), 2: torch.empty_like(ref)}, 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        for j in range(n):
            at = torch.arange(c + j + 1)
            k, v = (x[bt[b].long()[at // 64], at % 64].double() for x in (kc, vc))
            for h in range(nh):
                p = torch.exp(k[:, h // (nh // nk)] @ q[row, h].double() / math.sqrt(hd) - lse[row, h])
                hi = p.to(bf).double()
                for parts, pr in ((1, hi), (2, hi + (p - hi).to(bf).double())):
                    got[parts][row, h] = pr @ v[:, h // (nh // nk)]
            row += 1
    tol = pair_tolerance(ref, mag, max(n + c for n, c in zip(new, ctx)))
    assert ((got[2].to(bf).double() - ref).abs() <= tol).all()
    assert ((got[1].to(bf).double() - ref).abs() > tol).any()
