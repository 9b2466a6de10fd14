"""Key weights, eviction and sampling without a GPU: work lists, refusals, the cache's book-keeping."""
import ctypes

import numpy as np
import pytest
import torch

import prism_amd
from oracle import behind as ob
from prism_amd import _lib
from prism_amd.kv_cache import FlashAttnKVCache, KVCacheOutOfPages

A16 = 1 << 20


def _plan(new, ctx, nh, nk, window=0, rows=0, weighed=None, cus=256):
    lib = _lib.load()
    new, ctx = np.asarray(new, np.int32), np.asarray(ctx, np.int32)
    had = None if weighed is None else np.asarray(weighed, np.int32)
    counts = np.zeros(4, np.int32)
    args = (new.ctypes.data, ctx.ctypes.data, 0 if had is None else had.ctypes.data, len(new), nh, nk, window, rows, cus)
    assert lib.pkv_key_weights_plan(*args, 0, 0, counts.ctypes.data) == 0
    items = np.zeros((max(int(counts[:3].sum()), 1), 12), np.int32)
    assert lib.pkv_key_weights_plan(*args, items.ctypes.data, len(items), counts.ctypes.data) == 0
    few, many, merges = np.split(items[:counts[:3].sum()], np.cumsum(counts[:2]))
    return few, many, merges, int(counts[3])


@pytest.mark.parametrize("nh,nk", [(28, 4), (14, 2), (7, 1), (300, 2), (8, 8)])
@pytest.mark.parametrize("window", [0, 1, 33, 1000])
@pytest.mark.parametrize("rows", [0, 1, 9, 200])
def test_every_visible_pair_once(nh, nk, window, rows):
    """For every key that is written: its rows, over all items that list it, are those that see it (more may be listed,
    and mask themselves), each once; one item or one merge writes it."""
    rng = np.random.default_rng(nh + window + rows)
    g = nh // nk
    for trial in range(6):
        n = int(rng.integers(1, 12))
        new = np.where(rng.random(n) < 0.6, 1, rng.integers(0, 500, n))
        ctx = rng.integers(0, [1, 50, 3000, 30000][trial % 4], n)
        had = np.minimum(rng.integers(0, 4000, n), ctx) if trial % 2 else None
        few, many, merges, partials = _plan(new, ctx, nh, nk, window, rows, had, cus=[256, 8][trial % 2])
        tok0 = np.cumsum(new) - new
        written = {b: np.zeros(new[b] + ctx[b], int) for b in range(n) if new[b]}
        parts, rows_of = {}, {}
        for kind, items in (("few", few), ("many", many)):
            for t0, nt, pos0, b, k0, nk_, fresh, r0, nr, part, *_ in items.tolist():
                count = min(rows or new[b], new[b])
                assert (t0, nt, pos0) == (tok0[b] + new[b] - count, count, ctx[b] + new[b] - count)
                assert fresh == (ctx[b] if had is None else had[b])
                assert 0 < nk_ <= (3968 if kind == "few" else 256) and 0 <= r0 and r0 + nr <= nt * g
                if kind == "few":
                    assert (r0, nr, part) == (0, nt * g, -1) and nr <= 128
                else:
                    assert r0 % g == 0 or part >= 0
                rows_of.setdefault((b, k0, nk_), []).append((r0, nr))
                if part < 0:
                    written[b][k0:k0 + nk_] += 1
                else:
                    parts[part] = (b, k0, nk_, r0, nr)
        assert sorted(parts) == list(range(partials))
        for t0, nt, pos0, b, k0, nk_, fresh, r0, nr, part, count, _ in merges.tolist():
            written[b][k0:k0 + nk_] += 1
            assert [parts[part + i][:3] for i in range(count)] == [(b, k0, nk_)] * count and count > 1
        for b, w in written.items():
            count = min(rows or new[b], new[b])
            pos = np.arange(ctx[b] + new[b] - count, ctx[b] + new[b])
            lo = max(pos[0] - window + 1, 0) if window else 0
            start = min(lo, int(ctx[b] if had is None else had[b]))
            assert (w[start:] == 1).all() and (w[:start] == 0).all(), (b, start)
        for (b, k0, nk_), spans in rows_of.items():
            spans.sort()
            at = spans[0][0]
            for r0, nr in spans:
                assert r0 == at
                at += nr
            count = min(rows or new[b], new[b])
            pos = np.arange(ctx[b] + new[b] - count, ctx[b] + new[b])
            sees = (pos >= k0) & ((pos - (k0 + nk_ - 1) < window) if window else True)
            if sees.any():
                first, last = np.flatnonzero(sees)[[0, -1]]
                assert spans[0][0] <= first * g and at >= (last + 1) * g


def test_plan_refusals():
    lib = _lib.load()
    one, two, counts = np.ones(1, np.int32), np.full(1, 2, np.int32), np.zeros(4, np.int32)
    ok = dict(new=one, ctx=two, had=None, batch=1, nh=4, nk=2, window=0, rows=0, cus=256)

    def call(**over):
        a = {**ok, **over}
        ptr = lambda x: 0 if x is None else x.ctypes.data
        return lib.pkv_key_weights_plan(ptr(a["new"]), ptr(a["ctx"]), ptr(a["had"]), a["batch"], a["nh"], a["nk"], a["window"],
                                        a["rows"], a["cus"], 0, 0, counts.ctypes.data)

    assert call() == 0
    neg = np.full(1, -1, np.int32)
    for over in (dict(batch=-1), dict(nh=3), dict(nk=0), dict(window=-1), dict(rows=-1), dict(cus=0), dict(new=None),
                 dict(new=neg), dict(ctx=neg), dict(had=neg), dict(ctx=np.full(1, 1 << 27, np.int32))):
        assert call(**over) == _lib.PKV_EINVAL, over
    items = np.zeros((1, 12), np.int32)
    big = np.full(1, 20000, np.int32)
    assert lib.pkv_key_weights_plan(one.ctypes.data, big.ctypes.data, 0, 1, 4, 2, 0, 0, 256, items.ctypes.data, 1,
                                    counts.ctypes.data) == _lib.PKV_ENOSPC


def _batch(**over):
    kw = dict(page_size=16, num_pages=20, n_heads=4, n_kv=2, head_dim=64, device="cpu", weight_rows=None)
    kw.update(over)
    new, ctx, bt = kw.pop("new", [2, 1]), kw.pop("ctx", [10, 20]), kw.pop("bt", [[0, -1], [1, 2]])
    return prism_amd.PackedBatch(new, ctx, bt, **kw)


def test_batch_refusals():
    _batch()
    _batch(weight_rows=3, weighed=[0, 20])
    for over, msg in [(dict(weight_rows=-1), "weight_rows"), (dict(weight_rows=True), "weight_rows"),
                      (dict(weight_rows=1.5), "weight_rows"), (dict(weighed=[1]), "weighed"), (dict(weighed=[-1, 0]), "weighed"),
                      (dict(evicted=[1, 2, 3]), "evicted"), (dict(evicted=[-1, 0]), "evicted"),
                      (dict(evicted=[5, 0], windows=(8,)), "window"), (dict(bt=[[0, -1], [0, 2]], ctx=[17, 20]), "share|page")]:
        with pytest.raises(RuntimeError, match=msg):
            _batch(**over)
    # a page that two sequences read (a shared prefix) is fine without weights, not with them
    shared = dict(new=[1, 1], ctx=[17, 18], bt=[[5, 1], [5, 2]])
    _batch(**shared, weight_rows=0)
    with pytest.raises(RuntimeError, match="share a page"):
        _batch(**shared)
    # out of every counted row's window, and weighed: it may be shared, or gone
    _batch(**shared, windows=(2,))
    _batch(new=[1, 1], ctx=[17, 18], bt=[[-1, 1], [99, 2]], windows=(2,))


def test_evicted_tokens_move_the_positions():
    b = _batch(evicted=[100, 7], weight_rows=0)
    assert b.positions.tolist() == [110, 111, 27]
    assert b.slots.tolist() == [10, 11, 2 * 16 + 4]
    assert _batch(weight_rows=0).positions.tolist() == [10, 11, 20]
    with pytest.raises(RuntimeError, match="2.27"):
        _batch(evicted=[(1 << 27) - 11, 0])


def test_ops_need_the_device_and_the_layout():
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    kc, w, lse = torch.zeros(20, 16, 2, 64, dtype=torch.bfloat16), torch.zeros(20, 2, 16), torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="ROCm device"):
        prism_amd.packed_key_weights(q, kc, lse, w, _batch())
    with pytest.raises(RuntimeError, match="ROCm device"):
        prism_amd.sample_tokens(torch.zeros(2, 5), torch.zeros(2))
    with pytest.raises(RuntimeError, match="ROCm device"):
        i = torch.zeros(1, dtype=torch.int32)
        prism_amd.evict_keys(kc[None], kc[None], w[None], i[None], i, i, 4)


def _weights_call(lib, **over):
    a = dict(q=A16, q_st=256, q_sh=64, k=A16, page=2048, lse=A16, lse_st=4, w=A16, w_page=32, bt=A16, bt_st=2, items=A16,
             few=1, many=0, merges=0, partials=0, ws=0, ws_bytes=0, tokens=0, batch=1, nh=4, nk=2, hd=64, P=16, pages=20,
             blocks=2, window=0, scale=0.125)
    a.update(over)
    return lib.pkv_key_weights(*a.values(), None, None)


def test_weights_argument_errors():
    lib = _lib.load()
    assert _weights_call(lib, few=0) == 0
    for over, msg in [(dict(q=A16 + 2), "q"), (dict(q=0), "null"), (dict(q_st=3), "multiples of 8"), (dict(lse=0), "null"), (dict(w=0), "null"),
                      (dict(lse=A16 + 2), "4-byte"), (dict(w=A16 + 1), "4-byte"), (dict(lse_st=3), "overlap"),
                      (dict(w_page=31), "overlap"), (dict(items=0), "work list"), (dict(items=A16 + 4), "work list"),
                      (dict(partials=1), "workspace"), (dict(partials=1, ws=A16, ws_bytes=8), "workspace"),
                      (dict(tokens=-1), "sizes"), (dict(few=-1), "sizes"), (dict(many=-1), "sizes"), (dict(window=-1), "sizes"),
                      (dict(nh=3), "multiple"), (dict(hd=96), "head_dim"), (dict(P=24), "page_size"), (dict(scale=0.0), "scale"),
                      (dict(scale=float("nan")), "scale"), (dict(few=1 << 30, many=1 << 30), "too many"), (dict(page=16), "page stride")]:
        assert _weights_call(lib, **over) in (_lib.PKV_EINVAL, _lib.PKV_ENOSPC), over
        assert msg in lib.pkv_last_error().decode(), (over, lib.pkv_last_error())
    assert lib.pkv_key_weights_workspace_bytes(3, 4) == 3 * 4 * 256 * 4


def test_weights_work_lists_past_the_grid():
    """2^31 threads and more are refused, before anything is launched."""
    lib = _lib.load()
    for over in (dict(few=1 << 22), dict(few=1 << 21, many=1 << 21), dict(few=0, merges=1 << 22)):
        assert _weights_call(lib, **over) == _lib.PKV_EINVAL and b"too many" in lib.pkv_last_error(), over


def _evict_call(lib, **over):
    a = dict(k=A16, v=A16, layer=1 << 16, page=2048, w=A16, w_layer=640, w_page=32, bt=A16, bt_st=2, lens=A16, keeps=A16,
             kept=A16, layers=0, batch=1, nk=2, hd=64, P=16, pages=20, blocks=2, max_keep=4, first=0, recent=0, ws=A16,
             ws_bytes=1 << 20)
    a.update(over)
    return lib.pkv_evict(*a.values(), None, None)


def test_evict_argument_errors():
    lib = _lib.load()
    assert _evict_call(lib) == 0
    for over, msg in [(dict(k=A16 + 8), "aligned"), (dict(w=0), "null"), (dict(keeps=0), "null"), (dict(kept=0), "null"),
                      (dict(w=A16 + 4), "16-byte"), (dict(w_layer=6), "16-byte"), (dict(w_page=34), "16-byte"), (dict(kept=A16 + 2), "4-byte"),
                      (dict(layers=1, ws=0), "workspace"), (dict(layers=1, ws=A16 + 2), "workspace"),
                      (dict(layers=1, ws_bytes=8), "needed"), (dict(layer=12), "layer stride"), (dict(w_page=28), "overlap"),
                      (dict(layers=-1), "sizes"), (dict(max_keep=-1), "sizes"), (dict(first=-1), "sizes"), (dict(recent=-1), "sizes"),
                      (dict(layers=70000), "grid"), (dict(hd=80), "head_dim"), (dict(P=8), "page_size"), (dict(bt=0), "null"),
                      (dict(lens=0), "null")]:
        assert _evict_call(lib, **over) in (_lib.PKV_EINVAL, _lib.PKV_ENOSPC), over
        assert msg in lib.pkv_last_error().decode(), (over, lib.pkv_last_error())


def _sample_call(lib, **over):
    a = dict(x=A16, stride=100, dtype=_lib.PKV_FP32, u=A16, ts=0, t=1.0, ks=0, k=0, ps=0, p=1.0, ms=0, m=0.0, tokens=A16, lp=0,
             rows=0, vocab=100, ws=0, ws_bytes=0)
    a.update(over)
    return lib.pkv_sample(*a.values(), None)


def test_sample_argument_errors():
    lib = _lib.load()
    assert _sample_call(lib) == 0
    need = lib.pkv_sample_workspace_bytes(2, 100)
    assert need > 0 and lib.pkv_sample_workspace_bytes(0, 100) == 0
    two = dict(rows=2, ws=A16, ws_bytes=need)
    for over, msg in [(dict(rows=-1), "vocabulary"), (dict(vocab=0), "vocabulary"), (dict(vocab=1000001), "vocabulary"),
                      (dict(rows=65536), "grid"), (dict(dtype=3), "dtype"), (dict(two, x=0), "null"), (dict(two, u=0), "null"),
                      (dict(two, tokens=0), "null"), (dict(two, stride=99), "overlap"), (dict(two, x=A16 + 2), "aligned"),
                      (dict(two, ts=A16 + 1), "aligned"), (dict(two, tokens=A16 + 4), "8-byte"), (dict(two, ws=0), "workspace"),
                      (dict(two, ws_bytes=need - 1), "needed")]:
        assert _sample_call(lib, **over) in (_lib.PKV_EINVAL, _lib.PKV_ENOSPC), over
        assert msg in lib.pkv_last_error().decode(), (over, lib.pkv_last_error())


def test_the_sampling_oracle_on_rows_done_by_hand():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    cases = [((1.0, 0, 1.0, 0.0), [(0.05, 0), (0.1001, 1), (0.49, 1), (0.51, 2), (0.71, 3), (1.0, 3)]),
             ((1.0, 2, 1.0, 0.0), [(0.57, 1), (0.58, 3)]),              # tokens 1 and 3, 4 : 3
             ((1.0, 0, 0.65, 0.0), [(0.57, 1), (0.58, 3)]),             # 0.4 is short of 0.65, with 0.3 it is not
             ((1.0, 0, 1.0, 0.6), [(0.57, 1), (0.58, 3)]),              # 0.6 of 0.4 is 0.24
             ((0.0, 0, 1.0, 0.0), [(0.9, 1)])]
    for (t, k, p, m), draws in cases:
        for u, want in draws:
            assert ob.sample64(x, u, t, k, p, m)[0] == want, (t, k, p, m, u)
    assert ob.sample64(x, 0.2, 1.0, 2, 1.0, 0.0)[1] == pytest.approx(np.log(4 / 7))


def test_the_weights_oracle_is_softmax():
    g = torch.Generator().manual_seed(0)
    P, nk, hd, nh = 16, 2, 64, 4
    kc, q = torch.randn(4, P, nk, hd, generator=g), torch.randn(3, nh, hd, generator=g)
    bt = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    keys = kc[bt[0].long()].flatten(0, 1)[:40].double()
    lse, want = torch.zeros(3, nh, dtype=torch.float64), torch.zeros(40, nk, dtype=torch.float64)
    for j in range(3):
        for h in range(nh):
            s = keys[:38 + j, h // 2] @ q[j, h].double() / 8.0
            lse[j, h] = torch.logsumexp(s, 0)
            want[:38 + j, h // 2] += torch.softmax(s, 0)
    got, gain = ob.key_weights64(q, kc, lse, torch.zeros(4, nk, P), [3], [37], bt)
    flat = got[bt[0].long()].transpose(0, 1).reshape(nk, -1)[:, :40].T
    assert (flat - want).abs().max() < 1e-12 and torch.equal(got, gain)


def test_cache_book_keeping_without_a_device(monkeypatch):
    """evict's plan on a cache on the CPU: what it refuses changes nothing."""
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    kv.new_sequence(1)
    with pytest.raises(RuntimeError, match="enable_key_weights"):
        kv.evict([1], 10)
    with pytest.raises(RuntimeError, match="enable_key_weights"):
        kv.build_packed_batch([1], 1, 4, weight_rows=None)
    assert [t.shape for t in kv.enable_key_weights()] == [(12, 2, 16)] and kv.enable_key_weights() is kv.key_weights
    kv._ensure_capacity(1, 90)
    kv.build_packed_batch([1], 90, 4, weight_rows=None)
    kv.update_seqlens([1], 90)
    kv.fork_sequence(1, 2)
    state = lambda: (list(kv.free_pages), {s: list(p) for s, p in kv.seq_pages.items()}, dict(kv.seq_len), dict(kv._holders))
    before = state()
    for args, kw, error in [(([1], 0), {}, ValueError), (([1, 2], [5]), {}, ValueError), (([1, 1], 5), {}, ValueError),
                            (([1], 5), dict(first=-1), ValueError)]:
        with pytest.raises(error):
            kv.evict(*args, **kw)
    assert kv.evict([1], 90) == 0 and kv.evict([], 5) == 0
    # tokens of steps without weights
    kv.new_sequence(4)
    kv._ensure_capacity(4, 30)
    kv.build_packed_batch([4], 30, 4, weight_rows=None)
    kv.update_seqlens([4], 30)
    kv.update_seqlens([4], 10)
    with pytest.raises(RuntimeError, match="only 30 of the 32 tokens"):
        kv.evict([4], 20, recent=8)
    kv.free_sequence(4)
    assert state()[1:3] == before[1:3]
    kv.new_sequence(3)
    kv._ensure_capacity(3, 80)
    assert kv.pages_free < 4
    before = state()
    with pytest.raises(KVCacheOutOfPages, match="shared pages"):
        kv.evict([1, 2], 64)     # four pages to copy, one free
    with pytest.raises(RuntimeError, match="ROCm device"):
        kv.evict([1], 10)
    assert state() == before
    kv.seq_evicted[1] = 30
    assert kv.next_positions([1, 2]) == [120, 90]
    kv.free_sequence(2)
    kv.prepare_append([1], 1)
    assert kv.build_packed_batch([1], 1, 4).positions.tolist() == [120]
    with pytest.raises(RuntimeError, match="window"):
        kv.build_packed_batch([1], 1, 4, windows=(None, 64))
    with pytest.raises(RuntimeError, match="evicted"):
        prism_amd.PrefixCache(kv, 16).store(list(range(16)), kv.seq_pages[1][:1], "m")
    with pytest.raises(RuntimeError, match="evicted"):
        prism_amd.DecodeBatch(kv, 2).plan([1])
    kv.fork_sequence(1, 5)
    assert kv.seq_evicted[5] == 30
    kv.free_sequence(1)
    kv.free_sequence(5)
    assert not kv.seq_evicted


def test_a_prefix_whose_keys_were_never_weighed_starts_from_nothing():
    """Only pages that steps with weights filled count as weighed where they are a new sequence's prefix, whoever had
    them before."""
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    pc = prism_amd.PrefixCache(kv, 16)
    kv.enable_key_weights()

    def run(sid, counts, weights):
        for n, w in zip(counts, weights):
            kv.prepare_append([sid], n)
            kv.build_packed_batch([sid], n, 4, weight_rows=None if w else 0)
            kv.update_seqlens([sid], n)

    def weighed_as_prefix(tokens):
        pages, n = pc.lookup(tokens, "m")
        kv.new_sequence(9, prefix_pages=pages, prefix_len=n)
        got = kv._weighed[9]
        kv.free_sequence(9)
        return n, got

    for sid, weights, want in ((1, (1, 1), 48), (2, (0, 0), 0), (3, (0, 1), 48), (4, (1, 0), 32)):
        tokens = [100 * sid + i for i in range(48)]
        kv.new_sequence(sid)
        run(sid, (40, 8), weights)
        pc.store(tokens, kv.seq_pages[sid][:3], "m")
        assert weighed_as_prefix(tokens) == (48, want)
        kv.free_sequence(sid)
        pc.evict_lru(3)  # its pages go to the next one


def test_keys_written_over_weighed_ones_do_not_count_as_weighed():
    """Tokens rolled back, or cut away, and written again by steps without weights: the old keys' weights are not theirs."""
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    kv.enable_key_weights()

    def step(sid, n, weights):
        kv.prepare_append([sid], n)
        kv.build_packed_batch([sid], n, 4, weight_rows=None if weights else 0)
        kv.update_seqlens([sid], n)

    def weighed_as_prefix(sid, n):
        kv.new_sequence(9, prefix_pages=kv.seq_pages[sid][:n // 16], prefix_len=n)
        got = kv._weighed[9]
        kv.free_sequence(9)
        return got

    kv.new_sequence(1)
    step(1, 48, True)
    assert (kv._weighed[1], weighed_as_prefix(1, 48)) == (48, 48)
    kv.seq_len[1] = 20
    step(1, 28, False)
    assert (kv._weighed[1], weighed_as_prefix(1, 48)) == (20, 16)
    kv.seq_len[1] = 20
    step(1, 28, True)
    assert (kv._weighed[1], weighed_as_prefix(1, 48)) == (48, 48)
    # without prepare_append too: the pages are there
    kv.seq_len[1] = 40
    kv.build_packed_batch([1], 8, 4)
    kv.update_seqlens([1], 8)
    assert (kv._weighed[1], weighed_as_prefix(1, 48)) == (40, 32)


def test_a_page_copied_in_part_does_not_count_as_weighed(monkeypatch):
    """A prefix taken in part: what stands behind it in the copy is written by the sequence that copied it."""
    monkeypatch.setattr("prism_amd.kv_cache.copy_pages", lambda *a: None)
    monkeypatch.setattr("prism_amd.kv_cache.copy_key_weights", lambda *a: None)
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    kv.enable_key_weights()
    kv.new_sequence(1)
    kv.prepare_append([1], 32)
    kv.build_packed_batch([1], 32, 4, weight_rows=None)
    kv.update_seqlens([1], 32)
    for weights, want in ((0, 16), (None, 32)):
        kv.new_sequence(2, prefix_pages=kv.seq_pages[1][:2], prefix_len=20)
        kv.seq_pages[2].pop()  # (its fresh page)
        assert kv.prepare_append([2], 12) == 1
        kv.build_packed_batch([2], 12, 4, weight_rows=weights)
        kv.update_seqlens([2], 12)
        assert kv.seq_pages[1][1] in kv._weighed_pages
        kv.new_sequence(3, prefix_pages=kv.seq_pages[2][:2], prefix_len=32)
        assert kv._weighed[3] == want
        kv.free_sequence(3)
        kv.free_sequence(2)


def test_keys_written_without_a_packed_batch_do_not_count_as_weighed():
    """The growth of one sequence alone says that keys will be written, as prepare_append does."""
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    kv.enable_key_weights()
    kv.new_sequence(1)
    kv._ensure_capacity(1, 48)
    kv.build_packed_batch([1], 48, 4, weight_rows=None)
    kv.update_seqlens([1], 48)
    assert kv._weighed[1] == 48 and set(kv.seq_pages[1][:3]) <= kv._weighed_pages
    kv.seq_len[1] = 20
    kv._ensure_capacity(1, 48)
    kv.update_seqlens([1], 28)
    assert kv._weighed[1] == 20 and kv._weighed_pages == {kv.seq_pages[1][0]}


@pytest.mark.parametrize("weighing", [True, False])
def test_a_weighed_page_of_a_transferred_sequence_is_one(monkeypatch, weighing):
    """A prefix on it adds to its weights, and does not start them anew under the sequence that has them."""
    monkeypatch.setattr("prism_amd.kv_cache.copy_pages", lambda *a: None)
    monkeypatch.setattr("prism_amd.kv_cache.copy_key_weights", lambda *a: None)
    kv, other = (FlashAttnKVCache(1, 2, 64, 12, 16, "cpu") for _ in range(2))
    kv.enable_key_weights()
    if weighing:
        other.enable_key_weights()
    kv.new_sequence(1)
    kv.prepare_append([1], 40)
    kv.build_packed_batch([1], 40, 4, weight_rows=None)
    kv.update_seqlens([1], 40)
    assert kv.transfer_sequence(1, other, 7) == 3
    other.enable_key_weights()
    other.new_sequence(8, prefix_pages=other.seq_pages[7][:2], prefix_len=32)
    assert (other._weighed[7], other._weighed[8]) == ((40, 32) if weighing else (0, 0))


def _first_keys_without_weights(batch):
    """Per sequence, the key from which on the batch's packed_key_weights starts from nothing."""
    _, at, few, many, *_ = batch._weight_plans[None]
    items = batch._buf[(at - batch._buf.data_ptr()) // 4:][:12 * (few + many)].view(-1, 12)
    return {int(i[3]): int(i[6]) for i in items}


def _weighing_step(kv, sid, n):
    kv.prepare_append([sid], n)
    batch = kv.build_packed_batch([sid], n, 4, weight_rows=None)
    kv.update_seqlens([sid], n)
    return _first_keys_without_weights(batch)[0]


def _plain_step(kv, sid, n):
    kv.prepare_append([sid], n)
    kv.build_packed_batch([sid], n, 4)
    kv.update_seqlens([sid], n)


def test_weights_on_shared_pages_are_added_to(monkeypatch):
    """Sequences on pages that nobody weighed yet: the first one's step starts them, the second one's adds to them."""
    monkeypatch.setattr("prism_amd.kv_cache.copy_pages", lambda *a: None)
    monkeypatch.setattr("prism_amd.kv_cache.copy_key_weights", lambda *a: None)
    for n in (48, 41):  # whole pages, and a last one that each copies for itself
        kv = FlashAttnKVCache(1, 2, 64, 20, 16, "cpu")
        kv.enable_key_weights()
        kv.new_sequence(1)
        _plain_step(kv, 1, n)
        kv.fork_sequence(1, 2)
        kv.fork_sequence(1, 3)
        assert _weighing_step(kv, 1, 1) == 0
        # the whole pages are weighed; what lies on a page of its own is not
        assert _weighing_step(kv, 2, 1) == n // 16 * 16
        assert _weighing_step(kv, 2, 30) == n + 1
        assert _weighing_step(kv, 1, 1) == n + 1
        assert _weighing_step(kv, 3, 20) == n // 16 * 16


def test_weights_on_a_prefix_page_weighed_in_part_are_added_to():
    """A full page whose first keys alone were weighed, then taken as a prefix: what was weighed stays."""
    kv = FlashAttnKVCache(1, 2, 64, 20, 16, "cpu")
    kv.enable_key_weights()
    pc = prism_amd.PrefixCache(kv, 16)
    kv.new_sequence(1)
    assert _weighing_step(kv, 1, 40) == 0
    _plain_step(kv, 1, 8)
    pc.store(list(range(48)), kv.seq_pages[1], "m")
    pages, n = pc.lookup(list(range(48)), "m")
    kv.new_sequence(2, prefix_pages=pages, prefix_len=n)
    assert _weighing_step(kv, 2, 5) == 40
    assert _weighing_step(kv, 1, 1) == 48
    kv.free_sequence(1)
    kv.new_sequence(3, prefix_pages=pages, prefix_len=n)
    assert _weighing_step(kv, 3, 5) == 48
    # stored by steps without weights, weighed by the first that takes it
    kv.new_sequence(4)
    _plain_step(kv, 4, 32)
    pc.store(list(range(100, 132)), kv.seq_pages[4], "m")
    kv.free_sequence(4)
    pages, n = pc.lookup(list(range(100, 132)), "m")
    for sid, start in ((5, 0), (6, 32)):
        kv.new_sequence(sid, prefix_pages=pages, prefix_len=n)
        assert _weighing_step(kv, sid, 3) == start


def test_weights_of_pages_travel_with_them(monkeypatch):
    """Copies, transfers and migrations keep what a page weighed in part has; a page given back forgets it."""
    monkeypatch.setattr("prism_amd.kv_cache.copy_pages", lambda *a: None)
    monkeypatch.setattr("prism_amd.kv_cache.copy_key_weights", lambda *a: None)
    kv, other = (FlashAttnKVCache(1, 2, 64, 12, 16, "cpu") for _ in range(2))
    kv.enable_key_weights()
    other.enable_key_weights()
    kv.new_sequence(1)
    _weighing_step(kv, 1, 40)
    _plain_step(kv, 1, 8)
    kv.transfer_sequence(1, other, 1)
    other.new_sequence(2, prefix_pages=other.seq_pages[1][:3], prefix_len=48)
    assert _weighing_step(other, 2, 1) == 40
    target = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    target.enable_key_weights()
    kv.migrate_to(target)
    target.new_sequence(2, prefix_pages=target.seq_pages[1][:3], prefix_len=48)
    # rolled back into a page that another sequence lists too: its copy has the first keys' weights
    target.seq_len[1] = 37
    assert _weighing_step(target, 1, 1) == 37
    assert _weighing_step(target, 2, 1) == 40
    pages = list(target.seq_pages[2])
    target.free_all()
    target.new_sequence(3)
    _plain_step(target, 3, 180)
    assert set(pages) <= set(target.seq_pages[3])
    assert _weighing_step(target, 3, 1) == 0


def test_keys_counted_by_update_seqlens_alone_do_not_count_as_weighed(monkeypatch):
    """Tokens rolled back and written again by a step that says so to update_seqlens alone."""
    monkeypatch.setattr("prism_amd.kv_cache.copy_pages", lambda *a: None)
    monkeypatch.setattr("prism_amd.kv_cache.copy_key_weights", lambda *a: None)
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    kv.enable_key_weights()
    kv.new_sequence(1)
    assert _weighing_step(kv, 1, 48) == 0 and kv._weighed[1] == 48
    kv.seq_len[1] = 20
    kv.update_seqlens([1], 28)
    assert kv._weighed[1] == 20 and kv._weighed_pages == {kv.seq_pages[1][0]}
    assert _weighing_step(kv, 1, 1) == 20
    # a step with weights of which the first tokens alone are taken (the others were drafts), then one without
    kv.prepare_append([1], 6)
    kv.build_packed_batch([1], 6, 4, weight_rows=None)
    kv.update_seqlens([1], 4)
    assert kv._weighed_keys(1) == kv.seq_len[1] == 53
    kv.update_seqlens([1], 2)
    assert kv._weighed_keys(1) == 53 and kv.seq_len[1] == 55
    # a batch that was laid out, then another in its place: the last one counts
    for rows, want in ((0, 55), (None, 61)):
        kv.prepare_append([1], 3)
        kv.build_packed_batch([1], 3, 4, weight_rows=None)
        kv.build_packed_batch([1], 3, 4, weight_rows=rows)
        kv.update_seqlens([1], 3)
        assert kv._weighed_keys(1) == want
    # a batch that was laid out and given up, the tokens before it rolled back
    kv.prepare_append([1], 1)
    kv.build_packed_batch([1], 1, 4, weight_rows=None)
    kv.seq_len[1] = 57
    kv.update_seqlens([1], 2)
    assert kv._weighed_keys(1) == 57
    # the pages moved in between
    kv.prepare_append([1], 2)
    kv.build_packed_batch([1], 2, 4, weight_rows=None)
    kv.compact()
    kv.update_seqlens([1], 2)
    assert kv._weighed_keys(1) == kv.seq_len[1] == 61
    # of several sequences in one call, each by itself; none new is none written
    kv.new_sequence(2)
    kv.prepare_append([1, 2], [1, 9])
    kv.build_packed_batch([2], 9, 4, weight_rows=None)
    had = kv._weighed_keys(1)
    kv.update_seqlens([1, 2], [1, 9])
    assert (kv._weighed_keys(1), kv._weighed_keys(2)) == (had, 9)
    kv.update_seqlens([1, 2], 0)
    assert (kv._weighed_keys(1), kv._weighed_keys(2)) == (had, 9)


def test_lengths_of_a_cut_sequence_are_not_taken_for_positions():
    """As build_block_table returned them, whole or in part; not those of others, nor what was made of them."""
    from prism_amd.attention import refuse_lengths_of_cut
    kv = FlashAttnKVCache(1, 2, 64, 12, 16, "cpu")
    for sid in (1, 2, 3):
        kv.new_sequence(sid)
        kv._ensure_capacity(sid, 20)
        kv.update_seqlens([sid], 20)
    old = kv.build_block_table([1, 2, 3])[1]
    kv.seq_evicted[2] = 30
    refuse_lengths_of_cut(old, "x")
    _, sl = kv.build_block_table([1, 2, 3])
    assert sl.tolist() == [20, 20, 20]
    for bad in (sl, sl[1:], sl[1:2], sl[:2], old):
        with pytest.raises(RuntimeError, match="next_positions"):
            refuse_lengths_of_cut(bad, "x")
    for fine in (sl[:1], sl[2:], sl + 1, sl.clone(), torch.tensor(kv.next_positions([1, 2, 3]))):
        refuse_lengths_of_cut(fine, "x")
    sl[1] = 50
    refuse_lengths_of_cut(sl, "x")
    _, sl = kv.build_block_table([1, 3])
    refuse_lengths_of_cut(sl, "x")
    kv.free_sequence(2)
    refuse_lengths_of_cut(kv.build_block_table([1, 3])[1], "x")


def test_storing_a_prefix_looks_at_each_cut_sequence_once():
    """However many pages are stored: their owners' pages are gone through once, not for every page."""
    kv = FlashAttnKVCache(1, 2, 64, 400, 16, "cpu")
    pc = prism_amd.PrefixCache(kv, 16)
    looks = []

    class Pages(list):
        def __iter__(self):
            looks.append("all")
            return super().__iter__()

        def __contains__(self, page):
            looks.append(page)
            return super().__contains__(page)

    for sid in range(1, 6):
        kv.new_sequence(sid)
        kv._ensure_capacity(sid, 640)
        kv.seq_len[sid] = 640
    for sid in range(2, 6):
        kv.seq_evicted[sid] = 10
        kv.seq_pages[sid] = Pages(kv.seq_pages[sid])
    pc.store(list(range(640)), kv.seq_pages[1], "m")
    assert pc.num_cached_pages == 40 and len(looks) <= 4
    for pages in (kv.seq_pages[5][:1], kv.seq_pages[1][:3] + kv.seq_pages[3][-1:]):
        with pytest.raises(RuntimeError, match="evicted"):
            pc.store(list(range(64)), list(pages), "other")
    assert pc.num_cached_pages == 40
    pc.store(list(range(64)), [], "other")
