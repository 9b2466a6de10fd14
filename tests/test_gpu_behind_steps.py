"""The operators behind the attention together, as a server runs them: a decode loop whose cache stays within a budget
and whose tokens never leave the device."""
import numpy as np
import pytest
import torch

import prism_amd
from oracle import behind as ob
from oracle import packed as op
from prism_amd.kv_cache import KVCacheOutOfPages

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
L, NH, NK, HD, VOCAB = 2, 14, 2, 64, 3001


class Model:
    """Two layers without weights worth the name: enough to carry tokens through the operators."""

    def __init__(self, gpu, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: (torch.randn(*s, generator=g) / s[0] ** 0.5).to(BF16).to(gpu)
        self.emb = torch.randn(VOCAB, 256, generator=g).to(BF16).to(gpu)
        self.qkv = [r(256, (NH + 2 * NK) * HD) for _ in range(L)]
        self.out = [r(NH * HD, 256) for _ in range(L)]
        self.head = r(256, VOCAB)
        self.cos, self.sin = prism_amd.rotary_tables(HD, 4096, 1e4, device=gpu)

    def step(self, kv, batch, tokens, check=None, weigh=True):
        x = self.emb[tokens]
        for l in range(L):
            q = prism_amd.packed_rope_append(x @ self.qkv[l], kv.k_caches[l], kv.v_caches[l], batch, self.cos, self.sin)
            out, lse = prism_amd.packed_attention(q, kv.k_caches[l], kv.v_caches[l], batch, return_lse=True)
            if weigh:
                old = kv.key_weights[l].cpu() if check else None
                prism_amd.packed_key_weights(q, kv.k_caches[l], lse, kv.key_weights[l], batch)
            if check:
                check(l, q, out, lse, old)
            x = x + out.flatten(1) @ self.out[l]
        return x @ self.head


def _serve_step(model, kv, seqs, tokens, counts, check=True):
    kv.prepare_append(seqs, counts)
    batch = kv.build_packed_batch(seqs, counts, NH, weight_rows=None)
    want = np.concatenate([np.arange(p, p + n) for p, n in zip(kv.next_positions(seqs), counts)])
    assert np.array_equal(batch.positions.cpu().numpy(), want)
    bt, ctx = kv.block_table_host(seqs)
    had = [min(kv.seq_len[s], c) for s, c in zip(seqs, ctx)]

    def look(l, q, out, lse, old):
        k, v, bt_ = kv.k_caches[l].cpu(), kv.v_caches[l].cpu(), torch.from_numpy(bt)
        ref, ref_lse, mag = op.packed_attention64(q.cpu(), k, v, counts, ctx, bt_)
        # the probabilities and the output rounded to bf16, as test_gpu_packed derives it
        assert ((out.double().cpu() - ref).abs() <= ref.abs() * 2.0 ** -8 + (mag + ref.abs()) * (2.0 ** -8 + 2.0 ** -12)).all()
        w, gain = ob.key_weights64(q.cpu(), k, lse.cpu(), old, counts, ctx, bt_, weighed=had)
        err = (kv.key_weights[l].double().cpu() - w).abs()
        assert (err <= gain * (2.0 ** -12 + 7 * max(counts) * 2.0 ** -24) + (old.double() + gain) * 2.0 ** -23).all()

    logits = model.step(kv, batch, tokens, look if check else None)
    kv.update_seqlens(seqs, counts)
    return logits


def _evict(kv, seqs, budget, **how):
    """kv.evict, and every layer's pool against the restatement on the pools as they were."""
    n = [kv.seq_len[s] for s in seqs]
    keep = [min(x, budget) for x in n]
    bt, _ = kv.block_table_host(seqs)
    old = [x.cpu() for x in (kv.k_pool.view(torch.int16), kv.v_pool.view(torch.int16), kv.key_weight_pool)]
    seen = kv.next_positions(seqs)
    gained = kv.evict(seqs, budget, **how)
    want = ob.evict_np(*[x.numpy() for x in old], bt, n, keep, how.get("first", 4), how.get("recent", 64), max(keep))
    after, _ = kv.block_table_host(seqs)
    for i in range(len(seqs)):
        t = np.arange(keep[i])
        pg, was, row = after[i][t // kv.page_size], bt[i][t // kv.page_size], t % kv.page_size
        for got, ref in ((kv.k_pool.view(torch.int16), want[0]), (kv.v_pool.view(torch.int16), want[1])):
            assert np.array_equal(got.cpu().numpy()[:, pg, row], ref[:, was, row])
        assert np.array_equal(kv.key_weight_pool.cpu().numpy()[:, pg, :, row], want[2][:, was, :, row])
    assert [kv.seq_len[s] for s in seqs] == keep and kv.next_positions(seqs) == seen
    return gained


def test_a_server_within_its_budget(gpu):
    """Prompts, decode steps with sampled tokens, evictions whenever a sequence is over 160 tokens; a fork and a
    prefix-cached page on the way; transfer, migration and compaction of what is left."""
    model = Model(gpu)
    kv = prism_amd.FlashAttnKVCache(L, NK, HD, 90, 16, gpu)
    kv.enable_key_weights()
    pc = prism_amd.PrefixCache(kv, 16)
    rng = np.random.default_rng(0)
    g = torch.Generator(device=gpu).manual_seed(1)
    prompts = [rng.integers(0, VOCAB, n) for n in (150, 33, 170, 1)]
    seqs = [1, 2, 3, 4]
    for s in seqs:
        kv.new_sequence(s)
    tokens = torch.from_numpy(np.concatenate(prompts)).to(gpu)
    logits = _serve_step(model, kv, seqs, tokens, [len(p) for p in prompts])
    last = torch.from_numpy(np.cumsum([len(p) for p in prompts]) - 1).to(gpu)
    draw = lambda x: prism_amd.sample_tokens(x, torch.rand(len(x), generator=g, device=gpu), temperature=0.9, top_k=50, top_p=0.95)
    tokens = draw(logits[last])
    pc.store(prompts[0].tolist(), kv.seq_pages[1], "m")
    for step in range(22):
        over = [s for s in seqs if kv.seq_len[s] > 160]
        if over:
            free = kv.pages_free
            gained = _evict(kv, over, 128, recent=32)
            assert kv.pages_free == free + gained
            assert all(len(kv.seq_pages[s]) == 8 for s in over)
        if step == 5:
            kv.fork_sequence(3, 9)
            with pytest.raises(RuntimeError, match="share a page"):
                kv.prepare_append([3, 9], 1)
                kv.build_packed_batch([3, 9], 1, NH, weight_rows=None)
        tokens = draw(_serve_step(model, kv, seqs, tokens, [1] * len(seqs), check=step % 4 == 0))
        assert ((tokens >= 0) & (tokens < VOCAB)).all()
    assert kv.seq_evicted[1] > 0 and kv.seq_evicted[3] > 0 and 4 not in kv.seq_evicted
    # the fork kept what sequence 3 had at step 5; the cached prefix what the prompt wrote
    held = [x[:, kv.seq_pages[9]].clone() for x in (kv.k_pool, kv.v_pool, kv.key_weight_pool)]
    pages, n = pc.lookup(prompts[0].tolist(), "m")
    assert n == 144 and not set(pages) & set(kv.seq_pages[1])
    with pytest.raises(RuntimeError, match="evicted"):
        pc.store(list(range(128)), kv.seq_pages[1], "m")
    _evict(kv, [1, 3], 100, first=0, recent=1)
    assert all(torch.equal(a, x[:, kv.seq_pages[9]]) for a, x in zip(held, (kv.k_pool, kv.v_pool, kv.key_weight_pool)))
    # the state travels
    other = prism_amd.FlashAttnKVCache(L, NK, HD, 30, 16, gpu)
    other.enable_key_weights()
    kv.transfer_sequence(1, other, 5)
    assert other.next_positions([5]) == kv.next_positions([1])
    for a, b in ((kv.k_pool, other.k_pool), (kv.key_weight_pool, other.key_weight_pool)):
        assert torch.equal(a[:, kv.seq_pages[1]], b[:, other.seq_pages[5]])
    before = kv.key_weight_pool[:, kv.seq_pages[3]].clone()
    positions = kv.next_positions(seqs)
    kv.compact()
    assert torch.equal(before, kv.key_weight_pool[:, kv.seq_pages[3]]) and kv.next_positions(seqs) == positions
    assert kv.key_weights[0].data_ptr() == kv.key_weight_pool.data_ptr()
    _evict(kv, [3], 90)
    _serve_step(model, kv, seqs, tokens, [1] * len(seqs))


def test_sequences_that_share_pages_are_evicted_apart(gpu):
    """Forks evicted in one call, to different lengths: each gets its own copy of what it writes to, sources stay whole."""
    model = Model(gpu, 2)
    kv = prism_amd.FlashAttnKVCache(L, NK, HD, 40, 16, gpu)
    kv.enable_key_weights()
    kv.new_sequence(1)
    _serve_step(model, kv, [1], torch.arange(200, device=gpu), [200])
    kv.fork_sequence(1, 2)
    kv.fork_sequence(1, 3)
    third = [x[:, kv.seq_pages[3]].clone() for x in (kv.k_pool, kv.v_pool, kv.key_weight_pool)]
    bt, _ = kv.block_table_host([1, 2])
    old = [x.cpu().numpy() for x in (kv.k_pool.view(torch.int16), kv.v_pool.view(torch.int16), kv.key_weight_pool)]
    kv.evict([1, 2], [100, 170], first=2, recent=16)
    for i, keep in enumerate((100, 170)):
        want = ob.evict_np(*old, bt[i:i + 1], [200], [keep], 2, 16, keep)
        t = np.arange(keep)
        pages = np.array(kv.seq_pages[i + 1])
        assert len(pages) == -(-keep // 16)
        got = kv.k_pool.view(torch.int16).cpu().numpy()[:, pages[t // 16], t % 16]
        assert np.array_equal(got, want[0][:, bt[i][t // 16], t % 16])
        got = kv.key_weight_pool.cpu().numpy()[:, pages[t // 16], :, t % 16]
        assert np.array_equal(got, want[2][:, bt[i][t // 16], :, t % 16])
    assert not set(kv.seq_pages[1]) & set(kv.seq_pages[2]) and not set(kv.seq_pages[1]) & set(kv.seq_pages[3])
    assert all(torch.equal(a, x[:, kv.seq_pages[3]]) for a, x in zip(third, (kv.k_pool, kv.v_pool, kv.key_weight_pool)))
    free = kv.pages_free
    for s in (1, 2, 3):
        kv.free_sequence(s)
    assert kv.pages_free == 40 and free == 40 - 13 - 7 - 11
    # too few pages to copy into: nothing changes
    small = prism_amd.FlashAttnKVCache(1, NK, HD, 9, 16, gpu)
    small.enable_key_weights()
    small.new_sequence(1)
    small._ensure_capacity(1, 120)
    small.build_packed_batch([1], 120, NH, weight_rows=None)
    small.update_seqlens([1], 120)
    small.fork_sequence(1, 2)
    with pytest.raises(KVCacheOutOfPages):
        small.evict([1], 60)
    assert small.seq_pages[1] == small.seq_pages[2] and small.seq_len[1] == 120 and small.pages_free == 1


def test_a_copy_of_a_weighed_page_is_one(gpu):
    """Its weights came along: a prefix on it adds to them, as on the page itself."""
    kv = prism_amd.FlashAttnKVCache(2, 2, 64, 20, 16, gpu)
    kv.enable_key_weights()
    kv.new_sequence(1)
    kv.prepare_append([1], 64)
    kv.build_packed_batch([1], 64, 4, weight_rows=None)
    kv.key_weight_pool.copy_(torch.arange(kv.key_weight_pool.numel(), device=gpu).view(kv.key_weight_pool.shape))
    kv.update_seqlens([1], 64)
    kv.fork_sequence(1, 2)
    old = list(kv.seq_pages[2])
    kv._copy_on_write([(old[0], new := kv._pop_page(), 16)])
    assert {new, *old[:4]} <= kv._weighed_pages
    assert torch.equal(kv.key_weight_pool[:, new], kv.key_weight_pool[:, old[0]])
    kv.new_sequence(3, prefix_pages=[new, old[1]], prefix_len=32)
    assert kv._weighed[3] == 32


def test_a_captured_decode_step_draws_its_own_tokens(gpu):
    """Attention, weights and the draw in one graph: each replay against the eager calls on the same state."""
    model = Model(gpu, 3)
    kv = prism_amd.FlashAttnKVCache(L, NK, HD, 60, 16, gpu)
    kv.enable_key_weights()
    seqs, lens = [1, 2, 3], [70, 5, 200]
    for s in seqs:
        kv.new_sequence(s)
    _serve_step(model, kv, seqs, torch.arange(sum(lens), device=gpu) % VOCAB, lens)
    kv.prepare_append(seqs, 1)
    batch = kv.build_packed_batch(seqs, 1, NH, weight_rows=None)
    tokens, u = torch.tensor([5, 6, 7], device=gpu), torch.rand(3, device=gpu)
    state = [x.clone() for x in (kv.k_pool, kv.v_pool, kv.key_weight_pool)]

    def back():
        for a, b in zip((kv.k_pool, kv.v_pool, kv.key_weight_pool), state):
            a.copy_(b)

    def whole():
        return prism_amd.sample_tokens(model.step(kv, batch, tokens), u, top_p=0.9, return_logprobs=True)

    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        whole()
    torch.cuda.current_stream(gpu).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        drawn, logs = whole()
    for i in range(3):
        tokens.copy_((tokens * 7 + i) % VOCAB)
        u.uniform_()
        back()
        want, want_logs = whole()
        weights = kv.key_weight_pool.clone()
        back()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(drawn, want) and torch.equal(logs, want_logs) and torch.equal(kv.key_weight_pool, weights)
    batch.release()


def test_refusals(gpu):
    kv = prism_amd.FlashAttnKVCache(1, NK, HD, 8, 16, gpu)
    kc, w = kv.k_caches[0], kv.enable_key_weights()[0]
    batch = prism_amd.PackedBatch([3], [4], [[0]], page_size=16, num_pages=8, n_heads=NH, n_kv=NK, head_dim=HD,
                                  weight_rows=None, device=gpu)
    q, lse = torch.zeros(3, NH, HD, dtype=BF16, device=gpu), torch.zeros(3, NH, device=gpu)
    f = prism_amd.packed_key_weights
    f(q, kc, lse, w, batch)
    for a, kw in [((q.float(), kc, lse, w), {}), ((q[:2], kc, lse, w), {}), ((q, kc.float(), lse, w), {}), ((q, kc[:4], lse, w), {}),
                  ((q, kc, lse.double(), w), {}), ((q, kc, lse[:2], w), {}), ((q, kc, lse[:, :3], w), {}),
                  ((q, kc, lse.t().contiguous().t(), w), {}), ((q, kc, lse.cpu(), w), {}), ((q, kc, lse, w.half()), {}),
                  ((q, kc, lse, w[:4]), {}), ((q, kc, lse, w.transpose(1, 2)), {}), ((q, kc, lse, w.cpu()), {}),
                  ((q, kc, lse, w), dict(window=3)), ((q, kc, lse, w), dict(softmax_scale=0.0)),
                  ((q, kc, lse, w), dict(status=torch.zeros(1, device=gpu)))]:
        with pytest.raises(RuntimeError):
            f(*a, batch, **kw)
    plain = prism_amd.PackedBatch([3], [4], [[0]], page_size=16, num_pages=8, n_heads=NH, n_kv=NK, head_dim=HD, device=gpu)
    with pytest.raises(RuntimeError, match="weight_rows"):
        f(q, kc, lse, w, plain)
    # sampling
    x, u = torch.zeros(4, 10, device=gpu), torch.zeros(4, device=gpu)
    s = prism_amd.sample_tokens
    for a, kw in [((x.double(), u), {}), ((x[0], u), {}), ((x.t().contiguous().t(), u), {}), ((x, u[:3]), {}), ((x, u.double()), {}),
                  ((x, u.cpu()), {}), ((x[:, :0], u), {}), ((x, u), dict(temperature=-1.0)), ((x, u), dict(temperature=float("nan"))),
                  ((x, u), dict(top_p=float("nan"))), ((x, u), dict(min_p=float("nan"))), ((x, u), dict(top_k=u)),
                  ((x, u), dict(temperature=u.double())), ((x, u), dict(top_p=u[:2])), ((x, u), dict(min_p=u.cpu())),
                  ((x[:1].expand(4, 10), u), {})]:
        with pytest.raises(RuntimeError):
            s(*a, **kw)
    for kw in (dict(top_k=1.5), dict(top_p="a"), dict(temperature=None, top_k="x")):
        with pytest.raises(TypeError):
            s(x, u, **kw)
    # eviction
    i = torch.zeros(1, dtype=torch.int32, device=gpu)
    e, bt = prism_amd.evict_keys, torch.zeros(1, 2, dtype=torch.int32, device=gpu)
    k, v, wp = kv.k_pool, kv.v_pool, kv.key_weight_pool
    assert e(k, v, wp, bt, i, i, 3).tolist() == [[[[-1] * 3] * 2]]
    for a, kw in [((k[0], v[0], wp, bt, i, i, 3), {}), ((k.float(), v.float(), wp, bt, i, i, 3), {}), ((k, v[:, :4], wp, bt, i, i, 3), {}),
                  ((k.transpose(2, 3), v.transpose(2, 3), wp, bt, i, i, 3), {}), ((k, v, wp.double(), bt, i, i, 3), {}),
                  ((k, v, wp[:, :4], bt, i, i, 3), {}), ((k, v, wp, bt.long(), i, i, 3), {}), ((k, v, wp, bt[0], i, i, 3), {}),
                  ((k, v, wp, bt, i.cpu(), i, 3), {}), ((k, v, wp, bt, i, bt[0], 3), {}), ((k, v, wp, bt, i, i, -1), {}),
                  ((k, v, wp, bt, i, i, 3), dict(first=-1)), ((k, v, wp, bt, i, i, 3), dict(recent=2.0)),
                  ((k, v, wp, bt, i, i, 3), dict(status=i.float()))]:
        with pytest.raises(RuntimeError):
            e(*a, **kw)


def test_pages_of_a_cut_sequence_with_keys_never_weighed_do_not_count_as_weighed(gpu):
    """evict moves the last keys, which need no weights, into pages that were full of weighed ones."""
    kv = prism_amd.FlashAttnKVCache(1, NK, HD, 20, 16, gpu)
    kv.enable_key_weights()
    kv.new_sequence(1)
    for n, weights in ((64, None), (40, 0)):
        kv.prepare_append([1], n)
        kv.build_packed_batch([1], n, NH, weight_rows=weights)
        kv.update_seqlens([1], n)
    kv.evict([1], 60, recent=40)
    assert kv.seq_len[1] == 60 and kv._weighed[1] == 20
    assert kv._weighed_pages & set(kv.seq_pages[1]) == {kv.seq_pages[1][0]}
    kv.new_sequence(2, prefix_pages=kv.seq_pages[1][:3], prefix_len=48)
    assert kv._weighed[2] == 16


def test_lengths_of_a_cut_sequence_turn_nothing(gpu):
    """The decode calls that take cache_seqlens for positions refuse them; attention alone, and rotation by
    next_positions, go on."""
    kv = prism_amd.FlashAttnKVCache(1, NK, HD, 8, 256, gpu)
    kv.enable_key_weights()
    cos, sin = prism_amd.rope_tables(HD, 512, device=gpu)
    for sid in (1, 2):
        kv.new_sequence(sid)
        kv.prepare_append([sid], 300)
        kv.build_packed_batch([sid], 300, NH, weight_rows=None)
        kv.update_seqlens([sid], 300)
    kv.evict([2], 60)
    kv.prepare_append([1, 2], 1)
    bt, sl = kv.build_block_table([1, 2])
    qkv = torch.randn(2, 1, (NH + 2 * NK) * HD, device=gpu).to(BF16)
    kc, vc = kv.k_caches[0], kv.v_caches[0]
    before = kc.clone()
    append = dict(k_cache=kc, v_cache=vc, block_table=bt, cache_seqlens=sl)
    fused = lambda rows: prism_amd.rope_decode_attention(qkv[rows], kc, vc, cos, sin, cache_seqlens=sl[rows],
                                                         block_table=bt[rows], n_heads=NH, n_kv=NK)
    tables, one = prism_amd.rotary_tables(HD, 512, device=gpu), qkv[:, 0, :NH * HD].unflatten(1, (NH, HD))
    for call in (lambda: fused(slice(0, 2)), lambda: fused(slice(1, 2)), lambda: prism_amd.rotate_qk(one, None, sl, *tables),
                 lambda: prism_amd.rope_qk(qkv, sl, cos, sin, NH, NK, **append)):
        with pytest.raises(RuntimeError, match="next_positions"):
            call()
    assert torch.equal(kc, before)
    fused(slice(0, 1))
    positions = torch.tensor(kv.next_positions([1, 2]), dtype=torch.int32, device=gpu)
    q, _ = prism_amd.rope_qk(qkv, positions, cos, sin, NH, NK, **append)
    prism_amd.rotate_qk(one, None, positions, *tables)
    out = prism_amd.flash_attn_with_kvcache(q, kc, vc, cache_seqlens=sl + 1, block_table=bt, causal=True)
    assert out.isfinite().all()


def test_sequences_that_share_pages_weigh_them_in_turn(gpu):
    """Pages that steps without weights filled: both sequences' attention is in their sums, and decides the eviction."""
    model = Model(gpu, 4)
    kv = prism_amd.FlashAttnKVCache(L, NK, HD, 30, 16, gpu)
    kv.enable_key_weights()
    kv.new_sequence(1)
    kv.prepare_append([1], 96)
    model.step(kv, kv.build_packed_batch([1], 96, NH), torch.arange(96, device=gpu), weigh=False)
    kv.update_seqlens([1], 96)
    kv.fork_sequence(1, 2)
    shared = kv.seq_pages[1][:6]
    # (each step's weights against fp64: the old ones, zero before the first, and what the step adds)
    _serve_step(model, kv, [1], torch.arange(7, 20, device=gpu), [13])
    first = kv.key_weight_pool[:, shared].clone()
    _serve_step(model, kv, [2], torch.arange(40, 45, device=gpu), [5])
    assert (kv.key_weight_pool[:, shared] > first).all()
    _serve_step(model, kv, [1], torch.tensor([5], device=gpu), [1])
    _evict(kv, [1], 50, recent=16)
