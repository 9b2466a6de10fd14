"""packed_attention on the device against fp64, and the packed step as a whole."""
import numpy as np
import pytest
import torch

import prism_amd
from oracle import packed as op
from pkv_testutil import PAIR_CASES, pair_tolerance
from prism_amd.attention import read_status

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _tol(ref, mag, keys):
    """The probabilities are rounded to bf16 (half a step, 2^-8 of each), the sum that divides them is of the rounded
    ones: at most 2^-8 (sum_t p_t |v_t| + |out|).  Scores of N(0, 1) inputs (sums of magnitudes below 16 over 128
    products), exponentials and sums in fp32: below 2^-12 of the same, and 2^-24 per key summed.  The output is
    rounded once: 2^-8 of it."""
    return ref.abs() * 2.0 ** -8 + (mag + ref.abs()) * (2.0 ** -8 + max(2.0 ** -12, keys * 2.0 ** -24))


def _check(out, lse, want, keys, what):
    ref, ref_lse, mag = want
    got = out.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got - ref).abs()
    bad = err > _tol(ref, mag, keys)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(err[bad].max()):.3g}"
    if lse is not None:
        # fp32 scores (magnitudes below 16 over 128 products of 2^-24 each), their exponentials' sum, one logarithm
        e = (lse.double().cpu() - ref_lse).abs()
        tol = 2.0 ** -12 + keys * 2.0 ** -24 + ref_lse.abs() * 2.0 ** -22
        assert (e <= tol).all(), f"{what}: lse off by {float(e.max()):.3g}"


def _case(gpu, new, ctx, P, nh, nk, hd, seed, windows=(None,), extra=0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + c) // P) for n, c in zip(new, ctx)]
    ids = torch.randperm(sum(need) + 3, generator=g)
    bt = np.full((len(new), max(need + [1])), -1, np.int32)
    off = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[off:off + n].numpy()
        off += n
    pages = sum(need) + 3
    kc = torch.randn(pages, P, nk, hd, generator=g).to(BF16)
    vc = torch.randn(pages, P, nk, hd, generator=g).to(BF16)
    q = torch.randn(sum(new) + extra, nh, hd, generator=g).to(BF16)
    batch = prism_amd.PackedBatch(new, ctx, bt, page_size=P, num_pages=pages, n_heads=nh, n_kv=nk, head_dim=hd, windows=windows,
                                  device=gpu)
    return batch, torch.from_numpy(bt), kc, vc, q


LENGTHS = {
    "one": ([1], [0]),
    "short": ([1], [37]),
    "decode": ([1] * 9, [0, 1, 31, 32, 63, 64, 500, 255, 256]),
    "mixed": ([1, 65, 0, 1, 200, 3, 17], [700, 0, 50, 1, 129, 31, 64]),
    "chunk": ([333], [100]),
    "long": ([1, 2, 40], [5000, 3999, 2500]),
}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("nh,nk,hd", [(28, 4, 128), (14, 2, 64), (7, 1, 128), (8, 8, 128), (6, 3, 64), (200, 1, 64)])
@pytest.mark.parametrize("P", [16, 32, 64, 256])
def test_attention(gpu, lengths, nh, nk, hd, P):
    new, ctx = LENGTHS[lengths]
    window = 100 if (nh + P) % 3 == 0 else None
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, nh, nk, hd, seed=nh + P, windows=(None, 100))
    dk, dv, dq = kc.to(gpu), vc.to(gpu), q.to(gpu)
    for w in {None, window}:
        out, lse = prism_amd.packed_attention(dq, dk, dv, batch, window=w, return_lse=True)
        want = op.packed_attention64(q, kc, vc, new, ctx, bt, window=w)
        _check(out, lse, want, max(n + c for n, c in zip(new, ctx)), f"{lengths} window {w}")
        plain = prism_amd.packed_attention(dq, dk, dv, batch, window=w)
        assert torch.equal(plain, out)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 129, 5000])
@pytest.mark.parametrize("P,nh,nk,hd", [(16, 14, 2, 64), (256, 28, 4, 128), (16, 7, 1, 128), (64, 14, 2, 64)])
def test_windows_and_gone_pages(gpu, window, P, nh, nk, hd):
    new, ctx = [1, 70, 5, 1, 300], [900, 500, 63, 0, 33]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, nh, nk, hd, seed=window, windows=(window,))
    sinks = torch.randn(nh, generator=torch.Generator().manual_seed(1)) * 3
    want = op.packed_attention64(q, kc, vc, new, ctx, bt, window=window, sinks=sinks)
    # the pages wholly before the first row's window are gone, and what they held is NaN
    gone = bt.clone()
    for b in range(len(new)):
        first = max(ctx[b] - window + 1, 0) // P
        kc[bt[b, :first].long()] = float("nan")
        vc[bt[b, :first].long()] = float("nan")
        gone[b, :first] = -1
    batch = prism_amd.PackedBatch(new, ctx, gone, page_size=P, num_pages=len(kc), n_heads=nh, n_kv=nk, head_dim=hd,
                                  windows=(window,), device=gpu)
    out, lse = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, window=window, sinks=sinks.to(gpu),
                                          return_lse=True)
    _check(out, lse, want, 900, f"window {window}")
    with pytest.raises(RuntimeError, match="laid out for"):
        prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch)


@pytest.mark.parametrize("P", [16, 256])
def test_stale_rows_behind_the_last_key_do_not_matter(gpu, P):
    new, ctx = [1, 33, 7], [100, 0, 250]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, 14, 2, 64, seed=9)
    want = op.packed_attention64(q, kc, vc, new, ctx, bt)
    keep = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b in range(3):
        t = torch.arange(new[b] + ctx[b])
        keep[bt[b].long()[t // P], t % P] = True
    for bad in (float("nan"), float("inf"), torch.finfo(BF16).min):
        k2, v2 = kc.clone(), vc.clone()
        k2[~keep], v2[~keep] = bad, bad
        _check(prism_amd.packed_attention(q.to(gpu), k2.to(gpu), v2.to(gpu), batch), None, want, 300, f"stale {bad}")


@pytest.mark.parametrize("hd", [64, 128])
def test_extreme_scores_and_sinks(gpu, hd):
    """Scores of thousands: the softmax is a choice of one key, or of the sink."""
    new, ctx = [40, 1], [60, 1999]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, 64, 8, 2, hd, seed=4)
    q = q * 256
    # scores are exact up to 2^-24 of the magnitudes summed (below 256 * 16): 2^-12 of a unit, like N(0, 1) inputs'
    # 2^-12; rows whose two best keys are closer than that are still within the tolerance's p-weighted terms
    for sinks in (None, torch.tensor([-1e30, -3000.0, 0.0, 500.0, 1000.0, 5000.0, float("-inf"), 1e30])):
        want = op.packed_attention64(q, kc, vc, new, ctx, bt, sinks=sinks)
        out, lse = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, return_lse=True,
                                              sinks=sinks.to(gpu) if sinks is not None else None)
        assert torch.isfinite(out).all()
        # a score error d of up to 2^-24 * 128 * 4096 = 2^-5 moves p by p (1 - p) d
        # a weight below the smallest normal fp32 number (2^-126) may be lost: with fewer than 2^11 keys and |v| < 2^3
        # that is less than 2^-112 of the output (rows that a sink leaves next to nothing of)
        err = (out.double().cpu() - want[0]).abs()
        tol = _tol(want[0], want[2], 2000) + 2.0 ** -4 * (want[2] + want[0].abs()) + 2.0 ** -112
        assert (err <= tol).all(), f"{float((err / tol).max())} {float(want[0].flatten()[(err / tol).argmax()])}"
        e = (lse.double().cpu() - want[1]).abs()
        assert (e <= 2.0 ** -5 + want[1].abs() * 2.0 ** -22).all()


def test_scale_strides_out_and_padding(gpu):
    new, ctx = [3, 60, 1], [10, 70, 500]
    nh, nk, hd, P, total = 14, 2, 64, 64, 64
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, nh, nk, hd, seed=2, extra=6)
    want = op.packed_attention64(q[:total], kc, vc, new, ctx, bt, scale=0.3)
    # q a view into the fused projection, the caches views of one pool, out a view with a row of its own
    wide = torch.randn(total + 6, (nh + 4) * hd).to(BF16)
    wide[:, :nh * hd] = q.flatten(1)
    pool = torch.stack([kc, vc], 1).to(gpu)
    out = torch.full((total + 6, nh + 2, hd), 9.0, dtype=BF16, device=gpu)
    got = prism_amd.packed_attention(wide.to(gpu)[:, :nh * hd].unflatten(1, (nh, hd)), pool[:, 0], pool[:, 1], batch,
                                     softmax_scale=0.3, out=out[:, 1:-1])
    assert got.data_ptr() == out[:, 1:-1].data_ptr()
    _check(got[:total], None, want, 600, "views")
    assert (out[:, 0] == 9).all() and (out[:, -1] == 9).all() and (out[total:] == 9).all()
    own, lse = prism_amd.packed_attention(q.to(gpu), pool[:, 0], pool[:, 1], batch, softmax_scale=0.3, return_lse=True)
    assert torch.equal(own[:total], got[:total]) and not own[total:].any() and not lse[total:].any()


def test_nothing_new(gpu):
    for new, ctx in (([], []), ([0, 0], [5, 0])):
        batch, bt, kc, vc, q = _case(gpu, new, ctx, 16, 14, 2, 64, seed=2, extra=3)
        out, lse = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, return_lse=True)
        assert out.shape == (3, 14, 64) and not out.any() and not lse.any()
        cos, sin = prism_amd.rotary_tables(64, 4, device=gpu)
        x = torch.zeros(3, 18 * 64, dtype=BF16, device=gpu)
        assert not prism_amd.packed_rope_append(x, kc.to(gpu), vc.to(gpu), batch, cos, sin).any()


def test_a_page_that_goes_bad_is_flagged(gpu):
    for P in (16, 256):
        batch, bt, kc, vc, q = _case(gpu, [1, 30], [400, 300], P, 14, 2, 64, seed=2)
        batch.block_table[1, 0] = len(kc)
        prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch)
        assert read_status(gpu) == prism_amd._lib.PKV_STATUS_BAD_PAGE


def test_a_list_of_another_batch_is_flagged(gpu):
    """The C entry with the work list of a larger batch: rows outside the call's tensors are not touched."""
    big, bt, kc, vc, q = _case(gpu, [5, 60, 1], [10, 0, 30], 64, 14, 2, 64, seed=2)
    dq, dk, dv = q.to(gpu), kc.to(gpu), vc.to(gpu)
    lib, st = prism_amd._lib.load(), prism_amd.attention.status_tensor(gpu)
    window, items, n_items, merges, n_merges, partials, merge_rows = big._plans[None]
    assert partials == 0
    want = prism_amd.packed_attention(dq, dk, dv, big)
    for tokens, batch in ((65, 3), (66, 2)):     # the last sequence's token, or its block-table row, is not there
        out = torch.full((66, 14, 64), 3.0, dtype=BF16, device=gpu)
        rc = lib.pkv_packed_attn(dq.data_ptr(), 14 * 64, 64, dk.data_ptr(), dv.data_ptr(), dk.stride(0), big.block_table.data_ptr(),
                                 big.max_blocks, out.data_ptr(), 14 * 64, 64, 0, 0, items, n_items, merges, n_merges, partials,
                                 merge_rows, 0, 0, tokens, batch, 14, 2, 64, 64, big.num_pages, big.max_blocks, 0, 0.125,
                                 st.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and read_status(gpu) == prism_amd._lib.PKV_STATUS_BAD_PAGE
        assert torch.equal(out[:65], want[:65]) and (out[65] == 3.0).all()


def test_refusals(gpu):
    batch, bt, kc, vc, q = _case(gpu, [3], [4], 16, 4, 2, 64, seed=2)
    q, kc, vc = q.to(gpu), kc.to(gpu), vc.to(gpu)
    f = prism_amd.packed_attention
    for a, kw in [((q.float(), kc, vc, batch), {}), ((q[:2], kc, vc, batch), {}), ((q[:, :2], kc, vc, batch), {}),
                  ((q.transpose(1, 2).contiguous().transpose(1, 2), kc, vc, batch), {}), ((q, kc.float(), vc.float(), batch), {}),
                  ((q, kc[:, :8], vc[:, :8], batch), {}), ((q, kc[:2], vc[:2], batch), {}), ((q, kc, vc, batch), dict(window=3)),
                  ((q, kc, vc, batch), dict(sinks=torch.zeros(4, dtype=BF16, device=gpu))),
                  ((q, kc, vc, batch), dict(sinks=torch.zeros(3, device=gpu))), ((q, kc, vc, batch), dict(out=q[:, :2])),
                  ((q, kc, vc, batch), dict(out=q.float())), ((q, kc, vc, batch), dict(softmax_scale=0.0))]:
        with pytest.raises(RuntimeError):
            f(*a, **kw)
    with pytest.raises(RuntimeError, match="host"):
        prism_amd.PackedBatch(torch.tensor([1], device=gpu), [0], [[0]], page_size=16, num_pages=1, n_heads=4, n_kv=2, head_dim=64)
    with pytest.raises(RuntimeError, match="before the capture"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            _case(gpu, [3], [4], 16, 4, 2, 64, seed=2)


def test_captured_replayed_and_two_streams(gpu):
    """Calls that split their keys, in two graphs and eagerly on two streams at once: each has partials of its own."""
    new, ctx = [1, 1, 20], [3000, 6000, 2500]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, 64, 28, 4, 128, seed=8)
    assert batch._plans[None][4] > 0
    dk, dv = kc.to(gpu), vc.to(gpu)
    qs = [q.to(gpu), (q * 0.5).to(gpu)]
    graphs, outs = [], []
    for x in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(prism_amd.packed_attention(x, dk, dv, batch, return_lse=True))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for i in range(4):
        for x in qs:
            x.normal_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
            eager1 = prism_amd.packed_attention(qs[0], dk, dv, batch, return_lse=True)
        eager0 = prism_amd.packed_attention(qs[1], dk, dv, batch, return_lse=True)
        torch.cuda.synchronize()
        for a, b in ((outs[0], eager1), (outs[1], eager0)):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]), i
    want = op.packed_attention64(qs[0].cpu(), kc, vc, new, ctx, bt)
    _check(*outs[0], want, 6001, "replayed")


def test_same_bits_every_time(gpu):
    batch, bt, kc, vc, q = _case(gpu, [1, 50, 1], [9000, 2000, 10], 256, 28, 4, 128, seed=8)
    a = [prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, return_lse=True) for _ in range(5)]
    assert all(torch.equal(a[0][0], b[0]) and torch.equal(a[0][1], b[1]) for b in a[1:])


@pytest.mark.parametrize("nh,nk,hd,P,window", [(28, 4, 128, 256, None), (14, 2, 64, 16, 40), (7, 1, 128, 16, None)])
def test_steps_of_a_served_batch(gpu, nh, nk, hd, P, window):
    """Three steps (prompts; a mix with a forked sequence; decode) through the cache: every step's queries, cache and
    attention against a history kept in fp64 from the inputs, and the pages that others share left alone."""
    kv = prism_amd.FlashAttnKVCache(1, nk, hd, 64 if P == 256 else 200, P, gpu)
    g = torch.Generator().manual_seed(nh)
    cos, sin = prism_amd.rotary_tables(hd, 4096, 1e4, device=gpu)
    freq = 1e4 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    for s in (1, 2, 3):
        kv.new_sequence(s)
    hist = {s: [] for s in (1, 2, 3, 4)}
    steps = [([1, 2, 3], [300, 45, 1]), ([3, 1, 2], [1, 70, 1]), ([4, 1, 3, 2], [5, 1, 1, 130]), ([1, 2, 3, 4], [1, 1, 1, 1])]
    for ids, counts in steps:
        if 4 in ids and 4 not in kv.seq_pages:
            kv.fork_sequence(2, 4)
            hist[4] = list(hist[2])
        kv.prepare_append(ids, counts)
        batch = kv.build_packed_batch(ids, counts, nh, windows=(window,))
        x = torch.randn(sum(counts), (nh + 2 * nk) * hd, generator=g).to(BF16)
        q = prism_amd.packed_rope_append(x.to(gpu), kv.k_caches[0], kv.v_caches[0], batch, cos, sin)
        out, lse = prism_amd.packed_attention(q, kv.k_caches[0], kv.v_caches[0], batch, window=window, return_lse=True)
        ctx = [kv.seq_len[s] for s in ids]
        kv.update_seqlens(ids, counts)
        pos = batch.positions.cpu()
        want, mag = op.rotate64(x[:, :(nh + nk) * hd].unflatten(1, (nh + nk, hd)), pos, freq)
        tol = want.abs() * 2.0 ** -8 + mag * 2.0 ** -20
        assert ((q.double().cpu() - want[:, :nh]).abs() <= tol[:, :nh]).all()
        first = 0
        bt, _ = kv.block_table_host(ids)
        for s, n in zip(ids, counts):
            hist[s] += [(want[i, nh:], tol[i, nh:], x[i, (nh + nk) * hd:].unflatten(0, (nk, hd))) for i in range(first, first + n)]
            first += n
            at = torch.arange(len(hist[s]))
            row = torch.tensor(kv.seq_pages[s])[at // P]
            k, v = kv.k_caches[0].cpu()[row, at % P], kv.v_caches[0].cpu()[row, at % P]
            assert ((k.double() - torch.stack([h[0] for h in hist[s]])).abs() <= torch.stack([h[1] for h in hist[s]])).all()
            assert torch.equal(v, torch.stack([h[2] for h in hist[s]]))
        ref = op.packed_attention64(q.cpu(), kv.k_caches[0].cpu(), kv.v_caches[0].cpu(), counts, ctx, torch.from_numpy(bt), window=window)
        _check(out, lse, ref, 500, f"step {ids}")
        if window is None:
            # the framework's other attention, sequence by sequence over the same pages
            first = 0
            for i, (s, n) in enumerate(zip(ids, counts)):
                o = prism_amd.flash_attn_with_kvcache(q[None, first:first + n], kv.k_caches[0], kv.v_caches[0],
                                                      cache_seqlens=torch.tensor([kv.seq_len[s]], dtype=torch.int32, device=gpu),
                                                      block_table=torch.from_numpy(bt[i:i + 1]).to(gpu), causal=True)
                t = _tol(ref[0][first:first + n], ref[2][first:first + n], 500)
                assert ((o[0].double().cpu() - ref[0][first:first + n]).abs() <= t).all()
                first += n


def test_pages_past_32_bits(gpu):
    """A pool of 2.4e9 elements: pages whose offset does not fit 32 bits, of bytes or of elements."""
    P, nk, hd, nh = 256, 8, 128, 40
    pages = 9200
    kc = torch.zeros(pages, P, nk, hd, dtype=BF16, device=gpu)
    vc = torch.zeros_like(kc)
    bt = np.array([[9199, 9100], [4097, 8193]], np.int32)
    new, ctx = [3, 200], [300, 100]
    batch = prism_amd.PackedBatch(new, ctx, bt, page_size=P, num_pages=pages, n_heads=nh, n_kv=nk, head_dim=hd, device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    for p in bt.ravel().tolist():
        kc[p].normal_(generator=g)
        vc[p].normal_(generator=g)
    cos, sin = prism_amd.rotary_tables(hd, 400, device=gpu)
    x = torch.empty(203, (nh + 2 * nk) * hd, dtype=BF16, device=gpu).normal_(generator=g)
    q = prism_amd.packed_rope_append(x, kc, vc, batch, cos, sin)
    assert torch.equal(vc[9100, 44:47], x[:3, (nh + nk) * hd:].unflatten(1, (nk, hd)))
    assert torch.equal(vc[4097, 100:], x[3:159, (nh + nk) * hd:].unflatten(1, (nk, hd)))
    out, lse = prism_amd.packed_attention(q, kc, vc, batch, return_lse=True)
    ids = sorted(set(bt.ravel().tolist()))
    mini = torch.tensor([[ids.index(p) for p in row] for row in bt.tolist()])
    at = torch.tensor(ids, device=gpu)
    want = op.packed_attention64(q.cpu(), kc[at].cpu(), vc[at].cpu(), new, ctx, mini)
    _check(out, lse, want, 303, "far pages")
    del kc, vc
    torch.cuda.empty_cache()


def test_a_graph_outlives_the_batch_and_a_stream_its_use(gpu):
    new, ctx = [1, 40], [700, 300]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, 64, 14, 2, 64, seed=3)
    dq, dk, dv = q.to(gpu), kc.to(gpu), vc.to(gpu)
    want = prism_amd.packed_attention(dq, dk, dv, batch)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = prism_amd.packed_attention(dq, dk, dv, batch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prism_amd.packed_attention(dq, dk, dv, batch)
    size = batch._buf.numel()
    del batch
    for i in range(3):
        junk = [torch.full((size,), -7 - i, dtype=torch.int32, device=gpu) for _ in range(50)]   # would land in freed memory
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        del junk
    assert torch.equal(other, want)


@pytest.mark.parametrize("nh,nk,hd,P", [(28, 4, 128, 256), (14, 2, 64, 16)])
def test_many_ranges_of_one_block(gpu, nh, nk, hd, P):
    """One decode token and one short chunk on 20,000 keys: some twenty partials of a row to merge."""
    new, ctx = [1, 30], [20000, 9000]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, nh, nk, hd, seed=5, windows=(None, 7000))
    for w in (None, 7000):
        out, lse = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, window=w, return_lse=True)
        _check(out, lse, op.packed_attention64(q, kc, vc, new, ctx, bt, window=w), 20001, f"window {w}")


@pytest.mark.parametrize("new,ctx", [([1, 1], [5000, 40]), ([300, 1], [900, 2]), ([40, 6], [3000, 2900])])
def test_nan_stays_where_it_is_seen(gpu, new, ctx):
    """A NaN query spoils its head's row, a NaN key the rows that see it, whatever the ranges; nothing else."""
    batch, bt, kc, vc, q = _case(gpu, new, ctx, 64, 14, 2, 64, seed=6)
    clean, clean_lse = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, return_lse=True)
    bad_q = q.clone()
    bad_q[0, 5, 9] = float("nan")
    out, lse = prism_amd.packed_attention(bad_q.to(gpu), kc.to(gpu), vc.to(gpu), batch, return_lse=True)
    hit = torch.zeros(out.shape[:2], dtype=torch.bool, device=gpu)
    hit[0, 5] = True
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit])
    # key t of sequence 0, KV head 1: seen from position t on, by the second half of the heads
    for t in (3, ctx[0], ctx[0] + new[0] - 1):
        bad_k = kc.clone()
        bad_k[int(bt[0, t // 64]), t % 64, 1, 17] = float("nan")
        out, lse = prism_amd.packed_attention(q.to(gpu), bad_k.to(gpu), vc.to(gpu), batch, return_lse=True)
        hit = torch.zeros(out.shape[:2], dtype=torch.bool, device=gpu)
        hit[max(t - ctx[0], 0):new[0], 7:] = True
        assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all(), t
        assert torch.equal(out[~hit], clean[~hit]) and torch.equal(lse[~hit], clean_lse[~hit]), t


def test_ranges_merge_in_the_launch_and_behind_it(gpu):
    """Row blocks of 1 to 128 rows around the 32 that one wave holds, one to 70 ranges, replayed: the merge's two ways
    and its tags."""
    new, ctx = [1, 2, 4, 5, 18, 19, 1], [30000, 4000, 4000, 4000, 4000, 4000, 300]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, 256, 28, 4, 128, seed=12)
    dk, dv, dq = kc.to(gpu), vc.to(gpu), q.to(gpu)
    sinks = torch.randn(28, generator=torch.Generator().manual_seed(2))
    want = op.packed_attention64(q, kc, vc, new, ctx, bt, sinks=sinks)
    graph = torch.cuda.CUDAGraph()
    first = prism_amd.packed_attention(dq, dk, dv, batch, sinks=sinks.to(gpu), return_lse=True)
    sk = sinks.to(gpu)
    with torch.cuda.graph(graph):
        out, lse = prism_amd.packed_attention(dq, dk, dv, batch, sinks=sk, return_lse=True)
    for i in range(20):
        out.zero_()
        lse.zero_()
        graph.replay()
        if i % 5 == 0:
            torch.cuda.synchronize()
            eager = prism_amd.packed_attention(dq, dk, dv, batch, sinks=sk, return_lse=True)
            assert torch.equal(eager[0], out) and torch.equal(eager[1], lse), i
    assert torch.equal(first[0], out) and torch.equal(first[1], lse)
    _check(out, lse, want, 30001, "merged")


@pytest.mark.parametrize("keys", [70001, 300001])
def test_one_sequence_in_more_than_64_ranges(gpu, keys):
    """One row block on a card of its own: its ranges merge in the launch, or, where they are more than a wave's
    lanes, in a launch behind."""
    new, ctx = [1], [keys - 1]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, 256, 7, 1, 128, seed=13)
    merges, ranges = batch._plans[None][4:6]
    assert (merges, ranges > 64) == ((0, False) if keys < 100000 else (1, True)) and ranges > 32
    out, lse = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, return_lse=True)
    _check(out, lse, op.packed_attention64(q, kc, vc, new, ctx, bt), keys, "many ranges")


@pytest.mark.parametrize("nh,nk,hd", [(8, 2, 128), (8, 2, 64)])
def test_sinks_past_every_score(gpu, nh, nk, hd):
    """A sink of +inf, or one whose product with log2 e overflows, takes all of the weight: the row is 0 and its
    log-sum-exp the sink, decode rows and chunk rows alike, in one range or several."""
    new, ctx = [1, 40, 1, 9], [5, 60, 6000, 3000]
    batch, bt, kc, vc, q = _case(gpu, new, ctx, 64, nh, nk, hd, seed=4, windows=(None, 50))
    top = torch.finfo(torch.float32).max
    sinks = torch.tensor([float("inf"), top, 0.5, float("inf"), -top, 2.5e38, float("-inf"), 1.0])
    for window in (None, 50):
        out, lse = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch, window=window, sinks=sinks.to(gpu),
                                              return_lse=True)
        all_of_it = [0, 1, 3, 5]
        assert not out[:, all_of_it].any()
        assert torch.equal(lse[:, all_of_it].cpu(), sinks[all_of_it].expand(sum(new), 4))
        rest = [2, 4, 6, 7]
        want = op.packed_attention64(q, kc, vc, new, ctx, bt, window=window, sinks=sinks)
        _check(out[:, rest], lse[:, rest], [x[:, rest] for x in want], 6001, f"window {window}")


def test_a_status_word_elsewhere_is_refused(gpu):
    """The kernels write to the status word: one that is not the device's, or none, never reaches them."""
    batch, bt, kc, vc, q = _case(gpu, [3], [4], 16, 4, 2, 64, seed=2)
    q, kc, vc = q.to(gpu), kc.to(gpu), vc.to(gpu)
    cos, sin = prism_amd.rotary_tables(64, 8, device=gpu)
    x = torch.zeros(3, 8 * 64, dtype=BF16, device=gpu)
    for status in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int64, device=gpu),
                   torch.zeros(0, dtype=torch.int32, device=gpu)):
        for call in (lambda: prism_amd.packed_attention(q, kc, vc, batch, status=status),
                     lambda: prism_amd.packed_rope_append(x, kc, vc, batch, cos, sin, status=status),
                     lambda: prism_amd.rotate_qk(q, None, batch.positions, cos, sin, status=status)):
            with pytest.raises(RuntimeError, match="status"):
                call()
    own = torch.zeros(1, dtype=torch.int32, device=gpu)
    batch.block_table[0, 0] = -1
    prism_amd.packed_attention(q, kc, vc, batch, status=own)
    assert own.item() == prism_amd._lib.PKV_STATUS_BAD_PAGE and read_status(gpu) == 0


def test_captures_again_and_again_do_not_grow(gpu):
    """A graph captured anew for every batch, the old one released: the lists' memory comes back."""
    def step(seed):
        batch, bt, kc, vc, q = _case(gpu, [1, 40], [700, 300], 64, 14, 2, 64, seed=seed)
        dq, dk, dv = q.to(gpu), kc.to(gpu), vc.to(gpu)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = prism_amd.packed_attention(dq, dk, dv, batch)
        for _ in range(2):
            out.zero_()
            graph.replay()
            assert torch.equal(out, prism_amd.packed_attention(dq, dk, dv, batch))
        torch.cuda.synchronize()
        del graph
        batch.release()
    step(0)
    held, memory = len(prism_amd.packed._captured), torch.cuda.memory_allocated()
    for seed in range(1, 5):
        step(seed)
        assert len(prism_amd.packed._captured) == held and torch.cuda.memory_allocated() <= memory


@pytest.mark.parametrize("window", [None, 90])
@pytest.mark.parametrize("nh,nk,hd", [(4, 4, 128), (4, 4, 64), (4, 2, 128), (14, 2, 64)])
def test_a_bad_value_stays_in_its_blocks(gpu, nh, nk, hd, window):
    """A NaN or infinity in a V row: rows that see the key are not finite, rows of a block of 128 that sees one of the
    same 32 (64) keys may be (with one query head per KV head a block is 128 tokens), all others keep their bits."""
    new, ctx, P, g, tok = [400, 9, 1], [3000, 70, 900], 64, nh // nk, 32 if hd == 128 else 64
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, nh, nk, hd, seed=6, windows=(window,))
    dq, dk = q.to(gpu), kc.to(gpu)
    clean, lse = prism_amd.packed_attention(dq, dk, vc.to(gpu), batch, window=window, return_lse=True)
    first = [0, 400, 409]
    for b, t, bad in [(0, 3300, float("nan")), (0, 3127, float("inf")), (0, 2950, float("nan")), (1, 74, float("-inf")), (2, 850, float("nan"))]:
        v = vc.clone()
        v[int(bt[b, t // P]), t % P, 1, 5] = bad
        out, lse2 = prism_amd.packed_attention(dq, dk, v.to(gpu), batch, window=window, return_lse=True)
        assert torch.equal(lse, lse2)
        may, must = torch.zeros(out.shape[:2], dtype=torch.bool, device=gpu), torch.zeros(out.shape[:2], dtype=torch.bool, device=gpu)
        rows = torch.arange(new[b] * g, device=gpu)
        pos = ctx[b] + rows // g
        sees = (pos >= t) & (pos - t < (window or 1 << 30))
        for r0 in range(0, new[b] * g, 128):
            block = rows[r0:r0 + 128]
            lo, hi = int(pos[r0]) - (window or 1 << 30) + 1, int(pos[block[-1]])
            if max(lo, 0) // tok <= t // tok <= hi // tok:
                may[first[b] + block // g, g + block % g] = True
        must[first[b] + rows[sees] // g, g + rows[sees] % g] = True
        assert not torch.isfinite(out[must][:, 5]).any()
        assert torch.equal(out[~may], clean[~may])
        good = [d for d in range(hd) if d != 5]
        assert torch.equal(out[..., good], clean[..., good])


@pytest.mark.parametrize("new,ctx", PAIR_CASES)
@pytest.mark.parametrize("nh,nk,hd,P", [(7, 1, 128, 256), (14, 2, 64, 16), (8, 8, 128, 64)])
def test_decode_rows_round_their_probabilities_to_a_pair(gpu, new, ctx, nh, nk, hd, P):
    """Blocks of at most 16 rows, whole and in ranges: their outputs are off by little more than their own rounding."""
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, nh, nk, hd, seed=21)
    assert max(new) * (nh // nk) <= 16
    out = prism_amd.packed_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), batch)
    ref, _, mag = op.packed_attention64(q, kc, vc, new, ctx, bt)
    err = (out.double().cpu() - ref).abs()
    tol = pair_tolerance(ref, mag, max(n + c for n, c in zip(new, ctx)))
    assert (err <= tol).all(), f"{int((err > tol).sum())} off, worst {float((err / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("nh,nk,hd", [(28, 4, 128), (14, 2, 64)])
def test_a_list_with_more_partials_than_the_call(gpu, nh, nk, hd):
    """Work lists of split blocks, some merged in the launch and some behind it, with room for fewer partials than they
    name: blocks whose partials fit are done, of the others nothing is written, and nothing past the workspace or the
    tensors."""
    new, ctx, P = [1, 40, 1, 3, 40], [9000, 5000, 20, 7000, 30], 64
    batch, bt, kc, vc, q = _case(gpu, new, ctx, P, nh, nk, hd, seed=14)
    dq, dk, dv = q.to(gpu), kc.to(gpu), vc.to(gpu)
    lib, st = prism_amd._lib.load(), prism_amd.attention.status_tensor(gpu)
    _, items, n_items, merges, n_merges, partials, merge_rows = batch._plans[None]
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    lengths = [np.asarray(x, np.int32) for x in (new, ctx)]
    listed, merged, _ = batch._plan((lengths[0].ctypes.data, lengths[1].ctypes.data, len(new)), None, cus)
    assert len(listed) == n_items and len(merged) == n_merges > 0 and (listed[:, 9] > 0).any() and (listed[:, 7] < 0).any()
    want = prism_amd.packed_attention(dq, dk, dv, batch)
    total, g = sum(new), nh // nk
    for room in sorted({0, 1, partials // 3, partials // 2, partials - 1}):
        need = lib.pkv_packed_workspace_bytes(room, nk, hd)
        ws = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device=gpu)
        out = torch.full((total + 4, nh, hd), 3.0, dtype=BF16, device=gpu)
        rc = lib.pkv_packed_attn(dq.data_ptr(), nh * hd, hd, dk.data_ptr(), dv.data_ptr(), dk.stride(0), batch.block_table.data_ptr(),
                                 batch.max_blocks, out.data_ptr(), nh * hd, hd, 0, 0, items, n_items, merges, n_merges, room,
                                 merge_rows, ws.data_ptr(), need, total, len(new), nh, nk, hd, P, batch.num_pages,
                                 batch.max_blocks, 0, hd ** -0.5, st.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and read_status(gpu) == prism_amd._lib.PKV_STATUS_BAD_PAGE
        done = torch.zeros(total, nh, dtype=torch.bool)
        for t0, n, _, _, row0, _, _, slot, first, count, *_ in listed.tolist():
            last = slot if slot < 0 else first + count - 1 if count else \
                next(m[3] + m[4] - 1 for m in merged.tolist() if (m[0], m[2]) == (t0, row0))
            rows = torch.arange(row0, min(row0 + 128, n * g))
            for h in range(nk):
                done[t0 + rows // g, h * g + rows % g] = last < room
        done = done.to(gpu)
        assert done.any() and not done.all()
        assert torch.equal(out[:total][done], want[done]), room
        assert (out[:total][~done] == 3.0).all() and (out[total:] == 3.0).all(), room
        assert (ws[need:] == 0x5A).all(), room
