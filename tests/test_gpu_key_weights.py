"""packed_key_weights on the device against fp64."""
import numpy as np
import pytest
import torch

import prism_amd
from oracle import behind as ob
from prism_amd.attention import read_status

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _case(gpu, new, ctx, P, nh, nk, hd, seed, *, windows=(None,), rows=None, weighed=None, extra=0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + c) // P) for n, c in zip(new, ctx)]
    pages = sum(need) + 3
    ids = torch.randperm(pages, generator=g)
    bt = np.full((len(new), max(need + [1])), -1, np.int32)
    off = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[off:off + n].numpy()
        off += n
    kc = torch.randn(pages, P, nk, hd, generator=g).to(BF16)
    q = torch.randn(sum(new) + extra, nh, hd, generator=g).to(BF16)
    w = torch.rand(pages, nk, P, generator=g)
    seen = torch.cat([torch.arange(c, c + n) + 1.0 for n, c in zip(new, ctx)] + [torch.ones(extra)])
    lse = seen.log()[:, None] + q.float().square().sum(-1) / (2 * hd)
    batch = prism_amd.PackedBatch(new, ctx, bt, page_size=P, num_pages=pages, n_heads=nh, n_kv=nk, head_dim=hd,
                                  windows=windows, weight_rows=rows, weighed=weighed, device=gpu)
    return batch, torch.from_numpy(bt), kc, q, lse, w


def _check(got, want, gain, old, terms, what):
    """A term is exp of a score less its lse: the fp32 score is off by at most 128 roundings of 2^-24 of a magnitude
    below 16 (N(0, 1) inputs over sqrt(head_dim)), so 2^-13; in log2 units the difference (below 32) is rounded once
    more, 2^-24 of it, and the exponential by 2^-22 of itself: together below 2^-12 of each term.  Summing rounds every
    partial sum, 2^-24 for each term, and the sum with the old weight once."""
    got = got.double().cpu()
    tol = gain * (2.0 ** -12 + terms * 2.0 ** -24) + (old.double() + gain) * 2.0 ** -23
    err = (got - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - tol).max()):.3g}"
    assert torch.equal(got[gain == 0], want[gain == 0]), f"{what}: a key that nobody weighed changed"


LENGTHS = {
    "one": ([1], [0]),
    "short": ([1], [37]),
    "decode": ([1] * 9, [0, 1, 31, 32, 63, 64, 500, 255, 256]),
    "verify": ([5, 4, 1, 9], [700, 33, 0, 16]),
    "mixed": ([1, 65, 0, 1, 200, 3, 17], [700, 0, 50, 1, 129, 31, 64]),
    "chunk": ([333], [100]),
    "long": ([1, 2, 40], [5000, 3999, 2500]),
}


@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("nh,nk,hd", [(28, 4, 128), (14, 2, 64), (7, 1, 128), (8, 8, 128), (6, 3, 64), (200, 1, 64)])
@pytest.mark.parametrize("P", [16, 64, 256])
def test_weights(gpu, lengths, nh, nk, hd, P):
    new, ctx = LENGTHS[lengths]
    for rows in (None, 7):
        batch, bt, kc, q, lse, w = _case(gpu, new, ctx, P, nh, nk, hd, seed=nh + P, windows=(None, 100), rows=rows)
        for window in (None, 100):
            print("weights", lengths, nh, nk, hd, P, rows, window, flush=True)
            want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt, window=window, rows=rows)
            dw = w.to(gpu)
            got = prism_amd.packed_key_weights(q.to(gpu), kc.to(gpu), lse.to(gpu), dw, batch, window=window)
            assert got is dw or got.data_ptr() == dw.data_ptr()
            _check(got, want, gain, w, max(new) * (nh // nk), f"{lengths} rows {rows} window {window}")


@pytest.mark.parametrize("hd", [64, 128])
def test_row_counts_on_either_side_of_the_two_ways(gpu, hd):
    """128 query rows of a sequence stream its keys, 132 are streamed past them."""
    new, ctx = [32, 33, 31, 1], [5000, 300, 31, 4000]
    batch, bt, kc, q, lse, w = _case(gpu, new, ctx, 64, 16, 4, hd, seed=hd)
    assert batch._weight_plans[None][2] > 0 and batch._weight_plans[None][3] == 2  # 333 keys, blocks of 256
    want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt)
    got = prism_amd.packed_key_weights(q.to(gpu), kc.to(gpu), lse.to(gpu), w.to(gpu), batch)
    _check(got, want, gain, w, 33 * 4, f"head_dim {hd}")


@pytest.mark.parametrize("new,ctx,nh,nk,hd", [([2000], [0], 28, 4, 128), ([900, 1, 1400], [3000, 9000, 100], 14, 2, 64),
                                              ([700, 300], [0, 12000], 7, 1, 128)])
def test_split_rows(gpu, new, ctx, nh, nk, hd):
    """Blocks whose rows are cut into several items, merged in the list's order."""
    batch, bt, kc, q, lse, w = _case(gpu, new, ctx, 256, nh, nk, hd, seed=5)
    assert batch._weight_plans[None][4] > 0, "nothing was split"
    want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt)
    d = [x.to(gpu) for x in (q, kc, lse)]
    got = prism_amd.packed_key_weights(*d, w.to(gpu), batch)
    _check(got, want, gain, w, max(new) * (nh // nk), "split")
    assert torch.equal(prism_amd.packed_key_weights(*d, w.to(gpu), batch), got), "the bits do not repeat"


@pytest.mark.parametrize("window", [1, 2, 31, 33, 129, 5000])
@pytest.mark.parametrize("P,nh,nk,hd", [(16, 14, 2, 64), (256, 28, 4, 128)])
def test_gone_pages_and_masked_nans(gpu, window, P, nh, nk, hd):
    """Pages out of every row's window are gone, what is masked or behind the last key is NaN: neither matters."""
    new, ctx = [1, 70, 5, 1, 300], [900, 500, 63, 0, 33]
    batch, bt, kc, q, lse, w = _case(gpu, new, ctx, P, nh, nk, hd, seed=window, windows=(window,))
    want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt, window=window)
    gone, bad = bt.clone(), kc.clone()
    bad[:] = float("nan")
    for b in range(len(new)):
        lo, end = max(ctx[b] - window + 1, 0), ctx[b] + new[b]
        at = torch.arange(lo, end)
        bad[bt[b, at // P].long(), at % P] = kc[bt[b, at // P].long(), at % P]
        gone[b, :lo // P] = -1
    batch = prism_amd.PackedBatch(new, ctx, gone, page_size=P, num_pages=len(kc), n_heads=nh, n_kv=nk, head_dim=hd,
                                  windows=(window,), weight_rows=None, device=gpu)
    got = prism_amd.packed_key_weights(q.to(gpu), bad.to(gpu), lse.to(gpu), w.to(gpu), batch, window=window)
    _check(got, want, gain, w, 2100, f"window {window}")


def test_infinite_lse_weighs_nothing_and_nan_stays_with_what_sees_it(gpu):
    new, ctx, nh, nk, hd, P = [1, 1, 30], [50, 60, 70], 14, 2, 64, 16
    batch, bt, kc, q, lse, w = _case(gpu, new, ctx, P, nh, nk, hd, seed=3)
    lse[0, 2], lse[0, 5], lse[5, 1] = float("inf"), -float("inf"), -float("inf")
    want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt)
    args = [x.to(gpu) for x in (q, kc)]
    got = prism_amd.packed_key_weights(*args, lse.to(gpu), w.to(gpu), batch)
    _check(got, want, gain, w, 210, "infinite lse")
    lse[1, 0] = float("nan")   # sequence 1, head 0: KV head 0
    got = prism_amd.packed_key_weights(*args, lse.to(gpu), w.to(gpu), batch).cpu()
    nan = torch.zeros_like(w, dtype=torch.bool)
    at = torch.arange(61)
    nan[bt[1, at // P].long(), 0, at % P] = True
    assert torch.equal(got.isnan(), nan)


def test_keys_not_weighed_yet_start_from_nothing(gpu):
    new, ctx, P = [1, 40, 3], [100, 90, 0], 16
    for window in (None, 20):
        batch, bt, kc, q, lse, w = _case(gpu, new, ctx, P, 14, 2, 64, seed=8, weighed=[30, 90, 5], windows=(window,), rows=4)
        want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt, weighed=[30, 90, 5], window=window, rows=4)
        got = prism_amd.packed_key_weights(q.to(gpu), kc.to(gpu), lse.to(gpu), w.to(gpu), batch, window=window)
        _check(got, want, gain, w, 28, f"weighed, window {window}")


def test_strided_and_padded(gpu):
    """q inside a wider projection, pools with a page stride, rows behind the batch's tokens."""
    new, ctx, nh, nk, hd, P = [1, 90], [200, 30], 14, 2, 64, 16
    batch, bt, kc, q, lse, w = _case(gpu, new, ctx, P, nh, nk, hd, seed=4, extra=5)
    want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt)
    wide = torch.full((len(q), nh, 2 * hd), float("nan"), dtype=BF16, device=gpu)
    wide[..., :hd] = q.to(gpu)
    wide[91:] = float("nan")
    pool = torch.full((len(kc), 2, P, nk, hd), float("nan"), dtype=BF16, device=gpu)
    pool[:, 1] = kc.to(gpu)
    wpool = torch.full((len(kc), nk + 1, P), 7.0, device=gpu)
    wpool[:, :nk] = w.to(gpu)
    lpool = torch.zeros(len(q), nh + 3, device=gpu)
    lpool[:, :nh] = lse.to(gpu)
    got = prism_amd.packed_key_weights(wide[..., :hd], pool[:, 1], lpool[:, :nh], wpool[:, :nk], batch)
    _check(got, want, gain, w, 630, "strided")
    assert (wpool[:, nk] == 7.0).all()


def test_scale_streams_and_graphs(gpu):
    new, ctx, nh, nk, hd, P = [1, 1, 60], [300, 900, 100], 28, 4, 128, 64
    batch, bt, kc, q, lse, w = _case(gpu, new, ctx, P, nh, nk, hd, seed=6)
    want, gain = ob.key_weights64(q, kc, lse, w, new, ctx, bt, scale=0.05)
    d = [x.to(gpu) for x in (q, kc, lse)]
    eager = prism_amd.packed_key_weights(*d, w.to(gpu), batch, softmax_scale=0.05)
    _check(eager, want, gain, w, 420, "scale")
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        other = prism_amd.packed_key_weights(*d, w.to(gpu), batch, softmax_scale=0.05)
    side.synchronize()
    assert torch.equal(other, eager)
    dw = w.to(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        prism_amd.packed_key_weights(*d, dw, batch, softmax_scale=0.05)
    for _ in range(3):
        dw.copy_(w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, eager)
        prism_amd.packed_key_weights(*d, w.to(gpu), batch)
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(dw, eager)   # added to once more
    batch.release()


@pytest.mark.parametrize("nh,nk,hd", [(28, 4, 128), (14, 2, 64)])
def test_the_weights_of_a_step_sum_to_its_rows(gpu, nh, nk, hd):
    """With the lse that packed_attention returns, every (token, head) hands out a weight of one."""
    new, ctx, P = [1, 130, 7, 1], [1000, 20, 0, 64], 64
    batch, bt, kc, q, _, w = _case(gpu, new, ctx, P, nh, nk, hd, seed=7)
    dq, dk = q.to(gpu), kc.to(gpu)
    _, lse = prism_amd.packed_attention(dq, dk, dk, batch, return_lse=True)
    got = prism_amd.packed_key_weights(dq, dk, lse, torch.zeros_like(w, device=gpu), batch).double().cpu()
    # attention's own lse is within 2^-12 (test_gpu_packed), the weights' terms within 2^-12 of theirs
    for b, (n, c) in enumerate(zip(new, ctx)):
        at = torch.arange(n + c)
        per_head = got[bt[b, at // P].long(), :, at % P].sum(0)
        assert (per_head - n * nh // nk).abs().max() <= n * nh // nk * 2.0 ** -11, b


def test_pages_past_32_bits(gpu):
    """A pool whose last pages lie past 2^31 elements (and 2^32 bytes) of K."""
    P, nk, hd, nh = 256, 4, 128, 28
    pages = (1 << 31) // (P * nk * hd) + 40
    pool = torch.zeros(pages, P, nk, hd, dtype=BF16, device=gpu)
    new, ctx = [1, 20], [700, 300]
    g = torch.Generator().manual_seed(0)
    bt = torch.full((2, 3), -1, dtype=torch.int32)
    bt[0, :3] = torch.tensor([pages - 1, 5, pages - 7])
    bt[1, :2] = torch.tensor([pages - 3, pages - 2])
    used = torch.unique(bt[bt >= 0]).long()
    small = torch.randn(len(used), P, nk, hd, generator=g).to(BF16)
    pool[used.to(gpu)] = small.to(gpu)
    remap = torch.full((pages,), -1, dtype=torch.int32)
    remap[used] = torch.arange(len(used), dtype=torch.int32)
    q = torch.randn(21, nh, hd, generator=g).to(BF16)
    lse = torch.full((21, nh), 6.0)
    w = torch.zeros(pages, nk, P, device=gpu)
    batch = prism_amd.PackedBatch(new, ctx, bt, page_size=P, num_pages=pages, n_heads=nh, n_kv=nk, head_dim=hd,
                                  weight_rows=None, device=gpu)
    got = prism_amd.packed_key_weights(q.to(gpu), pool, lse.to(gpu), w, batch)
    small_bt = torch.where(bt >= 0, remap[bt.clamp(min=0).long()], -1)
    w0 = torch.zeros(len(used), nk, P)
    want, gain = ob.key_weights64(q, small, lse, w0, new, ctx, small_bt)
    _check(got[used.to(gpu)], want, gain, w0, 140, "far pages")
    assert int((got != 0).sum()) == int((got[used.to(gpu)] != 0).sum())


def test_a_list_of_another_batch_is_skipped_and_flagged(gpu):
    """Items that do not fit the call (here: fewer tokens) are left out, in bounds."""
    small, _, kc, q, lse, w = _case(gpu, [1], [100], 16, 14, 2, 64, seed=1)
    large, *_ = _case(gpu, [1, 1, 1], [100, 90, 80], 16, 14, 2, 64, seed=1)
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    mixed = prism_amd.PackedBatch([1], [100], small.block_table.cpu().numpy(), page_size=16, num_pages=len(kc), n_heads=14,
                                  n_kv=2, head_dim=64, weight_rows=None, device=gpu)
    mixed._weight_plans = large._weight_plans
    dw = w.to(gpu)
    prism_amd.packed_key_weights(q.to(gpu), kc.to(gpu), lse.to(gpu), dw, mixed, status=status)
    torch.cuda.synchronize()
    assert int(status) == prism_amd._lib.PKV_STATUS_BAD_PAGE
    assert read_status(gpu) == 0
