"""evict_keys on the device against a numpy restatement: everything it moves is moved bit for bit."""
import numpy as np
import pytest
import torch

import prism_amd
from oracle import behind as ob

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _pools(L, lens, P, nk, hd, seed, spare=3):
    rng = np.random.default_rng(seed)
    need = [-(-n // P) for n in lens]
    pages = sum(need) + spare
    ids = rng.permutation(pages)
    bt = np.full((len(lens), max(need + [1])), -1, np.int32)
    off = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[off:off + n]
        off += n
    k = rng.integers(-2 ** 15, 2 ** 15, size=(L, pages, P, nk, hd), dtype=np.int16)
    v = rng.integers(-2 ** 15, 2 ** 15, size=(L, pages, P, nk, hd), dtype=np.int16)
    w = (rng.exponential(size=(L, pages, nk, P)) ** 3).astype(np.float32)
    return k, v, w, bt


def _bf16(a, gpu):
    return torch.from_numpy(a).to(gpu).view(BF16)


def _run(gpu, k, v, w, bt, lens, keeps, first, recent, status=None):
    most = max([min(n, m) for n, m in zip(lens, keeps)] + [0])
    dk, dv, dw = _bf16(k, gpu), _bf16(v, gpu), torch.from_numpy(w).to(gpu)
    ints = [torch.from_numpy(np.asarray(a, np.int32)).to(gpu) for a in (bt, lens, keeps)]
    kept = prism_amd.evict_keys(dk, dv, dw, *ints, most, first=first, recent=recent, status=status)
    return dk.view(torch.int16).cpu().numpy(), dv.view(torch.int16).cpu().numpy(), dw.cpu().numpy(), kept.cpu().numpy()


def _same(got, want):
    for a, b, name in zip(got, want, ("K", "V", "weights", "kept")):
        assert a.shape == b.shape and a.dtype == b.dtype
        if a.dtype == np.float32:
            a, b = a.view(np.int32), b.view(np.int32)
        assert np.array_equal(a, b), f"{name}: {int((a != b).sum())} of {a.size} differ"


def _check(gpu, k, v, w, bt, lens, keeps, first, recent):
    most = max([min(n, m) for n, m in zip(lens, keeps)] + [0])
    want = ob.evict_np(k, v, w, bt, lens, keeps, first, recent, most)
    _same(_run(gpu, k, v, w, bt, lens, keeps, first, recent), want)


@pytest.mark.parametrize("L,nk,hd", [(1, 1, 64), (3, 2, 64), (2, 4, 128), (1, 8, 128), (1, 3, 64)])
@pytest.mark.parametrize("P", [16, 64, 256])
def test_evict(gpu, L, nk, hd, P):
    lens = [0, 1, 2, 63, 700, 1025, 2500, 300]
    keeps = [5, 1, 1, 40, 512, 1024, 300, 0]
    k, v, w, bt = _pools(L, lens, P, nk, hd, seed=P + nk)
    for first, recent in ((4, 64), (0, 0), (0, 1), (1000, 5), (3, 100000)):
        print("evict", L, nk, hd, P, first, recent, flush=True)
        _check(gpu, k, v, w, bt, lens, keeps, first, recent)


@pytest.mark.parametrize("lens,keeps", [([40000], [39999]), ([40000], [1]), ([33000, 9000], [4096, 8999]), ([20001], [10000])])
def test_long(gpu, lens, keeps):
    k, v, w, bt = _pools(1, lens, 64, 2, 64, seed=lens[0])
    _check(gpu, k, v, w, bt, lens, keeps, 4, 100)


@pytest.mark.parametrize("P", [16, 128])
@pytest.mark.parametrize("L,nk", [(1, 2), (8, 4)])
def test_short_tables(gpu, L, nk, P):
    """Up to 1024 tokens, and up to 4096 where the call has more than 256 heads."""
    for most in (1024, 4096):
        lens = [0, 1, 63, 64, 700, most, most - 1, most // 2 + 1, most - 130]
        keeps = [5, 1, 1, 40, 512, most // 2, most - 2, 3, most]
        k, v, w, bt = _pools(L, lens, P, nk, 64, seed=P + nk)
        assert bt.shape[1] * P == most
        w[:, :, 0] = np.round(w[:, :, 0])          # ties in one head of each layer
        w[:, :, 1, ::7] = -w[:, :, 1, ::7]         # negative ones, zeros of either sign and NaN in another
        w[:, 0, 1, 3] = np.nan
        for first, recent in ((4, 64), (0, 0), (3, 100000)):
            _check(gpu, k, v, w, bt, lens, keeps, first, recent)


def test_tables_wider_than_the_kernel_holds(gpu):
    """8200 columns, and a sequence that uses more than 8192 of them."""
    lens, keeps = [131200 - 5, 700], [9000, 300]
    k, v, w, bt = _pools(1, lens, 16, 1, 64, seed=8)
    assert bt.shape[1] > 8192
    _check(gpu, k, v, w, bt, lens, keeps, 4, 100)


def test_ties_and_odd_values(gpu):
    """Equal weights (zeros of both signs among them) go by age; NaN is above +inf, negative weights are below zero."""
    lens, keeps = [3000, 1500, 5000, 2000], [1000, 700, 4000, 900]
    k, v, w, bt = _pools(2, lens, 16, 2, 64, seed=1)
    rng = np.random.default_rng(2)
    w[0] = rng.integers(0, 3, size=w[0].shape)
    w[0][w[0] == 0] *= rng.choice([-1.0, 1.0], size=int((w[0] == 0).sum()))
    w[0][w[0] == 0] = np.where(rng.random(int((w[0] == 0).sum())) < 0.5, -0.0, 0.0)
    w[1] = rng.choice(np.array([np.nan, -np.nan, np.inf, -np.inf, -1.0, 1e-42, 0.0, 3.0e38], np.float32), size=w[1].shape)
    _check(gpu, k, v, w, bt, lens, keeps, 4, 64)
    w[:] = 0.0
    _check(gpu, k, v, w, bt, lens, keeps, 0, 0)


def test_strided_pools(gpu):
    """Layers and pages with space between them."""
    lens, keeps, L, P, nk, hd = [500, 90], [100, 80], 2, 16, 2, 64
    k, v, w, bt = _pools(L, lens, P, nk, hd, seed=5)
    want = ob.evict_np(k, v, w, bt, lens, keeps, 4, 16, 100)
    pages = k.shape[1]
    wide = torch.zeros(L, 2, pages, 3, P, nk, hd, dtype=torch.int16, device=gpu)
    wide[:, 0, :, 1] = torch.from_numpy(k).to(gpu)
    wide[:, 1, :, 1] = torch.from_numpy(v).to(gpu)
    before = wide.clone()
    ww = torch.full((L, pages, nk + 1, P), 5.0, device=gpu)
    ww[:, :, :nk] = torch.from_numpy(w).to(gpu)
    ints = [torch.from_numpy(np.asarray(a, np.int32)).to(gpu) for a in (bt, lens, keeps)]
    pools = wide.view(BF16)
    kept = prism_amd.evict_keys(pools[:, 0, :, 1], pools[:, 1, :, 1], ww[:, :, :nk], *ints, 100, first=4, recent=16)
    _same([x.cpu().numpy() for x in (wide[:, 0, :, 1], wide[:, 1, :, 1], ww[:, :, :nk], kept)], want)
    before[:, 0, :, 1], before[:, 1, :, 1] = wide[:, 0, :, 1], wide[:, 1, :, 1]
    assert torch.equal(before, wide) and (ww[:, :, nk] == 5.0).all()


def test_bad_pages_and_lengths_leave_the_sequence(gpu):
    lens, keeps = [500, 300, 200, 100, 90], [100, 50, 60, 30, 20]
    k, v, w, bt = _pools(1, lens, 16, 2, 64, seed=6)
    bt2, lens2, keeps2 = bt.copy(), list(lens), list(keeps)
    bt2[1, 3] = k.shape[1]
    bt2[2, 0] = -1
    lens2[3] = bt.shape[1] * 16 + 1
    keeps2[4] = -1
    status = torch.zeros(1, dtype=torch.int32, device=gpu)
    got = _run(gpu, k, v, w, bt2, lens2, keeps2, 4, 16, status=status)
    assert int(status) == prism_amd._lib.PKV_STATUS_BAD_PAGE
    want = ob.evict_np(k, v, w, bt[:1], lens[:1], keeps[:1], 4, 16, 100)
    _same(got[:3], want[:3])
    assert (got[3][:, 1:] == -1).all() and np.array_equal(got[3][:, :1], want[3])


def test_streams_and_graphs(gpu):
    lens, keeps = [800, 500], [300, 100]
    k, v, w, bt = _pools(2, lens, 16, 2, 64, seed=7)
    want = ob.evict_np(k, v, w, bt, lens, keeps, 4, 32, 300)
    ints = [torch.from_numpy(np.asarray(a, np.int32)).to(gpu) for a in (bt, lens, keeps)]
    fresh = [_bf16(k, gpu), _bf16(v, gpu), torch.from_numpy(w).to(gpu)]
    work = [x.clone() for x in fresh]
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        kept = prism_amd.evict_keys(*work, *ints, 300, first=4, recent=32)
    side.synchronize()
    out = lambda kept: [work[0].view(torch.int16).cpu().numpy(), work[1].view(torch.int16).cpu().numpy(),
                        work[2].cpu().numpy(), kept.cpu().numpy()]
    _same(out(kept), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = prism_amd.evict_keys(*work, *ints, 300, first=4, recent=32)
    for _ in range(3):
        for x, y in zip(work, fresh):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        _same(out(kept), want)
        prism_amd.evict_keys(*[x.clone() for x in fresh], *ints, 300, first=0, recent=0)
