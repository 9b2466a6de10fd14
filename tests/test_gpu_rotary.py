"""rotate_qk and packed_rope_append on the device, against fp64."""
import numpy as np
import pytest
import torch

import prism_amd
from oracle import packed as op
from prism_amd.attention import read_status

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _tol(ref, mag, dtype, norm):
    """One rounding to the output type (half a step: eps / 2 of the value, or half the smallest subnormal's step),
    and the fp32 arithmetic on the magnitudes that the element is made of: cos and sin rounded once (2^-24 each),
    two products and a sum (2^-24 each), and with the norm a sum of squares of up to 1024 terms and its tree, a
    reciprocal square root, a division and two products: 16 + 16 roundings in all, generously."""
    fi = torch.finfo(dtype)
    steps = 32 if norm else 16
    return ref.abs() * fi.eps / 2 + mag * steps * 2.0 ** -24 + fi.smallest_normal * fi.eps / 2


def _check(got, ref, mag, dtype, norm, what):
    err = (got.double().cpu() - ref).abs()
    bad = err > _tol(ref, mag, dtype, norm)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(err[bad].max()):.3g}"


def _tables(gpu, rd, n_pos, theta=1e4, scaling=None):
    freq, gain = prism_amd.epilogue._scaled_frequencies(rd, n_pos, theta, scaling)
    cos, sin = prism_amd.rotary_tables(rd, n_pos, theta, scaling=scaling, device=gpu)
    return freq, gain, cos, sin


@pytest.mark.parametrize("rd,n_pos,theta,scaling", [
    (128, 131072, 1e6, None), (2, 1, 1e4, None), (6, 77, 1e4, dict(rope_type="linear", factor=3.0)), (1024, 900, 5e5, None),
    (64, 40000, 1e4, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=8192)),
])
def test_rotary_tables_on_the_device(gpu, rd, n_pos, theta, scaling):
    """fp64 angles; cos and sin of the device's and the host's libraries are each within a few 2^-53 of the truth, and
    the rounding to fp32 is half a step of the value, 2^-24, of what is at most gain."""
    freq, gain, cos, sin = _tables(gpu, rd, n_pos, theta, scaling)
    angle = torch.arange(n_pos, dtype=torch.float64, device=gpu)[:, None] * freq.to(gpu)
    for got, want in ((cos, angle.cos() * gain), (sin, angle.sin() * gain)):
        assert got.shape == (n_pos, rd // 2) and got.dtype == torch.float32
        assert (got.double() - want).abs().max() <= gain * (2.0 ** -24 + 2.0 ** -45)
    f = torch.rand(rd // 2, generator=torch.Generator().manual_seed(1))
    c, s = prism_amd.rotary_tables(rd, 5, inv_freq=f.to(gpu), gain=0.5, device=gpu)
    a = torch.arange(5, dtype=torch.float64)[:, None] * f.double()
    assert (c.cpu().double() - a.cos() / 2).abs().max() <= 2.0 ** -24 and (s.cpu().double() - a.sin() / 2).abs().max() <= 2.0 ** -24


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("hd,rd", [(128, 128), (64, 64), (128, 32), (64, 16), (96, 96), (80, 48), (256, 64), (1024, 1024),
                                   (16, 16), (20, 10), (7, 6), (2, 2), (33, 32), (130, 2)])
@pytest.mark.parametrize("norm", [False, True])
def test_rotate_qk(gpu, dtype, inter, hd, rd, norm):
    g = torch.Generator().manual_seed(hd + rd)
    for tokens, nh, nk in [(1, 14, 2), (5, 3, 1), (67, 7, 5)]:
        q = torch.randn(tokens, nh, hd, generator=g).to(dtype)
        k = torch.randn(tokens, nk, hd, generator=g).to(dtype)
        wq, wk = ((1 + 0.2 * torch.randn(hd, generator=g)).to(dtype) if norm else None for _ in range(2))
        n_pos = 3000
        pos = torch.randint(0, n_pos, (tokens,), generator=g, dtype=torch.int32)
        freq, gain, cos, sin = _tables(gpu, rd, n_pos)
        dev = [t.to(gpu) if t is not None else None for t in (q, k, pos, wq, wk)]
        qo, ko = prism_amd.rotate_qk(*dev[:3], cos, sin, interleaved=inter, q_norm_w=dev[3], k_norm_w=dev[4])
        for got, x, w, name in ((qo, q, wq, "q"), (ko, k, wk, "k")):
            ref, mag = op.rotate64(x, pos, freq, gain=gain, interleaved=inter, norm_w=w)
            _check(got, ref, mag, dtype, norm, f"{name} {tokens} x {hd} / {rd}")


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("inter", [False, True])
def test_rotate_views_in_place_and_back(gpu, dtype, inter):
    g = torch.Generator().manual_seed(3)
    nh, nk, hd, rd, B, S = 6, 2, 64, 32, 3, 11
    qkv = torch.randn(B, S, (nh + 2 * nk) * hd, generator=g).to(dtype)
    pos = torch.randint(0, 500, (B, S), generator=g, dtype=torch.int32)
    freq, gain, cos, sin = _tables(gpu, rd, 500)
    x = qkv.to(gpu)
    q, k = x[..., :nh * hd].unflatten(2, (nh, hd)), x[..., nh * hd:(nh + nk) * hd].unflatten(2, (nk, hd))
    want, mag = op.rotate64(qkv.view(B * S, nh + 2 * nk, hd), pos.view(-1), freq, gain=gain, interleaved=inter)
    qo, ko = prism_amd.rotate_qk(q, k, pos.to(gpu), cos, sin, interleaved=inter)
    assert qo.shape == (B, S, nh, hd)
    _check(qo.view(B * S, nh, hd), want[:, :nh], mag[:, :nh], dtype, False, "views")
    # in place, q alone: k, v and nothing else changes
    got, none = prism_amd.rotate_qk(q, None, pos.to(gpu), cos, sin, interleaved=inter, q_out=q)
    assert none is None and got.data_ptr() == q.data_ptr() and torch.equal(q, qo)
    assert torch.equal(x[..., nh * hd:].cpu(), qkv[..., nh * hd:])
    prism_amd.rotate_qk(k, None, pos.to(gpu), cos, sin, interleaved=inter, q_out=k)
    assert torch.equal(k, ko)
    # turned back, by the rounded outputs: two roundings of a pair's magnitude
    back, _ = prism_amd.rotate_qk(q, None, pos.to(gpu), cos, -sin, interleaved=inter)
    err = (back.cpu().double() - qkv[..., :nh * hd].unflatten(2, (nh, hd)).double()).abs().view(B * S, nh, hd)
    assert (err <= mag[:, :nh] * (2 * torch.finfo(dtype).eps + 2.0 ** -19)).all()


def test_rotate_odd_addresses_and_strides(gpu):
    g = torch.Generator().manual_seed(4)
    tokens, nh, hd, rd = 9, 3, 32, 16
    buf = torch.randn(tokens, 131, generator=g).to(BF16)
    pos = torch.arange(tokens, dtype=torch.int32)
    freq, gain, cos, sin = _tables(gpu, rd, 16)
    for off in (0, 1, 8):
        q = buf.to(gpu)[:, off:off + nh * hd].unflatten(1, (nh, hd))   # rows 131 elements apart
        ref, mag = op.rotate64(buf[:, off:off + nh * hd].unflatten(1, (nh, hd)), pos, freq)
        qo, _ = prism_amd.rotate_qk(q, None, pos.to(gpu), cos, sin)
        _check(qo, ref, mag, BF16, False, f"offset {off}")
    # heads in front of tokens: any strides will do
    t = torch.randn(nh, tokens, hd, generator=g).to(BF16)
    ref, mag = op.rotate64(t.transpose(0, 1), pos, freq)
    qo, _ = prism_amd.rotate_qk(t.to(gpu).transpose(0, 1), None, pos.to(gpu), cos, sin)
    _check(qo, ref, mag, BF16, False, "heads first")


def test_rotate_far_positions_scaled(gpu):
    sc = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)
    freq, gain, cos, sin = _tables(gpu, 128, 131072, 1e6, sc)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(40, 4, 128, generator=g)
    pos = torch.randint(100000, 131072, (40,), generator=g, dtype=torch.int32)
    ref, mag = op.rotate64(q, pos, freq, gain=gain)
    got, _ = prism_amd.rotate_qk(q.to(gpu), None, pos.to(gpu), cos, sin)
    _check(got, ref, mag, FP32, False, "far")


def test_rotate_special_values(gpu):
    """Infinities and NaN stay in their pair; a head of zeros has a finite norm; no tokens is no work."""
    _, _, cos, sin = _tables(gpu, 64, 8)
    q = torch.ones(2, 2, 64, dtype=BF16, device=gpu)
    q[0, 0, 3], q[0, 1, 40] = float("inf"), float("nan")
    pos = torch.tensor([1, 2], dtype=torch.int32, device=gpu)
    out, _ = prism_amd.rotate_qk(q, None, pos, cos, sin)
    bad = ~torch.isfinite(out.cpu())
    want = torch.zeros_like(bad)
    want[0, 0, [3, 35]], want[0, 1, [8, 40]] = True, True
    assert torch.equal(bad, want)
    z, _ = prism_amd.rotate_qk(torch.zeros_like(q), None, pos, cos, sin, q_norm_w=torch.ones(64, dtype=BF16, device=gpu))
    assert torch.equal(z, torch.zeros_like(z))
    e, ek = prism_amd.rotate_qk(q[:0], q[:0], pos[:0], cos, sin)
    assert e.shape == ek.shape == (0, 2, 64)


def test_rotate_bad_positions_are_clamped_and_flagged(gpu):
    _, _, cos, sin = _tables(gpu, 64, 8)
    q = torch.randn(3, 2, 64, device=gpu).to(BF16)
    for hd_view in (q, q[..., :62]):   # the wide kernel and the other
        c, s = (cos, sin) if hd_view is q else prism_amd.rotary_tables(62, 8, device=gpu)
        pos = torch.tensor([-1, 3, 8], dtype=torch.int32, device=gpu)
        out, _ = prism_amd.rotate_qk(hd_view, None, pos, c, s)
        assert read_status(gpu) == prism_amd._lib.PKV_STATUS_BAD_POSITION
        ok, _ = prism_amd.rotate_qk(hd_view, None, pos.clamp(0, 7), c, s)
        assert torch.equal(out, ok) and read_status(gpu) == 0


def test_rotate_refusals(gpu):
    _, _, cos, sin = _tables(gpu, 64, 8)
    q = torch.zeros(3, 2, 64, dtype=BF16, device=gpu)
    pos = torch.zeros(3, dtype=torch.int32, device=gpu)
    w = torch.ones(64, dtype=BF16, device=gpu)
    big = torch.zeros(3, 2, 4, 64, dtype=BF16, device=gpu)
    for a, kw in [((q.double(), None, pos, cos, sin), {}), ((q, q.float(), pos, cos, sin), {}), ((q, q[:2], pos, cos, sin), {}),
                  ((q, None, pos.long(), cos, sin), {}), ((q, None, pos[:2], cos, sin), {}), ((q, None, pos.cpu(), cos, sin), {}),
                  ((q, None, pos, cos.bfloat16(), sin), {}), ((q, None, pos, cos[:4], sin), {}), ((q, None, pos, cos[:, ::2], sin), {}),
                  ((q[..., :62], None, pos, cos, sin), {}), ((q, None, pos, cos, sin), dict(q_norm_w=w.float())),
                  ((q, None, pos, cos, sin), dict(q_norm_w=w[:32])), ((q, None, pos, cos, sin), dict(k_norm_w=w)),
                  ((q, None, pos, cos, sin), dict(k_out=q)), ((q, None, pos, cos, sin), dict(q_out=q.float())),
                  ((q, None, pos, cos, sin), dict(q_out=q[:2])), ((q, None, pos, cos, sin), dict(eps=-1.0)),
                  ((q[0], None, pos, cos, sin), {}), ((q.transpose(1, 2), None, pos, cos[:, :1].contiguous(), sin[:, :1].contiguous()), {}),
                  ((big.transpose(0, 1), None, torch.zeros(6, dtype=torch.int32, device=gpu), cos, sin), {})]:
        with pytest.raises(RuntimeError):
            prism_amd.rotate_qk(*a, **kw)


def test_rotate_captured_and_on_another_stream(gpu):
    _, _, cos, sin = _tables(gpu, 128, 64)
    q, k = torch.randn(33, 4, 128, device=gpu).to(BF16), torch.randn(33, 2, 128, device=gpu).to(BF16)
    pos = torch.arange(33, dtype=torch.int32, device=gpu)
    want = prism_amd.rotate_qk(q, k, pos, cos, sin, interleaved=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = prism_amd.rotate_qk(q, k, pos, cos, sin, interleaved=True)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = prism_amd.rotate_qk(q, k, pos, cos, sin, interleaved=True)
    for i in range(3):
        q.normal_()
        pos.add_(i)
        graph.replay()
        want = prism_amd.rotate_qk(q, k, pos, cos, sin, interleaved=True)
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------------------------- append
def _case(new, ctx, P, nh, nk, hd, seed, extra=0):
    g = torch.Generator().manual_seed(seed)
    need = [-(-(n + c) // P) for n, c in zip(new, ctx)]
    ids = torch.randperm(sum(need) + 3, generator=g)
    bt = np.full((len(new), max(max(need), 1)), -1, np.int32)
    off = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[off:off + n].numpy()
        off += n
    pages = sum(need) + 3
    kc = torch.randn(pages, P, nk, hd, generator=g).to(BF16)
    vc = torch.randn(pages, P, nk, hd, generator=g).to(BF16)
    qkv = torch.randn(sum(new) + extra, (nh + 2 * nk) * hd, generator=g).to(BF16)
    return bt, kc, vc, qkv


@pytest.mark.parametrize("nh,nk,hd", [(28, 4, 128), (14, 2, 64), (7, 1, 128), (6, 3, 64)])
@pytest.mark.parametrize("P", [16, 64, 256])
@pytest.mark.parametrize("inter,rd_part,norm", [(False, 1, False), (True, 1, True), (False, 2, True), (True, 4, False)])
def test_append(gpu, nh, nk, hd, P, inter, rd_part, norm):
    new, ctx = [1, 37, 0, 1, 130, 3], [0, 15, 44, 255, 100, 1000]
    bt, kc, vc, qkv = _case(new, ctx, P, nh, nk, hd, seed=P + hd, extra=5)
    rd, total = hd // rd_part, sum(new)
    freq, gain, cos, sin = _tables(gpu, rd, 1100, scaling=dict(rope_type="yarn", factor=2.0,
                                                              original_max_position_embeddings=512))
    w = [(1 + 0.1 * torch.randn(hd, generator=torch.Generator().manual_seed(i))).to(BF16) if norm else None for i in (1, 2)]
    batch = prism_amd.PackedBatch(new, ctx, bt, page_size=P, num_pages=len(kc), n_heads=nh, n_kv=nk, head_dim=hd, device=gpu)
    dk, dv, x = kc.to(gpu), vc.to(gpu), qkv.to(gpu)
    q_out = torch.full((total + 5, nh, hd), 7.0, dtype=BF16, device=gpu)
    q = prism_amd.packed_rope_append(x, dk, dv, batch, cos, sin, interleaved=inter, q_out=q_out,
                                     q_norm_w=w[0].to(gpu) if norm else None, k_norm_w=w[1].to(gpu) if norm else None)
    assert q is q_out and (q[total:] == 7.0).all()
    pos, slots = batch.positions.cpu(), batch.slots.cpu().long()
    ref, mag = op.rotate64(qkv[:total, :nh * hd].unflatten(1, (nh, hd)), pos, freq, gain=gain, interleaved=inter, norm_w=w[0])
    _check(q[:total], ref, mag, BF16, norm, "q")
    ref, mag = op.rotate64(qkv[:total, nh * hd:(nh + nk) * hd].unflatten(1, (nk, hd)), pos, freq, gain=gain,
                           interleaved=inter, norm_w=w[1])
    got_k, got_v = dk.cpu().view(-1, nk, hd), dv.cpu().view(-1, nk, hd)
    _check(got_k[slots], ref, mag, BF16, norm, "k")
    assert torch.equal(got_v[slots], qkv[:total, (nh + nk) * hd:].unflatten(1, (nk, hd)))
    rest = torch.ones(len(got_k), dtype=torch.bool)
    rest[slots] = False
    assert torch.equal(got_k[rest], kc.view(-1, nk, hd)[rest]) and torch.equal(got_v[rest], vc.view(-1, nk, hd)[rest])
    # what rotate_qk gives for the same rows, bit for bit
    qr, kr = prism_amd.rotate_qk(x[:total, :nh * hd].unflatten(1, (nh, hd)), x[:total, nh * hd:(nh + nk) * hd].unflatten(1, (nk, hd)),
                                 batch.positions, cos, sin, interleaved=inter,
                                 q_norm_w=w[0].to(gpu) if norm else None, k_norm_w=w[1].to(gpu) if norm else None)
    assert torch.equal(qr, q[:total]) and torch.equal(kr.cpu(), got_k[slots])
    own = prism_amd.packed_rope_append(x, dk, dv, batch, cos, sin, interleaved=inter)
    assert own.shape == (total + 5, nh, hd) and not own[total:].any()


def test_append_other_positions_pool_views_and_bad_slots(gpu):
    nh, nk, hd, P = 4, 2, 64, 16
    new, ctx = [3, 2], [4, 30]
    bt, kc, vc, qkv = _case(new, ctx, P, nh, nk, hd, seed=1)
    freq, _, cos, sin = _tables(gpu, hd, 900)
    batch = prism_amd.PackedBatch(new, ctx, bt, page_size=P, num_pages=len(kc), n_heads=nh, n_kv=nk, head_dim=hd, device=gpu)
    # pages of a pool that holds K and V side by side: a page stride of its own
    pool = torch.stack([kc, vc], 1).to(gpu)
    pos = torch.tensor([800, 0, 5, 7, 899], dtype=torch.int32)
    q = prism_amd.packed_rope_append(qkv.to(gpu), pool[:, 0], pool[:, 1], batch, cos, sin, positions=pos.to(gpu))
    ref, mag = op.rotate64(qkv[:, :nh * hd].unflatten(1, (nh, hd)), pos, freq)
    _check(q, ref, mag, BF16, False, "q")
    ref, mag = op.rotate64(qkv[:, nh * hd:(nh + nk) * hd].unflatten(1, (nk, hd)), pos, freq)
    slots = batch.slots.cpu().long()
    _check(pool.cpu()[slots // P, 0, slots % P], ref, mag, BF16, False, "k")
    # a slot outside the pool is skipped and flagged
    before = pool.clone()
    good = batch.slots.clone()
    batch.slots[1], batch.slots[4] = -1, len(kc) * P
    prism_amd.packed_rope_append(qkv.to(gpu), pool[:, 0], pool[:, 1], batch, cos, sin, positions=pos.to(gpu))
    assert read_status(gpu) == prism_amd._lib.PKV_STATUS_BAD_PAGE
    assert torch.equal(pool, before)
    batch.slots.copy_(good)
    with pytest.raises(RuntimeError, match="positions"):
        prism_amd.packed_rope_append(qkv.to(gpu), pool[:, 0], pool[:, 1], batch, cos, sin, positions=pos[:3].to(gpu))
    with pytest.raises(RuntimeError, match="qkv"):
        prism_amd.packed_rope_append(qkv[:4].to(gpu), pool[:, 0], pool[:, 1], batch, cos, sin)
    with pytest.raises(RuntimeError, match="does not fit"):
        prism_amd.packed_rope_append(qkv.to(gpu), pool[:2, 0], pool[:2, 1], batch, cos, sin)
