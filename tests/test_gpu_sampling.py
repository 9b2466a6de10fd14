"""sample_tokens on the device against fp64."""
import numpy as np
import pytest
import torch

import prism_amd
from oracle import behind as ob

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _expect(x, u, t, k, p, m, got, logs, what):
    """Equal tokens.  The kernel's sums are within 2^-30 of the oracle's share (weights in fp64 or integers of 2^-42 of the
    largest, 2^20 of them at most): a number that lies nearer to a border than that decides nothing."""
    x, n = x.double().cpu().numpy(), len(u)
    per = lambda a: a.double().cpu().numpy() if torch.is_tensor(a) else np.full(n, np.float64(np.float32(a if a is not None else 0)))
    t, k, p, m = per(t), per(k), per(1.0 if p is None else p), per(m)
    u = u.double().cpu().numpy()
    got, logs = got.cpu().numpy(), None if logs is None else logs.double().cpu().numpy()
    for i in range(n):
        token, lp, near = ob.sample64(x[i], u[i], t[i], int(k[i]), p[i], m[i])
        if near < 2.0 ** -30:
            continue
        assert got[i] == token, f"{what} row {i}: {got[i]}, not {token} (t {t[i]} k {k[i]} p {p[i]} m {m[i]} u {u[i]})"
        if logs is not None:
            # the sum of the weights to 2^-30, the result rounded to fp32
            assert logs[i] == lp or abs(logs[i] - lp) <= 2.0 ** -29 + 2.0 ** -23 * abs(lp), f"{what} row {i}: {logs[i]} not {lp}"


def _draw(x, u, what, *, temperature=1.0, top_k=None, top_p=None, min_p=None):
    print(what, tuple(x.shape), x.dtype, flush=True)
    got, logs = prism_amd.sample_tokens(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                                        return_logprobs=True)
    _expect(x, u, temperature, top_k, top_p, min_p, got, logs, what)
    again = prism_amd.sample_tokens(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert torch.equal(again, got), f"{what}: another token with the same number"
    return got


def _logits(gpu, rows, vocab, dtype, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * spread
    for i in range(rows):
        at = torch.randperm(vocab, generator=g)[:min(30, vocab)]
        x[i, at] = 4 + torch.rand(len(at), generator=g) * 8
    return x.to(dtype).to(gpu), torch.rand(rows, generator=g).to(gpu)


RULES = {
    "plain": dict(),
    "cool": dict(temperature=0.6),
    "greedy": dict(temperature=0.0),
    "k": dict(top_k=50),
    "k1": dict(top_k=1),
    "p": dict(top_p=0.9),
    "m": dict(min_p=0.05),
    "kp": dict(temperature=0.8, top_k=40, top_p=0.95),
    "kpm": dict(temperature=1.2, top_k=400, top_p=0.9, min_p=0.02),
    "pm": dict(top_p=0.99, min_p=0.001),
    "wide k": dict(top_k=900, temperature=3.0),
    "wide p": dict(top_p=0.999, temperature=4.0),
    "wide m": dict(min_p=1e-4, temperature=2.0),
    "narrow": dict(top_p=1e-6),
    "first": dict(top_p=0.0),
    "top only": dict(min_p=1.0),
}


@pytest.mark.parametrize("rules", list(RULES))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [1, 2, 17, 1000, 4096, 32000, 151003])
def test_rules(gpu, rules, dtype, vocab):
    rows = 3 if vocab > 100000 else 12
    x, u = _logits(gpu, rows, vocab, dtype, seed=vocab)
    _draw(x, u, f"{rules} {vocab}", **RULES[rules])


@pytest.mark.parametrize("rules", ["plain", "kp", "p", "wide p", "wide k", "m"])
def test_flat_rows(gpu, rules):
    """Nothing stands out: what stays are tens of thousands of tokens, far more than the lists hold; all equal, the cut
    is among equals."""
    for dtype, vocab in ((torch.float32, 100003), (torch.bfloat16, 50000)):
        x, u = _logits(gpu, 4, vocab, dtype, seed=9, spread=0.3)
        x[:] = x.clamp(max=1.0)
        x[1] = 0.25
        x[2] = torch.where(x[2] > 0, 1.0, -1.0).to(dtype)
        for more in (dict(), dict(top_k=30000), dict(top_p=0.7), dict(top_k=20000, top_p=0.5, min_p=0.1)):
            _draw(x, u, f"flat {rules}", **{**RULES[rules], **more})


def test_masked_rows(gpu):
    """-inf, NaN and the type's lowest value as masks; rows with one token left, or none; +inf."""
    for dtype in DTYPES:
        x, u = _logits(gpu, 9, 9001, dtype, seed=3)
        x[0] = -float("inf")
        x[1] = float("nan")
        x[2, :] = -float("inf")
        x[2, 8999] = -3.0
        x[3, 100:] = float("nan")
        x[4, ::2] = torch.finfo(dtype).min
        x[5, 1:] = torch.finfo(dtype).min
        x[6, [5, 4097, 9000]] = float("inf")
        x[7, 4000:] = -float("inf")
        x[8] = torch.finfo(dtype).min
        for name, rules in RULES.items():
            got = _draw(x, u, f"masked {name}", **rules)
            assert got[0] == -1 and got[1] == -1 and got[2] == 8999
            assert int(got[6]) in (5, 4097, 9000)


def test_ties_go_to_the_lowest_token(gpu):
    x = torch.zeros(6, 20000, device=gpu)
    u = torch.tensor([0.0, 0.999999, 0.5, 0.3, 0.0, 1.0], device=gpu)
    assert _draw(x, u, "ties", temperature=0.0).tolist() == [0] * 6
    got = _draw(x, u, "ties", top_k=10)
    assert got.tolist() == [0, 9, 5, 3, 0, 9]
    x[:, 7000:7005] = 1.0
    assert _draw(x, u, "ties", top_k=2).tolist() == [7000, 7001, 7001, 7000, 7000, 7001]
    assert _draw(x, u, "ties", temperature=0.0).tolist() == [7000] * 6
    _draw(x, u, "ties", top_p=0.3)


def test_numbers_at_the_ends(gpu):
    x, _ = _logits(gpu, 6, 5000, torch.float32, seed=4)
    u = torch.tensor([0.0, 1.0, 1.0 - 2.0 ** -24, 2.0 ** -24, -3.0, 7.0], device=gpu)
    for name in ("plain", "k", "p", "kpm", "wide p"):
        _draw(x, u, f"ends {name}", **RULES[name])
    # the last tokens have no weight at all: 1.0 does not reach them
    x[:, 4000:] = -1e6
    got = _draw(x, u, "ends", temperature=0.5)
    assert int(got.max()) < 4000
    assert prism_amd.sample_tokens(x, u * float("nan")).tolist() == prism_amd.sample_tokens(x, u * 0).tolist()


def test_settings_of_each_row(gpu):
    rows = 40
    rng = np.random.default_rng(6)
    x, u = _logits(gpu, rows, 33001, torch.float32, seed=6)
    t = torch.from_numpy(rng.choice([0.0, 0.5, 1.0, 2.0, -1.0], rows).astype(np.float32)).to(gpu)
    k = torch.from_numpy(rng.choice([0, -5, 1, 30, 700, 33000, 33001, 10 ** 9], rows).astype(np.int32)).to(gpu)
    p = torch.from_numpy(rng.choice([0.0, 0.5, 0.95, 1.0, 2.0], rows).astype(np.float32)).to(gpu)
    m = torch.from_numpy(rng.choice([0.0, -1.0, 0.01, 0.3, 5.0], rows).astype(np.float32)).to(gpu)
    _draw(x, u, "rows", temperature=t, top_k=k, top_p=p, min_p=m)
    _draw(x, u, "rows", temperature=0.7, top_k=k, top_p=0.9, min_p=m)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab", [1500, 9000, 40000, 120001])
def test_hundreds_of_tokens_stay(gpu, dtype, vocab):
    """top-k whose last token lies in a class of values with many others, equal ones among them."""
    x, u = _logits(gpu, 6, vocab, dtype, seed=vocab)
    x[4] = (x[4].float() * 2).round().to(dtype) / 2
    x[5, 10:] = x[5, 10]
    for k in (513, 700, 900, 1023, 1024, 1400):
        _draw(x, u, f"top-k {k} of {vocab}", top_k=k)
        _draw(x, u, f"top-k {k} of {vocab}, with top-p", top_k=k, top_p=0.97, temperature=1.5)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("vocab,top_k", [(40009, 300), (60000, 700), (60000, 1000), (128000, 600)])
def test_long_lists_of_many_rows_are_thinned(gpu, dtype, vocab, top_k):
    """Rows whose lists hold more than 1024 tokens together, as many at a time as the device runs: every row goes the
    same way through the lists, whichever of its waves comes late."""
    x, u = _logits(gpu, 16, vocab, dtype, seed=vocab + top_k)
    got = _draw(x, u, f"thinned {top_k} of {vocab}", top_k=top_k, temperature=1.3)
    logs = prism_amd.sample_tokens(x, u, top_k=top_k, temperature=1.3, return_logprobs=True)[1]
    wide, many = x.repeat(32, 1), u.repeat(32)
    for _ in range(3):
        more, more_logs = prism_amd.sample_tokens(wide, many, top_k=top_k, temperature=1.3, return_logprobs=True)
        assert torch.equal(more, got.repeat(32)) and torch.equal(more_logs, logs.repeat(32))


def _expect_any(x, t, k, p, m, got, logs, what):
    """What holds for a row wherever its number lies: the token is one of those that stay, and the logarithm its own
    share, to _expect's tolerance.  Borders of top-p and min-p that lie nearer than 2^-30 may fall either way: the set
    and its sum lie between those of rules a little tighter and a little looser."""
    for i in range(len(got)):
        row, slack = x[i].double().cpu().numpy(), 2.0 ** -29
        loose, w, _ = ob.kept64(row, t, k, p * (1 + slack) if 0 < p < 1 else p, m * (1 - slack))
        _, tight, _ = ob.kept64(row, t, k, p * (1 - slack) if 0 < p < 1 else p, min(m, 1.0) * (1 + slack) if m < 1 else m)
        if len(loose) == 0:
            assert got[i] == -1 and logs[i] == -float("inf"), what
            continue
        at = np.flatnonzero(loose == int(got[i]))
        assert len(at) == 1 and w[at[0]] > 0, f"{what} row {i}: {got[i]} does not stay"
        lo, hi = np.log(w[at[0]] / w.sum()), np.log(w[at[0]] / tight.sum())
        assert lo - 2.0 ** -29 - 2.0 ** -23 * abs(lo) <= logs[i] <= hi + 2.0 ** -29 + 2.0 ** -23 * abs(hi), f"{what} row {i}"


@pytest.mark.parametrize("rules", list(RULES))
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_no_row_goes_unlooked_at(gpu, rules, dtype):
    """Ordinary rows with ordinary numbers are all far enough from a border to be compared with the oracle's tokens; rows
    whose numbers lie on borders (equal logits, 0 and 1) still get a token that stays, and its share."""
    r = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)
    r.update(RULES[rules])
    for vocab in (1000, 20000):
        x, u = _logits(gpu, 12, vocab, dtype, seed=vocab + 1)
        rule = [float(np.float32(r["temperature"])), r["top_k"], float(np.float32(r["top_p"])), float(np.float32(r["min_p"]))]
        near = [ob.sample64(x[i].double().cpu().numpy(), float(u[i]), *rule)[2] for i in range(12)]
        assert min(near) >= 2.0 ** -30, f"{rules} {vocab}: a row of this case decides nothing"
        ties = x.clone()
        ties[:4] = 0.5
        ties[4:8] = (x[4:8].float() / 4).round().to(dtype)
        ends = torch.tensor([0.0, 0.25, 0.5, 1.0] * 3, device=gpu)
        for what, a, b in (("rows", x, u), ("ties", ties, u), ("ties and ends", ties, ends), ("ends", x, ends)):
            got, logs = prism_amd.sample_tokens(a, b, temperature=r["temperature"], top_k=r["top_k"], top_p=r["top_p"],
                                                min_p=r["min_p"], return_logprobs=True)
            _expect_any(a, *rule, got.cpu().numpy(), logs.double().cpu().numpy(), f"{rules} {vocab} {what}")


def test_settings_of_rows_that_are_no_number(gpu):
    """NaN: no rule, and the largest logit as a temperature."""
    x, u = _logits(gpu, 4, 9001, torch.float32, seed=17)
    nan, one = torch.full((4,), float("nan"), device=gpu), torch.full((4,), 1.0, device=gpu)
    want = prism_amd.sample_tokens(x, u)
    assert torch.equal(prism_amd.sample_tokens(x, u, top_p=nan), want)
    assert torch.equal(prism_amd.sample_tokens(x, u, min_p=nan), want)
    assert torch.equal(prism_amd.sample_tokens(x, u, top_p=0.5 * one, min_p=nan), prism_amd.sample_tokens(x, u, top_p=0.5))
    assert torch.equal(prism_amd.sample_tokens(x, u, top_k=40, min_p=nan), prism_amd.sample_tokens(x, u, top_k=40))
    assert torch.equal(prism_amd.sample_tokens(x, u, temperature=nan), x.argmax(1))


def test_extreme_temperatures(gpu):
    x, u = _logits(gpu, 5, 3001, torch.float32, seed=11)
    x[4, :5] = torch.tensor([3e38, 3e38, 2.9e38, -3e38, 0.0])
    for t in (1e-45, 1e-30, 1e-3, 1e3, 1e30, float("inf")):
        for more in (dict(), dict(top_k=20), dict(top_p=0.5), dict(min_p=0.1)):
            _draw(x, u, f"t {t}", temperature=t, **more)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_strided_rows_at_any_alignment(gpu, dtype):
    wide, u = _logits(gpu, 5, 10007, dtype, seed=12)
    for off, n in ((0, 10007), (1, 10006), (3, 9999), (7, 1), (5, 4097), (2, 31)):
        x = wide[:, off:off + n]
        for name in ("plain", "kp", "p", "greedy", "wide p"):
            _draw(x, u, f"offset {off} {name}", **RULES[name])


@pytest.mark.parametrize("vocab", [262145, 999999, 1000000])
def test_large_vocabularies(gpu, vocab):
    x, u = _logits(gpu, 2, vocab, torch.bfloat16, seed=13)
    for name in ("plain", "kp", "p", "wide p", "greedy"):
        _draw(x, u, f"large {name}", **RULES[name])


def test_many_rows_and_none(gpu):
    x, u = _logits(gpu, 700, 999, torch.float32, seed=14)
    _draw(x, u, "many", top_k=20, top_p=0.9)
    _draw(x, u, "many")
    empty = prism_amd.sample_tokens(x[:0], u[:0])
    assert empty.shape == (0,) and empty.dtype == torch.int64


def test_the_draws_follow_the_distribution(gpu):
    """Numbers on a fine grid: each token is drawn as often as its share says, to one grid step at either end."""
    n = 20000
    x = torch.tensor([0.5, -1.0, 2.0, -float("inf"), 1.0, 1.9, -4.0], device=gpu).expand(n, 7).contiguous()
    u = (torch.arange(n, device=gpu) + 0.5) / n
    got = prism_amd.sample_tokens(x, u, temperature=0.7, top_k=4)
    share = torch.zeros(7, dtype=torch.float64)
    kept = torch.tensor([0, 2, 4, 5])
    share[kept] = torch.softmax(x[0, kept.to(gpu)].double().cpu() / float(np.float32(0.7)), 0)
    count = torch.bincount(got.cpu(), minlength=7).double()
    assert (count - share * n).abs().max() <= 2.0


def test_streams_and_graphs(gpu):
    x, u = _logits(gpu, 16, 40001, torch.bfloat16, seed=15)
    eager = prism_amd.sample_tokens(x, u, top_p=0.9)
    side = torch.cuda.Stream(gpu)
    side.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(side):
        other = prism_amd.sample_tokens(x, u, top_p=0.9)
    side.synchronize()
    assert torch.equal(eager, other)
    graph, v = torch.cuda.CUDAGraph(), u.clone()
    with torch.cuda.graph(graph):
        tokens, logs = prism_amd.sample_tokens(x, v, top_p=0.9, return_logprobs=True)
    for i in range(4):
        v.copy_((u + 0.17 * i) % 1.0)
        graph.replay()
        torch.cuda.synchronize()
        want, want_logs = prism_amd.sample_tokens(x, v, top_p=0.9, return_logprobs=True)
        assert torch.equal(tokens, want) and torch.equal(logs, want_logs)
