"""Sampling of a batch of rows with settings of their own, against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from inferi_b200.ops import BatchSampler, InferiError, Sampler

pytestmark = pytest.mark.gpu


def choose(x, T, k, top_p, min_p, coin):
    """(token, probability) of one row, in 64 bits (weights exact to 2^-52 here, to 2^-31 in the kernel: a border would have to be that near to a coin)."""
    x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
    if not T > 0 or x.max() == -np.inf:
        return int(np.argmax(x)), 1.0
    with np.errstate(over="ignore", under="ignore"):
        w = np.exp((x - x.max()) / float(np.float32(T)))
    n = len(x)
    by_k, by_p, by_min = 0 < k < n, 0 < top_p < 1, min_p > 0
    order = np.lexsort((np.arange(n), -x)) if by_k or by_p or by_min else np.arange(n)
    w = w[order]
    m = k if by_k else n
    sums = np.cumsum(w)
    if by_min:
        least = max(1, int((w >= float(np.float32(min_p))).sum()))
    if by_p:
        m = min(m, int((sums[:m] <= float(np.float32(top_p)) * sums[m - 1]).sum()) + 1)
    if by_min:
        m = min(m, least)
    at = min(int((sums[:m] <= float(np.float32(coin)) * sums[m - 1]).sum()), m - 1)
    return int(order[at]), float(w[at] / sums[m - 1])


def run(backend, logits, T, k, top_p, min_p, coin):
    """Lists, or None where no row has that limit."""
    f = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32, device="cuda")   # noqa: E731
    n = logits.shape[0]
    token, prob = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.full((n,), -7.0, device="cuda")
    BatchSampler(backend, logits.shape[1]).sample(logits, f(T), None if k is None else torch.tensor(k, dtype=torch.int32, device="cuda"), f(top_p), f(min_p), f(coin), token, prob)
    return token.tolist(), prob.tolist()


def check(backend, logits, T, k, top_p, min_p, coin):
    tokens, probs = run(backend, logits, T, k, top_p, min_p, coin)
    x = logits.cpu().numpy()
    for r in range(len(tokens)):
        want, p = choose(x[r], T[r], k[r] if k else 0, top_p[r] if top_p else 1.0, min_p[r] if min_p else 0.0, coin[r])
        assert tokens[r] == want, f"row {r}: token {tokens[r]} instead of {want} (T {T[r]}, k {k and k[r]}, top_p {top_p and top_p[r]}, min_p {min_p and min_p[r]}, coin {coin[r]})"
        # a weight and a sum, each to 2^-31 and 2^-44 of the largest weight per token, rounded to 32 bits
        assert abs(probs[r] - p) <= p * (2**-24 + 2**-29) + x.shape[1] * 2**-44, (r, probs[r], p)


def settings(n, seed):
    rng = np.random.default_rng(seed)
    pick = np.arange(n) % 8
    T = (0.3 + 1.4 * rng.random(n)).astype(np.float32).tolist()
    k = np.where(pick & 1, rng.integers(1, 300, n), 0).tolist()
    top_p = np.where(pick & 2, 0.3 + 0.69 * rng.random(n), 1.0).tolist()
    min_p = np.where(pick & 4, 0.3 * rng.random(n) ** 2, 0.0).tolist()
    return T, k, top_p, min_p, rng.random(n).astype(np.float32).clip(max=1 - 2**-24).tolist()


@pytest.mark.parametrize("sharp", [0.01, 0.7, 3.0, 30.0])
@pytest.mark.parametrize("vocab", [1, 2, 31, 512, 1000, 4096, 4097, 32003, 128256])
def test_against_the_definition(backend, vocab, sharp):
    n = 24
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn(n, vocab, generator=g, device="cuda") * sharp
    check(backend, logits, *settings(n, vocab))
    if vocab > 100:   # one filter alone, and none
        T, k, top_p, min_p, coin = settings(n, vocab + 1)
        for use in (0, 1, 2, 3):
            check(backend, logits, T, [5] * n if use == 1 else None, [0.9] * n if use == 2 else None, [0.02] * n if use == 3 else None, coin)


@pytest.mark.parametrize("vocab", [371000, 524288])
def test_vocabularies_that_shared_memory_does_not_hold(backend, vocab):
    logits = torch.randn(8, vocab, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 2
    check(backend, logits, *settings(8, 3))


@pytest.mark.parametrize("vocab", [50, 5000, 40000])
def test_ties(backend, vocab):
    """Equal logits: weights are equal, and index order decides.  Rows of one value, of two, of a few; a largest one that many tokens share."""
    rng = np.random.default_rng(vocab)
    rows = [np.zeros(vocab), np.where(np.arange(vocab) % 3 == 0, 1.0, 0.0), rng.integers(0, 4, vocab).astype(float), np.where(rng.random(vocab) < 0.5, 2.0, -np.inf),
            np.where(np.arange(vocab) >= vocab - 3, 0.0, -40.0)]
    logits = torch.tensor(np.stack(rows * 8), dtype=torch.float32, device="cuda")
    n = logits.shape[0]
    T, k, top_p, min_p, coin = settings(n, 7)
    pick = np.arange(n) // 5   # every kind of row with every combination of limits
    k, top_p, min_p = [np.where(pick & b, on, off).tolist() for b, on, off in ((1, vocab // 3 + 1, 0), (2, 0.6, 1.0), (4, 0.5, 0.0))]
    check(backend, logits, T, k, top_p, min_p, coin)
    check(backend, logits, [1.0] * n, [1] * n, None, None, coin)          # the first of the largest
    check(backend, logits, [1.0] * n, None, None, [1.0] * n, coin)        # all of the largest
    check(backend, logits, [1.0] * n, None, None, [1.5] * n, coin)        # the first alone
    check(backend, logits, [1.0] * n, [vocab - 1] * n, None, None, coin)


def test_coins_at_the_ends(backend):
    """Coin 0 is the first token that can come, a coin just below 1 the last one that is left."""
    logits = torch.tensor([[-math.inf, 0.0, -1.0, -math.inf, -50.0, -math.inf]] * 4, device="cuda")
    for coin, index, ranked in ((0.0, 1, 1), (1 - 2**-24, 2, 2)):
        tokens, _ = run(backend, logits, [1.0] * 4, [0, 2, 0, 0], [1.0, 1.0, 0.99, 1.0], [0.0, 0.0, 0.0, 0.1], [coin] * 4)
        assert tokens == [index, ranked, ranked, ranked]


def test_limits_that_are_none(backend):
    logits = torch.randn(8, 3000, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    coin = [0.1, 0.5, 0.9, 0.99, 0.3, 0.7, 0.2, 0.05]
    want = run(backend, logits, [0.8] * 8, None, None, None, coin)
    nan, inf = float("nan"), float("inf")
    assert run(backend, logits, [0.8] * 8, [0, -1, 3000, 3001, 2**31 - 1, -2**31, 0, 0], [1.0, 0.0, -1.0, nan, 2.0, inf, -inf, 1.0], [0.0, -1.0, nan, -inf, 0.0, -0.0, nan, 0.0], coin) == want
    # a row with a limit that keeps all of it, in the order of probabilities
    check(backend, logits, [0.8] * 8, [2999] * 8, [1 - 2**-24] * 8, [1e-30] * 8, coin)


def test_temperatures(backend):
    logits = torch.randn(9, 5000, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * 3
    logits[:, 77] = logits[:, 4000] = logits.max() + 1
    T = [0.0, -1.0, float("nan"), -float("inf"), 1e-6, 1e-30, 100.0, 1e6, 1e-2]
    tokens, probs = run(backend, logits, T, [0] * 9, [0.9] * 9, [0.0] * 9, [0.75] * 9)
    assert tokens[:4] == [77] * 4 and probs[:4] == [1.0] * 4
    assert tokens[4:6] == [4000] * 2 and probs[4:6] == [0.5] * 2    # two largest ones share everything
    check(backend, logits[6:], T[6:], None, [0.9] * 3, None, [0.75] * 3)
    check(backend, logits[6:], T[6:], None, None, None, [0.75] * 3)


def test_logits_that_are_no_numbers(backend):
    x = torch.randn(6, 700, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    x[0] = float("nan")
    x[1] = -math.inf
    x[2, ::2] = float("nan")
    x[3, 50] = x[3, 60] = math.inf
    x[4, 1:] = -math.inf
    x[5] = torch.finfo(torch.float32).min
    x[5, 9] = torch.finfo(torch.float32).max
    coin = [0.6] * 6
    for limits in ((None, None, None), ([3] * 6, [0.9] * 6, [0.1] * 6)):
        check(backend, x, [1.0] * 6, *limits, coin)
    assert run(backend, x, [0.0] * 6, None, None, None, coin)[0] == [0, 0, int(torch.where(x[2].isnan(), -math.inf, x[2]).argmax()), 50, 0, 9]


def test_agrees_with_the_sampler_of_one_row(backend):
    """Temperature and top-p are what `Sampler` makes of them (32-bit probabilities there: coins are kept away from borders)."""
    logits = torch.randn(1, 8000, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda") * 4
    for T, top_p in ((0.9, 0.8), (0.7, 1.0), (1.3, 0.95)):
        x = logits[0].double().cpu().numpy()
        w = np.exp((x - x.max()) / float(np.float32(T)))
        order = np.argsort(-x, kind="stable") if top_p < 1 else np.arange(8000)
        w = w[order]
        m = int((np.cumsum(w) <= top_p * w.sum()).sum()) + 1 if top_p < 1 else 8000
        sums = np.cumsum(w[:m]) / w[:m].sum()
        for at in np.argsort(-w[:m])[:6]:
            coin = float(np.float32(sums[at] - w[at] / w[:m].sum() / 2))
            one = Sampler(backend, 8000, T, top_p).sample(logits[0], coin).item()
            assert run(backend, logits, [T], None, [top_p], None, [coin])[0] == [one] == [order[at]]


def test_strided_rows_and_no_probabilities(backend):
    store = torch.randn(5, 1300, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")
    for cut in (store[:, :1000], store[:, 3:1004], store[1:2, 7:900]):
        n = cut.shape[0]
        T, coin = torch.full((n,), 0.9, device="cuda"), torch.full((n,), 0.4, device="cuda")
        k = torch.full((n,), 20, dtype=torch.int32, device="cuda")
        s = BatchSampler(backend, cut.shape[1])
        got = s.sample(cut, T, k, None, None, coin)
        assert got.dtype == torch.int32 and torch.equal(got, s.sample(cut.contiguous(), T, k, None, None, coin, torch.empty_like(got), torch.empty_like(T)))
        check(backend, cut, [0.9] * n, [20] * n, None, None, [0.4] * n)


def test_many_rows_captured(backend):
    n, vocab = 700, 9000
    logits = torch.randn(n, vocab, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda") * 3
    T, k, top_p, min_p, coin = settings(n, 8)
    check(backend, logits, T, k, top_p, min_p, coin)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")   # noqa: E731
    args = (f(T), torch.tensor(k, dtype=torch.int32, device="cuda"), f(top_p), f(min_p), f(coin))
    token = torch.empty(n, dtype=torch.int32, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        BatchSampler(backend, vocab).sample(logits, *args, token)
    args[-1].copy_(f(coin[::-1]))
    graph.replay()
    torch.cuda.synchronize()
    assert token.tolist() == run(backend, logits, T, k, top_p, min_p, coin[::-1])[0]


def test_no_rows(backend):
    e, before = torch.zeros(0, device="cuda"), backend.launch_count()
    assert BatchSampler(backend, 100).sample(torch.zeros(0, 100, device="cuda"), e, None, None, None, e).numel() == 0
    assert backend.launch_count() == before


def test_refusals(backend):
    x, one, i = torch.zeros(3, 100, device="cuda"), torch.zeros(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")

    def refused(message, vocab=100, x=x, T=one, k=i, p=one, m=one, coin=one, token=i, prob=one):
        with pytest.raises(InferiError, match=message):
            BatchSampler(backend, vocab).sample(x, T, k, p, m, coin, token, prob)

    refused("logits: expected", vocab=101)
    refused("logits: expected", x=x.half())
    refused("logits: expected", x=torch.zeros(3, 200, device="cuda")[:, ::2])
    refused("temperature", T=one[:2])
    refused("top_k", k=one)
    refused("top_p", p=one.double())
    refused("min_p", m=torch.zeros(6, device="cuda")[::2])
    refused("coin", coin=i)
    refused("token", token=i.long())
    refused("prob", prob=i)
    refused("on device", coin=one.cpu())
    refused("524289 tokens", vocab=524289, x=torch.zeros(3, 524289, device="cuda"))
    refused("0 tokens", vocab=0, x=torch.zeros(3, 0, device="cuda"))
    assert backend.lib.ib_sample_batch(backend.handle, None, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [70, 5000, 150000])
def test_zeros_of_either_sign_are_ties(backend, vocab):
    """-0 and 0 are the same logit: the lower index first, whatever the sign."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = -1.0 - torch.rand(8, vocab, generator=g, device="cuda")
    at = torch.randperm(vocab, generator=g, device="cuda")[:60]
    logits[:, at] = torch.where(torch.rand(8, 60, generator=g, device="cuda") < 0.5, -0.0, 0.0)
    coin = [0.0, 0.1, 0.25, 0.5, 0.75, 0.9, 0.99, 0.3]
    check(backend, logits, [0.1] * 8, [20] * 8, [0.9] * 8, None, coin)
    check(backend, logits, [0.1] * 8, [0] * 8, [0.5] * 8, [0.2] * 8, coin)
    tokens, _ = run(backend, logits, [0.0] * 8, None, None, None, coin)
    assert tokens == [int(at.min())] * 8


@pytest.mark.gpu
@pytest.mark.parametrize("rows, vocab", [(80, 128256), (160, 70000), (300, 33000)])
def test_many_rows_whose_histogram_reaches_as_far_as_a_sample_says(backend, rows, vocab):
    """Peaked and flat rows side by side: a few large logits that a sample misses, or finds; a border far behind them."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * torch.linspace(0.1, 4.0, rows, device="cuda")[:, None]
    top = torch.randint(0, vocab, (rows, 3), generator=g, device="cuda")
    logits.scatter_(1, top, torch.rand(rows, 3, generator=g, device="cuda") * 30)
    logits[: rows // 8, :4096] -= 20.0
    rng = np.random.default_rng(rows)
    T = (0.4 + rng.random(rows)).astype(np.float32).tolist()
    top_p = np.where(np.arange(rows) % 3 == 0, 0.9999, 0.5 + 0.49 * rng.random(rows)).astype(np.float32).tolist()
    coin = rng.random(rows).astype(np.float32).tolist()
    check(backend, logits, T, None, top_p, None, coin)
    check(backend, logits, T, np.where(np.arange(rows) % 2, rng.integers(1, 5000, rows), 0).tolist(), top_p, [1e-6] * rows, coin)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, vocab", [(200, 45000), (80, 128256)])
def test_odd_rows_among_many(backend, rows, vocab):
    """Rows of one value, of two, with one number only, with none, with infinities and NaN; temperatures from nothing to a million; limits at their ends - where a slice is large enough for
    a sample to say how far the histogram goes."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = torch.randn(rows, vocab, generator=g, device="cuda") * 2
    logits[0] = 3.0
    logits[1] = torch.where(torch.rand(vocab, generator=g, device="cuda") < 0.5, 1.0, -1.0)
    logits[2] = -math.inf
    logits[2, vocab - 3] = -5.0
    logits[3] = math.nan
    logits[4, ::3] = math.nan
    logits[5, 100:107] = math.inf
    logits[6] = torch.linspace(-1e30, 1e30, vocab, device="cuda")
    logits[7] = logits[7].round()
    logits[8, : vocab // 2] = -math.inf
    logits[9] = 1000.0 + logits[9] * 1e-3
    logits[10] = logits[10] * 1e-6
    logits[11, ::31] = 9.0    # (whatever a sample finds, or misses)
    logits[12, 5:13] = 30.0
    rng = np.random.default_rng(vocab)
    kinds = 20
    T = np.tile(np.array([1.0, 0.7, 1e-6, 1e6, 1e-30, 30.0, 0.9, 1.0], dtype=np.float32), rows)[:rows]
    T[:16] = 1.0
    coin = rng.random(rows).astype(np.float32)
    coin[::17], coin[5::17] = 0.0, np.float32(1 - 2**-24)
    for top_k, top_p, min_p in ((None, [0.9] * rows, None), ([1, 2, 50, vocab - 1, vocab, 0, 3000, 40000][:8] * (rows // 8), None, None),
                                (None, [1e-6, 1 - 2**-24, 0.5, 0.9999] * (rows // 4), [0.0, 1e-30, 0.5, 1.0] * (rows // 4)), ([200, 0] * (rows // 2), [0.8, 0.99] * (rows // 2), None)):
        tokens, probs = run(backend, logits, T.tolist(), top_k, top_p, min_p, coin.tolist())
        x = logits.cpu().numpy()
        for r in list(range(kinds)) + list(range(kinds, rows, 7)):
            want, p = choose(x[r], float(T[r]), top_k[r] if top_k else 0, top_p[r] if top_p else 1.0, min_p[r] if min_p else 0.0, coin[r])
            assert tokens[r] == want, (r, tokens[r], want)
            assert abs(probs[r] - p) <= p * (2**-24 + 2**-29) + vocab * 2**-44, (r, probs[r], p)


def tails(vocab, rows, seed):
    """Rows whose largest logits stand before a tail of equal values, or of few different ones, which has a part of the mass that is not small: what each of its weights is off by adds up."""
    rng = np.random.default_rng(seed)
    out = np.empty((rows, vocab), dtype=np.float32)
    down = math.log(vocab)   # a tail that far down weighs as much as the largest
    for r in range(rows):
        kind, share = r % 5, rng.uniform(-2.5, 1.5)
        if kind == 0:     # one value that takes rounding in every step
            tail = np.full(vocab, -(down + share) * 1.0123456789)
        elif kind == 1:   # few values
            tail = -(down + share) + rng.integers(0, 5, vocab) * 0.30103
        elif kind == 2:   # what a model in bf16 or f16 gives
            tail = torch.from_numpy(-(down + share) + rng.standard_normal(vocab)).to((torch.bfloat16, torch.float16)[r // 5 % 2]).double().numpy()
        elif kind == 3:   # all of it moved: the difference of two logits is rounded
            tail = np.full(vocab, -(down + share))
        else:
            tail = np.where(rng.random(vocab) < 0.5, -(down + share), -(down + share) - 7.7)
        x = tail.astype(np.float32)
        x[rng.integers(0, vocab, 1 + r % 3)] = 0.0
        out[r] = x + np.float32(20.3 if kind == 3 else 0.0)
    out[0] = -13.65625
    out[0, vocab // 7] = 0.0
    return torch.from_numpy(out).cuda()


def choices(x, T, k, top_p, min_p, coin, near):
    """`choose`, and what else may come out where a bound is up to `near` of the sum off."""
    x = x.astype(np.float64)
    w = np.exp((x - x.max()) / float(np.float32(T)))
    n = len(x)
    by_k, by_p, by_min = 0 < k < n, 0 < top_p < 1, min_p > 0
    order = np.lexsort((np.arange(n), -x)) if by_k or by_p or by_min else np.arange(n)
    w = w[order]
    least = max(1, int((w >= float(np.float32(min_p))).sum())) if by_min else n
    top, sums, out = k if by_k else n, np.cumsum(w), []
    for off in (-near, 0.0, near) if by_p else (0.0,):
        m = min(top, least, int(np.searchsorted(sums[:top], (float(np.float32(top_p)) + off) * sums[top - 1], side="right")) + 1 if by_p else n)
        for c in (-near, 0.0, near):
            at = min(int(np.searchsorted(sums[:m], (float(np.float32(coin)) + c) * sums[m - 1], side="right")), m - 1)
            out.append((int(order[at]), float(w[at] / sums[m - 1])))
    return out


def check_near(backend, logits, T, k, top_p, min_p, coin):
    """`check`, but where a coin or a top_p is so near to a border that the units decide, the token on either side of it will do; returns how many rows were decided.  A sum is off by half a
    unit and 2^-31 of itself per token, and so is the whole."""
    tokens, probs = run(backend, logits, T, k, top_p, min_p, coin)
    x, decided = logits.cpu().numpy(), 0
    for r in range(len(tokens)):
        may = choices(x[r], T[r], k[r] if k else 0, top_p[r] if top_p else 1.0, min_p[r] if min_p else 0.0, coin[r], logits.shape[1] * 2.0**-44 + 2.0**-30)
        assert any(tokens[r] == t and abs(probs[r] - p) <= p * (2**-24 + 2**-29) + x.shape[1] * 2**-44 for t, p in may), (r, tokens[r], probs[r], may, T[r], k and k[r], top_p and top_p[r], coin[r])
        decided += len({t for t, _ in may}) == 1
    return decided


@pytest.mark.parametrize("rows, vocab", [(3, 100000), (40, 100000), (24, 9000), (60, 32003), (300, 50000), (16, 524288)])
def test_tails_of_equal_logits(backend, rows, vocab):
    logits = tails(vocab, rows, vocab + rows)
    rng = np.random.default_rng(rows)
    coin = (1.0 - rng.random(rows) * 0.3).astype(np.float32).clip(max=1 - 2**-24).tolist()   # mostly in the tail, where the order is that of probabilities
    T = [1.0] * rows
    decided = []
    for _ in range(3):
        decided += [check_near(backend, logits, T, None, None, None, rng.random(rows).astype(np.float32).tolist())]
    decided += [check_near(backend, logits, T, None, (0.5 + 0.499 * rng.random(rows)).tolist(), None, coin)]
    decided += [check_near(backend, logits, T, [vocab - 1] * rows, (0.5 + 0.499 * rng.random(rows)).tolist(), None, coin)]
    decided += [check_near(backend, logits, T, None, [0.97] * rows, [1e-9] * rows, coin)]
    decided += [check_near(backend, logits, T, None, None, [1e-12] * rows, coin)]
    decided += [check_near(backend, logits, (0.8 + 0.4 * rng.random(rows)).astype(np.float32).tolist(), [0, vocab // 2] * (rows // 2) + [0] * (rows % 2), (0.9 + 0.0999 * rng.random(rows)).tolist(), None, coin)]
    assert sum(decided) >= 0.6 * rows * len(decided)   # (half a million tokens are some 3e-7 of the sum apart, at least, and the bounds 6e-8 wide)


def test_a_top_p_next_to_a_border(backend):
    """top_p and the coin so near to a border that the whole has to be known to a part in 10^8: on either side of it."""
    vocab, rows = 40000, 32
    logits = torch.randn(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(11), device="cuda").mul_(2.0).bfloat16().float()
    x = logits.cpu().numpy().astype(np.float64)
    top_p, coin = [], []
    for r in range(rows):
        w = np.sort(np.exp(x[r] - x[r].max()))[::-1]
        sums = np.cumsum(w)
        at = 200 + 37 * r                                   # that many tokens are left, or one more
        p = np.float32(sums[at - 1] / sums[-1])
        while abs(float(p) - sums[at - 1] / sums[-1]) < 3e-9:   # (not on the border itself)
            p = np.nextafter(p, np.float32(2))
        top_p.append(float(p))
        coin.append(1 - 2**-24)
    check(backend, logits, [1.0] * rows, None, top_p, None, coin)
    check(backend, logits, [1.0] * rows, None, [float(np.nextafter(np.float32(p), np.float32(0))) for p in top_p], None, coin)
