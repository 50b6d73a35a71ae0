"""Attention over a paged cache against its definition in 64 bits."""
import math

import pytest
import torch

from inferi_b200.ops import Backend, FusedAttention, AttnParams, InferiError, PagedAttention, PagedAttentionConfig

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


class Batch:
    """Requests with `cached` positions behind them and `new` tokens each, their pages shuffled over a cache whose unused rows hold NaN."""

    def __init__(self, cached, new, heads, mul, hs, P=16, dtype=torch.float16, pad=0, gap=0, q_pad=0, offset=0, seed=1, q_scale=1.0, spare=2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.cached, self.new, self.heads, self.mul, self.hs, self.P, self.gap = cached, new, heads, mul, hs, P, gap
        self.kv = [c + n for c, n in zip(cached, new)]
        kv_dim, n = heads // mul * hs, len(cached)
        pages = [-(-max(k, 0) // P) for k in self.kv]
        self.n_pages, width = sum(pages) + spare, max(pages) + 1
        ids = torch.randperm(self.n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
        self.store = torch.full((2, self.n_pages * (P * kv_dim + gap)), float("nan"), dtype=dtype, device="cuda")
        self.kc, self.vc = (s.as_strided((self.n_pages, P, kv_dim), (P * kv_dim + gap, kv_dim, 1)) for s in self.store)
        self.table = torch.full((n, width), 1 << 30, dtype=torch.int32)   # entries behind a request's pages are not looked at
        self.rows = []   # per request: [kv, kv_dim] of K and V as the cache holds them
        for r in range(n):
            mine, ids = ids[: pages[r]], ids[pages[r]:]
            self.table[r, : pages[r]] = torch.tensor(mine, dtype=torch.int32)
            k, v = (torch.randn(max(self.kv[r], 0), kv_dim, generator=g, device="cuda").to(dtype) for _ in range(2))
            for i, page in enumerate(mine):
                part = slice(i * P, min((i + 1) * P, self.kv[r]))
                self.kc[page, : part.stop - part.start], self.vc[page, : part.stop - part.start] = k[part], v[part]
            self.rows.append((k, v))
        self.table = self.table.cuda()
        self.start = [0]
        for c in new:
            self.start.append(self.start[-1] + c)
        self.row_start, self.kv_len = i32(self.start), i32(self.kv)
        tokens = self.start[-1] + pad

        def rows():
            return torch.randn(tokens * (heads * hs + q_pad) + offset, generator=g, device="cuda")[offset:].view(tokens, heads * hs + q_pad)[:, : heads * hs]

        self.q, self.out = rows(), rows()
        self.q *= q_scale

    def put(self, r, j, which, value):
        """Sets a position's row of K (0) or V (1), in the cache and in the copy."""
        self.rows[r][which][j] = value
        (self.kc, self.vc)[which][self.table[r, j // self.P].item(), j % self.P] = value

    def run(self, backend, window=0, sinks=0, longest_new=0):
        PagedAttention(backend).launch(PagedAttentionConfig(self.heads, self.mul, self.hs, window, sinks, longest_new), self.q, self.kc, self.vc, self.table, self.row_start, self.kv_len, self.out)
        return self.out

    def exact(self, r, window=0, sinks=0):
        """([new, heads, hs] of request r, how far a result may be off)"""
        n, kv, hs, G = self.new[r], self.kv[r], self.hs, self.mul
        k, v = (x.double().view(kv, self.heads // G, hs).permute(1, 0, 2) for x in self.rows[r])       # [kv heads, kv, hs]
        q = self.q[self.start[r]: self.start[r] + n].double().view(n, self.heads // G, G, hs).permute(1, 2, 0, 3)   # [kv heads, G, n, hs]
        p = torch.arange(kv - n, kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None, :]
        seen = j <= p
        if window:
            seen = seen & ((p - j < window) | (j < sinks))
        s = torch.einsum("hgnd,hkd->hgnk", q, k) / math.sqrt(hs)
        s = torch.where(seen, s, -math.inf)
        w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
        w = w / w.sum(-1, keepdim=True)
        w = torch.where(seen, w, 0.0)   # (rows that see nothing)
        # positions that a row does not see count for nothing, whatever they hold
        finite = torch.where(torch.isfinite(v), v, 0.0)
        out = torch.einsum("hgnk,hkd->hgnd", w, finite)
        odd = ~torch.isfinite(v).all(-1)
        for h, at in odd.nonzero().tolist():
            sees = seen[:, at]
            out[h][:, sees] = out[h][:, sees] + w[h][:, sees, at][..., None] * torch.where(torch.isfinite(v[h, at]), 0.0, v[h, at])
        # A score is off by at most the split of q (2^-23 of its terms' absolute sum A), hs / 8 truncated additions of two products (2^-23 of A each) and three roundings; a weight by twice that
        # (its own and the sum's) and the exponential's 2^-22, its split's 2^-22; the sum over positions adds 2^-23 per 16 of them and a rounding per step: all of it relative to the weighted sum of |v|.
        A = float(torch.einsum("hgnd,hkd->hgnk", q.abs(), torch.where(torch.isfinite(k), k, 0.0).abs()).max()) / math.sqrt(hs)
        tol = 2 * A * (hs / 8 + 4) * 2**-23 + (8 + kv / 16) * 2**-23
        return out.permute(2, 0, 1, 3).reshape(n, -1), tol * float(finite.abs().max()) + 1e-30

    def check(self, backend, window=0, sinks=0, longest_new=0, requests=None):
        before = self.out.clone()
        self.run(backend, window, sinks, longest_new)
        for r in requests if requests is not None else range(len(self.new)):
            if self.new[r] and self.kv[r] >= self.new[r]:
                want, tol = self.exact(r, window, sinks)
                got = self.out[self.start[r]: self.start[r + 1]].double()
                fine = torch.isfinite(want)
                assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"request {r}: other values that are no numbers"
                off = (got - want)[fine].abs().max() if fine.any() else 0.0
                assert off <= tol, f"request {r}: off by {float(off):.3e} > {tol:.1e}"
        assert torch.equal(self.out[self.start[-1]:], before[self.start[-1]:])   # rows behind the last request's stay
        return self.out.clone()


HEADS = [(32, 4, 64), (32, 4, 128), (4, 1, 64), (6, 2, 128), (16, 8, 64), (14, 7, 128), (12, 12, 64), (24, 24, 128), (64, 64, 64), (9, 3, 128), (20, 5, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("heads,mul,hs", HEADS)
def test_single_tokens(backend, heads, mul, hs, dtype):
    Batch([0, 1, 15, 16, 17, 63, 64, 65, 300, 1000], [1] * 10, heads, mul, hs, dtype=dtype, pad=3).check(backend)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("heads,mul,hs", HEADS)
def test_chunks(backend, heads, mul, hs, dtype):
    for longest in (0, 1, 129):
        Batch([0, 0, 7, 130, 64, 500, 31], [1, 70, 2, 129, 0, 33, 5], heads, mul, hs, P=32, dtype=dtype, pad=2).check(backend, longest_new=longest)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("cached,new,P", [(0, 1, 16), (0, 2, 1024), (5000, 1, 128), (0, 1000, 64), (3000, 300, 16), (17000, 9, 256), (0, 257, 16), (127, 128, 16), (128, 256, 16), (1, 255, 16)])
def test_one_request(backend, cached, new, P, dtype):
    Batch([cached], [new], 8, 4, 128, P=P, dtype=dtype).check(backend)
    Batch([cached], [new], 4, 2, 64, P=P, dtype=dtype).check(backend, longest_new=new)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 300), (16, 4), (63, 0), (64, 64), (100, 5), (129, 70), (400, 0), (1000, 200), (1 << 31, 0), (0xFFFFFFFF, 0xFFFFFFFF), (50, 0xFFFFFFFF)])
def test_windows_and_sinks(backend, window, sinks, dtype):
    Batch([0, 10, 700, 1500, 64, 333], [300, 1, 1, 65, 200, 8], 8, 4, 64, dtype=dtype).check(backend, window, sinks)
    Batch([900, 2100], [140, 1], 8, 4, 128, P=64, dtype=dtype).check(backend, window, sinks)


@pytest.mark.parametrize("gap,q_pad,offset", [(512, 0, 0), (64, 64, 0), (0, 3, 0), (0, 0, 1), (1024, 5, 2)])
def test_strides_and_alignment(backend, gap, q_pad, offset):
    for dtype in (torch.float16, torch.float32):
        Batch([5, 100, 40], [3, 1, 150], 8, 2, 64, dtype=dtype, gap=gap, q_pad=q_pad, offset=offset, pad=2).check(backend)
        Batch([5, 100], [1, 40], 4, 4, 128, dtype=dtype, gap=gap, q_pad=q_pad, offset=offset).check(backend, window=30, sinks=2)


def test_agrees_with_the_contiguous_op(backend):
    b = Batch([700], [1], 32, 4, 128)
    b.run(backend)
    k, v = b.rows[0]
    out = torch.empty(32 * 128, device="cuda")
    FusedAttention(backend).launch(AttnParams(701, 1024, 4, 32, 128, 700), b.q[0].contiguous(), k, v, out)
    assert (out - b.out[0]).abs().max() <= 2e-6


@pytest.mark.parametrize("n", [40, 127, 129, 200, 1000])
def test_many_requests(backend, n):
    """More requests than a CTA has threads, some without tokens; few units each and some long ones."""
    g = torch.Generator().manual_seed(n)
    cached, new = torch.randint(0, 60, (n,), generator=g).tolist(), torch.randint(0, 3, (n,), generator=g).tolist()
    cached[n // 3], new[n // 2], new[0], new[-1] = 4000, 90, 0, 1
    b = Batch(cached, new, 4, 2, 64)
    assert n < 1000 or len(cached) > 320
    b.check(backend, requests=[i for i in range(n) if i % 7 == 0 or new[i] > 3 or cached[i] > 100 or i == n - 1])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("scale", [1e-12, 1e-3, 30.0, 1e6])
def test_queries_of_any_size(backend, scale, dtype):
    """(At 1e6 the softmax is a choice of the largest score: the bound on a weight grows with the scores, and the check is of the choice where that is clear.)"""
    b = Batch([200, 64], [1, 70], 8, 4, 64, dtype=dtype, q_scale=scale)
    if scale < 1e5:
        b.check(backend)
    else:
        b.run(backend)
        for r in range(2):
            want, _ = b.exact(r)
            k = b.rows[r][0].double().view(b.kv[r], 2, 64)
            q = b.q[b.start[r]: b.start[r + 1]].double().view(-1, 8, 64)
            for h in range(8):
                s = q[:, h] @ k[:, h // 4].T
                s = s.masked_fill(torch.arange(b.kv[r], device="cuda")[None] > torch.arange(b.cached[r], b.kv[r], device="cuda")[:, None], -math.inf)
                top = s.topk(2, -1).values
                clear = (top[:, 0] - top[:, 1]) / 8.0 > top[:, 0].abs() * 1e-5 + 30
                got = b.out[b.start[r]: b.start[r + 1]].view(-1, 8, 64)[:, h]
                assert clear.any() and (got.double() - want.view(-1, 8, 64)[:, h])[clear].abs().max() <= 1e-5


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hs", [64, 128])
def test_masked_positions_may_hold_anything(backend, hs, dtype):
    """Infinities and NaN in rows of K and V that some rows of a tile see and others do not; the type's lowest and largest values."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    for new in (2, 40, 300):
        b = Batch([50, 90], [new, 1], 8, 4, hs, dtype=dtype, seed=new)
        b.put(0, 50 + new - 1, 1, float("nan"))       # the last token's V: only the last token sees it
        b.put(0, 50 + new // 2, 1, float("inf"))
        b.put(0, 50 + new // 2 + 1 if new > 2 else 0, 0, 0.0)
        b.check(backend)
        b = Batch([50, 90], [new, 1], 8, 4, hs, dtype=dtype, seed=new)
        b.put(0, 50 + new - 1, 0, float("nan"))       # ... and its K
        want, tol = b.exact(0)
        b.run(backend)
        assert torch.isnan(b.out[new - 1]).all() and (b.out[: new - 1].double() - want[: new - 1]).abs().max() <= tol
        # behind the window
        b = Batch([500], [new], 8, 4, hs, dtype=dtype, seed=new)
        for j, value in ((3, float("inf")), (200, float("nan")), (380, -float("inf")), (500 - 101, float("nan"))):
            b.put(0, j, 1, value)
        b.check(backend, window=100, sinks=2)
        # lowest and largest values: no overflow on the way where the result has none
        b = Batch([40], [new], 8, 4, hs, dtype=dtype, seed=new)
        b.put(0, 5, 1, high / 4)
        b.put(0, 40 + new - 1, 1, low / 4)
        b.check(backend)


def test_lengths_that_do_not_fit_together(backend):
    """Fewer cached positions than new tokens: the tokens at positions below 0 see nothing and get 0; rows never leave q."""
    b = Batch([4, 4], [6, 3], 8, 4, 64)
    b.kv_len = i32([2, 7])   # request 0: positions -4 .. 1
    b.out.fill_(5.0)
    b.run(backend)
    assert (b.out[:4] == 0).all() and torch.isfinite(b.out).all() and (b.out[4:6] != 0).any()
    assert torch.allclose(b.out[6:9].double(), b.exact(1)[0], atol=1e-5)
    for starts, kv in (([0, 9, 4], [10, 7]), ([-5, 6, 900], [10, 7]), ([3, 3, 3], [10, 7]), ([0, 6, 9], [-4, 1 << 30])):
        b.row_start, b.kv_len = i32(starts), i32(kv)
        b.run(backend)
    torch.cuda.synchronize()


def test_pages_outside_the_cache_do_not_reach_other_requests(backend):
    for longest in (0, 1, 50):
        b = Batch([200, 300, 90], [1, 50, 1], 8, 4, 128)
        for page in (-1, b.n_pages, 1 << 30, -(1 << 31)):
            b.table[0, 3] = page
            b.table[0, 0] = page
            b.check(backend, longest_new=longest, requests=[1, 2])


def test_nothing_to_do(backend):
    b = Batch([5, 6], [0, 0], 8, 4, 64, pad=4)
    b.check(backend)
    before = backend.launch_count()
    e = torch.zeros(0, 512, device="cuda")
    PagedAttention(backend).launch(PagedAttentionConfig(8, 4, 64), e, b.kc, b.vc, b.table, b.row_start, b.kv_len, e)
    PagedAttention(backend).launch(PagedAttentionConfig(8, 4, 64), b.q, b.kc, b.vc, b.table[:0], i32([0]), i32([]), b.out)
    assert backend.launch_count() == before


def test_results_repeat_bit_for_bit(backend):
    b = Batch([3000, 77, 900, 12000], [1, 300, 40, 1], 32, 4, 128, P=64)
    first = b.check(backend)
    for _ in range(5):
        assert torch.equal(b.run(backend), first)


def test_captured_first_call_and_replay_with_other_lengths(backend):
    """A context's first call while a stream is being captured; then lengths change and the graph is replayed."""
    own = Backend(0)
    b = Batch([800, 90, 0], [1, 60, 30], 8, 4, 64, pad=10)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        b.run(own)
    graph.replay()
    torch.cuda.synchronize()
    for r in range(3):
        want, tol = b.exact(r)
        assert (b.out[b.start[r]: b.start[r + 1]].double() - want).abs().max() <= tol
    b.new, b.kv, b.start = [2, 1, 20], [500, 80, 25], [0, 2, 3, 23]
    b.rows = [(k[:n], v[:n]) for (k, v), n in zip(b.rows, b.kv)]
    b.row_start.copy_(i32(b.start))
    b.kv_len.copy_(i32(b.kv))
    before = b.out.clone()
    graph.replay()
    torch.cuda.synchronize()
    for r in range(3):
        want, tol = b.exact(r)
        assert (b.out[b.start[r]: b.start[r + 1]].double() - want).abs().max() <= tol
    assert torch.equal(b.out[23:], before[23:])
    del graph
    own.close()


def test_two_contexts_side_by_side(backend):
    """Calls on two streams, a context each."""
    other = Backend(0)
    batches = [Batch([3000, 500], [1, 70], 8, 4, 128, seed=s) for s in (1, 2)]
    want = [b.check(backend) for b in batches]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for b, c, s in zip(batches, (backend, other), streams):
            with torch.cuda.stream(s):
                b.run(c)
    torch.cuda.synchronize()
    for b, w in zip(batches, want):
        assert torch.equal(b.out, w)
    other.close()


def test_a_cache_beyond_32_bit_offsets(backend):
    """Pages whose elements lie behind 2^32 bytes and 2^31 elements."""
    P, kv_dim, n_pages = 1024, 1024, 2200   # 2.3e9 elements
    kc = torch.empty(n_pages, P, kv_dim, dtype=torch.float16, device="cuda")
    vc = torch.empty(n_pages, P, kv_dim, dtype=torch.float16, device="cuda")
    for cached, new in ((1500, 1), (1100, 200)):
        b = Batch([cached], [new], 32, 4, 128, P=P)
        b.table[0, :2] = i32([n_pages - 1, n_pages - 2])
        for c, rows in ((kc, b.rows[0][0]), (vc, b.rows[0][1])):
            c[n_pages - 1], c[n_pages - 2, : b.kv[0] - P] = rows[:P], rows[P:]
        b.kc, b.vc, b.n_pages = kc, vc, n_pages
        b.check(backend)


def test_refusals(backend):
    b = Batch([20, 30], [1, 2], 8, 4, 64)

    def refused(message, heads=8, mul=4, hs=64, window=0, sinks=0, q=b.q, kc=b.kc, vc=b.vc, table=b.table, starts=b.row_start, kv=b.kv_len, out=b.out):
        with pytest.raises(InferiError, match=message):
            PagedAttention(backend).launch(PagedAttentionConfig(heads, mul, hs, window, sinks), q, kc, vc, table, starts, kv, out)

    refused("kv_mul=3", mul=3)
    refused("kv_mul=0", mul=0)
    refused("kv_mul=128", heads=128, mul=128, q=torch.zeros(3, 128 * 64, device="cuda"), out=torch.zeros(3, 128 * 64, device="cuda"))
    refused("q: expected", hs=128)
    refused("head_size=32", hs=32, q=torch.zeros(3, 256, device="cuda"), out=torch.zeros(3, 256, device="cuda"))
    refused("kv_dim=128", mul=8)
    refused("q: expected", q=b.q.half())
    refused("out: expected", out=b.out[:2])
    refused("window: -1", window=-1)
    refused("sinks", sinks=1 << 32)
    refused("row_start", starts=b.row_start[:2])
    refused("row_start", starts=b.row_start.long())
    refused("block_table: expected", table=b.table.T.contiguous().T)
    refused("block table", table=b.table[:1])
    refused("on device", kv=b.kv_len.cpu())
    refused("float16 or both float32", vc=b.vc.float())
    refused("contiguous pages", kc=b.kc.transpose(0, 1), vc=b.vc.transpose(0, 1))
    assert backend.lib.ib_paged_attention(backend.handle, None, None, None) == 1


def gives_up(backend, hs):
    """A launch whose waits are given 0.3 ms, thirty times what they take otherwise, and rows whose results take milliseconds: every row sees an infinite value, which does each of them again element by
    element, while the tensor cores' warps wait for the next tile's queries.  More query tiles than CTAs, so that most CTAs have a part of one, a whole one or more, and a part of another."""
    b = Batch([3000], [4100], 16, 4, hs, P=64)
    b.put(0, 5, 1, float("inf"))
    backend.set_wait_limit(300_000)
    b.run(backend)
    backend.set_wait_limit(2_000_000_000)
    return backend.lib.ib_stream_sync(backend.handle, torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("hs", [64, 128])
def test_a_wait_that_gives_up_ends_the_launch(hs):
    """Some warps of a CTA give up, others do not: the launch ends, and the next synchronising call says so, once."""
    own = Backend(0)
    assert gives_up(own, hs) == 5 and b"gave up waiting" in own.lib.ib_last_error_string()
    torch.cuda.synchronize()
    assert own.lib.ib_stream_sync(own.handle, torch.cuda.current_stream().cuda_stream) == 0
    own.close()


@pytest.mark.parametrize("hs", [64, 128])
def test_a_wait_that_gave_up_leaves_no_arrivals_for_later_launches(hs):
    """CTAs that gave up had parts of tiles left, whose other parts had arrived: later launches find counters that are zero, and merge what is there."""
    own, fresh = Backend(0), Backend(0)
    b = Batch([2900], [4100], 16, 4, hs, P=64, seed=2)
    want = b.run(fresh).clone()
    for _ in range(2):
        assert gives_up(own, hs) == 5
        for _ in range(3):
            b.out.fill_(float("nan"))
            assert torch.equal(b.run(own), want)
    assert own.lib.ib_stream_sync(own.handle, torch.cuda.current_stream().cuda_stream) == 0
    exact, tol = b.exact(0)
    assert (want.double() - exact).abs().max() <= tol
    own.close()
    fresh.close()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("new", [1, 2, 3, 40, 300])
def test_infinities_in_keys(backend, hs, new, dtype):
    """A key with an infinite element gives a score of an infinity, by the sign of q's: weight 0 for rows where that is negative, no number for the others; for both signs in a key, none either.  The
    elements of q are of any size, so that the remainders that the kernels split off have either sign, or are 0."""
    inf = float("inf")

    def key(b, r, j, *elements):
        k = b.rows[r][0][j].clone()
        for at, value in elements:
            k[at] = value
        b.put(r, j, 0, k)

    for cached, window, sinks in ((50, 0, 0), (700, 0, 0), (700, 90, 3)):
        b = Batch([cached, 20, 20], [new, 1, 2], 8, 4, hs, dtype=dtype, seed=new + cached)
        b.q[:, ::3] = b.q[:, ::3].half().float()   # (no remainder)
        b.q[:, 1::7] *= 1e-6
        key(b, 0, cached - 3, (3, inf))                       # the first kv head's
        key(b, 0, cached - 40, (hs + 5, -inf), (hs + 7, 2.0))   # the second one's
        key(b, 0, 1, (0, -inf))
        key(b, 1, 0, (hs - 1, inf))
        key(b, 2, 7, (9, -inf), (hs + 30, inf))
        if new > 1:
            key(b, 0, cached + new // 2, (2 * hs - 1, inf))
        b.check(backend, window, sinks)
        assert torch.isfinite(b.out).any() and torch.isnan(b.out).any()
        key(b, 0, cached - 3, (4, -inf))                      # both signs, mostly
        b.put(0, cached - 5, 1, inf)                          # and an infinite value next to it
        b.put(2, 7, 1, float("nan"))                          # at a weight of 0, or beside a score that is none: none
        b.check(backend, window, sinks)
    # no key but such: nothing to weigh
    b = Batch([0], [new], 8, 4, hs, dtype=dtype, seed=new)
    for j in range(new):
        key(b, 0, j, (6, inf), (hs + 6, -inf))
    b.check(backend)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("new,kv", [(3, 2), (6, 2), (40, 11), (300, 290), (300, 1)])
def test_rows_that_see_nothing_beside_values_that_are_no_numbers(backend, hs, new, kv, dtype):
    """Tokens ahead of position 0 get 0, also where rows of K and V that the tile's other tokens see hold anything."""
    b = Batch([0], [new], 8, 4, hs, dtype=dtype, seed=new)
    b.put(0, 0, 1, float("nan"))
    b.put(0, kv - 1, 1, float("inf"))
    b.put(0, kv - 1, 0, float("nan"))
    b.kv_len = i32([kv])
    b.out.fill_(5.0)
    b.run(backend)
    assert (b.out[: new - kv] == 0).all() and torch.isnan(b.out[new - kv:]).all()


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("bits", [0x7F800001, 0x7F801FFF, 0x7FC00000, 0x7FFFFFFF, -0x007FFFFF, -0x007FE001, -1])
def test_nan_of_any_payload_in_a_32_bit_cache(backend, hs, which, bits):
    """A NaN is one also where its payload is in the bits that tf32 does not hold: the rows that see it are NaN (of V: in its element), the others are as without it."""
    for new in (1, 2, 40):
        b = Batch([300], [new], 8, 4, hs, dtype=torch.float32, seed=new)
        clean = b.run(backend).clone()
        at = 300 + new // 2
        (b.kc, b.vc)[which].view(torch.int32)[b.table[0, at // 16].item(), at % 16, hs + 9] = bits   # the second kv head's
        got = b.run(backend).view(new, 8, hs)
        nan = torch.zeros_like(got, dtype=torch.bool)
        if which == 0:
            nan[new // 2:, 4:] = True
        else:
            nan[new // 2:, 4:, 9] = True
        assert torch.equal(torch.isnan(got), nan)
        assert (got - clean.view(new, 8, hs))[~nan].abs().max() <= 1e-5   # (rows done again are in another order)


LONG = [(5000, 1, 128), (12000, 1, 16), (17000, 9, 256), (3000, 300, 16), (6000, 40, 32)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("cached,new,P", LONG)
def test_rows_of_long_requests_by_their_own_size(backend, cached, new, P, hs, dtype):
    """Every row's error by its own norm.  A score is off by the 2^-22 of q's split and by hs / 8 truncations of two products, 2^-23 each, of partial sums that are of its own size (1 here, 4 at most):
    2e-6 where all go one way; what all of a row's scores have in common cancels, and what they do not adds up as the row's own elements do.  Twice that for the sums.  (A product without its remainder is
    off by 2^-12 of a score's terms.)"""
    b = Batch([cached, 700], [new, 1], 8, 4, hs, P=P, dtype=dtype, seed=cached + new)
    for window, sinks in ((0, 0), (2500, 130)):
        b.run(backend, window, sinks)
        want = b.exact(0, window, sinks)[0].view(new, 8, hs)
        off = (b.out[:new].view(new, 8, hs).double() - want).norm(dim=-1) / want.norm(dim=-1)
        assert off.max() <= 4e-6, f"off by {float(off.max()):.2e} of a row's norm"


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("cached,new,P,window,sinks", [c + (0, 0) for c in LONG] + [(0, 700, 64, 0, 0), (4000, 1, 64, 1100, 70), (3000, 260, 16, 900, 200)])
def test_every_position_counts_once(backend, cached, new, P, window, sinks, hs, dtype):
    """Values that are 1 in a column of their own for a position each, and 0 otherwise: the result is the weights, one by one, at every border of ranges, tiles and pages.  The bound is that of a weight in
    `Batch.exact`, relative to itself, and half a step of the remainders of f16 (2^-24 of 2^14 times the largest weight)."""
    b = Batch([cached, 70], [new, 1], 8, 4, hs, P=P, dtype=dtype, seed=cached + new + window)
    kv = cached + new
    k = b.rows[0][0].double().view(kv, 2, hs)
    q = b.q[:new].double().view(new, 2, 4, hs)
    s = torch.einsum("nhgd,khd->nhgk", q, k) / math.sqrt(hs)
    p, j = torch.arange(cached, kv, device="cuda")[:, None, None, None], torch.arange(kv, device="cuda")
    seen = (j <= p) & ((p - j < window) | (j < sinks)) if window else j <= p
    w = torch.where(seen, s, -math.inf).softmax(-1)
    A = float(torch.einsum("nhgd,khd->nhgk", q.abs(), k.abs()).max()) / math.sqrt(hs)
    tol = 2 * A * (hs / 8 + 4) * 2**-23 + (8 + kv / 16) * 2**-23
    pages = b.table[0, : -(-kv // P)].long()
    for first in range(0, kv, 2 * hs):
        values = torch.zeros(len(pages) * P, 2, hs, dtype=dtype, device="cuda")
        at = torch.arange(2 * hs, device="cuda")
        at = at[first + at < kv]
        values[first + at, at // hs, at % hs] = 1.0
        values[kv:] = float("nan")
        b.vc[pages] = values.view(len(pages), P, 2 * hs)
        b.run(backend, window, sinks)
        got = b.out[:new].view(new, 2, 4, hs).double().permute(0, 2, 1, 3).reshape(new, 4, 2 * hs)[..., : len(at)]
        want = torch.stack([w[:, h // hs, :, first + h] for h in range(len(at))], -1)
        off = (got - want).abs() - tol * want - torch.where(want > 0, 2.0**-38, 0.0) * w.amax()
        assert off.max() <= 0, f"position {first + int(off.amax((0, 1)).argmax())}"


def test_infinities_in_a_long_prompt(backend):
    """Every row of a chunk behind 260,000 positions sees an infinity, so each is done again: 256 of them, while other warps of the CTA wait for the next tile, take two thirds of the waits' limit."""
    b = Batch([260000], [2400], 32, 4, 128, P=256)
    clean = b.run(backend).clone()
    k, v = (b.rows[0][which][at].clone() for which, at in ((0, 250000), (1, 5)))
    b.put(0, 5, 1, float("inf"))
    odd = k.clone()
    odd[130] = -float("inf")   # a score of an infinity for the second kv head: weight 0, or no number
    b.put(0, 250000, 0, odd)
    b.run(backend)
    assert backend.lib.ib_stream_sync(backend.handle, torch.cuda.current_stream().cuda_stream) == 0
    out, lost = b.out.view(2400, 32, 128), b.q.view(2400, 32, 128)[:, 4:8, 2] < 0
    assert torch.isposinf(out[:, :4]).all() and torch.isposinf(out[:, 8:]).all()
    assert torch.isnan(out[:, 4:8][lost]).all() and torch.isposinf(out[:, 4:8][~lost]).all() and lost.any() and (~lost).any()
    b.put(0, 5, 1, v)
    b.put(0, 250000, 0, k)
    assert torch.equal(b.run(backend), clean)


def test_synchronize_says_that_a_launch_gave_up():
    own = Backend(0)
    own.synchronize()
    b = Batch([3000], [4100], 16, 4, 64, P=64)
    b.put(0, 5, 1, float("inf"))
    own.set_wait_limit(300_000)
    b.run(own)
    with pytest.raises(InferiError) as e:
        own.synchronize()
    assert e.value.code == 5 and "gave up waiting" in e.value.message
    own.synchronize()
    own.set_wait_limit(2_000_000_000)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b.run(own)
        own.synchronize()
        assert side.query()
    own.close()
