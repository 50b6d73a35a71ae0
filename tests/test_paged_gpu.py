"""Block tables, slot maps and cache appends of a paged cache, against plain restatements on the host."""
import ctypes as C

import numpy as np
import pytest
import torch

from inferi_b200 import ops
from inferi_b200.ops import InferiError, PagedAppend, PagedAppendConfig, PagePlan

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def plan_by_hand(P, cached, new, table, free, n_free, room, n_pages):
    """One request after the other, with a list for the stack."""
    table, n = table.copy(), len(cached)
    stack, back = list(free[:n_free]), []
    for i in range(n):
        if new[i] < 0 and 0 <= cached[i] <= table.shape[1] * P:
            back += list(table[i, : -(-cached[i] // P)])
    stack += back
    size = len(stack)
    free = free.copy()
    free[:size] = stack
    kv, starts, status, positions, slots = [0] * n, [0], [0] * n, [], []
    asked_tokens = asked_pages = 0
    for i in range(n):
        if cached[i] < 0 or cached[i] > table.shape[1] * P:
            status[i] = ops.PLAN_INVALID
        elif new[i] >= 0:
            kv[i] = cached[i]
            have, need = -(-cached[i] // P), -(-(cached[i] + new[i]) // P) - -(-cached[i] // P)
            if have + need > table.shape[1]:
                status[i] = ops.PLAN_TABLE_FULL
            elif new[i] > 0:
                asked_tokens += new[i]
                if asked_tokens > room:
                    status[i] = ops.PLAN_NO_ROOM
                else:
                    asked_pages += need
                    if need and asked_pages > size:
                        status[i] = ops.PLAN_NO_PAGES
                    else:
                        for j in range(need):
                            table[i, have + j] = stack.pop()
                        kv[i] = cached[i] + new[i]
                        for p in range(cached[i], kv[i]):
                            page = table[i, p // P]
                            positions.append(p)
                            slots.append(page * P + p % P if 0 <= page < n_pages else -1)
        starts.append(len(positions))
    pad = room - len(positions)
    return dict(table=table, free=free, kv=kv, starts=starts, status=status, positions=positions + [0] * pad, slots=slots + [-1] * pad, n_free=len(stack))


def run_plan(backend, P, cached, new, table, free, n_free, room, in_place=False):
    d = dict(cached=i32(cached), new=i32(new), table=i32(table), free=i32(free), n_free=i32([n_free]), starts=i32([-7] * (len(cached) + 1)), positions=i32([-7] * room), slots=i32([-7] * room),
             status=i32([-7] * len(cached)))
    d["kv"] = d["cached"] if in_place else i32([-7] * len(cached))
    n_free_out = d["n_free"] if in_place else i32([-7])
    PagePlan(backend).launch(P, d["cached"], d["new"], d["table"], d["free"], d["n_free"], d["kv"], d["starts"], d["positions"], d["slots"], n_free_out, d["status"])
    return dict({k: d[k].cpu().numpy() for k in ("table", "free", "kv", "starts", "status", "positions", "slots")}, n_free=int(n_free_out))


def check_plan(backend, P, cached, new, width, n_free, room, n_pages, in_place=False, table=None, seed=0):
    rng = np.random.default_rng(seed)
    ids = rng.permutation(n_pages)
    if table is None:
        table, at = np.full((len(cached), width), -1), 0
        for i, c in enumerate(cached):
            have = min(max(0, -(-c // P)), width)
            table[i, :have] = ids[at:at + have]
            at += have
        assert at + n_free <= n_pages
        ids = ids[at:]
    free = np.full(n_pages, -5)
    free[:n_free] = ids[:n_free]
    got, want = run_plan(backend, P, cached, new, table, free, n_free, room, in_place), plan_by_hand(P, cached, new, table, free, n_free, room, n_pages)
    for name, w in want.items():
        assert np.array_equal(got[name], w), f"{name}: {got[name]} instead of {w}"
    return got


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,P,longest,chunk", [(1, 16, 40, 1), (1, 16, 0, 700), (3, 32, 100, 90), (31, 16, 500, 1), (256, 64, 900, 20), (257, 16, 300, 5), (1024, 16, 100, 3), (1025, 1024, 4000, 100),
                                               (2500, 16, 64, 40)])
def test_plan_against_one_request_after_the_other(backend, n, P, longest, chunk, in_place):
    rng = np.random.default_rng(n + P)
    cached, new = rng.integers(0, longest + 1, n), rng.integers(0, chunk + 1, n)
    new[rng.random(n) < 0.2] = -1
    held, asked = int((-(-cached // P)).sum()), int((-(-(cached + np.maximum(new, 0)) // P) + cached // -P).sum())
    for n_free in (0, asked // 2, asked + 3):
        for room in (max(1, int(np.maximum(new, 0).sum()) // 2), int(np.maximum(new, 0).sum()) + 5):
            check_plan(backend, P, cached, new, (longest + chunk) // P + 2, n_free, room, held + n_free + 1, in_place)


def test_plan_refuses_requests_one_by_one(backend):
    # a negative length, one beyond its row, one whose tokens the row has no room for, one that fits to the last entry
    got = check_plan(backend, 16, [-3, 65, 60, 60, 64, 64], [2, 1, 5, 4, 0, 1], 4, 9, 50, 40, table=np.arange(24).reshape(6, 4))
    assert list(got["status"]) == [ops.PLAN_INVALID, ops.PLAN_INVALID, ops.PLAN_TABLE_FULL, 0, 0, ops.PLAN_TABLE_FULL]
    # behind a request that gets no pages, those that need none go on
    got = check_plan(backend, 16, [0, 5, 16, 3], [40, 2, 1, 13], 8, 2, 60, 40)
    assert list(got["status"]) == [ops.PLAN_NO_PAGES, 0, ops.PLAN_NO_PAGES, 0] and list(got["kv"]) == [0, 7, 16, 16]
    # ended requests with lengths that are no lengths return nothing; all of them ended
    check_plan(backend, 16, [-1, 1000, 20], [-1, -1, -5], 2, 1, 4, 12, table=np.arange(6).reshape(3, 2))


def test_plan_follows_no_page_outside_the_cache(backend):
    """Stack and table entries that are no pages of the cache come out as they are, and give no slots."""
    table = np.full((2, 3), -1)
    table[0, 0], table[1, 0] = 1000, 2
    free = np.array([3, -9, 77, 5, -5, -5, -5, -5])
    got = run_plan(backend, 16, [10, 16], [3, 17], table, free, 3, 40)
    assert list(got["slots"][:3]) == [-1] * 3 and list(got["table"][1]) == [2, 77, -9] and (got["slots"][3:20] == -1).all() and got["n_free"] == 1


def test_plan_with_more_pages_than_there_are(backend):
    """Pages that come back twice do not run over the stack's end."""
    table = np.tile(np.arange(4), (3, 1))
    got = run_plan(backend, 16, [64, 64, 64], [-1, -1, -1], table, np.full(6, -5), 2, 4)
    assert got["n_free"] == 6 and list(got["kv"]) == [0, 0, 0]
    got = run_plan(backend, 16, [64, 64, 16], [-1, -1, 30], table, np.full(6, -5), 1 << 20, 40)
    assert got["n_free"] == 4 and (got["slots"] == -1).all()


def test_plan_steps_of_a_server_and_its_graph(backend):
    """Thirty steps in place through one captured launch: every page is in one row or on the stack, once."""
    rng = np.random.default_rng(5)
    n, P, width, n_pages, room = 40, 16, 8, 200, 300
    cached, table, free, n_free = i32([0] * n), i32(np.full((n, width), -1)), i32(rng.permutation(n_pages)), i32([n_pages])
    new, starts, positions, slots, status = i32([0] * n), i32([0] * (n + 1)), i32([0] * room), i32([0] * room), i32([0] * n)
    args = (P, cached, new, table, free, n_free, cached, starts, positions, slots, n_free, status)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            PagePlan(backend).launch(*args)
    for step in range(30):
        add = rng.integers(0, 30, n)
        add[rng.random(n) < 0.2] = -1
        before = {k: v.cpu().numpy().copy() for k, v in (("cached", cached), ("table", table), ("free", free))}
        n_before = int(n_free)
        new.copy_(i32(add))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = plan_by_hand(P, before["cached"], add, before["table"], before["free"], n_before, room, n_pages)
        got = dict(table=table, kv=cached, starts=starts, status=status, positions=positions, slots=slots)
        for name, t in got.items():
            assert np.array_equal(t.cpu().numpy(), want[name]), (step, name)
        held = [p for i in range(n) for p in table[i, : -(-int(cached[i]) // P)].tolist()]
        assert sorted(held + free[: int(n_free)].tolist()) == list(range(n_pages))


def append_by_hand(variant, hs, base, q, k, v, positions):
    """Rotated q and k, in 64 bits."""
    theta = float(np.float32(base)) ** (-np.arange(0, hs, 2) / hs)
    angle = positions.astype(np.float64)[:, None, None] * theta

    def turn(x):
        x = x.astype(np.float64).reshape(len(x), -1, hs)
        a, b = (x[..., 0::2], x[..., 1::2]) if variant == ops.ROPE_ORIGINAL else (x[..., : hs // 2], x[..., hs // 2:])
        u, w = np.cos(angle) * a - np.sin(angle) * b, np.sin(angle) * a + np.cos(angle) * b
        out = np.empty_like(x)
        if variant == ops.ROPE_ORIGINAL:
            out[..., 0::2], out[..., 1::2] = u, w
        else:
            out[..., : hs // 2], out[..., hs // 2:] = u, w
        return out.reshape(len(x), -1)

    return turn(q), turn(k), v.astype(np.float64)


def check_append(backend, variant, hs, heads, kv_heads, n, P, dtype, far, base=500000.0, q_pad=0, offset=0, gap=0, in_place=False, seed=1):
    """q_pad: floats between q's rows; offset: floats by which the rows start off their buffers' 16-byte boundaries; gap: elements between pages."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    q_dim, kv_dim, n_pages = heads * hs, kv_heads * hs, n // P + 3

    def rows(dim, pad):
        return torch.randn(n * (dim + pad) + offset, generator=g, device="cuda")[offset:].view(n, dim + pad)[:, :dim]

    q, k, v = rows(q_dim, q_pad), rows(kv_dim, q_pad), rows(kv_dim, 0)
    positions = torch.randint(-3 if far < 100 else 0, far + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    slots = torch.randperm(n_pages * P, generator=g, device="cuda")[:n].to(torch.int32)
    slots[::7] = torch.tensor([-1, n_pages * P, -(1 << 31), (1 << 31) - 1], device="cuda", dtype=torch.int32)[torch.arange(len(slots[::7]), device="cuda") % 4]
    store = torch.randn(2, n_pages * (P * kv_dim + gap), generator=g, device="cuda").to(dtype)
    kc, vc = (s.as_strided((n_pages, P, kv_dim), (P * kv_dim + gap, kv_dim, 1)) for s in store)
    q_out = q if in_place else rows(q_dim, q_pad)
    before, q_before = store.clone(), q_out.clone()
    wq, wk, wv = append_by_hand(variant, hs, base, q.cpu().numpy(), k.cpu().numpy(), v.cpu().numpy(), positions.cpu().numpy())
    PagedAppend(backend).launch(variant, PagedAppendConfig(hs, base), q, k, v, positions, slots, q_out, kc, vc)
    s = slots.cpu().numpy().astype(np.int64)
    there = (s >= 0) & (s < n_pages * P)
    # a rotated element is two products of a cosine or sine that is off by 3e-7 at most (an angle within 2^-23 pi of a turn's half, plus half a step) and their rounded sum: 8e-7 of the pair's
    # length; the cache's type rounds once more, by at most half a step
    pair = lambda x: np.abs(x).max(axis=1, keepdims=True) * 1.5   # noqa: E731
    off = np.abs(q_out.cpu().numpy() - wq)
    assert (off[there] <= 8e-7 * pair(wq)[there] + 1e-30).all()
    assert np.array_equal(q_out.cpu().numpy()[~there], q_before.cpu().numpy()[~there])
    half_step = np.finfo(np.float16).eps / 2 if dtype == torch.float16 else np.finfo(np.float32).eps / 2
    for cache, want, rotated in ((kc, wk, True), (vc, wv, False)):
        got = cache.float().cpu().numpy().astype(np.float64).reshape(n_pages * P, kv_dim)[s[there]]
        assert (np.abs(got - want[there]) <= (8e-7 * pair(want)[there] if rotated else 0.0) + half_step * np.abs(want[there]) + 1e-7).all()
    for cache in (kc, vc):   # nothing else was written
        cache.reshape(n_pages * P, kv_dim) if gap == 0 else None
        flat = torch.tensor(s[there], device="cuda")
        cache[flat // P, flat % P] = 0
    for c, b in zip(store, before):
        view = b.as_strided((n_pages, P, kv_dim), (P * kv_dim + gap, kv_dim, 1))
        view[flat // P, flat % P] = 0
        assert torch.equal(c, b)


@pytest.mark.parametrize("variant", [ops.ROPE_ORIGINAL, ops.ROPE_NEOX])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hs,heads,kv_heads,n,P,far", [(128, 32, 8, 1, 16, 10), (64, 32, 8, 65, 16, 4000), (128, 28, 4, 40, 64, 131071), (64, 5, 5, 7, 32, 0), (8, 3, 1, 33, 16, 50),
                                                       (256, 2, 1, 9, 1024, 2**31 - 1), (96, 4, 2, 21, 16, 1 << 20)])
def test_append(backend, variant, dtype, hs, heads, kv_heads, n, P, far):
    check_append(backend, variant, hs, heads, kv_heads, n, P, dtype, far)


@pytest.mark.parametrize("variant", [ops.ROPE_ORIGINAL, ops.ROPE_NEOX])
@pytest.mark.parametrize("q_pad,offset,gap,in_place", [(64, 0, 0, False), (0, 0, 2048, True), (3, 0, 0, False), (0, 1, 8, False), (5, 3, 0, True), (128, 4, 64, True)])
def test_append_strides_and_alignment(backend, variant, q_pad, offset, gap, in_place):
    for dtype in (torch.float16, torch.float32):
        check_append(backend, variant, 64, 6, 2, 37, 16, dtype, 5000, q_pad=q_pad, offset=offset, gap=gap, in_place=in_place)


@pytest.mark.parametrize("hs,heads,kv_heads", [(2, 8, 8), (6, 4, 4), (12, 10, 2), (250, 4, 4)])
def test_append_head_sizes_that_are_no_multiples_of_8(backend, hs, heads, kv_heads):
    for variant in (ops.ROPE_ORIGINAL, ops.ROPE_NEOX):
        check_append(backend, variant, hs, heads, kv_heads, 19, 16, torch.float32, 300, base=10000.0)


def test_append_agrees_with_the_op_for_one_row(backend):
    """A row is what RoPE.launch makes of it (whose angles are 32-bit products: position 7, where they are exact to 7 * 2^-24)."""
    q, k, v = (torch.randn(1, d, device="cuda") for d in (2048, 512, 512))
    kc, vc, q_out = torch.zeros(1, 16, 512, device="cuda"), torch.zeros(1, 16, 512, device="cuda"), torch.empty_like(q)
    for variant in (ops.ROPE_ORIGINAL, ops.ROPE_NEOX):
        PagedAppend(backend).launch(variant, PagedAppendConfig(64, 1e4), q, k, v, i32([7]), i32([5]), q_out, kc, vc)
        q1, k1 = q[0].clone(), k[0].clone()
        ops.RoPE(backend).launch(variant, ops.RoPEConfig(64, 512, 7, 1e4), q1, k1)
        assert (q1 - q_out[0]).abs().max() <= 5e-6 and (k1 - kc[0, 5]).abs().max() <= 5e-6 and torch.equal(vc[0, 5], v[0])


def test_append_of_no_rows_launches_nothing(backend):
    e, kc = torch.zeros(0, 64, device="cuda"), torch.zeros(2, 16, 64, device="cuda")
    before = backend.launch_count()
    PagedAppend(backend).launch(ops.ROPE_ORIGINAL, PagedAppendConfig(64, 1e4), e, e, e, i32([]), i32([]), e, kc, kc.clone())
    assert backend.launch_count() == before


def test_refusals(backend):
    n, z = 3, lambda *s: torch.zeros(*s, device="cuda")   # noqa: E731
    q, kv, kc, vc, idx = z(n, 256), z(n, 128), z(4, 16, 128), z(4, 16, 128), i32([0, 1, 2])

    def append(message, variant=0, hs=64, base=1e4, q=q, k=kv, v=kv, positions=idx, slots=idx, q_out=q, kc=kc, vc=vc):
        with pytest.raises(InferiError, match=message):
            PagedAppend(backend).launch(variant, PagedAppendConfig(hs, base), q, k, v, positions, slots, q_out, kc, vc)

    append("unknown variant", variant=2)
    append("head_size=48", hs=48)
    append("head_size=0", hs=0)
    append("head_size", hs=-64)
    append("base_freq", base=0.0)
    append("base_freq", base=float("nan"))
    append("q: expected", q=q.half())
    append("q: expected", q=z(n, 512)[:, ::2])
    append("k: expected", k=z(n, 64))
    append("v: expected", v=z(2, 128))
    append("q_out: expected", q_out=z(n, 128))
    append("positions", positions=idx.long())
    append("slots", slots=i32([0, 1]))
    append("on device", slots=idx.cpu())
    append("float16 or both float32", kc=kc.double(), vc=vc.double())
    append("float16 or both float32", vc=vc.half())
    append("contiguous pages", kc=z(4, 16, 256)[:, :, :128], vc=z(4, 16, 256)[:, :, :128])
    append("page_size=24", kc=z(4, 24, 128), vc=z(4, 24, 128))
    append("page_size=8", kc=z(4, 8, 128), vc=z(4, 8, 128))
    append("16-byte aligned", kc=z(4 * 16 * 128 + 1)[1:].view(4, 16, 128), vc=z(4 * 16 * 128 + 1)[1:].view(4, 16, 128))
    append("multiples of 16 bytes", hs=2, k=z(n, 2), v=z(n, 2), kc=z(4, 16, 2), vc=z(4, 16, 2))

    def plan(message, page=16, cached=idx, new=idx, table=None, free=idx, n_free=None, slots=idx, status=idx):
        table, one = i32(np.zeros((3, 2))) if table is None else table, i32([1])
        with pytest.raises(InferiError, match=message):
            PagePlan(backend).launch(page, cached, new, table, free, one if n_free is None else n_free, idx.clone(), i32([0] * 4), slots.clone(), slots, one.clone(), status)

    plan("page_size=20", page=20)
    plan("page_size", page=-16)
    plan("new_len", new=idx[:2])
    plan("block table", table=i32([0, 0, 0]))
    plan("block table", table=i32(np.zeros((2, 2))))
    plan("n_free", n_free=idx)
    plan("status", status=idx.float())
    plan("on device", free=idx.cpu())
    plan("0 tokens", slots=i32([]))
    plan("0 pages", free=i32([]))
    a = ops.PagePlanArgs(9000, 1, 1, 1, 16, *[idx.data_ptr()] * 11)
    assert backend.lib.ib_page_plan(backend.handle, None, C.byref(a)) == 1 and b"9000 requests" in backend.lib.ib_last_error_string()
    assert backend.lib.ib_page_plan(backend.handle, None, None) == 1 and backend.lib.ib_paged_append(backend.handle, None, None, None) == 1


@pytest.mark.parametrize("n", [32, 33, 128, 129, 8192])
def test_plan_at_the_borders_of_its_launches(backend, n):
    test_plan_against_one_request_after_the_other(backend, n, 16, 90, 7, True)


@pytest.mark.parametrize("offset,room", [(0, 41), (1, 40), (2, 43), (3, 8)])
def test_plan_writes_its_rows_and_no_others(backend, offset, room):
    """Positions and slots that begin off the 16-byte boundaries, and end where four do not."""
    n, P = 6, 16
    cached, new, free = i32([0, 15, 16, 40, 3, 31]), i32([5, 2, -1, 9, 0, 11]), i32(np.arange(30))
    table = i32(np.arange(100, 100 + 6 * 4).reshape(6, 4) % 30)
    d = [i32([-7] * 60) for _ in range(2)]
    positions, slots = (t[offset: offset + room] for t in d)
    kv, starts, status, n_free = i32([0] * n), i32([0] * (n + 1)), i32([0] * n), i32([20])
    PagePlan(backend).launch(P, cached, new, table, free, n_free, kv, starts, positions, slots, n_free, status)
    for t in d:
        assert (t[:offset] == -7).all() and (t[offset + room:] == -7).all()
    total = int(starts[-1])
    assert total == (27 if room > 8 else 7)
    assert (positions[total:] == 0).all() and (slots[total:] == -1).all() and (slots[:total] >= 0).all()
    want = [p for c, a, b in zip(cached.tolist(), starts.tolist(), starts.tolist()[1:]) for p in range(c, c + b - a)]
    assert positions[:total].tolist() == want
    assert [s % P for s in slots[:total].tolist()] == [p % P for p in want]
    assert [s // P for s in slots[:total].tolist()] == [int(table[r, p // P]) for r, (c, a, b) in enumerate(zip(cached.tolist(), starts.tolist(), starts.tolist()[1:])) for p in range(c, c + b - a)]


@pytest.mark.parametrize("variant", [ops.ROPE_ORIGINAL, ops.ROPE_NEOX])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hs,heads,kv_heads,n", [(64, 4, 2, 1776), (64, 4, 2, 1777), (128, 3, 3, 2500), (8, 40, 2, 2000)])
def test_append_of_more_rows_than_have_a_place_together(backend, variant, dtype, hs, heads, kv_heads, n):
    check_append(backend, variant, hs, heads, kv_heads, n, 32, dtype, 2000)


def test_plan_of_no_requests(backend):
    """A server's step without any: no tokens, and the stack as it was."""
    for room, in_place in ((1, False), (9, True), (5000, False)):
        got = run_plan(backend, 16, [], [], np.zeros((0, 3)), np.arange(7), 5, room, in_place)
        assert list(got["starts"]) == [0] and (got["positions"] == 0).all() and (got["slots"] == -1).all() and got["n_free"] == 5 and list(got["free"]) == list(range(7))
