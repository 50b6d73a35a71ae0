"""The operators of a serving step together - plan, append, attention, sampling - and both ways to launch them; what needs no GPU: the structs' layouts and refusals."""
import ctypes as C
import importlib
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from inferi_b200 import _lib, ops
from inferi_b200.ops import BatchSampler, InferiError, PagedAppend, PagedAppendConfig, PagedAttention, PagedAttentionConfig, PagePlan

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---- without a GPU ----
@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_struct_layouts_are_the_headers(tmp_path):
    structs = {"ib_paged_cache": _lib.PagedCache, "ib_page_plan_args": _lib.PagePlanArgs, "ib_paged_append_args": _lib.PagedAppendArgs, "ib_paged_attn_args": _lib.PagedAttnArgs,
               "ib_sample_batch_args": _lib.SampleBatchArgs}
    lines = [f'printf("%zu", sizeof({s}));' + "".join(f'printf(" %zu", offsetof({s}, {f[0]}));' for f in t._fields_) + 'puts("");' for s, t in structs.items()]
    (tmp_path / "layout.c").write_text('#include <stddef.h>\n#include <stdio.h>\n#include "inferi_b200.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    printed = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines()
    for (name, t), line in zip(structs.items(), printed):
        assert [C.sizeof(t)] + [getattr(t, f[0]).offset for f in t._fields_] == [int(x) for x in line.split()], name


def test_null_contexts_are_rejected_without_touching_a_device():
    lib = _lib.load()
    assert lib.ib_page_plan(None, None, None) == 1 and lib.ib_paged_append(None, None, None, None) == 1
    assert lib.ib_paged_attention(None, None, None, None) == 1 and lib.ib_sample_batch(None, None, None) == 1
    assert b"null context" in lib.ib_last_error_string()


def test_the_binding_takes_nothing_that_it_cannot_check():
    binding = pytest.importorskip("inferi_b200._binding")
    i, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 64)
    plan = (16, i, i, i.view(4, 1), i, i, i, i, i, i, i, i)
    for args in [(1, 0) + plan, (0, 0) + plan, (1, 0) + plan[:-1], (1, "x") + plan, (None, 0) + plan, ()]:
        assert binding.page_plan(*args) == -1
    for args in [(1, 0, 0, 64, 1e4, f, f, f, i, i, f, f, f), (1, 0, 0, 64, None, f, f, f, i, i, f, f, f), (1, 0, 0, 64, 1e4, f, f, f, i, i, f, f), (1, 0, 0, -1, 1e4, f, f, f, i, i, f, f, 5)]:
        assert binding.paged_append(*args) == -1
    for args in [(1, 0, 1, 1, 64, 0, 0, 0, f, f, f, i, i, i, f), (1, 0, 2**40, 1, 64, 0, 0, 0, f, f, f, i, i, i, f), (1, 0, 1, 1, 64, 0, 0, -1, f, f, f, i, i, i, f), (1, 0, 1, 1, 64, 0, 0, 0, f)]:
        assert binding.paged_attention(*args) == -1
    for args in [(1, 0, 64, f, f, None, None, None, f, i, None), (1, 0, -5, f, f, None, None, None, f, i, None), (1, 0, 64, f, f, 3, None, None, f, i, None), (1, 0, 64)]:
        assert binding.sample_batch(*args) == -1


class NoDevice:
    """A context that is never launched with: every call on host tensors is refused before"""
    handle, _address, device, lib = None, 0, 0, None


def test_tensors_of_the_host_are_refused():
    b, i, f = NoDevice(), torch.zeros(4, dtype=torch.int32), torch.zeros(4, 64)
    cache = torch.zeros(2, 16, 64)
    for call in [lambda: PagePlan(b).launch(16, i, i, i.view(4, 1), i, i[:1], i, torch.zeros(5, dtype=torch.int32), i, i, i[:1], i),
                 lambda: PagedAppend(b).launch(0, PagedAppendConfig(64, 1e4), f, f, f, i, i, f, cache, cache),
                 lambda: PagedAttention(b).launch(PagedAttentionConfig(1, 1, 64), f, cache, cache, i.view(4, 1), torch.zeros(5, dtype=torch.int32), i, f),
                 lambda: BatchSampler(b, 64).sample(f, f[:, 0].contiguous(), None, None, None, f[:, 0].contiguous(), i)]:
        with pytest.raises((InferiError, ValueError)):
            call()


# ---- a step of a server ----
def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


class Server:
    """A model of one layer: the rows of q, k and v that a token has are a table's, and logits are the attention's output times a matrix.  `launch` is a step."""
    heads, mul, hs, vocab, P, base = 8, 2, 64, 700, 16, 10000.0

    def __init__(self, backend, n, n_pages, width, room, dtype, window=0, sinks=0):
        g = torch.Generator(device="cuda").manual_seed(n)
        self.n, self.dtype, self.window, self.sinks, self.room = n, dtype, window, sinks, room
        self.q_dim, self.kv_dim = self.heads * self.hs, self.heads // self.mul * self.hs
        self.tables = [torch.randn(self.vocab, d, generator=g, device="cuda") for d in (self.q_dim, self.kv_dim, self.kv_dim)]
        self.head = torch.randn(self.q_dim, self.vocab, generator=g, device="cuda") * 0.3
        self.kc, self.vc = (torch.full((n_pages, self.P, self.kv_dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.kv_len, self.new, self.status, self.n_free = i32([0] * n), i32([0] * n), i32([0] * n), i32([n_pages])
        self.table, self.free = i32(np.full((n, width), -1)), i32(np.random.default_rng(n).permutation(n_pages))
        self.row_start, self.positions, self.slots, self.ids = i32([0] * (n + 1)), i32([0] * room), i32([0] * room), torch.zeros(room, dtype=torch.int64, device="cuda")
        self.out, self.logits = torch.zeros(room, self.q_dim, device="cuda"), torch.zeros(n, self.vocab, device="cuda")
        self.temperature, self.top_p, self.min_p, self.coin = (torch.zeros(n, device="cuda") for _ in range(4))
        self.top_k, self.token, self.prob = i32([0] * n), i32([0] * n), torch.zeros(n, device="cuda")
        self.ops = PagePlan(backend), PagedAppend(backend), PagedAttention(backend), BatchSampler(backend, self.vocab)

    def launch(self):
        plan, append, attention, sampler = self.ops
        plan.launch(self.P, self.kv_len, self.new, self.table, self.free, self.n_free, self.kv_len, self.row_start, self.positions, self.slots, self.n_free, self.status)
        q, k, v = (t[self.ids] for t in self.tables)
        append.launch(ops.ROPE_NEOX, PagedAppendConfig(self.hs, self.base), q, k, v, self.positions, self.slots, q, self.kc, self.vc)
        attention.launch(PagedAttentionConfig(self.heads, self.mul, self.hs, self.window, self.sinks), q, self.kc, self.vc, self.table, self.row_start, self.kv_len, self.out)
        last = (self.row_start[1:] - 1).clamp(min=0).long()
        self.logits.copy_(self.out[last] @ self.head)
        sampler.sample(self.logits, self.temperature, self.top_k, self.top_p, self.min_p, self.coin, self.token, self.prob)

    def turned(self, x, positions):
        angle = positions.double()[:, None, None] * torch.tensor(float(np.float32(self.base)) ** (-np.arange(0, self.hs, 2) / self.hs), device="cuda")
        a, b = x.double().view(len(x), -1, self.hs).chunk(2, dim=-1)
        return torch.cat((angle.cos() * a - angle.sin() * b, angle.sin() * a + angle.cos() * b), dim=-1)

    def exact(self, ids, new):
        """Attention of the last `new` of a request's tokens, in 64 bits, and how far it may be off."""
        kv, half = len(ids), 2.0**-11 if self.dtype == torch.float16 else 2.0**-24   # rounding of the cache
        t = torch.tensor(ids, device="cuda")
        q, k, v = (x[t] for x in self.tables)
        at = torch.arange(kv, device="cuda")
        q, k = self.turned(q, at)[-new:].view(new, -1, self.mul, self.hs), self.turned(k, at)
        v = v.double().view(kv, -1, self.hs)
        s = torch.einsum("nhgd,khd->hgnk", q, k) / self.hs**0.5
        p = at[-new:, None]
        seen = at[None] <= p
        if self.window:
            seen = seen & ((p - at[None] < self.window) | (at[None] < self.sinks))
        w = torch.where(seen, s, -torch.inf).softmax(-1)
        # A score moves by the cache's rounding, half * A, a weight by twice that relative to itself, a value by half of itself.  The kernels: a score by (hs / 8 + 4) * 2^-23 * A as the
        # attention has it and 4 * 2^-23 * A by the rotations, a weight by twice that, hs = 64: 2^-18 * A; (8 + kv / 16) * 2^-23 of the sum, kv < 128: below 2^-18.
        A = float(torch.einsum("nhgd,khd->hgnk", q.abs(), k.abs()).max()) / self.hs**0.5
        return torch.einsum("hgnk,khd->nhgd", w, v).reshape(new, -1), float(v.abs().max()) * (2 * half * A + half + 2.0**-18 * (1 + A))


def chosen(x, T, k, top_p, min_p, coin):
    """(token, how near the coin is to another one, of the whole) of a row of logits, in 64 bits"""
    x = x.astype(np.float64)
    if not T > 0:
        return int(x.argmax()), 1.0
    w = np.exp((x - x.max()) / float(np.float32(T)))
    order = np.lexsort((np.arange(len(x)), -x)) if 0 < k < len(x) or 0 < top_p < 1 or min_p > 0 else np.arange(len(x))
    w = w[order]
    m, sums = k if 0 < k < len(x) else len(x), np.cumsum(w)
    near = 1.0
    if 0 < top_p < 1:
        limit = top_p * sums[m - 1]
        near, m = np.abs(sums[:m] - limit).min() / sums[m - 1], min(m, int((sums[:m] <= limit).sum()) + 1)
    if min_p > 0:
        near, m = min(near, np.abs(w - min_p).min()), min(m, max(1, int((w >= min_p).sum())))
    limit = coin * sums[m - 1]
    near = min(near, np.abs(sums[:m] - limit).min() / sums[m - 1])
    return int(order[min(int((sums[:m] <= limit).sum()), m - 1)]), near


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 3)])
def test_steps_of_a_server(backend, captured, dtype, window, sinks):
    """Prompts in chunks, decoding, requests that end and others that take their places, one that waits for pages: each step's tokens, attention and choice against 64 bits, from what
    the requests have been given so far."""
    rng = np.random.default_rng(3)
    n, room = 7, 120
    s = Server(backend, n, n_pages=20, width=9, room=room, dtype=dtype, window=window, sinks=sinks)
    s.temperature.copy_(torch.tensor([0.0, 0.7, 1.0, 1.3, 0.9, 0.8, 1.1]))
    s.top_k.copy_(torch.tensor([0, 0, 40, 0, 5, 0, 0]))
    s.top_p.copy_(torch.tensor([0.0, 0.9, 0.0, 0.95, 0.8, 0.0, 0.0]))
    s.min_p.copy_(torch.tensor([0.0, 0.0, 0.05, 0.0, 0.0, 0.1, 0.0]))
    settings = [t.tolist() for t in (s.temperature, s.top_k, s.top_p, s.min_p)]
    side, graph = torch.cuda.Stream(), None
    held = [[] for _ in range(n)]       # tokens of each request that are in the cache
    due = [rng.integers(0, s.vocab, rng.integers(1, 60)).tolist() for _ in range(n)]   # tokens that a request waits with
    statuses, told = set(), 0
    for step in range(24):
        new = [min(len(d), 25) for d in due]
        for r in range(n):
            if len(held[r]) > 70 or (step > 5 and rng.random() < 0.04):
                new[r], held[r], due[r] = -1, [], rng.integers(0, s.vocab, rng.integers(1, 60)).tolist()   # ended; the next one begins with the next step
        s.new.copy_(i32(new))
        coin = rng.random(n).astype(np.float32)
        s.coin.copy_(torch.from_numpy(coin))
        # the tokens of the rows, by the plan's rules: who has room, then who gets pages
        free, width = int(s.n_free) + sum(-(-int(s.kv_len[r]) // s.P) for r in range(n) if new[r] < 0), s.table.shape[1]
        ids, gets, used, asked = [], [0] * n, 0, 0
        for r in range(n):
            need = -(-(len(held[r]) + max(new[r], 0)) // s.P) - -(-len(held[r]) // s.P) if new[r] > 0 else 0
            fits = -(-(len(held[r]) + max(new[r], 0)) // s.P) <= width
            asked += new[r] if new[r] > 0 and fits else 0
            fits = fits and asked <= room
            used += need if fits else 0
            gets[r] = new[r] if new[r] > 0 and fits and (need == 0 or used <= free) else 0
            ids += due[r][: gets[r]]
        s.ids.zero_()
        s.ids[: len(ids)] = torch.tensor(ids, dtype=torch.int64, device="cuda")
        s.out.fill_(7.0)
        torch.cuda.synchronize()
        if captured and graph is None and step == 1:   # (the first step has set everything up)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                s.launch()
        if graph is not None:
            graph.replay()
        else:
            s.launch()
        torch.cuda.synchronize()
        starts, status = s.row_start.tolist(), s.status.tolist()
        statuses |= set(status)
        assert [b - a for a, b in zip(starts, starts[1:])] == gets, step
        assert torch.equal(s.slots[starts[-1]:], torch.full_like(s.slots[starts[-1]:], -1)) and bool((s.out[starts[-1]:] == 7.0).all())
        tokens, logits = s.token.tolist(), s.logits.cpu().numpy()
        for r in range(n):
            if gets[r] == 0:
                continue
            held[r] += due[r][: gets[r]]
            due[r] = due[r][gets[r]:]
            assert int(s.kv_len[r]) == len(held[r])
            want, tol = s.exact(held[r], gets[r])
            off = float((s.out[starts[r]: starts[r + 1]].double() - want).abs().max())
            assert off <= tol, (step, r, off, tol)
            token, near = chosen(logits[r], *(x[r] for x in settings), coin[r])
            if near > 1e-7:   # (the kernel is good to 1e-9)
                assert tokens[r] == token, (step, r)
                told += 1
            if not due[r]:
                due[r] = [tokens[r]]
    pages = [p for r in range(n) for p in s.table[r, : -(-int(s.kv_len[r]) // s.P)].tolist()]
    assert sorted(pages + s.free[: int(s.n_free)].tolist()) == list(range(20))
    assert {1, 3} <= statuses and told > 60   # somebody had to wait for pages, somebody for room


# ---- the compiled way and the Python way ----
class PythonOnly:
    page_plan = paged_append = paged_attention = sample_batch = staticmethod(lambda *a: -1)


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_both_ways_launch_the_same(backend, monkeypatch, captured):
    def steps():
        s = Server(backend, 5, 40, 8, 90, torch.float16)
        s.temperature.fill_(0.9)
        s.top_p.fill_(0.9)
        s.coin.copy_(torch.linspace(0, 0.99, 5))
        s.ids.copy_(torch.arange(90, device="cuda") * 7 % s.vocab)
        out = []
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for new in ([20, 1, 30, 0, 16], [1, 1, 1, 30, 1], [-1, 1, 1, 1, 1]):
                s.new.copy_(i32(new))
                if captured:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=side):
                        s.launch()
                    graph.replay()
                else:
                    s.launch()
                out += [t.clone() for t in (s.kv_len, s.table, s.free, s.row_start, s.positions, s.slots, s.status, s.out, s.token, s.prob)]
        side.synchronize()
        return out

    assert ops._fast is importlib.import_module("inferi_b200._binding")
    fast = steps()
    monkeypatch.setattr(ops, "_fast", PythonOnly)
    for a, b in zip(fast, steps()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_both_ways_refuse_the_same(backend, monkeypatch):
    b = backend
    i, f = (lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")), (lambda *s, **k: torch.zeros(*s, device="cuda", **k))
    cache, half = f(2, 16, 64), f(2, 16, 64, dtype=torch.float16)

    def plan(page=16, n=4, table=(4, 2), starts=5, status=4, slots=8, free=6):
        return lambda: PagePlan(b).launch(page, i(n), i(n), i(*table), i(free), i(1), i(n), i(starts), i(8), i(slots), i(1), i(status))

    def append(variant=0, hs=64, q=(3, 128), k=(3, 64), slots=3, kc=cache, vc=cache):
        return lambda: PagedAppend(b).launch(variant, PagedAppendConfig(hs, 1e4), f(*q), f(*k), f(3, 64), i(3), i(slots), f(*q), kc, vc)

    def attention(heads=2, mul=2, hs=64, q=(3, 128), out=(3, 128), table=(2, 2), starts=3, kc=cache, vc=cache, **more):
        return lambda: PagedAttention(b).launch(PagedAttentionConfig(heads, mul, hs, **more), f(*q), kc, vc, i(*table), i(starts), i(2), f(*out))

    def sample(vocab=50, logits=(4, 50), T=4, k=None, token=None):
        return lambda: BatchSampler(b, vocab).sample(f(*logits), f(T), k, None, None, f(4), token)

    def in_place():
        q = f(3, 128)
        PagedAttention(b).launch(PagedAttentionConfig(2, 2, 64), q, cache, cache, i(2, 2), i(3), i(2), q)

    refused = [plan(page=24), plan(page=8), plan(table=(3, 2)), plan(table=(8,)), plan(starts=4), plan(status=3), plan(slots=7), plan(free=0), plan(n=9000, table=(9000, 1), starts=9001, status=9000),
               append(variant=7), append(hs=48), append(hs=512, q=(3, 512)), append(q=(3, 100)), append(k=(3, 128)), append(slots=2), append(vc=half), append(kc=f(2, 16, 60), vc=f(2, 16, 60)),
               append(kc=f(2, 17, 64), vc=f(2, 17, 64)), append(kc=cache[0], vc=cache[0]),
               attention(hs=32, heads=4), attention(mul=1), attention(mul=3, heads=3, q=(3, 192), out=(3, 192), kc=half), attention(out=(2, 128)), attention(q=(3, 64)), attention(table=(3, 2)), attention(starts=2),
               attention(heads=0), attention(window=-1), attention(vc=cache[:, :, :32]), attention(heads=130, mul=130, q=(3, 130 * 64), out=(3, 130 * 64)),
               in_place, sample(vocab=51), sample(vocab=600000, logits=(4, 600000)), sample(T=3), sample(k=f(4)), sample(token=f(4)), sample(token=i(5))]

    def answers():
        out = []
        for call in refused:
            with pytest.raises((InferiError, ValueError)) as e:
                call()
            out.append((type(e.value), str(e.value)))
        return out

    fast = answers()
    monkeypatch.setattr(ops, "_fast", PythonOnly)
    assert answers() == fast
