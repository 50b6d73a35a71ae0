"""The operators that serve a batch of requests over a paged cache: their plain forms, and the calls that a user makes of the framework's.

A case is a dict of plain values.  Its `kind` says which operator it is:

  plan      block tables, positions and slots of a step from the requests' lengths (`PagePlan.launch`)
  append    rotation of queries and keys at every token's own position, keys and values into their slots (`PagedAppend.launch`)
  attention new tokens of several requests over the paged cache, single tokens and chunks of a prompt, with a sliding window and first tokens that stay
            visible, or without (`PagedAttention.launch`)
  sample    a token and its probability for every row of logits: temperature, top-k, top-p and min-p per row, given random numbers (`BatchSampler.sample`)

Head counts and vocabularies are those of `inferi_b200.llama2`'s two configurations (1B: 32 heads of 64, 8B: 32 heads of 128, both 8 kv heads) and generic ones.
"""
from __future__ import annotations

import math

import torch

own = False

ORIGINAL, NEOX = 0, 1
PAD_POSITION, NO_SLOT = 0, -1
OK, NO_PAGES, TABLE_FULL, NO_ROOM, INVALID = 0, 1, 2, 3, 4

_backend = None


def backend():
    """One context per process, as a host program keeps it."""
    global _backend
    if _backend is None:
        from inferi_b200.ops import Backend
        _backend = Backend(torch.cuda.current_device())
    return _backend


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    att = dict(kind="attention", page=16, window=0, sinks=0, pad=0, kv="f16")
    return [
        # a decode step of a small server: sixteen requests, one token each
        dict(name="plan 16 decoding", kind="plan", requests=16, page=16, longest=2000, chunk=0, ended=0.1, short=False),
        # a step of a large one: prompts' chunks between decoding requests, some of which have ended, and fewer free pages than are asked for
        dict(name="plan 2000 mixed", kind="plan", requests=2000, page=32, longest=8000, chunk=256, ended=0.05, short=True),
        # a decode step's keys and values, 1B heads
        dict(name="append 64 tokens", kind="append", tokens=64, heads=32, mul=4, hs=64, page=16, variant=ORIGINAL, far=4000, pad=0, kv="f16"),
        # chunks of prompts at far positions, 8B heads
        dict(name="append 8001 tokens", kind="append", tokens=8001, heads=32, mul=4, hs=128, page=64, variant=NEOX, far=120000, pad=191, kv="f16"),
        # one request decoding, 1B heads: latency
        dict(att, name="decode 1 of 500", requests=1, new=1, same=True, cached=500, heads=32, mul=4, hs=64),
        # a ragged decode batch, 8B heads: the cache's bytes count
        dict(att, name="decode 64 up to 8000", requests=64, new=1, same=True, cached=8000, heads=32, mul=4, hs=128, pad=3),
        # a chunk of a long prompt behind what is cached already, 8B heads
        dict(att, name="chunk 1000 after 15000", requests=1, new=1000, same=True, cached=15000, heads=32, mul=4, hs=128, page=64),
        # several prompts of a batch together, with the window that a model with a sliding window has, 1B heads
        dict(att, name="chunks window and sinks", requests=7, new=700, same=False, cached=5000, heads=32, mul=4, hs=64, page=32, window=1024, sinks=4, pad=55),
        # a few proposed tokens per request to be verified, 32-bit cache
        dict(att, name="verify 32-bit cache", requests=24, new=5, same=False, cached=3000, heads=32, mul=8, hs=128, kv="f32"),
        # one row of an 8B vocabulary: latency
        dict(name="sample 1 row", kind="sample", rows=1, vocab=128256, sharp=3.0, filters="top-p"),
        # a batch with settings of every request's own
        dict(name="sample 250 rows", kind="sample", rows=250, vocab=128256, sharp=3.0, filters="mixed"),
        # a smaller vocabulary, hot: long tails are kept
        dict(name="sample 33 rows hot", kind="sample", rows=33, vocab=32003, sharp=0.7, filters="mixed"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "attention", "attention", "attention", "sample"])
    heads = rng.choice([(32, 4, 64), (32, 4, 128), (8, 1, 64), (16, 2, 128), (64, 8, 64), (12, 4, 128), (16, 8, 128), (5, 1, 128), (28, 7, 128), (40, 5, 64)])
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        return dict(kind="plan", requests=_log_int(rng, 1, 2000), page=page, longest=_log_int(rng, 16, 8000), chunk=rng.choice([0, 1, rng.randint(2, 256)]),
                    ended=rng.choice([0.0, rng.uniform(0.0, 0.5)]), short=rng.random() < 0.5)
    if kind == "append":
        return dict(kind="append", tokens=_log_int(rng, 1, 8000), heads=heads[0], mul=heads[1], hs=heads[2], page=page, variant=rng.choice([ORIGINAL, NEOX]), far=_log_int(rng, 1, 130000),
                    pad=rng.choice([0, rng.randint(1, 64)]), kv=rng.choice(["f16", "f16", "f32"]))
    if kind == "sample":
        return dict(kind="sample", rows=_log_int(rng, 1, 250), vocab=_log_int(rng, 50, 128256), sharp=rng.uniform(0.5, 4.0), filters=rng.choice(["mixed", "top-p", "top-k", "min-p", "none"]))
    requests = _log_int(rng, 1, 64)
    new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 1500)
    cached = _log_int(rng, 1, 15000)
    while requests * new * (cached + new) * heads[0] > 300e6:   # (scores of a padded batch; the longest listed chunk has 512e6)
        requests, new, cached = max(1, requests // 2), max(1, new * 3 // 4), max(1, cached * 3 // 4)
    kv = rng.choice(["f16", "f16", "f32"])
    while requests * (cached + new) * heads[0] // heads[1] * heads[2] > (350e6 if kv == "f16" else 175e6):   # (elements of K; 390e6 in the largest listed decode step)
        requests, cached = max(1, requests // 2), max(1, cached * 3 // 4)
    window = rng.choice([0, 0, _log_int(rng, 1, 4096)])
    return dict(kind="attention", requests=requests, new=new, same=rng.random() < 0.5, cached=cached, heads=heads[0], mul=heads[1], hs=heads[2], page=page, window=window,
                sinks=rng.choice([0, 4, rng.randint(1, 200)]) if window else 0, pad=rng.choice([0, rng.randint(1, 64)]), kv=kv)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _cache_type(case):
    return torch.float16 if case["kv"] == "f16" else torch.float32


def _spread(n, lo, hi, g):
    """n numbers spread evenly over lo .. hi, in an order of the seed's."""
    return (lo + (hi - lo) * (torch.arange(n) + 0.5) / n).round().long()[torch.randperm(n, generator=g)]


def _lengths(case, seed):
    """(cached, new) of every request on the host: ragged, the same totals whatever the seed."""
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    n, top, new = case["requests"], case["cached"], case["new"]
    cached = _spread(n, top // 2, top, g) if n > 1 else torch.tensor([max(0, top - int(torch.randint(0, 8, (1,), generator=g)))])
    return cached, torch.full((n,), new, dtype=torch.long) if case["same"] else _spread(n, 0.3 * new, new, g).clamp(min=1)


def _plan_lengths(case, g):
    n = case["requests"]
    cached, new = _spread(n, 0, case["longest"], g), torch.ones(n, dtype=torch.long)
    kind = torch.randperm(n, generator=g)
    chunks, ended = int(0.2 * n) if case["chunk"] else 0, int(case["ended"] * n)
    new[kind[:chunks]] = _spread(chunks, 0, case["chunk"], g) if chunks else new[:0]
    new[kind[n - ended:]] = -1
    return cached, new


def _prepare_plan(case, seed):
    g = torch.Generator().manual_seed(seed)
    n, P = case["requests"], case["page"]
    cached, new = _plan_lengths(case, g)
    have = (cached + P - 1) // P
    added = new.clamp(min=0)
    asked = int(((cached + added + P - 1) // P - have).sum())
    n_free = max(1, asked * 7 // 10) if case["short"] else asked + 100
    most = (case["longest"] + max(case["chunk"], 1) + P - 1) // P + 1
    n_pages = n * most + 100
    ids = torch.randperm(n_pages, generator=g)
    table = torch.full((n, most), -1, dtype=torch.int32)
    table[torch.arange(most)[None, :] < have[:, None]] = ids[: int(have.sum())].to(torch.int32)
    free = torch.full((n_pages,), -1, dtype=torch.int32)
    free[:n_free] = ids[int(have.sum()):][:n_free].to(torch.int32)
    room = n + int(0.2 * n) * max(case["chunk"], 1)
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(cached=cached.to(**i32), new=new.to(**i32), table=table.cuda(), free=free.cuda(), n_free=torch.tensor([n_free], **i32), kv_len=torch.zeros(n, **i32),
                row_start=torch.zeros(n + 1, **i32), positions=torch.zeros(room, **i32), slots=torch.zeros(room, **i32), n_free_out=torch.zeros(1, **i32), status=torch.zeros(n, **i32))


def _prepare_append(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, pad, hs, kv_heads = case["tokens"], case["pad"], case["hs"], case["heads"] // case["mul"]
    q_dim, kv_dim = case["heads"] * hs, kv_heads * hs
    q, kv = torch.randn(n + pad, q_dim, generator=g, device="cuda"), torch.randn(n + pad, 2 * kv_dim, generator=g, device="cuda")   # (keys and values of one product)
    n_pages = (n + case["page"] - 1) // case["page"] + 5
    slots = torch.randperm(n_pages * case["page"], generator=g, device="cuda")[: n + pad].to(torch.int32) if n + pad <= n_pages * case["page"] else \
        torch.cat([torch.randperm(n_pages * case["page"], generator=g, device="cuda")[:n], torch.zeros(pad, dtype=torch.long, device="cuda")]).to(torch.int32)
    positions = torch.randint(0, case["far"] + 1, (n + pad,), generator=g, device="cuda", dtype=torch.int32)
    slots[n:], positions[n:] = NO_SLOT, PAD_POSITION
    cache = dict(generator=g, device="cuda")
    state = dict(q=q, k=kv[:, :kv_dim], v=kv[:, kv_dim:], positions=positions, slots=slots, q_out=torch.zeros(n + pad, q_dim, device="cuda"),
                 key_cache=torch.randn(n_pages, case["page"], kv_dim, **cache).to(_cache_type(case)), value_cache=torch.randn(n_pages, case["page"], kv_dim, **cache).to(_cache_type(case)))
    return state


def _prepare_attention(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    cached, new = _lengths(case, seed)
    n, P, hs = case["requests"], case["page"], case["hs"]
    q_dim, kv_dim = case["heads"] * hs, case["heads"] // case["mul"] * hs
    kv = cached + new
    pages = (kv + P - 1) // P
    max_pages = (case["cached"] + case["new"] + P - 1) // P + 1
    n_pages = n * max_pages
    host = torch.Generator().manual_seed(seed)
    table = torch.full((n, max_pages), -1, dtype=torch.int32)
    table[torch.arange(max_pages)[None, :] < pages[:, None]] = torch.randperm(n_pages, generator=host)[: int(pages.sum())].to(torch.int32)
    row_start = torch.zeros(n + 1, dtype=torch.int32)
    row_start[1:] = torch.cumsum(new, 0)
    tokens = n * case["new"] + case["pad"]   # rows of a batch of a fixed size: those behind the last request's stay as they are
    q = torch.randn(tokens, q_dim, generator=g, device="cuda") * 1.5
    key = torch.randn(n_pages, P, kv_dim, generator=g, device="cuda").to(_cache_type(case))
    value = torch.randn(n_pages, P, kv_dim, generator=g, device="cuda").to(_cache_type(case))
    # (host copies of the lengths' maxima: what a server that made the lengths knows)
    return dict(q=q, key_cache=key, value_cache=value, table=table.cuda(), row_start=row_start.cuda(), kv_len=kv.to(torch.int32).cuda(), out=torch.zeros(tokens, q_dim, device="cuda"),
                longest_new=int(new.max()), longest_kv=int(kv.max()))


def _prepare_sample(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, vocab = case["rows"], case["vocab"]
    logits = torch.randn(n, vocab, generator=g, device="cuda") * case["sharp"]
    logits[torch.rand(n, vocab, generator=g, device="cuda") < 0.001] = -math.inf   # forbidden tokens
    logits[:, vocab // 2] = logits[:, vocab // 3]                                     # ties
    rand = lambda: torch.rand(n, generator=g, device="cuda")   # noqa: E731
    temperature, coin = 0.5 + rand(), rand()
    top_k = torch.randint(1, 200, (n,), generator=g, device="cuda", dtype=torch.int32)
    top_p, min_p = 0.5 + 0.49 * rand(), 0.2 * rand()
    which = {"none": 0, "top-k": 1, "top-p": 2, "min-p": 3}.get(case["filters"])
    pick = torch.randint(0, 8, (n,), generator=g, device="cuda") if which is None else torch.full((n,), 1 << which >> 1, device="cuda")
    if which is None:
        temperature[rand() < 0.1] = 0.0
    top_k[(pick & 1) == 0] = 0
    top_p[(pick & 2) == 0] = 1.0
    min_p[(pick & 4) == 0] = 0.0
    return dict(logits=logits, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, coin=coin, token=torch.zeros(n, dtype=torch.int32, device="cuda"),
                prob=torch.zeros(n, device="cuda"))


def prepare(case, seed):
    state = {"plan": _prepare_plan, "append": _prepare_append, "attention": _prepare_attention, "sample": _prepare_sample}[case["kind"]](case, seed)
    return dict(state, case=case)


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _own_plan(s):
    from inferi_b200.ops import PagePlan
    PagePlan(backend()).launch(s["case"]["page"], s["cached"], s["new"], s["table"], s["free"], s["n_free"], s["kv_len"], s["row_start"], s["positions"], s["slots"], s["n_free_out"], s["status"])
    return _plan_outputs(s)


def _own_append(s):
    from inferi_b200.ops import PagedAppend, PagedAppendConfig
    c = s["case"]
    PagedAppend(backend()).launch(c["variant"], PagedAppendConfig(c["hs"], 500000.0), s["q"], s["k"], s["v"], s["positions"], s["slots"], s["q_out"], s["key_cache"], s["value_cache"])
    return dict(q=s["q_out"], key_cache=s["key_cache"], value_cache=s["value_cache"])


def _own_attention(s):
    from inferi_b200.ops import PagedAttention, PagedAttentionConfig
    c = s["case"]
    PagedAttention(backend()).launch(PagedAttentionConfig(c["heads"], c["mul"], c["hs"], c["window"], c["sinks"], s["longest_new"]), s["q"], s["key_cache"], s["value_cache"], s["table"], s["row_start"], s["kv_len"], s["out"])
    return s["out"]


def _own_sample(s):
    from inferi_b200.ops import BatchSampler
    BatchSampler(backend(), s["case"]["vocab"]).sample(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["coin"], s["token"], s["prob"])
    return dict(token=s["token"], prob=s["prob"])


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _plan_outputs(s):
    return {n: s[n] for n in ("table", "free", "kv_len", "row_start", "positions", "slots", "n_free_out", "status")}


def _before(v):
    """Sums of what is ahead of each element."""
    return torch.cumsum(v, 0) - v


def _plain_plan(s):
    P, table, free, room = s["case"]["page"], s["table"], s["free"], s["slots"].numel()
    n, width = table.shape
    cached, new = s["cached"].long(), s["new"].long()
    ended = new < 0
    have = (cached + P - 1) // P
    bad = (cached < 0) | (have > width)
    # pages of ended requests on top of the stack, in the order of requests and positions
    column = torch.arange(width, device=table.device)
    back = torch.where(ended & ~bad, have, 0)
    n_free = s["n_free"].long()
    place = n_free + _before(back)[:, None] + column[None, :]
    returned = column[None, :] < back[:, None]
    spill = torch.zeros(free.numel() + 1, dtype=free.dtype, device=free.device)
    spill[:-1] = free
    spill.scatter_(0, torch.where(returned, place, free.numel()).reshape(-1), table.reshape(-1))
    size = n_free + back.sum()
    free.copy_(spill[:-1])
    # who has room
    status = torch.where(bad, INVALID, OK)
    want = torch.where(bad | ended, 0, new)
    need = torch.where(want > 0, (cached + want + P - 1) // P - have, 0)
    status = torch.where((status == OK) & (have + need > width), TABLE_FULL, status)
    want = torch.where(status == OK, want, 0)
    status = torch.where((want > 0) & (_before(want) + want > room), NO_ROOM, status)
    need = torch.where(status == OK, need, 0)
    status = torch.where((need > 0) & (_before(need) + need > size), NO_PAGES, status)
    fine = status == OK
    want, need = torch.where(fine, want, 0), torch.where(fine, need, 0)
    # (the refused ones are behind everybody who got pages, so the sums ahead of those are the same with them and without)
    top = size - 1 - _before(need)
    nth = column[None, :] - have[:, None]
    taken = (nth >= 0) & (nth < need[:, None])
    table.copy_(torch.where(taken, free[(top[:, None] - nth).clamp(0, free.numel() - 1)], table))
    s["n_free_out"].copy_(size - need.sum())
    s["kv_len"].copy_(torch.where(bad | ended, 0, cached + want))
    ends = torch.cumsum(want, 0)
    s["row_start"][0] = 0
    s["row_start"][1:].copy_(ends)
    s["status"].copy_(status)
    t = torch.arange(room, device=table.device)
    of = torch.searchsorted(ends, t, right=True).clamp(max=n - 1)
    pos = cached[of] + t - (ends - want)[of]
    there = t < ends[-1]
    s["positions"].copy_(torch.where(there, pos, PAD_POSITION))
    slot = table[of, (pos // P).clamp(0, width - 1)].long() * P + pos % P
    s["slots"].copy_(torch.where(there, slot, NO_SLOT))
    return _plan_outputs(s)


def _rotated(x, positions, hs, variant):
    theta = 500000.0 ** (-torch.arange(0, hs, 2, device=x.device, dtype=torch.float64) / hs)
    angle = positions.double()[:, None, None] * theta
    c, sn = torch.cos(angle).float(), torch.sin(angle).float()
    x = x.reshape(x.shape[0], -1, hs)
    a, b = (x[..., 0::2], x[..., 1::2]) if variant == ORIGINAL else (x[..., : hs // 2], x[..., hs // 2:])
    u, w = c * a - sn * b, sn * a + c * b
    return torch.stack((u, w), -1).flatten(1) if variant == ORIGINAL else torch.cat((u, w), -1).flatten(1)


def _plain_append(s):
    c = s["case"]
    there = s["slots"] >= 0
    s["q_out"].copy_(torch.where(there[:, None], _rotated(s["q"], s["positions"], c["hs"], c["variant"]), s["q_out"]))
    for rows, cache in ((_rotated(s["k"], s["positions"], c["hs"], c["variant"]), s["key_cache"]), (s["v"], s["value_cache"])):
        flat = cache.view(-1, cache.shape[-1])
        flat[s["slots"][: c["tokens"]].long()] = rows[: c["tokens"]].to(cache.dtype)
    return dict(q=s["q_out"], key_cache=s["key_cache"], value_cache=s["value_cache"])


def _plain_attention(s):
    """Requests padded to the longest: scores [requests, kv heads, new * heads of a group, positions]."""
    c, hs, mul = s["case"], s["case"]["hs"], s["case"]["mul"]
    kv_heads, P, Lq, Lk = c["heads"] // mul, c["page"], s["longest_new"], s["longest_kv"]
    dev = s["q"].device
    row_start, kv_len = s["row_start"].long(), s["kv_len"].long()
    new = row_start[1:] - row_start[:-1]
    n = new.numel()
    at = torch.arange(Lk, device=dev)
    slot = s["table"].long()[:, at // P].clamp(min=0) * P + at % P
    key, value = (x.view(-1, kv_heads, hs)[slot].float().permute(0, 2, 1, 3) for x in (s["key_cache"], s["value_cache"]))       # [n, kv heads, Lk, hs]
    i = torch.arange(Lq, device=dev)
    row = (row_start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    there = i < new[:, None]
    q = s["q"][row].view(n, Lq, kv_heads, mul, hs).permute(0, 2, 1, 3, 4).reshape(n, kv_heads, Lq * mul, hs)
    pos = (kv_len - new)[:, None] + i
    gap = pos[:, :, None] - at
    seen = gap >= 0
    if c["window"]:
        seen = seen & ((gap < c["window"]) | (at < c["sinks"]))
    seen = (seen & there[:, :, None])[:, None, :, None, :]
    x = (q @ key.transpose(2, 3)).mul_(1.0 / math.sqrt(hs)).view(n, kv_heads, Lq, mul, Lk)
    x = x.masked_fill_(~seen, -math.inf)
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = x.sum(-1, keepdim=True)
    o = x.view(n, kv_heads, Lq * mul, Lk) @ value.masked_fill((at >= kv_len[:, None])[:, None, :, None], 0.0)
    o = (o.view(n, kv_heads, Lq, mul, hs) / total).permute(0, 2, 1, 3, 4).reshape(n, Lq, -1)
    rows = torch.arange(s["q"].shape[0], device=dev)
    of = torch.searchsorted(row_start[1:], rows, right=True).clamp(max=n - 1)
    o = o[of, (rows - row_start[of]).clamp(0, Lq - 1)]
    s["out"].copy_(torch.where((rows < row_start[-1])[:, None], o, s["out"]))
    return s["out"]


def _plain_sample(s):
    """Running sums next to a border: in 64 bits."""
    x, n, vocab = s["logits"].double(), s["logits"].shape[0], s["case"]["vocab"]
    hot = s["temperature"] > 0
    T = torch.where(hot, s["temperature"], 1.0).double()[:, None]
    w = ((x - x.amax(-1, keepdim=True)) / T).exp()
    top_k, top_p, min_p = s["top_k"].long()[:, None], s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    by_k, by_p, by_min = (top_k > 0) & (top_k < vocab), (top_p > 0) & (top_p < 1), min_p > 0
    filtered = by_k | by_p | by_min
    order = torch.where(filtered, torch.sort(x, dim=-1, descending=True, stable=True)[1], torch.arange(vocab, device=x.device))
    w = w.gather(-1, order)
    rank = torch.arange(vocab, device=x.device)[None, :]
    w = torch.where(by_k & (rank >= top_k), 0.0, w)
    sums = w.cumsum(-1)
    keep = ~(by_p & (sums - w > top_p * sums[:, -1:])) & ~(by_min & (w < min_p)) | (rank == 0)
    w = torch.where(keep, w, 0.0)
    sums = w.cumsum(-1)
    coin = s["coin"].double()[:, None]
    at = (sums <= coin * sums[:, -1:]).sum(-1, keepdim=True)
    last = vocab - 1 - (w > 0).flip(-1).int().argmax(-1, keepdim=True)
    at = torch.minimum(at, last)
    token, prob = order.gather(-1, at)[:, 0], (w.gather(-1, at) / sums[:, -1:])[:, 0]
    greedy = torch.where(x == x.amax(-1, keepdim=True), rank, vocab).amin(-1)
    s["token"].copy_(torch.where(hot, token, greedy))
    s["prob"].copy_(torch.where(hot, prob, 1.0))
    return dict(token=s["token"], prob=s["prob"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attention": _own_attention, "sample": _own_sample}[kind](state)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[kind](state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _pairs(cached, new, window, sinks):
    """Visible (token, position) pairs of a request, and how many positions any of its tokens sees."""
    if not window:
        return new * cached + new * (new + 1) // 2, cached + new
    p = torch.arange(cached, cached + new)
    near = (p + 1).clamp(max=window)
    first = (p + 1 - near).clamp(max=sinks)
    low = max(0, cached - window + 1)
    return int((near + first).sum()), cached + new - low + min(low, sinks)


def work(case):
    if case["kind"] == "plan":   # lengths in; lengths, starts and status out; positions and slots; table entries written; returned pages read and written
        cached, new = _plan_lengths(case, torch.Generator().manual_seed(1))
        P, added = case["page"], new.clamp(min=0)
        pages, back = int(((cached + added + P - 1) // P - (cached + P - 1) // P).sum()), int(((cached + P - 1) // P)[new < 0].sum())
        return {"bytes": case["requests"] * 5 * 4 + int(added.sum()) * 2 * 4 + 8 * (pages + back), "flops": 0}
    if case["kind"] == "append":
        q_dim, kv_dim = case["heads"] * case["hs"], case["heads"] // case["mul"] * case["hs"]
        elem = 2 if case["kv"] == "f16" else 4
        return {"bytes": case["tokens"] * (8 * q_dim + 2 * kv_dim * (4 + elem) + 8), "flops": case["tokens"] * 3 * (q_dim + kv_dim)}
    if case["kind"] == "attention":
        cached, new = _lengths(case, 1)
        seen = [_pairs(int(a), int(b), case["window"], case["sinks"]) for a, b in zip(cached, new)]
        q_dim, kv_dim = case["heads"] * case["hs"], case["heads"] // case["mul"] * case["hs"]
        elem = 2 if case["kv"] == "f16" else 4
        return {"bytes": int(new.sum()) * 8 * q_dim + sum(r for _, r in seen) * 2 * kv_dim * elem, "flops": 4 * q_dim * sum(p for p, _ in seen)}
    return {"bytes": 4 * case["rows"] * case["vocab"], "flops": 0}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_append(case, s):
    hs, n = case["hs"], case["tokens"]
    half = torch.arange(hs // 2, device="cuda", dtype=torch.float64)
    turn = s["positions"][:n].double()[:, None] * torch.exp(half * (-2.0 / hs * math.log(500000.0)))[None, :]
    spin = torch.polar(torch.ones_like(turn), turn)[:, None, :]

    def rotate(rows):
        r = rows[:n].double().reshape(n, -1, hs)
        if case["variant"] == ORIGINAL:
            return torch.view_as_real(torch.view_as_complex(r.reshape(n, -1, hs // 2, 2).contiguous()) * spin).reshape(n, -1)
        z = torch.complex(r[..., : hs // 2], r[..., hs // 2:]) * spin
        return torch.cat((z.real, z.imag), -1).reshape(n, -1)

    q, key, value = s["q_out"].double(), s["key_cache"].double(), s["value_cache"].double()
    q[:n] = rotate(s["q"])
    to = s["slots"][:n].long()
    key.view(-1, key.shape[-1])[to] = rotate(s["k"])
    value.view(-1, value.shape[-1])[to] = s["v"][:n].double()
    return dict(q=q, key_cache=key, value_cache=value)


def _exact_attention(case, s):
    hs, mul, P = case["hs"], case["mul"], case["page"]
    starts, lens = s["row_start"].tolist(), s["kv_len"].tolist()
    out = s["out"].double()
    for r, length in enumerate(lens):
        lo, hi = starts[r], starts[r + 1]
        pages = s["table"][r, : (length + P - 1) // P].long()
        key, value = (x[pages].reshape(-1, case["heads"] // mul, hs)[:length].double() for x in (s["key_cache"], s["value_cache"]))
        p = torch.arange(length - (hi - lo), length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        hidden = j > p
        if case["window"]:
            hidden = hidden | ((p - j >= case["window"]) & (j >= case["sinks"]))
        for h in range(case["heads"]):
            score = (s["q"][lo:hi, h * hs:(h + 1) * hs].double() @ key[:, h // mul].T) / math.sqrt(hs)
            out[lo:hi, h * hs:(h + 1) * hs] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ value[:, h // mul]
    return out


def _exact_sample(case, s):
    """The probability of the token that each row's coin falls on."""
    probs = []
    for r in range(case["rows"]):
        T, k, top, least, coin = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "coin"))
        if not T > 0:
            probs.append(1.0)
            continue
        x = s["logits"][r].double()
        p = torch.softmax(x / T, 0)
        if k > 0 or 0 < top < 1 or least > 0:
            p, _ = torch.sort(p, descending=True)
            m = int(k) if 0 < k < case["vocab"] else case["vocab"]
            if 0 < top < 1:
                m = min(m, 1 + int((p[:m].cumsum(0) <= top * p[:m].sum()).sum()))
            m = max(1, min(m, int((p >= least * p[0]).sum()) if least > 0 else m))
            p = p[:m]
        run_sum = p.cumsum(0)
        i = min(int((run_sum <= coin * run_sum[-1]).sum()), p.numel() - 1)
        probs.append(float(p[i] / run_sum[-1]))
    return dict(token=None, prob=torch.tensor(probs, dtype=torch.float64, device="cuda"))


def exact(case, seed):
    if case["kind"] == "plan":
        return None   # whole numbers
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](case, s)
