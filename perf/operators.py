"""The operators of a serving step over a paged K/V cache, as cases that can be timed and compared.

A serving engine that keeps the paging metadata itself does four things per step around the layers of a model:

* ``plan``: from the requests' lengths and the tokens that each is fed, page allocation, the block tables, the index
  pointers that attention reads, and the cache slot and position of every new token (``plan_step``);
* ``append``: QK norm and rotary embedding of the new rows, K and V into their slots (``rotate_append``);
* ``attention``: the new tokens of every request over its pages, causal, with or without a sliding window and first
  tokens that stay visible; one new token per request (decode), chunks of a prompt, or both in one batch
  (``chunk_attention``);
* ``sample``: a token per request from its last row of logits, with temperature, top-k, top-p and min-p and given
  random numbers (``sample_tokens``).

``own`` false: plain forms in elementary torch operations.  ``own`` true: the framework's calls.
"""
import math

import torch

own = False

D = 128  # head dimension of the framework
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# (q heads, kv heads) of the framework's geometries and tests, and of the 30B-A3B one
HEADS = [(4, 2), (8, 2), (8, 8), (16, 8), (32, 8), (32, 8), (32, 4)]


def listed():
    def attn(name, requests, new_lo, new_hi, cached_lo, cached_hi, heads, page, **kw):
        c = {"name": name, "kind": "attention", "requests": requests, "new_lo": new_lo, "new_hi": new_hi, "cached_lo": cached_lo,
             "cached_hi": cached_hi, "decode": 0, "n_q": heads[0], "n_kv": heads[1], "page": page, "window": 0, "sinks": 0,
             "pad": 0, "dtype": "bf16"}
        c.update(kw)
        return c

    return [
        # eight running requests of different ages, one token each: latency alone
        {"name": "plan_b8", "kind": "plan", "requests": 8, "len_lo": 90, "len_hi": 1100, "chunk": 0, "page": 64, "ended": 0, "dry": False},
        # a large server's step: 512 requests up to 8000 tokens old, every 16th fed a prompt chunk, some just ended
        {"name": "plan_b512", "kind": "plan", "requests": 512, "len_lo": 1, "len_hi": 8000, "chunk": 256, "page": 16, "ended": 9, "dry": False},
        # one layer's rows of a decode step over sixteen requests
        {"name": "append_b16", "kind": "append", "tokens": 16, "n_q": 32, "n_kv": 8, "page": 64, "norm": True, "pad": 0, "dtype": "bf16"},
        # one layer's rows of a 4000-token prompt chunk, in a padded batch of 4096
        {"name": "append_chunk", "kind": "append", "tokens": 4000, "n_q": 32, "n_kv": 8, "page": 64, "norm": True, "pad": 96, "dtype": "bf16"},
        # one user of a small model: latency alone
        attn("decode_b1", 1, 1, 1, 1200, 1200, (8, 2), 64),
        # a decode step over 64 requests of different ages
        attn("decode_b64", 64, 1, 1, 90, 2200, (32, 8), 16),
        # four users with long documents, few kv heads
        attn("decode_long", 4, 1, 1, 20000, 32700, (32, 4), 64),
        # decode and prompt chunks in one batch, padded
        attn("mixed_b24", 24, 40, 333, 0, 1900, (32, 8), 64, decode=18, pad=13),
        # the last chunk of a long prompt
        attn("chunk_long", 1, 2048, 2048, 6111, 6111, (32, 8), 64, dtype="fp16"),
        # two prompts from their beginning, each row seeing 1024 positions and the first four
        attn("window_prefill", 2, 3500, 4096, 0, 0, (32, 8), 64, window=1024, sinks=4),
        # one user's next token from the benchmark's vocabulary
        {"name": "sample_b1", "kind": "sample", "requests": 1, "chunk": 1, "vocab": 151936, "dtype": "bf16", "mode": "top_k_top_p"},
        # 64 users with settings of their own, greedy ones among them, behind a mixed step
        {"name": "sample_b64", "kind": "sample", "requests": 64, "chunk": 2, "vocab": 151936, "dtype": "fp32", "mode": "mixed"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 200.0)


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["plan", "append", "attention", "attention", "attention", "sample"])
        if kind == "plan":
            lo = rng.choice([0, 1, _log_int(rng, 1, 1000)])
            case = {"kind": kind, "requests": _log_int(rng, 1, 600), "len_lo": lo, "len_hi": lo + _log_int(rng, 1, 8000),
                    "chunk": rng.choice([0, _log_int(rng, 1, 500)]), "page": rng.choice([1, 8, 16, 16, 64, 64, 128]),
                    "ended": rng.choice([0, 0, rng.randint(1, 9)]), "dry": rng.random() < 0.2}
            if case["requests"] * case["len_hi"] / case["page"] > 600000:
                continue
        elif kind == "append":
            n_q, n_kv = rng.choice(HEADS)
            case = {"kind": kind, "tokens": _log_int(rng, 1, 4200), "n_q": n_q, "n_kv": n_kv, "page": rng.choice([1, 8, 16, 64, 64, 128]),
                    "norm": rng.random() < 0.7, "pad": rng.choice([0, rng.randint(1, 100)]), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        elif kind == "attention":
            n_q, n_kv = rng.choice(HEADS + [(12, 4), (14, 2)])
            shape = rng.choice(["decode", "decode", "few", "chunk", "chunk", "mixed"])
            r = _log_int(rng, 1, 96)
            lo, hi = _log_int(rng, 1, 4000), _log_int(rng, 1, 4000)
            case = {"kind": kind, "requests": r, "new_lo": 1, "new_hi": 1, "cached_lo": min(lo, hi) - 1, "cached_hi": max(lo, hi), "decode": 0,
                    "n_q": n_q, "n_kv": n_kv, "page": rng.choice([1, 8, 16, 16, 64, 64, 128])}
            if shape == "decode" and r <= 8 and rng.random() < 0.4:
                case["cached_hi"] = _log_int(rng, 4000, 33000)
            if shape == "few":
                case["new_hi"] = rng.randint(2, 20)
            elif shape in ("chunk", "mixed"):
                a, b = _log_int(rng, 2, 4096), _log_int(rng, 2, 4096)
                case["new_lo"], case["new_hi"] = min(a, b), max(a, b)
                if shape == "mixed":
                    case["decode"] = rng.randint(0, r)
            case["window"] = rng.choice([0, 0, 0, _log_int(rng, 1, 2000)])
            case["sinks"] = rng.choice([0, 1, 4, rng.randint(1, 300)]) if case["window"] else 0
            case["pad"] = rng.choice([0, 0, rng.randint(1, 50)])
            case["dtype"] = rng.choice(["bf16", "bf16", "fp16"])
            if r * n_q * case["new_hi"] * (case["cached_hi"] + case["new_hi"]) > 1.2e9:  # scores of the plain form
                continue
            if r * n_kv * (case["cached_hi"] + case["new_hi"]) > 1.2e7:  # its rows of K
                continue
        else:
            case = {"kind": kind, "requests": _log_int(rng, 1, 96), "chunk": rng.choice([1, 1, 2]), "vocab": rng.choice([2048, 8192, 32008, 151936, 151936, _log_int(rng, 2, 200000)]),
                    "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32", "fp32"]), "mode": rng.choice(["plain", "top_k", "top_p", "min_p", "top_k_top_p", "mixed", "mixed"])}
        if _cost(case) <= limit:
            return case


# ------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------
def _spread(lo, hi, n):
    """n lengths over [lo, hi], in a mixed order (the same for every seed)."""
    if n == 1:
        return [hi]
    v = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return [v[(i * 5) % n] for i in range(n)] if n % 5 else v[::-1]


def _plan_lengths(case):
    """(cached, new) tokens of every request; new -1: the request has ended."""
    cached = _spread(case["len_lo"], case["len_hi"], case["requests"])
    new = [1] * len(cached)
    for i in range(0, len(cached), 16):
        new[i] = case["chunk"] or 1
    for i in range(case["ended"]):
        new[(7 * i + 3) % len(new)] = -1
    for i in range(5, len(new), 40):
        new[i] = 0  # idle
    return cached, new


def _attention_lengths(case):
    """(new, cached) tokens of every request."""
    r = case["requests"]
    new = _spread(case["new_lo"], case["new_hi"], r)
    new = [1 if i < case["decode"] else n for i, n in enumerate(new)]
    return new, _spread(case["cached_lo"], case["cached_hi"], r)


def _pages(n, page):
    return (n + page - 1) // page


class _State:
    pass


def _prepare_plan(case, s, gen, dev):
    page = case["page"]
    cached, new = _plan_lengths(case)
    s.page = page
    held = [_pages(n, page) for n in cached]
    most = max(_pages(n + max(0, t), page) for n, t in zip(cached, new)) + 1
    need = sum(_pages(n + t, page) - h for n, t, h in zip(cached, new, held) if t > 0)
    pool = sum(held) + need + 7
    perm = torch.randperm(pool, generator=gen, device=dev).to(torch.int32)
    s.lengths = torch.tensor(cached, dtype=torch.int32, device=dev)
    s.new_tokens = torch.tensor(new, dtype=torch.int32, device=dev)
    h = torch.tensor(held, device=dev)
    first = torch.cumsum(h, 0) - h
    col = torch.arange(most, device=dev)
    s.block_table = torch.where(col < h[:, None], perm[(first[:, None] + col).clamp_max(pool - 1)], -1).to(torch.int32)
    # the free pages sit in a ring that has wrapped round
    left = pool - sum(held)
    head = pool - left // 2 + 3 * pool
    s.free_pages = torch.full((pool,), -1, dtype=torch.int32, device=dev)
    s.free_pages[(head + torch.arange(left, device=dev)) % pool] = perm[sum(held):]
    tail = head + (max(0, need // 2) if case["dry"] else left)  # dry: the pool runs out in this step
    s.free_range = torch.tensor([head, tail], dtype=torch.int64, device=dev)
    R, T = len(cached), sum(max(0, t) for t in new) + 5
    i32 = dict(dtype=torch.int32, device=dev)
    s.plan = {"qo_indptr": torch.zeros(R + 1, **i32), "kv_indptr": torch.zeros(R + 1, **i32), "kv_indices": torch.zeros(pool, **i32),
              "last_page_len": torch.zeros(R, **i32), "slots": torch.zeros(T, dtype=torch.int64, device=dev), "positions": torch.zeros(T, **i32),
              "granted": torch.zeros(R, **i32), "free_range": torch.zeros(2, dtype=torch.int64, device=dev)}


def _prepare_append(case, s, gen, dev):
    T, pad, n_q, n_kv, page, dt = case["tokens"], case["pad"], case["n_q"], case["n_kv"], case["page"], DTYPES[case["dtype"]]
    rows = T + pad
    qkv = torch.randn(rows, (n_q + 2 * n_kv) * D, generator=gen, device=dev, dtype=torch.float32).to(dt)
    s.q, s.k, s.v = (x.view(rows, -1, D) for x in qkv.split([n_q * D, n_kv * D, n_kv * D], dim=1))
    most = 2 * T + 70
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D))
    ang = torch.arange(most, dtype=torch.float64, device=dev)[:, None] * inv[None, :]
    ang = torch.cat((ang, ang), dim=-1)
    s.cos, s.sin = ang.cos().to(dt), ang.sin().to(dt)
    pool = _pages(T, page) + 3
    perm = torch.randperm(pool, generator=gen, device=dev)
    at = torch.arange(T, device=dev)
    s.slots = torch.full((rows,), -1, dtype=torch.int64, device=dev)
    s.slots[:T] = perm[at // page] * page + at % page
    s.positions = torch.zeros(rows, dtype=torch.int32, device=dev)
    s.positions[:T] = (at + T // 2).to(torch.int32)
    s.k_cache = torch.randn(pool, page, n_kv, D, generator=gen, device=dev, dtype=torch.float32).to(dt)
    s.v_cache = torch.randn(pool, page, n_kv, D, generator=gen, device=dev, dtype=torch.float32).to(dt)
    s.q_norm = s.k_norm = None
    if case["norm"]:
        s.q_norm, s.k_norm = (1.0 + 0.25 * (2 * torch.rand(2, D, generator=gen, device=dev) - 1)).to(dt)
    s.eps = 1e-6
    s.out = torch.zeros(rows, n_q, D, dtype=dt, device=dev)


def _prepare_attention(case, s, gen, dev):
    n_q, n_kv, page, dt = case["n_q"], case["n_kv"], case["page"], DTYPES[case["dtype"]]
    new, cached = _attention_lengths(case)
    total = [n + c for n, c in zip(new, cached)]
    pages = [_pages(n, page) for n in total]
    pool = sum(pages) + 5
    s.max_new, s.max_len = max(new), max(total)
    s.window, s.sinks = case["window"], case["sinks"]

    def indptr(v):
        t = torch.zeros(len(v) + 1, dtype=torch.int64)
        t[1:] = torch.cumsum(torch.tensor(v), 0)
        return t.to(torch.int32).to(dev)

    s.qo_indptr, s.kv_indptr = indptr(new), indptr(pages)
    s.kv_indices = torch.randperm(pool, generator=gen, device=dev)[: sum(pages)].to(torch.int32)
    s.last_page_len = torch.tensor([n - (p - 1) * page for n, p in zip(total, pages)], dtype=torch.int32, device=dev)
    rows = sum(new) + case["pad"]
    # rows as QK norm and rotation leave them: of length sqrt(128), a few positions with larger weights
    s.q = (1.3 * torch.randn(rows, n_q, D, generator=gen, device=dev)).to(dt)
    s.k_cache = torch.randn(pool, page, n_kv, D, generator=gen, device=dev, dtype=dt)
    s.v_cache = torch.randn(pool, page, n_kv, D, generator=gen, device=dev, dtype=dt)
    s.out = torch.zeros(rows, n_q, D, dtype=dt, device=dev)
    s.lse = torch.zeros(rows, n_q, dtype=torch.float32, device=dev)


def _prepare_sample(case, s, gen, dev):
    R, V, chunk = case["requests"], case["vocab"], case["chunk"]
    # requests that were fed nothing, one token, or a chunk: a row of logits per token
    fed = [1 + (i * 3) % chunk if not (chunk > 1 and i % 13 == 12) else 0 for i in range(R)]
    qo = torch.zeros(R + 1, dtype=torch.int64)
    qo[1:] = torch.cumsum(torch.tensor(fed), 0)
    s.qo_indptr = qo.to(torch.int32).to(dev)
    T = max(1, int(qo[-1]))
    # a broad bulk and, as a trained model has them, a few tokens far above it
    logits = 1.8 * torch.randn(T, V, generator=gen, device=dev)
    top = torch.randint(0, V, (T, 40), generator=gen, device=dev)
    logits.scatter_(1, top, 9.0 + 4.0 * torch.randn(T, 40, generator=gen, device=dev))
    s.logits = logits.to(DTYPES[case["dtype"]])
    s.u = torch.rand(R, generator=gen, device=dev)

    def per_request(*choices):
        pick = torch.randint(0, len(choices), (R,), generator=gen, device=dev)
        return torch.tensor(choices, device=dev)[pick]

    mode = case["mode"]
    temperatures = (0.0, 0.6, 0.8, 1.0, 1.3) if mode == "mixed" else (0.7, 1.0)
    s.temperature = per_request(*temperatures)
    s.top_k = per_request(*((0, 20, 50, 1000) if mode == "mixed" else (20, 50) if "top_k" in mode else (0, 0))).to(torch.int32)
    s.top_p = per_request(*((1.0, 0.95, 0.8) if mode == "mixed" else (0.95, 0.9) if "top_p" in mode else (1.0, 1.0)))
    s.min_p = per_request(*((0.0, 0.0, 0.05) if mode == "mixed" else (0.02, 0.1) if mode == "min_p" else (0.0, 0.0)))


def prepare(case, seed):
    dev = torch.device("cuda")
    s = _State()
    s.kind = case["kind"]
    gen = torch.Generator(device=dev).manual_seed(seed)
    {"plan": _prepare_plan, "append": _prepare_append, "attention": _prepare_attention, "sample": _prepare_sample}[s.kind](case, s, gen, dev)
    return s


# ------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------
def _own(s):
    import fleet_chiplet_megakernel_b200 as mk

    if s.kind == "plan":
        if not isinstance(s.plan, mk.StepPlan):
            s.plan = mk.StepPlan(**s.plan)
        p = mk.plan_step(s.lengths, s.new_tokens, s.block_table, s.free_pages, s.free_range, s.page, s.plan)
        return {"qo_indptr": p.qo_indptr, "kv_indptr": p.kv_indptr, "kv_indices": p.kv_indices, "last_page_len": p.last_page_len, "slots": p.slots,
                "positions": p.positions, "granted": p.granted, "free_range": p.free_range, "block_table": s.block_table, "free_pages": s.free_pages}
    if s.kind == "append":
        mk.rotate_append(s.q, s.k, s.v, s.cos, s.sin, s.positions, s.slots, s.k_cache, s.v_cache, q_norm=s.q_norm, k_norm=s.k_norm, eps=s.eps, out=s.out)
        return {"q": s.out, "k_cache": s.k_cache, "v_cache": s.v_cache}
    if s.kind == "attention":
        mk.chunk_attention(s.q, s.k_cache, s.v_cache, s.qo_indptr, s.kv_indptr, s.kv_indices, s.last_page_len, window=s.window, sinks=s.sinks,
                           out=s.out, lse=s.lse, max_new=s.max_new)
        return {"out": s.out, "lse": s.lse}
    tokens, logprobs = mk.sample_tokens(s.logits, s.u, temperature=s.temperature, top_k=s.top_k, top_p=s.top_p, min_p=s.min_p, qo_indptr=s.qo_indptr,
                                        return_logprobs=True)
    return {"tokens": tokens, "logprobs": logprobs}


# ------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------
def _plain_plan(s):
    """Requests take pages and token rows in order.  One that does not get all its pages or rows gets nothing, and those
    behind it that need pages (or rows) neither; the pages of ended requests go to the ring's tail first."""
    page, p = s.page, s.plan
    length, new = s.lengths.long().clamp_min(0), s.new_tokens.long()
    R, M = s.block_table.shape
    ring, T = s.free_pages.numel(), p["slots"].numel()
    dev = length.device
    held = (length + page - 1) // page
    ended = new < 0
    col = torch.arange(M, device=dev)
    head, tail = s.free_range[0], s.free_range[1]
    # ended requests: their pages behind the tail
    back = torch.where(ended, held, 0)
    first = torch.cumsum(back, 0) - back
    give = col < back[:, None]
    at = torch.where(give, (tail + first[:, None] + col) % ring, ring)
    grown = torch.cat((s.free_pages, s.free_pages.new_zeros(1)))
    grown.scatter_(0, at.flatten(), s.block_table.flatten())
    s.free_pages.copy_(grown[:ring])
    tail = tail + back.sum()
    # pages for the others
    want = torch.where(ended, 0, new)
    after = (length + want + page - 1) // page
    valid = (want > 0) & (after <= M)
    need = torch.where(valid, after - held, 0)
    upto = torch.cumsum(need, 0)
    fits = valid & ((need == 0) | (upto <= tail - head))
    rows = torch.cumsum(torch.where(fits, want, 0), 0)
    granted = torch.where(fits & (rows <= T), want, 0)
    served = granted > 0
    need = torch.where(served, need, 0)
    before = torch.cumsum(need, 0) - need
    grow = (col >= held[:, None]) & (col < (held + need)[:, None])
    page_of = s.free_pages[((head + before[:, None] + col - held[:, None]) % ring)]
    s.block_table.copy_(torch.where(grow, page_of, s.block_table))
    # index pointers
    kv_len = torch.where(ended, 0, length + granted)
    pages = torch.where(ended, 0, held + need)
    p["granted"].copy_(granted)
    p["qo_indptr"][1:] = torch.cumsum(granted, 0)
    p["kv_indptr"][1:] = torch.cumsum(pages, 0)
    p["last_page_len"].copy_(torch.where(pages > 0, kv_len - (pages - 1) * page, 0))
    p["free_range"][0], p["free_range"][1] = head + need.sum(), tail
    kv_first = torch.cumsum(pages, 0) - pages
    n = p["kv_indices"].numel()
    to = torch.where(col < pages[:, None], (kv_first[:, None] + col).clamp_max(n), n)
    grown = torch.cat((p["kv_indices"], p["kv_indices"].new_zeros(1)))
    grown.scatter_(0, to.flatten(), s.block_table.flatten())
    p["kv_indices"].copy_(grown[:n])
    # slot and position of every new token, rows behind the last one -1 and 0
    t = torch.arange(T, device=dev)
    ends = torch.cumsum(granted, 0)
    r = torch.searchsorted(ends, t, right=True).clamp_max(R - 1)
    live = t < ends[-1]
    pos = torch.where(live, length[r] + t - (ends - granted)[r], 0)
    p["positions"].copy_(pos)
    p["slots"].copy_(torch.where(live, s.block_table[r, (pos // page).clamp_max(M - 1)].long() * page + pos % page, -1))
    return dict(p, block_table=s.block_table, free_pages=s.free_pages)


def _plain_append(s):
    def rotated(x, norm):
        x = x.float()
        if norm is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s.eps) * norm.float()
        cos, sin = s.cos[s.positions.long()].float()[:, None], s.sin[s.positions.long()].float()[:, None]
        return x * cos + torch.cat((-x[..., D // 2:], x[..., : D // 2]), -1) * sin

    n_kv = s.k.shape[1]
    live = s.slots >= 0
    s.out.copy_(torch.where(live[:, None, None], rotated(s.q, s.q_norm).to(s.out.dtype), s.out))
    for cache, rows in ((s.k_cache, rotated(s.k, s.k_norm).to(s.k_cache.dtype)), (s.v_cache, s.v)):
        flat = cache.view(-1, n_kv * D)
        grown = torch.cat((flat, flat[:1]))  # rows without a slot go to a row of their own behind the cache
        grown.scatter_(0, torch.where(live, s.slots, flat.shape[0])[:, None].expand(-1, n_kv * D), rows.reshape(-1, n_kv * D))
        flat.copy_(grown[:-1])
    return {"q": s.out, "k_cache": s.k_cache, "v_cache": s.v_cache}


def _plain_attention(s):
    T, n_q, _ = s.q.shape
    _, page, n_kv, _ = s.k_cache.shape
    dev = s.q.device
    qo, kv = s.qo_indptr.long(), s.kv_indptr.long()
    R = qo.numel() - 1
    n = qo[1:] - qo[:-1]
    length = (kv[1:] - kv[:-1] - 1) * page + s.last_page_len
    j = torch.arange(s.max_len, device=dev)
    there = j < length[:, None]
    at = torch.where(there, kv[:-1, None] + j // page, 0)
    slot = s.kv_indices[at].long() * page + j % page
    k = s.k_cache.view(-1, n_kv, D)[slot].float().permute(0, 2, 3, 1)  # [R, kv head, D, position]
    v = torch.where(there[:, :, None, None], s.v_cache.view(-1, n_kv, D)[slot].float(), 0.0).transpose(1, 2)
    i = torch.arange(s.max_new, device=dev)
    q = s.q[(qo[:-1, None] + i).clamp_max(T - 1)].float()
    q = q.view(R, s.max_new, n_kv, n_q // n_kv, D).permute(0, 2, 1, 3, 4).reshape(R, n_kv, -1, D)
    p = (length - n)[:, None] + i  # position of every query
    sees = there[:, None, :] & (j <= p[:, :, None])
    if s.window:
        sees &= (j > p[:, :, None] - s.window) | (j < s.sinks)
    score = (q @ k).mul_(1.0 / math.sqrt(D)).view(R, n_kv, s.max_new, -1, s.max_len)
    score.masked_fill_(~sees[:, None, :, None, :], -math.inf)
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    w = score.sub_(m).exp_()
    total = w.sum(-1, keepdim=True)
    o = w.view(R, n_kv, -1, s.max_len) @ v
    o = torch.where(total > 0, o.view(R, n_kv, s.max_new, -1, D) / total, 0.0)
    lse = (m + total.log()).squeeze(-1)
    # rows of the batch; those behind the last sequence stay as they are
    t = torch.arange(T, device=dev)
    r = torch.searchsorted(qo[1:], t, right=True).clamp_max(R - 1)
    c = (t - qo[r]).clamp(0, s.max_new - 1)
    live = t < qo[-1]
    s.out.copy_(torch.where(live[:, None, None], o[r, :, c].reshape(T, n_q, D).to(s.out.dtype), s.out))
    s.lse.copy_(torch.where(live[:, None], lse[r, :, c].reshape(T, n_q), s.lse))
    return {"out": s.out, "lse": s.lse}


def _plain_sample(s):
    """Weights exp((l - max) / temperature) in 64 bits; top-k, top-p and min-p each keep a prefix of the order by logit
    (ties by index); the token is the first, by index, at which the kept weights' running sum exceeds u times their sum."""
    q0, q1 = s.qo_indptr[:-1].long(), s.qo_indptr[1:].long()
    V = s.logits.shape[1]
    l = s.logits[(q1 - 1).clamp_min(0)].double()
    t = s.temperature.double()[:, None]
    m = l.amax(1, keepdim=True)
    w = ((l - m) / torch.where(t > 0, t, 1.0)).exp()
    order = torch.sort(l, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(V, device=l.device)
    k = s.top_k.long()[:, None]
    ws = torch.where((rank < k) | (k <= 0), ws, 0.0)
    c = torch.cumsum(ws, 1)
    p = s.top_p.double()[:, None]
    keep = (ws > 0) & ((c - ws < p * c[:, -1:]) | (p >= 1) | (rank == 0)) & (ws >= s.min_p.double()[:, None])
    keep &= (t > 0) | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    c = torch.cumsum(torch.where(kept, w, 0.0), 1)
    total = c[:, -1:]
    token = (c > s.u.double()[:, None] * total).to(torch.int8).argmax(1)
    logprob = (w.gather(1, token[:, None]) / total).log().squeeze(1)
    fed = q1 > q0
    return {"tokens": torch.where(fed, token, -1), "logprobs": torch.where(fed, logprob, -math.inf).float()}


def run(state):
    if own:
        return _own(state)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[state.kind](state)


# ------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------
def _exact_append(s):
    def turn(x, norm):
        x = x.double()
        if norm is not None:
            x = norm.double() * x / (x.pow(2).sum(-1, keepdim=True) / D + s.eps).sqrt()
        half = D // 2
        a, b = x[..., :half], x[..., half:]
        c, n = s.cos.double()[s.positions.long(), None], s.sin.double()[s.positions.long(), None]
        return torch.cat((a * c[..., :half] - b * n[..., :half], b * c[..., half:] + a * n[..., half:]), -1)

    q, k, v = s.out.double(), s.k_cache.double(), s.v_cache.double()
    live = torch.nonzero(s.slots >= 0).flatten()
    q[live] = turn(s.q, s.q_norm)[live]
    k.view(-1, *k.shape[2:])[s.slots[live]] = turn(s.k, s.k_norm)[live]
    v.view(-1, *v.shape[2:])[s.slots[live]] = s.v.double()[live]
    return {"q": q, "k_cache": k, "v_cache": v}


def _exact_attention(s):
    out, lse = s.out.double(), s.lse.double()
    n_kv, page = s.k_cache.shape[2], s.k_cache.shape[1]
    per = s.q.shape[1] // n_kv
    qo, kv, last = s.qo_indptr.tolist(), s.kv_indptr.tolist(), s.last_page_len.tolist()
    for r in range(len(last)):
        n, pages = qo[r + 1] - qo[r], s.kv_indices[kv[r]:kv[r + 1]].long()
        length = (len(pages) - 1) * page + last[r]
        k = s.k_cache[pages].flatten(0, 1)[:length].double()
        v = s.v_cache[pages].flatten(0, 1)[:length].double()
        at = torch.arange(length - n, length, device=k.device)[:, None]
        j = torch.arange(length, device=k.device)[None, :]
        hidden = j > at
        if s.window:
            hidden |= (j <= at - s.window) & (j >= s.sinks)
        for h in range(n_kv):  # one kv head at a time: scores in 64 bits are large
            q = s.q[qo[r]:qo[r + 1], h * per:(h + 1) * per].double()
            score = torch.einsum("thd,jd->htj", q, k[:, h]) / math.sqrt(D)
            score.masked_fill_(hidden, -math.inf)
            l = torch.logsumexp(score, -1)
            o = torch.einsum("htj,jd->thd", score.sub_(l[..., None]).exp_(), v[:, h])
            out[qo[r]:qo[r + 1], h * per:(h + 1) * per] = o
            lse[qo[r]:qo[r + 1], h * per:(h + 1) * per] = l.T
    return {"out": out, "lse": lse}


def _exact_sample(s):
    qo = s.qo_indptr.tolist()
    tokens, logprobs = [], []
    for r in range(len(qo) - 1):
        if qo[r + 1] == qo[r]:
            tokens.append(-1)
            logprobs.append(-math.inf)
            continue
        l = s.logits[qo[r + 1] - 1].double()
        t, k, p, least = float(s.temperature[r]), int(s.top_k[r]), float(s.top_p[r]), float(s.min_p[r])
        if t <= 0:
            tokens.append(int((l == l.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        by = torch.argsort(l, descending=True, stable=True)
        if k > 0:
            by = by[:k]
        w = torch.exp((l[by] - l.max()) / t)
        n = len(w)
        if p < 1:
            before = torch.cat((w.new_zeros(1), torch.cumsum(w, 0)[:-1]))
            n = max(1, int((before < p * w.sum()).sum()))
        n = min(n, int((w >= least).sum()))
        by, w = by[:n], w[:n]
        by, turn = by.sort()
        w = w[turn]
        c = torch.cumsum(w, 0)
        i = int((c <= float(s.u[r]) * c[-1]).sum())
        tokens.append(int(by[i]))
        logprobs.append(math.log(float(w[i] / c[-1])))
    return {"tokens": torch.tensor(tokens), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers only
    return {"append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](prepare(case, seed))


# ------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "plan":
        cached, new = _plan_lengths(case)
        page = case["page"]
        held = sum(_pages(n, page) for n in cached)
        pages = sum(_pages(n + t, page) for n, t in zip(cached, new) if t >= 0)
        tokens = sum(max(0, t) for t in new) + 5
        # lengths, new tokens and held pages in; pages, index pointers, last pages, grants, slots and positions out
        return {"bytes": 4.0 * (2 * len(cached) + held + pages + 4 * len(cached) + 2) + 12.0 * tokens, "flops": 0.0}
    if case["kind"] == "append":
        T, heads = case["tokens"], case["n_q"] + 2 * case["n_kv"]
        return {"bytes": T * (4.0 * heads * D + 4.0 * D + 12) + 8.0 * case["pad"], "flops": 8.0 * T * (case["n_q"] + case["n_kv"]) * D}
    if case["kind"] == "attention":
        new, cached = _attention_lengths(case)
        w, sinks = case["window"], case["sinks"]
        seen = rows = 0.0
        for n, c in zip(new, cached):
            if not w:
                seen += n * c + n * (n + 1) / 2
                rows += n + c
                continue
            for p in range(c, c + n):
                seen += min(p + 1, w) + max(0, min(sinks, p + 1 - w))
            rows += min(n + c, n + w - 1 + sinks)
        q = sum(new) * case["n_q"]
        return {"bytes": 4.0 * rows * case["n_kv"] * D + q * (4.0 * D + 4), "flops": 4.0 * D * case["n_q"] * seen}
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": float(case["requests"]) * (case["vocab"] * size + 32), "flops": 4.0 * case["requests"] * case["vocab"]}
