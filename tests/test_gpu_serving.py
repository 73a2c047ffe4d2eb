"""The operators of a serving step against plain implementations in 64 bits: ``plan_step``, ``rotate_append``, ``chunk_attention``,
``sample_tokens``.

Tolerances.  A rounding to the 16-bit type is off by at most half a step, h = finfo.eps / 2 relative to the value.  fp32 sums of n
terms are off by less than n 2^-24 times the sum of the magnitudes.  Attention: a score is a sum of 128 products and its weight is off by the
factor exp(d), d <= 130 * 2^-24 * scale * sum |q k|; the sum of weights and the weighted sum of V add positions * 2^-24 each, and weights
enter the second product rounded to the 16-bit type (h).  With A = sum w |v| / sum w the output is off by at most
h |out| + (h + 2 max(d) + 2 positions 2^-24) A, the logarithm of the sum of weights by max(d) + positions 2^-24 + 2^-22 (|lse| + 1)."""
import math

import pytest
import torch

import fleet_chiplet_megakernel_b200 as mk

pytestmark = pytest.mark.gpu
D = 128
BF, FP = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rnd(g, *shape, dtype=BF, scale=1.0):
    return (scale * torch.randn(*shape, generator=g, device="cuda")).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------
# plan_step
# ------------------------------------------------------------------------------------
def plan_reference(lengths, new, table, ring, free, page, tokens_max, width):
    """The definition, request by request.  table: list of page lists; ring: list; free: (head, tail)."""
    head, tail = free
    ring, table = list(ring), [list(t) for t in table]
    P = len(ring)
    held = [-(-n // page) for n in lengths]
    for r, t in enumerate(new):
        if t < 0:
            for k in range(held[r]):
                ring[tail % P] = table[r][k]
                tail += 1
    granted, pages, slots, positions = [], [], [], []
    left, rows, blocked_pages, blocked_rows = tail - head, 0, False, False
    for r, t in enumerate(new):
        g = 0
        after = -(-(lengths[r] + max(t, 0)) // page)
        if t > 0 and after <= width:
            need = after - held[r]
            if need and (blocked_pages or need > left):
                blocked_pages = True  # nobody behind it gets pages either
            elif blocked_rows or rows + t > tokens_max:
                blocked_rows = True
                left -= need
            else:
                g = t
                rows += t
                left -= need
                for k in range(held[r], after):
                    table[r][k] = ring[head % P]
                    head += 1
        granted.append(g)
        n = 0 if t < 0 else lengths[r] + g
        mine = table[r][: -(-n // page)]
        pages.append(mine)
        for pos in range(lengths[r], lengths[r] + g):
            slots.append(table[r][pos // page] * page + pos % page)
            positions.append(pos)
    last = [(0 if not p else (lengths[r] + granted[r]) - (len(p) - 1) * page) for r, p in enumerate(pages)]
    return granted, pages, last, slots, positions, table, ring, (head, tail)


def run_plan(lengths, new, page, spare, tokens_max, width_more=1, wrap=5, strided=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    P = max(1, sum(held) + spare)
    perm = torch.randperm(P, generator=g).tolist()
    width = max(-(-(n + max(t, 0)) // page) for n, t in zip(lengths, new)) + width_more
    width = max(width, 1)
    table, at = [], 0
    for h in held:
        table.append(perm[at:at + h] + [-7] * (width - h))
        at += h
    head = 3 * P + wrap
    ring = [-9] * P
    for k, pg in enumerate(perm[at:]):
        ring[(head + k) % P] = pg
    free = (head, head + len(perm) - at)
    want = plan_reference(lengths, new, table, ring, free, page, tokens_max, width)

    R = len(lengths)
    bt = torch.full((R, width + 3), 99, dtype=torch.int32, device="cuda")
    view = bt[:, :width] if strided else torch.empty(R, width, dtype=torch.int32, device="cuda")
    view.copy_(torch.tensor(table, dtype=torch.int32))
    rt, fr = i32(ring), torch.tensor(free, dtype=torch.int64, device="cuda")
    plan = mk.StepPlan.empty(R, tokens_max, P)
    plan.kv_indices.fill_(-5)
    for again in range(2):  # the same call gives the same plan
        mk.plan_step(i32(lengths), i32(new), view, rt, fr, page, plan)
    granted, pages, last, slots, positions, table, ring, free = want
    assert plan.granted.tolist() == granted
    qo, kv = [0], [0]
    for a, b in zip(granted, pages):
        qo.append(qo[-1] + a)
        kv.append(kv[-1] + len(b))
    assert plan.qo_indptr.tolist() == qo and plan.kv_indptr.tolist() == kv
    flat = sum(pages, [])
    assert plan.kv_indices.tolist() == flat + [-5] * (P - len(flat))
    assert plan.last_page_len.tolist() == last
    assert plan.slots.tolist() == slots + [-1] * (tokens_max - len(slots))
    assert plan.positions.tolist() == positions + [0] * (tokens_max - len(positions))
    assert view.tolist() == table and rt.tolist() == ring
    assert plan.free_range.tolist() == list(free) and fr.tolist() == [head, head + P - sum(held)]
    if strided:
        assert bool((bt[:, width:] == 99).all())


@pytest.mark.parametrize("page", [1, 8, 16, 24, 64])
@pytest.mark.parametrize("lengths,new", [
    ([0], [1]), ([0], [0]), ([5], [-1]), ([63], [1]), ([64], [1]), ([0, 0, 0], [130, 1, 64]), ([1000], [1]),
    ([10, 64, 0, 127, 128, 3], [1, 1, 70, 1, 1, 0]), ([10, 64, 0, 127, 128, 3], [-1, 1, -1, 1, 200, -1]),
    ([33] * 40, [1] * 40), (list(range(70)), [(-1 if i % 5 == 0 else i % 7) for i in range(70)])])
def test_plan_against_the_definition(lengths, new, page):
    spare = sum(-(-max(0, t) // page) + 1 for t in new)
    total = max(1, sum(max(0, t) for t in new))
    run_plan(lengths, new, page, spare, total + 3)
    run_plan(lengths, new, page, spare, total, strided=True, wrap=0, seed=1)


@pytest.mark.parametrize("spare", [0, 1, 2, 5, 9])
def test_plan_when_pages_run_out(spare):
    run_plan([16, 3, 16, 32, 5, 16, 48], [1, 1, 1, 1, 40, 1, 2], 16, spare, 100)
    # what ended requests give back is used in the same step
    run_plan([16, 3, 40, 32, 5, 16, 48], [1, 1, -1, 1, 40, -1, 2], 16, spare, 100, wrap=1)


@pytest.mark.parametrize("budget", [1, 2, 5, 43])
def test_plan_when_token_rows_run_out(budget):
    run_plan([16, 3, 16, 32, 5, 16, 48], [1, 1, 1, 1, 40, 1, 2], 16, 20, budget)


def test_plan_where_a_table_row_is_too_short():
    run_plan([16, 3, 30], [1, 30, 1], 16, 9, 50, width_more=-1)


def test_plan_of_more_tokens_than_there_are_positions():
    """A request for as many tokens as an int holds, on pages of one token, is granted nothing and takes nothing from those behind it."""
    for page in (1, 2):
        lengths, new = i32([9, 4, 3]), i32([2 ** 31 - 1, 2, 5])
        table = torch.full((3, 12), -7, dtype=torch.int32, device="cuda")
        held = [-(-n // page) for n in (9, 4, 3)]
        for r, h in enumerate(held):
            table[r, :h] = torch.arange(h, dtype=torch.int32, device="cuda") + 20 * r
        plan = mk.StepPlan.empty(3, 16, 40)
        after = [-(-n // page) for n in (9, 6, 8)]
        free = sum(after) - sum(held) - 1  # one page too few for the last
        mk.plan_step(lengths, new, table, i32(list(range(100, 110))), torch.tensor([0, free], device="cuda"), page, plan)
        assert plan.granted.tolist() == [0, 2, 0] and plan.qo_indptr.tolist() == [0, 0, 2, 2]
        assert plan.free_range.tolist() == [after[1] - held[1], free]
        assert plan.positions.tolist() == [4, 5] + [0] * 14


def test_plan_with_a_page_index_that_is_too_short():
    """The index ends where its tensor ends; tables, slots and positions are those of the whole step."""
    plan, short = mk.StepPlan.empty(2, 8, 12), mk.StepPlan.empty(2, 8, 3)
    tables = []
    for p in (plan, short):
        table = torch.tensor([[0, 1, -7, -7], [2, 3, -7, -7]], dtype=torch.int32, device="cuda")
        mk.plan_step(i32([8, 7]), i32([2, 6]), table, i32([9, 8, 7]), torch.tensor([0, 3], device="cuda"), 4, p)
        tables.append(table)
    assert tables[0].tolist() == [[0, 1, 9, -7], [2, 3, 8, 7]] and torch.equal(tables[0], tables[1])
    assert plan.kv_indices.tolist() == [0, 1, 9, 2, 3, 8, 7] + [0] * 5 and short.kv_indices.tolist() == [0, 1, 9]
    assert torch.equal(plan.slots, short.slots) and torch.equal(plan.positions, short.positions) and torch.equal(plan.free_range, short.free_range)


def test_plan_many_requests():
    new = [(-1 if i % 31 == 7 else i % 3) for i in range(2500)]
    run_plan([(i * 37) % 300 for i in range(2500)], new, 16, 2000, 2600)


# ------------------------------------------------------------------------------------
# rotate_append
# ------------------------------------------------------------------------------------
def rotate_reference(x, norm, eps, cos, sin, pos):
    x = x.double()
    size = x.abs()
    if norm is not None:
        f = norm.double() / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        x, size = x * f, size * f.abs()
    c, s = cos.double()[pos.long(), None], sin.double()[pos.long(), None]
    turned = torch.cat((-x[..., 64:], x[..., :64]), -1)
    size = size * c.abs() + torch.cat((size[..., 64:], size[..., :64]), -1) * s.abs()
    return x * c + turned * s, size


def close_rounded(got, want, size, what):
    """One rounding to the 16-bit type, and some 150 fp32 roundings (a sum of 128 squares, its root, four products) in front of it."""
    t = torch.finfo(got.dtype)
    off = (got.double() - want).abs()
    assert bool((off <= t.eps / 2 * want.abs() * (1 + 2.0 ** -8) + 160 * 2.0 ** -24 * size + t.smallest_normal * t.eps).all()), f"{what}: off by {float(off.max())}"


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("tokens,n_q,n_kv,page,norm,tables,layout", [
    (1, 4, 2, 64, True, "same", "fused"), (3, 32, 8, 16, True, "same", "fused"), (17, 8, 8, 1, False, "fp32", "apart"), (130, 14, 2, 24, True, "fp32", "odd"),
    (64, 5, 1, 64, True, "same", "odd"), (7, 1, 1, 8, False, "same", "expanded")])
def test_rotate_append_against_the_definition(dtype, tokens, n_q, n_kv, page, norm, tables, layout):
    g = gen(tokens)
    pad = 5
    rows = tokens + pad
    if layout == "fused":
        q, k, v = (x.view(rows, -1, D) for x in rnd(g, rows, (n_q + 2 * n_kv) * D, dtype=dtype).split([n_q * D, n_kv * D, n_kv * D], 1))
    elif layout == "odd":  # rows that start at no multiple of 16 bytes
        q, k, v = (rnd(g, rows, n, D + 3, dtype=dtype)[..., 1:D + 1] for n in (n_q, n_kv, n_kv))
    elif layout == "expanded":
        q, k, v = (rnd(g, 1, n, D, dtype=dtype).expand(rows, n, D) for n in (n_q, n_kv, n_kv))
    else:
        q, k, v = (rnd(g, n, rows, D, dtype=dtype).transpose(0, 1) for n in (n_q, n_kv, n_kv))
    td = torch.float32 if tables == "fp32" else dtype
    ang = torch.rand(300, D, generator=g, device="cuda") * 6
    cos, sin = ang.cos().to(td), ang.sin().to(td)
    qn, kn = (rnd(g, D, dtype=dtype) for _ in range(2)) if norm else (None, None)
    pages = -(-tokens // page) + 2
    kc, vc = (rnd(g, 2, pages, page, n_kv, D, dtype=dtype)[1] for _ in range(2))
    slots = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    slots[:tokens] = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    pos = torch.randint(0, 300, (rows,), generator=g, device="cuda", dtype=torch.int32)
    slots[tokens + 1], pos[tokens + 2], slots[tokens + 3] = pages * page, 300, 1 << 40
    slots[tokens + 2] = -2
    want_k, want_v = kc.clone(), vc.clone()
    out = rnd(g, rows, n_q, D, dtype=dtype)
    kept = out.clone()
    mk.rotate_append(q, k, v, cos, sin, pos, slots, kc, vc, qn, kn, eps=1e-6, out=out)
    live, p = slice(0, tokens), pos[:tokens]
    ref, size = rotate_reference(q[live], qn, 1e-6, cos, sin, p)
    close_rounded(out[live], ref, size, "q")
    assert torch.equal(out[tokens:], kept[tokens:])
    ref, size = rotate_reference(k[live], kn, 1e-6, cos, sin, p)
    close_rounded(kc.flatten(0, 1)[slots[live]], ref, size, "k")
    want_v.view(-1, n_kv, D)[slots[live]] = v[live]
    assert torch.equal(vc, want_v)
    free = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    free[slots[live]] = False
    assert torch.equal(kc.view(-1, n_kv, D)[free], want_k.view(-1, n_kv, D)[free])


def test_rotate_append_position_and_slot_bounds():
    """A token whose position has no row in the tables, or whose slot no row in the cache, changes nothing."""
    g = gen(0)
    q, k, v = (rnd(g, 3, 2, D) for _ in range(3))
    cos = sin = torch.ones(4, D, device="cuda", dtype=BF)
    kc, vc, out = torch.zeros(1, 2, 2, D, device="cuda", dtype=BF), torch.zeros(1, 2, 2, D, device="cuda", dtype=BF), torch.zeros(3, 2, D, device="cuda", dtype=BF)
    mk.rotate_append(q, k, v, cos, sin, i32([4, -1, 0]), torch.tensor([0, 1, 2], device="cuda"), kc, vc, out=out)
    assert not kc.any() and not vc.any() and not out.any()


def test_rotate_append_in_place():
    g = gen(3)
    x = rnd(g, 70, 10 * D).view(70, 10, D)
    q, k, v = x.split([6, 2, 2], 1)
    ang = torch.rand(80, D, generator=g, device="cuda")
    args = (ang.cos(), ang.sin(), torch.arange(70, device="cuda", dtype=torch.int32), torch.arange(70, device="cuda"))
    caches = [torch.zeros(5, 16, 2, D, device="cuda", dtype=BF) for _ in range(4)]
    want = mk.rotate_append(q, k, v, *args, *caches[:2], rnd(g, D), rnd(g, D), 1e-6)
    g2 = gen(3)
    rnd(g2, 70, 10 * D), torch.rand(80, D, generator=g2, device="cuda")
    kept = x[:, 6:].clone()
    assert mk.rotate_append(q, k, v, *args, *caches[2:], rnd(g2, D), rnd(g2, D), 1e-6, out=q) is q
    assert torch.equal(q, want) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3]) and torch.equal(x[:, 6:], kept)


# ------------------------------------------------------------------------------------
# chunk_attention
# ------------------------------------------------------------------------------------
class Batch:
    """Requests of (cached, new) tokens over pages scattered over a pool; what is behind a request's last token holds NaN."""

    def __init__(self, requests, n_q, n_kv, page, dtype=BF, seed=0, pad=0, spoil=True, scale=1.0):
        g = gen(seed)
        self.n_q, self.n_kv, self.page, self.dtype, self.requests = n_q, n_kv, page, dtype, requests
        lens = [c + n for c, n in requests]
        pages = [-(-n // page) for n in lens]
        pool = sum(pages) + 3
        perm = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        self.k = rnd(g, pool, page, n_kv, D, dtype=dtype, scale=scale)
        self.v = rnd(g, pool, page, n_kv, D, dtype=dtype)
        self.kv_indices = perm[: sum(pages)].contiguous()
        qo, kv = [0], [0]
        for (_, n), p in zip(requests, pages):
            qo.append(qo[-1] + n)
            kv.append(kv[-1] + p)
        self.qo, self.kv = qo, kv
        self.qo_indptr, self.kv_indptr = i32(qo), i32(kv)
        self.last = i32([n - (p - 1) * page if p else 0 for n, p in zip(lens, pages)])
        if spoil:
            for r, n in enumerate(lens):
                if n % page:
                    pg = int(self.kv_indices[kv[r + 1] - 1])
                    self.k[pg, n % page:], self.v[pg, n % page:] = math.nan, math.inf
            for pg in perm[sum(pages):].tolist():
                self.k[pg], self.v[pg] = math.nan, math.nan
        self.q = rnd(g, qo[-1] + pad, n_q, D, dtype=dtype)
        self.out = rnd(g, qo[-1] + pad, n_q, D, dtype=dtype)
        self.lse = torch.full((qo[-1] + pad, n_q), 7.0, device="cuda")

    def run(self, **kw):
        return mk.chunk_attention(self.q, self.k, self.v, self.qo_indptr, self.kv_indptr, self.kv_indices, self.last, out=self.out, lse=self.lse, **kw)

    def reference(self, window=0, sinks=0, scale=D ** -0.5):
        """(out, lse, allowed error of out, of lse), rows of live tokens."""
        h = torch.finfo(self.dtype).eps / 2
        outs = []
        for r, (c, n) in enumerate(self.requests):
            if not n:
                continue
            pages = self.kv_indices[self.kv[r]:self.kv[r + 1]].long()
            k, v = (x[pages].flatten(0, 1)[: c + n].double().repeat_interleave(self.n_q // self.n_kv, 1) for x in (self.k, self.v))
            q = self.q[self.qo[r]:self.qo[r + 1]].double()
            at, j = torch.arange(c, c + n, device="cuda")[:, None], torch.arange(c + n, device="cuda")
            sees = j <= at
            if window:
                sees &= (j > at - window) | (j < sinks)
            s = torch.einsum("thd,jhd->htj", q, k) * scale
            size = torch.einsum("thd,jhd->htj", q.abs(), k.abs()) * abs(scale)
            s = s.masked_fill(~sees, -math.inf)
            d = 130 * 2.0 ** -24 * size.masked_fill(~sees, 0).amax(-1) + (c + n) * 2.0 ** -24  # [head, token]
            w = torch.softmax(s, -1)
            v = torch.where(sees.any(0)[:, None, None], v, 0.0)
            out = torch.einsum("htj,jhd->thd", w, v)
            mean = torch.einsum("htj,jhd->thd", w, v.abs())
            lse = torch.logsumexp(s, -1)
            outs.append((out, lse.T, h * out.abs() * (1 + h) + (h + 2 * d.T[..., None]) * mean + torch.finfo(self.dtype).smallest_normal, d.T + 2.0 ** -22 * (lse.T.abs() + 1)))
        return [torch.cat(x) for x in zip(*outs)]

    def check(self, **kw):
        before, lse_before = self.out.clone(), self.lse.clone()
        scale = kw.get("scale")
        want, lse, tol, lse_tol = self.reference(kw.get("window", 0), kw.get("sinks", 0), D ** -0.5 if scale is None else scale)
        assert self.run(**kw) is self.out
        n = self.qo[-1]
        off, lse_off = (self.out[:n].double() - want).abs(), (self.lse[:n].double() - lse).abs()
        assert bool((off <= tol).all()), f"out off by {float((off / tol).max())} of what is allowed"
        assert bool((lse_off <= lse_tol).all()), f"lse off by {float((lse_off / lse_tol).max())} of what is allowed"
        assert torch.equal(self.out[n:], before[n:]) and torch.equal(self.lse[n:], lse_before[n:])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n_q,n_kv,page", [(8, 2, 64), (4, 4, 16), (32, 4, 16), (14, 2, 8), (12, 4, 24), (40, 2, 1), (3, 1, 128)])
def test_attention_of_single_tokens(n_q, n_kv, page, dtype):
    Batch([(0, 1), (1, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (300, 1), (1211, 1)], n_q, n_kv, page, dtype, pad=2).check()


@pytest.mark.parametrize("cached", [0, 1, 127, 128, 4000])
@pytest.mark.parametrize("max_new", [0, 1])
def test_attention_of_one_request(cached, max_new):
    Batch([(cached, 1)], 8, 2, 64).check(max_new=max_new)


@pytest.mark.parametrize("requests", [250, 288, 300, 319, 320, 1000])
def test_attention_of_many_single_tokens(requests):
    """The table of the requests and the stages share the row kernel's shared memory."""
    Batch([((7 * i) % 50, 1) for i in range(requests)], 8, 2, 16).check()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("n_q,n_kv,page", [(8, 2, 64), (4, 4, 16), (32, 4, 8), (14, 2, 16), (12, 4, 24), (40, 2, 1), (16, 1, 128)])
@pytest.mark.parametrize("requests", [[(0, 2)], [(0, 33), (5, 7)], [(64, 64), (0, 1), (3, 0), (200, 129)], [(1000, 3), (0, 0), (0, 257), (31, 32)]])
def test_attention_of_chunks(requests, n_q, n_kv, page, dtype):
    Batch(requests, n_q, n_kv, page, dtype, pad=3).check()


@pytest.mark.parametrize("count", [31, 32, 33, 70])
def test_attention_of_many_chunks(count):
    """Requests of equal and of different lengths, empty ones and single tokens among them."""
    requests = [((13 * (i // 3)) % 200, (0, 1, 9, 33, 40, 90)[(5 * i) % 6 if i % 4 else i % 6]) for i in range(count)]
    Batch(requests, 8, 2, 16, pad=3).check()
    Batch(requests[::-1], 4, 4, 8, dtype=FP).check(window=40, sinks=3)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 4), (128, 4), (200, 130), (64, 1000), (5000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("requests", [[(700, 1), (0, 1), (15, 1), (129, 1)], [(0, 300), (500, 140), (90, 1)]])
def test_attention_with_window_and_sinks(requests, window, sinks):
    Batch(requests, 8, 2, 16).check(window=window, sinks=sinks)


def test_attention_scale_and_lengths():
    Batch([(513, 1), (40, 9)], 8, 8, 64).check(scale=0.3)
    Batch([(513, 1), (40, 90)], 8, 8, 64).check(scale=0.0)
    Batch([(20000, 1), (9000, 70)], 4, 2, 64).check()


@pytest.mark.parametrize("new", [1, 5, 200])
def test_attention_large_scores(new):
    """Scores of some hundreds: one position takes all weight, and its place moves along the row."""
    Batch([(700, new)], 8, 2, 64, scale=40.0).check()


@pytest.mark.parametrize("new", [2, 150])
def test_attention_values_that_are_not_finite_reach_only_rows_that_see_them(new):
    b = Batch([(300, new), (80, 2)], 8, 2, 16, spoil=False)
    at = 300 + new // 2  # position of a new token: rows before it do not see it
    page = int(b.kv_indices[at // 16])
    want, _, tol, _ = b.reference()  # (the rows that see neither value do not depend on them; a plain product with weight 0 would)
    b.v[page, at % 16, 1, 5] = math.inf
    b.k[page, at % 16, 0, 3] = math.nan
    b.run()
    hit = torch.zeros(b.qo[-1], 8, D, dtype=torch.bool, device="cuda")
    hit[new // 2:new, :4] = True        # NaN scores of kv head 0
    hit[new // 2:new, 4:, 5] = True     # an infinite value in one dim of kv head 1
    assert bool(torch.isfinite(b.out[: b.qo[-1]][~hit]).all())
    assert bool(b.out[new // 2:new, :4].isnan().all()) and bool((b.out[new // 2:new, 4:, 5] == math.inf).all())
    assert bool(((b.out[: b.qo[-1]].double() - want).abs() <= tol)[~hit].all())


@pytest.mark.parametrize("new", [1, 140])
def test_attention_rows_that_see_nothing(new):
    """More new rows than positions: the first rows have none, their outputs are zero; a request without pages likewise."""
    b = Batch([(0, new), (30, new)], 8, 2, 16)
    b.last[0] = 0 if new == 1 else new % 16 - 3  # three positions fewer than rows (none at all)
    gone = 3 if new > 1 else 1
    if new == 1:
        b.kv_indptr = i32([0, 0, b.kv[2] - b.kv[1]])
        b.kv_indices = b.kv_indices[b.kv[1]:].contiguous()
    b.run()
    assert not b.out[:gone].any() and bool((b.lse[:gone] == -math.inf).all())
    assert bool(b.out[gone:b.qo[-1]].isfinite().all()) and bool(b.out[gone:b.qo[-1]].any())


@pytest.mark.parametrize("new", [1, 140])
def test_attention_pages_and_pointers_out_of_range(new):
    """What the index tensors say is held against the tensors' sizes: outputs of such rows mean nothing, but all others are right and nothing faults."""
    b = Batch([(100, new), (77, new)], 8, 2, 16)
    b.kv_indices[b.kv[0] + 1], b.kv_indices[b.kv[0] + 2] = 10 ** 9, -3
    want, _, tol, _ = b.reference_of_last()
    b.run()
    assert bool(((b.out[b.qo[1]:].double() - want).abs() <= tol).all())
    b.qo_indptr, b.kv_indptr, b.last = i32([-5, 10 ** 9, 3]), i32([-1, 10 ** 9, 2]), i32([10 ** 9, -4])
    b.run()
    torch.cuda.synchronize()


def _reference_of_last(self):
    lone = object.__new__(Batch)
    lone.__dict__.update(self.__dict__, requests=[(0, 0)] * (len(self.requests) - 1) + [self.requests[-1]])
    return Batch.reference(lone)


Batch.reference_of_last = _reference_of_last


def test_attention_of_strided_tensors():
    """Caches of one layer out of a joint tensor, q out of a fused projection, an output with a pitch of its own."""
    for requests in ([(200, 1), (17, 1)], [(200, 150), (17, 1)]):
        b = Batch(requests, 8, 2, 16)
        joint = torch.full((b.k.shape[0], 3, 16, 2, 2, D), math.nan, dtype=BF, device="cuda")
        joint[:, 1, :, :, 0], joint[:, 1, :, :, 1] = b.k, b.v
        b.k, b.v = joint[:, 1, :, :, 0], joint[:, 1, :, :, 1]
        wide = torch.zeros(b.q.shape[0], 12, D, dtype=BF, device="cuda")
        wide[:, 2:10] = b.q
        b.q = wide[:, 2:10]
        b.out = torch.zeros(8, b.q.shape[0], D, dtype=BF, device="cuda").transpose(0, 1)
        b.lse = torch.zeros(8, b.q.shape[0], device="cuda").T
        b.check()


def far_apart(shape, dtype=BF):
    """Two caches whose pages are 2^30 elements apart, one between the other's."""
    pages, rest = shape[0], shape[1] * shape[2] * shape[3]
    pool = torch.empty((pages - 1) * 2 ** 30 + 2 ** 29 + rest, dtype=dtype, device="cuda")
    stride = (2 ** 30, shape[2] * shape[3], shape[3], 1)
    return pool.as_strided(shape, stride), pool.as_strided(shape, stride, 2 ** 29)


@pytest.mark.parametrize("requests", [[(200, 1), (17, 1)], [(130, 80), (17, 1)]])
def test_attention_over_a_cache_past_32_bits(requests):
    b = Batch(requests, 8, 2, 64)
    k, v = far_apart(b.k.shape)
    b.k, b.v = k.copy_(b.k), v.copy_(b.v)
    b.check()


def test_rotate_append_into_a_cache_past_32_bits():
    g = gen(1)
    kc, vc = far_apart((6, 16, 2, D))
    kc.zero_(), vc.zero_()
    x, cos, sin = rnd(g, 40, 8, D), torch.ones(40, D, device="cuda"), torch.zeros(40, D, device="cuda")
    slots = torch.randperm(96, generator=g, device="cuda")[:40]
    out = mk.rotate_append(x[:, :4], x[:, 4:6], x[:, 6:], cos, sin, torch.arange(40, device="cuda", dtype=torch.int32), slots, kc, vc)
    assert torch.equal(out, x[:, :4])  # (no rotation, no norm: as they were)
    for cache, rows in ((kc, x[:, 4:6]), (vc, x[:, 6:])):
        want = torch.zeros(96, 2, D, dtype=BF, device="cuda")
        want[slots] = rows
        assert torch.equal(cache.reshape(96, 2, D), want)


def test_sample_from_rows_past_32_bits():
    g = gen(2)
    near = rnd(g, 6, 5000, scale=2.0)
    pool = torch.empty(5 * 2 ** 30 + 5000, dtype=BF, device="cuda")
    logits = pool.as_strided((6, 5000), (2 ** 30, 1)).copy_(near)
    u = torch.rand(6, generator=g, device="cuda")
    for kw in ({}, {"top_k": 40}, {"top_p": 0.9}):
        assert torch.equal(mk.sample_tokens(logits, u, **kw), mk.sample_tokens(near, u, **kw))


def test_attention_is_the_same_each_time():
    for requests in ([(2000, 1)] * 3, [(700, 200), (9, 1)]):
        b = Batch(requests, 8, 2, 64)
        first = b.run().clone()
        for _ in range(3):
            assert torch.equal(b.run(), first)


# ------------------------------------------------------------------------------------
# sample_tokens
# ------------------------------------------------------------------------------------
def sample_reference(logits, u, t, k, p, m):
    l = logits.double()
    l = torch.where(l.isnan(), -math.inf, l)
    top = l.max()
    if top == -math.inf:
        return -1, -math.inf
    if t <= 0:
        return int((l == top).nonzero()[0]), 0.0
    by = torch.argsort(l, descending=True, stable=True)
    if 0 < k < len(by):
        by = by[:k]
    w = torch.where(l[by] == top, 1.0, torch.exp((l[by] - top) / torch.tensor(t, dtype=torch.float32).double().item()))
    n = len(w)
    if p < 1:
        before = torch.cat((w.new_zeros(1), torch.cumsum(w, 0)[:-1]))
        n = max(1, int((before < float(torch.tensor(p)) * w.sum()).sum()))
    n = min(n, int((w >= min(float(torch.tensor(m)), 1.0)).sum()))
    by, turn = by[:n].sort()
    w = w[:n][turn]
    c = torch.cumsum(w, 0)
    i = min(int((c <= float(u) * c[-1]).sum()), int((w > 0).nonzero()[-1]))
    return int(by[i]), math.log(float(w[i] / c[-1]))


def check_sample(logits, u, t, k, p, m, **kw):
    tokens, lp = mk.sample_tokens(logits, u, t, k, p, m, return_logprobs=True, **kw)
    tokens, lp = tokens.tolist(), lp.tolist()
    for r in range(len(u)):
        a = [x[r].item() if isinstance(x, torch.Tensor) else x for x in (t, k, p, m)]
        want, want_lp = sample_reference(logits[r], u[r], *a)
        assert tokens[r] == want, f"request {r}, settings {a}: token {tokens[r]}, {want} expected"
        # the weights' ratio in 64 bits, its logarithm rounded to fp32
        assert lp[r] == want_lp or abs(lp[r] - want_lp) <= 2.0 ** -23 * abs(want_lp) + 1e-12


@pytest.mark.parametrize("dtype", [BF, FP, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 2048, 32008, 151936])
@pytest.mark.parametrize("settings", [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.02),
                                      (2.5, 0, 0.999, 0.0), (0.01, 7, 0.5, 0.0), (1.0, 5000, 0.3, 1.0)])
def test_sample_against_the_definition(settings, vocab, dtype):
    g = gen(vocab)
    logits = rnd(g, 7, vocab, dtype=dtype, scale=3.0)
    u = torch.rand(7, generator=g, device="cuda")
    u[0], u[1] = 0.0, 1.0 - 2.0 ** -24
    check_sample(logits, u, *settings)


def test_sample_settings_per_request_and_many_rows():
    g = gen(3)
    for R, V in ((200, 5003), (64, 40001), (20, 151936)):
        pick = lambda *c: torch.tensor(c, device="cuda")[torch.randint(0, len(c), (R,), generator=g, device="cuda")]  # noqa: E731
        logits = rnd(g, R, V, dtype=torch.float32, scale=2.5)
        check_sample(logits, torch.rand(R, generator=g, device="cuda"), pick(0.0, 0.5, 1.0, 1.7), pick(0, 1, 3, 64, 2000, 10 ** 9).to(torch.int32),
                     pick(1.0, 0.99, 0.6, 0.0), pick(0.0, 0.01, 0.3))


@pytest.mark.parametrize("vocab", [7, 3000, 20000])
@pytest.mark.parametrize("kind", ["equal", "two_values", "lowest", "minus_inf", "plus_inf", "nan", "nothing", "zeros", "tiny", "steep"])
def test_sample_rows_that_are_hard_to_cut(kind, vocab):
    """Equal logits by the thousand, masked ones, infinities, NaN."""
    g = gen(vocab)
    l = rnd(g, 6, vocab, dtype=torch.float32, scale=2.0)
    if kind == "equal":
        l = torch.full_like(l, 1.5)
    elif kind == "two_values":
        l = torch.where(l > 0, 1.0, 0.5)
    elif kind == "lowest":
        l = torch.where(l > 1.0, l, torch.finfo(torch.float32).min)
    elif kind == "minus_inf":
        l = torch.where(l > 1.0, l, -math.inf)
        l[:, 0] = 0.0
    elif kind == "plus_inf":
        l[:, ::3] = math.inf
    elif kind == "nan":
        l[:, ::2] = math.nan
    elif kind == "nothing":
        l = torch.full_like(l, -math.inf)
        l[:, ::2] = math.nan
    elif kind == "zeros":
        l = torch.where(l > 0, 0.0, -0.0)
    elif kind == "tiny":
        l = l * 1e-40
    elif kind == "steep":
        l = l * 1e30
    u = torch.rand(6, generator=g, device="cuda")
    for settings in ((1.0, 0, 1.0, 0.0), (1.0, vocab // 2, 1.0, 0.0), (0.5, 0, 0.7, 0.0), (1.0, vocab - 1, 0.5, 0.1), (0.0, 3, 0.5, 0.0), (1.0, 2, 0.0, 0.0)):
        check_sample(l, u, *settings)


def test_sample_wide_spread_of_weights():
    """Rows whose border lies far down: most weight in few tokens and top_p next to 1."""
    g = gen(9)
    l = torch.cat((rnd(g, 4, 50, dtype=torch.float32, scale=1.0) + 30, rnd(g, 4, 60000, dtype=torch.float32, scale=4.0)), 1)
    u = torch.rand(4, generator=g, device="cuda")
    for p in (0.5, 0.99999, 1 - 2.0 ** -23, 1 - 2.0 ** -24):
        check_sample(l, u, 1.0, 0, p, 0.0)
        check_sample(l, u, 3.0, 0, p, 0.0)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("vocab", [5000, 40001, 151936])
@pytest.mark.parametrize("temperature,top_p,top_k", [(1.3, 0.95, 0), (1.0, 0.5, 0), (2.0, 0.9, 0), (1.0, 0.99, 20000), (0.5, 0.9, 3000), (1.0, 1 - 2.0 ** -20, 0)])
def test_sample_rows_that_keep_thousands(temperature, top_p, top_k, vocab, dtype):
    """Broad rows: top_p and top_k leave more tokens than one list holds."""
    g = gen(vocab + 1)
    logits = rnd(g, 4, vocab, dtype=dtype, scale=1.5)
    check_sample(logits, torch.rand(4, generator=g, device="cuda"), temperature, top_k, top_p, 0.0)


@pytest.mark.parametrize("dtype", [BF, FP, torch.float32])
@pytest.mark.parametrize("vocab", [900, 20000, 151936])
@pytest.mark.parametrize("rest", [-30.0, -20.0, -math.inf])
def test_sample_borders_that_are_too_close_for_32_bits(rest, vocab, dtype):
    """Eight equal weights and a rest that is 1e-13 to 3e-4 of them: the weights before the third, or the fifth, are the limit but for that."""
    g = gen(vocab)
    for top_p in (0.25, 0.5):
        logits = torch.full((16, vocab), rest, device="cuda")
        for r in range(16):
            logits[r, torch.randperm(vocab, generator=g, device="cuda")[:8]] = 3.0
        u = torch.arange(16, device="cuda") / 16 + 1 / 32
        check_sample(logits.to(dtype), u, 1.0, 0, top_p, 0.0)


def test_sample_of_the_last_rows_of_requests():
    g = gen(1)
    logits, u = rnd(g, 9, 5000, dtype=torch.float32, scale=2.0)[:, 7:4007], torch.rand(5, generator=g, device="cuda")
    qo = i32([0, 1, 1, 4, 9, 9])
    tokens, lp = mk.sample_tokens(logits, u, 0.9, 30, qo_indptr=qo, return_logprobs=True)
    for r, row in enumerate((0, None, 3, 8, None)):
        if row is None:
            assert int(tokens[r]) == -1 and float(lp[r]) == -math.inf
        else:
            assert int(tokens[r]) == sample_reference(logits[row], u[r], 0.9, 30, 1.0, 0.0)[0]
    # pointers outside the rows
    assert mk.sample_tokens(logits, u, qo_indptr=i32([0, 10, 11, -4, 2 ** 31 - 1, 5])).tolist()[:1] == [-1]
