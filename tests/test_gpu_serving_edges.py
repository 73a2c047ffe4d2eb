"""The serving operators at the edges of what their documentation allows: calls without rows or pages, vocabularies of millions, weights that a
16-bit type has no value for, positions next to 2^31, tangents, tensors that share memory, waits that run out."""
import ctypes as C
import math
import subprocess
import sys

import pytest
import torch

import fleet_chiplet_megakernel_b200 as mk
from fleet_chiplet_megakernel_b200 import _cabi
from tests.conftest import ROOT
from tests.test_gpu_serving import Batch, check_sample, gen, i32, rnd

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
D = 128


@pytest.mark.parametrize("top_p", [0.3, 0.513, 0.9])
def test_sample_from_a_vocabulary_of_millions(top_p):
    """Twelve million logits of two values that are next to each other, and one above them: what is summed over a bin of the histograms does not
    fit 32 bits in units of 1 / 1024 of a bin."""
    logits = torch.full((1, 12_000_001), -0.0615, device="cuda")
    logits[0, 1::2] = -0.0305
    logits[0, 7_654_320] = 0.0
    u = torch.tensor([0.0, 0.37, 0.86, 1 - 2.0 ** -24], device="cuda")
    check_sample(logits.expand(4, -1), u, 1.0, 0, top_p, 0.0)
    check_sample(logits.expand(4, -1), u, 1.0, 7_000_000, top_p, 0.0)


def test_sample_of_a_step_without_rows():
    """Nothing was granted: no row of logits, and -1 for every request."""
    logits, u = rnd(gen(0), 4, 50, dtype=torch.float32), torch.rand(3, device="cuda")
    for none in (logits[:0], torch.empty(0, 50, device="cuda")):
        tokens, lp = mk.sample_tokens(none, u, 0.8, 5, qo_indptr=i32([0, 0, 0, 0]), return_logprobs=True)
        assert tokens.tolist() == [-1] * 3 and lp.tolist() == [-math.inf] * 3


@pytest.mark.parametrize("rows", [2, 140])
def test_attention_of_requests_without_pages(rows):
    """An index without entries: every row sees nothing."""
    q = rnd(gen(rows), rows + 1, 8, D)
    cache = torch.full((3, 16, 2, D), math.nan, dtype=BF, device="cuda")
    out, lse = torch.full_like(q, 7.0), torch.full((rows + 1, 8), 7.0, device="cuda")
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    mk.chunk_attention(q, cache, cache, i32([0, rows, rows]), i32([0, 0, 0]), empty, i32([0, 0]), out=out, lse=lse)
    assert not out[:rows].any() and bool((lse[:rows] == -math.inf).all())
    assert bool((out[rows] == 7).all()) and bool((lse[rows] == 7).all())


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("gap", [12.0, 15.0, 17.5, 20.0])
@pytest.mark.parametrize("requests", [[(20000, 1)], [(9000, 3), (20000, 6)], [(20000, 80), (300, 1)]])
def test_attention_of_many_small_weights(requests, gap, dtype):
    """One position has a score `gap` above all others, which are what the output consists of: their weights exp(-gap) are small against 2^-14, below
    which fp16 has fewer bits, and at last against 2^-25, from where on it has none.  On top of what every case may be off by, an fp16 weight
    may by 2^-36 of the largest (it is carried 2^11 times as large or more, in steps of 2^-24)."""
    b = Batch(requests, 4, 2, 64, dtype)
    b.q.zero_(), b.k.zero_()
    b.q[..., 0] = 16.0
    b.v.abs_().mul_(500.0)
    first = b.kv_indices[torch.tensor(b.kv[:-1], device="cuda")].long()
    b.k[first, 0, :, 0] = gap / (16.0 * D ** -0.5)
    b.v[first, 0] = 0.0
    want, lse, tol, lse_tol = b.reference()
    if dtype == FP:
        for r, (c, n) in enumerate(requests):
            v = b.v[b.kv_indices[b.kv[r]:b.kv[r + 1]].long()].flatten(0, 1)[: c + n].double().sum(0).repeat_interleave(2, 0)
            tol[b.qo[r]:b.qo[r + 1]] += 2.0 ** -36 * v  # (the sum of weights is 1 or more of the largest)
    b.run()
    n = b.qo[-1]
    off = (b.out[:n].double() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off / want.abs()).nan_to_num(0).max())} of the value, {float((off / tol).max())} of what is allowed"
    assert bool(((b.lse[:n].double() - lse).abs() <= lse_tol).all())


# ------------------------------------------------------------------------------------
# waits that run out
# ------------------------------------------------------------------------------------
def _call(b, wait_ns):
    """chunk_attention through its C entry point, which has a limit of the kernel's waits."""
    lib, a = _cabi.load(), _cabi.MkChunkAttentionArgs()
    for name, t in (("q", b.q), ("k_cache", b.k), ("v_cache", b.v), ("qo_indptr", b.qo_indptr), ("kv_indptr", b.kv_indptr), ("kv_indices", b.kv_indices),
                    ("last_page_len", b.last), ("out", b.out), ("lse", b.lse)):
        setattr(a, name, t.data_ptr())
    a.q_stride[:], a.out_stride[:], a.lse_stride[:] = b.q.stride()[:2], b.out.stride()[:2], b.lse.stride()
    a.k_cache_stride[:], a.v_cache_stride[:] = b.k.stride()[:3], b.v.stride()[:3]
    a.scale, a.dtype, a.requests, a.tokens = D ** -0.5, _cabi.MK_BF16 if b.dtype == BF else _cabi.MK_F16, len(b.requests), b.q.shape[0]
    a.q_heads, a.kv_heads, a.pages, a.page_size, a.num_indices, a.wait_ns = b.n_q, b.n_kv, b.k.shape[0], b.page, b.kv_indices.numel(), wait_ns
    a.workspace_bytes = lib.mk_chunk_attention_workspace(C.byref(a))
    workspace = torch.empty(a.workspace_bytes, dtype=torch.uint8, device="cuda")
    a.workspace = workspace.data_ptr()
    rc = lib.mk_chunk_attention(C.byref(a), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("requests", [[(0, 300)], [(500, 140), (90, 1), (0, 70)], [(2000, 2100)]])
def test_attention_whose_waits_run_out(requests, dtype):
    """A limit below what a copy takes: the kernel ends, says so to the host, and leaves NaN in rows of its tiles; nothing else is lost.  Whatever the limit, a
    row that is not NaN is right, and the calls behind are."""
    b = Batch(requests, 8, 2, 16, dtype, pad=3)
    mk.serving.check_waits()
    want, _, tol, _ = b.reference()
    n = b.qo[-1]
    tiles = torch.cat([torch.full((k,), 4 * k > 32, device="cuda") for _, k in requests])  # rows of the tile kernel, of 4 q heads a kv head
    for wait_ns in (1, 300, 1000, 2000, 4000, 10000, 30000, 90000):
        b.out.fill_(7.0), b.lse.fill_(7.0)
        assert _call(b, wait_ns) == 0
        lost = b.out[:n].isnan().any(-1)
        right = ((b.out[:n].double() - want).abs() <= tol).all(-1)
        assert bool((lost | right).all()) and bool((b.out[n:] == 7).all()) and bool((b.lse[n:] == 7).all())
        assert torch.equal(lost, b.lse[:n].isnan()) and not bool(lost[~tiles].any())
        if wait_ns == 1:
            assert bool(lost[tiles].all())
        if bool(lost.any()):
            with pytest.raises(RuntimeError, match=r"wait for .* ran out \(CTA \d+\)"):
                if wait_ns % 3000 == 0:  # reported by whichever comes first
                    mk.serving.check_waits()
                else:
                    b.run()
            assert bool((lost == b.out[:n].isnan().any(-1)).all())  # (and that call has done nothing)
        else:
            try:  # (a warp whose rows are all behind the last one may have given up)
                mk.serving.check_waits()
            except RuntimeError as e:
                assert "ran out" in str(e)
        mk.serving.check_waits()
        assert _call(b, 0) == 0 and bool(((b.out[:n].double() - want).abs() <= tol).all())
    b.check()
    mk.serving.check_waits()


# ------------------------------------------------------------------------------------
# tensors that share memory
# ------------------------------------------------------------------------------------
def test_tensors_that_share_memory_are_refused_and_slices_beside_each_other_are_not():
    b = Batch([(200, 2), (0, 50)], 8, 2, 16)
    rows = b.qo[-1]
    b.check()
    joint = torch.zeros(rows + 1, 16, D, dtype=BF, device="cuda")
    joint[1:, :8] = b.q
    b.q, kept = joint[1:, :8], b.out
    for out in (joint[:-1, :8], joint[1:, 1:9], b.k.view(-1)[: rows * 8 * D].view(rows, 8, D)):
        b.out = out
        with pytest.raises(ValueError, match="out and (q|k_cache) share memory"):
            b.run()
    b.out = joint[1:, 8:]
    b.check()
    b.out, lse = kept, b.lse
    b.lse = kept.view(torch.float32).view(-1)[: rows * 8].view(rows, 8)
    with pytest.raises(ValueError, match="out and lse share memory"):
        b.run()
    b.lse = lse
    assert torch.equal(joint[1:, :8], b.q) and not joint[0].any()

    g = gen(0)
    x = rnd(g, 6, 8, D)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    cos, sin = torch.ones(6, D, device="cuda"), torch.zeros(6, D, device="cuda")
    kv = torch.zeros(4, 2, 4, 2, D, dtype=BF, device="cuda")
    flat = kv.view(-1)
    args = dict(q=q, k=k, v=v, cos=cos, sin=sin, positions=torch.arange(6, dtype=torch.int32, device="cuda"), slots=torch.arange(6, device="cuda"),
                k_cache=kv[:3, 0], v_cache=kv[:3, 1])
    row_later = flat.as_strided((3, 4, 2, D), kv[:3, 0].stride(), 2 * D)
    for change, text in ((dict(v_cache=row_later), "k_cache and v_cache"), (dict(out=x[:, 2:6]), "out and (k|q)"), (dict(out=kv[0, 0].reshape(-1)[: 6 * D].view(6, 1, D).expand(6, 4, D)), "share memory"),
                         (dict(out=flat[: 6 * 4 * D].view(6, 4, D)), "k_cache and out"), (dict(k=kv[:2].view(-1, 2, D)[:6]), "k_cache and k")):
        with pytest.raises(ValueError, match=text):
            mk.rotate_append(**{**args, **change})
    assert not kv.any()
    out = mk.rotate_append(**args, out=q)
    assert torch.equal(out, q) and torch.equal(kv[:3, 0].reshape(12, 2, D)[:6], k) and torch.equal(kv[:3, 1].reshape(12, 2, D)[:6], v)

    logits, buf = rnd(g, 4, 50, dtype=torch.float32), torch.ones(8, dtype=torch.float32, device="cuda")
    for kw in (dict(u=buf[:4]), dict(u=buf[4:]), dict(u=torch.rand(4, device="cuda"), temperature=buf[2:6]), dict(u=torch.rand(4, device="cuda"), top_k=buf.view(torch.int32)[:4])):
        with pytest.raises(ValueError, match="out and .* share memory"):
            mk.sample_tokens(logits, out=buf.view(torch.int64), **kw)
    with pytest.raises(ValueError, match="out and logits share memory"):
        mk.sample_tokens(logits, torch.rand(4, device="cuda"), out=logits.view(-1)[:8].view(torch.int64))
    with pytest.raises(ValueError, match="out and qo_indptr"):
        mk.sample_tokens(logits, torch.rand(3, device="cuda"), qo_indptr=buf.view(torch.int32)[:4], out=buf.view(torch.int64)[:3])


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    b = Batch([(40, 2)], 8, 2, 16)
    logits, u = rnd(gen(0), 2, 50, dtype=torch.float32), torch.rand(2, device="cuda")
    cos = torch.ones(4, D, device="cuda")
    x = rnd(gen(1), 2, 4, D)
    caches = [torch.zeros(1, 4, 2, D, dtype=BF, device="cuda") for _ in range(2)]
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        with pytest.raises(ValueError, match="q carries a forward-mode tangent"):
            mk.chunk_attention(dual(b.q), b.k, b.v, b.qo_indptr, b.kv_indptr, b.kv_indices, b.last)
        with pytest.raises(ValueError, match="v_cache carries"), torch.no_grad():
            mk.chunk_attention(b.q, b.k, dual(b.v), b.qo_indptr, b.kv_indptr, b.kv_indices, b.last)
        with pytest.raises(ValueError, match="sin carries"):
            mk.rotate_append(x, x[:, :2], x[:, 2:], cos, dual(cos), i32([0, 1]), torch.arange(2, device="cuda"), *caches)
        with pytest.raises(ValueError, match="logits carries"):
            mk.sample_tokens(dual(logits), u)
        with pytest.raises(ValueError, match="temperature carries"):
            mk.sample_tokens(logits, u, dual(torch.ones(2, device="cuda")))
        mk.sample_tokens(fw.unpack_dual(dual(logits)).primal, u)
    mk.sample_tokens(logits, u)


def test_logprobs_are_asked_for_by_any_true_value():
    import numpy as np
    logits, u = rnd(gen(0), 2, 50, dtype=torch.float32), torch.rand(2, device="cuda")
    want = mk.sample_tokens(logits, u, return_logprobs=True)
    for yes in (1, np.True_, "yes"):
        got = mk.sample_tokens(logits, u, return_logprobs=yes)
        assert isinstance(got, tuple) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for no in (0, np.False_, None):
        assert torch.equal(mk.sample_tokens(logits, u, return_logprobs=no), want[0])


def test_plan_grants_no_position_past_32_bits():
    """A request may grow to 2^31 - 1 tokens; one token more, and its positions (and its length) would not fit their type."""
    page, top = 1 << 20, 2 ** 31 - 1
    for more in (3, 4):
        table = torch.full((2, 2100), -7, dtype=torch.int32, device="cuda")
        table[0, :2048] = torch.arange(2048, dtype=torch.int32, device="cuda")
        plan = mk.StepPlan.empty(2, 8, 2200)
        mk.plan_step(i32([top - 3, 0]), i32([more, 2]), table, i32([2050, 2051]), torch.tensor([0, 2], device="cuda"), page, plan)
        granted = 3 if more == 3 else 0
        assert plan.granted.tolist() == [granted, 2]
        own = [(2047 * page + page - 4 + i, top - 3 + i) for i in range(granted)]
        assert list(zip(plan.slots.tolist(), plan.positions.tolist()))[: granted + 2] == own + [(2050 * page, 0), (2050 * page + 1, 1)]
        assert plan.last_page_len.tolist() == [page - 4 + granted, 2]


@pytest.mark.parametrize("max_new", [1, 2, 9, 100, 10 ** 6, 2 ** 31 - 1])
def test_attention_whatever_the_caller_says_of_its_longest_chunk(max_new):
    """max_new chooses kernels; one that is too small or too large leaves the results within what every case is allowed."""
    Batch([(300, 1), (64, 90), (0, 33), (700, 7), (5, 0)], 8, 2, 16, pad=2).check(max_new=max_new)
    Batch([(200, 40)], 14, 2, 8, dtype=FP).check(max_new=max_new, window=50, sinks=2)


def test_the_first_call_of_a_process_may_be_a_captured_one():
    """What a process sets up once (shared memory of the kernels, tensor maps, the word that waits report to) is no part of the graph."""
    code = """
import torch, fleet_chiplet_megakernel_b200 as mk
from tests.test_gpu_serving import Batch
b = Batch([(40, 2), (0, 300), (9, 1)], 8, 2, 16)
logits, u = torch.randn(3, 5000, device="cuda"), torch.rand(3, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    b.run()
    tokens = mk.sample_tokens(logits, u, 0.9, 0, 0.9)
g.replay()
torch.cuda.synchronize()
got = b.out.clone()
b.check()
assert torch.equal(got, b.out) and torch.equal(tokens, mk.sample_tokens(logits, u, 0.9, 0, 0.9))
mk.serving.check_waits()
print("captured first")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and "captured first" in r.stdout, (r.returncode, r.stdout, r.stderr[-2000:])


def test_tensors_that_are_negated_lazily_are_refused():
    """A view that only records a sign (of the imaginary part of a conjugate, for instance) holds other numbers than its memory."""
    b = Batch([(40, 2)], 8, 2, 16)
    logits, u = rnd(gen(0), 2, 50, dtype=torch.float32), torch.rand(2, device="cuda")
    b.q = torch._neg_view(b.q)
    with pytest.raises(ValueError, match="q is negated"):
        b.run()
    with pytest.raises(ValueError, match="logits is negated"):
        mk.sample_tokens(torch._neg_view(logits), u)
    assert torch.equal(mk.sample_tokens(torch._neg_view(logits).resolve_neg(), u), mk.sample_tokens(-logits, u))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("at", [200, 130, 400, 470])
@pytest.mark.parametrize("requests,heads", [([(420, 60)] * 11, (32, 8)), ([(5000, 60)], (8, 2))])
def test_attention_whose_scores_grow_by_the_range_of_a_float(requests, heads, at, dtype):
    """All scores are 0 but one position's, which lie 120 to 134 above in base 2, row by row: in the bf16 tiles its weight is next to the largest float, or beyond
    it, until the base of the row follows (it never does behind the last tile), and what the weights are scaled by then is next to the smallest."""
    b = Batch(requests, *heads, 64, dtype, spoil=False)
    per_log2 = 1 / (D ** -0.5 * math.log2(math.e))
    b.k.zero_(), b.q.zero_()
    b.q[..., 0] = 1.0
    b.q[..., 1] = torch.linspace(-1, 1, b.q.shape[0] * b.n_q, device="cuda").view(b.q.shape[0], b.n_q).to(dtype)
    for r, (c, n) in enumerate(requests):
        p = c + n - 480 + at  # (a position that the cache has)
        page = b.kv_indices[b.kv[r] + p // 64].long()
        b.k[page, p % 64, :, 0], b.k[page, p % 64, :, 1] = round(127 * per_log2 / 4) * 4, round(7 * per_log2)
    b.check()
