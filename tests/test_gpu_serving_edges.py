"""The serving operators at the edges of what their documentation allows: calls without rows or pages, vocabularies of millions, weights that a
16-bit type has no value for, positions next to 2^31, tangents, tensors that share memory, waits that run out."""
import math

import pytest
import torch

import fleet_chiplet_megakernel_b200 as mk
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
