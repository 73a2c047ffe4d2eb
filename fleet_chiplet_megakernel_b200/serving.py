"""Operators of a serving step for a host that keeps the paging metadata itself.

A serving engine drives the megakernel a pass at a time in mode ``online_notoken`` (``PersistentKernel``, ``MPK``) over page tables and
lengths that it owns.  What it does around the layers of a model stands here, each one call that enqueues its work on the current
stream, allocates no more than its outputs and a workspace from torch's allocator, and can be captured into a CUDA graph:

* ``plan_step``: page allocation, block tables, the index pointers that the attention layers read, slots and positions of the new tokens;
* ``rotate_append``: QK norm and rotary embedding of new rows, K and V into their cache slots;
* ``chunk_attention``: attention of the new tokens of every request over its pages, single tokens and long chunks alike, with an
  optional sliding window and first tokens that stay visible;
* ``sample_tokens``: temperature, top-k, top-p and min-p from given random numbers, where the megakernel takes the largest logit.

The caches have the layout of the attention layers, ``[pages, page_size, kv_heads, 128]``, so the megakernel goes on from what these
calls leave in them.  Tensors may be on any CUDA device (all of a call on one); wrong types, shapes and strides raise ``ValueError``,
sizes beyond what a kernel takes ``NotImplementedError``.  A tensor that is written and shares memory with another one of the call is refused as well
(slices beside each other in one buffer share none).  None of them has a derivative: a tensor that requires a gradient is refused while gradients are
recorded, one with a forward-mode tangent always.  What index tensors hold is on the device and is not checked here: the kernels stay
inside the tensors whatever it is.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _cabi

HEAD_DIM = 128
_I32, _I64 = torch.int32, torch.int64
_native = None


def _load():
    """The binding, with the entry points of the loaded library; there is no fallback without either."""
    global _native
    lib = _cabi.load()
    try:
        from . import _serving_native as native
    except ImportError as e:
        raise RuntimeError("the binding of the serving operators is missing or does not fit this torch: build it with "
                           "`python -m fleet_chiplet_megakernel_b200._build --force`") from e
    native.bind(*(C.cast(getattr(lib, name), C.c_void_p).value for name in
                  ("mk_plan_step", "mk_rotate_append", "mk_chunk_attention_workspace", "mk_chunk_attention", "mk_sample_tokens", "mk_op_error", "mk_op_check")))
    _native = native
    return native


def check_waits() -> None:
    """Raises ``RuntimeError`` if a wait inside a kernel has run out (after 2 seconds) in a ``chunk_attention`` call that is done: rows of its output
    may be NaN.  The next ``chunk_attention`` raises it as well, before it does anything.  Synchronize first, as before reading the output."""
    (_native or _load()).check_waits()


# ------------------------------------------------------------------------------------
# the plan of a step
# ------------------------------------------------------------------------------------
@dataclass
class StepPlan:
    """What ``plan_step`` writes, for ``len(granted)`` requests and up to ``len(slots)`` token rows.  The first four may be the meta
    tensors of a ``PersistentKernel``.  No two tensors of a call may share memory."""
    qo_indptr: torch.Tensor      # [requests + 1] int32: first token row of every request
    kv_indptr: torch.Tensor      # [requests + 1] int32: its first entry of kv_indices
    kv_indices: torch.Tensor     # [pages] int32: the pages of every request in order (those behind its end are left out)
    last_page_len: torch.Tensor  # [requests] int32: tokens in its last page, the new ones included (0: no page)
    slots: torch.Tensor          # [tokens] int64: cache row (page * page_size + row in the page) of every new token, -1 behind the last
    positions: torch.Tensor      # [tokens] int32: its position in its request
    granted: torch.Tensor        # [requests] int32: new tokens of this step, 0 where pages or token rows ran out
    free_range: torch.Tensor     # [2] int64: the ring's free part behind this step

    @classmethod
    def empty(cls, max_requests: int, max_tokens: int, max_pages: int, device="cuda") -> "StepPlan":
        def z(n, dt=_I32):
            return torch.zeros(n, dtype=dt, device=device)
        return cls(z(max_requests + 1), z(max_requests + 1), z(max_pages), z(max_requests), z(max_tokens, _I64), z(max_tokens), z(max_requests), z(2, _I64))


def plan_step(lengths, new_tokens, block_table, free_pages, free_range, page_size: int, plan: StepPlan) -> StepPlan:
    """Plan a step on the GPU: ``lengths[r]`` tokens of request r are in the cache, on the pages ``block_table[r, : ceil(length / page_size)]``,
    and it is to be fed ``new_tokens[r]`` more (0: idle; -1: it has ended and gives its pages back).

    Free pages are ``free_pages[i % len(free_pages)]`` for ``free_range[0] <= i < free_range[1]``.  Requests take pages and token rows in their
    order; one that cannot have all of them is granted nothing, nor are those behind it that need any.  One whose row of the table is too short, or that
    would pass 2^31 - 1 tokens, is granted nothing and holds up nobody.  Pages of ended requests go behind the ring's tail first and can be taken
    in the same step.  ``block_table`` and ``free_pages`` are brought up to date in place; the step counts once the caller takes ``plan.free_range`` and
    ``lengths + plan.granted`` (0 for ended requests) into its next one: until then the same call gives the same plan."""
    if not isinstance(plan, StepPlan):
        raise ValueError("plan: a StepPlan is needed")
    (_native or _load()).plan_step(lengths, new_tokens, block_table, free_pages, free_range, page_size, plan.qo_indptr, plan.kv_indptr, plan.kv_indices,
                                   plan.last_page_len, plan.slots, plan.positions, plan.granted, plan.free_range)
    return plan


# ------------------------------------------------------------------------------------
# rows into the cache
# ------------------------------------------------------------------------------------
def rotate_append(q, k, v, cos, sin, positions, slots, k_cache, v_cache, q_norm=None, k_norm=None, eps: float = 0.0, out=None):
    """What stands between the QKV projection and attention: ``out[t] = rope(norm(q[t]))``, and ``rope(norm(k[t]))`` and ``v[t]`` into row
    ``slots[t]`` of the caches.

    q [tokens, q_heads, 128], k and v [tokens, kv_heads, 128]: bf16 or fp16, any token and head stride (slices of one projection).  cos and
    sin [positions, 128], of the rows' type or fp32; row ``positions[t]`` is used.  norm(x) = w x / sqrt(mean(x^2) + eps) where ``q_norm`` /
    ``k_norm`` [128] are given.  fp32 throughout, rounded once.  Tokens with a slot or position outside (-1: padding) are left out,
    their rows of ``out`` as they were.  A slot may not occur twice; ``out`` may be q."""
    return (_native or _load()).rotate_append(q, k, v, cos, sin, positions, slots, k_cache, v_cache, q_norm, k_norm, eps, out)


# ------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------
def chunk_attention(q, k_cache, v_cache, qo_indptr, kv_indptr, kv_indices, last_page_len, scale: float | None = None, window: int = 0, sinks: int = 0,
                    out=None, lse=None, max_new: int = 0):
    """Causal attention of new tokens over a paged cache that already holds their K and V.

    Request r has rows ``qo_indptr[r] <= t < qo_indptr[r + 1]`` of q [tokens, q_heads, 128] and the pages ``kv_indices[kv_indptr[r] : kv_indptr[r + 1]]``
    of k_cache and v_cache [pages, page_size, kv_heads, 128] (bf16 or fp16), the last filled up to ``last_page_len[r]``; its new rows are its
    last positions.  One new token each (decode), chunks, or both in one batch.  ``window`` > 0: a row at position p sees positions above
    p - window and the first ``sinks``.  ``scale``: 1/sqrt(128) if None.  Rows behind the last request are left as they were; a row that
    sees nothing is zero.  ``lse`` [tokens, q_heads] fp32, if given, takes the natural logarithm of each row's sum of weights.
    ``max_new``: the largest number of new tokens of a request, if the caller knows it (0: no); say it for a batch of single tokens, which then need not
    pass by the kernel for chunks.  It only chooses kernels and may be wrong.  Both kernels hold scores, weights' sums and outputs in fp32.  Requests of up to
    32 rows (new tokens x q heads of a kv head) enter the product with V with weights of two 16-bit parts, longer chunks with weights rounded to the
    cache's type, which adds about as much error as the rounding of ``out``; so the last bits of a row depend on the kernel that takes it.
    Returns ``out`` [tokens, q_heads, 128], which may not share memory with q."""
    return (_native or _load()).chunk_attention(q, k_cache, v_cache, qo_indptr, kv_indptr, kv_indices, last_page_len, scale, window, sinks, out, lse, max_new)


# ------------------------------------------------------------------------------------
# sampling
# ------------------------------------------------------------------------------------
def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, qo_indptr=None, out=None, return_logprobs: bool = False):
    """A token per request from its row of ``logits`` [rows, vocab] (bf16, fp16 or fp32) and its random number ``u[r]`` in [0, 1).

    Row r belongs to request r; with ``qo_indptr`` [requests + 1] int32 (``StepPlan``) its last one does, and a request without rows gets -1.
    ``temperature``, ``top_p``, ``min_p`` (fp32) and ``top_k`` (int32) are numbers or a tensor [requests] each.  temperature 0: the largest logit,
    the lowest index on ties.  Otherwise weights exp((l - max) / temperature); top_k (0: off) keeps the k largest, top_p (1: off) of
    these the ones before which less than top_p of their weight lies, min_p (0: off; above 1 it counts as 1) those of at least min_p times the largest;
    equal logits count in the order of the index.  The token is the first by index at which the running sum of the kept weights exceeds
    u times their sum.  NaN logits count as minus infinity; a row of nothing else gives -1.  Returns tokens int64 [requests] (``out``), and
    with ``return_logprobs`` the logarithms of the probabilities with which they were drawn as well."""
    return (_native or _load()).sample_tokens(logits, u, temperature, top_k, top_p, min_p, qo_indptr, out, return_logprobs)
