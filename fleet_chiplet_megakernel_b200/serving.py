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
sizes beyond what a kernel takes ``NotImplementedError``.  What index tensors hold is on the device and is not checked here: the
kernels stay inside the tensors whatever it is.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _cabi

HEAD_DIM = 128
_DTYPES = {torch.bfloat16: _cabi.MK_BF16, torch.float16: _cabi.MK_F16, torch.float32: _cabi.MK_F32}
_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32


def _check(rc, what):
    if rc >= 0:
        return rc
    buf = C.create_string_buffer(512)
    _cabi.load().mk_op_error(buf, 512)
    msg = buf.value.decode() or what
    if rc in (_cabi.MK_E_UNSUPPORTED, _cabi.MK_E_TOO_LARGE):
        raise NotImplementedError(msg)
    if rc == _cabi.MK_E_INVALID:
        raise ValueError(msg)
    raise RuntimeError(msg)


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def _tensor(t, what, dtype, device, shape=None, least=None):
    """A tensor argument: type, device, shape (None in it: any), contiguous; ``least``: at least so many entries of one dimension."""
    _need(isinstance(t, torch.Tensor), f"{what}: a tensor is needed")
    _need(t.dtype == dtype, f"{what}.dtype: {t.dtype}, {dtype} is needed")
    _need(t.device == device, f"{what} is on {t.device}, the others on {device}")
    if shape is not None:
        _need(t.dim() == len(shape) and all(s is None or s == d for s, d in zip(shape, t.shape)), f"{what}.shape: {tuple(t.shape)}, {shape} is needed")
    if least is not None:
        _need(t.dim() == 1 and t.shape[0] >= least, f"{what}.shape: {tuple(t.shape)}, one dimension of at least {least} is needed")
    _need(t.is_contiguous(), f"{what} must be contiguous")
    return t.data_ptr()


def _rows(t, what, dtype, device, heads=None, tokens=None):
    """Rows [tokens, heads, 128] with any token and head stride."""
    _need(isinstance(t, torch.Tensor), f"{what}: a tensor is needed")
    _need(t.dim() == 3 and t.shape[2] == HEAD_DIM, f"{what}.shape: {tuple(t.shape)}, [tokens, heads, {HEAD_DIM}] is needed")
    _need(t.dtype == dtype, f"{what}.dtype: {t.dtype}, {dtype} is needed")
    _need(t.device == device, f"{what} is on {t.device}, the others on {device}")
    _need(heads is None or t.shape[1] == heads, f"{what} has {t.shape[1]} heads, {heads} are needed")
    _need(tokens is None or t.shape[0] == tokens, f"{what} has {t.shape[0]} rows, {tokens} are needed")
    s = t.stride()
    _need(s[2] == 1, f"{what}: the elements of a row must be contiguous")
    return t.data_ptr(), s[:2]


def _no_overlap(strides, shape, what):
    """Rows that are written may not share memory, as those of an expanded tensor do."""
    at = sorted((s, n) for s, n in zip(strides, shape) if n > 1)
    reach = HEAD_DIM
    for s, n in at:
        _need(s >= reach, f"{what}: its rows share memory")
        reach = s * (n - 1) + reach


def _cache(t, what, dtype, device):
    _need(isinstance(t, torch.Tensor), f"{what}: a tensor is needed")
    _need(t.dim() == 4 and t.shape[3] == HEAD_DIM, f"{what}.shape: {tuple(t.shape)}, [pages, page_size, kv_heads, {HEAD_DIM}] is needed")
    _need(t.dtype == dtype, f"{what}.dtype: {t.dtype}, {dtype} is needed")
    _need(t.device == device, f"{what} is on {t.device}, the others on {device}")
    s = t.stride()
    _need(s[3] == 1, f"{what}: the elements of a row must be contiguous")
    return t.data_ptr(), s[:3]


def _cuda(t, what):
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{what} must be a CUDA tensor; there is no CPU fallback")
    return t.device


def _call(fn, args, device, what):
    """The native call on the current stream of the tensors' device."""
    if device.index == torch.cuda.current_device():
        rc = fn(C.byref(args), torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(args), torch.cuda.current_stream(device).cuda_stream)
    if rc < 0:
        _check(rc, what)


# ------------------------------------------------------------------------------------
# the plan of a step
# ------------------------------------------------------------------------------------
@dataclass
class StepPlan:
    """What ``plan_step`` writes, for up to ``len(granted)`` requests and ``len(slots)`` token rows.  The first four may be the meta
    tensors of a ``PersistentKernel``."""
    qo_indptr: torch.Tensor      # [requests + 1] int32: first token row of every request
    kv_indptr: torch.Tensor      # [requests + 1] int32: its first entry of kv_indices
    kv_indices: torch.Tensor     # [pages] int32: the pages of every request in order
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
    order; one that cannot have all of them is granted nothing, nor are those behind it that need any.  Pages of ended requests
    go behind the ring's tail first and can be taken in the same step.  ``block_table`` and ``free_pages`` are brought up to date in place;
    the step counts once the caller takes ``plan.free_range`` and ``lengths + plan.granted`` (0 for ended requests) into its next one:
    until then the same call gives the same plan."""
    dev = _cuda(lengths, "lengths")
    a = _cabi.MkStepPlanArgs()
    _need(isinstance(plan, StepPlan), "plan: a StepPlan is needed")
    _need(lengths.dim() == 1 and lengths.shape[0] > 0, "lengths: one dimension, a length per request, is needed")
    R = lengths.shape[0]
    a.lengths = _tensor(lengths, "lengths", _I32, dev)
    a.new_tokens = _tensor(new_tokens, "new_tokens", _I32, dev, (R,))
    _need(isinstance(block_table, torch.Tensor) and block_table.dim() == 2 and block_table.shape[0] == R and block_table.shape[1] > 0 and
          block_table.dtype == _I32 and block_table.device == dev, f"block_table: int32 [{R}, pages of the longest request] on {dev} is needed")
    stride = block_table.stride()
    _need(stride[1] == 1 and (R == 1 or stride[0] >= block_table.shape[1]), "block_table: rows must be contiguous and apart")
    a.block_table, a.table_stride, a.table_width = block_table.data_ptr(), max(stride[0], block_table.shape[1]), block_table.shape[1]
    a.free_pages = _tensor(free_pages, "free_pages", _I32, dev, least=1)
    a.free_range_in = _tensor(free_range, "free_range", _I64, dev, (2,))
    a.qo_indptr = _tensor(plan.qo_indptr, "plan.qo_indptr", _I32, dev, (R + 1,))
    a.kv_indptr = _tensor(plan.kv_indptr, "plan.kv_indptr", _I32, dev, (R + 1,))
    a.kv_indices = _tensor(plan.kv_indices, "plan.kv_indices", _I32, dev, least=1)
    a.last_page_len = _tensor(plan.last_page_len, "plan.last_page_len", _I32, dev, (R,))
    a.slots = _tensor(plan.slots, "plan.slots", _I64, dev, least=1)
    T = plan.slots.shape[0]
    a.positions = _tensor(plan.positions, "plan.positions", _I32, dev, (T,))
    a.granted = _tensor(plan.granted, "plan.granted", _I32, dev, (R,))
    a.free_range_out = _tensor(plan.free_range, "plan.free_range", _I64, dev, (2,))
    _need(a.free_range_out != a.free_range_in, "plan.free_range may not be free_range: the call reads one and writes the other")
    _need(page_size >= 1, "page_size must be positive")
    a.requests, a.ring_size, a.max_indices, a.max_tokens, a.page_size = R, free_pages.shape[0], plan.kv_indices.shape[0], T, page_size
    _call(_cabi.load().mk_plan_step, a, dev, "plan_step")
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
    their rows of ``out`` as they were.  A slot may not occur twice."""
    dev = _cuda(q, "q")
    a = _cabi.MkRotateAppendArgs()
    dt = q.dtype
    _need(dt in (torch.bfloat16, torch.float16), f"q.dtype: {dt}, bf16 or fp16 is needed")
    a.q, a.q_stride[:] = _rows(q, "q", dt, dev)
    a.k, a.k_stride[:] = _rows(k, "k", dt, dev, tokens=q.shape[0])
    a.v, a.v_stride[:] = _rows(v, "v", dt, dev, k.shape[1], q.shape[0])
    T, n_q, n_kv = q.shape[0], q.shape[1], k.shape[1]
    a.k_cache, a.k_cache_stride[:] = _cache(k_cache, "k_cache", dt, dev)
    a.v_cache, a.v_cache_stride[:] = _cache(v_cache, "v_cache", dt, dev)
    _need(k_cache.shape[2] == n_kv and v_cache.shape == k_cache.shape, f"caches {tuple(k_cache.shape)} and {tuple(v_cache.shape)} for {n_kv} kv heads")
    for t, what in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _no_overlap(t.stride()[:3], t.shape[:3], what)
    for t, what in ((cos, "cos"), (sin, "sin")):
        _need(isinstance(t, torch.Tensor) and t.dim() == 2 and t.shape[1] == HEAD_DIM and t.shape[0] > 0 and t.stride(1) == 1 and t.device == dev and
              t.dtype == cos.dtype and t.dtype in (dt, _F32) and t.shape == cos.shape,
              f"{what}: [positions, {HEAD_DIM}] of type {dt} or fp32 on {dev}, cos and sin alike, is needed")
    a.cos, a.sin, a.table_stride[:] = cos.data_ptr(), sin.data_ptr(), (cos.stride(0), sin.stride(0))
    for t, what in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        if t is not None:
            setattr(a, what, _tensor(t, what, dt, dev, (HEAD_DIM,)))
    a.positions = _tensor(positions, "positions", _I32, dev, (T,))
    a.slots = _tensor(slots, "slots", _I64, dev, (T,))
    if out is None:
        out = torch.zeros(T, n_q, HEAD_DIM, dtype=dt, device=dev)
    a.out, a.out_stride[:] = _rows(out, "out", dt, dev, n_q, T)
    _no_overlap(out.stride()[:2], out.shape[:2], "out")
    a.eps, a.dtype, a.table_dtype = eps, _DTYPES[dt], _DTYPES[cos.dtype]
    a.tokens, a.q_heads, a.kv_heads, a.pages, a.page_size, a.table_rows = T, n_q, n_kv, k_cache.shape[0], k_cache.shape[1], cos.shape[0]
    if T:
        _call(_cabi.load().mk_rotate_append, a, dev, "rotate_append")
    return out


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
    ``max_new``: the largest number of new tokens of a request, if the caller knows it; it chooses kernels, nothing else depends on it.
    Returns ``out`` [tokens, q_heads, 128]."""
    dev = _cuda(q, "q")
    a = _cabi.MkChunkAttentionArgs()
    dt = q.dtype
    _need(dt in (torch.bfloat16, torch.float16), f"q.dtype: {dt}, bf16 or fp16 is needed")
    a.q, a.q_stride[:] = _rows(q, "q", dt, dev)
    T, n_q = q.shape[0], q.shape[1]
    a.k_cache, a.k_cache_stride[:] = _cache(k_cache, "k_cache", dt, dev)
    a.v_cache, a.v_cache_stride[:] = _cache(v_cache, "v_cache", dt, dev)
    pages, page, n_kv, _ = k_cache.shape
    _need(v_cache.shape == k_cache.shape, f"k_cache is {tuple(k_cache.shape)}, v_cache {tuple(v_cache.shape)}")
    _need(n_kv > 0 and n_q % n_kv == 0, f"{n_q} q heads on {n_kv} kv heads")
    _need(isinstance(last_page_len, torch.Tensor) and last_page_len.dim() == 1, "last_page_len: one dimension, a length per request, is needed")
    R = last_page_len.shape[0]
    a.last_page_len = _tensor(last_page_len, "last_page_len", _I32, dev)
    a.qo_indptr = _tensor(qo_indptr, "qo_indptr", _I32, dev, (R + 1,))
    a.kv_indptr = _tensor(kv_indptr, "kv_indptr", _I32, dev, (R + 1,))
    a.kv_indices = _tensor(kv_indices, "kv_indices", _I32, dev, least=0)
    if out is None:
        out = torch.zeros(T, n_q, HEAD_DIM, dtype=dt, device=dev)
    a.out, a.out_stride[:] = _rows(out, "out", dt, dev, n_q, T)
    _no_overlap(out.stride()[:2], out.shape[:2], "out")
    if lse is not None:
        _need(isinstance(lse, torch.Tensor) and lse.dtype == _F32 and lse.shape == (T, n_q) and lse.device == dev, f"lse: fp32 [{T}, {n_q}] on {dev} is needed")
        a.lse, a.lse_stride[:] = lse.data_ptr(), lse.stride()
    _need(0 <= window < 1 << 31 and 0 <= sinks < 1 << 31 and 0 <= max_new < 1 << 31, "window, sinks and max_new may not be negative")
    a.scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else scale
    a.dtype, a.requests, a.tokens, a.q_heads, a.kv_heads, a.page_size, a.pages = _DTYPES[dt], R, T, n_q, n_kv, page, pages
    a.num_indices, a.window, a.sinks, a.max_new = kv_indices.shape[0], window, sinks, max_new
    if T == 0 or R == 0:
        return out
    lib = _cabi.load()
    if dev.index == torch.cuda.current_device():
        need = lib.mk_chunk_attention_workspace(C.byref(a))
    else:
        with torch.cuda.device(dev):
            need = lib.mk_chunk_attention_workspace(C.byref(a))
    _check(need, "chunk_attention")
    workspace = torch.empty(need, dtype=torch.uint8, device=dev)  # (of the current stream's pool, or the capturing graph's)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), need
    _call(lib.mk_chunk_attention, a, dev, "chunk_attention")
    return out


# ------------------------------------------------------------------------------------
# sampling
# ------------------------------------------------------------------------------------
def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, qo_indptr=None, out=None, return_logprobs: bool = False):
    """A token per request from its row of ``logits`` [rows, vocab] (bf16, fp16 or fp32) and its random number ``u[r]`` in [0, 1).

    Row r belongs to request r; with ``qo_indptr`` [requests + 1] int32 (``StepPlan``) its last one does, and a request without rows gets -1.
    ``temperature``, ``top_p``, ``min_p`` (fp32) and ``top_k`` (int32) are numbers or a tensor [requests] each.  temperature 0: the largest logit,
    the lowest index on ties.  Otherwise weights exp((l - max) / temperature); top_k (0: off) keeps the k largest, top_p (1: off) of
    these the ones before which less than top_p of their weight lies, min_p (0: off) those of at least min_p times the largest;
    equal logits count in the order of the index.  The token is the first by index at which the running sum of the kept weights exceeds
    u times their sum.  NaN logits count as minus infinity; a row of nothing else gives -1.  Returns tokens int64 [requests] (``out``), and
    with ``return_logprobs`` the logarithms of the probabilities with which they were drawn as well."""
    dev = _cuda(logits, "logits")
    a = _cabi.MkSampleArgs()
    _need(logits.dtype in _DTYPES, f"logits.dtype: {logits.dtype}, bf16, fp16 or fp32 is needed")
    _need(logits.dim() == 2 and logits.shape[1] > 0, f"logits.shape: {tuple(logits.shape)}, [rows, vocab] is needed")
    _need(logits.stride(1) == 1 or logits.shape[1] == 1, "logits: the elements of a row must be contiguous")
    _need(isinstance(u, torch.Tensor) and u.dim() == 1, "u: one dimension, a number per request, is needed")
    R = u.shape[0]
    a.u = _tensor(u, "u", _F32, dev)
    for name, value, dt in (("temperature", temperature, _F32), ("top_p", top_p, _F32), ("min_p", min_p, _F32), ("top_k", top_k, _I32)):
        if isinstance(value, torch.Tensor):
            setattr(a, name, _tensor(value, name, dt, dev, (R,)))
        else:
            setattr(a, name + "_value", value)
    if qo_indptr is not None:
        a.qo_indptr = _tensor(qo_indptr, "qo_indptr", _I32, dev, (R + 1,))
    else:
        _need(logits.shape[0] >= R, f"{logits.shape[0]} rows of logits for {R} requests")
    if out is None:
        out = torch.empty(R, dtype=_I64, device=dev)
    a.tokens = _tensor(out, "out", _I64, dev, (R,))
    logprobs = torch.empty(R, dtype=_F32, device=dev) if return_logprobs else None
    if return_logprobs:
        a.logprobs = logprobs.data_ptr()
    a.logits, a.row_stride, a.dtype = logits.data_ptr(), logits.stride(0), _DTYPES[logits.dtype]
    a.requests, a.rows, a.vocab = R, logits.shape[0], logits.shape[1]
    if R:
        _call(_cabi.load().mk_sample_tokens, a, dev, "sample_tokens")
    return (out, logprobs) if return_logprobs else out
