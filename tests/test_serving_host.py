"""Refusals of the serving operators, without a GPU: the Python checks and those behind the C entry points (which look at the
arguments before any CUDA call is made)."""
import ctypes as C

import pytest
import torch

import fleet_chiplet_megakernel_b200 as mk
from fleet_chiplet_megakernel_b200 import _cabi

FAKE = 1 << 20  # an aligned address that nothing reads: the calls end at their checks


def refused(lib, fn, args, code, text):
    assert getattr(lib, fn)(C.byref(args) if args is not None else None, None) == code
    buf = C.create_string_buffer(512)
    assert lib.mk_op_error(buf, 512) == 0
    assert text in buf.value.decode(), buf.value


def filled(cls, **kw):
    a = cls()
    for name, kind in cls._fields_:
        if kind is C.c_void_p:
            setattr(a, name, FAKE)
        elif kind is C.c_int32:
            setattr(a, name, 1)
    for name, value in kw.items():
        if isinstance(value, tuple):
            getattr(a, name)[:] = value
        else:
            setattr(a, name, value)
    return a


def test_cpu_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        mk.plan_step(z(1, dtype=torch.int32), z(1, dtype=torch.int32), z(1, 1, dtype=torch.int32), z(1, dtype=torch.int32), z(2, dtype=torch.int64), 16,
                     mk.StepPlan.empty(1, 1, 1, device="cpu"))
    q = z(1, 2, 128, dtype=torch.bfloat16)
    cache = z(1, 16, 1, 128, dtype=torch.bfloat16)
    ptr = z(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        mk.chunk_attention(q, cache, cache, ptr, ptr, ptr, ptr[:1])
    with pytest.raises(ValueError, match="CUDA"):
        mk.rotate_append(q, q[:, :1], q[:, :1], z(1, 128), z(1, 128), ptr[:1], z(1, dtype=torch.int64), cache, cache)
    with pytest.raises(ValueError, match="CUDA"):
        mk.sample_tokens(z(1, 4), z(1))


@pytest.mark.parametrize("change,code,text", [
    ({"slots": None}, _cabi.MK_E_INVALID, "null"), ({"requests": 0}, _cabi.MK_E_INVALID, "requests"), ({"requests": 8193}, _cabi.MK_E_TOO_LARGE, "requests"),
    ({"page_size": 0}, _cabi.MK_E_INVALID, "positive"), ({"table_stride": 0}, _cabi.MK_E_INVALID, "overlap"), ({"ring_size": 0}, _cabi.MK_E_INVALID, "positive"),
    ({"requests": 8000, "table_width": 1 << 20, "table_stride": 1 << 20}, _cabi.MK_E_TOO_LARGE, "2^31")])
def test_plan_refusals(native_lib, change, code, text):
    refused(native_lib, "mk_plan_step", filled(_cabi.MkStepPlanArgs, **{"table_stride": 1, **change}), code, text)


@pytest.mark.parametrize("change,text", [
    ({"k_cache": None}, "null"), ({"dtype": _cabi.MK_F32}, "bf16 or fp16"), ({"dtype": _cabi.MK_BF16, "table_dtype": _cabi.MK_F16}, "rows' type"),
    ({"q_heads": 0}, "positive"), ({"tokens": -1}, "positive"), ({"page_size": 0}, "positive")])
def test_rotate_append_refusals(native_lib, change, text):
    refused(native_lib, "mk_rotate_append", filled(_cabi.MkRotateAppendArgs, **{"dtype": _cabi.MK_F16, "table_dtype": _cabi.MK_F16, **change}), _cabi.MK_E_INVALID, text)


@pytest.mark.parametrize("change,code,text", [
    ({"q": None}, _cabi.MK_E_INVALID, "null"), ({"dtype": _cabi.MK_I32}, _cabi.MK_E_INVALID, "bf16 or fp16"), ({"q_heads": 3, "kv_heads": 2}, _cabi.MK_E_INVALID, "3 q heads"),
    ({"window": -1}, _cabi.MK_E_INVALID, "negative"), ({"sinks": -1}, _cabi.MK_E_INVALID, "negative"), ({"requests": 5000}, _cabi.MK_E_TOO_LARGE, "requests"),
    ({"out": FAKE + 8}, _cabi.MK_E_INVALID, "aligned"), ({"k_cache_stride": (128, 4, 128)}, _cabi.MK_E_INVALID, "caches"), ({"q_stride": (132, 128)}, _cabi.MK_E_INVALID, "q and out"),
    ({"tokens": 1 << 30, "q_heads": 4}, _cabi.MK_E_TOO_LARGE, "rows"), ({"workspace_bytes": 16}, _cabi.MK_E_INVALID, "workspace"), ({"workspace": None}, _cabi.MK_E_INVALID, "workspace")])
def test_chunk_attention_refusals(native_lib, change, code, text):
    base = {"dtype": _cabi.MK_BF16, "q_stride": (128, 128), "out_stride": (128, 128), "k_cache_stride": (128, 128, 128), "v_cache_stride": (128, 128, 128), "workspace_bytes": 1 << 40}
    refused(native_lib, "mk_chunk_attention", filled(_cabi.MkChunkAttentionArgs, **{**base, **change}), code, text)


@pytest.mark.parametrize("change,code,text", [
    ({"u": None}, _cabi.MK_E_INVALID, "null"), ({"dtype": _cabi.MK_I32}, _cabi.MK_E_INVALID, "fp32"), ({"vocab": 0}, _cabi.MK_E_INVALID, "sizes"),
    ({"qo_indptr": None, "requests": 2}, _cabi.MK_E_INVALID, "rows of logits"), ({"requests": 1 << 29, "rows": 1 << 29}, _cabi.MK_E_TOO_LARGE, "requests")])
def test_sample_refusals(native_lib, change, code, text):
    refused(native_lib, "mk_sample_tokens", filled(_cabi.MkSampleArgs, **{"dtype": _cabi.MK_F32, **change}), code, text)


def test_arrays_that_share_memory_are_refused(native_lib):
    names = [n for n, kind in _cabi.MkStepPlanArgs._fields_ if kind is C.c_void_p]
    apart = {n: FAKE + (k << 12) for k, n in enumerate(names)}
    written = [n for n in names if n not in ("lengths", "new_tokens", "free_range_in")]
    for name in written:
        for other in names:
            if other != name:
                refused(native_lib, "mk_plan_step", filled(_cabi.MkStepPlanArgs, **{**apart, "table_stride": 1, "requests": 4, "max_indices": 4, "max_tokens": 4, "ring_size": 4, other: apart[name] + 4}),
                        _cabi.MK_E_INVALID, "share memory")
    a = filled(_cabi.MkRotateAppendArgs, dtype=_cabi.MK_BF16, table_dtype=_cabi.MK_F32)
    refused(native_lib, "mk_rotate_append", a, _cabi.MK_E_INVALID, "k_cache and v_cache share")


def test_null_arguments_and_empty_calls(native_lib):
    for fn in ("mk_plan_step", "mk_rotate_append", "mk_chunk_attention", "mk_sample_tokens"):
        refused(native_lib, fn, None, _cabi.MK_E_INVALID, "null")
    assert native_lib.mk_chunk_attention_workspace(None) == _cabi.MK_E_INVALID
    assert native_lib.mk_op_error(None, 0) == _cabi.MK_E_INVALID
    # no tokens, no requests: nothing to do, and no device is touched
    assert native_lib.mk_rotate_append(C.byref(filled(_cabi.MkRotateAppendArgs, dtype=_cabi.MK_BF16, table_dtype=_cabi.MK_F32, tokens=0)), None) == 0
    assert native_lib.mk_sample_tokens(C.byref(filled(_cabi.MkSampleArgs, dtype=_cabi.MK_F32, requests=0)), None) == 0
    a = filled(_cabi.MkChunkAttentionArgs, dtype=_cabi.MK_BF16, tokens=0)
    assert native_lib.mk_chunk_attention(C.byref(a), None) == 0


def test_workspace_does_not_depend_on_the_data(native_lib):
    """The bytes follow from sizes alone, and a longer batch never needs less."""
    last = 0
    for tokens in (1, 8, 64, 512, 4096):
        a = filled(_cabi.MkChunkAttentionArgs, dtype=_cabi.MK_BF16, tokens=tokens, q_heads=32, kv_heads=8, page_size=64, pages=100, requests=1)
        need = native_lib.mk_chunk_attention_workspace(C.byref(a))
        assert need > 0
        a.workspace = None
        assert native_lib.mk_chunk_attention_workspace(C.byref(a)) == need
        last = max(last, need)
