"""The serving operators at the edges of what their documentation allows, as far as no GPU is needed."""
import ctypes as C
import dataclasses
import os
import random
import socket
import subprocess
import sys

import pytest
import torch
import torch.multiprocessing as mp

import fleet_chiplet_megakernel_b200 as mk
from fleet_chiplet_megakernel_b200 import _cabi
from tests.conftest import ROOT
from tests.test_serving_host import FAKE, filled, refused

NAMES = {"q": "self_attn.q_proj.weight", "k": "self_attn.k_proj.weight", "v": "self_attn.v_proj.weight", "o": "self_attn.o_proj.weight",
         "qn": "self_attn.q_norm.weight", "kn": "self_attn.k_norm.weight", "gate": "mlp.gate_proj.weight", "up": "mlp.up_proj.weight",
         "down": "mlp.down_proj.weight", "ln1": "input_layernorm.weight", "ln2": "post_attention_layernorm.weight"}


# ------------------------------------------------------------------------------------
# MPK.sample_tokens
# ------------------------------------------------------------------------------------
def _wrapper(world_size=1, rank=0, shard_lm_head=True, with_lm_head=True, vocab=2048, padded=0):
    """MPK in mode online_notoken over this rank's shard, built (without a GPU nothing can be compiled)."""
    H, L, n_q, n_kv, mlp = 512, 1, 4, 2, 1024
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    w = {"embed": z(vocab, H), "norm": z(H), "lm_head": z(padded or vocab, H)}
    for s, shape in {"q": (n_q * 128, H), "k": (n_kv * 128, H), "v": (n_kv * 128, H), "o": (H, n_q * 128), "qn": (128,), "kn": (128,), "gate": (mlp, H), "up": (mlp, H),
                     "down": (H, mlp), "ln1": (H,), "ln2": (H,)}.items():
        w[f"l0.{s}"] = z(*shape)
    w = mk.shard_qwen3_weights(w, world_size, rank, shard_lm_head)
    sd = {"model.embed_tokens.weight": w["embed"], "model.norm.weight": w["norm"], "lm_head.weight": w["lm_head"]}
    sd.update({f"model.layers.0.{long}": w[f"l0.{s}"] for s, long in NAMES.items()})
    caches = [z(8, 16, n_kv // world_size, 128) for _ in range(2)]
    config = mk.MirageModelConfig(hidden_size=H, intermediate_size=mlp, vocab_size=vocab, local_num_q_heads=n_q // world_size, local_num_kv_heads=n_kv // world_size,
                                  head_dim=128, num_layers=L, k_cache=caches[:1], v_cache=caches[1:], position_embeddings=(z(64, 128), z(64, 128)), state_dict=sd,
                                  with_lm_head=with_lm_head)
    m = mk.MPK(mk.MPKMetadata(mode="online_notoken", total_num_requests=2, max_seq_length=64, max_num_batched_requests=2, max_num_batched_tokens=2, max_num_pages=8,
                              page_size=16, device="cpu", world_size=world_size, rank=rank, model_config=config, logits=z(2, w["lm_head"].shape[0])))
    m.build()
    return m


def _rank(rank, ws, port, ret):
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    torch.distributed.init_process_group("gloo", rank=rank, world_size=ws)
    said = []
    for shard, padded in ((True, 0), (False, 0), (False, 2304)):
        m = _wrapper(shard_lm_head=shard, world_size=ws, rank=rank, padded=padded)
        try:
            m.sample_tokens(torch.zeros(2))
        except (ValueError, NotImplementedError) as e:
            said.append((type(e).__name__, str(e)))
        m.finalize()
    ret[rank] = said
    torch.distributed.barrier()
    torch.distributed.destroy_process_group()


def test_mpk_draws_from_no_slice_of_the_logits(native_lib):
    """Two ranks: with the head cut by vocabulary rows every rank refuses; with the head whole, padded or not, the call goes on to the operator (which wants a GPU)."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ret = mp.Manager().dict()
    mp.spawn(_rank, args=(2, port, ret), nprocs=2, join=True)
    for rank in (0, 1):
        (kind, text), *whole = ret[rank]
        assert kind == "NotImplementedError" and "1024 of 2048" in text and "sharded" in text
        assert len(whole) == 2 and all(k == "ValueError" and "CUDA" in t for k, t in whole)


def test_mpk_draws_from_no_logits_that_nothing_fills(native_lib):
    m = _wrapper(with_lm_head=False)
    with pytest.raises(ValueError, match="with_lm_head"):
        m.sample_tokens(torch.zeros(2))
    m.finalize()
    m = _wrapper()
    with pytest.raises(ValueError, match="CUDA"):
        m.sample_tokens(torch.zeros(2))
    m.finalize()


# ------------------------------------------------------------------------------------
# arguments of the C entry points
# ------------------------------------------------------------------------------------
def test_arrays_without_entries_need_no_address(native_lib):
    """No rows of logits, no pages: the call goes on to its next check; with one entry an address is needed."""
    refused(native_lib, "mk_sample_tokens", filled(_cabi.MkSampleArgs, dtype=_cabi.MK_F32, logits=None, rows=0, vocab=0), _cabi.MK_E_INVALID, "sizes")
    refused(native_lib, "mk_sample_tokens", filled(_cabi.MkSampleArgs, dtype=_cabi.MK_F32, logits=None, rows=1), _cabi.MK_E_INVALID, "null")
    base = {"dtype": _cabi.MK_BF16, "kv_indices": None, "workspace": None}
    refused(native_lib, "mk_chunk_attention", filled(_cabi.MkChunkAttentionArgs, **base, num_indices=0), _cabi.MK_E_INVALID, "workspace")
    refused(native_lib, "mk_chunk_attention", filled(_cabi.MkChunkAttentionArgs, **base, num_indices=1), _cabi.MK_E_INVALID, "null")


# ------------------------------------------------------------------------------------
# tensors that share memory
# ------------------------------------------------------------------------------------
def _memory(at, reach, sizes, strides):
    v = [at, reach, len(sizes)] + (list(sizes) + [1] * 3)[:3] + (list(strides) + [0] * 3)[:3]
    return (C.c_int64 * 9)(*v)


def _bytes(at, reach, sizes, strides):
    starts = [at]
    for n, s in zip(sizes, strides):
        starts = [x + i * s for x in starts for i in range(n)]
    return {x + k for x in starts for k in range(reach)}


def test_shared_memory_is_found_exactly(native_lib):
    """Against the sets of bytes: slices, permutations and views of other shapes of one buffer, broadcast and empty ones."""
    rng = random.Random(5)
    seen = [0, 0]
    for _ in range(4000):
        def one():
            dims = rng.randint(0, 3)
            strides, at = [], 1
            for _ in range(dims):  # nested, with gaps or without; some of them broadcast
                at *= rng.choice([1, 2, 3, 4, 5, 8])
                strides.append(0 if rng.random() < 0.05 else 4 * at)
            sizes = [rng.choice([0, 1, 2, 3, 4]) if rng.random() < 0.9 else 7 for _ in range(dims)]
            rng.shuffle(strides)
            return 4096 + 4 * rng.randint(0, 60), rng.choice([4, 8, 16]), sizes, strides
        a, b = one(), one()
        if rng.random() < 0.4:  # the same strides, another slice
            b = (b[0], b[1], b[2][: len(a[2])] + [1] * (len(a[2]) - len(b[2])), a[3])
        want = bool(_bytes(*a) & _bytes(*b))
        assert native_lib.mk_debug_share_memory(_memory(*a), _memory(*b)) == want, (a, b)
        assert native_lib.mk_debug_share_memory(_memory(*b), _memory(*a)) == want, (a, b)
        seen[want] += 1
    assert min(seen) > 500


def test_shared_memory_of_real_layouts(native_lib):
    meet = lambda a, b: native_lib.mk_debug_share_memory(_memory(*a), _memory(*b))  # noqa: E731
    T, row = 4096, 256
    base = 0x7f0000000000
    part = lambda first, heads: (base + first * row, row, (T, heads), (48 * row, row))  # noqa: E731 (slices of one projection)
    assert [meet(part(0, 32), part(32, 8)), meet(part(0, 32), part(40, 8)), meet(part(0, 33), part(32, 8)), meet(part(0, 32), part(31, 1))] == [0, 0, 1, 1]
    # K and V interleaved by page, by row and by head; one page, row or head too many
    for strides, gap in (((2 * 64 * 8 * row, 8 * row, row), 64 * 8 * row), ((64 * 16 * row, 16 * row, row), 8 * row), ((64 * 16 * row, 16 * row, 2 * row), row)):
        k, v = (base, row, (1000, 64, 8), strides), (base + gap, row, (1000, 64, 8), strides)
        assert meet(k, v) == 0 and meet(k, (base + gap - 2, row, (1000, 64, 8), strides)) == 1
        assert meet(k, (base + strides[0], row, (1000, 64, 8), strides)) == 1
    # two caches whose pages are 2 GB apart, an output inside the gap and one that is not
    far = (base, row, (6, 16, 2), (1 << 31, 2 * row, row))
    assert meet(far, (base + (1 << 30), row, (6, 16, 2), far[3])) == 0
    assert meet(far, (base + 32 * row, row, (1000, 32), (32 * row, row))) == 0 and meet(far, (base + 31 * row, row, (1000, 32), (32 * row, row))) == 1
    # strides that no address has
    assert meet((base, row, (1 << 31, 1 << 31), (1 << 62, 1 << 62)), (base - row, row, (), ())) == 0


def test_operators_refuse_what_shares_memory(native_lib):
    """Every tensor that is written with every other of the call, at one element past its beginning (all other tensors are apart)."""
    for cls, fn, written, more in (
            (_cabi.MkRotateAppendArgs, "mk_rotate_append", ("out", "k_cache", "v_cache"),
             dict(dtype=_cabi.MK_BF16, table_dtype=_cabi.MK_F32, q_stride=(128, 128), k_stride=(128, 128), v_stride=(128, 128), out_stride=(128, 128), table_stride=(128, 128),
                  k_cache_stride=(128, 128, 128), v_cache_stride=(128, 128, 128), tokens=8)),
            (_cabi.MkChunkAttentionArgs, "mk_chunk_attention", ("out", "lse", "workspace"),
             dict(dtype=_cabi.MK_BF16, q_stride=(128, 128), out_stride=(128, 128), lse_stride=(1, 1), k_cache_stride=(128, 128, 128), v_cache_stride=(128, 128, 128),
                  workspace_bytes=1 << 40, tokens=8, requests=8, num_indices=8)),
            (_cabi.MkSampleArgs, "mk_sample_tokens", ("tokens", "logprobs"), dict(dtype=_cabi.MK_F32, rows=8, requests=8, vocab=8, row_stride=8))):
        names = [n for n, kind in cls._fields_ if kind is C.c_void_p]
        apart = {n: FAKE + (k << 26) for k, n in enumerate(names)}
        for name in written:
            for other in names:
                if other == name or (name, other) == ("out", "q") and cls is _cabi.MkRotateAppendArgs:
                    continue
                refused(native_lib, fn, filled(cls, **{**apart, **more, other: apart[name] + 16}), _cabi.MK_E_INVALID, "share memory")
    # out may be q, but not q moved by a row
    base = dict(dtype=_cabi.MK_BF16, table_dtype=_cabi.MK_F32, q_stride=(128, 128), out_stride=(128, 128), tokens=8)
    names = [n for n, kind in _cabi.MkRotateAppendArgs._fields_ if kind is C.c_void_p]
    apart = {n: FAKE + (k << 26) for k, n in enumerate(names)}
    refused(native_lib, "mk_rotate_append", filled(_cabi.MkRotateAppendArgs, **{**apart, **base, "out": apart["q"] + 256}), _cabi.MK_E_INVALID, "out and q share")


# ------------------------------------------------------------------------------------
# the binding
# ------------------------------------------------------------------------------------
def test_the_binding_shares_the_process_c_plus_plus_runtime(native_lib):
    """torch's macros format numbers through a C++ stream in the module; with a runtime of its own (linked statically) that ends the process."""
    code = "import torch, fleet_chiplet_megakernel_b200.serving as s\ntry: s._load().plan_step(1, 2, 3)\nexcept RuntimeError as e: print(e)"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert r.returncode == 0 and "3 arguments, 14 are needed" in r.stdout, (r.returncode, r.stdout, r.stderr)


# ------------------------------------------------------------------------------------
# the workspace of chunk_attention
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("page,max_new", [(64, 0), (64, 1), (12, 0)])
def test_workspace_follows_from_the_shapes_alone(native_lib, page, max_new):
    """It may be asked for before there is any memory, and has to be asked for every shape: chunks of few rows are cut into pieces, longer ones are not."""
    row = 8 * 128
    need = {}
    for tokens in (1, 8, 64, 512, 4096):
        a = filled(_cabi.MkChunkAttentionArgs, dtype=_cabi.MK_BF16, tokens=tokens, q_heads=32, kv_heads=8, page_size=page, pages=100, requests=1, max_new=max_new, scale=0.1, window=0, sinks=0,
                   q_stride=(32 * 128, 128), out_stride=(32 * 128, 128), k_cache_stride=(page * row, row, 128), v_cache_stride=(page * row, row, 128))
        need[tokens] = native_lib.mk_chunk_attention_workspace(C.byref(a))
        assert need[tokens] > 0
        for name, kind in _cabi.MkChunkAttentionArgs._fields_:
            if kind is C.c_void_p:
                setattr(a, name, None)
        assert native_lib.mk_chunk_attention_workspace(C.byref(a)) == need[tokens]
    if page == 64 and max_new == 0:
        tile = lambda tokens, splits: splits * tokens * 32 * 130 * 4  # noqa: E731 (as many pieces as there are SMs for, of 64 tokens and a kv head each)
        assert need[64] == tile(64, 16) and need[512] == tile(512, 2) and need[4096] == 16 and need[8] < need[64] > need[4096]
    else:
        assert len(set(need.values())) <= 2  # of the kernel for few rows: a share per SM


def test_operators_refuse_addresses_between_elements(native_lib):
    """Every pointer of every call, one byte on (all tensors are apart): the kernels' loads want whole elements."""
    for cls, fn, more in ((_cabi.MkStepPlanArgs, "mk_plan_step", dict(table_stride=1)),
                          (_cabi.MkRotateAppendArgs, "mk_rotate_append", dict(dtype=_cabi.MK_BF16, table_dtype=_cabi.MK_F32)),
                          (_cabi.MkChunkAttentionArgs, "mk_chunk_attention", dict(dtype=_cabi.MK_BF16, workspace_bytes=1 << 40)),
                          (_cabi.MkSampleArgs, "mk_sample_tokens", dict(dtype=_cabi.MK_BF16))):
        names = [n for n, kind in cls._fields_ if kind is C.c_void_p]
        apart = {n: FAKE + (k << 26) for k, n in enumerate(names)}
        for name in names:
            refused(native_lib, fn, filled(cls, **{**apart, **more, name: apart[name] + 1}), _cabi.MK_E_INVALID, "aligned" if name in ("q", "out", "k_cache", "v_cache", "workspace") and cls is _cabi.MkChunkAttentionArgs else "multiple of")


def test_mpk_metadata_keeps_the_order_of_its_fields():
    """By position, the fields that were there before stand where they stood: what is new comes last."""
    names = [f.name for f in dataclasses.fields(mk.MPKMetadata)]
    assert names[-4:] == ["use_cutlass_kernel", "eos_token_id", "extra", "logits"]
    values = [None] * (len(names) - 1)
    values[-1] = {"numerics": "mpk"}
    assert mk.MPKMetadata(*values).extra == {"numerics": "mpk"} and mk.MPKMetadata(*values).logits is None


def test_a_vocabulary_beyond_the_counters_is_a_limit_and_no_mistake(native_lib):
    refused(native_lib, "mk_sample_tokens", filled(_cabi.MkSampleArgs, dtype=_cabi.MK_F32, vocab=1 << 30), _cabi.MK_E_TOO_LARGE, "vocabulary")
