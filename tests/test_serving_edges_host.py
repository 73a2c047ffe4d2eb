"""The serving operators at the edges of what their documentation allows, as far as no GPU is needed."""
import ctypes as C
import os
import socket

import pytest
import torch
import torch.multiprocessing as mp

import fleet_chiplet_megakernel_b200 as mk
from fleet_chiplet_megakernel_b200 import _cabi
from tests.test_serving_host import filled, refused

NAMES = {"q": "self_attn.q_proj.weight", "k": "self_attn.k_proj.weight", "v": "self_attn.v_proj.weight", "o": "self_attn.o_proj.weight",
         "qn": "self_attn.q_norm.weight", "kn": "self_attn.k_norm.weight", "gate": "mlp.gate_proj.weight", "up": "mlp.up_proj.weight",
         "down": "mlp.down_proj.weight", "ln1": "input_layernorm.weight", "ln2": "post_attention_layernorm.weight"}


# ------------------------------------------------------------------------------------
# MPK.sample_tokens
# ------------------------------------------------------------------------------------
def _wrapper(world_size=1, rank=0, shard_lm_head=True, with_lm_head=True, vocab=2048):
    """MPK in mode online_notoken over this rank's shard, built (without a GPU nothing can be compiled)."""
    H, L, n_q, n_kv, mlp = 512, 1, 4, 2, 1024
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    w = {"embed": z(vocab, H), "norm": z(H), "lm_head": z(vocab, H)}
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
    for shard in (True, False):
        m = _wrapper(shard_lm_head=shard, world_size=ws, rank=rank)
        try:
            m.sample_tokens(torch.zeros(2))
        except (ValueError, NotImplementedError) as e:
            said.append((type(e).__name__, str(e)))
        m.finalize()
    ret[rank] = said
    torch.distributed.barrier()
    torch.distributed.destroy_process_group()


def test_mpk_draws_from_no_slice_of_the_logits(native_lib):
    """Two ranks: with the head cut by vocabulary rows every rank refuses; with the head whole the call goes on to the operator (which wants a GPU)."""
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ret = mp.Manager().dict()
    mp.spawn(_rank, args=(2, port, ret), nprocs=2, join=True)
    for rank in (0, 1):
        (kind, text), (kind_whole, text_whole) = ret[rank]
        assert kind == "NotImplementedError" and "1024 of 2048" in text and "sharded" in text
        assert kind_whole == "ValueError" and "CUDA" in text_whole


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
