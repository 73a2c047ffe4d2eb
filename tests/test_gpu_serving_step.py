"""The serving operators as an engine uses them: around passes of the megakernel over one cache, in captured graphs, on several
streams; and what they refuse of tensors on the GPU."""
import math

import pytest
import torch

import fleet_chiplet_megakernel_b200 as mk
from oracle import qwen3_oracle as O
from tests.test_gpu_serving import Batch, check_sample, gen, i32, rnd, sample_reference

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
TOL = 2e-2  # logits against the oracle, of the row's largest: the megakernel's own
D = 128

NAMES = {"q": "self_attn.q_proj.weight", "k": "self_attn.k_proj.weight", "v": "self_attn.v_proj.weight", "o": "self_attn.o_proj.weight",
         "qn": "self_attn.q_norm.weight", "kn": "self_attn.k_norm.weight", "gate": "mlp.gate_proj.weight", "up": "mlp.up_proj.weight",
         "down": "mlp.down_proj.weight", "ln1": "input_layernorm.weight", "ln2": "post_attention_layernorm.weight"}


class Engine:
    """MPK in mode online_notoken over paging state that lives here."""

    def __init__(self, requests, budget, pool, page, max_seq):
        self.geom, self.page, self.requests, self.max_seq = O.TINY, page, requests, max_seq
        self.w = O.make_weights(self.geom, 0, norm_jitter=0.25)
        self.dw = {k: v.cuda() for k, v in self.w.items()}
        g = self.geom
        sd = {"model.embed_tokens.weight": self.dw["embed"], "model.norm.weight": self.dw["norm"], "lm_head.weight": self.dw["lm_head"]}
        for i in range(g.layers):
            for s, l in NAMES.items():
                sd[f"model.layers.{i}.{l}"] = self.dw[f"l{i}.{s}"]
        self.kc = [torch.full((pool, page, g.n_kv, D), math.nan, dtype=BF, device="cuda") for _ in range(g.layers)]
        self.vc = [torch.full_like(t, math.nan) for t in self.kc]
        self.cos, self.sin = mk.qwen3_graph.rope_tables(mk.Qwen3Geometry(), max_seq, "cuda")
        self.logits = torch.zeros(budget, g.vocab, dtype=BF, device="cuda")
        config = mk.MirageModelConfig(hidden_size=g.hidden, intermediate_size=g.mlp, vocab_size=g.vocab, local_num_q_heads=g.n_q, local_num_kv_heads=g.n_kv,
                                      head_dim=D, num_layers=g.layers, k_cache=self.kc, v_cache=self.vc, position_embeddings=(self.cos, self.sin), state_dict=sd)
        self.m = mk.MPK(mk.MPKMetadata(mode="online_notoken", total_num_requests=requests, max_seq_length=max_seq, max_num_batched_requests=requests,
                                       max_num_batched_tokens=budget, max_num_pages=pool, page_size=page, model_config=config, logits=self.logits,
                                       extra={"numerics": "mpk"}))
        self.m.build()
        self.m.compile()
        self.lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.table = torch.zeros(requests, -(-max_seq // page), dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(pool, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        self.free = torch.tensor([0, pool], dtype=torch.int64, device="cuda")

    def plan(self, new, run=None):
        """Plans a step, takes it over into the paging state and returns the granted tokens."""
        new = i32(new)
        p = self.m.plan_step(self.lengths, new, self.table, self.ring, self.free) if run is None else run(new)
        self.lengths = torch.where(new < 0, 0, self.lengths + p.granted).to(torch.int32)
        self.free = p.free_range.clone()
        return p.granted.tolist()


def test_a_server_of_megakernel_passes():
    """Requests of all ages through plan, pass and sampling: prompts in chunks, a request that waits for pages, one that ends and hands its pages on, a new one in its
    place.  Logits against the oracle, tokens against the definition of sampling on those logits."""
    page = 8
    e = Engine(requests=3, budget=8, pool=7, page=page, max_seq=40)
    prompts = {0: [5, 9, 2, 77, 31, 8, 4, 100, 3], 1: [11, 12, 13], 2: [400, 401, 402, 403, 404]}
    g = gen(3)
    seqs, refs, fed, settings = {}, {}, {}, {0: (0.0, 0, 1.0, 0.0), 1: (0.8, 20, 0.9, 0.0), 2: (1.2, 0, 1.0, 0.05)}

    def begin(slot, tokens):
        seqs[slot], fed[slot] = list(tokens), 0
        refs[slot] = O.MpkRefModel(e.geom, e.w, e.max_seq)

    for slot in prompts:
        begin(slot, prompts[slot])
    waited = ended = 0
    for step in range(26):
        new, budget = [], 8
        for r in range(3):
            left = min(len(seqs[r]) - fed[r], 4, budget)
            new.append(left)
            budget -= left
        if step == 12:
            new[1] = -1  # request 1 ends; its pages are free in this step already
            ended += 1
        granted = e.plan(new)
        waited += sum(1 for a, b in zip(granted, new) if a < max(b, 0))
        rows = [t for r in range(3) for t in seqs[r][fed[r]:fed[r] + granted[r]]]
        e.m.input_tokens[: len(rows), 0] = torch.tensor(rows, dtype=torch.int64, device="cuda")
        e.m()
        t, k, p, m = (torch.tensor([settings[r][i] for r in range(3)], device="cuda") for i in range(4))
        u = torch.rand(3, generator=g, device="cuda")
        tokens, _ = e.m.sample_tokens(u, t, k.to(torch.int32), p, m, return_logprobs=True)
        tokens = tokens.tolist()
        at = 0
        for r in range(3):
            for i in range(fed[r], fed[r] + granted[r]):
                want = refs[r].step(seqs[r][i], i)
            at += granted[r]
            fed[r] += granted[r]
            if not granted[r]:
                assert tokens[r] == -1
                continue
            row = e.logits[at - 1]
            assert O.max_rel_err(row.cpu()[None], want[None]) < TOL, f"step {step}, request {r}"
            assert tokens[r] == sample_reference(row, u[r], *settings[r])[0]
            if fed[r] == len(seqs[r]) and len(seqs[r]) < 30:
                seqs[r].append(tokens[r])
        if step == 12:
            begin(1, [900, 901, 902, 903, 904, 905])
    assert waited > 0 and ended and len(seqs[1]) > 6 and len(seqs[0]) > 12
    e.m.finalize()


def _prefill_by_operators(e, plan, tokens):
    """The model's layers over the planned rows, by torch's products and the serving operators, in the megakernel's roundings."""
    g, w = e.geom, e.dw
    T = len(tokens)

    def norm(x, weight):
        f = x.float()
        return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * weight.float()).to(BF)

    x = w["embed"][torch.tensor(tokens, device="cuda")]
    for i in range(g.layers):
        h = norm(x, w[f"l{i}.ln1"])
        q, k, v = ((h @ w[f"l{i}.{n}"].T).view(T, -1, D) for n in "qkv")
        q = mk.rotate_append(q, k, v, e.cos, e.sin, plan.positions[:T], plan.slots[:T], e.kc[i], e.vc[i], w[f"l{i}.qn"], w[f"l{i}.kn"], eps=1e-6)
        a = mk.chunk_attention(q, e.kc[i], e.vc[i], plan.qo_indptr, plan.kv_indptr, plan.kv_indices, plan.last_page_len)
        x = x + a.view(T, -1) @ w[f"l{i}.o"].T
        h = norm(x, w[f"l{i}.ln2"])
        x = x + (torch.nn.functional.silu((h @ w[f"l{i}.gate"].T).float()) * (h @ w[f"l{i}.up"].T).float()).to(BF) @ w[f"l{i}.down"].T
    return norm(x, w["norm"]) @ w["lm_head"].T


@pytest.mark.parametrize("page", [8, 16, 64])
def test_prompts_by_operators_and_tokens_by_the_megakernel(page):
    """Long prompts through the operators in one chunk each (beside a request that is already decoding), then passes of the megakernel over the same cache."""
    e = Engine(requests=3, budget=8, pool=600 // page + 6, page=page, max_seq=260)
    big = mk.StepPlan.empty(3, 512, e.ring.shape[0])
    prompts = [O.make_prompt(e.geom, n, r).tolist() for r, n in enumerate((150, 37, 201))]
    refs = [O.MpkRefModel(e.geom, e.w, e.max_seq) for _ in prompts]

    def step(feed):
        granted = e.plan([len(f) for f in feed], lambda new: mk.plan_step(e.lengths, new, e.table, e.ring, e.free, page, big))
        assert granted == [len(f) for f in feed]
        logits = _prefill_by_operators(e, big, sum(feed, []))
        ends = big.qo_indptr.tolist()
        return logits, [ends[r + 1] - 1 for r in range(3)]

    step([[], prompts[1], []])
    logits, last = step([prompts[0], [7], prompts[2]])  # a chunk, one token, a chunk
    sent = [prompts[0], prompts[1] + [7], prompts[2]]
    for r, ref in enumerate(refs):
        for i, t in enumerate(sent[r]):
            want = ref.step(t, i)
        assert O.max_rel_err(logits[last[r]].cpu()[None], want[None]) < TOL, f"request {r} behind the operators"
    tokens = mk.sample_tokens(logits, torch.zeros(3, device="cuda"), 0.0, qo_indptr=big.qo_indptr).tolist()
    assert tokens == [int(logits[i].argmax()) for i in last]
    for n in range(4):  # the megakernel goes on from what the operators have left in the cache
        assert e.plan([1, 1, 1]) == [1, 1, 1]
        e.m.input_tokens[:3, 0] = torch.tensor(tokens, device="cuda")
        e.m()
        for r, ref in enumerate(refs):
            want = ref.step(tokens[r], len(sent[r]))
            sent[r].append(tokens[r])
            assert O.max_rel_err(e.logits[r].cpu()[None], want[None]) < TOL, f"request {r}, token {n} by the megakernel"
        tokens = e.m.sample_tokens(torch.zeros(3, device="cuda"), 0.0).tolist()
    e.m.finalize()


def test_mpk_refuses_what_its_mode_does_itself():
    e = Engine(requests=1, budget=2, pool=4, page=16, max_seq=40)
    e.m.metadata.logits = None
    with pytest.raises(ValueError, match="logits"):
        e.m.sample_tokens(torch.zeros(1, device="cuda"))
    e.m.metadata.mode = "offline"
    with pytest.raises(ValueError, match="offline"):
        e.m.plan_step(e.lengths, i32([1]), e.table, e.ring, e.free)
    e.m.finalize()


# ------------------------------------------------------------------------------------
# graphs, streams
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("requests", [[(300, 1), (17, 1), (1000, 1)], [(200, 130), (0, 1), (64, 64)], [(0, 300)]])
def test_attention_in_captured_graphs(requests):
    """Two graphs with workspaces of their own, replayed in turn and at once on two streams with new inputs, give what eager calls give."""
    bs = [Batch(requests, 8, 2, 16, seed=s) for s in (0, 1)]
    for b in bs:
        b.run()
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for b in bs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.run()
        graphs.append(g)
    for turn in range(3):
        for k, b in enumerate(bs):
            b.q.copy_(rnd(gen(10 * turn + k), *b.q.shape))
        want = [b.run().clone() for b in bs]
        for b in bs:
            b.out[: b.qo[-1]] = 0
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for b, w in zip(bs, want):
            assert torch.equal(b.out, w)


def test_a_step_in_one_graph():
    """Plan, append, attention and sampling captured together; replays follow the lengths that the inputs hold."""
    g = gen(2)
    R, page, pool, n_q, n_kv, V = 4, 16, 40, 8, 2, 5000
    lengths, new = i32([0, 33, 15, 64]), i32([20, 1, 1, 1])
    table = torch.zeros(R, 10, dtype=torch.int32, device="cuda")
    ring = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    free = torch.tensor([0, pool], dtype=torch.int64, device="cuda")
    first = mk.StepPlan.empty(R, 200, pool)
    mk.plan_step(i32([0] * R), lengths, table, ring, free, page, first)  # pages for what is there already
    free = first.free_range.clone()
    plan = mk.StepPlan.empty(R, 32, pool)
    kc, vc = (rnd(g, pool, page, n_kv, D) for _ in range(2))
    qkv = rnd(g, 32, n_q + 2 * n_kv, D)
    q, k, v = qkv[:, :n_q], qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:]
    ang = torch.rand(200, D, generator=g, device="cuda") * 6
    logits, u = rnd(g, 32, V, dtype=torch.float32, scale=3.0), torch.rand(R, generator=g, device="cuda")

    def step():
        mk.plan_step(lengths, new, table, ring, free, page, plan)
        x = mk.rotate_append(q, k, v, ang.cos(), ang.sin(), plan.positions, plan.slots, kc, vc)
        o = mk.chunk_attention(x, kc, vc, plan.qo_indptr, plan.kv_indptr, plan.kv_indices, plan.last_page_len)
        return o, mk.sample_tokens(logits, u, 0.9, 40, 0.95, qo_indptr=plan.qo_indptr)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, tokens = step()
    for n in ([20, 1, 1, 1], [1, 0, 9, 1], [0, 1, 1, 0], [5, 5, 5, 5]):
        new.copy_(i32(n))
        u.copy_(torch.rand(R, generator=g, device="cuda"))
        graph.replay()
        got, got_tokens, granted = out.clone(), tokens.clone(), plan.granted.tolist()
        assert granted == n
        want, want_tokens = step()
        assert torch.equal(got, want) and torch.equal(got_tokens, want_tokens)
        assert [t >= 0 for t in got_tokens.tolist()] == [x > 0 for x in n]


def test_calls_on_several_streams():
    """The same operators on three streams at once, each with tensors of its own."""
    streams = [torch.cuda.Stream() for _ in range(3)]
    bs = [Batch([(900, 1), (40, 120), (333, 2)], 8, 2, 16, seed=s) for s in range(3)]
    want = [b.run().clone() for b in bs]
    logits, u = rnd(gen(5), 6, 32008, dtype=torch.float32, scale=3.0), torch.rand(6, generator=gen(6), device="cuda")
    tokens = mk.sample_tokens(logits, u, 0.8, 50, 0.9)
    for b in bs:
        b.out[: b.qo[-1]] = 0
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for s, b in zip(streams, bs):
            with torch.cuda.stream(s):
                b.run()
                got.append(mk.sample_tokens(logits, u, 0.8, 50, 0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(b.out, w) for b, w in zip(bs, want)) and all(torch.equal(t, tokens) for t in got)


def test_sampling_settings_as_numbers_and_as_tensors():
    g = gen(8)
    logits, u = rnd(g, 5, 3001, dtype=torch.float16, scale=3.0), torch.rand(5, generator=g, device="cuda")
    full = lambda x, dt=torch.float32: torch.full((5,), x, dtype=dt, device="cuda")  # noqa: E731
    a = mk.sample_tokens(logits, u, 0.7, 30, 0.9, 0.01)
    b = mk.sample_tokens(logits, u, full(0.7), full(30, torch.int32), full(0.9), full(0.01))
    out = torch.zeros(5, dtype=torch.int64, device="cuda")
    assert mk.sample_tokens(logits, u, 0.7, 30, 0.9, 0.01, out=out) is not None
    assert torch.equal(a, b) and torch.equal(a, out)
    check_sample(logits, u, 1.0, 0, 1.0, 2.0)  # min_p above 1: the largest alone
    check_sample(logits, u, 1.0, -3, 1.0, 0.0)


# ------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------
def test_attention_refusals():
    b = Batch([(40, 2), (3, 1)], 8, 2, 16)
    ok = dict(q=b.q, k_cache=b.k, v_cache=b.v, qo_indptr=b.qo_indptr, kv_indptr=b.kv_indptr, kv_indices=b.kv_indices, last_page_len=b.last)
    before = b.out.clone()
    wide = torch.zeros(3, 8, 132, dtype=BF, device="cuda")
    for change, text in [(dict(q=b.q.float()), "bf16 or fp16"), (dict(q=b.q.half()), "dtype"), (dict(q=b.q[:, :7]), "7 q heads"), (dict(q=b.q[..., :64]), "128"),
                         (dict(k_cache=b.k[:, :, :1]), "v_cache"), (dict(kv_indices=b.kv_indices.long()), "dtype"), (dict(qo_indptr=b.qo_indptr[:2]), "qo_indptr"),
                         (dict(last_page_len=b.last[None]), "one dimension"), (dict(window=-1), "window"), (dict(sinks=-2), "sinks"), (dict(out=b.q), "may not be q"),
                         (dict(out=b.out[:1].expand(3, 8, D)), "share memory"), (dict(out=b.out.cpu()), "is on cpu"), (dict(lse=torch.zeros(3, 7, device="cuda")), "lse"),
                         (dict(lse=torch.zeros(3, 1, device="cuda").expand(3, 8)), "share memory"),
                         (dict(q=wide[..., :D]), "multiples of 16 bytes"), (dict(kv_indices=torch.zeros(40, dtype=torch.int32, device="cuda")[::2]), "contiguous"),
                         (dict(q=[1]), "tensor is needed"), (dict(q=b.q.clone().requires_grad_()), "gradient")]:
        with pytest.raises(ValueError, match=text):
            mk.chunk_attention(**{**ok, "out": b.out, **change})
    assert torch.equal(b.out, before)
    with torch.no_grad():
        mk.chunk_attention(**{**ok, "q": b.q.clone().requires_grad_()})
    assert mk.chunk_attention(**{**ok, "q": b.q[:0]}).shape == (0, 8, D)
    with pytest.raises(NotImplementedError, match="requests"):
        big = torch.zeros(5001, dtype=torch.int32, device="cuda")
        mk.chunk_attention(**{**ok, "qo_indptr": big, "kv_indptr": big, "last_page_len": big[:5000]})


def test_other_refusals():
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    plan = mk.StepPlan.empty(2, 4, 8)
    ok = dict(lengths=i32([1, 2]), new_tokens=i32([1, 1]), block_table=z(2, 3, dt=torch.int32), free_pages=i32([5, 6]), free_range=z(2, dt=torch.int64), page_size=4, plan=plan)
    for change, text in [(dict(new_tokens=i32([1])), "new_tokens"), (dict(block_table=z(3, 3, dt=torch.int32)), "block_table"), (dict(page_size=0), "page_size"),
                         (dict(free_range=plan.free_range), "may not be"), (dict(plan=None), "StepPlan"), (dict(block_table=z(1, 3, dt=torch.int32).expand(2, 3)), "apart"),
                         (dict(lengths=torch.ones(2, device="cuda")), "dtype"), (dict(new_tokens=plan.granted), "granted and new_tokens share"),
                         (dict(lengths=plan.positions[1:3]), "positions and lengths share"), (dict(free_pages=plan.kv_indices), "free_pages and kv_indices share")]:
        with pytest.raises(ValueError, match=text):
            mk.plan_step(**{**ok, **change})
    qq = z(3, 4, D, dt=BF)
    q, kv, cache, t = z(3, 4, D, dt=BF), z(3, 2, D, dt=BF), z(2, 4, 2, D, dt=BF), z(9, D, dt=BF)
    ok = dict(q=q, k=kv, v=kv, cos=t, sin=t, positions=i32([0, 1, 2]), slots=z(3, dt=torch.int64), k_cache=cache, v_cache=cache.clone())
    for change, text in [(dict(k=kv[:2]), "k.shape"), (dict(v=z(3, 1, D, dt=BF)), "v.shape"), (dict(cos=t.half()), "dtype"), (dict(sin=t[:4]), "sin"),
                         (dict(positions=z(3, dt=torch.int64)), "dtype"), (dict(k_cache=z(2, 4, 1, D, dt=BF)), "kv heads"), (dict(q_norm=z(64, dt=BF)), "q_norm"),
                         (dict(k_cache=cache[:1].expand(2, 4, 2, D)), "share memory"), (dict(out=z(3, 4, D)), "dtype"),
                         (dict(v_cache=cache), "k_cache and v_cache share"), (dict(q=qq, out=qq.as_strided((3, 4, D), (D, 3 * D, 1))), "other strides")]:
        with pytest.raises(ValueError, match=text):
            mk.rotate_append(**{**ok, **change})
    for args, text in [((z(2, 9).double(), z(2)), "fp32"), ((z(2, 9), z(3)), "rows of logits"), ((z(2, 9), z(2).double()), "dtype"), ((z(9), z(1)), "vocab"),
                       ((z(2, 9), z(2), z(3)), "temperature"), ((z(2, 9), z(2), 1.0, z(2)), "top_k"), ((z(9, 2).T, z(2)), "contiguous")]:
        with pytest.raises(ValueError, match=text):
            mk.sample_tokens(*args)
    assert mk.sample_tokens(z(0, 9), z(0)).shape == (0,)
