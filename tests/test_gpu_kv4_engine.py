"""The engine with its cache held in 4 bits and with drawn tokens (MI355X).

Logits of the 4-bit path are compared with the same model and the same cache
contents under a plain float32 attention over the stored values, read back row
by row: the bound is the engine tests' own (fp16 activations rounded after every
operation, 1e-2 of the largest logit).  Tokens are held to the float64 sampler
on the very logits that they were drawn from.
"""

from __future__ import annotations

import pytest
import torch

from nanoserve_amd import Int4PagedKVCache, gather_cache_int4
from nanoserve_amd.attention import get_attention_backend
from nanoserve_amd.block_manager import BlockSpaceManager
from nanoserve_amd.engine import LLMEngine, ModelRunner, SamplingParams, SchedulerConfig, Sequence
from nanoserve_amd.kv_cache import PagedKVCache
from nanoserve_amd.model import Qwen2Config, Qwen2ForCausalLM, random_init_
from nanoserve_amd.quant import quantize_model
from oracle.qwen2 import relative_error
from oracle.sampling import sample_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 1e-2
# Head size 64, two query heads per KV head.
TINY = dict(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2,
            num_attention_heads=4, num_key_value_heads=2, rope_theta=10000.0, tie_word_embeddings=False)


def _model(dtype=torch.float16, int4=True, seed=0, kv_bits=4, cfg=TINY):
    m = random_init_(Qwen2ForCausalLM(Qwen2Config(**cfg), max_position=2048), std=0.05, seed=seed).to(dtype).to(DEV)
    if int4:
        quantize_model(m, 128)
    return m.fuse_projections(kv_bits=kv_bits).eval().requires_grad_(False)


def _tokens(n, seed, vocab=512):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _runner(model, num_blocks=64, block_size=16, cache=Int4PagedKVCache, **kw):
    c = cache(num_blocks, block_size, model.num_layers, model.num_kv_heads, model.head_dim,
              model.model.embed_tokens.weight.dtype, DEV)
    return ModelRunner(model, c, BlockSpaceManager(block_size, num_blocks, watermark=0.0), DEV, **kw)


def _seq(i, tokens, max_new=8, **sampling):
    return Sequence(i, list(tokens), SamplingParams(max_new_tokens=max_new, ignore_eos=True, **sampling))


def _attention_over_stored_values(query, kc, vc, md, scale):
    """attn_fn in float32 over the rows that gather_cache_int4 reads back."""
    bs, out = kc.shape[2], torch.empty_like(query)
    for i in range(md.num_seqs):
        a, b = md.query_start_loc_cpu[i:i + 2]
        n, ql = md.seq_lens_cpu[i], b - a
        pos = torch.arange(n, device=DEV)
        slots = md.block_tables[i][pos // bs].long() * bs + pos % bs
        k, v = (x.float() for x in gather_cache_int4(kc, vc, slots, query.dtype))
        q = query[a:b].float().view(ql, k.shape[1], -1, query.shape[2])
        s = (q[:, :, :, None] * k.transpose(0, 1)[None, :, None]).sum(-1) * scale
        seen = pos <= (n - ql + torch.arange(ql, device=DEV))[:, None]
        p = s.masked_fill(~seen[:, None, None], -torch.inf).softmax(-1)
        out[a:b] = (p[..., None] * v.transpose(0, 1)[None, :, None]).sum(3).reshape(ql, -1, query.shape[2])
    return out


@torch.inference_mode()
def _step(runner, plan, attn_fn=None):
    for s, q in plan:
        assert runner.block_manager.allocate(s, s.num_computed_tokens + q)
    ids, pos, md, si, _ = runner.build_inputs(plan)
    hidden = runner.model(ids, pos, runner.kv_cache, md, attn_fn or runner.attn_fn)
    for s, q in plan:
        s.mark_computed(q)
    return runner.model.compute_logits(hidden, si)


@pytest.mark.parametrize("dtype,int4,block,kv_bits", [(torch.float16, True, 16, 4), (torch.float16, True, 16, 16),
                                                      (torch.float16, False, 32, 4), (torch.bfloat16, True, 16, 4),
                                                      (torch.float16, True, 8, 4)])
def test_forward_matches_attention_over_the_stored_values(dtype, int4, block, kv_bits):
    """kv_bits 16: projections fused for the 16-bit cache's epilogue serve the 4-bit one too."""
    model = _model(dtype, int4, kv_bits=kv_bits)
    got, want = (_runner(model, block_size=block) for _ in range(2))
    tol = TOL if dtype == torch.float16 else 3 * TOL
    seqs = [[_seq(i, _tokens(n, i)) for i, n in enumerate((21, 90, 33))] for _ in range(2)]
    plans = [[(0, 21), (1, 50)], [(0, 1), (1, 40), (2, 33)], [(0, 1), (1, 1), (2, 1)]]
    for step, plan in enumerate(plans):
        if step:
            for pair in seqs:
                for i, _ in plan:
                    if pair[i].num_computed_tokens == pair[i].num_tokens:
                        pair[i].output_token_ids.append(7 + i)
        a = _step(got, [(seqs[0][i], q) for i, q in plan])
        b = _step(want, [(seqs[1][i], q) for i, q in plan], _attention_over_stored_values)
        assert relative_error(a, b.float().cpu()) < tol, f"step {step}"
    # Later layers' rows follow from earlier layers' attention; the first layer's are the same bytes.
    assert torch.equal(got.kv_cache.k_cache[0], want.kv_cache.k_cache[0])


def test_chunked_prefill_and_graphs_agree_with_one_shot():
    model = _model()
    toks = _tokens(100, 3)
    one = _runner(model)
    want = _step(one, [(_seq(0, toks), 100)])
    chunked, s = _runner(model), _seq(0, toks)
    for q in (33, 1, 66):
        got = _step(chunked, [(s, q)]) if s.num_computed_tokens + q == 100 else _chunk(chunked, s, q)
    assert relative_error(got, want.float().cpu()) < TOL
    # A captured decode step against an eager one.
    graphed = _runner(model, use_graphs=True, max_model_len=512, graph_batch_sizes=(1, 2))
    sg, se = _seq(0, toks), _seq(0, toks)
    _step(graphed, [(sg, 100)])
    eager = _runner(model)
    _step(eager, [(se, 100)])
    for step in range(4):
        sg.output_token_ids.append(5 + step)
        se.output_token_ids.append(5 + step)
        want = _step(eager, [(se, 1)])
        assert graphed.block_manager.allocate(sg, sg.num_computed_tokens + 1)
        (_, tok), = graphed.execute([(sg, 1)])
        logits = graphed.graphs.last_logits
        assert relative_error(logits, want.float().cpu()) < TOL
        assert tok == int(logits.argmax())


@torch.inference_mode()
def _chunk(runner, s, q):
    assert runner.block_manager.allocate(s, s.num_computed_tokens + q)
    ids, pos, md, _, _ = runner.build_inputs([(s, q)])
    runner.model(ids, pos, runner.kv_cache, md, runner.attn_fn)
    s.mark_computed(q)


_LENS = [(5, 6), (33, 3), (17, 9), (70, 4), (2, 12), (40, 7)]  # (prompt, output) lengths


def _run(model, sampling, kv_bits=4, num_blocks=64, graphs=True, pipeline=True, max_tokens=64):
    eng = LLMEngine(model, num_blocks=num_blocks, block_size=16, device=DEV,
                    scheduler_config=SchedulerConfig(max_num_batched_tokens=max_tokens, max_num_seqs=8),
                    max_model_len=256, use_graphs=graphs, pipeline_decode=pipeline, kv_bits=kv_bits)
    for i, (p, n) in enumerate(_LENS):
        eng.add_request(_tokens(p, 400 + i), SamplingParams(max_new_tokens=n, ignore_eos=True, **sampling(i)))
    out = eng.run_all()
    assert [len(s.output_token_ids) for s in out] == [n for _, n in _LENS]
    assert eng.block_manager.num_free_blocks == num_blocks
    return [s.output_token_ids for s in out]


def _draws(i):
    return dict(temperature=0.9, top_k=(0, 40)[i % 2], top_p=(0.95, 1.0)[i % 2], min_p=0.01 * (i % 3), seed=50 + i)


@pytest.mark.parametrize("graphs", [False, True])
def test_requests_with_a_4_bit_cache_and_drawn_tokens_end_at_their_lengths(graphs):
    model = _model()
    a = _run(model, _draws, graphs=graphs)
    assert a == _run(model, _draws, graphs=graphs)  # the seeds decide
    b = _run(model, lambda i: dict(_draws(i), seed=90 + i), graphs=graphs)
    assert sum(x != y for p, q in zip(a, b) for x, y in zip(p, q)) > 0.5 * sum(n for _, n in _LENS)
    # Under memory pressure requests are evicted and recomputed, and still end.
    _run(model, _draws, graphs=graphs, num_blocks=9)


def test_pipelined_draws_are_the_unpipelined_ones():
    model = _model(seed=3)
    assert _run(model, _draws, pipeline=True) == _run(model, _draws, pipeline=False)


@pytest.mark.parametrize("kv_bits", [4, 16])
@pytest.mark.parametrize("graphs", [False, True])
def test_tokens_are_the_float64_samplers_on_the_steps_logits(graphs, kv_bits):
    model = _model(seed=5, kv_bits=kv_bits)
    runner = _runner(model, cache=Int4PagedKVCache if kv_bits == 4 else PagedKVCache, use_graphs=graphs,
                     max_model_len=256, graph_batch_sizes=(4,))
    seqs = [_seq(i, _tokens(10 + i, i), **s) for i, s in enumerate(
        (dict(temperature=1.0, seed=1), dict(), dict(temperature=0.7, top_k=20, top_p=0.9, min_p=0.02, seed=2),
         dict(temperature=1.3, top_p=0.8)))]
    taken = []
    compute = model.compute_logits

    def keep(*args):
        taken.append(compute(*args))
        return taken[-1]

    model.compute_logits = keep
    for step in range(5):
        plan = [(s, s.pending_tokens) for s in seqs]
        for s, q in plan:
            assert runner.block_manager.allocate(s, s.num_computed_tokens + q)
        u = [s.uniform(len(s.output_token_ids)) for s in seqs]
        results = runner.execute(plan)
        logits = (runner.graphs.last_logits if graphs and step else taken[-1]).float().cpu().numpy()
        p = [s.sampling for s in seqs]
        want = sample_ref(logits, u, [torch.tensor(x.temperature).item() for x in p], [x.top_k for x in p],
                          [torch.tensor(x.top_p).item() for x in p], [torch.tensor(x.min_p).item() for x in p])
        assert [t for _, t in results] == want, f"step {step}"
        for s, t in results:
            s.output_token_ids.append(t)


def test_greedy_requests_keep_their_tokens_beside_drawing_ones():
    model = _model(seed=7, kv_bits=16)
    greedy = _run(model, lambda i: {}, kv_bits=16)
    mixed = _run(model, lambda i: _draws(i) if i % 2 else {}, kv_bits=16)
    # The same greedy requests in a batch of the same shapes: the same logits, the same tokens.
    assert all(greedy[i] == mixed[i] for i in range(0, len(_LENS), 2))


def test_a_4_bit_cache_holds_more_in_less_and_refuses_other_widths():
    args = (32, 16, 2, 2, 64, torch.float16, DEV)
    assert PagedKVCache(*args).num_bytes / Int4PagedKVCache(*args).num_bytes > 3.5
    with pytest.raises(ValueError):
        LLMEngine(_model(), num_blocks=8, device=DEV, kv_bits=8)
    with pytest.raises(ValueError):
        get_attention_backend("auto", kv_bits=2)
    assert get_attention_backend("hip", kv_bits=4)[1] == "hip-int4"
