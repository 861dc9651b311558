"""The engine with drafted tokens (MI355X).

Drafts decide how many tokens a step yields, never which: every request's tokens
are those of the same engine without drafts.  The models are float32, so that the
logits of the two (a row among others, a row alone) differ by some 1e-5 of their
spread and a near tie, which either may decide otherwise, is out of the question
for the seeds used; in half precision the tokens are held to the logits instead.
"""

from __future__ import annotations

import pytest
import torch

from nanoserve_amd.attention import AttentionMetadata
from nanoserve_amd.drafting import NgramDrafter
from nanoserve_amd.engine import LLMEngine, SamplingParams, SchedulerConfig
from nanoserve_amd.model import Qwen2Config, Qwen2ForCausalLM, random_init_
from nanoserve_amd.quant import quantize_model

pytestmark = pytest.mark.gpu
DEV = "cuda"
TINY = dict(vocab_size=96, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
            num_attention_heads=2, num_key_value_heads=1, rope_theta=10000.0, tie_word_embeddings=False)


def _model(dtype=torch.float32, seed=0, int4=False, **over):
    cfg = {**TINY, **over}
    m = random_init_(Qwen2ForCausalLM(Qwen2Config(**cfg), max_position=1024), std=0.08, seed=seed).to(dtype).to(DEV)
    if int4:
        quantize_model(m, 128)
    return m.fuse_projections().eval().requires_grad_(False)


class Oracle:
    """Drafts the tokens that a run without drafts gave, with wrong branches before and behind them."""

    def __init__(self, truth, wrong=0.3, seed=0):
        self.truth, self.wrong = truth, wrong
        self.g = torch.Generator().manual_seed(seed)
        self.asked = []

    def draft(self, seq, limit, depth):
        self.asked.append((limit, depth))
        rest = self.truth[seq.seq_id][len(seq.output_token_ids):][:depth]
        tokens, parents, row = [], [], 0
        for t in rest:
            if len(tokens) + 2 > limit:
                break
            tokens += [(t + 1) % 96, t]  # a sibling that is wrong, then the right one
            parents += [row, row]
            row = len(tokens)
            if torch.rand(1, generator=self.g).item() < self.wrong:
                tokens[-1] = (t + 5) % 96
                break
        return tokens, parents


def _prompts():
    g = torch.Generator().manual_seed(5)
    out = []
    for n in (3, 17, 40, 9, 64, 25):
        phrase = torch.randint(0, 96, (max(2, n // 3),), generator=g).tolist()
        out.append((phrase * 4)[:n])
    return out


def _run(model, sampling, draft_tokens=0, drafter=None, num_blocks=96, block_size=8, eos=None, config=None, **kw):
    e = LLMEngine(model, num_blocks, block_size, DEV, scheduler_config=config, eos_token_id=eos, max_model_len=512,
                  draft_tokens=draft_tokens, drafter=drafter, **kw)
    for i, p in enumerate(_prompts()):
        e.add_request(p, sampling(i))
    steps = 0
    done = {}
    while e.has_unfinished_requests:
        for s in e.step():
            done[s.seq_id] = s.output_token_ids
        steps += 1
    assert e.block_manager.num_free_blocks == num_blocks
    return done, steps, e


def _greedy(i):
    return SamplingParams(max_new_tokens=20 + 7 * i, ignore_eos=True)


@pytest.mark.parametrize("draft_tokens", [1, 5, 63])
def test_greedy_tokens_do_not_depend_on_drafts(draft_tokens):
    model = _model()
    plain, steps, _ = _run(model, _greedy)
    drafted, fewer, e = _run(model, _greedy, draft_tokens)
    assert drafted == plain
    assert e.num_drafted > 0 and 0 < e.num_accepted <= e.num_drafted
    assert fewer < steps
    assert all(len(t) == 20 + 7 * i for i, t in plain.items())


@pytest.mark.parametrize("block_size,over", [(16, dict(head=64)), (4, dict(head=64)), (16, dict(head=32))])
def test_wrong_and_right_branches(block_size, over):
    """Trees whose right chain lies behind wrong siblings: rows move in the cache in every step."""
    heads = 128 // over["head"]
    model = _model(num_attention_heads=heads, num_key_value_heads=1)
    plain, steps, _ = _run(model, _greedy, block_size=block_size)
    drafter = Oracle(plain)
    drafted, fewer, e = _run(model, _greedy, 12, drafter, block_size=block_size)
    assert drafted == plain and fewer < steps
    assert e.num_accepted > 0.2 * e.num_drafted
    assert all(limit <= 12 for limit, _ in drafter.asked)


def test_drawn_tokens_do_not_depend_on_drafts():
    model = _model(seed=3)
    sampling = lambda i: SamplingParams(max_new_tokens=30, ignore_eos=True, temperature=0.0 if i == 2 else 0.7,  # noqa: E731
                                        top_k=8, seed=11 * i)
    plain, steps, _ = _run(model, sampling)
    drafted, fewer, _ = _run(model, sampling, 10, Oracle(plain))
    assert drafted == plain and fewer < steps


def test_a_request_ends_inside_a_draft():
    """At its end-of-sequence token, with what was accepted behind it dropped, and at its length."""
    model = _model()
    plain, _, _ = _run(model, _greedy)
    eos = plain[4][9]
    stop = lambda i: SamplingParams(max_new_tokens=40)  # noqa: E731
    want, _, _ = _run(model, stop, eos=eos)
    got, _, _ = _run(model, stop, 8, Oracle(plain, wrong=0.0), eos=eos)
    assert got == want
    assert any(t[-1] == eos and len(t) < 40 for t in got.values())


def test_drafts_with_evictions_chunked_prompts_and_graphs():
    """A cache and a budget so small that requests are evicted and rows are cut from drafts."""
    model = _model()
    config = lambda: SchedulerConfig(max_num_batched_tokens=24, max_num_seqs=4)  # noqa: E731
    plain, _, _ = _run(model, _greedy, num_blocks=24, config=config())
    drafted, _, e = _run(model, _greedy, 9, Oracle(plain), num_blocks=24, config=config())
    assert drafted == plain and e.num_accepted > 0
    graphs, _, e = _run(model, _greedy, 9, NgramDrafter(branches=1), num_blocks=24, config=config(), use_graphs=True)
    assert graphs == plain and e.num_accepted > 0


def test_half_precision_tokens_follow_from_their_logits():
    """INT4 model in float16 on the matrix-core kernels: every token is the largest logit of its
    prefix, computed in one prompt step, or within the rounding of it."""
    model = _model(torch.float16, int4=True, hidden_size=256, intermediate_size=512, num_attention_heads=4,
                   num_key_value_heads=2)
    out, _, e = _run(model, _greedy, 15, NgramDrafter(branches=3), block_size=16)
    assert e.num_accepted > 0
    for i, prompt in enumerate(_prompts()):
        text = prompt + out[i]
        one = LLMEngine(model, 64, 16, DEV, max_model_len=512)
        n = len(text)
        blocks = torch.arange(-(-n // 16), device=DEV)
        pos = torch.arange(n, device=DEV)
        md = AttentionMetadata(slot_mapping=pos, query_start_loc=torch.tensor([0, n], device=DEV),
                               seq_lens=torch.tensor([n], device=DEV), block_tables=blocks[None], max_query_len=n,
                               max_seq_len=n, num_seqs=1, num_tokens=n, is_decode_only=False)
        with torch.inference_mode():
            hidden = model(torch.tensor(text, device=DEV), pos, one.kv_cache, md, one.runner.attn_fn)
            logits = model.compute_logits(hidden).float()
        for j, t in enumerate(out[i]):
            row = logits[len(prompt) + j - 1]
            assert row[t] >= row.max() - 1e-2 * row.abs().max(), (i, j)


def test_refusals():
    model = _model()
    for kw, match in ((dict(draft_tokens=64), "draft_tokens"), (dict(draft_tokens=-1), "draft_tokens"),
                      (dict(draft_tokens=4, kv_bits=4), "16-bit")):
        with pytest.raises(ValueError, match=match):
            LLMEngine(model, 16, 8, DEV, **kw)

    class Bad:
        def draft(self, seq, limit, depth):
            return [96], [0]

    e = LLMEngine(model, 32, 8, DEV, max_model_len=128, draft_tokens=4, drafter=Bad())
    e.add_request([1, 2, 3], SamplingParams(max_new_tokens=8))
    with pytest.raises(ValueError, match="vocabulary"):
        e.run_all()
