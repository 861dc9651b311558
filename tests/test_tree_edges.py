"""A drafted step at its edges, as far as the host decides them (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import nanoserve_amd
from nanoserve_amd import _lib, tree
from nanoserve_amd.engine import LLMEngine
from nanoserve_amd.model import Qwen2Config, Qwen2ForCausalLM
from nanoserve_amd.scheduling import SamplingParams


class Devices:
    """torch's current device and a library on two devices of different sizes, stood in for on the CPU."""

    current = 0

    def __init__(self, index):
        self.index = getattr(index, "index", index)

    def __enter__(self):
        self.before, Devices.current = Devices.current, self.index

    def __exit__(self, *_):
        Devices.current = self.before

    @staticmethod
    def ns_paged_attention_tree_counters():
        return (64, 256)[Devices.current]


@pytest.fixture
def devices(monkeypatch):
    monkeypatch.setattr(torch.cuda, "device", Devices)
    monkeypatch.setattr(tree._lib, "load", lambda: Devices)
    monkeypatch.setattr(tree, "_counters", {})
    monkeypatch.setattr(torch, "zeros", lambda n, **_: n)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)


@pytest.mark.parametrize("capturing", [False, True])
def test_counters_are_those_of_the_tensors_device(devices, capturing):
    """One a workgroup of the device that the call runs on, whichever is current."""
    assert tree._arrivals(torch.device("cuda:1"), capturing) == 256
    assert tree._arrivals(torch.device("cuda:0"), capturing) == 64
    with Devices(1):
        assert tree._arrivals(torch.device("cuda:0"), capturing) == 64


def test_a_capture_is_looked_for_on_the_tensors_device(devices, monkeypatch):
    """Device 1 records a graph while device 0 is current, and the other way round."""
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: Devices.current, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: Devices.current == 1, raising=False)
    assert tree._capturing(1) and not tree._capturing(0)
    with Devices(1):
        assert tree._capturing(1) and not tree._capturing(0)


# ---- the C entry points' limits: refused before any launch ------------------------

BIG = 1 << 40  # aligned, never read
UNSUPPORTED = _lib.NS_ERR_UNSUPPORTED


def _commit(caches=(BIG, 2 * BIG), **over):
    array = (ctypes.c_void_p * max(len(caches), 1))(*caches)
    a = dict(counts=BIG, tokens=BIG, chosen=BIG, ids=BIG, parents=BIG, i64=1, qsl=BIG, qsl64=1, slots=BIG, slots64=1, S=2, T=16,
             maxr=8, array=ctypes.addressof(array), n=len(caches), num_slots=512, row_bytes=256, stream=None)
    a.update(over)
    return _lib.load().ns_commit_drafts(*a.values())


@pytest.mark.parametrize("over", [dict(S=1 << 24), dict(S=1 << 31), dict(row_bytes=(1 << 20) + 1), dict(maxr=65)])
def test_commit_refuses_what_no_grid_holds(over):
    assert _commit(**over) == UNSUPPORTED


@pytest.mark.parametrize("over", [
    dict(counts=None), dict(tokens=None), dict(chosen=None), dict(ids=None), dict(parents=None), dict(qsl=None),
    dict(slots=None), dict(S=-1), dict(T=-1), dict(maxr=-1), dict(array=None), dict(n=-1), dict(num_slots=-1),
    dict(row_bytes=-1), dict(row_bytes=0), dict(caches=(BIG, 0)), dict(counts=BIG + 4), dict(chosen=BIG + 4),
    dict(qsl=BIG + 4), dict(slots=BIG + 4), dict(chosen=BIG + 2, i64=0),
])
def test_commit_refuses_with_caches_beside_one_another(over):
    assert _commit(**over) == _lib.NS_ERR_INVALID_ARG


def test_commit_refuses_caches_that_overlap():
    """A row in two caches would be moved twice: the second move may read what the first has written."""
    size = 512 * 256
    for caches in ((BIG, BIG), (BIG, BIG + size - 16), (BIG + 256, 2 * BIG, BIG), (3 * BIG, 2 * BIG, 3 * BIG - size + 1)):
        assert _commit(caches=caches) == _lib.NS_ERR_INVALID_ARG


@pytest.mark.parametrize("dtype,D,bs", [(_lib.NS_DTYPE_F32, 64, 16), (_lib.NS_DTYPE_F16, 8, 16), (_lib.NS_DTYPE_F16, 64, 4)])
def test_attention_refuses_what_no_grid_holds(dtype, D, bs):
    T = 1 << 26
    assert _lib.load().ns_paged_attention_tree(
        BIG, BIG, BIG, BIG, BIG, 64, 64, 1, BIG, 1, BIG, 1, BIG, 2, T, 8, 64, 1, 1, D, bs, 128, 0.125, dtype, None, None, 0,
        None) == UNSUPPORTED


# ---- the engine, its model stood in for --------------------------------------------


class Drafter:
    """Three drafted tokens in a chain, or what room there is for them."""

    def draft(self, seq, limit, depth):
        n = min(3, limit, depth)
        return [7, 8, 9][:n], list(range(n))


def _engine(kept, **kw):
    """An engine past its request's prompt, whose drafted steps give the lists of `kept` in turn."""
    model = Qwen2ForCausalLM(Qwen2Config(vocab_size=16, hidden_size=16, intermediate_size=16, num_hidden_layers=1,
                                         num_attention_heads=2, num_key_value_heads=1, tie_word_embeddings=False))
    e = LLMEngine(model, 16, 4, "cpu", max_model_len=64, draft_tokens=3, drafter=Drafter(), **kw)

    def prompt(scheduled):
        for seq, q in scheduled:
            seq.mark_computed(q)
        return [(seq, 1) for seq, _ in scheduled]

    e.runner.execute = prompt
    e.add_request([1, 2, 3, 4, 5], SamplingParams(max_new_tokens=12))
    e.step()
    if kept is not None:
        kept = iter(kept)
        e.runner.execute_drafted = lambda seqs, drafts: [next(kept) for _ in seqs]
    return e


@pytest.mark.parametrize("kept,text,accepted", [
    ([[5]], [5], 0), ([[7, 5]], [7, 5], 1), ([[7, 8, 9, 5]], [7, 8, 9, 5], 3),
    # the end of the text: at the model's own token, at a drafted one, with more of them behind
    ([[7, 0]], [7, 0], 1), ([[7, 8, 9, 0]], [7, 8, 9, 0], 3), ([[0]], [0], 0), ([[0, 8]], [0], 1),
    ([[7, 0, 9, 5]], [7, 0], 2), ([[0, 8, 9, 5]], [0], 1), ([[7, 5], [7, 0, 9]], [7, 5, 7, 0], 3),
])
def test_accepted_tokens_are_those_that_the_text_keeps(kept, text, accepted):
    e = _engine(kept, eos_token_id=0)
    seq = e.scheduler.running[0]
    for _ in kept:
        e.step()
    assert seq.output_token_ids == [1, *text]
    assert (e.num_drafted, e.num_accepted) == (3 * len(kept), accepted)


@pytest.mark.parametrize("what", ["_stage", "step_inputs"])
def test_a_step_that_never_reached_the_device_leaves_no_blocks_named(what, monkeypatch):
    """The device's tables lack the blocks of a step that failed before its launch: the next one names them again."""
    e = _engine(None)
    seq = e.scheduler.running[0]

    def fails(*a, **kw):
        raise RuntimeError("out of memory")

    with monkeypatch.context() as m:
        if what == "_stage":
            m.setattr(e.runner, what, fails)
        else:
            m.setattr("nanoserve_amd.engine.step_inputs", fails)
        for _ in range(2):
            with pytest.raises(RuntimeError, match="memory"):
                e.step()
    rows, held, start, blocks = e.runner._tables.place([seq])
    assert held == [0] and blocks == seq.block_table and start == [0, len(blocks)]


# ---- what a user imports ------------------------------------------------------------


def test_what_goes_with_a_drafted_step_is_exported():
    for name in ("AttentionMetadata", "BlockTables", "NgramDrafter", "commit_drafts", "paged_attention_tree", "step_inputs"):
        assert name in nanoserve_amd.__all__ and hasattr(nanoserve_amd, name)
