"""Drafts, the tables that a drafting engine keeps, and the oracle of a step over
drafted trees (no GPU)."""

from __future__ import annotations

import pytest
import torch

from nanoserve_amd import commit_drafts, paged_attention_tree, step_inputs
from nanoserve_amd.block_manager import BlockSpaceManager
from nanoserve_amd.drafting import NgramDrafter, check_draft
from nanoserve_amd.scheduling import SamplingParams, Sequence
from nanoserve_amd.tree import BlockTables
from oracle.paged_attention import paged_attention_ref
from oracle.tree import ancestors, commit_ref, signed, step_inputs_ref, tree_attention_ref
from tests._helpers import build_paged, make_md


def _seq(i, tokens, out=()):
    s = Sequence(i, list(tokens), SamplingParams())
    s.output_token_ids = list(out)
    return s


# ---- drafts ------------------------------------------------------------------


def test_the_longest_match_comes_first_and_shorter_ones_branch():
    d = NgramDrafter(max_ngram=2, branches=2)
    #          0  1  2  3  4  5  6  7
    s = _seq(0, [5, 6, 7, 9, 6, 8, 5, 6])
    # (5, 6) stood before 7 9 6 8; (6,) alone also before 8 5 6.
    assert d.draft(s, 8, 3) == ([7, 9, 6, 8, 5, 6], [0, 1, 2, 0, 4, 5])
    assert d.draft(s, 4, 3) == ([7, 9, 6, 8], [0, 1, 2, 0])
    assert d.draft(s, 8, 1) == ([7, 8], [0, 0])
    assert d.draft(s, 0, 3) == ([], []) == d.draft(s, 3, 0)


def test_chains_that_begin_alike_share_rows():
    d = NgramDrafter(max_ngram=1, branches=3)
    s = _seq(0, [1, 2, 3, 1, 2, 4, 1, 2, 3, 5, 1])
    tokens, parents = d.draft(s, 20, 3)
    # latest first: 2 3 5, then 2 4 1, then 2 3 1
    assert (tokens, parents) == ([2, 3, 5, 4, 1, 1], [0, 1, 2, 1, 4, 2])


def test_the_index_follows_the_output_and_forgets():
    d = NgramDrafter()
    s = _seq(3, [1, 2, 3])
    assert d.draft(s, 4, 4) == ([], [])
    s.output_token_ids += [1, 2]
    assert d.draft(s, 4, 4) == ([3, 1, 2], [0, 1, 2])
    d.forget(s)
    d.forget(s)
    assert d.draft(s, 4, 4) == ([3, 1, 2], [0, 1, 2])
    for bad in (dict(max_ngram=0), dict(branches=0)):
        with pytest.raises(ValueError):
            NgramDrafter(**bad)


def test_what_a_drafter_may_return():
    check_draft([], [], 0, 0, 10)
    check_draft([1, 2, 3], [0, 1, 0], 3, 2, 10)
    for args in (([1], [], 3, 3, 10), ([1, 2], [0, 0], 1, 3, 10), ([10], [0], 3, 3, 10), ([-1], [0], 3, 3, 10),
                 ([1], [1], 3, 3, 10), ([1], [-1], 3, 3, 10), ([1, 2], [0, 1], 3, 1, 10), ([1], [0], 0, 3, 10)):
        with pytest.raises(ValueError):
            check_draft(*args)


# ---- tables ------------------------------------------------------------------


def test_tables_name_only_what_is_new():
    bm = BlockSpaceManager(4, 64, watermark=0.0)
    t = BlockTables(16, "cpu", rows=2)
    a, b, c = (_seq(i, [0]) for i in range(3))
    assert bm.allocate(a, 9) and bm.allocate(b, 4)
    rows, held, start, new = t.place([a, b])
    assert sorted(rows) == [0, 1] and held == [0, 0] and start == [0, 3, 4] and new == [*a.block_table, *b.block_table]
    assert bm.allocate(a, 13)
    assert t.place([a, b]) == (rows, [3, 1], [0, 1, 1], a.block_table[3:])
    # a shorter table of the same blocks keeps its entries, and what comes next is new
    bm.trim(a, 5)
    t.trimmed(a)
    assert bm.allocate(c, 4) and bm.allocate(a, 9)
    _, held, start, new = t.place([a])
    assert held == [2] and new == a.block_table[2:]
    # a table that was freed and filled again is another
    bm.free(a)
    assert bm.allocate(a, 9)
    assert t.place([a])[1] == [0]
    # a request without a row takes that of one outside the batch, or the tables grow
    rows, held, _, _ = t.place([a, c])
    assert held == [3, 0] and len(set(rows)) == 2
    rows, held, _, _ = t.place([a, b, c])
    assert held == [3, 0, 1] and len(set(rows)) == 3 and t.tensor.shape[0] >= 3
    t.forget(b)
    t.forget(b)
    assert t.place([b])[1] == [0]


def test_trim_returns_the_blocks_behind_and_no_others():
    bm = BlockSpaceManager(4, 8, watermark=0.0)
    a, b = _seq(0, [0]), _seq(1, [0])
    assert bm.allocate(a, 20) and bm.allocate(b, 4)
    table = a.block_table
    bm.trim(a, 20)
    assert a.block_table is table and bm.num_free_blocks == 2
    bm.trim(a, 9)
    assert a.block_table == table[:3] and a.block_table is not table and bm.num_free_blocks == 4
    assert bm.allocate(a, 13) and a.block_table[3] == table[3]  # the first of them is the next one out
    bm.trim(a, 0)
    assert a.block_table == [] and bm.num_free_blocks == 7
    bm.free(a)
    bm.free(b)
    assert bm.num_free_blocks == 8


# ---- the oracle ----------------------------------------------------------------


def test_ancestors_and_their_bits():
    assert ancestors([-1, 0, 0, 2, 1]) == [0b1, 0b11, 0b101, 0b1101, 0b10011]
    assert ancestors([3, 1, -5]) == [1, 2, 4]  # no earlier row: a root
    chain = ancestors([j - 1 for j in range(66)])
    assert chain[63] == (1 << 64) - 1 and chain[64:] == [0, 0]
    assert signed(chain[63]) == -1 and signed(1 << 63) == -(1 << 63) and signed(5) == 5


def test_a_chain_is_causal_attention():
    seqs, rows, heads, d, bs = [37, 16, 5], [7, 1, 5], (4, 2), 16, 8
    kc, vc, tables, _ = build_paged(seqs, 16, bs, heads[1], d)
    md = make_md(seqs, rows, tables, bs)
    q = torch.randn(sum(rows), heads[0], d, generator=torch.Generator().manual_seed(1))
    masks = [m for n in rows for m in ancestors([j - 1 for j in range(n)])]
    out, mag = tree_attention_ref(q, kc, vc, md.query_start_loc_cpu, seqs, tables, masks, 0.3)
    assert torch.allclose(out.float(), paged_attention_ref(q, kc, vc, md, 0.3), atol=2e-6)
    assert (mag >= out.abs() - 1e-12).all()


def test_a_tree_is_attention_over_each_path():
    """Every row equals causal attention of the sequence that holds its path alone."""
    base, parents, d, bs = 11, [-1, 0, 0, 2, 1, 3], 8, 4
    n = base + len(parents)
    kc, vc, tables, ((k, v),) = build_paged([n], 8, bs, 1, d)
    q = torch.randn(len(parents), 2, d, generator=torch.Generator().manual_seed(2))
    masks = ancestors(parents)
    out, _ = tree_attention_ref(q, kc, vc, [0, len(parents)], [n], tables, masks, 0.4)
    for j, m in enumerate(masks):
        keys = [*range(base), *[base + i for i in range(6) if m >> i & 1]]
        kk, vv = k[keys].double(), v[keys].double()
        for h in range(2):
            w = torch.tensor([float(q[j, h].double() @ x[0]) * 0.4 for x in kk], dtype=torch.float64).softmax(0)
            assert torch.allclose(out[j, h], w @ vv[:, 0], atol=1e-12)
    empty, _ = tree_attention_ref(q[:1], kc, vc, [0, 1], [1], tables, [0], 0.4)
    assert (empty == 0).all()


def test_addresses_by_hand():
    tables = [[9, 9, 9], [4, 7, 0]]
    got = step_inputs_ref(tables, [1], [5], [4], 6, 4, 3, new=[[8]], held=[2], parents=[-1, 0, 0, 2, 0, 0])
    assert tables[1] == [4, 7, 8]
    assert got == ([0, 4], [9], [5, 6, 6, 7, 0, 0], [29, 30, 31, 32, -1, -1], [[4, 7, 8]],
                   [0b1, 0b11, 0b101, 0b1101, 0, 0])


def test_a_walk_by_hand():
    cache = torch.arange(8.0).view(8, 1)
    #        row 0 chose 7: rows 1 (6) no, 2 (7) yes; row 2 chose 3: row 4; row 4 chose 1: nobody
    counts, tokens = commit_ref([7, 9, 3, 0, 1], [5, 6, 7, 3, 3], [-1, 0, 0, 1, 2], [0, 5], [3, 4, 5, 6, 7], 5, [cache], 8)
    assert counts == [3] and tokens == [[7, 3, 1, -1, -1]]
    assert cache.flatten().tolist() == [0, 1, 2, 3, 5, 7, 6, 7]


# ---- refusals without a GPU -------------------------------------------------------


def test_cpu_tensors_are_refused():
    i = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        step_inputs(torch.zeros(2, 4, dtype=torch.int64), i, i, i, 1, 16, 4)
    with pytest.raises(ValueError, match="GPU"):
        commit_drafts(i, i, i, torch.zeros(2, dtype=torch.int64), i, [], [], 1)
    kc, vc, tables, _ = build_paged([4], 2, 4, 1, 8)
    md = make_md([4], [1], tables, 4)
    md.tree_mask = torch.ones(1, dtype=torch.int64)
    with pytest.raises(ValueError, match="GPU"):
        paged_attention_tree(torch.zeros(1, 1, 8), kc, vc, md, 1.0)
