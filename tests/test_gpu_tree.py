"""Attention for trees of drafted tokens, the step's addresses and the commit of
accepted rows, on the GPU against plain float64 and integer restatements
(oracle/tree.py).

Tolerance of attention.  With u half a step of the dtype, an output is off by u of
itself when it is rounded.  A weight is off by u of itself when it enters the second
product (float16: by 2^-25 besides, below its normal range), and the same weights
are summed, so their part is at most 2 u (1 + u) times the weighted mean of |V|.
Scores are float32 sums of D products, off by at most (D / 8) 2^-24 (blocks of
eight are summed at once) times sum |q k| scale, which is below 64 for these data; a
weight is off by as much of itself.  64 more roundings of 2^-24 of that size cover
the exponentials, the rescaling and the joins."""

from __future__ import annotations

import pytest
import torch

from nanoserve_amd import AttentionMetadata, commit_drafts, get_attention_backend, paged_attention_tree, step_inputs
from oracle.tree import ancestors, commit_ref, signed, step_inputs_ref, tree_attention_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP = [torch.float16, torch.bfloat16]


def random_parents(q, g):
    return ([-1] + [int(torch.randint(max(0, j - 4), j, (1,), generator=g)) for j in range(1, q)])[:q]


class Case:
    """A batch on the CPU, and its metadata on the GPU."""

    def __init__(self, bases, rows, heads, dtype, block_size=16, index=torch.int64, seed=0, spare=3, masks=None,
                 fill=float("nan")):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d = heads
        self.bs, self.rows = block_size, rows
        self.lens = [b + q for b, q in zip(bases, rows)]
        self.starts = [0]
        for q in rows:
            self.starts.append(self.starts[-1] + q)
        T = self.starts[-1]
        need = [-(-n // block_size) for n in self.lens]
        nb = sum(need) + spare
        perm = torch.randperm(nb, generator=g).tolist()
        self.tables, cur = [], 0
        shape = (nb, block_size, self.hkv, self.d)
        # What no sequence holds is NaN: a kernel that reads it into a result shows.
        self.kc, self.vc = torch.full(shape, fill), torch.full(shape, fill)
        for n, L in zip(need, self.lens):
            t = perm[cur:cur + n]
            cur += n
            self.tables.append(t)
            for c in (self.kc, self.vc):
                x = torch.full((n * block_size, self.hkv, self.d), fill)
                x[:L] = torch.randn(L, self.hkv, self.d, generator=g)
                c[t] = x.view(n, block_size, self.hkv, self.d)
        self.kc, self.vc = self.kc.to(dtype), self.vc.to(dtype)
        self.query = torch.randn(T, self.hq, self.d, generator=g).to(dtype)
        self.parents = [random_parents(q, g) for q in rows]
        self.masks = masks if masks is not None else [m for p in self.parents for m in ancestors(p)]
        self.scale = self.d ** -0.5
        self.index = index

    def md(self, host=True, width=0):
        wide = max([len(t) for t in self.tables] + [1, width])
        bt = torch.zeros(len(self.lens), wide, dtype=self.index)
        for i, t in enumerate(self.tables):
            bt[i, :len(t)] = torch.tensor(t, dtype=self.index)
        to = lambda v: torch.tensor(v, dtype=self.index, device=DEV)  # noqa: E731
        return AttentionMetadata(
            slot_mapping=torch.zeros(self.starts[-1], dtype=torch.int64, device=DEV), query_start_loc=to(self.starts),
            seq_lens=to(self.lens), block_tables=bt.to(DEV), max_query_len=max(self.rows),
            max_seq_len=max(self.lens), num_seqs=len(self.lens), num_tokens=self.starts[-1], is_decode_only=False,
            query_start_loc_cpu=self.starts if host else None,
            tree_mask=torch.tensor([signed(m) for m in self.masks], dtype=torch.int64, device=DEV))

    def reference(self):
        return tree_attention_ref(self.query, self.kc, self.vc, self.starts, self.lens, self.tables, self.masks,
                                  self.scale)

    def check(self, out, ref=None):
        ref, mag = ref or self.reference()
        close(out, ref, mag, self.query.dtype, self.d, max(self.lens))

    def run(self, md=None, fn=paged_attention_tree):
        return fn(self.query.to(DEV), self.kc.to(DEV), self.vc.to(DEV), md or self.md(), self.scale)


def close(out, ref, mag, dtype, d, keys):
    u = torch.finfo(dtype).eps / 2
    weights = 2 * u * (1 + u) if dtype is not torch.float32 else 0.0
    tiny = keys * 2.0 ** -25 if dtype is torch.float16 else 0.0
    tol = u * ref.abs() + (weights + (d / 8 + 64) * 64 * 2.0 ** -24) * mag + tiny * mag.amax() + 1e-30
    err = (out.double().cpu() - ref).abs()
    assert torch.isfinite(out).all()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", FP)
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128), (8, 8, 64), (16, 1, 128), (6, 2, 64), (34, 2, 128)])
@pytest.mark.parametrize("block_size,index", [(16, torch.int64), (48, torch.int32)])
def test_ragged_trees(dtype, heads, block_size, index):
    """Prefixes of 0 to a few hundred keys around the tiles' and chunks' borders, trees of 1 to 64 rows."""
    bases = [0, 1, 15, 16, 17, 31, 33, 63, 100, 0, 257]
    rows = [1, 2, 3, 16, 17, 5, 64, 1, 8, 64, 33]
    c = Case(bases, rows, heads, dtype, block_size, index)
    c.check(c.run())


@pytest.mark.parametrize("dtype", FP)
@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)])
def test_long_contexts_in_ranges(dtype, heads):
    """Contexts that are cut into key ranges, beside short ones."""
    c = Case([3000, 20, 1025, 4100, 0], [8, 3, 1, 24, 5], heads, dtype)
    c.check(c.run())


@pytest.mark.parametrize("dtype,heads,block_size", [
    (torch.float32, (14, 2, 64), 16), (torch.float32, (4, 2, 8), 4), (torch.float16, (6, 3, 96), 16),
    (torch.bfloat16, (2, 1, 256), 16), (torch.float16, (14, 2, 64), 8), (torch.bfloat16, (4, 4, 33), 5),
    (torch.float16, (14, 2, 128), 1)])
def test_other_shapes(dtype, heads, block_size):
    c = Case([0, 1, 63, 64, 65, 200], [1, 64, 3, 17, 2, 9], heads, dtype, block_size)
    c.check(c.run())


@pytest.mark.parametrize("dtype,heads", [(torch.float16, (14, 2, 64)), (torch.bfloat16, (28, 4, 128)),
                                         (torch.float32, (4, 2, 40))])
def test_masks_of_all_kinds(dtype, heads):
    """No bits (keys of the prefix alone, or none), every bit, bits past the rows, bits ahead of the row."""
    bases, rows = [0, 0, 40, 40, 0, 17], [4, 64, 4, 64, 1, 1]
    g = torch.Generator().manual_seed(3)
    masks = []
    for b, q in zip(bases, rows):
        for j in range(q):
            kind = j % 4
            masks.append((0, (1 << 64) - 1, 1 << j, int(torch.randint(0, 1 << 62, (1,), generator=g)) << 2)[kind])
    masks[-1] = 0
    c = Case(bases, rows, heads, dtype, masks=masks)
    out = c.run()
    c.check(out)
    assert torch.equal(out[0].cpu(), torch.zeros_like(out[0].cpu()))  # no prefix and no bits


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
@pytest.mark.parametrize("dtype,heads", [(torch.float16, (14, 2, 64)), (torch.bfloat16, (28, 4, 128)),
                                         (torch.float32, (4, 2, 40))])
def test_values_that_a_row_does_not_see(dtype, heads, bad):
    """K and V of row 2 of a tree, in no other row's way to the root: only row 2 may notice."""
    bad = torch.finfo(dtype).min if bad == "lowest" else bad
    parents = [-1, 0, 0, 1, 3, 1]
    masks = ancestors(parents)
    for base in (0, 5, 29, 200):
        c = Case([base, 40], [6, 3], heads, dtype, masks=masks + ancestors([-1, 0, 1]))
        clean = c.reference()
        at = base + 2
        blk, off = c.tables[0][at // 16], at % 16
        for cache in (c.kc, c.vc):
            cache[blk, off, :, 1::3] = bad
        out = c.run().cpu()
        keep = [0, 1, 3, 4, 5, 6, 7, 8]
        ref, mag = (x[keep] for x in clean)
        close(out[keep], ref, mag, dtype, c.d, max(c.lens))
        if bad != bad:
            assert torch.isnan(out[2, :, 1::3].float()).all()


@pytest.mark.parametrize("dtype,heads", [(torch.float16, (14, 2, 64)), (torch.bfloat16, (28, 4, 128))])
def test_values_that_are_seen_and_not_finite(dtype, heads):
    """An infinite V in the tree reaches the rows that see it as the formula says; the others' dims stay."""
    parents = [-1, 0, 1, 0]
    c = Case([50], [4], heads, dtype, masks=ancestors(parents))
    clean = c.reference()
    at = 51
    c.vc[c.tables[0][at // 16], at % 16, :, 4] = float("inf")
    out = c.run().cpu().float()
    assert torch.isinf(out[1, :, 4]).all() and torch.isinf(out[2, :, 4]).all()
    rest = [d for d in range(c.d) if d != 4]
    ref, mag = clean
    close(out[:, :, rest].to(dtype), ref[:, :, rest], mag[:, :, rest], dtype, c.d, 54)
    close(out[[0, 3], :, 4].to(dtype), ref[[0, 3], :, 4], mag[[0, 3], :, 4], dtype, c.d, 54)


@pytest.mark.parametrize("scale", [0.0, -0.125, 3.0])
def test_scales(scale):
    c = Case([100, 0], [7, 20], (14, 2, 64), torch.float16)
    c.query = c.query * 0.3
    c.scale = scale
    c.check(c.run())


def test_blocks_outside_the_cache():
    """Rows of that sequence are NaN, nothing is read, the others stay."""
    for heads in ((14, 2, 64), (6, 3, 96)):
        c = Case([100, 2500, 30], [4, 8, 2], heads, torch.float16)
        ref, mag = c.reference()
        for bad in (-1, c.kc.shape[0], 1 << 40):
            md = c.md()
            md.block_tables[1, 3] = bad
            out = c.run(md).cpu()
            assert torch.isnan(out[4:12]).all()
            keep = [0, 1, 2, 3, 12, 13]
            close(out[keep], ref[keep], mag[keep], torch.float16, c.d, 2508)


def test_rows_of_no_sequence_and_empty_sequences():
    c = Case([10, 20, 30, 0], [3, 0, 5, 0], (14, 2, 64), torch.float16)
    ref = c.reference()
    out = c.run(c.md(host=False))
    c.check(out, ref)
    # four rows behind the last sequence
    md = c.md(host=False)
    md.num_tokens += 4
    md.tree_mask = torch.cat((md.tree_mask, torch.full((4,), -1, dtype=torch.int64, device=DEV)))
    q = torch.cat((c.query, torch.full((4, 14, 64), float("nan"), dtype=torch.float16))).to(DEV)
    got = paged_attention_tree(q, c.kc.to(DEV), c.vc.to(DEV), md, c.scale)
    c.check(got[:8], ref)
    assert (got[8:] == 0).all()


def test_offsets_and_lengths_that_leave_the_batch():
    """Device lengths past max_seq_len are cut there, offsets outside the query are not followed."""
    c = Case([10, 20], [3, 4], (14, 2, 64), torch.float16)
    md = c.md(host=False, width=64)
    md.query_start_loc = torch.tensor([0, 3, 1 << 40], device=DEV)
    out = c.run(md)
    ref, mag = c.reference()
    close(out[:3].cpu(), ref[:3], mag[:3], torch.float16, 64, 24)
    assert (out[3:] == 0).all()
    md = c.md(host=False, width=64)
    md.seq_lens = torch.tensor([13, 1 << 40], device=DEV)  # cut to max_seq_len, which is its length
    c.check(c.run(md))


def test_more_sequences_than_a_launch_schedules():
    n = 1100
    g = torch.Generator().manual_seed(5)
    bases = torch.randint(0, 40, (n,), generator=g).tolist()
    rows = torch.randint(0, 4, (n,), generator=g).tolist()
    c = Case(bases, rows, (4, 2, 64), torch.float16)
    c.check(c.run())


def test_one_row_sequences_without_offsets():
    c = Case([30, 0, 700], [1, 1, 1], (14, 2, 64), torch.bfloat16)
    md = c.md()
    md.query_start_loc = None
    md.is_decode_only = True
    c.check(c.run(md))


def test_strides_and_32_bit_indices():
    c = Case([30, 5], [3, 40], (14, 2, 64), torch.float16, index=torch.int32)
    md = c.md()
    wide = torch.full((2, 64), -7, dtype=torch.int32, device=DEV)
    w = md.block_tables.shape[1]
    wide[:, :w] = md.block_tables
    md.block_tables = wide[:, :w]
    q = torch.stack((c.query, torch.zeros_like(c.query)), 1).to(DEV)[:, 0]
    c.check(paged_attention_tree(q, c.kc.to(DEV), c.vc.to(DEV), md, c.scale))
    lens, starts = md.seq_lens, md.query_start_loc
    md.seq_lens = torch.stack((lens, lens * 0), 1)[:, 0]
    md.query_start_loc = torch.stack((starts, starts * 0), 1)[:, 0]
    c.check(c.run(md))


def test_a_cache_past_32_bit_offsets():
    c = Case([400, 100], [5, 12], (14, 2, 64), torch.float16)
    ref = c.reference()
    row = 2 * 64 * 2 * 16  # bytes of a block
    big = (1 << 32) // row + 2048
    kc, vc = (torch.zeros(big, 16, 2, 64, dtype=torch.float16, device=DEV) for _ in range(2))
    n = c.kc.shape[0]
    kc[-n:], vc[-n:] = c.kc.to(DEV), c.vc.to(DEV)
    md = c.md()
    md.block_tables += big - n
    c.check(paged_attention_tree(c.query.to(DEV), kc, vc, md, c.scale), ref)


def test_the_16_bit_backend_takes_trees_and_the_4_bit_one_refuses():
    c = Case([30, 5], [3, 12], (14, 2, 64), torch.float16)
    fn, _ = get_attention_backend("auto")
    md = c.md()
    fn.prepare(md, c.kc.to(DEV))
    assert md.decode_plan is None
    c.check(c.run(md, fn))
    fn4, _ = get_attention_backend("auto", 4)
    small = torch.zeros(c.kc.shape[0], 2, 16, 36, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="tree_mask"):
        fn4(c.query.to(DEV), small, small, md, c.scale)


def test_equal_calls_give_equal_bits_on_any_stream():
    """Joined ranges are summed in their order, whoever arrives last; calls on two streams share nothing."""
    c = Case([6000, 3000, 9], [8, 24, 2], (14, 2, 64), torch.float16)
    md, q, k, v = c.md(), c.query.to(DEV), c.kc.to(DEV), c.vc.to(DEV)
    first = paged_attention_tree(q, k, v, md, c.scale)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(paged_attention_tree(q, k, v, md, c.scale))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)
    c.check(first)


def test_captured_calls_follow_the_device():
    """A graph of two calls, replayed for other lengths, masks and offsets, with eager calls between."""
    a = Case([3000, 64, 0, 7], [8, 30, 1, 25], (14, 2, 64), torch.float16, seed=1)
    b = Case([90, 2800, 11, 0], [1, 3, 40, 20], (14, 2, 64), torch.float16, seed=2)
    b.starts = [0, 1, 4, 44, 64]
    T = 64
    nb = max(a.kc.shape[0], b.kc.shape[0])
    kc, vc = (torch.zeros(nb, 16, 2, 64, dtype=torch.float16, device=DEV) for _ in range(2))
    q = torch.zeros(T, 14, 64, dtype=torch.float16, device=DEV)
    md = a.md(host=False, width=200)
    md.max_query_len, md.max_seq_len = 64, 3200

    def load(c):
        m = c.md(width=200)
        n = c.kc.shape[0]
        kc[:n], vc[:n], q[:c.starts[-1]] = c.kc.to(DEV), c.vc.to(DEV), c.query.to(DEV)
        md.block_tables.copy_(m.block_tables)
        md.seq_lens.copy_(m.seq_lens)
        md.query_start_loc.copy_(m.query_start_loc)
        md.tree_mask.copy_(m.tree_mask)

    load(a)
    assert a.starts[-1] == b.starts[-1] == T
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged_attention_tree(q, kc, vc, md, a.scale)
    s.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        one = paged_attention_tree(q, kc, vc, md, a.scale)
        two = paged_attention_tree(q * 2, kc, vc, md, a.scale / 2)
    with torch.cuda.graph(other, stream=s):
        three = paged_attention_tree(q, kc, vc, md, a.scale)
    for c in (b, a, b, b, a):
        load(c)
        ref = c.reference()
        graph.replay()
        torch.cuda.synchronize()
        c.check(one, ref)
        c.check(two, ref)
        eager = paged_attention_tree(q, kc, vc, md, c.scale)
        c.check(eager, ref)
        # two graphs at once
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(one, eager) and torch.equal(three, eager)


def test_attention_refusals():
    c = Case([30, 5], [3, 12], (14, 2, 64), torch.float16)
    q, k, v = c.query.to(DEV), c.kc.to(DEV), c.vc.to(DEV)

    def refused(error, match, q=q, k=k, v=v, **over):
        md = c.md()
        for n, x in over.items():
            setattr(md, n, x)
        with pytest.raises(error, match=match):
            paged_attention_tree(q, k, v, md, c.scale)

    refused(ValueError, "tree_mask", tree_mask=None)
    refused(ValueError, "tree_mask", tree_mask=torch.zeros(3, dtype=torch.int64, device=DEV))
    refused(TypeError, "tree_mask", tree_mask=torch.zeros(15, dtype=torch.int32, device=DEV))
    refused(TypeError, "tree_mask", tree_mask=torch.zeros(15, device=DEV))
    refused(ValueError, "expected cuda", tree_mask=torch.zeros(15, dtype=torch.int64))
    refused(ValueError, "64 rows", max_query_len=65)
    refused(ValueError, "tokens", num_tokens=14)
    refused(ValueError, "block_tables", block_tables=torch.zeros(1, 4, dtype=torch.int64, device=DEV))
    refused(ValueError, "columns", max_seq_len=1000)
    refused(ValueError, "query_start_loc", query_start_loc=torch.zeros(2, dtype=torch.int64, device=DEV))
    refused(ValueError, "one row", query_start_loc=None)
    refused(ValueError, "seq_lens", seq_lens=torch.zeros(1, dtype=torch.int64, device=DEV))
    refused(TypeError, "alike", q=q.float())
    refused(ValueError, "head_dim", q=q[:, :, :32])
    refused(ValueError, "query heads", q=q[:, :13].contiguous())
    refused(ValueError, "GPU", q=q.cpu())
    refused(ValueError, "contiguous", k=k.transpose(1, 2).contiguous().transpose(1, 2))
    empty = c.md()
    empty.num_tokens, empty.tree_mask = 0, empty.tree_mask[:0]
    assert paged_attention_tree(q[:0], k, v, empty, c.scale).shape == (0, 14, 64)


# ---- the step's addresses ------------------------------------------------------


def _inputs_case(computed, rows, block_size, width, g, tree, pool=None, pad=0):
    n = len(computed)
    pool = pool or n + 2
    tables = torch.randint(0, 10000, (pool, width), generator=g).tolist()
    place = torch.randperm(pool, generator=g)[:n].tolist()
    held = [-(-c // block_size) for c in computed]
    new = [torch.randint(0, 10000, (max(0, -(-(c + q) // block_size) - h),), generator=g).tolist()
           for c, q, h in zip(computed, rows, held)]
    parents = [p for q in rows for p in random_parents(q, g)] if tree else None
    T = sum(rows) + pad
    if tree:
        parents += [0] * pad
    return tables, place, held, new, parents, T


def _check_inputs(computed, rows, block_size, width, g, tree=True, index=torch.int64, table=torch.int64, pad=0,
                  max_blocks=None, new_blocks=True):
    tables, place, held, new, parents, T = _inputs_case(computed, rows, block_size, width, g, tree, pad=pad)
    if max_blocks is None:
        max_blocks = max([-(-(c + q) // block_size) for c, q in zip(computed, rows)] + [1])
    to = lambda v: torch.tensor(v, dtype=index, device=DEV)  # noqa: E731
    dev = torch.tensor(tables, dtype=table, device=DEV)
    starts = [0]
    for b in new:
        starts.append(starts[-1] + len(b))
    more = dict(new_blocks=to([b for x in new for b in x]), new_start=to(starts), held=to(held)) if new_blocks else {}
    x = step_inputs(dev, to(place), to(computed), to(rows), T, block_size, max_blocks,
                    parents=None if parents is None else to(parents), **more)
    want = step_inputs_ref(tables, place, computed, rows, T, block_size, max_blocks, new if new_blocks else None, held,
                           parents)
    got = (x.query_start_loc, x.seq_lens, x.positions, x.slot_mapping, x.block_tables)
    for a, b in zip(got, want):
        assert a.tolist() == b
    assert dev.tolist() == tables
    assert x.block_tables.dtype is table and x.positions.dtype is torch.int64
    assert (x.tree_mask is None) if parents is None else x.tree_mask.tolist() == want[5]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("index,table", [(torch.int64, torch.int32), (torch.int32, torch.int64)])
@pytest.mark.parametrize("block_size", [1, 7, 16, 32])
def test_step_inputs(tree, index, table, block_size):
    g = torch.Generator().manual_seed(block_size)
    _check_inputs([0], [1], block_size, 64, g, tree, index, table)
    _check_inputs([0, 5, 16, 31, 100, 0, 3], [1, 64, 2, 17, 33, 0, 8], block_size, 200, g, tree, index, table, pad=5)
    n = torch.randint(0, 60, (300,), generator=g).tolist()
    q = torch.randint(0, 9, (300,), generator=g).tolist()
    _check_inputs(n, q, block_size, 90, g, tree, index, table, pad=1)


def test_step_inputs_of_long_prompts_and_wide_tables():
    g = torch.Generator().manual_seed(9)
    _check_inputs([0, 4000, 17], [5000, 1, 3001], 16, 700, g, tree=False)
    _check_inputs([30000] * 9, [3] * 9, 16, 2048, g, table=torch.int32)
    _check_inputs([100, 50], [3, 4], 16, 20, g, new_blocks=False)
    _check_inputs([100, 50], [3, 4], 16, 20, g, max_blocks=0)
    _check_inputs([100, 50], [3, 4], 16, 20, g, max_blocks=40)


def test_step_inputs_at_the_tables_edges():
    """Blocks past the table, requests without a row of it, negative lengths: -1, and no write outside."""
    g = torch.Generator().manual_seed(4)
    tables = torch.randint(0, 99, (3, 4), generator=g).tolist()
    guard = torch.full((5, 4), 77, dtype=torch.int64, device=DEV)
    guard[1:4] = torch.tensor(tables)
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    place, computed, rows = [0, 5, -1, 2, 1], [60, 3, 0, -4, 10], [9, 2, 3, 2, -7]
    new, held = [[11, 12, 13], [14], [15], [16], []], [3, 0, 0, -1, 0]
    x = step_inputs(guard[1:4], to(place), to(computed), to(rows), 20, 16, 6, new_blocks=to([11, 12, 13, 14, 15, 16]),
                    new_start=to([0, 3, 4, 5, 6, 6]), held=to(held))
    want = step_inputs_ref(tables, place, computed, rows, 20, 16, 6, new, held)
    for a, b in zip((x.query_start_loc, x.seq_lens, x.positions, x.slot_mapping, x.block_tables), want):
        assert a.tolist() == b
    assert guard[1:4].tolist() == tables
    assert (guard[0] == 77).all() and (guard[4] == 77).all()


def test_step_inputs_of_odd_parents():
    """A parent that is no earlier row makes a root; rows past the 64th are in no tree."""
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    parents = [5, 1, -9, 2, 1 << 40, 4, 3] + [j - 1 for j in range(70)]
    tables = [[1, 2, 3, 4, 5, 6, 7, 8], [9, 10, 11, 12, 13, 14, 15, 16]]
    want = step_inputs_ref(tables, [0, 1], [3, 4], [7, 70], 77, 16, 6, parents=parents)
    x = step_inputs(to(tables), to([0, 1]), to([3, 4]), to([7, 70]), 77, 16, 6, parents=to(parents))
    assert x.positions.tolist() == want[2] and x.tree_mask.tolist() == want[5] and x.slot_mapping.tolist() == want[3]


def test_step_inputs_of_an_empty_step():
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    x = step_inputs(torch.zeros(2, 4, dtype=torch.int64, device=DEV), to([]), to([]), to([]), 3, 16, 4)
    assert x.query_start_loc.tolist() == [0] and x.slot_mapping.tolist() == [-1] * 3 and x.block_tables.shape == (0, 4)
    x = step_inputs(torch.zeros(0, 4, dtype=torch.int64, device=DEV), to([0]), to([2]), to([1]), 1, 16, 4)
    assert x.slot_mapping.tolist() == [-1] and x.block_tables.tolist() == [[-1, 0, 0, 0]]


# ---- commit --------------------------------------------------------------------


def _commit_case(rows, g, vocab=4, follow=0.7):
    """Few different tokens, so that siblings share some, and choices that follow the tree often."""
    parents = [random_parents(q, g) for q in rows]
    ids, chosen = [], []
    for p in parents:
        i = torch.randint(0, vocab, (len(p),), generator=g).tolist()
        c = torch.randint(0, vocab, (len(p),), generator=g).tolist()
        for j, up in enumerate(p):
            if up >= 0 and torch.rand(1, generator=g).item() < follow:
                c[up] = i[j]
        ids += i
        chosen += c
    return [x for p in parents for x in p], ids, chosen


@pytest.mark.parametrize("heads,dtype,layers", [((2, 64), torch.float16, 3), ((4, 128), torch.bfloat16, 1),
                                                ((1, 33), torch.float16, 2), ((3, 5), torch.float32, 70),
                                                ((1, 3), torch.uint8, 2)])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_commit(heads, dtype, layers, index):
    g = torch.Generator().manual_seed(heads[1] + layers)
    rows = [1, 2, 64, 0, 17, 5, 40, 33]
    parents, ids, chosen = _commit_case(rows, g)
    starts = [0]
    for q in rows:
        starts.append(starts[-1] + q)
    # The widest tree has a path of more rows than a thread holds at once.
    at = 0
    for j in range(1, 64):
        ids[starts[2] + j] = 1000 + j
        parents[starts[2] + j] = at
        if j % 3:
            chosen[starts[2] + at] = 1000 + j
            at = j
    T, nb = starts[-1], 40
    slots = torch.randperm(nb * 16, generator=g)[:T].tolist()
    slots[3], slots[70] = -1, nb * 16 + 5  # rows without a place
    caches = [torch.randint(0, 200, (nb, 16, *heads), generator=g).to(dtype) for _ in range(2 * layers)]
    dev = [c.to(DEV) for c in caches]
    to = lambda v: torch.tensor(v, dtype=index, device=DEV)  # noqa: E731
    counts, tokens = commit_drafts(to(chosen), to(ids), to(parents), to(starts), to(slots), dev[:layers], dev[layers:], 64)
    want = commit_ref(chosen, ids, parents, starts, slots, 64, [c.view(nb * 16, -1) for c in caches], nb * 16)
    assert counts.tolist() == want[0] and tokens.tolist() == want[1]
    assert want[0][2] == 43
    for a, b in zip(dev, caches):
        assert torch.equal(a.cpu(), b)
    # without caches, and with rows cut off
    counts, tokens = commit_drafts(to(chosen), to(ids), to(parents), to(starts), to(slots), [], [], 3)
    want = commit_ref(chosen, ids, parents, starts, slots, 3, [], 0)
    assert counts.tolist() == want[0] and tokens.tolist() == want[1]


def test_commit_along_overlapping_moves():
    """A path whose every row moves onto the place of an earlier row of the path."""
    n = 30
    parents = [-1, 0] + [j - 1 for j in range(2, n)]
    parents[2] = 0
    ids, chosen = list(range(100, 100 + n)), [0] * n
    chosen[0] = ids[2]
    for j in range(2, n - 1):
        chosen[j] = ids[j + 1]
    cache = torch.arange(48 * 8.0).view(3, 16, 1, 8)
    dev = [cache.half().to(DEV)]
    slots = list(range(5, 5 + n))
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    flat = cache.half().view(48, -1)
    counts, tokens = commit_drafts(to(chosen), to(ids), to(parents), to([0, n]), to(slots), dev, [], n)
    want = commit_ref(chosen, ids, parents, [0, n], slots, n, [flat], 48)
    assert counts.tolist() == want[0] == [n - 1] and tokens.tolist() == want[1]
    assert torch.equal(dev[0].view(48, -1).cpu(), flat)


def test_commit_of_odd_trees():
    """Later roots, parents that are no earlier row, equal siblings, negative tokens."""
    parents = [-1, -1, 0, 0, 9, 2, 3, 2]
    ids = [1, 7, 7, 7, 7, -1, 8, 9]
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    for chosen in ([7, 7, -1, 8, 0, 5, 5, 5], [7, 7, 9, 8, 0, 5, 5, 5], [3] * 8, [7, 7, 7, 7, 7, 7, 7, 7]):
        counts, tokens = commit_drafts(to(chosen), to(ids), to(parents), to([0, 8]), to(range(8)), [], [], 8)
        want = commit_ref(chosen, ids, parents, [0, 8], list(range(8)), 8, [], 0)
        assert counts.tolist() == want[0] and tokens.tolist() == want[1]
    # offsets that leave the batch
    counts, tokens = commit_drafts(to([7] * 8), to(ids), to(parents), to([0, 9, 3, -2]), to(range(8)), [], [], 8)
    assert counts.tolist() == [0, 0, 0] and (tokens == -1).all()


def test_refusals_of_step_inputs_and_commit():
    to = lambda v, t=torch.int64: torch.tensor(v, dtype=t, device=DEV)  # noqa: E731
    tables = torch.zeros(4, 8, dtype=torch.int64, device=DEV)
    ok = dict(tables=tables, rows=to([0]), computed=to([3]), query_lens=to([2]), num_tokens=2, block_size=16, max_blocks=2)

    def refused(error, match, **over):
        with pytest.raises(error, match=match):
            step_inputs(**{**ok, **over})

    refused(ValueError, "GPU", tables=tables.cpu())
    refused(ValueError, "tables", tables=tables.float())
    refused(ValueError, "tables", tables=tables[0])
    refused(ValueError, "overlap", tables=tables.t())
    refused(ValueError, "overlap", tables=tables[:1].expand(4, 8))
    refused(ValueError, "computed", computed=to([3, 4]))
    refused(ValueError, "expected", query_lens=to([2]).cpu())
    refused(TypeError, "int32 or int64", rows=to([0.0], torch.float32))
    refused(ValueError, "together", new_blocks=to([1]))
    refused(ValueError, "new_start", new_blocks=to([1]), new_start=to([0]), held=to([0]))
    refused(ValueError, "parents", parents=to([0]))
    refused(ValueError, "sizes", block_size=0)
    refused(ValueError, "sizes", num_tokens=-1)

    cache = torch.zeros(2, 16, 2, 64, dtype=torch.float16, device=DEV)
    ok2 = dict(chosen=to([1, 2]), input_ids=to([1, 2]), parents=to([-1, 0]), query_start_loc=to([0, 2]),
               slot_mapping=to([0, 1]), k_caches=[cache], v_caches=[cache.clone()], max_rows=2)

    def refused2(error, match, **over):
        with pytest.raises(error, match=match):
            commit_drafts(**{**ok2, **over})

    refused2(ValueError, "max_rows", max_rows=65)
    refused2(ValueError, "max_rows", max_rows=-1)
    refused2(ValueError, "input_ids", input_ids=to([1]))
    refused2(ValueError, "parents", parents=to([1]))
    refused2(ValueError, "slot_mapping", slot_mapping=to([1]))
    refused2(TypeError, "int32 or int64", parents=to([0.0, 0.0], torch.float32))
    refused2(ValueError, "query_start_loc", query_start_loc=to(3))
    refused2(ValueError, "GPU", chosen=to([1, 2]).cpu())
    refused2(ValueError, "one shape", v_caches=[cache.float()])
    refused2(ValueError, "one shape", v_caches=[cache[:1]])
    refused2(ValueError, "one shape", v_caches=[cache.cpu()])
    refused2(ValueError, "one shape", k_caches=[cache[:, ::2]], v_caches=[cache[:, ::2]])
    refused2(ValueError, "kv_heads", k_caches=[cache[0]], v_caches=[])
    counts, tokens = commit_drafts(**ok2)
    assert counts.tolist() == [1] and tokens.tolist() == [[1, -1]]


# ---- together --------------------------------------------------------------------


def test_a_step_from_lengths_to_commit():
    """Addresses, cache write, attention and commit of one step, as they are used: the
    cache then holds what a step of the accepted tokens alone would have written."""
    from nanoserve_amd import reshape_and_cache

    g = torch.Generator().manual_seed(11)
    bases, rows, hq, hkv, d, bs = [37, 0, 120], [9, 1, 16], 14, 2, 64, 16
    c = Case(bases, rows, (hq, hkv, d), torch.float16, seed=4, fill=0.0)
    T = sum(rows)
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    tables = torch.zeros(3, 32, dtype=torch.int64, device=DEV)
    held = [-(-b // bs) for b in bases]
    for i, h in enumerate(held):
        tables[i, :h] = to(c.tables[i][:h])
    new = [t[h:] for t, h in zip(c.tables, held)]
    starts = [0]
    for b in new:
        starts.append(starts[-1] + len(b))
    parents = [x for p in c.parents for x in p]
    x = step_inputs(tables, to([0, 1, 2]), to(bases), to(rows), T, bs, 32, to([b for n in new for b in n]), to(starts),
                    to(held), to(parents))
    assert x.tree_mask.tolist() == [signed(m) for m in c.masks]
    kc, vc = c.kc.to(DEV), c.vc.to(DEV)
    key, value = (torch.randn(T, hkv, d, generator=g).half() for _ in range(2))
    reshape_and_cache(key.to(DEV), value.to(DEV), kc, vc, x.slot_mapping)
    md = AttentionMetadata(slot_mapping=x.slot_mapping, query_start_loc=x.query_start_loc, seq_lens=x.seq_lens,
                           block_tables=x.block_tables, max_query_len=16, max_seq_len=max(c.lens), num_seqs=3,
                           num_tokens=T, is_decode_only=False, tree_mask=x.tree_mask)
    out = paged_attention_tree(c.query.to(DEV), kc, vc, md, c.scale)
    slots = x.slot_mapping.tolist()
    for t, s in enumerate(slots):
        c.kc.view(-1, hkv, d)[s], c.vc.view(-1, hkv, d)[s] = key[t], value[t]
    c.check(out)
    _, ids, chosen = _commit_case(rows, g)
    counts, tokens = commit_drafts(to(chosen), to(ids), to(parents), x.query_start_loc, x.slot_mapping, [kc], [vc], 16)
    flat = [c.kc.view(-1, hkv, d), c.vc.view(-1, hkv, d)]
    want = commit_ref(chosen, ids, parents, c.starts, slots, 16, flat, c.kc.shape[0] * bs)
    assert counts.tolist() == want[0] and tokens.tolist() == want[1]
    assert torch.equal(kc.cpu(), c.kc) and torch.equal(vc.cpu(), c.vc)


def test_step_inputs_and_commit_replay_from_a_graph():
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    g = torch.Generator().manual_seed(6)
    B, T, bs, W = 3, 40, 16, 12
    tables = torch.zeros(4, W, dtype=torch.int64, device=DEV)
    rows, computed, lens, held = (torch.zeros(B, dtype=torch.int64, device=DEV) for _ in range(4))
    start = torch.zeros(B + 1, dtype=torch.int64, device=DEV)
    new, parents, ids, chosen = (torch.zeros(T, dtype=torch.int64, device=DEV) for _ in range(4))
    caches = [torch.zeros(16, bs, 1, 8, dtype=torch.float16, device=DEV) for _ in range(4)]
    step = lambda: step_inputs(tables, rows, computed, lens, T, bs, W, new, start, held, parents)  # noqa: E731
    end = lambda x: commit_drafts(chosen, ids, parents, x.query_start_loc, x.slot_mapping, caches[:2], caches[2:], 32)  # noqa: E731
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        end(step())
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        x = step()
        counts, tokens = end(x)
    for it in range(4):
        q = torch.randint(1, 14, (B,), generator=g).tolist()
        c = torch.randint(0, 100, (B,), generator=g).tolist()
        blocks = torch.randperm(16, generator=g).tolist()
        h = [-(-v // bs) for v in c]
        host = torch.zeros(4, W, dtype=torch.int64)
        fresh = [[blocks.pop()] if -(-(a + b) // bs) > k else [] for a, b, k in zip(c, q, h)]
        p, i, ch = _commit_case(q, g)
        pad = T - len(p)
        tables.copy_(host)
        for dst, v in ((rows, [2, 0, 3]), (computed, c), (lens, q), (held, h),
                       (start, [0, len(fresh[0]), len(fresh[0] + fresh[1]), sum(map(len, fresh))]),
                       (new[:sum(map(len, fresh))], [b for f in fresh for b in f]), (parents, p + [-1] * pad),
                       (ids, i + [0] * pad), (chosen, ch + [0] * pad)):
            dst.copy_(to(v))
        for k in caches:
            k.normal_()
        before = [k.cpu() for k in caches]
        graph.replay()
        torch.cuda.synchronize()
        tab = host.tolist()
        want = step_inputs_ref(tab, [2, 0, 3], c, q, T, bs, W, fresh, h, p + [-1] * pad)
        assert [v.tolist() for v in (x.query_start_loc, x.seq_lens, x.positions, x.slot_mapping, x.block_tables)] == list(want[:5])
        assert x.tree_mask.tolist()[:len(p)] == want[5][:len(p)]
        flat = [k.view(16 * bs, -1) for k in before]
        done = commit_ref(ch, i, p, want[0], want[3], 32, flat, 16 * bs)
        assert counts.tolist() == done[0] and tokens.tolist() == done[1]
        for a, b in zip(caches, before):
            assert torch.equal(a.cpu(), b)
