"""Attention for drafted trees at every width of its column blocks, for both head
sizes, with batches that fill the device and batches that do not, against plain
float64 (oracle/tree.py).  The tolerance is that of test_gpu_tree.py, derived there."""

from __future__ import annotations

import pytest
import torch

from nanoserve_amd import paged_attention_tree, step_inputs
from oracle.tree import ancestors, signed, step_inputs_ref, tree_attention_ref

from tests.test_gpu_tree import DEV, Case, close

pytestmark = pytest.mark.gpu
FP = [torch.float16, torch.bfloat16]
# Eight query heads a KV head: rows / 2 column tiles of 16.  Blocks take up to 16 tiles at
# head size 64 and 8 at 128: all widths, and a second block that is not full.
WIDTHS = [(64, r) for r in (2, 4, 7, 15, 31, 45)] + [(128, r) for r in (2, 4, 7, 15, 21, 40)]


def batch(n, rows, g):
    """n sequences around the chunks' borders; one has `rows` rows and a context that is cut
    into ranges, where there are few workgroups' worth of others."""
    edges = [0, 1, 15, 16, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 129, 160]
    bases = [edges[i % len(edges)] for i in range(n)]
    q = [rows] + torch.randint(1, rows + 1, (n - 1,), generator=g).tolist()
    bases[0] = 1500
    return bases, q


@pytest.mark.parametrize("dtype", FP)
@pytest.mark.parametrize("D,rows", WIDTHS)
def test_full_batches(dtype, D, rows):
    g = torch.Generator().manual_seed(rows)
    bases, q = batch(33, rows, g)
    c = Case(bases, q, (16, 2, D), dtype, seed=rows)
    c.check(c.run())


@pytest.mark.parametrize("dtype", FP)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,rows,heads", [(1, 1, (2, 2)), (1, 3, (14, 2)), (1, 64, (8, 1)), (2, 33, (12, 1)),
                                          (5, 17, (28, 4)), (3, 64, (40, 2))])
def test_small_batches(dtype, D, n, rows, heads):
    """Narrow blocks of columns and ranges: few sequences, one of 4000 keys."""
    g = torch.Generator().manual_seed(n)
    bases, q = batch(n, rows, g)
    bases[0] = 4000
    c = Case(bases, q, (*heads, D), dtype, seed=n)
    c.check(c.run())


@pytest.mark.parametrize("D,rows", WIDTHS)
def test_prefixes_that_end_everywhere_in_a_step(D, rows):
    """Contexts one key apart over two steps of all key groups: groups that have no chunk in the last one."""
    q = rows
    bases = list(range(0, 33 * 16, 16)) + [511 + i for i in range(4)]
    c = Case(bases, [q] + [1] * (len(bases) - 1), (16, 2, D), torch.float16, seed=5)
    c.check(c.run())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("D,rows", WIDTHS)
def test_rows_that_do_not_see_a_bad_key(D, rows, bad):
    """K and V of one drafted row, a leaf, hold NaN or infinities: every other row is as without."""
    g = torch.Generator().manual_seed(1)
    bases, q = batch(33, rows, g)
    c = Case(bases, q, (16, 2, D), torch.bfloat16, seed=2)
    clean, mag = c.reference()
    leaves = []
    for i, n in enumerate(q):
        children = set(c.parents[i])
        leaf = max((j for j in range(1, n) if j not in children), default=None)
        if leaf is None or i % 3 == 2:
            continue
        leaves.append(c.starts[i] + leaf)
        at = bases[i] + leaf
        for cache in (c.kc, c.vc):
            cache[c.tables[i][at // 16], at % 16, :, ::5] = bad
    keep = [t for t in range(c.starts[-1]) if t not in set(leaves)]
    out = c.run().cpu()
    close(out[keep], clean[keep], mag[keep], torch.bfloat16, D, max(c.lens))


@pytest.mark.parametrize("D,rows", WIDTHS)
def test_an_infinite_value_reaches_the_rows_that_see_it(D, rows):
    """V of row 0 holds an infinity in one dim: every row of the request sees it, and no other dim or request."""
    g = torch.Generator().manual_seed(3)
    bases, q = batch(33, rows, g)
    c = Case(bases, q, (16, 2, D), torch.float16, seed=3)
    clean, mag = c.reference()
    for i in range(0, 33, 2):
        at = bases[i]
        c.vc[c.tables[i][at // 16], at % 16, :, 3] = float("inf")
    out = c.run().cpu()
    hit = [t for i in range(0, 33, 2) for t in range(c.starts[i], c.starts[i + 1])]
    assert torch.isinf(out[hit][:, :, 3].float()).all()
    rest = [d for d in range(D) if d != 3]
    close(out[:, :, rest], clean[:, :, rest], mag[:, :, rest], torch.float16, D, max(c.lens))
    other = [t for t in range(c.starts[-1]) if t not in set(hit)]
    close(out[other], clean[other], mag[other], torch.float16, D, max(c.lens))


@pytest.mark.parametrize("D,rows", WIDTHS)
def test_large_scores_move_the_reference(D, rows):
    """Scores that rise along the context by far more than a float's range of weights: the last keys take all."""
    g = torch.Generator().manual_seed(4)
    bases, q = batch(33, rows, g)
    c = Case(bases, q, (16, 2, D), torch.float16, seed=6)
    # q . k grows with the key's place: one dim of q is 8, of k its place's height up to 8.
    c.query[:, :, 0] = 8.0
    for i, L in enumerate(c.lens):
        for p in range(L):
            c.kc[c.tables[i][p // 16], p % 16, :, 0] = 8.0 * p / L
    c.scale = 1.0 if D == 64 else 0.5
    ref, mag = c.reference()
    out = c.run().cpu()
    # Scores reach 64 + 8 |noise| at scale 1: below 160 in size, 2.5 times what close() counts on.
    u = 2.0 ** -11
    tol = u * ref.abs() + (2 * u * (1 + u) + (D / 8 + 64) * 160 * 2.0 ** -24) * mag + max(c.lens) * 2.0 ** -25 * mag.amax()
    assert torch.isfinite(out).all()
    assert ((out.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("heads", [(14, 2, 64), (28, 4, 128)])
def test_rows_past_the_64th_stay(heads):
    """The device's offsets give a sequence 80 rows: its first 64 are computed, the others left as they are (zero)."""
    c = Case([20, 3], [80, 9], heads, torch.float16, seed=8)
    md = c.md(host=False)
    md.max_query_len = 64
    ref, mag = c.reference()
    out = c.run(md).cpu()
    keep = [*range(64), *range(80, 89)]
    close(out[keep], ref[keep], mag[keep], torch.float16, heads[2], max(c.lens))
    assert torch.equal(out[64:80], torch.zeros_like(out[64:80]))


def test_one_device_batch_of_each_kind_in_one_graph():
    """Both head sizes captured together, replayed with other masks."""
    cases = [Case([900, 40, 3], [9, 2, 30], (14, 2, 64), torch.float16, seed=1),
             Case([700, 80], [20, 5], (28, 4, 128), torch.bfloat16, seed=2)]
    mds = [c.md(host=False) for c in cases]
    args = [[x.to(DEV) for x in (c.query, c.kc, c.vc)] for c in cases]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for c, a, m in zip(cases, args, mds):
            paged_attention_tree(*a, m, c.scale)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        outs = [paged_attention_tree(*a, m, c.scale) for c, a, m in zip(cases, args, mds)]
    for it in range(3):
        for c, m in zip(cases, mds):
            if it:
                c.masks = [x for q in c.rows for x in ancestors([-1] + [max(0, j - it) for j in range(1, q)])]
                m.tree_mask.copy_(torch.tensor([signed(x) for x in c.masks]))
        graph.replay()
        torch.cuda.synchronize()
        for c, o in zip(cases, outs):
            c.check(o, tree_attention_ref(c.query, c.kc, c.vc, c.starts, c.lens, c.tables, c.masks, c.scale))


def test_columns_and_rows_at_the_ends_of_64_bits():
    """New blocks named for columns and table rows that no table has are not written anywhere."""
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    far = 2 ** 63 - 1
    tables = to([[10, 11, 12, 13], [20, 21, 22, 23], [30, 31, 32, 33], [40, 41, 42, 43]])
    plain = tables.tolist()
    rows, held, new = [0, 1, far, -far, 3], [far, far - 1, 0, 0, 4], [[1, 2], [3, 4, 5], [6], [7], [8]]
    start = [0, 2, 5, 6, 7, 8]
    computed, lens = [17, 3, 5, 0, 33], [2, 1, 4, 2, 3]
    x = step_inputs(tables, to(rows), to(computed), to(lens), 12, 16, 4, to([b for n in new for b in n]), to(start), to(held))
    want = step_inputs_ref(plain, rows, computed, lens, 12, 16, 4, new, held)
    got = [v.tolist() for v in (x.query_start_loc, x.seq_lens, x.positions, x.slot_mapping, x.block_tables)]
    assert got == list(want[:5])
    assert tables.tolist() == plain
