"""A drafted step at its edges, on the GPU.  Attention's tolerance is that of
test_gpu_tree.py, derived there."""

from __future__ import annotations

import pytest
import torch

from nanoserve_amd import commit_drafts, paged_attention_hip
from tests.test_gpu_tree import DEV, Case, close

pytestmark = pytest.mark.gpu
KERNELS = [(torch.float16, (14, 2, 64), 16), (torch.bfloat16, (28, 4, 128), 16),  # matrix cores
           (torch.float16, (6, 3, 96), 16), (torch.float32, (4, 2, 40), 4), (torch.float16, (14, 2, 64), 8)]  # plain


@pytest.mark.parametrize("dtype,heads,block_size", KERNELS)
@pytest.mark.parametrize("base", [32, 3040])
def test_a_block_outside_the_cache_under_drafted_rows(dtype, heads, block_size, base):
    """The sequence's last block, whose keys only some of its rows see: all of its rows are NaN, no others."""
    q = 20
    masks = [1 << j for j in range(5)] + [1 << j for j in range(q)] + [1, 2, 0]
    c = Case([30, base, 7], [5, q, 3], heads, dtype, block_size, masks=masks)
    ref, mag = c.reference()
    for bad in (-1, c.kc.shape[0], 1 << 40):
        md = c.md()
        md.block_tables[1, len(c.tables[1]) - 1] = bad
        out = c.run(md).cpu()
        assert torch.isnan(out[5:25]).all()
        keep = [*range(5), 25, 26, 27]
        close(out[keep], ref[keep], mag[keep], dtype, c.d, base + q)


@pytest.mark.parametrize("row_bytes,caches", [((1 << 20) - 1, 34), ((1 << 20) - 2, 70), ((1 << 20) - 4, 130),
                                              (1 << 20, 5), (6, 300)])
def test_commit_of_rows_of_a_mebibyte(row_bytes, caches):
    """More units of rows than one launch's grid holds."""
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    held = [torch.zeros(3, 1, 1, row_bytes, dtype=torch.uint8, device=DEV) for _ in range(caches)]
    g = torch.Generator(device=DEV).manual_seed(row_bytes)
    row = torch.randint(0, 256, (row_bytes,), dtype=torch.uint8, device=DEV, generator=g)
    for i, c in enumerate(held):
        c[2, 0, 0] = row + i
    counts, tokens = commit_drafts(to([7, 0, 3]), to([1, 5, 7]), to([-1, 0, 0]), to([0, 3]), to([0, 1, 2]),
                                   held[:caches // 2], held[caches // 2:], 3)
    assert counts.tolist() == [2] and tokens.tolist() == [[7, 3, -1]]
    for i, c in enumerate(held):
        assert torch.equal(c[1, 0, 0], row + i) and torch.equal(c[2], c[1]) and not c[0].any()


def test_commit_refuses_a_cache_that_is_listed_twice():
    to = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)  # noqa: E731
    both = torch.arange(2 * 3 * 16 * 8, device=DEV).half().view(2, 3, 16, 1, 8)
    before = both.clone()
    k, v = both.unbind()
    args = to([7, 0, 3]), to([1, 5, 7]), to([-1, 0, 0]), to([0, 3]), to([0, 1, 2])
    for caches in (([k, v], [k]), ([k], [k.view(3, 16, 1, 8)])):
        with pytest.raises(ValueError, match="twice"):
            commit_drafts(*args, *caches, 3)
    with pytest.raises(RuntimeError, match="invalid"):
        commit_drafts(*args, [both[0]], [both.view(6, 16, 1, 8)[1:4]], 3)
    assert torch.equal(both, before)
    commit_drafts(*args, [k], [v], 3)  # neighbours do not overlap
    assert torch.equal(both[:, 0, 1], before[:, 0, 2]) and torch.equal(both[:, 0, 2:], before[:, 0, 2:])


@pytest.mark.parametrize("dtype,heads,block_size", KERNELS)
def test_rows_whose_scores_are_all_minus_infinity(dtype, heads, block_size):
    """Count as rows without keys, in one range and in many, and as paged_attention_hip has them;
    one finite score among them takes all of the weight."""
    c = Case([40, 3000, 40, 0], [1, 1, 1, 1], heads, dtype, block_size, fill=0.0)
    c.query = c.query.abs() + 0.5
    for i in (0, 1, 3):
        c.kc[c.tables[i]] = -float("inf")
    md = c.md()
    out = c.run(md).cpu()
    ref, mag = c.reference()  # NaN in these rows
    zero = [0, 1, 3]
    assert (out[zero] == 0).all()
    close(out[2:3], ref[2:3], mag[2:3], dtype, c.d, 41)
    md.tree_mask, md.is_decode_only, md.query_start_loc = None, True, None
    assert (c.run(md, paged_attention_hip).cpu()[zero] == 0).all()
    for i, at in ((0, 40), (1, 1700), (3, 0)):  # a row of the tree, one of the prefix
        c.kc[c.tables[i][at // block_size], at % block_size] = 0.25
    c.check(c.run())
