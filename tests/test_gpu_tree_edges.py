"""A drafted step at its edges, on the GPU.  Attention's tolerance is that of
test_gpu_tree.py, derived there."""

from __future__ import annotations

import pytest
import torch

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
