"""The sampler's oracle, pinned on the CPU, and what the product refuses without a GPU."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nanoserve_amd import _lib, sample_rows
from oracle.sampling import sample_ref, sample_row


def _kept(z, **settings):
    """The tokens that some uniform number draws."""
    return sorted({sample_row(z, u, 1.0, **settings) for u in np.linspace(0, 1, 20001, endpoint=False)})


def test_filters_on_a_small_row():
    p = np.array([0.1, 0.4, 0.05, 0.3, 0.15])
    z = np.log(p)
    assert _kept(z) == [0, 1, 2, 3, 4]
    assert _kept(z, top_k=2) == [1, 3]
    assert _kept(z, top_p=0.4) == [1] and _kept(z, top_p=0.41) == [1, 3]
    assert _kept(z, top_p=0.0) == [1] and _kept(z, top_k=1, top_p=0.5) == [1]
    # After top-k the probabilities are 0.4 / 0.85, 0.3 / 0.85, 0.15 / 0.85.
    assert _kept(z, top_k=3, top_p=0.83) == [1, 3, 4] and _kept(z, top_k=3, top_p=0.81) == [1, 3]
    assert _kept(z, min_p=0.3) == [1, 3, 4] and _kept(z, min_p=1.5) == [1]


def test_the_share_of_uniform_numbers_is_the_probability():
    z = np.random.default_rng(0).normal(size=6) * 2
    t = 0.7
    p = np.exp(z / t) / np.exp(z / t).sum()
    u = (np.arange(200000) + 0.5) / 200000
    got = np.bincount([sample_row(z, x, t) for x in u[::20]], minlength=6) / len(u[::20])
    assert np.abs(got - p).max() < 6 / 10000  # each border is off by less than one of 10000 points


def test_ties_go_to_the_lower_index_first():
    z = np.zeros(4)
    assert [sample_row(z, u, 1.0) for u in (0.0, 0.24, 0.26, 0.51, 0.99)] == [0, 0, 1, 2, 3]
    assert _kept(z, top_k=2) == [0, 1]


def test_greedy_rows():
    nan, inf = math.nan, math.inf
    assert sample_row([1.0, 3.0, 3.0], 0.9, 0.0) == 1
    assert sample_row([1.0, nan, 3.0], 0.9, 1.0) == 1
    assert sample_row([1.0, inf, inf], 0.9, 1.0) == 1
    assert sample_row([-inf, -inf], 0.9, 1.0) == 0
    assert sample_row([0.0, -inf, 0.0], 0.9, math.inf) == 2  # an infinite temperature: the finite ones alike


def test_against_torch_on_random_rows():
    g = torch.Generator().manual_seed(0)
    z = torch.randn(8, 50, generator=g, dtype=torch.float64)
    u = torch.rand(8, generator=g, dtype=torch.float64)
    got = sample_ref(z.numpy(), u.numpy(), [0.8] * 8, top_k=[20] * 8, top_p=[0.9] * 8)
    for i in range(8):
        v, at = (z[i] / 0.8).sort(descending=True)
        v[20:] = -math.inf
        p = v.softmax(0)
        p[p.cumsum(0) - p >= 0.9] = 0
        p /= p.sum()
        assert got[i] == int(at[(p.cumsum(0) > u[i]).nonzero()[0]])


def test_the_product_has_no_cpu_path():
    with pytest.raises(ValueError, match="GPU"):
        sample_rows(torch.zeros(2, 5), torch.zeros(2), 1.0)
    with pytest.raises(ValueError):
        sample_rows(torch.zeros(5), torch.zeros(2), 1.0)


INV, UNS, WS = _lib.NS_ERR_INVALID_ARG, _lib.NS_ERR_UNSUPPORTED, _lib.NS_ERR_WORKSPACE


def _args(**over):
    a = dict(out=16, x=16, st=1000, M=4, N=1000, dtype=_lib.NS_DTYPE_F16, u=16, t=16, k=None, k64=1, p=None, mp=None,
             ws=16, ws_bytes=1 << 30, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(out=None), INV), (dict(x=None), INV), (dict(u=None), INV), (dict(t=None), INV), (dict(M=-1), INV),
    (dict(N=0), INV), (dict(st=999), INV), (dict(M=65536), INV), (dict(N=1 << 31, st=1 << 31), INV), (dict(x=17), INV),
    (dict(out=12), INV), (dict(u=18), INV), (dict(k=12), INV), (dict(k=18, k64=0), INV), (dict(p=18), INV),
    (dict(mp=18), INV), (dict(dtype=7), UNS), (dict(ws=None), WS), (dict(ws_bytes=100), WS), (dict(ws=20), WS),
])
def test_sample_rejects_bad_arguments(over, code):
    assert _lib.load().ns_sample_rows(*_args(**over)) == code


def test_no_rows_is_a_no_op_and_the_workspace_grows_with_the_rows():
    lib = _lib.load()
    assert lib.ns_sample_rows(*_args(M=0, out=None)) == _lib.NS_OK
    size = lib.ns_sample_rows_workspace_size
    assert 0 < size(1, 5) < size(1, 151936) < size(32, 151936)
    assert size(0, 5) == 0 and size(5, 0) == 0 and size(65536, 5) == 0
