"""ns_sample_rows against the float64 oracle on an MI355X: the tokens are equal.

The kernel's weights are exact to 2^-45 of a row's largest and its sums exact,
so a token can differ from the oracle's only where a uniform number or a filter
falls within ~1e-11 of a border; none of the drawn ones does."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nanoserve_amd import argmax_rows, sample_rows
from nanoserve_amd.capture import graph_capture
from oracle.sampling import sample_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _dev(x):
    return None if x is None else x.to(DEV)


def _check(z, u, t, k=None, p=None, mp=None):
    got = sample_rows(z.to(DEV), _dev(u), _dev(t), _dev(k), _dev(p), _dev(mp))
    assert got.dtype == torch.int64 and got.shape == (z.shape[0],)
    want = sample_ref(z.float().numpy(), u.numpy(), t.numpy(), *(None if x is None else x.numpy() for x in (k, p, mp)))
    assert got.tolist() == want


def _settings(M, seed, which="tkpm"):
    g = _g(seed)
    pick = lambda v, ty: torch.tensor(v, dtype=ty)[torch.randint(0, len(v), (M,), generator=g)]  # noqa: E731
    return (torch.rand(M, generator=g), pick([0.5, 0.8, 1.0, 1.7], torch.float32),
            pick([0, 1, 5, 50, 1000, 1 << 30], torch.int64) if "k" in which else None,
            pick([0.3, 0.9, 0.95, 0.999, 1.0], torch.float32) if "p" in which else None,
            pick([0.0, 0.01, 0.1, 0.5], torch.float32) if "m" in which else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["t", "tk", "tp", "tm", "tkpm"])
@pytest.mark.parametrize("M,N", [(1, 151936), (24, 20011), (5, 1), (9, 13), (40, 777), (3, 4096)])
def test_matches_float64(M, N, which, dtype):
    z = (torch.randn(M, N, generator=_g(N)) * 2.5).to(dtype)
    _check(z, *_settings(M, N + 1, which))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(1024, 300), (300, 9001), (200, 20011), (110, 30000), (70, 4097)])
def test_many_rows_with_a_top_k(M, N, dtype):
    """Every way in which rows are cut, top-k on both sides of the number of groups of threads."""
    z = (torch.randn(M, N, generator=_g(N)) * 2.5).to(dtype)
    u, t, k, p, mp = _settings(M, M)
    k = torch.tensor([1, 2, 40, 400, 768, 1000, 1023, 1024, 1025, 4096, 0])[torch.arange(M) % 11]
    _check(z, u, t, k, p, mp)
    _check(z, u, t, k.int())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M", [2, 200])
def test_more_equal_largest_elements_than_are_listed(M, dtype):
    """The first bin holds from half a workgroup's share of the list to more than the whole list."""
    N = 20000
    z = torch.randn(M, N, generator=_g(1))
    for r in range(M):
        n = (500, 1025, 3000, 4096, 4097, 20000)[r % 6]
        z[r, r:r + n] = 9.0                                 # side by side: one slice's
        z[r, torch.randperm(N, generator=_g(r))[:n // 2]] = 9.0
    z[0, 5:9] = -torch.inf
    u, t, _, p, mp = _settings(M, 3)
    _check(z.to(dtype), u, t, torch.tensor([50, 3, 1000, 700])[torch.arange(M) % 4], p, mp)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_and_few_values(dtype):
    """Bins that hold far more elements than the last stage sorts at once."""
    N = 60000
    z = torch.zeros(6, N)
    z[1, 100:200] = 1.0
    z[2] = torch.randint(0, 3, (N,), generator=_g(0)).float()
    z[3] = torch.randint(0, 40, (N,), generator=_g(1)).float() / 64
    z[4] = -50.0
    z[4, 7] = 0.0                       # one token and a far tail
    z[5] = torch.randn(N, generator=_g(2)) * 1e-3
    z = z.to(dtype)
    u, one = torch.tensor([0.0, 0.3, 0.61, 0.99, 0.5, 0.77]), torch.ones(6)
    _check(z, u, one)
    _check(z, u, one, k=torch.full((6,), 20000))
    _check(z, u, one, p=torch.full((6,), 0.37))
    _check(z, u, one, k=torch.full((6,), 30001, dtype=torch.int32), p=torch.full((6,), 0.83), mp=torch.full((6,), 0.4))
    _check(z, u, torch.full((6,), 1e-3))
    _check(z, u, torch.full((6,), 50.0))


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_logits_and_greedy_rows(dtype):
    N = 5000
    z = (torch.randn(8, N, generator=_g(0)) * 2).to(dtype)
    z[0, 100:] = -torch.inf
    z[1] = -torch.inf
    z[1, 4000] = -1.0                  # a single choice
    z[2] = -torch.inf                  # no choice: the first index
    z[3, 77] = torch.nan
    z[4, 9], z[4, 50] = torch.inf, torch.inf
    z[6, ::2] = torch.finfo(dtype).min
    u = torch.linspace(0.05, 0.95, 8)
    t = torch.tensor([1.0, 1.0, 1.0, 1.0, 1.0, 0.0, 1.0, -1.0])
    _check(z, u, t)
    _check(z, u, t, k=torch.full((8,), 300), p=torch.full((8,), 0.9), mp=torch.full((8,), 0.02))
    # Rows without a temperature are argmax_rows'.
    got = sample_rows(z.to(DEV), u.to(DEV), 0.0)
    assert torch.equal(got, argmax_rows(z.to(DEV)))
    _check(z, u, torch.full((8,), torch.inf))


def test_settings_at_and_past_their_limits():
    N = 3000
    z = torch.randn(1, N, generator=_g(3)).repeat(12, 1)
    u = torch.tensor([0.0, 1.0, 0.99999994, -1.0, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5, 0.5])
    t = torch.tensor([1.0] * 11 + [1e-30])
    k = torch.tensor([0, 0, 0, 0, -3, N, N + 1, 1, N - 1, 0, 0, 0])
    p = torch.tensor([1.0, 1.0, 1.0, 1.0, 2.0, 1.0, 0.0, -1.0, 1.0, 1e-30, 0.99999994, 1.0])
    mp = torch.tensor([0.0, 0.0, 0.0, 0.0, -1.0, 1.0, 0.0, 0.0, 0.0, 2.0, 1e-30, 0.0])
    _check(z, u, t, k, p, mp)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_and_unaligned_rows(dtype):
    base = (torch.randn(9, 2011, generator=_g(0)) * 2).to(dtype)
    dev = base.to(DEV)
    u, t, k, p, mp = _settings(9, 1)
    for lo, hi in ((0, 2011), (1, 2000), (3, 5), (7, 2011)):
        z = dev[:, lo:hi]
        want = sample_ref(base[:, lo:hi].float().numpy(), u.numpy(), t.numpy(), k.numpy(), p.numpy(), mp.numpy())
        assert sample_rows(z, u.to(DEV), t.to(DEV), k.to(DEV), p.to(DEV), mp.to(DEV)).tolist() == want
    z = dev.t().contiguous().t()  # no unit stride
    want = sample_ref(base.float().numpy(), u.numpy(), t.numpy())
    assert sample_rows(z, u.to(DEV), t.to(DEV)).tolist() == want
    assert sample_rows(dev[2:3].expand(4, 2011), u[:4].to(DEV), t[:4].to(DEV)).tolist() == sample_ref(
        base[2:3].expand(4, 2011).float().numpy(), u.numpy(), t.numpy())


def test_numbers_for_all_rows_and_an_output():
    z = torch.randn(5, 900, generator=_g(0))
    u = torch.rand(5, generator=_g(1))
    out = torch.full((5,), -1, dtype=torch.int64, device=DEV)
    got = sample_rows(z.to(DEV), u.to(DEV), 0.7, top_k=30, top_p=0.8, min_p=0.05, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert out.tolist() == sample_ref(z.numpy(), u.numpy(), np.full(5, np.float32(0.7)), [30] * 5,
                                      np.full(5, np.float32(0.8)), np.full(5, np.float32(0.05)))


def test_draws_follow_the_probabilities():
    """20000 draws from one row: each count within five standard deviations."""
    n = 20000
    z = torch.tensor([2.0, 1.0, 0.0, -1.0, 3.0, -4.0])
    u = torch.rand(n, generator=_g(5))
    got = sample_rows(z.to(DEV).expand(n, 6), u.to(DEV), 1.0)
    p = torch.softmax(z.double(), 0)
    count = torch.bincount(got.cpu(), minlength=6)
    assert ((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()


def test_refuses_what_it_cannot_take():
    z, u = torch.zeros(3, 50, device=DEV), torch.zeros(3, device=DEV)
    for kw, err in ((dict(uniform=u[:2]), ValueError), (dict(uniform=u.double()), TypeError),
                    (dict(uniform=None), ValueError), (dict(uniform=u.cpu()), ValueError),
                    (dict(temperature=u[None]), ValueError), (dict(top_k=u), TypeError),
                    (dict(top_p=u.half()), TypeError), (dict(out=torch.zeros(3, device=DEV)), ValueError),
                    (dict(logits=z.int()), TypeError), (dict(logits=z[0]), ValueError),
                    (dict(logits=z[:, :0]), RuntimeError)):
        with pytest.raises(err):
            sample_rows(**{**dict(logits=z, uniform=u, temperature=1.0), **kw})
    assert sample_rows(z[:0], u[:0], 1.0).shape == (0,)


def test_graph_replays_with_eager_calls_between_and_streams():
    M, N = 7, 30000
    z = (torch.randn(M, N, generator=_g(0)) * 2).half().to(DEV)
    settings = [x.to(DEV) for x in _settings(M, 4)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        sample_rows(z, *settings)
    s.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with graph_capture(g, s):
            outs.append(sample_rows(z, *settings))
        graphs.append(g)
    for step in range(4):
        z.copy_((torch.randn(M, N, generator=_g(step + 10)) * 2).half())
        settings[0].copy_(torch.rand(M, generator=_g(step)))
        want = sample_rows(z, *settings)
        torch.cuda.synchronize()
        for g in graphs:  # both at once
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        assert want.tolist() == sample_ref(z.float().cpu().numpy(), *(x.cpu().numpy() for x in settings))
