"""Request settings of the sampler, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nanoserve_amd.sampling import SamplerInputs
from nanoserve_amd.scheduling import SamplingParams, Sequence


@pytest.mark.parametrize("bad", [dict(temperature=-0.1), dict(temperature=float("inf")), dict(temperature=float("nan")),
                                 dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.01), dict(min_p=-0.1), dict(min_p=1.1),
                                 dict(top_p=float("nan")), dict(seed=-1)])
def test_settings_out_of_range_are_refused(bad):
    with pytest.raises(ValueError):
        SamplingParams(**bad)


@pytest.mark.parametrize("bad", [dict(seed=1.5), dict(seed=float("nan")), dict(seed="7"), dict(top_k=float("nan"))])
def test_settings_that_would_fail_in_a_later_step_are_refused(bad):
    with pytest.raises(ValueError):
        SamplingParams(**bad)
    assert SamplingParams(seed=np.int64(7), top_k=np.int32(5)).seed == 7


def test_the_default_is_greedy():
    assert not SamplingParams().draws and SamplingParams(temperature=0.5).draws


def test_uniform_numbers_follow_the_seed_and_the_index_alone():
    a, b = (Sequence(i, [1], SamplingParams(max_new_tokens=5, temperature=1.0, seed=9)) for i in (0, 4))
    assert [a.uniform(i) for i in range(5)] == [b.uniform(i) for i in range(5)]
    assert b.uniform(3) == a.uniform(3)
    c, d = (Sequence(i, [1], SamplingParams(max_new_tokens=5, temperature=1.0)) for i in (0, 4))
    assert [c.uniform(i) for i in range(5)] != [d.uniform(i) for i in range(5)]  # the request's id
    u = [a.uniform(i) for i in range(5)]
    assert all(0 <= x < 1 for x in u) and len(set(u)) == 5
    assert a.uniform(20) < 1 and [a.uniform(i) for i in range(5)] == u  # past the length: the same start


def test_a_request_without_an_end_holds_no_more_numbers_than_it_has_used():
    a = Sequence(0, [1], SamplingParams(max_new_tokens=1 << 40, temperature=1.0, seed=2))
    b = Sequence(1, [1], SamplingParams(temperature=1.0, seed=2))
    b.uniform(5000)
    assert [a.uniform(i) for i in range(300)] == [b.uniform(i) for i in range(300)]
    assert len(a._uniform) < 1024


def test_staged_settings_are_the_requests():
    inputs = SamplerInputs(torch.device("cpu"), rows=2)
    seqs = [Sequence(i, [1], SamplingParams(temperature=0.5 + i, top_k=1 << (8 * i), top_p=0.9, min_p=0.1 * i, seed=i))
            for i in range(5)]  # more than there is room for
    seqs[2].output_token_ids = [4, 4]
    got = inputs.stage(seqs)
    assert got["temperature"].tolist() == [0.5, 1.5, 2.5, 3.5, 4.5]
    assert got["top_k"].dtype == torch.int32 and got["top_k"].tolist() == [1, 1 << 8, 1 << 16, 1 << 24, 0x7FFFFFFF]
    assert got["uniform"].tolist() == [s.uniform(len(s.output_token_ids)) for s in seqs]
    assert np.allclose(got["min_p"].numpy(), [0.0, 0.1, 0.2, 0.3, 0.4]) and np.allclose(got["top_p"].numpy(), 0.9)
