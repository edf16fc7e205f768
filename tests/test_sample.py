"""sample_tokens without a GPU: refusals, and the tests' own oracle."""

import math

import pytest
import torch

import cutilegpt_amd as cg
from cutilegpt_amd import _lib
from sample_ref import draw, kept

P = 1 << 20  # a pointer that is never followed
EINVAL, EDTYPE, ESHAPE = -1, -2, -3


def call(**change):
    a = dict(x=P, rows=0, cols=100, ld=100, dtype=_lib.CGPT_F32, u=P, temperature=None, top_k=None, top_p=None, min_p=None,
             temperature_all=1.0, top_k_all=0, top_p_all=1.0, min_p_all=0.0, ids=P)
    assert set(change) <= set(a)
    a.update(change)
    return _lib.load().cgpt_sample(*a.values(), None)


def test_c_entry_refuses():
    assert call() == 0
    for change, status in ((dict(rows=-1), EINVAL), (dict(cols=0), EINVAL), (dict(ld=99), EINVAL), (dict(dtype=5), EDTYPE),
                           (dict(cols=(1 << 20) + 1, ld=1 << 21), ESHAPE), (dict(rows=1 << 23), ESHAPE),
                           (dict(temperature_all=-1.0), EINVAL), (dict(temperature_all=math.nan), EINVAL),
                           (dict(top_k_all=-1), EINVAL), (dict(top_p_all=-0.1), EINVAL), (dict(top_p_all=math.nan), EINVAL),
                           (dict(min_p_all=1.5), EINVAL), (dict(min_p_all=math.nan), EINVAL)):
        assert call(**change) == status, change
    for change in (dict(x=0), dict(u=0), dict(ids=0), dict(x=P + 2), dict(ids=P + 4), dict(u=P + 2), dict(temperature=P + 1),
                   dict(top_k=P + 3), dict(top_p=P + 1), dict(min_p=P + 2), dict(x=P + 1, dtype=_lib.CGPT_BF16)):
        assert call(rows=1, **change) == EINVAL, change
    # A setting of the rows makes the common one unread.
    assert call(temperature=P, temperature_all=-1.0, top_k=P, top_k_all=-1, top_p=P, top_p_all=math.nan, min_p=P, min_p_all=9.0) == 0


def test_wrapper_refuses_host_tensors():
    with pytest.raises(ValueError, match="one GPU"):
        cg.sample_tokens(torch.zeros(1, 5), torch.zeros(1))
    with pytest.raises(ValueError, match="one GPU"):
        cg.sample_tokens([1.0], torch.zeros(1))


def test_oracle_cuts():
    x = torch.tensor([1.0, 3.0, 3.0, -math.inf, 2.0, math.nan])
    assert kept(x, 1.0, 0, 1.0, 0.0)[0] == [1, 2, 4, 0]
    assert kept(x, 1.0, 2, 1.0, 0.0)[0] == [1, 2] and kept(x, 1.0, 1, 1.0, 0.0)[0] == [1]
    # Weights 1, 1, e^-1, e^-2: two thirds of the sum 2.503 are reached by the second.
    assert kept(x, 1.0, 0, 0.66, 0.0)[0] == [1, 2] and kept(x, 1.0, 0, 0.82, 0.0)[0] == [1, 2, 4]
    assert kept(x, 1.0, 2, 0.5, 0.0)[0] == [1] and kept(x, 1.0, 0, 0.0, 0.0)[0] == [1]
    assert kept(x, 1.0, 0, 1.0, 0.3)[0] == [1, 2, 4] and kept(x, 1.0, 0, 1.0, 1.0)[0] == [1, 2]
    assert kept(x, 0.0, 0, 1.0, 0.0)[0] == [1]
    assert draw(x, 0.0)[0] == 0 and draw(x, 0.999)[0] == 4 and draw(x[3:4], 0.5)[0] == -1


def test_oracle_frequencies():
    """Draws at evenly spaced numbers hit every token as often as its weight says."""
    x = torch.tensor([0.3, -1.0, 2.0, 0.3, 1.1])
    n = 4000
    hits = torch.zeros(5)
    for i in range(n):
        hits[draw(x, (i + 0.5) / n, T=0.7)[0]] += 1
    assert bool(((hits / n - torch.softmax(x / 0.7, 0)).abs() <= 1.0 / n).all())
