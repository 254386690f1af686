"""The plain path of drawing from given numbers, against extended precision; its refusals."""

import math

import numpy as np
import pytest
import torch

from astrai_b200.inference.sample import sample_given
from tests.sample_oracle import oracle


@pytest.mark.parametrize("s", [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=5, top_p=0.9), dict(top_k=40),
                               dict(top_p=0.8), dict(min_p=0.1), dict(temperature=2.0, top_p=0.9, min_p=0.05), dict(top_p=0.0),
                               dict(min_p=1.0), dict(top_k=1000)])
def test_against_the_definition(s):
    g = torch.Generator().manual_seed(0)
    x = 2 * torch.randn(40, 60, generator=g)
    x[:5] = x[:5].round()
    x[5, 7:] = -math.inf
    u = torch.rand(40, generator=g)
    token, logprob = sample_given(x, u, return_logprobs=True, **s)
    for r in range(40):
        t, p, m = (float(np.float32(s.get(n, d))) for n, d in (("temperature", 1.0), ("top_p", 1.0), ("min_p", 0.0)))
        want, lp, near = oracle(x[r].double().numpy(), float(u[r]), t, s.get("top_k", 0), p, m)
        assert near < 1e-12 or int(token[r]) == want
        assert near < 1e-12 or abs(float(logprob[r]) - lp) <= 1e-6


def test_rows_without_a_distribution():
    x = torch.zeros(4, 5)
    x[0] = -math.inf
    x[1, 0] = math.nan
    x[1, 3] = 2.0
    x[2] = math.nan
    x[3, 2] = math.inf
    token, logprob = sample_given(x, torch.rand(4), return_logprobs=True)
    assert token.tolist() == [0, 3, 0, 2] and logprob.isnan().all()


def test_refusals():
    x, u = torch.randn(3, 10), torch.rand(3)
    for bad in (dict(temperature=-1.0), dict(top_k=-1), dict(top_p=1.5), dict(top_p=math.nan), dict(min_p=-0.1),
                dict(uniform=u[:2]), dict(top_k=torch.zeros(2)), dict(logits=x[0])):
        with pytest.raises(ValueError):
            sample_given(**{"logits": x, "uniform": u, **bad})


def test_top_k_beyond_32_bits_is_off():
    g = torch.Generator().manual_seed(1)
    x, u = torch.randn(8, 30, generator=g), torch.rand(8, generator=g)
    off = sample_given(x, u)
    for k in (2 ** 31 + 1, 2 ** 32 + 1, 2 ** 40 + 3, -1, -2 ** 32 + 1):
        for n in (1, 8):
            assert torch.equal(sample_given(x, u, top_k=torch.full((n,), k)), off)
