"""Drawn tokens where no token reaches a limit, on each way through a row."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_cases import say
from tests.test_gpu_sample import DTYPES, INF, _check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
def test_min_p_above_one(device, dtype):
    """No token's weight reaches min_p: the first one is kept alone, with a logprob of 0, by short lists,
    by lists of a small top_k, and past both."""
    say("sample min_p above 1", dtype)
    g = torch.Generator().manual_seed(1)
    rows, vocab = 6, 151936
    logits = torch.randn(rows, vocab, generator=g) * torch.tensor([0.5, 3.0, 0.01, 1.0, 0.5, 2.0])[:, None]
    logits[3] = 0.0
    logits[3, 5::3] = 7.0                 # more of the largest than one list holds
    logits[4, 70:] = -INF
    logits = logits.to(dtype)
    u = torch.tensor([0.0, 0.3, 0.5, 0.9, 0.99, 1.0])
    m = torch.tensor([1.5, 1.0 + 2.0 ** -23, 2.0, 1e30, INF, 3.4e38])
    k = torch.tensor([5000, 50, 0, 20000, 7, 100000], dtype=torch.int32)
    p = torch.full((rows,), 0.9)
    for limits in (dict(), dict(top_k=k), dict(top_p=p), dict(top_k=k, top_p=p),
                   dict(top_k=k.flip(0), top_p=p, temperature=torch.tensor([0.5, 2.0, 30.0, 1.0, 1e-3, 1e6]))):
        got = _check(device, logits, u, min_p=m, **limits)
        assert (got.logprobs == 0).all()
