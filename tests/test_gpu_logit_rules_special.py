"""Logit rules on logits that are infinite or NaN, and rules that make them so."""

from __future__ import annotations

import pytest
import torch

from helios_amd import ops
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lead", [0, 3])
def test_nan_logits_under_rules(device, dtype, lead):
    """A NaN that a rule touches stays one and counts as the largest, one that a rule makes does too
    (inf - inf), and one that is not allowed does neither; rows on and off 16-byte addresses, in
    place and into rows that lie otherwise."""
    say("logit rules nan", dtype, lead)
    vocab = 9000
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(6, vocab, generator=g)
    logits[0, 4500] = NAN                       # touched by a token
    logits[1, 8999] = logits[1, 77] = NAN       # touched by a bias; the other by nothing
    logits[2, 300] = INF                        # inf - inf
    logits[3, 5000] = -NAN                      # not allowed
    logits[4, 20] = -INF                        # -inf * 2, -inf + bias
    logits[5, 4096] = INF                       # inf / 2 stays the largest
    logits = logits.to(dtype)
    tokens = torch.tensor([[4500, 2], [1, 2], [300, 5], [5000, 6], [20, 7], [4096, 8]], dtype=torch.int32)
    presence = torch.tensor([0.5, 0.5, INF, 0.5, 0.5, 0.5])
    bias_ids = torch.tensor([[3], [8999], [3], [3], [20], [3]], dtype=torch.int32)
    bias = torch.full((6, 1), 0.25)
    allowed = torch.full((6, 282), -1, dtype=torch.int32)
    allowed[3, 5000 // 32] &= ~(1 << 5000 % 32)
    x = logits.float().clone()
    for r in range(6):
        for t in tokens[r].tolist():
            l = x[r, t]
            x[r, t] = (l / 2 if l > 0 else l * 2) - (0.0 + presence[r])
        x[r, bias_ids[r, 0]] += 0.25
    want = x.to(dtype)
    want[3, 5000] = -INF
    ids = [4500, 77, 300, int(want[3].float().argmax()), int(want[4].float().argmax()), 4096]
    rules = ops.LogitRules(
        tokens=tokens.to(device), lengths=torch.full((6,), 2, dtype=torch.int32, device=device),
        repetition=torch.full((6,), 2.0, device=device), presence=presence.to(device), bias_ids=bias_ids.to(device),
        bias_values=bias.to(device), allowed=allowed.to(device))
    wide = torch.zeros(6, vocab + 8, dtype=dtype, device=device)
    wide[:, lead:lead + vocab] = logits.to(device)
    rows = wide[:, lead:lead + vocab]
    place = wide.clone()[:, lead:lead + vocab]
    for got in (ops.apply_logit_rules(rows, rules), ops.apply_logit_rules(place, rules, out=place),
                ops.apply_logit_rules(rows, rules, return_logits=False)):
        assert got.token_ids.tolist() == ids
        if got.logits is not None:
            out = got.logits.float().cpu()
            assert torch.equal(torch.isnan(out), torch.isnan(want.float()))
            fine = ~torch.isnan(out)
            assert torch.equal(out[fine], want.float()[fine])
