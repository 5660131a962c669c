"""Selection and attention over selected blocks where bounds, keys or values are infinite or NaN."""

from __future__ import annotations

import pytest
import torch

from helios_amd import ops
from oracle import decode_ops as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")


def _scores(q, bounds, heads):
    """Scores [heads, blocks] of a query row [hq, d] for bounds [blocks, heads, 2, d] by their
    definition in 64 bits, a NaN as +inf."""
    qd = q.double().view(heads, -1, 1, q.shape[1])
    low, high = bounds.double().permute(2, 1, 0, 3)[:, :, None]
    s = torch.maximum(qd * low, qd * high).sum(dim=(1, 3))
    return torch.where(torch.isnan(s), INF, s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,hq,heads,d,count", [
    (1, 1, 1, 8, 300), (2, 6, 2, 64, 300), (1, 4, 4, 96, 150), (2, 5, 1, 128, 130), (1, 3, 1, 256, 70),
    (64, 8, 8, 16, 1200)])
def test_selection_by_bounds_with_one_infinity(device, rows, hq, heads, d, count, dtype):
    """One infinite bound in a dim whose queries all have one sign: the other bound's product is
    the larger, and the block's score stays finite. The score is infinite where the infinity is
    the larger, and where a query is 0 (0 * inf is a NaN, which counts as infinity). NaN bounds
    and infinite scores are equal: the earlier block goes first."""
    say("select one infinity", rows, hq, heads, d, count, dtype)
    g = torch.Generator().manual_seed(d + count)
    per_page = 16
    width = -(-count // per_page)
    mid, half = torch.randn(2, rows * width, per_page, heads, d, generator=g)
    bounds = torch.stack((mid - half.abs(), mid + half.abs()), dim=3).to(dtype)
    table = torch.randperm(rows * width, generator=g).view(rows, width).to(torch.int32)
    q = torch.randn(rows, hq, d, generator=g).to(dtype)
    q[..., 0], q[..., 1] = q[..., 0].abs() + 0.125, -q[..., 1].abs() - 0.125
    q[:, ::hq // heads, d - 1] = 0
    of = bounds[table.long()].flatten(1, 2)  # a copy: [rows, blocks, heads, 2, d]
    for step in range(0, count - 60, 60):
        of[:, step + 3, :, 0, 0] = -INF      # 0 * -inf is not in the definition
        of[:, step + 9, :, 1, 1] = INF
        of[:, step + 14, :, :, 0] = -INF     # the score is -inf
        of[:, step + 20, :, :, 1] = INF      # the score is -inf
        of[:, step + 25, :, 1, 0] = INF      # +inf
        of[:, step + 30, :, 0, d - 1] = -INF  # a query is 0 here
        of[:, step + 31, :, :, 2] = -NAN
        of[:, step + 33, :, 0, 0], of[:, step + 33, :, 1, 1] = -INF, INF
        of[:, step + 36, :, 0, 0], of[:, step + 36, :, 1, 0] = -INF, INF
    bounds[table.long()] = of.view(rows, width, per_page, heads, 2, d)
    scores = torch.stack([_scores(q[r], of[r, :count], heads) for r in range(rows)]).tolist()
    keys = torch.full((rows,), 16 * count - 3, dtype=torch.int32, device=device)
    args = [t.to(device) for t in (q, bounds, table)]
    for budget in (3, 4, 5, 9, 20, count // 2, count - 3, count - 1):
        want = torch.tensor([[oracle.select(s, count, budget, 1, 1) for s in row] for row in scores], dtype=torch.int32)
        got = ops.select_blocks(*args, keys, budget, block_size=16, sink=1, recent=1)
        assert torch.equal(got.cpu(), want), budget
