"""Selection and attention over selected blocks where bounds, keys or values are infinite or NaN,
and the bits of the attention's weights."""

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


def _pool(ends, heads, d, dtype, seed):
    """K and V pools [pages, 256, heads, d] and a page table; NaN behind the last keys."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // 256) for n in ends]
    k, v = (torch.full((sum(need), 256, heads, d), NAN) for _ in range(2))
    order = torch.randperm(sum(need), generator=g).tolist()
    table = torch.zeros(len(ends), max(need), dtype=torch.int32)
    for b, n in enumerate(ends):
        for j in range(need[b]):
            p, fill = order.pop(), min(256, n - 256 * j)
            table[b, j] = p
            k[p, :fill] = torch.randn(fill, heads, d, generator=g)
            v[p, :fill] = torch.randn(fill, heads, d, generator=g)
    return k.to(dtype), v.to(dtype), table


def _attend(device, q, k, v, table, ends, block, budget, scale):
    """The kernel's result (double, on the host) and the definition's, over all blocks."""
    blocks = torch.arange(budget, dtype=torch.int32).view(1, 1, -1).repeat(len(ends), k.shape[2], 1)
    got = ops.block_sparse_attn(*(t.to(device) for t in (q, k, v, blocks, table)),
                                torch.tensor(ends, dtype=torch.int32, device=device), block_size=block, scale=scale)
    ref = oracle.sparse_attention(q, k, v, blocks, table, ends, range(len(ends)), block, scale)
    return got.double().cpu(), ref


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_keep_24_bits(device, dtype):
    """Two keys whose weights 1 and 1 - 2^-13 .. 1 - 2^-12 nearly cancel in V. Scores are exact
    in fp32 but for a rounding of 2^-24 of at most 2^-4; exp2 is within 2^-23 of a weight, the
    sums and the quotient within 2^-23 of 1 each: 2^-21 in all beside the output's own half
    step, which is 2^-21 at most. Weights of 16 bits are off by up to 2^-18."""
    say("sparse 24 bits", dtype)
    k, v = torch.zeros(1, 256, 1, 32), torch.zeros(1, 256, 1, 32)
    k[0, 0, 0, 0], k[0, 1, 0, 0] = 1, 1 + 2.0 ** -7
    v[0, 0], v[0, 1] = -1, 1
    q = torch.zeros(16, 8, 32)
    q[..., 0] = (2.0 ** -6 * (1 + torch.arange(128) / 128)).view(16, 8)
    got, ref = _attend(device, q.to(dtype), k.to(dtype), v.to(dtype), torch.zeros(16, 1, dtype=torch.int32), [2] * 16,
                       16, 1, 1.0)
    off = torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -7) + 2.0 ** -21
    assert ((got - ref).abs() <= off).all(), ((got - ref).abs() / off).max()


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_small_weights(device, dtype):
    """A key of weight 1 and V = 0 in every unit of 16, the others' weights e^-18 and V = 1024:
    all of the result comes from weights of 2^-26. Their exponent 25.97 is rounded to 2^-20,
    exp2 and up to 1000 sums in fp32 to 2^-23 + 1000 * 2^-24: within 2^-13 of the result."""
    say("sparse small weights", dtype)
    k, v = torch.full((4, 256, 1, 32), 0.0), torch.full((4, 256, 1, 32), 1024.0)
    k[..., 0] = -18
    k[:, ::16, 0, 0], v[:, ::16] = 0, 0
    q = torch.zeros(3, 2, 32)
    q[..., 0] = 1
    got, ref = _attend(device, q.to(dtype), k.to(dtype), v.to(dtype), torch.arange(4, dtype=torch.int32).repeat(3, 1),
                       [1000, 1024, 100], 64, 16, 1.0)
    assert ((got - ref).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -13) * ref.abs()).all()
