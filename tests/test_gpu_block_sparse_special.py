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


def _expect(got, ref, dtype, most):
    """NaN and infinities where the definition has them; elsewhere its values to the output's half
    step, and 2^-16 of the values weighed (weights, exp and sums in fp32)."""
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf])
    fine = torch.isfinite(ref)
    off = torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -16 * most
    assert ((got - ref).abs()[fine] <= off[fine]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,ends", [
    (4, 1, 64, [256, 40, 1000]), (16, 2, 128, [300] * 3), (3, 1, 200, [17, 900]), (8, 8, 128, [1000] * 40)])
def test_infinite_and_nan_values(device, hq, heads, d, ends, dtype):
    """An infinite or NaN element of V that a row sees makes that element of its result infinite or
    NaN, for every head of the group and at any weight, and no other element."""
    say("sparse infinite values", hq, heads, d, dtype)
    k, v, table = _pool(ends, heads, d, dtype, seed=d + hq)
    q = torch.randn(len(ends), hq, d, generator=torch.Generator().manual_seed(1)).to(dtype)
    for b, n in enumerate(ends):
        at = lambda t: (int(table[b, t // 256]), t % 256, b % heads)  # noqa: E731
        v[at(n - 1)][5] = INF
        v[at(0)][9] = -INF
        v[at(n // 2)][12], v[at(n // 3)][12] = INF, -INF
        v[at(n // 2)][d - 1] = NAN
        v[at(n // 3)][13] = v[at(n - 2)][13] = -INF
        # This key's weight is e^-60 or less of the largest for every query.
        far = at(n // 4)
        k[far] = 0
        v[far][20] = INF
    k[..., 0] += 60
    q[..., 0] = 9 * (d / 64) ** 0.5
    for b, n in enumerate(ends):
        k[int(table[b, n // 4 // 256]), n // 4 % 256, b % heads, 0] = 0
    got, ref = _attend(device, q, k, v, table, ends, 64, 16, d ** -0.5)
    _expect(got, ref, dtype, 6.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ends", [[100, 40, 256, 17], [1000] * 4])
def test_infinite_and_nan_keys(device, ends, dtype):
    """A score of -inf is a weight of 0, one of +inf or NaN makes the row NaN, for the heads that
    have it alone; a row whose scores are all -inf gets zeros."""
    say("sparse infinite keys", dtype)
    k, v, table = _pool(ends, 1, 64, dtype, seed=11)
    q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    q[:, :, 0] = torch.tensor([1.0, -1.0, 2.0, 0.0])
    first = table[:, 0].tolist()
    k[first[0], 7, 0, 0] = -INF      # head 0, 2: no weight; 1: NaN (+inf); 3: NaN (0 * inf)
    k[first[1], 16, 0, 3] = NAN      # all of the row
    k[first[2], :, 0, 0] = -INF      # every key of the sequence
    for p in table[2].tolist():
        k[p, :, 0, 0] = torch.where(torch.isnan(k[p, :, 0, 0]), k[p, :, 0, 0], torch.tensor(-INF, dtype=dtype))
    got, ref = _attend(device, q, k, v, table, ends, 64, 16, 0.125)
    assert torch.isnan(ref[0, [1, 3]]).all() and torch.isfinite(ref[0, [0, 2]]).all() and torch.isnan(ref[1]).all()
    assert torch.isnan(ref[2]).all() and (got[2, [0, 2]] == 0).all() and torch.isnan(got[2, [1, 3]]).all()
    keep = [0, 1, 3]
    _expect(got[keep], ref[keep], dtype, 6.0)
