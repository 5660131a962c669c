"""Products with 4-bit weights of rows with infinite and NaN elements, the bits of normalised rows,
and memory behind the operands."""

from __future__ import annotations

import pytest
import torch

from helios_amd import ops
from oracle import decode_ops as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")


def _weight(rows, k, group, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    values = torch.randint(0, 16, (rows, k), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(k // group, rows, generator=g)) * 0.3 * k ** -0.5).to(dtype)
    zeros = torch.randint(0, 16, (k // group, rows), generator=g, dtype=torch.uint8)
    return values, scales, zeros


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,k,group", [(2, 40, 160, 32), (7, 33, 512, 128), (16, 100, 576, 64), (20, 2100, 160, 32),
                                               (64, 50, 2560, 128)])
def test_infinite_elements_of_x(device, rows, cols, k, group, dtype):
    """y has the infinities and NaN of sum_k x[k] W[k]: an infinity times a weight, NaN where that
    weight is 0 or infinities of both signs meet. Finite rows are the same bit for bit."""
    say("int4 infinite x", rows, cols, k, group, dtype)
    parts = _weight(cols, k, group, dtype, seed=rows)
    w = oracle.int4_matrix(*parts)
    packed = ops.int4_pack(*(p.to(device) for p in parts))
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(k)).to(dtype)
    residual = torch.randn(rows, cols, generator=torch.Generator().manual_seed(1)).to(dtype).to(device)
    clean = ops.int4_linear(x.to(device), packed, residual=residual)
    bad = x.clone()
    bad[0, k - 1] = INF
    bad[1, 3] = -INF
    spoiled = [0, 1]
    if rows > 5:
        bad[4, 5], bad[4, k // 2] = INF, -INF
        bad[5, 9] = NAN
        bad[rows - 1, k // 3], bad[rows - 1, 2] = INF, INF
        spoiled += [4, 5, rows - 1]
    got = ops.int4_linear(bad.to(device), packed, residual=residual)
    keep = [r for r in range(rows) if r not in spoiled]
    assert torch.equal(got[keep], clean[keep])
    y = torch.stack([(bad[r].double() * w).sum(1) for r in spoiled])
    got = got[spoiled].double().cpu()
    assert not torch.isfinite(y).any() and torch.isinf(y).any() and torch.isnan(y).any()
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    assert torch.equal(got[torch.isinf(y)], y[torch.isinf(y)])


def test_elements_near_the_end_of_the_range(device):
    """bfloat16 elements whose products with 16 + q leave fp32 where the result does not: fp32 sums
    of k terms of at most |x W|, k + 16 roundings."""
    say("int4 near the end of the range")
    parts = _weight(70, 256, 64, torch.bfloat16, seed=4)
    parts = (parts[0], parts[1] * 2.0 ** -8, parts[2])
    w = oracle.int4_matrix(*parts)
    x = torch.randn(18, 256, generator=torch.Generator().manual_seed(3))
    x[5] = 3e37 + 1e36 * x[5]
    x[17] *= 1e37
    x = x.to(torch.bfloat16)
    got = ops.int4_linear(x.to(device), ops.int4_pack(*(p.to(device) for p in parts))).double().cpu()
    y = x.double() @ w.t()
    most = x.double().abs() @ w.abs().t()
    off = 2.0 ** -8 * y.abs() + 2.0 ** -24 * (256 + 16) * 31 * most
    assert ((got - y).abs() <= off).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 4, 5, 8, 11, 16, 17, 40, 64])
def test_normalised_rows_keep_24_bits(device, rows, dtype):
    """Two elements, in groups of their own with weights of 15 s and -15 s, that normalise to values
    2^-12 of themselves apart. h = x r norm is rounded in fp32 (and r cancels but for 2^-20 of
    the small y); a group's sums are of 31 h, 16 h and 15 h with a rounding of 2^-24 each for every
    of three parts, so 220 h 2^-24 covers both. An h of 16 bits is off by up to 2^-17. Norm weights of
    2^-24 to 2^18, one of them 2^10 times the others where x is 0."""
    say("int4 24 bits", rows, dtype)
    g = torch.Generator().manual_seed(rows)
    values = torch.zeros(24, 64, dtype=torch.uint8)
    zeros = torch.zeros(2, 24, dtype=torch.uint8)
    values[:, 7], zeros[1] = 15, 15
    values[:, 32:] = 15
    values[:, 50] = 0
    scales = torch.ones(2, 24).to(dtype)
    x = torch.zeros(rows, 64)
    x[:, 7] = x[:, 50] = 1 + torch.rand(rows, generator=g)
    x = x.to(dtype)
    for seed in range(8):
        g = torch.Generator().manual_seed(seed)
        norm = torch.ones(64)
        norm[7] = 1 + torch.rand(1, generator=g)
        norm[50] = norm[7] * (1 + 2.0 ** -12 * (0.5 + torch.rand(1, generator=g)))
        norm[20] = 2.0 ** 10
        norm *= 2.0 ** (6 * (seed - 4))
        packed = ops.int4_pack(*(t.to(device) for t in (values, scales, zeros)))
        got = ops.int4_linear(x.to(device), packed, norm_weight=norm.to(device), eps=1e-6).double().cpu()
        h = x.double() / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6) * norm.double()
        y = h @ oracle.int4_matrix(values, scales, zeros).t()
        off = (torch.finfo(dtype).eps / 2 + 2.0 ** -19) * y.abs() + 2.0 ** -24 * 220 * h[:, 50:51].abs() \
            + torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2  # half of the smallest step
        assert ((got - y).abs() <= off).all(), ((got - y).abs() / off).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,group", [(1, 160, 32), (4, 32, 32), (7, 192, 64), (16, 96, 32), (33, 160, 32)])
def test_memory_behind_the_operands(device, rows, k, group, dtype):
    """K that ends inside a packed block of 128: what lies in memory behind x, the norm's weights,
    the packed weights and their steps does not show."""
    say("int4 memory behind", rows, k, group, dtype)
    parts = _weight(33, k, group, dtype, seed=k)
    w = ops.int4_pack(*(p.to(device) for p in parts))
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(1)).to(dtype).to(device)
    norm = 1 + 0.1 * torch.rand(k, generator=torch.Generator().manual_seed(2)).to(device)

    def inside(t, fill):
        flat = torch.full((t.numel() + 8192,), fill, dtype=t.dtype, device=device)
        flat[:t.numel()] = t.flatten()
        return flat[:t.numel()].view(t.shape)

    far = w._replace(packed=inside(w.packed, 255), steps=inside(w.steps, -1))  # steps of NaN
    for n in (None, norm):
        want = ops.int4_linear(x, w, norm_weight=n, eps=1e-6)
        got = ops.int4_linear(inside(x, NAN), far, norm_weight=None if n is None else inside(n, NAN), eps=1e-6)
        assert torch.isfinite(want).all() and torch.equal(got, want)
