"""Products with 4-bit weights against 64 bits: row tiles, groups, odd widths and K that end
inside a packed block, each step that rides on the product."""

from __future__ import annotations

import pytest
import torch

from helios_amd import ops
from oracle import decode_ops as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def _weight(rows, k, group, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    values = torch.randint(0, 16, (rows, k), generator=g, dtype=torch.uint8)
    scales = ((0.5 + torch.rand(k // group, rows, generator=g)) * 0.3 * k ** -0.5).to(dtype)
    zeros = torch.randint(0, 16, (k // group, rows), generator=g, dtype=torch.uint8)
    return values, scales, zeros


def _packed(values, scales, zeros, device):
    return ops.int4_pack(values.to(device), scales.to(device), zeros.to(device))


def _check(got, x, values, scales, zeros, norm, residual, swiglu):
    """y is a fp32 sum: groups of up to 128 terms of at most 31 s |h|, the correction of the same
    size, then up to k / 32 groups and 8 waves: (128 + 128 + k / 32 + 16) roundings of the sum of
    those terms at most. A normalised h is two bf16 numbers: within 2^-17 of itself; rsqrt and
    the mean within 2^-20. The output's own rounding is half a step."""
    dtype, k = x.dtype, x.shape[1]
    w = oracle.int4_matrix(values, scales, zeros)
    h = x.double()
    if norm is not None:
        h = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * norm.double()
    y = h @ w.t()
    group = k // scales.shape[0]
    most = h.abs() @ (31 * scales.double().t().repeat_interleave(group, 1)).t()
    off = 2.0 ** -24 * (272 + k / 32) * most
    if norm is not None:
        off += (2.0 ** -17 + 2.0 ** -20) * (h.abs() @ w.abs().t())
    if swiglu:
        gate, up = y.chunk(2, 1)
        go, uo = off.chunk(2, 1)
        y = gate * torch.sigmoid(gate) * up
        # |silu'| <= 1.1, |silu(g)| <= |g|; silu and the product to a few fp32 steps
        off = 1.1 * go * (up.abs() + uo) + (gate.abs() + go) * uo + 2.0 ** -21 * y.abs()
    if residual is not None:
        y = residual.double() + y
        off += 2.0 ** -24 * y.abs()
    off = off * (1 + torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * y.abs() + torch.finfo(dtype).tiny
    err = (got.double().cpu() - y).abs()
    assert (err <= off).all(), (err / off).max()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,k,group", [(1, 16, 128, 128), (3, 1, 32, 32), (16, 40, 576, 64), (17, 33, 160, 32),
                                               (32, 48, 1152, 128), (33, 17, 2560, 128), (64, 130, 1344, 64), (50, 2100, 160, 32),
                                               (50, 4200, 96, 32)])
def test_int4_linear(device, rows, cols, k, group, dtype):
    say("int4_linear", rows, cols, k, group, dtype)
    g = torch.Generator().manual_seed(rows + cols + k)
    x = torch.randn(rows, k, generator=g).to(dtype)
    norm = 1 + 0.1 * torch.randn(k, generator=g)
    residual = torch.randn(rows, cols, generator=g).to(dtype)
    parts = _weight(2 * cols, k, group, dtype, seed=rows * k)
    half = tuple(t[:cols] if i == 0 else t[:, :cols].contiguous() for i, t in enumerate(parts))
    both, one = _packed(*parts, device), _packed(*half, device)
    xd, rd = x.to(device), residual.to(device)
    for n in (None, norm):
        nd = None if n is None else n.to(device)
        kw = dict(norm_weight=nd, eps=1e-6)
        _check(ops.int4_linear(xd, one, **kw), x, *half, n, None, False)
        _check(ops.int4_linear(xd, one, residual=rd, **kw), x, *half, n, residual, False)
        _check(ops.int4_linear(xd, both, swiglu=True, **kw), x, *parts, n, None, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_int4_linear_large_values(device, dtype):
    """x * norm_weight beyond the type's range, where the normalised row is not."""
    say("int4 large", dtype)
    x = torch.full((2, 256), 3e4 if dtype == torch.float16 else 1e18).to(dtype)
    x[1] = -x[1] * torch.linspace(0.1, 1, 256).to(dtype)
    norm = torch.full((256,), 8.0)
    parts = _weight(24, 256, 32, dtype, seed=3)
    _check(ops.int4_linear(x.to(device), _packed(*parts, device), norm_weight=norm.to(device), eps=1e-6), x, *parts,
           norm, None, False)


@pytest.mark.parametrize("rows", [2, 20, 64])
def test_int4_rows_do_not_mix(device, rows):
    """A row's infinities and NaN stay in it; rows equal bit for bit whatever their neighbours."""
    say("int4 rows", rows)
    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 512, generator=g).to(torch.bfloat16).to(device)
    w = _packed(*_weight(48, 512, 128, torch.bfloat16, seed=5), device)
    norm = torch.ones(512, device=device)
    for n in (None, norm):
        clean = ops.int4_linear(x, w, norm_weight=n, eps=1e-6)
        spoiled = x.clone()
        spoiled[1] = float("nan")
        spoiled[rows - 1, 7] = float("inf") if rows > 2 else float("nan")
        got = ops.int4_linear(spoiled, w, norm_weight=n, eps=1e-6)
        keep = [r for r in range(rows) if r not in (1, rows - 1)]
        assert torch.equal(got[keep], clean[keep])
        assert not torch.isfinite(got[1]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,group", [(1, 32, 32), (17, 192, 64), (100, 2560, 128), (16, 96, 32)])
def test_int4_dequantize(device, rows, k, group, dtype):
    say("int4_dequantize", rows, k, group, dtype)
    parts = _weight(rows, k, group, dtype, seed=rows + k)
    got = ops.int4_dequantize(_packed(*parts, device))
    # scale (8 or 11 bits) times an integer of at most 4: exact in fp32, one rounding
    assert torch.equal(got.cpu(), oracle.int4_matrix(*parts).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_quantize(device, group, dtype):
    """Every weight within half a step of its group's 16 values, groups of one sign and of
    zeros among them."""
    say("int4_quantize", group, dtype)
    g = torch.Generator().manual_seed(group)
    w = torch.randn(33, 384, generator=g)
    w[3, :group] = 0
    w[4, :group] = 2 + torch.rand(group, generator=g)
    w[5, :group] = -7.5
    w = w.to(dtype)
    q = ops.int4_quantize(w.to(device), group)
    assert (q.rows, q.k, q.group) == (33, 384, group)
    back = ops.int4_dequantize(q).cpu().double()
    scales = (q.steps & 0xffff).to(torch.int16).view(dtype).permute(1, 3, 0, 2).reshape(-1, 48)
    step = scales.cpu().double()[:, :33].t().repeat_interleave(group, 1)[:, :384]
    # half a step; the scale's own rounding (half an eps of 15 steps) may push an end past the
    # last value; and the result's rounding
    most = step * (0.5 + 15 * torch.finfo(dtype).eps) + torch.finfo(dtype).eps / 2 * w.double().abs()
    assert ((back - w.double()).abs() <= most).all()
    assert (back[3, :group] == 0).all()


def test_int4_in_two_graphs(device):
    """Captured into two graphs that share their memory, one with normalised rows that go through
    a workspace, replayed in turn with new inputs and eager calls between."""
    say("int4 graphs")
    parts = _weight(64, 1024, 128, torch.bfloat16, seed=9)
    w = _packed(*parts, device)
    x = torch.randn(40, 1024, device=device).to(torch.bfloat16)
    norm = torch.ones(1024, device=device)
    ops.int4_linear(x, w, norm_weight=norm, eps=1e-6)
    graphs, outs = [], []
    for rows in (5, 40, 33):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append((ops.int4_linear(x[:rows], w, norm_weight=norm, eps=1e-6), rows))
        graphs.append(graph)
    for seed in range(3):
        x.copy_(torch.randn(40, 1024, generator=torch.Generator().manual_seed(seed)))
        for graph, (got, rows) in zip(graphs, outs):
            graph.replay()
            assert torch.equal(got, ops.int4_linear(x[:rows], w, norm_weight=norm, eps=1e-6))


def test_int4_of_no_rows_and_on_a_side_stream(device):
    w = _packed(*_weight(48, 128, 128, torch.bfloat16, seed=2), device)
    assert ops.int4_linear(torch.empty(0, 128, dtype=torch.bfloat16, device=device), w).shape == (0, 48)
    x = torch.randn(2, 3, 128, device=device).to(torch.bfloat16)
    want = ops.int4_linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.int4_linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert want.shape == (2, 3, 48) and torch.equal(got, want)


def test_int4_refusals(device):
    parts = _weight(32, 256, 64, torch.bfloat16, seed=1)
    w = _packed(*parts, device)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=device)
    bad = [
        lambda: ops.int4_linear(torch.zeros(65, 256, dtype=torch.bfloat16, device=device), w),
        lambda: ops.int4_linear(x.half(), w),
        lambda: ops.int4_linear(x[:, :128].contiguous(), w),
        lambda: ops.int4_linear(x.t().contiguous().t(), w),
        lambda: ops.int4_linear(torch.zeros(1025, dtype=torch.bfloat16, device=device)[1:].view(4, 256), w),
        lambda: ops.int4_linear(x, w, residual=torch.zeros(4, 31, dtype=torch.bfloat16, device=device)),
        lambda: ops.int4_linear(x, w, residual=torch.zeros(4, 16, dtype=torch.bfloat16, device=device), swiglu=True),
        lambda: ops.int4_linear(x, w, norm_weight=torch.ones(255, device=device)),
        lambda: ops.int4_linear(x, w, norm_weight=torch.ones(256, device=device), eps=-1.0),
        lambda: ops.int4_linear(x, w._replace(packed=w.packed[:1])),
        lambda: ops.int4_linear(x, w._replace(steps=w.steps.float())),
        lambda: ops.int4_linear(x, w._replace(steps=w.steps.cpu())),
        lambda: ops.int4_linear(x, w._replace(dtype=torch.float32)),
        lambda: ops.int4_dequantize(w._replace(rows=64)),
        lambda: ops.int4_pack(parts[0].to(device), parts[1].to(device), parts[2].to(device) + 16),
        lambda: ops.int4_quantize(torch.full((16, 128), float("nan"), dtype=torch.bfloat16, device=device)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(i)
    with pytest.raises(RuntimeError):
        ops.int4_linear(x.cpu(), w)
