"""Attention over the 8-bit cache where single roundings show (weights that differ by half an fp16 step,
queries of very different sizes side by side, scores past fp32's small steps), and plans of other runs."""

from __future__ import annotations

import math

import pytest
import torch

from helios_amd import _capi, ops
from oracle import kv8 as oracle
from tests.gpu_cases import say
from tests.test_gpu_kv8 import CODES, DTYPES, HALF, _attend, _pool, _u8

pytestmark = pytest.mark.gpu


def _close(got, q, cache, table, cu, used, window, scale=None):
    """One rounding of the output, whatever the rows' kind and type: weights within 2^-22 of themselves
    (two fp16, each off by half a step, 2^-11; 2^-20 allowed), of scores whose fp32 sums of d products
    and exponents are off by e, in the quotient's numerator and denominator; and 2^-31 of the largest
    weight for each key, twice what fp16 loses below its smallest step."""
    d = q.shape[2]
    keys, vals = oracle.values(cache.keys, cache.key_scales), oracle.values(cache.values, cache.value_scales)
    want, mag, reach, peak = oracle.attention(q, keys, vals, table, cu, used, window, scale or d ** -0.5)
    e = (d / 2 + 16) * 2.0 ** -24 * reach + 2.0 ** -18
    tol = HALF[q.dtype] * want.abs() + (2.0 ** -20 + 2 * e) * mag + int(used.max()) * 2.0 ** -31 * peak + 2.0 ** -25
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), (float((off / tol).max()), bad.nonzero()[:5].tolist())


def _lengths(seqs):
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32)
    return cu, torch.tensor([c + n for c, n in seqs], dtype=torch.int32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("rows", [1, 3, 50])
def test_weights_half_a_step_apart(device, rows, code, dtype):
    """Values that cancel but for weights of 1 and 2043.5 / 2048, which 11 bits take to a neighbour: 2^-12
    of a value of 100, an eighth of what is left."""
    say("kv8 weights half a step apart", rows, code, dtype)
    n, d = 200 + rows, 64
    cache, table = _pool([n], 256, 1, d, code, seed=1, stale=False)
    _u8(cache.keys).zero_()
    cache.keys[:, :, 0, 0] = torch.ones((), dtype=code)
    cache.key_scales.fill_(0.0)
    cache.key_scales[:, :, 1::2] = 8 * math.log(2043.5 / 2048)
    top = torch.full((), 100.0 if code == torch.int8 else 104.0).to(code)
    _u8(cache.values)[:, ::2] = _u8(top)
    _u8(cache.values)[:, 1::2] = _u8((-top.float()).to(code))
    cache.value_scales.fill_(1.0)
    q = torch.zeros(rows, 2, d)
    q[..., 0] = 1.0
    q = q.to(dtype)
    cu, used = _lengths([(200, rows)])
    _, got = _attend(device, q, cache, table, cu, used, rows, n, (-1, -1), scale=1 / 8)
    _close(got, q, cache, table, cu, used, (-1, -1), scale=1 / 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
def test_rows_of_every_kind_are_rounded_once(device, code, dtype):
    """Decode rows, drafted ones and chunks of one tick, with windows and without."""
    say("kv8 rounded once", code, dtype)
    seqs = [(900, 1), (300, 70), (0, 129), (77, 4), (500, 16)]
    cu, used = _lengths(seqs)
    cache, table = _pool([c + n for c, n in seqs], 64, 2, 128, code, seed=11)
    q = torch.randn(int(cu[-1]), 8, 128, generator=torch.Generator().manual_seed(11)).to(dtype)
    for window in ((-1, 0), (150, 0)):
        _, got = _attend(device, q, cache, table, cu, used, 129, int(used.max()), window)
        _close(got, q, cache, table, cu, used, window)


@pytest.mark.parametrize("rows", [1, 3, 40, 130])
@pytest.mark.parametrize("power", [20, 32, 40, 60, 110])
def test_queries_far_apart(device, power, rows):
    """Rows and heads, neighbours of one sequence, up to 2^110 apart: the small ones get their own answer
    (not the values' mean), the large ones the value of their best key."""
    say("kv8 queries far apart", power, rows)
    cu, used = _lengths([(300 - rows, rows), (300 - rows, rows)])
    cache, table = _pool([300, 300], 64, 2, 64, torch.float8_e4m3fn, seed=21)
    g = torch.Generator().manual_seed(power + rows)
    q = 3 * torch.randn(2 * rows, 8, 64, generator=g)
    large = (torch.arange(2 * rows)[:, None] + torch.arange(8)) % 3 == 0
    q = torch.where(large[..., None], q * 2.0 ** power, q).to(torch.bfloat16)
    _, got = _attend(device, q, cache, table, cu, used, rows, 300, (-1, 0))
    # (A large row's scores are off by more than 1: its bound holds for whatever its keys weigh.)
    _close(got, q, cache, table, cu, used, (-1, 0))
    assert torch.isfinite(got).all()
    # Each row by itself has the same answer.
    cu, used = _lengths([(299, 1)])
    _, one = _attend(device, q[rows - 1:rows], cache, table[:1], cu, used, 1, 300, (-1, 0))
    _close(one, q[rows - 1:rows], cache, table[:1], cu, used, (-1, 0))

@pytest.mark.parametrize("rows", [1, 40])
def test_small_half_precision_queries_beside_large_ones(device, rows):
    """The whole range of fp16 in one block, subnormal elements among them, whose keys are large."""
    say("kv8 fp16 queries far apart", rows)
    cu, used = _lengths([(300 - rows, rows)])
    cache, table = _pool([300], 64, 1, 64, torch.int8, seed=22, stale=False)
    cache.key_scales.mul_(2.0 ** 12)
    q = torch.randn(rows, 8, 64, generator=torch.Generator().manual_seed(22))
    q = torch.where((torch.arange(8) % 2 == 0)[:, None], q * 2.0 ** 12, q * 2.0 ** -13).to(torch.float16)
    _, got = _attend(device, q, cache, table, cu, used, rows, 300, (-1, 0))
    _close(got, q, cache, table, cu, used, (-1, 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_scores_past_the_steps_of_fp32(device, rows, dtype):
    """Scores up to 2^40, where fp32's own steps reach those of the weights' reference: equal keys share a
    row, all others are far below it. Scores of equal keys are equal, so the mean of their values is off
    by the weights' and the output's rounding alone."""
    say("kv8 large scores", rows, dtype)
    d, n = 64, 200 + rows
    cache, table = _pool([n], 64, 1, d, torch.int8, seed=23, stale=False)
    _u8(cache.keys).zero_()
    token = torch.zeros(n, dtype=torch.int8)
    token[:] = 126
    token[::3] = 127
    for j in range(-(-n // 64)):
        part = token[64 * j:64 * j + 64]
        cache.keys[table[0, j], :part.shape[0], 0, 0] = part
    cache.value_scales.fill_(1.0)
    vals = cache.values[table[0].long()].flatten(0, 1)[:n, 0].double()
    cu, used = _lengths([(200, rows)])
    q = torch.zeros(rows, 8, d)
    q[..., 0] = 1 + torch.arange(8) / 8  # exact in both types, scores at any part of fp32's steps
    q = q.to(dtype)
    want = torch.stack([vals[:200 + r + 1:3].mean(dim=0) for r in range(rows)])[:, None]
    mag = torch.stack([vals[:200 + r + 1:3].abs().mean(dim=0) for r in range(rows)])[:, None]
    for power in range(9, 34):  # scores of 127 * q * 2^power, in powers of two 1.44 times as much
        cache.key_scales.fill_(2.0 ** power * (1 + 2.0 ** -9))
        _, got = _attend(device, q, cache, table, cu, used, rows, n, (-1, 0), scale=1.0)
        off = (got.double().cpu() - want).abs()
        assert (off <= HALF[dtype] * want.abs() + 2.0 ** -20 * mag).all(), (power, float(off.max()))


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("windows,widths", [(((40, 0), (-1, 0)), (5, 5)), (((-1, 0), (40, 0)), (5, 5)), (((-1, 0), (-1, 7)), (5, 5)),
                                            (((-1, 0), (-1, 0)), (5, 4)), (((-1, 0), (-1, 0)), (4, 5))])
def test_plan_of_other_windows_or_tables_is_flagged(device, windows, widths, new):
    """A plan's key ranges follow its windows and its table's width: a run with others writes nothing and
    says so."""
    say("kv8 plan of others", windows, widths, new)
    cu, used = _lengths([(250 - new, new), (180, 1)])
    cache, table = _pool([250, 181], 64, 1, 64, torch.int8, seed=24)
    on = ops.Kv8Cache(*(t.to(device) for t in cache))
    wide = torch.zeros(2, 5, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = table.to(device)
    q = torch.randn(new + 1, 4, 64, device=device).to(torch.bfloat16)
    plan = ops.Kv8AttnPlan(cu.to(device), used.to(device), total_q=new + 1, max_q=new, max_k=250, n_q_heads=4, n_kv_heads=1,
                           head_dim=64, page_size=64, window=windows[0], block_table_width=widths[0])
    good = plan.run(q, on, wide)
    assert plan.error_word() == 0 and torch.isfinite(good).all()
    plan.window, plan.width = windows[1], widths[1]
    out = torch.full_like(q, 3.0)
    plan.run(q, on, wide, out=out)
    assert plan.error_word() == _capi.HX_WERR_PLAN_MISMATCH and (out == 3).all()


@pytest.mark.parametrize("power", [-78, -40, 60, 110])
@pytest.mark.parametrize("rows", [1, 40])
def test_values_of_every_size(device, rows, power):
    """Values 2^-78 to 2^110 of the usual, at 40000 keys: the outputs are as much smaller or larger. (The
    scales' logarithms, up to 2^7, are off by 2^-17 with the scores' last places: within twice e.)"""
    say("kv8 values of every size", rows, power)
    n = 40000
    cu, used = _lengths([(n - rows, rows)])
    cache, table = _pool([n], 64, 1, 16, torch.float8_e4m3fn, seed=25, stale=False)
    q = 2 * torch.randn(rows, 4, 16, generator=torch.Generator().manual_seed(25)).to(torch.bfloat16)
    far = cache._replace(value_scales=cache.value_scales * 2.0 ** power)
    _, got = _attend(device, q, far, table, cu, used, rows, n, (-1, 0))
    _close(got.double() * 2.0 ** -power, q, cache, table, cu, used, (-1, 0))


@pytest.mark.parametrize("rows", [1, 40])
def test_rows_of_zeros_beside_large_values(device, rows):
    """Values stored as zeros (a scale of 2^-100) count in the weights' sum beside values of 2^20."""
    say("kv8 zeros beside large values", rows)
    n = 3000
    cu, used = _lengths([(n - rows, rows)])
    cache, table = _pool([n], 64, 1, 64, torch.int8, seed=26, stale=False)
    cache.value_scales.mul_(2.0 ** 20)
    _u8(cache.values)[:, ::3] = 0
    cache.value_scales[:, :, ::3] = 2.0 ** -100
    q = torch.randn(rows, 4, 64, generator=torch.Generator().manual_seed(26)).to(torch.bfloat16)
    _, got = _attend(device, q, cache, table, cu, used, rows, n, (-1, 0))
    _close(got, q, cache, table, cu, used, (-1, 0))
