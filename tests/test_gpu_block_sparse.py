"""Attention over selected blocks of the paged cache against 64 bits: key bounds, selection,
the attention, and the three in turn over a growing cache."""

from __future__ import annotations

import math

import pytest
import torch

from helios_amd import ops
from oracle import decode_ops as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
NAN, INF = float("nan"), float("inf")


def _pools(ends, heads, d, dtype, seed, page=256, spare=2):
    """K and V pools and a page table (CPU) for sequences of these lengths; pages nobody holds
    and everything behind a last key are NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in ends]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.zeros(len(ends), max(need + [1]) + 1, dtype=torch.int32)
    k = torch.full((pages, page, heads, d), NAN)
    v = torch.full((pages, page, heads, d), NAN)
    at = 0
    for b, n in enumerate(ends):
        for j in range(need[b]):
            p = order[at]
            at += 1
            table[b, j] = p
            fill = min(page, n - j * page)
            k[p, :fill] = torch.randn(fill, heads, d, generator=g) + torch.randn(heads, d, generator=g)
            v[p, :fill] = torch.randn(fill, heads, d, generator=g)
    return k.to(dtype), v.to(dtype), table


def _same(got, want):
    """Equal values (0 and -0 alike), NaN where the other has one."""
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    keep = ~torch.isnan(want)
    assert torch.equal(got[keep], want[keep])


# ------------------------------------------------------------------------- key bounds
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,d,block,page,ticks", [
    (1, 8, 16, 256, [(0, 1), (15, 1), (16, 1), (255, 2)]),
    (8, 128, 64, 256, [(63, 1), (64, 1), (100, 400), (0, 257), (511, 1), (5, 0)]),
    (2, 96, 256, 256, [(0, 300), (255, 1), (256, 1)]),
    (3, 256, 128, 512, [(500, 30), (0, 1030)]),
    (5, 40, 32, 96, [(90, 20), (31, 2)])])
def test_block_bounds(device, heads, d, block, page, ticks, dtype):
    say("block bounds", heads, d, block, dtype)
    cached, new = [c for c, _ in ticks], [n for _, n in ticks]
    ends = [c + n for c, n in ticks]
    k, _, table = _pools(ends, heads, d, dtype, seed=heads * d + block, page=page)
    k[k.isnan()] = 99.0  # stale keys behind the last one
    bounds = torch.randn(k.shape[0], page // block, heads, 2, d).to(dtype)
    want = oracle.block_bounds(k, bounds, table, cached, new)
    on = bounds.to(device)
    cu = torch.tensor([0] + new).cumsum(0).to(torch.int32).to(device)
    used = torch.tensor(ends, dtype=torch.int32, device=device)
    for max_q in (max(new), 1):  # a grid for fewer tokens than there are gives the same
        on.copy_(bounds)
        ops.kv_block_bounds(k.to(device), on, table.to(device), cu, used, max_q=max_q)
        _same(on, want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_block_bounds_special_keys(device, dtype):
    """Infinities are bounds, a NaN makes both NaN in its dim and head alone; a page outside the
    pool or past the table leaves everything as it was."""
    say("block bounds special", dtype)
    k, _, table = _pools([70, 300], 2, 16, dtype, seed=4)
    p = int(table[0, 0])
    k[p, 3, 0, 5], k[p, 9, 0, 5] = INF, -INF
    k[p, 66, 1, 7] = NAN
    k[p, 5, 1, 2] = -NAN
    bounds = torch.zeros(k.shape[0], 4, 2, 2, 16).to(dtype)
    want = oracle.block_bounds(k, bounds, table, [0, 0], [70, 300])
    on, table = bounds.to(device), table.to(device)
    cu = torch.tensor([0, 70, 370], dtype=torch.int32, device=device)
    used = torch.tensor([70, 300], dtype=torch.int32, device=device)
    ops.kv_block_bounds(k.to(device), on, table, cu, used, max_q=300)
    _same(on, want)
    on.fill_(3)
    for bad in (-1, k.shape[0], 2 ** 31 - 1):
        ops.kv_block_bounds(k.to(device), on, torch.full_like(table, bad), cu, used, max_q=300)
    assert (on == 3).all()
    # more keys than the table has pages for
    ops.kv_block_bounds(k.to(device), on, table[:, :1], torch.tensor([0, 0, 1], dtype=torch.int32, device=device),
                        torch.tensor([0, 300], dtype=torch.int32, device=device), max_q=1)
    assert (on == 3).all()


# -------------------------------------------------------------------------- selection
def _bounds(pages, per_page, heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    mid, half = torch.randn(2, pages, per_page, heads, d, generator=g)
    return torch.stack((mid - half.abs(), mid + half.abs()), dim=3).to(dtype)


def _select_ref(q, bounds, table, keys, seqs, rows, budget, sink, recent, block):
    heads = bounds.shape[2]
    group = q.shape[1] // heads
    out = []
    for i, n in enumerate(keys):
        count = -(-n // block)
        out.append([oracle.select(
            oracle.block_scores(q[rows[i]], bounds, table[seqs[i]], count, h, group) if count > budget else None,
            count, budget, sink, recent) for h in range(heads)])
    return torch.tensor(out, dtype=torch.int32).view(len(keys), heads, budget)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,block,keys,budget,sink,recent", [
    (2, 1, 8, 16, [0, 1, 16, 17, 500, 512], 3, 0, 1),
    (8, 2, 128, 64, [4000, 700, 65, 4096, 2111], 6, 1, 2),
    (12, 4, 96, 64, [1500, 1501], 10, 2, 1),
    (10, 1, 256, 256, [5000], 2, 1, 1),
    (4, 4, 24, 16, [3000, 2999], 64, 0, 2),
    (4, 2, 64, 32, [700, 90], 40, 3, 3)])
def test_select_blocks(device, hq, heads, d, block, keys, budget, sink, recent, dtype):
    say("select blocks", hq, heads, d, block, dtype)
    width = -(-max(keys) // 256) + 1
    g = torch.Generator().manual_seed(d + block)
    pages = len(keys) * width
    table = torch.randperm(pages, generator=g).view(len(keys), width).to(torch.int32)
    bounds = _bounds(pages, 256 // block, heads, d, dtype, seed=d)
    q = torch.randn(len(keys), hq, d, generator=g).to(dtype)
    at = list(range(len(keys)))
    want = _select_ref(q, bounds, table, keys, at, at, budget, sink, recent, block)
    args = (bounds.to(device), table.to(device))
    got = ops.select_blocks(q.to(device), *args, torch.tensor(keys, dtype=torch.int32, device=device), budget,
                            block_size=block, sink=sink, recent=recent)
    assert torch.equal(got.cpu(), want)
    # The same rows named in another order, of queries with other strides.
    rows, seqs = at[::-1], at[::-1]
    wide = torch.zeros(len(keys), hq + 1, d + 8, dtype=dtype)
    wide[:, :hq, :d] = q
    again = ops.select_blocks(
        wide.to(device)[:, :hq, :d], *args, torch.tensor(keys[::-1], dtype=torch.int32, device=device), budget,
        block_size=block, sink=sink, recent=recent, rows=torch.tensor(rows, device=device),
        row_seq=torch.tensor(seqs, dtype=torch.int32, device=device))
    assert torch.equal(again.cpu(), want.flip(0))


@pytest.mark.parametrize("blocks", [900, 2000, 3000, 5000, 16384])
def test_select_blocks_of_long_sequences(device, blocks):
    """As many blocks as there may be, with scores that differ in few values: ties go to the
    earlier block."""
    say("select long", blocks)
    per_page, d = 16, 8
    width = -(-blocks // per_page)
    g = torch.Generator().manual_seed(blocks)
    bounds = torch.randint(-2, 3, (width, per_page, 1, 1, d), generator=g).repeat(1, 1, 1, 2, 1).to(torch.bfloat16)
    q = torch.tensor([[[1.0, 2, 0, 0, -1, 0, 0, 1]]]).to(torch.bfloat16)
    table = torch.randperm(width, generator=g).view(1, width).to(torch.int32)
    scores = (bounds[table[0].long()].reshape(-1, 2, d)[:blocks, 0].double() * q[0, 0].double()).sum(1)
    for budget in (1, 7, 700, blocks - 1, blocks, blocks + 3):
        want = oracle.select(scores, blocks, budget, 0, 1)
        got = ops.select_blocks(q.to(device), bounds.to(device), table.to(device),
                                torch.tensor([blocks * 16 - 5], dtype=torch.int32, device=device), budget,
                                block_size=16, sink=0, recent=1)
        assert got[0, 0].tolist() == want


@pytest.mark.parametrize("dtype", DTYPES)
def test_select_blocks_special_scores(device, dtype):
    """Infinite and NaN bounds, equal scores, pages outside the pool."""
    say("select special", dtype)
    bounds = _bounds(8, 4, 1, 16, dtype, seed=3)
    q = torch.randn(1, 2, 16).to(dtype)
    table = torch.arange(8, dtype=torch.int32).view(1, 8)
    bounds[1, 2, 0, :, 4] = NAN
    bounds[3, 0, 0, 1] = INF
    bounds[3, 0, 0, 0] = 0
    bounds[4, 1, 0, 0] = -INF
    bounds[4, 1, 0, 1] = -INF
    bounds[5] = bounds[2]
    table[0, 6] = 99
    for budget in (3, 5, 9, 20, 31):
        want = _select_ref(q, bounds, table, [8 * 256], [0], [0], budget, 1, 1, 64)
        got = ops.select_blocks(q.to(device), bounds.to(device), table.to(device),
                                torch.tensor([8 * 256], dtype=torch.int32, device=device), budget, block_size=64,
                                sink=1, recent=1)
        assert torch.equal(got.cpu(), want), budget


def test_select_blocks_of_rows_that_are_not_there(device):
    """Rows and sequences outside the tensors: -1. Negative counts: no keys. Counts past the
    table: the table's."""
    say("select absent")
    bounds = _bounds(4, 4, 2, 16, torch.bfloat16, seed=1).to(device)
    q = torch.randn(2, 4, 16, device=device).to(torch.bfloat16)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=device)
    i32 = dict(dtype=torch.int32, device=device)
    got = ops.select_blocks(q, bounds, table, torch.tensor([512, 512, 512, 512, -3, 9999], **i32), 12, block_size=64,
                            rows=torch.tensor([0, 2, -1, 0, 1, 1], device=device),
                            row_seq=torch.tensor([2, 0, 0, -1, 1, 1], **i32)).cpu()
    assert (got[:5] == -1).all()
    assert got[5, 0].tolist() == list(range(8)) + [-1] * 4


# -------------------------------------------------------------------------- attention
def _tolerance(q, v, ref, dtype, scale):
    """The output's half step; weights of 16 bits or more (2^-16 of the values they weigh, which
    are at most max |v|); fp32 scores, |scale q k| up to 60 to 2^-20 of itself through exp, and
    sums of up to 2^13 keys in parts: 2^-14 of max |v| covers them."""
    return torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -14 * v[v.isfinite()].double().abs().max() \
        + torch.finfo(dtype).tiny


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,heads,d,block,ends,budget", [
    (2, 1, 8, 16, [1, 16, 17, 300], 4),
    (8, 2, 128, 64, [700, 64, 65, 1023, 1], 9),
    (12, 4, 96, 64, [900, 333], 20),
    (16, 1, 256, 256, [1000, 100], 3),
    (4, 4, 64, 32, [500, 31], 12),
    (20, 2, 128, 16, [450], 70),
    (3, 1, 136, 128, [600, 129], 2)])
def test_block_sparse_attn(device, hq, heads, d, block, ends, budget, dtype):
    say("sparse attention", hq, heads, d, block, dtype)
    k, v, table = _pools(ends, heads, d, dtype, seed=d + block)
    g = torch.Generator().manual_seed(budget)
    q = torch.randn(len(ends), hq, d, generator=g).to(dtype)
    blocks = torch.full((len(ends), heads, budget), -1, dtype=torch.int32)
    for i, n in enumerate(ends):
        for h in range(heads):
            count = -(-n // block)
            pick = torch.randperm(count, generator=g)[:budget].sort().values
            blocks[i, h, :len(pick)] = pick.to(torch.int32)
    for scale in (None, 0.7, -0.2):
        s = d ** -0.5 if scale is None else scale
        ref = oracle.sparse_attention(q, k, v, blocks, table, ends, range(len(ends)), block, s)
        got = ops.block_sparse_attn(q.to(device), k.to(device), v.to(device), blocks.to(device), table.to(device),
                                    torch.tensor(ends, dtype=torch.int32, device=device), block_size=block, scale=scale)
        assert ((got.double().cpu() - ref).abs() <= _tolerance(q, v, ref, dtype, s)).all()


@pytest.mark.parametrize("d", [64, 128])
def test_block_sparse_attn_many_rows(device, d):
    """Enough rows and heads that a list is not split, and one so long that it is cut for its
    length."""
    say("sparse many rows", d)
    block, budget, n = 64, 24, 40
    ends = [64 * 24 + 7 * i for i in range(n)]
    k, v, table = _pools(ends, 8, d, torch.bfloat16, seed=d)
    g = torch.Generator().manual_seed(d)
    q = (2 * torch.randn(n, 16, d, generator=g)).to(torch.bfloat16)
    blocks = torch.stack([torch.stack([torch.randperm(-(-e // block), generator=g)[:budget].sort().values
                                       for _ in range(8)]) for e in ends]).to(torch.int32)
    ref = oracle.sparse_attention(q, k, v, blocks, table, ends, range(n), block, d ** -0.5)
    got = ops.block_sparse_attn(q.to(device), k.to(device), v.to(device), blocks.to(device), table.to(device),
                                torch.tensor(ends, dtype=torch.int32, device=device), block_size=block)
    assert ((got.double().cpu() - ref).abs() <= _tolerance(q, v, ref, torch.bfloat16, d ** -0.5)).all()


@pytest.mark.parametrize("d", [64, 160])
def test_block_sparse_attn_many_splits(device, d):
    """One row's list in more parts than a wave has lanes (88 of 128 keys: sums in 216 steps, 2^-16
    of max |v|)."""
    say("sparse many splits", d)
    k, v, table = _pools([11190], 1, d, torch.bfloat16, seed=d)
    g = torch.Generator().manual_seed(d)
    q = torch.randn(1, 3, d, generator=g).to(torch.bfloat16)
    blocks = torch.arange(700, dtype=torch.int32).view(1, 1, 700)
    ref = oracle.sparse_attention(q, k, v, blocks, table, [11190], [0], 16, d ** -0.5)
    got = ops.block_sparse_attn(q.to(device), k.to(device), v.to(device), blocks.to(device), table.to(device),
                                torch.tensor([11190], dtype=torch.int32, device=device), block_size=16)
    assert ((got.double().cpu() - ref).abs() <= _tolerance(q, v, ref, torch.bfloat16, d ** -0.5)).all()


def test_block_sparse_attn_lists(device):
    """Lists in any order, with repeats (they count twice), ids past the keys, pages outside the
    pool, gaps of -1 in the middle, and nothing at all."""
    say("sparse lists")
    k, v, table = _pools([600, 200, 70], 2, 32, torch.bfloat16, seed=9)
    table[1, 0] = 77  # not in the pool
    q = torch.randn(3, 4, 32).to(torch.bfloat16)
    blocks = torch.tensor([[[9, 3, 3, -1, 0, 50], [8, -1, -1, -1, -1, 2]],
                           [[0, 1, 2, 3, -1, -1], [3, 2, 1, 0, 9, 9]],
                           [[-1] * 6, [1, 1, 2, 2 ** 31 - 1, -2 ** 31, -7]]], dtype=torch.int32)
    args = [t.to(device) for t in (q, k, v, blocks, table)]
    got = ops.block_sparse_attn(*args, torch.tensor([600, 200, 70], dtype=torch.int32, device=device), block_size=64)
    ref = oracle.sparse_attention(q, k, v, blocks, table, [600, 200, 70], [0, 1, 2], 64, 32 ** -0.5)
    assert (ref[1] == 0).all() and (ref[2, :2] == 0).all()
    assert ((got.double().cpu() - ref).abs() <= _tolerance(q, v, ref, torch.bfloat16, 1)).all()


def test_block_sparse_attn_row_maps(device):
    """Drafted rows of one sequence, rows written where they are named and nowhere else, queries
    and outputs inside wider tensors."""
    say("sparse rows")
    k, v, table = _pools([300, 700], 2, 64, torch.float16, seed=5)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(6, 4, 64, generator=g).half()
    rows, seqs, keys = [4, 0, 3], [1, 0, 1], [699, 300, 0]
    blocks = torch.arange(11, dtype=torch.int32).view(1, 1, 11).repeat(3, 2, 1)
    ref = oracle.sparse_attention(q[rows], k, v, blocks, table, keys, seqs, 64, 0.125)
    wide = torch.zeros(6, 5, 72, dtype=torch.float16, device=device)
    wide[:, :4, :64] = q.to(device)
    out = torch.full((6, 7, 66), 5.0, dtype=torch.float16, device=device)
    kw = dict(block_size=64, rows=torch.tensor(rows, device=device),
              row_seq=torch.tensor(seqs, dtype=torch.int32, device=device))
    args = (k.to(device), v.to(device), blocks.to(device), table.to(device),
            torch.tensor(keys, dtype=torch.int32, device=device))
    got = ops.block_sparse_attn(wide[:, :4, :64], *args, out=out[:, 1:5, 2:], **kw)
    assert ((got[rows].double().cpu() - ref).abs() <= _tolerance(q, v, ref, torch.float16, 1)).all()
    assert (got[3] == 0).all()
    mask = torch.ones_like(out, dtype=torch.bool)
    mask[rows, 1:5, 2:] = False
    assert (out[mask] == 5).all()
    fresh = ops.block_sparse_attn(q.to(device), *args, **kw)
    assert torch.equal(fresh[rows], got[rows]) and (fresh[[1, 2, 5]] == 0).all()
    # A query whose rows are not 16-byte aligned is copied first.
    odd = torch.zeros(6, 4, 65, dtype=torch.float16, device=device)[..., 1:]
    odd.copy_(q)
    assert torch.equal(ops.block_sparse_attn(odd, *args, **kw), fresh)
    # Rows and sequences outside their tensors: nothing written, zeros.
    kw["rows"] = torch.tensor([6, -1, 2], device=device)
    kw["row_seq"] = torch.tensor([0, 0, 2], dtype=torch.int32, device=device)
    out.fill_(5)
    ops.block_sparse_attn(q.to(device), *args, out=out[:, 1:5, 2:], **kw)
    assert (out[2, 1:5, 2:] == 0).all() and (out[[0, 1, 3, 4, 5]] == 5).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_block_sparse_attn_special_values(device, dtype):
    """What a row does not see never reaches it; what it sees does. A dominant key, scores of
    any size, and the lowest values."""
    say("sparse special", dtype)
    big = 200.0 if dtype == torch.float16 else 1e4
    k, v, table = _pools([256] * 4, 1, 64, dtype, seed=8)
    k, v = k.clone(), v.clone()
    q = torch.randn(4, 2, 64).to(dtype)
    blocks = torch.tensor([[[0, 2]]] * 4, dtype=torch.int32)
    p = table[:, 0].tolist()
    k[p[0], 64:128] = NAN       # block 1: not listed
    v[p[0], 192:] = INF         # block 3: not listed
    v[p[1], 130] = INF          # seen
    k[p[2], 3, 0] = big * q[2, 0].sign()  # dominates head 0
    v[p[3], :] = torch.finfo(dtype).min
    args = [t.to(device) for t in (q, k, v, blocks, table)]
    got = ops.block_sparse_attn(*args, torch.tensor([256] * 4, dtype=torch.int32, device=device),
                                block_size=64).double().cpu()
    ref = oracle.sparse_attention(q, k, v, blocks, table, [256] * 4, range(4), 64, 0.125)
    tol = _tolerance(q, v[p[0], :64], ref, dtype, 1)
    assert ((got[0] - ref[0]).abs() <= tol[0]).all()
    assert not torch.isfinite(got[1]).any()
    assert ((got[2] - ref[2]).abs() <= tol[2]).all()
    # weights sum to 1 within 2^-20, and 1 step of the type
    assert ((got[3] - ref[3]).abs() <= torch.finfo(dtype).eps * ref[3].abs()).all()


def test_block_sparse_attn_equals_dense(device):
    """All blocks of every sequence: the framework's own attention over all keys."""
    say("sparse equals dense")
    ends = [900, 256, 33, 1500]
    k, v, table = _pools(ends, 8, 128, torch.bfloat16, seed=21)
    k, v, table = k.nan_to_num(0).to(device), v.nan_to_num(0).to(device), table.to(device)
    q = torch.randn(4, 32, 128, device=device).to(torch.bfloat16)
    used = torch.tensor(ends, dtype=torch.int32, device=device)
    blocks = torch.arange(24, dtype=torch.int32, device=device).view(1, 1, 24).repeat(4, 8, 1)
    got = ops.block_sparse_attn(q, k, v, blocks, table, used, block_size=64)
    cu = torch.arange(5, dtype=torch.int32, device=device)
    want = ops.varlen_attn(q, k, v, cu, None, 1, 1500, window_size=(-1, 0), enable_gqa=True, seqused_k=used,
                           block_table=table)
    # two kernels, each within its rounding and the other's 16-bit partials
    assert (got.float() - want.float()).abs().max() <= 2e-2
    assert (got.float() - want.float()).abs().mean() <= 2e-3


def test_pool_rows_past_32_bits(device):
    """Pages whose elements lie beyond 2^31 from the pool's start."""
    say("sparse long pool")
    pages = 2 ** 31 // (256 * 8 * 128) + 3
    k = torch.zeros(pages, 256, 8, 128, dtype=torch.bfloat16, device=device)
    v = torch.zeros_like(k)
    bounds = torch.zeros(pages, 4, 8, 2, 128, dtype=torch.bfloat16, device=device)
    table = torch.tensor([[pages - 1, 0, pages - 2]], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    for p in table[0].tolist():
        k[p] = torch.randn(256, 8, 128, generator=g).to(torch.bfloat16)
        v[p] = torch.randn(256, 8, 128, generator=g).to(torch.bfloat16)
    q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16)
    used = torch.tensor([600], dtype=torch.int32, device=device)
    cu = torch.tensor([0, 600], dtype=torch.int32, device=device)
    ops.kv_block_bounds(k, bounds, table.to(device), cu, used, max_q=600)
    blocks = ops.select_blocks(q.to(device), bounds, table.to(device), used, 4, block_size=64)
    got = ops.block_sparse_attn(q.to(device), k, v, blocks, table.to(device), used, block_size=64)
    few = table[0].long()
    small = torch.arange(3, dtype=torch.int32).view(1, 3)
    kc, vc = k[few.to(device)].cpu(), v[few.to(device)].cpu()
    bc = oracle.block_bounds(kc, torch.zeros(3, 4, 8, 2, 128), small, [0], [600]).to(torch.bfloat16)
    want = _select_ref(q, bc, small, [600], [0], [0], 4, 1, 2, 64)
    assert torch.equal(blocks.cpu(), want)
    ref = oracle.sparse_attention(q, kc, vc, want, small, [600], [0], 64, 128 ** -0.5)
    assert ((got.double().cpu() - ref).abs() <= _tolerance(q, vc, ref, torch.bfloat16, 1)).all()


def test_block_sparse_step_in_two_graphs(device):
    """Bounds, selection and attention of a tick captured twice into graphs that share their
    memory, replayed in turn, new keys and eager calls between."""
    say("sparse graphs")
    ends = [1000, 640]
    k, v, table = _pools(ends, 2, 64, torch.bfloat16, seed=6)
    k, v, table = k.nan_to_num(0).to(device), v.nan_to_num(0).to(device), table.to(device)
    bounds = torch.zeros(k.shape[0], 4, 2, 2, 64, dtype=torch.bfloat16, device=device)
    used = torch.tensor(ends, dtype=torch.int32, device=device)
    cu = torch.tensor([0, 1000, 1640], dtype=torch.int32, device=device)
    q = torch.randn(2, 8, 64, device=device).to(torch.bfloat16)

    def step(budget):
        ops.kv_block_bounds(k, bounds, table, cu, used, max_q=1000)
        blocks = ops.select_blocks(q, bounds, table, used, budget, block_size=64)
        return blocks, ops.block_sparse_attn(q, k, v, blocks, table, used, block_size=64)

    step(4)
    graphs, outs = [], []
    for budget in (4, 7):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(step(budget))
        graphs.append(graph)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        k.copy_(torch.randn(k.shape, generator=g))
        q.copy_(torch.randn(q.shape, generator=g))
        for graph, out, budget in zip(graphs, outs, (4, 7)):
            graph.replay()
            want = step(budget)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_block_sparse_refusals(device):
    bf = dict(dtype=torch.bfloat16, device=device)
    i32 = dict(dtype=torch.int32, device=device)
    k = torch.zeros(4, 256, 2, 64, **bf)
    bounds = torch.zeros(4, 4, 2, 2, 64, **bf)
    table, keys = torch.zeros(2, 3, **i32), torch.ones(2, **i32)
    q, blocks = torch.zeros(2, 4, 64, **bf), torch.zeros(2, 2, 5, **i32)
    cu = torch.zeros(3, **i32)
    bad = [
        lambda: ops.kv_block_bounds(k, bounds[:, :3].contiguous(), table, cu, keys, max_q=1),
        lambda: ops.kv_block_bounds(k, bounds.half(), table, cu, keys, max_q=1),
        lambda: ops.kv_block_bounds(k[:, ::2], bounds, table, cu, keys, max_q=1),
        lambda: ops.kv_block_bounds(k, bounds, table, cu[:2], keys, max_q=1),
        lambda: ops.kv_block_bounds(k, bounds, table[:1], cu, keys, max_q=1),
        lambda: ops.kv_block_bounds(k, bounds, table.long(), cu, keys, max_q=1),
        lambda: ops.kv_block_bounds(k, bounds, table, cu, keys, max_q=-1),
        lambda: ops.kv_block_bounds(k.float(), bounds.float(), table, cu, keys, max_q=1),
        lambda: ops.select_blocks(q, bounds, table, keys, 2, block_size=64),
        lambda: ops.select_blocks(q, bounds, table, keys, 5, block_size=64, recent=0),
        lambda: ops.select_blocks(q, bounds, table, keys, 5, block_size=64, sink=-1),
        lambda: ops.select_blocks(q, bounds, table, keys, 5, block_size=48),
        lambda: ops.select_blocks(q[:, :3], bounds, table, keys, 5, block_size=64),
        lambda: ops.select_blocks(q.half(), bounds, table, keys, 5, block_size=64),
        lambda: ops.select_blocks(q, bounds, table, keys[:1], 5, block_size=64),
        lambda: ops.select_blocks(q, bounds, table[:1], keys, 5, block_size=64),
        lambda: ops.select_blocks(q, bounds, torch.zeros(2, 4097, **i32), keys, 5, block_size=64),
        lambda: ops.select_blocks(q, bounds, table, keys, 5, block_size=64, rows=torch.zeros(2, **i32)),
        lambda: ops.select_blocks(q, bounds, table, keys, 5, block_size=64, row_seq=keys.long()),
        lambda: ops.block_sparse_attn(q, k, k[:3], blocks, table, keys, block_size=64),
        lambda: ops.block_sparse_attn(q, k, k.half(), blocks, table, keys, block_size=64),
        lambda: ops.block_sparse_attn(q[:, :3], k, k, blocks, table, keys, block_size=64),
        lambda: ops.block_sparse_attn(q, k, k, blocks[:1], table, keys, block_size=64),
        lambda: ops.block_sparse_attn(q, k, k, blocks.long(), table, keys, block_size=64),
        lambda: ops.block_sparse_attn(q, k, k, blocks, table, keys, block_size=512),
        lambda: ops.block_sparse_attn(q, k, k, blocks, table, keys, block_size=64, out=q[:1]),
        lambda: ops.block_sparse_attn(q, k, k, blocks, table, keys, block_size=64,
                                      rows=torch.zeros(3, dtype=torch.int64, device=device)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(i)
    with pytest.raises(RuntimeError):
        ops.select_blocks(q.cpu(), bounds, table, keys, 5, block_size=64)
    none = torch.zeros(0, **i32)
    assert ops.select_blocks(q[:0], bounds, table, none, 5, block_size=64).shape == (0, 2, 5)
    assert ops.block_sparse_attn(q[:0], k, k, blocks[:0], table, none, block_size=64).shape == (0, 4, 64)
