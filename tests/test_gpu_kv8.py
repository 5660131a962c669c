"""The 8-bit KV cache against its definitions: quantising writes, norms and rotation, reading
back, and attention over it."""

from __future__ import annotations

import math

import pytest
import torch

from helios_amd import _capi, ops
from oracle import kv8 as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]
CODES = [torch.float8_e4m3fn, torch.int8]
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NAN, INF = float("nan"), float("inf")


def _u8(t):
    return t.view(torch.uint8)


def _bits(t):
    return t.contiguous().view(torch.int32)


def _cache(pages, page, heads, d, code, device, fill=0x55):
    """A pool that nothing has been written to: known bytes."""
    codes = torch.full((2, pages, page, heads, d), fill, dtype=torch.uint8, device=device).view(code)
    scales = torch.full((2, pages, heads, page), 3.0, device=device)
    return ops.Kv8Cache(codes[0], codes[1], scales[0], scales[1])


# ------------------------------------------------------------------------------ append
def _expected_append(cache, slots, k, v):
    """CPU copies of the cache after the append."""
    out = [t.cpu().clone() for t in cache]
    page = cache.keys.shape[1]
    for i, x in ((0, k), (1, v)):
        codes, scales = oracle.quantise(x, cache.keys.dtype)
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < cache.keys.shape[0] * page:
                _u8(out[i])[s // page, s % page] = _u8(codes)[t]
                out[2 + i][s // page, :, s % page] = scales[t]
    return out


def _same_cache(cache, want):
    for got, exp in zip(cache, want):
        got = got.cpu()
        if got.dtype == torch.float32:
            assert torch.equal(got.isnan(), exp.isnan())
            assert torch.equal(got.nan_to_num(7.0), exp.nan_to_num(7.0))
        else:
            assert torch.equal(_u8(got), _u8(exp))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads,d,page,tokens", [(8, 128, 256, 70), (4, 64, 256, 300), (1, 16, 64, 1), (3, 96, 320, 33),
                                                 (2, 256, 128, 129), (5, 176, 64, 17)])
def test_append(device, heads, d, page, tokens, code, dtype):
    say("kv8 append", heads, d, page, tokens, code, dtype)
    g = torch.Generator().manual_seed(heads * d + tokens)
    pages = -(-tokens // page) + 2
    cache = _cache(pages, page, heads, d, code, device)
    slots = torch.randperm(pages * page, generator=g)[:tokens]
    if tokens > 16:
        slots[3], slots[9], slots[11] = -1, pages * page, 2 ** 40
    # Values as slices of one projection, keys with rows that no 16-byte load takes.
    k = (torch.randn(tokens, heads, d + 1, generator=g) * torch.exp(3 * torch.randn(tokens, 1, 1, generator=g))).to(dtype)[..., 1:]
    v = torch.randn(tokens, 2 * heads * d, generator=g).to(dtype)[:, heads * d:].unflatten(1, (heads, d))
    kd = torch.empty(tokens, heads, d + 1, dtype=dtype, device=device)[..., 1:]
    kd.copy_(k)
    vd = torch.empty(tokens, 2 * heads * d, dtype=dtype, device=device)[:, heads * d:].unflatten(1, (heads, d))
    vd.copy_(v)
    for keys in (kd, kd.contiguous()):
        want = _expected_append(cache, slots, k, v)
        ops.kv8_append(cache, slots.to(device), keys, vd)
        _same_cache(cache, want)


@pytest.mark.parametrize("code", CODES)
def test_append_of_any_magnitude(device, code):
    """Rows at every power of two that bfloat16 has, subnormal ones among them, with 0 and -0."""
    say("kv8 append magnitudes", code)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(320, 2, 64, generator=g).double() * 2.0 ** torch.randint(-9, 1, (320, 2, 64), generator=g)
    x = (x * 2.0 ** (torch.arange(320) * 0.8 - 133)[:, None, None]).float().clamp(-3e38, 3e38).to(torch.bfloat16)
    x[:, :, 5], x[:, :, 6] = 0.0, -0.0
    cache = _cache(3, 128, 2, 64, code, device)
    slots = torch.randperm(384, generator=g)[:320]
    want = _expected_append(cache, slots, x, -x)
    ops.kv8_append(cache, slots.to(device), x.to(device), (-x).to(device))
    _same_cache(cache, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
def test_append_special_rows(device, code, dtype):
    """Zeros, the type's largest and smallest numbers, equal magnitudes, halves between codes,
    infinities and NaN."""
    say("kv8 append special", code, dtype)
    d = 32
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    rows = torch.zeros(10, d)
    rows[1, 3] = big
    rows[2] = big
    rows[2, ::2] = -big
    rows[3, :4] = torch.tensor([tiny, -tiny, tiny / 2, 0.0])
    rows[4] = torch.arange(d) - 15.5
    rows[4, 0] = 127.0
    rows[5, 7] = INF
    rows[6, 8] = -INF
    rows[7, 9] = NAN
    rows[8] = -0.0
    rows[9] = torch.linspace(-448, 448, d)
    x = rows.to(dtype)[:, None]
    cache = _cache(1, 64, 1, d, code, device)
    slots = torch.arange(10) * 3
    want = _expected_append(cache, slots, x, x.flip(0))
    ops.kv8_append(cache, slots.to(device), x.to(device), x.flip(0).to(device))
    _same_cache(cache, want)
    back = ops.kv8_gather(cache.keys, cache.key_scales, [0], 28, torch.float32)[0, 0].cpu()[::3]
    assert torch.isnan(back[5:8]).all() and torch.isfinite(back[:5]).all() and (back[0] == 0).all()
    # Reading back is within half a step: of the largest element (int8), of its own binade (e4m3).
    for r in (1, 2, 4, 9):
        top = x[r].double().abs().max()
        off = (back[r].double() - x[r, 0].double()).abs()
        step = top / 127 / 2 if code == torch.int8 else torch.maximum(x[r, 0].double().abs() * 2.0 ** -4, top / 448 * 2.0 ** -10)
        assert (off <= step * (1 + 2.0 ** -20)).all()


def test_append_nothing(device):
    cache = _cache(1, 64, 2, 32, torch.int8, device)
    before = [t.clone() for t in cache]
    empty = torch.empty(0, 2, 32, dtype=torch.bfloat16, device=device)
    ops.kv8_append(cache, torch.empty(0, dtype=torch.int64, device=device), empty, empty)
    assert all(torch.equal(_u8(a) if a.dtype != torch.float32 else a, _u8(b) if b.dtype != torch.float32 else b)
               for a, b in zip(cache, before))


# ------------------------------------------------------------------- norms and rotation
def _tables(rows, d):
    inv = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    angle = torch.cat((angle, angle), dim=1)
    return torch.cos(angle).float(), torch.sin(angle).float()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hkv,d,rows", [(4, 128, 300), (1, 256, 129), (3, 80, 65), (2, 16, 7)])
def test_rotated_keys_have_the_codes_of_their_values(device, hkv, d, rows, code):
    """Bit for bit those of 64 bits: both round ratios of at most 2^9 to fp32 and then to the code, from
    values within 2^-50 of themselves, so that of the 2^17 elements here one differs with less than
    2^17 * 2^-50 * 2^25 = 2^-8. A scale is the fp32 root of the squares' mean times one rounding."""
    say("kv8 rotated keys' codes", hkv, d, rows, code)
    g = torch.Generator().manual_seed(d + rows)
    k = torch.randn(rows, hkv, d, generator=g).to(torch.bfloat16)
    w = 1 + 0.3 * torch.randn(d, generator=g)
    cos, sin = _tables(500, d)
    pos = torch.randint(0, 500, (rows,), generator=g)
    cache = _cache(-(-rows // 64), 64, hkv, d, code, device)
    ops.kv8_norm_rope_append(*(t.to(device) for t in (k, k, k, w, w, cos, sin, pos)), cache,
                             torch.arange(rows, device=device), 1e-6)
    want = oracle.rotate(k, w, cos, sin, pos, 1e-6)
    scale = want.abs().amax(dim=-1) / oracle.MOST[code]
    ratio = (want / scale[..., None]).float()
    codes = (ratio.round() if code == torch.int8 else ratio).to(code)
    assert torch.equal(_u8(cache.keys.cpu().flatten(0, 1))[:rows], _u8(codes))
    got = cache.key_scales.cpu().transpose(1, 2).flatten(0, 1)[:rows].double()
    assert ((got - scale).abs() <= (d / 16 + 8) * 2.0 ** -24 * scale).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d,rows", [(32, 8, 128, 65), (16, 4, 64, 7), (5, 1, 16, 1), (12, 4, 96, 40), (4, 2, 256, 20),
                                           (1, 1, 48, 3)])
def test_norm_rope_append(device, hq, hkv, d, rows, code, dtype):
    say("kv8 norm rope append", hq, hkv, d, rows, code, dtype)
    g = torch.Generator().manual_seed(hq + d + rows)
    eps, page, table_rows = 1e-6, 64, 300
    pages = -(-rows // page) + 1
    x = torch.randn(rows, (hq + 2 * hkv) * d, generator=g).to(dtype)
    x[rows // 2, :d] = 0  # a head of zeros: eps alone under the root
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g) for _ in range(2))
    cos, sin = _tables(table_rows, d)
    pos = torch.randint(0, table_rows, (rows,), generator=g)
    if rows > 4:
        pos[1], pos[2] = -5, 10 ** 12  # clamped to the tables
    slots = torch.randperm(pages * page, generator=g)[:rows]
    if rows > 4:
        slots[4] = -7  # a row that is not stored still has its queries
    q, k, v = (t.unflatten(1, (-1, d)) for t in x.split([hq * d, hkv * d, hkv * d], dim=1))
    want_q, want_k = (oracle.rotate(t, w, cos, sin, pos, eps) for t, w in ((q, qw), (k, kw)))
    # A sum of squares of d fp32 terms, the root, the products and the rotation's two terms: each
    # within a few 2^-24 of the terms' magnitude.
    off = (d / 16 + 16) * 2.0 ** -24
    mag = torch.maximum(want_q.abs(), oracle.rotate(q, qw, cos.abs(), -sin.abs(), pos, eps).abs())
    mag = torch.maximum(mag, oracle.rotate(q, qw, cos.abs(), sin.abs(), pos, eps).abs())
    for strided in (False, True):
        cache = _cache(pages, page, hkv, d, code, device)
        before = [t.cpu().clone() for t in cache]
        on = x.to(device)
        if strided:  # rows that no 16-byte load takes, and a given output
            wide = torch.empty(rows, x.shape[1] + 3, dtype=dtype, device=device)[:, 1:1 + x.shape[1]]
            wide.copy_(on)
            on = wide
            out = torch.full((rows, hq, d + 2), 9.0, dtype=dtype, device=device)[..., :d]
        else:
            out = None
        qd, kd, vd = (t.unflatten(1, (-1, d)) for t in on.split([hq * d, hkv * d, hkv * d], dim=1))
        got = ops.kv8_norm_rope_append(qd, kd, vd, qw.to(device), kw.to(device), cos.to(device), sin.to(device),
                                       pos.to(device), cache, slots.to(device), eps, out=out)
        if strided:
            assert got.data_ptr() == out.data_ptr()
        err = (got.double().cpu() - want_q).abs()
        assert (err <= HALF[dtype] * want_q.abs() + 4 * off * mag + 2.0 ** -24).all(), float(err.max())
        kept = (slots >= 0).nonzero()[:, 0]
        at = slots[kept]
        for i, want in ((0, want_k), (1, v.double())):
            codes = cache[i].cpu().flatten(0, 1)
            codes = _u8(codes)[at].view(code)
            scales = cache[2 + i].cpu()[at // page, :, at % page].double()
            exact = want[kept].abs().amax(dim=-1) / oracle.MOST[code]
            assert ((scales - exact).abs() <= exact * 8 * off + 2.0 ** -100).all()
            # An element's error is relative to the terms it is the difference of, at most 2.5 of
            # the row's largest: in codes, that many of the largest code.
            ratio = want[kept] / scales[..., None]
            slack = 24 * off * oracle.MOST[code]
            lo, hi = ratio - slack, ratio + slack
            c = codes.to(torch.float32).double()
            rnd = (lambda y: y.round()) if code == torch.int8 else (lambda y: y.clamp(-448, 448).float().to(code).double())
            assert ((c >= rnd(lo)) & (c <= rnd(hi))).all()
        # Nothing else was written.
        others = torch.ones(pages * page, dtype=torch.bool)
        others[at] = False
        assert torch.equal(_u8(cache.keys.cpu()).flatten(0, 1)[others], _u8(before[0]).flatten(0, 1)[others])
        assert torch.equal(cache.value_scales.cpu().transpose(1, 2).flatten(0, 1)[others],
                           before[3].transpose(1, 2).flatten(0, 1)[others])


# ---------------------------------------------------------------------------- read back
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("heads,d,page,length", [(8, 128, 256, 1000), (4, 64, 64, 64), (1, 16, 64, 1), (3, 96, 320, 700),
                                                 (2, 256, 128, 129), (5, 176, 64, 0)])
@pytest.mark.parametrize("dtype", [*DTYPES, torch.float32])
def test_gather(device, heads, d, page, length, dtype, code):
    say("kv8 gather", heads, d, page, length, dtype, code)
    g = torch.Generator().manual_seed(d + length)
    n = -(-length // page)
    pages = n + 2
    codes, scales = oracle.quantise(torch.randn(pages, page, heads, d, generator=g), code)
    scales = scales.transpose(1, 2).contiguous()
    order = torch.randperm(pages, generator=g)[:n].to(torch.int32)
    got = ops.kv8_gather(codes.to(device), scales.to(device), order.to(device), length, dtype)
    want = oracle.values(codes, scales)[order.long()].flatten(0, 1)[:length].transpose(0, 1)[None].to(dtype)
    assert got.shape == (1, heads, length, d) and torch.equal(got.cpu(), want)
    if length > 64:  # pages outside the pool read as zeros
        bad = order.clone()
        bad[0], bad[-1] = -1, pages
        got = ops.kv8_gather(codes.to(device), scales.to(device), bad.to(device), length, dtype).cpu()
        assert (got[0, :, :page] == 0).all()
        last = (n - 1) * page
        assert (got[0, :, last:] == 0).all() and torch.equal(got[0, :, page:last], want[0, :, page:last])


# --------------------------------------------------------------------------- attention
def _pool(ends, page, heads, d, code, seed, spread=0.3, spare=2, stale=True):
    """A cache (CPU) of sequences of these lengths, and their table. Codes and scales of pages that
    nobody holds and behind a last key are NaN where the type has one, and wild otherwise."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in ends]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.zeros(len(ends), max(need + [1]), dtype=torch.int32)
    out = []
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(ends):
        for j in range(need[b]):
            table[b, j] = order[at]
            used[order[at], :min(page, n - j * page)] = True
            at += 1
    for _ in range(2):
        x = torch.randn(pages, page, heads, d, generator=g) * torch.exp(spread * torch.randn(pages, page, heads, 1, generator=g))
        codes, scales = oracle.quantise(x, code)
        scales = scales.transpose(1, 2).contiguous()
        if stale:
            _u8(codes)[~used] = 0x7f
            scales[~used[:, None].expand(-1, heads, -1)] = NAN
        out.append((codes, scales))
    return ops.Kv8Cache(out[0][0], out[1][0], out[0][1], out[1][1]), table


def _attend(device, q, cache, table, cu, used, max_q, max_k, window, scale=None, **kw):
    on = ops.Kv8Cache(*(t.to(device) for t in cache))
    plan = ops.Kv8AttnPlan(cu.to(device), used.to(device), total_q=q.shape[0], max_q=max_q, max_k=max_k,
                           n_q_heads=q.shape[1], n_kv_heads=cache.keys.shape[2], head_dim=q.shape[2],
                           page_size=cache.keys.shape[1], window=window, **kw)
    return plan, plan.run(q.to(device), on, table.to(device), scale=scale)


def _tolerance(dtype, want, mag, reach, peak, keys, d):
    """One rounding of the output; weights of 2^-11 relative (one fp16, chunks of bf16 rows) or
    better, of scores whose fp32 sums of d products and exponents are off by E, in the quotient's
    numerator and denominator; and what fp16 loses below its smallest step: 2^-32 of the largest
    weight for each key."""
    e = (d / 2 + 16) * 2.0 ** -24 * reach + 2.0 ** -18
    one = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -20
    return HALF[dtype] * want.abs() + (one + 2 * e) * mag + keys * 2.0 ** -31 * peak + 2.0 ** -25


def _check(got, q, cache, table, cu, used, window, scale=None):
    d = q.shape[2]
    keys, vals = oracle.values(cache.keys, cache.key_scales), oracle.values(cache.values, cache.value_scales)
    want, mag, reach, peak = oracle.attention(q, keys, vals, table, cu, used, window, scale or d ** -0.5)
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    tol = _tolerance(q.dtype, want, mag, reach, peak, int(used.max()) if len(used) else 0, d)
    off = (got - want).abs()
    past = (got == torch.sign(want) * INF) & (want.abs() + tol >= torch.finfo(q.dtype).max)  # rounds to infinity
    bad = ~(off <= tol) & ~want.isnan() & ~past
    assert not bad.any(), (float(off[bad].max()), bad.nonzero()[:5].tolist())


SHAPES = [
    # hq, hkv, d, page, (cached, new) per sequence
    (32, 8, 128, 256, [(0, 1), (1, 1), (30, 1), (31, 1), (255, 1), (256, 1), (700, 1), (2100, 1)]),  # decode rows
    (32, 8, 128, 256, [(700, 4), (0, 4), (33, 2), (300, 1), (5, 0), (90, 3)]),  # few rows, a sequence without any
    (32, 8, 128, 256, [(0, 300), (100, 129), (511, 1), (0, 5), (1000, 64), (20, 63)]),  # chunks beside decode rows
    (16, 4, 64, 64, [(130, 5), (63, 1), (0, 64), (500, 70)]),
    (12, 4, 96, 320, [(319, 1), (320, 2), (10, 100)]),
    (16, 1, 256, 128, [(127, 1), (300, 1), (40, 30)]),  # 16 heads to a KV head
    (32, 1, 64, 64, [(200, 1), (0, 1), (100, 3)]),  # two blocks of them
    (40, 2, 48, 64, [(200, 1), (90, 20)]),
    (5, 1, 16, 64, [(64, 3), (64, 4), (0, 1)]),
    (8, 8, 128, 256, [(400, 16), (400, 17), (256, 1)]),  # a head each
    (128, 1, 32, 64, [(70, 1), (65, 2)]),
]


@pytest.mark.parametrize("window", [(-1, 0), (-1, -1), (100, 0), (0, 0), (40, 7)])
@pytest.mark.parametrize("index", range(len(SHAPES)))
def test_attention(device, index, window):
    hq, hkv, d, page, seqs = SHAPES[index]
    dtype, code = DTYPES[index % 2], CODES[(index // 2 + window[0]) % 2]
    say("kv8 attention", SHAPES[index], window, dtype, code)
    ends = [c + n for c, n in seqs]
    cache, table = _pool(ends, page, hkv, d, code, seed=index)
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32)
    used = torch.tensor(ends, dtype=torch.int32)
    q = torch.randn(int(cu[-1]), hq, d, generator=torch.Generator().manual_seed(index)).to(dtype)
    lens = [n for _, n in seqs]
    plan, got = _attend(device, q, cache, table, cu, used, max(lens), max(ends), window, q_lens=lens)
    assert plan.error_word() == 0
    _check(got, q, cache, table, cu, used, window)
    # Larger bounds and no host lengths: the same bits from another launch.
    plan, again = _attend(device, q, cache, table, cu, used, max(lens) + 9, max(ends) + 1000, window,
                          block_table_width=table.shape[1])
    assert plan.error_word() == 0
    assert torch.equal(got.nan_to_num(), again.nan_to_num())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
def test_attention_long(device, code, dtype):
    """Sequences that split many times, past 64 pages a chunk, beside short ones."""
    say("kv8 attention long", code, dtype)
    seqs = [(9000, 1), (7000, 3), (5000, 20), (17, 1), (4500, 1)]
    ends = [c + n for c, n in seqs]
    cache, table = _pool(ends, 64, 2, 64, code, seed=5)
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32)
    used = torch.tensor(ends, dtype=torch.int32)
    q = torch.randn(int(cu[-1]), 8, 64, generator=torch.Generator().manual_seed(5)).to(dtype) * 3
    _, got = _attend(device, q, cache, table, cu, used, 20, max(ends), (-1, 0))
    _check(got, q, cache, table, cu, used, (-1, 0))


def test_attention_many_sequences(device):
    """More sequences than the planner has threads, rows of every kind among them."""
    say("kv8 attention many sequences")
    g = torch.Generator().manual_seed(8)
    seqs = [(int(torch.randint(0, 90, (1,), generator=g)), [1, 1, 2, 9, 0][i % 5]) for i in range(2100)]
    ends = [c + n for c, n in seqs]
    cache, table = _pool(ends, 64, 1, 16, torch.int8, seed=8)
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32)
    used = torch.tensor(ends, dtype=torch.int32)
    q = torch.randn(int(cu[-1]), 4, 16, generator=g).to(torch.bfloat16)
    plan, got = _attend(device, q, cache, table, cu, used, 9, max(ends), (-1, 0))
    assert plan.error_word() == 0
    _check(got, q, cache, table, cu, used, (-1, 0))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_scales_far_apart(device, dtype, rows):
    """Keys' and values' scales over 2^60, queries over 2^40 of a row and of the rows; values of
    zeros (the least scale) at the keys with the largest weights."""
    say("kv8 attention scales", dtype, rows)
    g = torch.Generator().manual_seed(3)
    cache, table = _pool([300], 64, 2, 64, torch.float8_e4m3fn, seed=3, stale=False)
    cache.value_scales.mul_(torch.exp2(torch.randint(-30, 31, cache.value_scales.shape, generator=g).float()))
    cache.value_scales[:, :, ::7] = 2.0 ** -100
    _u8(cache.values)[:, ::7] = 0
    cache.key_scales.mul_(torch.exp2(torch.randint(-8, 2, cache.key_scales.shape, generator=g).float()))
    q = torch.randn(rows, 8, 64, generator=g) * torch.exp2(torch.randint(-5, 3, (rows, 8, 1), generator=g).float())
    q[:, :, ::5] *= 2.0 ** (-20 if dtype == torch.bfloat16 else -8)
    q = q.to(dtype)
    cu, used = torch.tensor([0, rows], dtype=torch.int32), torch.tensor([300], dtype=torch.int32)
    _, got = _attend(device, q, cache, table, cu, used, rows, 300, (-1, 0))
    _check(got, q, cache, table, cu, used, (-1, 0))


@pytest.mark.parametrize("rows", [1, 3, 50])
def test_attention_cancelling_values(device, rows):
    """Values that cancel but for weights 2^-9 apart: the output is what is left of them."""
    say("kv8 attention cancelling", rows)
    n, d = 200 + rows, 64
    cache, table = _pool([n], 256, 1, d, torch.int8, seed=1, stale=False)
    _u8(cache.keys).zero_()
    cache.keys[:, :, 0, 0] = 1
    cache.key_scales.fill_(0.0)
    cache.key_scales[:, :, ::2] = 8 * 2.0 ** -9  # score 2^-9 of every second key
    cache.values[:, ::2] = 100
    cache.values[:, 1::2] = -100
    cache.value_scales.fill_(1.0)
    q = torch.zeros(rows, 2, d)
    q[..., 0] = 1.0
    q = q.to(torch.float16)
    cu, used = torch.tensor([0, rows], dtype=torch.int32), torch.tensor([n], dtype=torch.int32)
    _, got = _attend(device, q, cache, table, cu, used, rows, n, (-1, -1), scale=1 / 8)
    _check(got, q, cache, table, cu, used, (-1, -1), scale=1 / 8)


@pytest.mark.parametrize("rows", [1, 4, 40])
def test_attention_of_rows_stored_as_nan(device, rows):
    """A key or value stored as NaN makes the rows that see it NaN in its head, and no others."""
    say("kv8 attention nan", rows)
    n = 500
    cache, table = _pool([n, n, n], 256, 2, 64, torch.float8_e4m3fn, seed=2)
    key = n - rows // 2 - 1  # hidden from the first half of the rows
    for b, scales in ((0, cache.key_scales), (1, cache.value_scales)):
        scales[int(table[b, key // 256]), 1, key % 256] = NAN
    cu = torch.tensor([0, rows, 2 * rows, 3 * rows], dtype=torch.int32)
    used = torch.tensor([n, n, n], dtype=torch.int32)
    q = torch.randn(3 * rows, 4, 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    _, got = _attend(device, q, cache, table, cu, used, rows, n, (-1, 0))
    nan = got.isnan().cpu()
    first = rows - rows // 2 - 1
    want = torch.zeros_like(nan)
    for b in (0, 1):
        want[b * rows + first:(b + 1) * rows, 2:] = True
    assert torch.equal(nan, want)
    keys, vals = oracle.values(cache.keys, cache.key_scales), oracle.values(cache.values, cache.value_scales)
    keys, vals = keys.nan_to_num(0.0), vals.nan_to_num(0.0)
    out, mag, reach, peak = oracle.attention(q, keys, vals, table, cu, used, (-1, 0), 1 / 8)
    off = (got.double().cpu() - out).abs()
    assert (off[~want] <= _tolerance(q.dtype, out, mag, reach, peak, n, 64)[~want]).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_of_infinite_queries(device, rows):
    """An infinite or NaN element makes its own row and head NaN, and no others."""
    say("kv8 attention odd queries", rows)
    cache, table = _pool([300], 256, 1, 64, torch.int8, seed=4)
    cu, used = torch.tensor([0, rows], dtype=torch.int32), torch.tensor([300], dtype=torch.int32)
    q = torch.randn(rows, 4, 64, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    _, clean = _attend(device, q, cache, table, cu, used, rows, 300, (-1, 0))
    odd = q.clone()
    odd[rows // 2, 1, 5], odd[rows - 1, 2, 6] = INF, NAN
    _, got = _attend(device, odd, cache, table, cu, used, rows, 300, (-1, 0))
    keep = torch.ones(rows, 4, dtype=torch.bool)
    keep[rows // 2, 1] = keep[rows - 1, 2] = False
    keep = keep.to(device)
    assert got[~keep].isnan().all() and torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("new", [1, 20])
def test_attention_of_bad_metadata(device, new):
    """Pages outside the pool are no keys; lengths past their bounds are cut; both are flagged, and
    rows of a malformed cu_seq_q stay as they were."""
    say("kv8 attention bad metadata", new)
    cache, table = _pool([600, 600], 256, 2, 64, torch.int8, seed=6)
    cu, used = torch.tensor([0, new, 2 * new], dtype=torch.int32), torch.tensor([600, 600], dtype=torch.int32)
    q = torch.randn(2 * new, 4, 64, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = -1, cache.keys.shape[0]
    plan, got = _attend(device, q, cache, bad, cu, used, new, 600, (-1, 0))
    assert plan.error_word() == _capi.HX_WERR_BAD_PAGE
    with pytest.raises(RuntimeError, match="page id"):
        plan.check_errors()
    _check(got, q, cache, bad, cu, used, (-1, 0))
    # all pages bad: no key is left
    _, got = _attend(device, q, cache, torch.full_like(table, -1), cu, used, new, 600, (-1, 0))
    assert (got == 0).all()
    # longer than max_k, and negative
    plan, got = _attend(device, q, cache, table, cu, torch.tensor([700, -3], dtype=torch.int32), new, 600, (-1, 0))
    assert plan.error_word() == _capi.HX_WERR_CLAMPED_LEN
    _check(got, q, cache, table, cu, torch.tensor([600, 0], dtype=torch.int32), (-1, 0))
    # fewer keys than rows: the first rows have none
    _, got = _attend(device, q, cache, table, cu, torch.tensor([new // 2, 0], dtype=torch.int32), new, 600, (-1, 0))
    _check(got, q, cache, table, cu, torch.tensor([new // 2, 0], dtype=torch.int32), (-1, 0))
    assert (got[new:] == 0).all()
    # a cu_seq_q that runs backwards
    on = ops.Kv8Cache(*(t.to(device) for t in cache))
    plan = ops.Kv8AttnPlan(torch.tensor([0, 2 * new, new], dtype=torch.int32, device=device), used.to(device), total_q=2 * new,
                           max_q=2 * new, max_k=600, n_q_heads=4, n_kv_heads=2, head_dim=64, page_size=256)
    plan.run(q.to(device), on, table.to(device))
    assert plan.error_word() == _capi.HX_WERR_BAD_CU_SEQ


def test_attention_layouts(device):
    """Strided queries, tables wider than planned, given outputs; rows behind the last sequence
    stay as they were."""
    say("kv8 attention layouts")
    seqs = [(300, 1), (100, 30), (40, 2)]
    ends = [c + n for c, n in seqs]
    cache, table = _pool(ends, 64, 2, 64, torch.float8_e4m3fn, seed=7)
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32)
    used = torch.tensor(ends, dtype=torch.int32)
    total = int(cu[-1])
    q = torch.randn(total, 8, 64, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16)
    _, want = _attend(device, q, cache, table, cu, used, 30, max(ends), (-1, 0))
    on = ops.Kv8Cache(*(t.to(device) for t in cache))
    wide = torch.full((len(seqs), table.shape[1] + 5), -9, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = table.to(device)
    padded = torch.cat((q, q[:7])).to(device)
    plan = ops.Kv8AttnPlan(cu.to(device), used.to(device), total_q=total + 7, max_q=30, max_k=max(ends), n_q_heads=8,
                           n_kv_heads=2, head_dim=64, page_size=64)
    for make in (lambda: padded,
                 lambda: padded.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda: torch.cat((padded, padded), dim=2)[..., 64:],
                 lambda: torch.nn.functional.pad(padded, (1, 2))[..., 1:65]):
        out = torch.full((total + 7, 8, 66), 5.0, dtype=torch.bfloat16, device=device)[..., :64]
        got = plan.run(make(), on, wide[:, :table.shape[1] + 2], out=out)
        assert got.data_ptr() == out.data_ptr()
        assert torch.equal(out[:total], want) and (out[total:] == 5).all()
    assert plan.error_word() == 0
    one = ops.kv8_attn(q.to(device), on, cu.to(device), used.to(device), table.to(device), max_q=30, max_k=max(ends),
                       window_size=(-1, 0))
    assert torch.equal(one, want)
    causal = ops.kv8_attn(q.to(device), on, cu.to(device), used.to(device), table.to(device), max_q=30, max_k=max(ends),
                          is_causal=True)
    assert torch.equal(causal, want)


def test_attention_and_append_past_32_bits(device):
    """Codes more than 2^32 bytes and scales more than 2^32 / 16 elements into their pools."""
    say("kv8 past 32 bits")
    page, heads, d = 256, 8, 128
    pages = 2 ** 32 // (page * heads * d) + 3
    codes = torch.empty((2, pages, page, heads, d), dtype=torch.int8, device=device)
    scales = torch.empty((2, pages, heads, page), device=device)
    cache = ops.Kv8Cache(codes[0], codes[1], scales[0], scales[1])
    tail = ops.Kv8Cache(*(t[-3:].contiguous() for t in cache))
    g = torch.Generator(device=device).manual_seed(9)
    k, v = (torch.randn(600, heads, d, generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    at = torch.arange(600, device=device)
    ops.kv8_append(cache, at + (pages - 3) * page, k, v)
    ops.kv8_append(tail, at, k, v)
    for high in (1, 25):
        q = torch.randn(high, 32, d, generator=g, device=device).to(torch.bfloat16)
        cu = torch.tensor([0, high], dtype=torch.int32, device=device)
        used = torch.tensor([600], dtype=torch.int32, device=device)
        outs = [ops.kv8_attn(q, c, cu, used, torch.arange(first, first + 3, dtype=torch.int32, device=device)[None],
                             max_q=high, max_k=600, is_causal=True) for c, first in ((cache, pages - 3), (tail, 0))]
        assert torch.equal(*outs) and torch.isfinite(outs[0]).all()
    back = [ops.kv8_gather(c.keys, c.key_scales, list(range(first, first + 3)), 600, torch.float32)
            for c, first in ((cache, pages - 3), (tail, 0))]
    assert torch.equal(*back)


# -------------------------------------------------------------- streams, graphs, refusals
def _tick(device, seed, lens=((300, 1), (90, 40), (700, 3))):
    ends = [c + n for c, n in lens]
    cache, table = _pool(ends, 256, 2, 64, torch.float8_e4m3fn, seed=seed, stale=False)
    cu = torch.tensor([0] + [n for _, n in lens]).cumsum(0).to(torch.int32)
    q = torch.randn(int(cu[-1]), 8, 64, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
    return (ops.Kv8Cache(*(t.to(device) for t in cache)), table.to(device), cu.to(device),
            torch.tensor(ends, dtype=torch.int32, device=device), q.to(device), ends, [n for _, n in lens])


def test_whole_step_in_a_graph(device):
    """Append, plan and attention captured once and replayed on other data and lengths, with eager
    work between the replays."""
    say("kv8 graph")
    cache, table, cu, used, q, ends, lens = _tick(device, 1)
    total = q.shape[0]
    k, v = (torch.randn(total, 2, 64, device=device).to(torch.bfloat16) for _ in range(2))
    pos = torch.cat([torch.arange(e - n, e) for e, n in zip(ends, lens)]).to(device)
    of = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)]).to(device)
    slots = table.long()[of, pos // 256] * 256 + pos % 256

    def step():
        ops.kv8_append(cache, slots, k, v)
        return ops.kv8_attn(q, cache, cu, used, table, max_q=40, max_k=1024, is_causal=True)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
    for turn in range(5):
        g = torch.Generator(device=device).manual_seed(turn)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=device))
        used.copy_(torch.tensor([300 - turn, 130, 703 - 100 * turn], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())


def test_two_graphs_share_memory(device):
    """Two captured steps in one memory pool, replayed in turn."""
    say("kv8 two graphs")
    ticks = [_tick(device, s) for s in (1, 2)]
    wants = [ops.kv8_attn(q, c, cu, used, table, max_q=40, max_k=1024, is_causal=True) for c, table, cu, used, q, _, _ in ticks]
    stream, pool, graphs, outs = torch.cuda.Stream(), None, [], []
    with torch.cuda.stream(stream):
        for c, table, cu, used, q, _, _ in ticks:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream, pool=pool):
                outs.append(ops.kv8_attn(q, c, cu, used, table, max_q=40, max_k=1024, is_causal=True))
            pool = graph.pool()
            graphs.append(graph)
    for turn in range(4):
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[turn % 2], wants[turn % 2])


def test_runs_on_another_stream(device):
    say("kv8 stream")
    cache, table, cu, used, q, _, _ = _tick(device, 3)
    want = ops.kv8_attn(q, cache, cu, used, table, max_q=40, max_k=1024, is_causal=True)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        busy = torch.randn(4096, 4096, device=device)
        for _ in range(3):
            busy = busy @ busy * 1e-3
        fresh = q * 1  # ready only after the products
        got = ops.kv8_attn(fresh, cache, cu, used, table, max_q=40, max_k=1024, is_causal=True)
    stream.synchronize()
    assert torch.equal(got, want)


def test_plan_of_another_shape_is_flagged(device):
    """A run whose workspace holds another tick's plan writes nothing and says so."""
    say("kv8 plan mismatch")
    cache, table, cu, used, q, _, _ = _tick(device, 4)
    make = lambda total: ops.Kv8AttnPlan(cu, used, total_q=total, max_q=40, max_k=1024, n_q_heads=8, n_kv_heads=2,  # noqa: E731
                                         head_dim=64, page_size=256, block_table_width=table.shape[1])
    plan, other = make(q.shape[0]), make(q.shape[0] + 1)
    other._shape, other._q_shape = plan._shape, plan._q_shape
    out = torch.full_like(q, 3.0)
    other.run(q, cache, table, out=out)
    assert other.error_word() == _capi.HX_WERR_PLAN_MISMATCH and (out == 3).all()


def test_refusals(device):
    say("kv8 refusals")
    cache, table, cu, used, q, _, _ = _tick(device, 5)
    k = torch.randn(4, 2, 64, device=device).to(torch.bfloat16)
    slots = torch.arange(4, device=device)
    with pytest.raises(ValueError, match="float8_e4m3fn or int8"):
        ops.kv8_append(cache._replace(keys=cache.keys.view(torch.uint8)), slots, k, k)
    with pytest.raises(ValueError, match="same dtypes"):
        ops.kv8_append(cache._replace(values=cache.values[:1]), slots, k, k)
    with pytest.raises(ValueError, match="float32"):
        ops.kv8_append(cache._replace(key_scales=cache.key_scales.double()), slots, k, k)
    with pytest.raises(ValueError, match="one dtype"):
        ops.kv8_append(cache, slots, k, k.half())
    with pytest.raises(ValueError, match="one dtype"):
        ops.kv8_append(cache, slots, k.float(), k.float())
    with pytest.raises(ValueError, match="int64"):
        ops.kv8_append(cache, slots.int(), k, k)
    with pytest.raises(ValueError, match="heads"):
        ops.kv8_append(cache, slots, k[:, :1], k[:, :1])
    with pytest.raises(ValueError, match="contiguous head_dim"):
        ops.kv8_append(cache, slots, k.transpose(1, 2).contiguous().transpose(1, 2), k)
    odd = ops.Kv8Cache(*(torch.zeros(1, 64, 1, 24, dtype=torch.int8, device=device),) * 2,
                       *(torch.zeros(1, 1, 64, device=device),) * 2)
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.kv8_append(odd, slots, k[:, :1, :24], k[:, :1, :24])
    with pytest.raises(ValueError, match="length"):
        ops.kv8_gather(cache.keys, cache.key_scales, [0], 257, torch.bfloat16)
    with pytest.raises(ValueError, match="gives"):
        ops.kv8_gather(cache.keys, cache.key_scales, [0], 7, torch.float64)
    cos = torch.ones(4, 64, device=device)
    w = torch.ones(64, device=device)
    with pytest.raises(ValueError, match="positions"):
        ops.kv8_norm_rope_append(k, k, k, w, w, cos, cos, slots[:3], cache, slots, 1e-6)
    with pytest.raises(ValueError, match="at least one row"):
        ops.kv8_norm_rope_append(k, k, k, w, w, cos[:0], cos[:0], slots, cache, slots, 1e-6)
    with pytest.raises(ValueError, match="queries"):
        ops.kv8_norm_rope_append(k[:3], k, k, w, w, cos, cos, slots, cache, slots, 1e-6)
    plan = ops.Kv8AttnPlan(cu, used, total_q=q.shape[0], max_q=40, max_k=703, n_q_heads=8, n_kv_heads=2, head_dim=64,
                           page_size=256)
    with pytest.raises(ValueError, match="as planned"):
        plan.run(q[:-1], cache, table)
    with pytest.raises(ValueError, match="block_table"):
        plan.run(q, cache, table[:, :1])
    with pytest.raises(ValueError, match="block_table"):
        plan.run(q, cache, table[:2])
    with pytest.raises(ValueError, match="scale"):
        plan.run(q, cache, table, scale=-1.0)
    with pytest.raises(ValueError, match="out"):
        plan.run(q, cache, table, out=q.float())
    with pytest.raises(RuntimeError, match="ROCm device only"):
        plan.run(q.cpu(), cache, table)
    for kw, text in ((dict(head_dim=72), "Unsupported"), (dict(page_size=96), "Unsupported"), (dict(n_q_heads=7), "multiple"),
                     (dict(n_q_heads=258), "Unsupported"), (dict(max_q=-1), "non-negative")):
        given = dict(total_q=4, max_q=4, max_k=64, n_q_heads=8, n_kv_heads=2, head_dim=64, page_size=256) | kw
        with pytest.raises(ValueError, match=text):
            ops.Kv8AttnPlan(cu, used, **given)


def test_empty_ticks(device):
    """No sequences, no rows, no keys."""
    say("kv8 empty")
    cache, table, _, _, q, _, _ = _tick(device, 6)
    none = torch.zeros(1, dtype=torch.int32, device=device)
    out = ops.kv8_attn(q[:0], cache, none, none[:0], table[:0], max_q=1, max_k=10)
    assert out.shape == (0, 8, 64)
    cu = torch.tensor([0, 0, 1], dtype=torch.int32, device=device)
    out = ops.kv8_attn(q[:1], cache, cu, torch.zeros(2, dtype=torch.int32, device=device), table[:2], max_q=1, max_k=0)
    assert (out == 0).all()


def test_scale_and_mean(device):
    """A scale so large that only the best key counts, and one so small that all count alike."""
    cache, table, cu, used, q, ends, lens = _tick(device, 7)
    for scale in (1e4, 1e-8):
        got = ops.kv8_attn(q, cache, cu, used, table, max_q=40, max_k=1024, is_causal=True, scale=scale)
        host = ops.Kv8Cache(*(t.cpu() for t in cache))
        if scale < 1:
            _check(got, q.cpu(), host, table.cpu(), cu.cpu(), used.cpu(), (-1, 0), scale=scale)
        else:
            keys, vals = (oracle.values(c, s).double() for c, s in ((host.keys, host.key_scales), (host.values, host.value_scales)))
            row, L = 0, ends[0]
            pages = table[0].long().cpu()
            k, v = keys[pages].flatten(0, 1)[:L, 0], vals[pages].flatten(0, 1)[:L, 0]
            best = int((k @ q[row, 0].double().cpu()).argmax())
            assert (got[row, 0].double().cpu() - v[best]).abs().max() <= HALF[torch.bfloat16] * v[best].abs().max()
    assert math.isfinite(float(got.float().sum()))
