"""Drawn tokens against the definition in 64 bits: every limit and their combinations, ties,
special logits, and numbers at the ends of their range."""

from __future__ import annotations

import math

import pytest
import torch

from helios_amd import ops
from oracle import kv8 as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NAN, INF = float("nan"), float("inf")


def _check(device, logits, u, got=None, **limits):
    """Tokens are the definition's; a logprob is one fp32 rounding of it (2^-24 of itself), of sums
    of weights that are each within 2^-45 of the largest: vocab * 2^-44 of W >= 1."""
    on = {k: None if t is None else t.to(device) for k, t in limits.items()}
    if got is None:
        got = ops.sample_tokens(logits.to(device), u.to(device), **on)
    ids, logs = oracle.sample(logits, u, **limits)
    assert got.token_ids.dtype == torch.int64 and got.logprobs.dtype == torch.float32
    assert got.token_ids.tolist() == ids.tolist()
    have = got.logprobs.double().cpu()
    same = have == logs  # infinities
    assert ((have - logs).abs()[~same] <= 2.0 ** -23 * logs.abs()[~same] + logits.shape[1] * 2.0 ** -44 + 2.0 ** -45).all()
    return got


def _limits(rows, g, k=None, p=None, m=None, t=None):
    def some(low, high):
        return low + (high - low) * torch.rand(rows, generator=g)
    return dict(
        temperature=None if t is None else some(*t),
        top_k=None if k is None else torch.randint(k[0], k[1] + 1, (rows,), generator=g).to(torch.int32),
        top_p=None if p is None else some(*p), min_p=None if m is None else some(*m))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 1000, 4099])
@pytest.mark.parametrize("spread", [0.01, 1.0, 6.0])
def test_small_vocabularies(device, vocab, spread, dtype):
    """Every combination of limits, rows of each."""
    say("sample", vocab, spread, dtype)
    g = torch.Generator().manual_seed(vocab)
    rows = 6
    for which in range(16):
        logits = (torch.randn(rows, vocab, generator=g) * spread).to(dtype)
        limits = _limits(rows, g, k=(1, max(1, vocab // 2)) if which & 1 else None, p=(0.0, 1.0) if which & 2 else None,
                         m=(0.0, 0.6) if which & 4 else None, t=(0.2, 3.0) if which & 8 else None)
        _check(device, logits, torch.rand(rows, generator=g), **limits)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [151936, 151669, 1 << 18])
def test_large_vocabularies(device, vocab, dtype):
    """Rows of a few and of most tokens kept, by each limit: lists of one launch's size and past it."""
    say("sample", vocab, dtype)
    g = torch.Generator().manual_seed(vocab % 1000)
    limits = dict(
        temperature=torch.tensor([0.7, 1.0, 1.0, 5.0, 1.0, 0.0, 1.3, 1.0]),
        top_k=torch.tensor([50, 0, 5000, 100000, -3, 7, 0, vocab + 5], dtype=torch.int32),
        top_p=torch.tensor([0.9, 0.95, 0.99, 0.9, 1.0, 0.1, 0.5, 2.0]),
        min_p=torch.tensor([0.0, 0.001, 0.0, 1e-5, 0.0, 0.9, 1e-30, 0.0]))
    logits = (torch.randn(8, vocab, generator=g) * torch.tensor([3.0, 3, 0.5, 0.3, 2, 1, 1, 0.01])[:, None]).to(dtype)
    _check(device, logits, torch.rand(8, generator=g), **limits)


@pytest.mark.parametrize("dtype", DTYPES)
def test_ties(device, dtype):
    """More equal logits than a launch orders at once: the lower id first, at every border."""
    say("sample ties", dtype)
    vocab = 20000
    logits = torch.zeros(9, vocab)
    logits[1] = 3.0
    logits[1, ::3] = 4.0                  # 6667 of the largest
    logits[2, 100:] = -1.0                # 100, then 19900 equal ones
    logits[3, 5] = 2.0
    logits[4, 19999] = 1e-3
    logits[5] = -0.0
    logits[5, ::2] = 0.0                  # 0 and -0 are equal
    logits[6] = -INF
    logits[6, 7000:14000] = 1.0           # an allowed range, all alike
    logits[7, 3:] = -INF
    logits[8] = (torch.arange(vocab) % 5).float()
    logits = logits.to(dtype)
    u = torch.tensor([0.3, 0.99, 0.7, 0.5, 0.25, 0.6, 0.123, 0.9, 0.8])
    for limits in (dict(), dict(top_k=torch.tensor([3000, 7000, 5000, 1, 19999, 9, 7000, 2, 4001], dtype=torch.int32)),
                   dict(top_p=torch.tensor([0.5, 0.25, 0.9, 1.0, 0.75, 0.125, 0.5, 0.6, 0.3])),
                   dict(top_k=torch.full((9,), 6000, dtype=torch.int32), top_p=torch.full((9,), 0.5), min_p=torch.full((9,), 0.5)),
                   dict(temperature=torch.full((9,), 0.01), min_p=torch.full((9,), 1.0))):
        _check(device, logits, u, **limits)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [20011, 151936])
def test_small_top_k(device, vocab, dtype):
    """A small top_k where its first tokens lie together, are tied, or few are allowed at all: more
    tokens at its bound than one list holds, and fewer than top_k."""
    say("sample small top_k", vocab, dtype)
    g = torch.Generator().manual_seed(vocab % 97)
    rising = torch.arange(vocab) * (8.0 / vocab)
    logits = torch.zeros(11, vocab)
    logits[0] = torch.randn(vocab, generator=g) * 3
    logits[1] = rising.flip(0)
    logits[2] = rising
    logits[3, 77::7] = 2.0                # a seventh of the largest
    logits[4] = -INF
    logits[4, 5000:8000] = torch.randn(3000, generator=g)
    logits[5] = torch.finfo(dtype).min
    logits[5, 9::400] = torch.randn(logits[5, 9::400].shape, generator=g)
    logits[6] = -INF
    logits[6, vocab - 1] = -2.0
    logits[7, :100] = 1.0
    logits[8] = torch.randn(vocab, generator=g)
    logits[8, 40:72] += 20.0              # a group's 32 tokens far above the others
    logits[9] = torch.randn(vocab, generator=g) * 1e-3
    logits[10] = -INF
    logits[10, ::97] = 1.5
    logits = logits.to(dtype)
    u = torch.rand(11, generator=g)
    k = torch.tensor([1, 33, 200, 64, 150, 100, 5, 120, 207, 208, 90], dtype=torch.int32)
    _check(device, logits, u, top_k=k)
    _check(device, logits, u, top_k=k, top_p=torch.rand(11, generator=g), temperature=0.1 + 2 * torch.rand(11, generator=g))
    _check(device, logits, u, top_k=k.flip(0), min_p=torch.rand(11, generator=g))
    _check(device, logits, u, top_k=7 * k, top_p=torch.full((11,), 0.99), min_p=torch.full((11,), 1e-4))
    store = torch.zeros(11, vocab + 3, dtype=dtype)
    store[:, 1:vocab + 1] = logits       # rows that begin anywhere
    got = ops.sample_tokens(store.to(device)[:, 1:vocab + 1], u.to(device), top_k=k.to(device))
    _check(device, logits, u, got, top_k=k)


def test_small_top_k_of_many_rows(device):
    """One workgroup a row, and rows of every kind side by side."""
    say("sample small top_k, many rows")
    g = torch.Generator().manual_seed(3)
    rows = 900
    logits = torch.randn(rows, 4099, generator=g) * 2
    _check(device, logits, torch.rand(rows, generator=g), top_k=torch.randint(-1, 90, (rows,), generator=g).to(torch.int32),
           top_p=0.5 + torch.rand(rows, generator=g), temperature=torch.rand(rows, generator=g))


def test_special_logits(device):
    """Infinities and NaN; rows that nothing is allowed in."""
    say("sample special")
    for dtype in DTYPES:
        logits = torch.randn(8, 500, generator=torch.Generator().manual_seed(1))
        logits[0, 70] = INF
        logits[0, 90] = INF
        logits[1, 80] = NAN
        logits[1, 20] = INF
        logits[2] = -INF
        logits[3, 1:] = -INF
        logits[4, ::2] = -INF
        logits[5] = -INF
        logits[5, 499] = -3.0
        logits[6] = torch.finfo(dtype).max
        logits[7] = -torch.finfo(dtype).max
        logits[7, 33] = torch.finfo(dtype).max
        logits = logits.to(dtype)
        u = torch.linspace(0.05, 0.95, 8)
        _check(device, logits, u)
        _check(device, logits, u, top_k=torch.full((8,), 400, dtype=torch.int32), top_p=torch.full((8,), 0.9),
               min_p=torch.full((8,), 1e-3), temperature=torch.full((8,), 2.0))


def test_ends_of_the_ranges(device):
    """Numbers at and past 0 and 1, limits at and past theirs, temperatures of every size."""
    say("sample ends")
    g = torch.Generator().manual_seed(2)
    row = torch.randn(1, 3001, generator=g)
    u = torch.tensor([0.0, -1.0, 1.0 - 2.0 ** -24, 1.0, 7.0, 2.0 ** -149])
    logits = row.expand(6, -1).contiguous()
    for limits in (dict(), dict(top_k=torch.full((6,), 2500, dtype=torch.int32)), dict(top_p=torch.full((6,), 0.3))):
        _check(device, logits, u, **{k: v for k, v in limits.items()})
    half = torch.full((6,), 0.5)
    _check(device, logits, half, top_p=torch.tensor([0.0, -1.0, 1.0, 1.5, 1e-30, 1 - 2.0 ** -24]))
    _check(device, logits, half, min_p=torch.tensor([0.0, -1.0, 1.0, 2.0, 1e-38, 1 - 2.0 ** -24]))
    _check(device, logits, half, temperature=torch.tensor([1e-30, 1e-6, 1e6, 1e30, 0.0, -2.0]))
    _check(device, logits * 1e4, half, temperature=torch.tensor([1e-3, 1.0, 1e3, 1e4, 1e5, 1e9]))
    _check(device, logits * 1e-20, half, temperature=torch.tensor([1e-20, 1e-21, 1.0, 1e-25, 1e-19, 1e9]))
    top = ops.sample_tokens(logits.to(device), half.to(device), temperature=torch.full((6,), INF, device=device))
    assert ((top.logprobs + math.log(3001)).abs() <= 2.0 ** -23 * math.log(3001)).all()  # all alike
    got = ops.sample_tokens(logits[:0].to(device), u[:0].to(device))
    assert got.token_ids.shape == (0,) and got.logprobs.shape == (0,)


def test_logits_far_from_zero(device):
    """Logits whose differences are a few of their last places: borders do not move with them."""
    say("sample far")
    g = torch.Generator().manual_seed(3)
    logits = 10000 + torch.randint(0, 40, (5, 30000), generator=g) * 2.0 ** -10
    for p, m in ((0.5, None), (None, 0.99), (0.9, 0.97)):
        _check(device, logits, torch.rand(5, generator=g), top_p=None if p is None else torch.full((5,), p),
               min_p=None if m is None else torch.full((5,), m))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows(device, dtype):
    """Rows of a wider tensor, at every alignment; a single row of any stride."""
    say("sample strides", dtype)
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(4, 9001, generator=g).to(dtype)
    on = wide.to(device)
    u = torch.rand(4, generator=g)
    k = torch.full((4,), 300, dtype=torch.int32)
    for lead in range(9):
        part = wide[:, lead:lead + 8000]
        got = ops.sample_tokens(on[:, lead:lead + 8000], u.to(device), top_k=k.to(device))
        _check(device, part, u, got=got, top_k=k)
    got = ops.sample_tokens(on[2:3, 1:], u[:1].to(device))
    _check(device, wide[2:3, 1:], u[:1], got=got)


def test_many_rows(device):
    say("sample many rows")
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(3000, 40, generator=g)
    _check(device, logits, torch.rand(3000, generator=g), **_limits(3000, g, k=(0, 30), p=(0.1, 1.0), t=(0.0, 2.0)))


def test_shares(device):
    """Over evenly spaced numbers every kept token comes up as often as its weight says."""
    say("sample shares")
    n = 4096
    logits = torch.log(torch.tensor([[8.0, 4.0, 2.0, 1.0, 1.0]]))
    u = (torch.arange(n, dtype=torch.float32) + 0.5) / n
    got = ops.sample_tokens(logits.expand(n, -1).contiguous().to(device), u.to(device)).token_ids.cpu()
    assert torch.bincount(got, minlength=5).tolist() == [n // 2, n // 4, n // 8, n // 16, n // 16]


def test_in_a_graph(device):
    """Captured once and replayed on other logits and limits, two graphs in one pool in turn, with
    eager work between."""
    say("sample graph")
    g = torch.Generator(device=device).manual_seed(6)
    sets, graphs, outs, pool = [], [], [], None
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for rows in (3, 20):
            s = dict(logits=torch.randn(rows, 151936, device=device), uniforms=torch.rand(rows, device=device),
                     temperature=torch.ones(rows, device=device), top_k=torch.full((rows,), 40, dtype=torch.int32, device=device),
                     top_p=torch.full((rows,), 0.9, device=device))
            ops.sample_tokens(**s)
            stream.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream, pool=pool):
                outs.append(ops.sample_tokens(**s))
            pool = graph.pool()
            sets.append(s)
            graphs.append(graph)
    for turn in range(6):
        s = sets[turn % 2]
        s["logits"].copy_(3 * torch.randn(s["logits"].shape, generator=g, device=device))
        s["uniforms"].copy_(torch.rand(s["uniforms"].shape, generator=g, device=device))
        s["top_k"].fill_(turn * 900)  # 0: none
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs[turn % 2]]
        want = ops.sample_tokens(**s)
        assert torch.equal(got[0], want.token_ids) and torch.equal(got[1], want.logprobs)


def test_refusals(device):
    logits, u = torch.zeros(2, 8, device=device), torch.zeros(2, device=device)
    with pytest.raises(ValueError, match="rows, vocab"):
        ops.sample_tokens(logits.double(), u)
    with pytest.raises(ValueError, match="rows, vocab"):
        ops.sample_tokens(logits[:, :0], u)
    with pytest.raises(ValueError, match="at most"):
        ops.sample_tokens(torch.zeros(1, (1 << 18) + 1, device=device), u[:1])
    with pytest.raises(ValueError, match="overlap"):
        ops.sample_tokens(logits.t(), torch.zeros(8, device=device))
    with pytest.raises(ValueError, match="uniforms"):
        ops.sample_tokens(logits, u.double())
    with pytest.raises(ValueError, match="top_k"):
        ops.sample_tokens(logits, u, top_k=u)
    with pytest.raises(ValueError, match="min_p"):
        ops.sample_tokens(logits, u, min_p=u[:1])
    with pytest.raises(ValueError, match="top_p"):
        ops.sample_tokens(logits, u, top_p=u.cpu())
    with pytest.raises(RuntimeError, match="ROCm device only"):
        ops.sample_tokens(logits.cpu(), u.cpu())
