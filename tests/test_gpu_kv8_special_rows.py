"""Infinite and NaN elements through the quantising append with norms and rotation."""

from __future__ import annotations

import pytest
import torch

from helios_amd import ops
from oracle import kv8 as oracle
from tests.gpu_cases import say
from tests.test_gpu_kv8 import CODES, DTYPES, INF, NAN, _bits, _cache, _tables, _u8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [16, 64, 80, 128, 176, 256])
def test_infinite_and_nan_elements(device, d, code, dtype):
    """A key or value with such an element is stored as zeros under a NaN scale, also where its cosine,
    sine or norm weight is 0; a query's NaN are the formula's; every other head row has the bits that
    it has beside finite ones."""
    say("kv8 norm rope append of odd elements", d, code, dtype)
    hq, hkv, rows, eps = 4, 3, 12, 1e-6
    g = torch.Generator().manual_seed(d)
    q = torch.randn(rows, hq, d, generator=g).to(dtype)
    k, v = (torch.randn(rows, hkv, d, generator=g).to(dtype) for _ in range(2))
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g) for _ in range(2))
    cos, sin = _tables(rows, d)
    cos[5], sin[6] = 0.0, 0.0
    kw[3] = qw[3] = 0.0
    pos = torch.arange(rows)
    odd = [(1, 0, 0, INF), (2, 1, d - 1, -INF), (3, 2, d // 2, NAN), (5, 0, 1, INF), (6, 1, 2, -INF), (7, 0, 3, INF),
           (8, 2, 3, NAN), (9, 1, d // 2 + 3, INF), (10, 0, 5, INF), (10, 0, 7, -INF)]
    bad = [t.clone() for t in (q, k, v)]
    for row, head, at, x in odd:
        for t in bad:
            t[row, head, at] = x
    caches, outs = [], []
    for given in ((q, k, v), bad):
        cache = _cache(1, 64, hkv, d, code, device)
        outs.append(ops.kv8_norm_rope_append(*(t.to(device) for t in (*given, qw, kw, cos, sin, pos)), cache,
                                             torch.arange(rows, device=device) * 3, eps).cpu())
        caches.append([t.cpu() for t in cache])
    hit = torch.zeros(rows, hkv, dtype=torch.bool)
    for row, head, _, _ in odd:
        hit[row, head] = True
    for i in (0, 1):
        clean, got = (_u8(c[i])[0, :3 * rows:3] for c in caches)
        assert (got[hit] == 0).all() and torch.equal(got[~hit], clean[~hit])
        clean, got = (c[2 + i][0, :, :3 * rows:3].t() for c in caches)
        assert got[hit].isnan().all() and torch.equal(_bits(got[~hit]), _bits(clean[~hit]))
    want = oracle.rotate(bad[0], qw, cos, sin, pos, eps)
    assert torch.equal(outs[1].isnan(), want.isnan()) and (outs[1][~want.isnan()].abs() < INF).all()
    asked = torch.zeros(rows, hq, dtype=torch.bool)
    asked[:, :hkv] = hit
    assert torch.equal(outs[1][~asked], outs[0][~asked])
