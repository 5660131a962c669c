"""Attention over the 8-bit cache at head dims past 128, in every type, with rows of each kind and sequences
cut into few and many parts."""

from __future__ import annotations

import pytest
import torch

from tests.gpu_cases import say
from tests.test_gpu_kv8 import CODES, DTYPES, _attend, _pool
from tests.test_gpu_kv8_special import _close, _lengths

pytestmark = pytest.mark.gpu

# hq, hkv, page, (cached, new) per sequence
TICKS = [
    (8, 2, 64, [(8999, 1), (1500, 1), (0, 1), (63, 2), (900, 4)]),          # few rows in 12, 2 and no parts
    (16, 1, 128, [(2000, 1), (700, 30), (4000, 90), (0, 70), (127, 5)]),    # chunks beside them
    (3, 3, 256, [(6000, 17), (255, 129), (1, 40)]),                         # chunks alone
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("tick", range(len(TICKS)))
@pytest.mark.parametrize("d", [144, 176, 192, 240, 256])
def test_wide_heads(device, d, tick, code, dtype):
    hq, hkv, page, seqs = TICKS[tick]
    say("kv8 wide heads", d, TICKS[tick], code, dtype)
    cu, used = _lengths(seqs)
    cache, table = _pool([c + n for c, n in seqs], page, hkv, d, code, seed=d + tick)
    q = torch.randn(int(cu[-1]), hq, d, generator=torch.Generator().manual_seed(d)).to(dtype)
    lens = [n for _, n in seqs]
    for window in ((-1, 0), (1000, 0)):
        plan, got = _attend(device, q, cache, table, cu, used, max(lens), int(used.max()), window, q_lens=lens)
        assert plan.error_word() == 0
        _close(got, q, cache, table, cu, used, window)
