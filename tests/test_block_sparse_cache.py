"""Host side of block-sparse attention: pools with key bounds and the settings that are refused
(no GPU work)."""

from __future__ import annotations

import pytest
import torch

from helios_amd.config import Qwen3Config
from helios_amd.decoder import PagedQwen3Decoder
from helios_amd.paged_cache import BlockSparse, KVPagePool, PackedBatchCache, PagedKVCache


def _config(**change):
    base = dict(vocab_size=64, context_length=2048, hidden_size=32, n_heads=2, n_layers=2, hidden_dim=64, head_dim=8,
                n_kv_heads=1, dtype=torch.bfloat16)
    return Qwen3Config(**{**base, **change})


def test_pool_with_bounds():
    pool = KVPagePool(_config(), 3, device="cpu", block_size=64)
    assert len(pool.bounds) == 2
    for layer in pool.bounds:
        assert layer.shape == (3, 4, 1, 2, 8) and layer.is_contiguous() and layer.dtype == torch.bfloat16
    assert KVPagePool(_config(), 3, device="cpu").bounds is None
    assert pool.bytes_per_token == KVPagePool(_config(), 3, device="cpu").bytes_per_token


@pytest.mark.parametrize("block", [0, 8, 48, 512, 2048, -16])
def test_pool_refuses_block_sizes(block):
    with pytest.raises(ValueError):
        KVPagePool(_config(), 3, device="cpu", block_size=block)


@pytest.mark.parametrize("change", [dict(dtype=torch.float32), dict(head_dim=12), dict(head_dim=264)])
def test_pool_refuses_heads_without_bounds(change):
    with pytest.raises(ValueError):
        KVPagePool(_config(**change), 3, device="cpu", block_size=64)


@pytest.mark.parametrize("args", [(2, 1, 2), (4, -1, 2), (4, 1, 0), (0, 0, 1)])
def test_budgets(args):
    with pytest.raises(ValueError):
        BlockSparse(*args)


def test_batches_need_bounds_and_few_enough_blocks():
    plain, pool = (KVPagePool(_config(), 3, device="cpu", block_size=b) for b in (None, 64))
    with pytest.raises(ValueError, match="bounds"):
        PackedBatchCache([PagedKVCache(plain, 512)], sparse=BlockSparse(8))
    batch = PackedBatchCache([PagedKVCache(pool, 512)], sparse=BlockSparse(8))
    batch.prepare_packed([300])  # bookkeeping runs without a device
    batch.advance_packed()
    long = KVPagePool(_config(context_length=16 * 16384 + 1), 3, device="cpu", block_size=16)
    with pytest.raises(ValueError, match="16384"):
        PackedBatchCache([PagedKVCache(long, 512)], sparse=BlockSparse(8))


def test_refresh_bounds_refusals():
    plain, pool = (KVPagePool(_config(), 3, device="cpu", block_size=b) for b in (None, 64))
    with pytest.raises(RuntimeError, match="no key bounds"):
        PagedKVCache(plain, 512).refresh_bounds()
    cache = PagedKVCache(pool, 512)
    cache.refresh_bounds()  # nothing committed, nothing to do
    PackedBatchCache([cache]).prepare_packed([3])
    with pytest.raises(RuntimeError, match="in flight"):
        cache.refresh_bounds()


def test_decoder_weight_bits():
    with pytest.raises(ValueError):
        PagedQwen3Decoder(_config(), "cpu", weight_bits=8)
    with pytest.raises(ValueError):  # hidden 32 does not divide into groups of 128
        PagedQwen3Decoder(_config(), "cpu", weight_bits=4)
    with pytest.raises(ValueError):  # nor do the heads' 16 elements into groups of 32
        PagedQwen3Decoder(_config(), "cpu", weight_bits=4, group_size=32)
    model = PagedQwen3Decoder(_config(head_dim=16), "cpu", weight_bits=4, group_size=32)
    assert model.layers[0]["qkv"].rows == 64 and model.layers[0]["down"].k == 64
