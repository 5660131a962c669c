"""The 8-bit cache and drawn tokens without a GPU: the C entries' refusals before any launch, the
pool's sizes and refusals, and the oracle's own properties."""

from __future__ import annotations

import math

import pytest
import torch

from helios_amd import _capi, ops
from helios_amd.config import Qwen3Config
from helios_amd.paged_cache import KVPagePool, PackedBatchCache, PagedKVCache
from oracle import kv8 as oracle

MIB = 1 << 20
BAD, NOT, WORK = _capi.HX_E_INVALID_ARG, _capi.HX_E_UNSUPPORTED, _capi.HX_E_WORKSPACE


def test_append_refusals():
    lib = _capi.lib()
    base = [MIB, 2 * MIB, 3 * MIB, 4 * MIB, 4, 256, 8, 128, 0, 5 * MIB, 1024, 128, 6 * MIB, 1024, 128, 7 * MIB, 1, 0, None]

    def call(**kw):
        args = list(base)
        for at, value in kw.items():
            args[int(at[1:])] = value
        return lib.hx_kv8_append(*args)

    assert call(_7=120) == NOT and call(_7=264) == NOT and call(_8=2) == NOT and call(_17=2) == NOT
    assert call(_4=0) == BAD and call(_6=0) == BAD and call(_16=-1) == BAD
    assert call(_0=MIB + 8) == BAD and call(_2=None) == BAD and call(_15=None) == BAD
    assert call(_16=0) == _capi.HX_OK
    assert call(_16=1 << 40) == NOT  # a launch of more work-items than the hardware counts


def test_norm_rope_append_refusals():
    lib = _capi.lib()
    base = [MIB, 4096, 128, 2 * MIB, 1024, 128, 3 * MIB, 1024, 128, 4 * MIB, 5 * MIB, 6 * MIB, 7 * MIB, 100, 8 * MIB, 1,
            32, 8, 128, 1e-6, 0, 9 * MIB, 4096, 128, 10 * MIB, 11 * MIB, 12 * MIB, 13 * MIB, 4, 256, 1, 14 * MIB, None]

    def call(**kw):
        args = list(base)
        for at, value in kw.items():
            args[int(at[1:])] = value
        return lib.hx_kv8_norm_rope_append(*args)

    assert call(_18=40) == NOT and call(_20=2) == NOT and call(_30=7) == NOT
    assert call(_13=0) == BAD and call(_19=-1.0) == BAD and call(_19=math.nan) == BAD and call(_16=0) == BAD
    assert call(_9=4 * MIB + 4) == BAD and call(_11=6 * MIB + 8) == BAD and call(_31=None) == BAD
    assert call(_15=0) == _capi.HX_OK


def test_gather_refusals():
    lib = _capi.lib()

    def call(heads=8, d=128, code=0, pages=2, length=300, dtype=0, out=4 * MIB):
        return lib.hx_kv8_gather(MIB, 2 * MIB, 4, 256, heads, d, code, 3 * MIB, pages, length, dtype, out, None)

    assert call(d=100) == NOT and call(code=3) == NOT and call(dtype=5) == NOT
    assert call(length=513) == BAD and call(length=-1) == BAD and call(out=4 * MIB + 8) == BAD
    assert call(length=0, out=None) == _capi.HX_OK


def test_attention_refusals():
    lib = _capi.lib()
    size = lib.hx_kv8_attn_workspace_bytes
    assert size(64, 64, 1, 4096, 32, 8, 128, 256) > 0
    assert size(0, 0, 0, 0, 32, 8, 128, 256) > 0
    for bad in ((1, 1, 1, 1, 30, 8, 128, 256), (1, 1, 1, 1, 32, 8, 72, 256), (1, 1, 1, 1, 32, 8, 272, 256), (1, 1, 1, 1, 32, 8, 128, 96),
                (1, 1, 1, 1, 258, 2, 128, 256), (-1, 1, 1, 1, 32, 8, 128, 256), (1, 1, 1, 0x7fffffff, 32, 8, 128, 256)):
        assert size(*bad) == 0, bad
    need = size(2, 5, 4, 1000, 32, 8, 128, 256)

    def plan(batch=2, d=128, ws=256 * MIB, nbytes=need, used=2 * MIB, width=4):
        return lib.hx_kv8_attn_plan(MIB, used, batch, 5, 4, 1000, 32, 8, d, 256, width, -1, 0, ws, nbytes, None)

    assert plan(ws=None) == WORK and plan(ws=256 * MIB + 16) == WORK and plan(nbytes=need - 1) == WORK
    assert plan(d=24) == NOT and plan(used=None) == BAD and plan(width=0) == BAD and plan(batch=-1) == BAD
    assert plan(batch=0, ws=None) == _capi.HX_OK

    def run(q=MIB, q_row=4096, out=8 * MIB, out_row=4096, stride=4, scale=0.1, dtype=0, code=0, pages=9, ws=256 * MIB, nbytes=need,
            k_scale=4 * MIB):
        return lib.hx_kv8_attn_run(q, q_row, 128, 2 * MIB, 3 * MIB, k_scale, 5 * MIB, pages, 256, code, 6 * MIB, stride, 4, 2, 5,
                                   4, 1000, 32, 8, 128, scale, -1, 0, dtype, out, out_row, 128, 3, ws, nbytes, None)

    assert run(q=MIB + 8) == BAD and run(q_row=4097) == BAD and run(out=8 * MIB + 2) == BAD and run(out_row=4095) == BAD
    assert run(stride=3) == BAD and run(scale=0.0) == BAD and run(scale=math.nan) == BAD and run(scale=math.inf) == BAD
    assert run(dtype=2) == NOT and run(code=9) == NOT and run(pages=0) == BAD and run(k_scale=4 * MIB + 4) == BAD
    assert run(ws=None) == WORK and run(nbytes=need - 1) == WORK


def test_sample_refusals():
    lib = _capi.lib()
    size = lib.hx_sample_workspace_bytes
    assert size(4, 1000) > 0 and size(0, 10) == 0 and size(1, (1 << 18) + 1) == 0

    def call(rows=4, vocab=1000, dtype=0, logits=MIB, stride=1000, u=2 * MIB, ids=3 * MIB, ws=4 * MIB, nbytes=size(4, 1000)):
        return lib.hx_sample_tokens(logits, stride, rows, vocab, dtype, u, None, None, None, None, ids, None, ws, nbytes, None)

    assert call(dtype=3) == NOT and call(vocab=(1 << 18) + 1, stride=1 << 20) == NOT and call(rows=(1 << 20) + 1) == NOT
    assert call(vocab=0) == BAD and call(stride=999) == BAD and call(logits=MIB + 1) == BAD and call(u=None) == BAD
    assert call(logits=MIB + 2, dtype=2) == BAD and call(ids=None) == BAD
    assert call(ws=None) == WORK and call(ws=4 * MIB + 4) == WORK and call(nbytes=100) == WORK
    assert call(rows=0, logits=None) == _capi.HX_OK


def test_pool_sizes_and_refusals():
    config = Qwen3Config(n_layers=2)
    pool = KVPagePool(config, 3, device="meta", kv_dtype=torch.float8_e4m3fn)
    assert pool.keys[1].shape == (3, 256, 8, 128) and pool.keys[0].dtype == torch.float8_e4m3fn
    assert pool.key_scales[0].shape == pool.value_scales[1].shape == (3, 8, 256)
    assert pool.bytes_per_token == 2 * 2 * 8 * (128 + 4) and pool.bytes_per_page == 256 * pool.bytes_per_token
    assert isinstance(pool.kv8(1), ops.Kv8Cache)
    assert KVPagePool(config, 3, device="meta").bytes_per_token == 2 * 2 * 8 * 128 * 2
    for kw, text in ((dict(kv_dtype=torch.uint8), "float8_e4m3fn or int8"), (dict(kv_dtype=torch.int8, block_size=64), "16-bit")):
        with pytest.raises(ValueError, match=text):
            KVPagePool(config, 3, device="meta", **kw)
    for bad in (dict(head_dim=40), dict(dtype=torch.float32), dict(n_heads=256, n_kv_heads=1)):
        with pytest.raises(ValueError, match="8-bit pool needs"):
            KVPagePool(Qwen3Config(n_layers=1, **bad), 3, device="meta", kv_dtype=torch.int8)
    small = Qwen3Config(n_layers=1, context_length=512)
    pool = KVPagePool(small, 4, device="cpu", kv_dtype=torch.int8)
    batch = PackedBatchCache([PagedKVCache(pool, 512)])
    batch.prepare_packed([3])  # the bookkeeping works without a GPU
    q, k = torch.zeros(1, 32, 3, 128, dtype=torch.bfloat16), torch.zeros(1, 8, 3, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm device only"):
        batch.attend(0, q, k, k)
    with pytest.raises(ValueError, match="8-bit pool"):
        PackedBatchCache([PagedKVCache(pool, 512)], prefix_cascade=True)


def test_oracle_quantise():
    """Codes are within half a step of their rows, and a code's own value comes back as itself."""
    g = torch.Generator().manual_seed(0)
    for code in (torch.float8_e4m3fn, torch.int8):
        x = torch.randn(200, 64, generator=g) * torch.exp(4 * torch.randn(200, 1, generator=g))
        codes, scales = oracle.quantise(x, code)
        back = codes.to(torch.float32).double() * scales.double()[:, None]
        top = x.abs().amax(dim=1, keepdim=True).double()
        step = top / 254 if code == torch.int8 else torch.maximum(x.abs().double() * 2.0 ** -4, top / 448 * 2.0 ** -10)
        assert ((back - x.double()).abs() <= step * (1 + 2.0 ** -20)).all()
        again, _ = oracle.quantise(back.float(), code)
        assert torch.equal(again.view(torch.uint8), codes.view(torch.uint8))


def test_oracle_sample():
    """Shares of the weights, in order of falling logit."""
    logits = torch.tensor([[0.0, math.log(3.0), math.log(4.0), -math.inf]]).expand(8, -1)
    u = torch.tensor([0.0, 0.49, 0.51, 0.86, 0.88, 0.99, 1.0, -1.0])
    ids, logs = oracle.sample(logits, u)
    assert ids.tolist() == [2, 2, 1, 1, 0, 0, 0, 2]
    assert torch.allclose(logs.exp(), torch.tensor([4.0, 4, 3, 3, 1, 1, 1, 4], dtype=torch.float64) / 8, rtol=1e-6)
    assert oracle.sample(logits, u, top_k=torch.full((8,), 1))[0].tolist() == [2] * 8
    assert oracle.sample(logits, u, top_p=torch.full((8,), 0.6))[0].tolist() == [2, 2, 2, 1, 1, 1, 1, 2]
    assert oracle.sample(logits, u, min_p=torch.full((8,), 0.75))[0].tolist() == [2, 2, 2, 1, 1, 1, 1, 2]
    assert oracle.sample(logits, u, temperature=torch.zeros(8))[0].tolist() == [2] * 8


def test_attention_refuses_more_tiles_than_the_plan_counts():
    """Sequences of few rows are dealt by their 32-key tiles, counted in 32 bits: 2^16 sequences of up to
    2^20 keys are 2^31 of them."""
    lib = _capi.lib()
    size = lib.hx_kv8_attn_workspace_bytes
    for batch, max_k in ((1 << 16, 1 << 20), (1 << 20, 1 << 16), (40, 0x7ffffd00), (1 << 28, 1)):
        assert size(batch, batch, 1, max_k, 1, 1, 16, 256) == 0
        assert lib.hx_kv8_attn_plan(MIB, 2 * MIB, batch, batch, 1, max_k, 1, 1, 16, 256, 1 << 20, -1, 0, 256 * MIB, 1 << 60,
                                    None) == NOT
    assert size((1 << 16) - 64, 1 << 16, 1, 1 << 20, 1, 1, 16, 256) > 0 and size(31, 31, 1, 0x7ffffd00, 1, 1, 16, 256) > 0
