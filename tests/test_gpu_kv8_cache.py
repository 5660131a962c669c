"""The 8-bit pool in the cache classes and the decoder: growing batches, prefix pages, ticks whose
tokens are drawn."""

from __future__ import annotations

import pytest
import torch

from helios_amd import ops
from helios_amd.config import Qwen3Config
from helios_amd.decoder import PagedQwen3Decoder
from helios_amd.paged_cache import BlockSparse, KVPagePool, PackedBatchCache, PagedBatchCache, PagedKVCache
from oracle import kv8 as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu

CODES = [torch.float8_e4m3fn, torch.int8]


def _config(**kw):
    given = dict(vocab_size=1000, context_length=4096, hidden_size=256, n_heads=8, n_kv_heads=2, head_dim=64, n_layers=2,
                 hidden_dim=512, dtype=torch.bfloat16) | kw
    return Qwen3Config(**given)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("device_metadata", [True, False])
def test_growing_batch(device, code, device_metadata):
    """Prompts in chunks, decode ticks and drafted tokens over one pool: every tick's attention is
    that of everything written so far, as its codes stand for."""
    say("kv8 batch", code, device_metadata)
    config = _config()
    pool = KVPagePool(config, 12, device=device, kv_dtype=code)
    caches = [PagedKVCache(pool, 1024) for _ in range(3)]
    batch = PackedBatchCache(caches, device_metadata=device_metadata)
    g = torch.Generator().manual_seed(1)
    for counts in ([300, 5, 1], [1, 1, 1], [3, 60, 1], [1, 300, 2], [1, 1, 1]):
        total = sum(counts)
        q, k, v = (torch.randn(1, h, total, 64, generator=g).to(torch.bfloat16) for h in (8, 2, 2))
        batch.prepare_packed(counts)
        out = batch.attend(1, q.to(device), k.to(device), v.to(device))
        batch.advance_packed()
        cache = ops.Kv8Cache(*(t.cpu() for t in pool.kv8(1)))
        table = torch.zeros(3, 4, dtype=torch.int32)
        for b, c in enumerate(caches):
            table[b, :len(c.pages)] = torch.tensor([p.index for p in c.pages], dtype=torch.int32)
        cu = torch.tensor([0] + counts).cumsum(0)
        used = torch.tensor([c.length for c in caches])
        keys, vals = oracle.values(cache.keys, cache.key_scales), oracle.values(cache.values, cache.value_scales)
        # What was just stored is the definition's codes.
        for x, pool_codes, pool_scales in ((k, cache.keys, cache.key_scales), (v, cache.values, cache.value_scales)):
            codes, scales = oracle.quantise(x[0].transpose(0, 1), code)
            at = torch.cat([torch.arange(c.length - n, c.length) for c, n in zip(caches, counts)])
            of = torch.repeat_interleave(torch.arange(3), torch.tensor(counts))
            page = table[of, at // 256].long()
            assert torch.equal(pool_codes.view(torch.uint8)[page, at % 256], codes.view(torch.uint8))
            assert torch.equal(pool_scales.transpose(1, 2)[page, at % 256], scales)
        rows = q[0].transpose(0, 1)
        want, mag, _, _ = oracle.attention(rows, keys, vals, table, cu, used, (-1, 0), 1 / 8)
        got = out[0].transpose(0, 1).double().cpu()
        # One rounding of the output (2^-8), weights within 2^-11 and what their scores are off by.
        assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * mag + 2.0 ** -20).all()


def test_attend_projected_matches_the_operators(device):
    """attend_projected over requests of one length is norms, rotation, append and attention."""
    say("kv8 attend projected")
    config = _config(n_heads=16, n_kv_heads=4, head_dim=128)
    pool = KVPagePool(config, 6, device=device, kv_dtype=torch.float8_e4m3fn)
    caches = [PagedKVCache(pool, 512) for _ in range(2)]
    batch = PagedBatchCache(caches)
    model = PagedQwen3Decoder(config, device, seed=0)
    g = torch.Generator(device=device).manual_seed(2)
    own = ops.Kv8Cache(*(torch.zeros_like(t) for t in pool.kv8(0)))
    for t in own:
        (t if t.dtype == torch.float32 else t.view(torch.uint8)).zero_()
    w = 1 + 0.1 * torch.randn(128, generator=g, device=device)
    start = 0
    for tokens in (40, 1, 3):
        q, k, v = (torch.randn(2, tokens, h * 128, generator=g, device=device).to(torch.bfloat16) for h in (16, 4, 4))
        batch.prepare(tokens)
        out = batch.attend_projected(0, q, k, v, w, w, model.cos, model.sin, 1e-6)
        rot = ops.kv8_norm_rope_append(
            q.view(-1, 16, 128), k.view(-1, 4, 128), v.view(-1, 4, 128), w, w, model.cos, model.sin,
            torch.arange(start, start + tokens, device=device).repeat(2), own, batch.write_slots, 1e-6)
        want = ops.kv8_attn(rot, own, batch.cu_seq_q, batch.seqused_k, batch.block_table, max_q=tokens, max_k=start + tokens,
                            is_causal=True)
        assert out.shape == (2, 16, tokens, 128)
        assert torch.equal(out.transpose(1, 2).reshape(-1, 16, 128), want)
        batch.advance(tokens)
        start += tokens
    with pytest.raises(RuntimeError, match="prepare"):
        batch.attend_projected(0, q, k, v, w, w, model.cos, model.sin, 1e-6)


@pytest.mark.parametrize("code", CODES)
def test_prefix_pages(device, code):
    """A restored prefix, shared, copied or with a private tail, answers as the request it came from;
    a copy's later writes do not reach it."""
    say("kv8 prefix", code)
    config = _config()
    pool = KVPagePool(config, 16, device=device, kv_dtype=code)
    first = PagedKVCache(pool, 1024)
    g = torch.Generator(device=device).manual_seed(3)
    new = lambda n, h: torch.randn(1, h, n, 64, generator=g, device=device).to(torch.bfloat16)  # noqa: E731
    batch = PackedBatchCache([first])
    batch.prepare_packed([512])
    for layer in range(2):
        batch.attend(layer, new(512, 8), new(512, 2), new(512, 2))
    batch.advance_packed()
    block = first.snapshot_block(0, 512)
    assert block.memory_bytes == 2 * pool.bytes_per_page == 2 * 256 * 2 * 2 * 2 * (64 + 4)
    q, k, v = new(1, 8), new(1, 2), new(1, 2)
    outs = []
    for kw in ({}, {"copy": True}, {"private_tail": True}):
        cache = PagedKVCache(pool, 1024)
        cache.restore_blocks([block], **kw)
        if kw:
            cache.truncate(511)  # into a page of its own
        batch = PackedBatchCache([cache])
        batch.prepare_packed([1])
        outs.append(batch.attend(1, q, k, v))
        batch.advance_packed()
        cache.close()
    assert torch.equal(outs[1], outs[2]) and not torch.equal(outs[0], outs[1])
    before = [t.clone() for t in outs[:1]]
    cache = PagedKVCache(pool, 1024)
    cache.restore_blocks([block])
    batch = PackedBatchCache([cache])
    batch.prepare_packed([1])
    assert torch.equal(batch.attend(1, q, k, v), before[0])  # the shared pages are as they were


def _ticks(model, pool, config, device, sampled, steps):
    """Prompts, then decode ticks that feed the drawn tokens back; every tick's result."""
    caches = [PagedKVCache(pool, config.context_length) for _ in range(3)]
    batch = PackedBatchCache(caches)
    g = torch.Generator(device=device).manual_seed(5)
    ids = torch.randint(0, config.vocab_size, (1, 146), generator=g, device=device)
    out = []
    for step in range(steps):
        counts = [5, 140, 1] if step == 0 else [1, 1, 1]
        batch.prepare_packed(counts)
        u = torch.rand(3, generator=g, device=device)
        result = model.forward_packed(ids, batch, **sampled(u))
        if isinstance(result, ops.SampledTokens):
            out.append(result)
        else:
            out.append((result, ops.sample_tokens(result, **sampled(u, True)._asdict())))
            result = out[-1][1]
        ids = result.token_ids[None]
    return out


@pytest.mark.parametrize("code", [None, *CODES])
def test_decoder_draws_its_tokens(device, code):
    """forward_packed(sampling=...) over a 16-bit or 8-bit pool draws what sample_tokens draws from
    the same tick's logits, tick after tick."""
    say("kv8 decoder", code)
    config = _config() if code is not None else _config(head_dim=128)  # what the 16-bit pool's fused append takes
    model = PagedQwen3Decoder(config, device, seed=2, std=0.05)
    full = lambda t: torch.full((3,), t, device=device)  # noqa: E731

    def drawn(u, bare=False):
        s = ops.Sampling(u, temperature=full(0.8), top_k=torch.full((3,), 40, dtype=torch.int32, device=device), top_p=full(0.9))
        return s if bare else dict(sampling=s)

    got = _ticks(model, KVPagePool(config, 8, device=device, kv_dtype=code), config, device, drawn, 4)
    want = _ticks(model, KVPagePool(config, 8, device=device, kv_dtype=code), config, device,
                  lambda u, bare=False: drawn(u, True) if bare else {}, 4)
    for a, (logits, b) in zip(got, want):
        assert logits.shape == (3, 1000) and torch.isfinite(logits).all()
        assert torch.equal(a.token_ids, b.token_ids) and torch.equal(a.logprobs, b.logprobs)
        assert (a.token_ids >= 0).all() and (a.token_ids < 1000).all()
    with pytest.raises(ValueError, match="not both"):
        model.forward_packed(torch.zeros(1, 3, dtype=torch.int64, device=device), None, greedy=True, sampling=drawn(full(0.5), True))


def test_decoder_rules_then_draw(device):
    """Tokens are drawn from the ruled logits: none that is not allowed, -1 where nothing is."""
    say("kv8 decoder rules")
    config = _config()
    model = PagedQwen3Decoder(config, device, seed=2, std=0.05)
    pool = KVPagePool(config, 8, device=device, kv_dtype=torch.int8)
    batch = PackedBatchCache([PagedKVCache(pool, 256) for _ in range(3)])
    allowed = torch.zeros(3, 32, dtype=torch.int32, device=device)
    allowed[0, 5] = 1 << 7   # token 167 alone
    allowed[1, :] = 0x0f
    for u in (0.0, 0.4, 0.999):
        batch.prepare_packed([2, 2, 2])
        got = model.forward_packed(torch.arange(6, device=device)[None], batch, rules=ops.LogitRules(allowed=allowed),
                                   sampling=ops.Sampling(torch.full((3,), u, device=device)))
        ids = got.token_ids.tolist()
        assert ids[0] == 167 and ids[1] % 32 < 4 and ids[2] == -1


def test_eight_bit_ticks_stay_close_to_sixteen(device):
    """One layer's attention from an 8-bit pool against the 16-bit one: keys and values half a step
    off. e4m3: 2^-4 of an element at most; int8: 1/254 of a row's largest."""
    say("kv8 against 16 bits")
    config = _config(n_layers=1)
    g = torch.Generator(device=device).manual_seed(6)
    q = torch.randn(1, 8, 300, 64, generator=g, device=device).to(torch.bfloat16)
    k, v = (torch.randn(1, 2, 300, 64, generator=g, device=device).to(torch.bfloat16) for _ in range(2))
    outs = {}
    for code in (None, *CODES):
        batch = PackedBatchCache([PagedKVCache(KVPagePool(config, 2, device=device, kv_dtype=code), 512)])
        batch.prepare_packed([300])
        outs[code] = batch.attend(0, q, k, v).double()
    for code in CODES:
        # Scores off by |q| |dk| / 8 at most, so weights by e^2x that; values by half a step.
        step = {CODES[0]: 2.0 ** -4 * k.abs().double(), CODES[1]: k.abs().amax(-1, keepdim=True).double() / 254}[code]
        x = (q.abs().double().view(1, 2, 4, 300, 64) @ step.expand_as(k).transpose(2, 3).contiguous()[:, :, None]).amax() / 8
        v_off = {CODES[0]: 2.0 ** -4 * v.abs().max().double(), CODES[1]: v.abs().max().double() / 254}[code]
        bound = torch.expm1(2 * x) * v.abs().max().double() + v_off + 2.0 ** -7 * v.abs().max().double()
        assert (outs[code] - outs[None]).abs().max() <= bound
        assert (outs[code] - outs[None]).norm() <= 0.06 * outs[None].norm()  # and far less where errors average


def test_refusals(device):
    config = _config()
    for kw, text in ((dict(kv_dtype=torch.float8_e5m2), "float8_e4m3fn or int8"), (dict(kv_dtype=torch.int8, block_size=64), "16-bit")):
        with pytest.raises(ValueError, match=text):
            KVPagePool(config, 2, device=device, **kw)
    pool = KVPagePool(config, 2, device=device, kv_dtype=torch.int8)
    cache = PagedKVCache(pool, 256)
    for kw in (dict(overlap=True), dict(prefix_cascade=True)):
        with pytest.raises(ValueError, match="8-bit pool"):
            PackedBatchCache([cache], **kw)
    with pytest.raises(ValueError, match="key bounds"):
        PackedBatchCache([cache], sparse=BlockSparse(4))
    with pytest.raises(RuntimeError, match="kv_dtype"):
        KVPagePool(config, 2, device=device).kv8(0)
