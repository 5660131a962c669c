"""The operators of a long-context decode tick as the cache and the decoder use them: key bounds
under every append, sparse and mixed ticks, 4-bit products, logit rules, and all of them in
one run of ticks."""

from __future__ import annotations

import math

import pytest
import torch

from helios_amd import ops
from helios_amd.config import Qwen3Config
from helios_amd.decoder import PagedQwen3Decoder
from helios_amd.paged_cache import BlockSparse, KVPagePool, PackedBatchCache, PagedBatchCache, PagedKVCache
from oracle import decode_ops as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu


def _config(**change):
    base = dict(vocab_size=1000, context_length=4096, hidden_size=256, n_heads=8, n_layers=2, hidden_dim=512,
                n_kv_heads=2, dtype=torch.bfloat16)
    return Qwen3Config(**{**base, **change})


def _filled(config, device, lengths, block_size, seed=4, pages=40):
    """A pool of random keys and values with requests of these lengths, bounds refreshed."""
    pool = KVPagePool(config, pages, device=device, block_size=block_size)
    g = torch.Generator(device=device).manual_seed(seed)
    for t in pool.keys + pool.values:
        t.normal_(generator=g)
    caches = []
    for n in lengths:
        cache = PagedKVCache(pool, config.context_length)
        cache.pages.extend(pool.acquire(-(-n // 256)))
        cache.length = n
        if block_size is not None:
            cache.refresh_bounds()
        caches.append(cache)
    return pool, caches


def _expect_bounds(pool, caches):
    """Every block of every request holds the bounds of its keys."""
    for layer in range(pool.config.n_layers):
        k, got = pool.keys[layer].cpu(), pool.bounds[layer].cpu()
        for cache in caches:
            table = torch.tensor([[p.index for p in cache.pages]])
            want = oracle.block_bounds(k, got, table, [0], [cache.length])
            assert torch.equal(got.double(), want)


def _rows(config, tokens, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)

    def make(heads):
        return torch.randn(1, heads, tokens, config.head_dim, generator=g, device=device).to(config.dtype)

    return make(config.n_heads), make(config.n_kv_heads), make(config.n_kv_heads)


@pytest.mark.parametrize("kw", [dict(), dict(device_metadata=False), dict(overlap=True), dict(sparse=BlockSparse(4))])
def test_every_append_keeps_the_bounds(device, kw):
    """attend (fused, with an unaligned K, under a cascade), attend_projected and a uniform batch."""
    say("bounds under appends", kw.keys())
    config = _config()
    pool, caches = _filled(config, device, [300, 511, 64], 64)
    batch = PackedBatchCache(caches, **kw)
    for tick, counts in enumerate([[1, 1, 1], [70, 1, 1], [1, 1, 200]]):
        batch.prepare_packed(counts)
        for layer in range(config.n_layers):
            q, k, v = _rows(config, sum(counts), tick * 7 + layer, device)
            if tick == 1:
                k = torch.cat((k, k), -1)[..., 1:129]  # rows no 16-byte load may take
            batch.attend(layer, q, k, v)
        batch.advance_packed()
    model = PagedQwen3Decoder(config, device, seed=1, std=0.05)
    batch.prepare_packed([1, 5, 1])
    model.forward_packed(torch.randint(0, 1000, (1, 7), device=device), batch)
    _expect_bounds(pool, caches)
    uniform = PagedBatchCache(caches, **kw)
    uniform.prepare(1)
    for layer in range(config.n_layers):
        q, k, v = _rows(config, 3, layer, device)
        uniform.attend(layer, *(t[0].transpose(0, 1).unsqueeze(2) for t in (q, k, v)))
    uniform.advance(1)
    _expect_bounds(pool, caches)


def test_shared_prefix_copies_and_truncation(device):
    """A restored prefix has its bounds, shared or copied; tokens forgotten and written anew leave
    no trace."""
    say("bounds of restored pages")
    config = _config()
    pool, caches = _filled(config, device, [600], 64)
    blocks = [caches[0].snapshot_block(0, 512)]
    for kw in (dict(), dict(copy=True), dict(private_tail=True)):
        cache = PagedKVCache(pool, config.context_length)
        cache.restore_blocks(blocks, **kw)
        if kw:
            cache.truncate(450)
        batch = PackedBatchCache([cache], sparse=BlockSparse(4))
        batch.prepare_packed([1])
        for layer in range(config.n_layers):
            batch.attend(layer, *_rows(config, 1, layer, device))
        batch.advance_packed()
        caches.append(cache)
    _expect_bounds(pool, caches)
    caches[0].truncate(520)
    batch = PackedBatchCache([caches[0]])
    batch.prepare_packed([9])
    for layer in range(config.n_layers):
        batch.attend(layer, *_rows(config, 9, 30 + layer, device))
    batch.advance_packed()
    _expect_bounds(pool, caches)


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [1, 40, 1, 3]])
def test_sparse_ticks(device, counts):
    """Decode rows attend to their selections, chunk rows and short rows to everything."""
    say("sparse ticks", counts)
    config = _config(head_dim=64)
    pool, caches = _filled(config, device, [2000, 700, 100, 1500], 64)
    sparse = BlockSparse(6, sink=1, recent=2)
    batch = PackedBatchCache(caches, sparse=sparse)
    batch.prepare_packed(counts)
    q, k, v = _rows(config, sum(counts), 3, device)
    got = batch.attend(0, q, k, v)[0].transpose(0, 1)
    batch.advance_packed()
    table = batch.block_table.cpu()
    kc, vc, bounds, qc = pool.keys[0].cpu(), pool.values[0].cpu(), pool.bounds[0].cpu(), q[0].transpose(0, 1).cpu()
    start = 0
    for b, n in enumerate(counts):
        for i in range(n):
            keys = caches[b].length - n + i + 1
            count, row = -(-keys // 64), start + i
            lists = []
            for h in range(2):
                if n > 1 or count <= sparse.budget:
                    lists.append(list(range(count)))
                else:
                    scores = oracle.block_scores(qc[row], bounds, table[b], count, h, 4)
                    lists.append(oracle.select(scores, count, sparse.budget, 1, 2))
            ref = oracle.sparse_attention(qc[row:row + 1], kc, vc, torch.tensor([lists]), table, [keys], [b], 64, 0.125)
            # the chunk rows' kernel keeps its weights in 24 bits, the sparse one in 16
            tol = 2.0 ** -8 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -14 * vc.double().abs().max()
            assert ((got[row].double().cpu() - ref[0]).abs() <= tol).all(), (b, i)
        start += n


def test_sparse_budget_above_the_cache_changes_nothing(device):
    """No row has more blocks than the budget: the tick is the dense one, bit for bit."""
    say("sparse budget above")
    outs = []
    for sparse in (None, BlockSparse(64)):
        config = _config()
        _, caches = _filled(config, device, [2000, 700], 64)
        batch = PackedBatchCache(caches, sparse=sparse)
        batch.prepare_packed([1, 1])
        outs.append(batch.attend(0, *_rows(config, 2, 3, device)))
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("rows", [3, 40, 90])
def test_int4_decoder_matches_its_dequantised_weights(device, rows):
    """The 4-bit decoder against one that holds the same values in 16 bits: fused products for few
    rows, dequantised ones for many."""
    say("int4 decoder", rows)
    config = _config()
    model = PagedQwen3Decoder(config, device, seed=3, std=0.05, weight_bits=4, group_size=64)
    dense = PagedQwen3Decoder(config, device, seed=3, std=0.05)
    for layer, of in zip(dense.layers, model.layers):
        for name in ("qkv", "o", "gate_up", "down"):
            layer[name] = ops.int4_dequantize(of[name])
    ids = torch.randint(0, 1000, (1, rows + 1), generator=torch.Generator().manual_seed(rows)).to(device)
    logits = []
    for m, kw in ((model, {}), (dense, dict(fused_rope=False)), (model, dict(fused_rope=False))):
        _, caches = _filled(config, device, [300, 30], None)
        batch = PackedBatchCache(caches)
        batch.prepare_packed([rows, 1])
        logits.append(m.forward_packed(ids, batch, **kw).float())
    # as between the 16-bit sequences: products in other orders and roundings, two layers
    scale = max(logits[1].abs().max().item(), 1.0)
    assert (logits[0] - logits[1]).abs().max().item() <= 2e-2 * scale
    # the same sequence of operations on the same values
    assert torch.equal(logits[2], logits[1])


def test_rules_in_the_decoder(device):
    """The logits and ids of a tick with rules are its logits, then the rules: on the fused heads
    and on the library's."""
    say("decoder rules")
    config = _config()
    model = PagedQwen3Decoder(config, device, seed=2, std=0.05)
    g = torch.Generator().manual_seed(1)
    rules = ops.LogitRules(
        tokens=torch.randint(0, 1000, (3, 20), generator=g, dtype=torch.int32).to(device),
        lengths=torch.tensor([20, 3, 0], dtype=torch.int32, device=device),
        repetition=torch.full((3,), 1.3, device=device), presence=torch.full((3,), 0.5, device=device),
        allowed=torch.tensor([[-1] * 32, [0] * 32, [0, 6] + [0] * 30], dtype=torch.int32, device=device))
    ids = torch.randint(0, 1000, (1, 7), generator=g).to(device)
    for kw in (dict(), dict(fused_rope=False)):
        outs = []
        for more in (dict(), dict(rules=rules), dict(rules=rules, greedy=True)):
            _, caches = _filled(config, device, [300, 30, 5], None)
            batch = PackedBatchCache(caches)
            batch.prepare_packed([1, 5, 1])
            outs.append(model.forward_packed(ids, batch, **kw, **more))
        want = ops.apply_logit_rules(outs[0], rules)
        assert torch.equal(outs[1], want.logits) and torch.equal(outs[2], want.token_ids)
        assert outs[2][1] == -1 and int(outs[2][2]) in (33, 34)


def test_ticks_with_all_of_them(device, monkeypatch):
    """A 4-bit decoder on long caches with a sparse budget and rules, four ticks: every call that
    the ticks make of the operators is right for what it was given, and each greedy id is the
    best allowed one, with what was said fed back."""
    say("all together")
    calls = {}

    def spy(name):
        real = getattr(ops, name)

        def wrapped(*args, **kw):
            keep = [a.clone() if isinstance(a, torch.Tensor) else a for a in args]
            got = real(*args, **kw)
            calls.setdefault(name, []).append((keep, dict(kw), got))
            return got
        monkeypatch.setattr(ops, name, wrapped)

    for name in ("int4_linear", "select_blocks", "block_sparse_attn", "apply_logit_rules"):
        spy(name)
    config = _config()
    model = PagedQwen3Decoder(config, device, seed=5, std=0.05, weight_bits=4, group_size=128)
    pool, caches = _filled(config, device, [1900, 1100, 60], 64)
    batch = PackedBatchCache(caches, sparse=BlockSparse(5, sink=1, recent=1))
    history = torch.full((3, 8), -1, dtype=torch.int32, device=device)
    allowed = torch.full((3, 32), -1, dtype=torch.int32, device=device)
    allowed[1, 2:] = 0
    ids = torch.tensor([[3, 5, 7]], device=device)
    for tick in range(4):
        history[:, tick] = ids[0].to(torch.int32)
        rules = ops.LogitRules(
            tokens=history, lengths=torch.full((3,), tick + 1, dtype=torch.int32, device=device),
            repetition=torch.full((3,), 1.2, device=device), frequency=torch.full((3,), 0.8, device=device),
            allowed=allowed)
        batch.prepare_packed([1, 1, 1])
        ids = model.forward_packed(ids, batch, greedy=True, rules=rules).view(1, 3)
        assert int(ids[0, 1]) < 64
    _expect_bounds(pool, caches)
    assert [len(calls[n]) for n in ("int4_linear", "select_blocks", "block_sparse_attn", "apply_logit_rules")] \
        == [4 * 2 * 4, 8, 8, 4]

    for (x, w), kw, got in calls["int4_linear"]:
        m = ops.int4_dequantize(w).double()  # bf16 values of 8-bit scales: within half a step each
        h = x.double()
        norm = kw.get("norm_weight")
        if norm is not None:
            h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + config.rms_norm_eps) * norm.double()
        y = h @ m.t()
        off = 2.0 ** -8 * (h.abs() @ m.abs().t())  # the 16-bit values' own rounding
        if kw.get("swiglu"):
            (gate, up), (go, uo) = y.chunk(2, -1), off.chunk(2, -1)
            y, off = gate * torch.sigmoid(gate) * up, 1.1 * go * (up.abs() + uo) + (gate.abs() + go) * uo
        if kw.get("residual") is not None:
            y = y + kw["residual"].double()
        assert ((got.double() - y).abs() <= off + 2.0 ** -8 * y.abs() * (1 + 2.0 ** -8) + 1e-6).all()
    for (q, bounds, table, keys, budget), kw, got in calls["select_blocks"]:
        q, bounds, table = q.cpu(), bounds.cpu(), table.cpu()
        for b, n in enumerate(keys.tolist()):
            count = -(-n // 64)
            for h in range(2):
                scores = oracle.block_scores(q[b], bounds, table[b], count, h, 4)
                assert got[b, h].tolist() == oracle.select(scores, count, budget, 1, 1)
    for (q, k, v, blocks, table, keys), kw, got in calls["block_sparse_attn"]:
        ref = oracle.sparse_attention(q.cpu(), k.cpu(), v.cpu(), blocks.cpu(), table.cpu(), keys.tolist(), range(3), 64,
                                      config.head_dim ** -0.5)
        tol = 2.0 ** -8 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -14 * v.double().abs().max().item()
        assert ((got.double().cpu() - ref).abs() <= tol).all()
    for tick, ((logits, rules), _, got) in enumerate(calls["apply_logit_rules"]):
        for r in range(3):
            # the history buffer has grown since: its first columns are this tick's
            bits = ((allowed[r].cpu().long()[:, None] >> torch.arange(32)) & 1).flatten()[:1000].bool()
            known = history[r, :tick + 1].tolist()
            ref = oracle.logit_rules(logits[r].cpu(), known, 0, float(rules.repetition[r]), 0.0,
                                     float(rules.frequency[r]), [], bits)
            top = ref.max()
            pick = ref[int(got.token_ids[r])]
            assert math.isfinite(float(pick)) and pick >= top - 2.0 ** -7 * top.abs() - 1e-6


def test_norm_rows_of_a_mixed_int4_tick(device):
    """A tick of more rows than int4_linear takes, then one of fewer, on one cache: the keys the
    first wrote are those the second reads (values equal to the reference sequence's)."""
    say("int4 mixed ticks")
    config = _config()
    model = PagedQwen3Decoder(config, device, seed=7, std=0.05, weight_bits=4)
    outs = []
    for fused in (True, False):
        _, caches = _filled(config, device, [700, 20], 64)
        batch = PackedBatchCache(caches)
        g = torch.Generator().manual_seed(3)
        for counts in ([1, 100], [1, 1]):
            batch.prepare_packed(counts)
            ids = torch.randint(0, 1000, (1, sum(counts)), generator=g).to(device)
            out = model.forward_packed(ids, batch, fused_rope=fused)
        outs.append(out.float())
    assert (outs[0] - outs[1]).abs().max() <= 2e-2 * max(outs[1].abs().max().item(), 1.0)
