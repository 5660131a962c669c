"""Logit rules against their definition row by row: rounding, slices' edges, masks that leave
a row empty, ties, repeated and foreign ids, aliasing."""

from __future__ import annotations

import math

import pytest
import torch

from helios_amd import ops
from oracle import decode_ops as oracle
from tests.gpu_cases import say

pytestmark = pytest.mark.gpu


def _rules(rows, vocab, history, n_bias, masked, seed):
    g = torch.Generator().manual_seed(seed)
    tokens = (torch.rand(rows, history, generator=g) ** 3 * (vocab + 1)).to(torch.int32) - int(history > 3)
    lengths = torch.randint(0, history + 1, (rows,), generator=g, dtype=torch.int32)
    prompt = (lengths * torch.rand(rows, generator=g)).to(torch.int32)
    bias = torch.randint(-1, vocab + 1, (rows, n_bias), generator=g, dtype=torch.int32)
    if n_bias > 2:
        bias[:, 2] = bias[:, 0]  # listed twice
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g).to(torch.int32) if masked else None
    if masked:
        allowed[0] = 0
    return ops.LogitRules(
        tokens=tokens, lengths=lengths, prompt_lens=prompt, repetition=0.7 + torch.rand(rows, generator=g),
        presence=torch.randn(rows, generator=g), frequency=torch.randn(rows, generator=g),
        bias_ids=bias if n_bias else None, bias_values=torch.randn(rows, n_bias, generator=g) * 4 if n_bias else None,
        allowed=allowed)


def _to(rules, device):
    return ops.LogitRules(*(None if t is None else t.to(device) for t in rules))


def _bits(rules, r, vocab):
    if rules.allowed is None:
        return None
    word = rules.allowed[r].long()
    return ((word[:, None] >> torch.arange(32)) & 1).flatten()[:vocab].bool()


def _check(got, logits, rules):
    """Five fp32 roundings of intermediates at most, then the type's own half step."""
    rows, vocab = logits.shape
    out, ids = got.logits.cpu(), got.token_ids.cpu()
    assert out.dtype == logits.dtype and ids.dtype == torch.int64 and ids.shape == (rows,)
    for r in range(rows):
        known = rules.tokens[r, :int(rules.lengths[r])].tolist()
        bias = [] if rules.bias_ids is None else list(zip(rules.bias_ids[r].tolist(),
                                                          rules.bias_values[r].double().tolist()))
        p = [float(rules.repetition[r]), float(rules.presence[r]), float(rules.frequency[r])]
        allowed = _bits(rules, r, vocab)
        ref = oracle.logit_rules(logits[r], known, int(rules.prompt_lens[r]), *p, bias, allowed)
        fine = torch.isfinite(ref)
        assert torch.equal(out[r][~fine].double(), ref[~fine])
        size = logits[r].double().abs() * (1 + p[0] + 1 / p[0]) + abs(p[1]) + abs(p[2]) * (1 + len(known)) \
            + max([abs(x) for _, x in bias], default=0.0)
        off = 5 * 2.0 ** -24 * size[fine] + torch.finfo(logits.dtype).eps / 2 * ref[fine].abs() * (1 + 2.0 ** -20)
        assert ((out[r][fine].double() - ref[fine]).abs() <= off).all()
        usable = torch.ones(vocab, dtype=torch.bool) if allowed is None else allowed
        if not usable.any():
            assert ids[r] == -1
            continue
        top = out[r].double().masked_fill(~usable, -math.inf)
        assert ids[r] == int((usable & (top == top.max())).nonzero()[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,history,n_bias,masked", [
    (1, 1, 1, 1, False), (3, 31, 5, 3, True), (2, 4096, 300, 0, True), (5, 4097, 1000, 9, True),
    (2, 50257, 700, 300, False), (4, 12288, 4000, 64, True)])
def test_logit_rules(device, rows, vocab, history, n_bias, masked, dtype):
    say("logit rules", rows, vocab, history, n_bias, masked, dtype)
    rules = _rules(rows, vocab, history, n_bias, masked, seed=vocab + rows)
    logits = (3 * torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab))).to(dtype)
    on = _to(rules, device)
    got = ops.apply_logit_rules(logits.to(device), on)
    _check(got, logits, rules)
    alone = ops.apply_logit_rules(logits.to(device), on, return_logits=False)
    assert alone.logits is None and torch.equal(alone.token_ids, got.token_ids)
    place = logits.to(device)
    again = ops.apply_logit_rules(place, on, out=place)
    assert again.logits is place and torch.equal(place, got.logits) and torch.equal(again.token_ids, got.token_ids)


@pytest.mark.parametrize("vocab", [1000, 8191])
def test_rows_inside_wider_rows(device, vocab):
    """Logits and tables whose rows lie in wider ones, at addresses no vector load may take: the
    columns behind a row stay as they were."""
    say("logit rules strides", vocab)
    rules = _rules(3, vocab, 50, 4, True, seed=vocab)
    wide = torch.randn(3, vocab + 13, device=device).to(torch.bfloat16)
    on = _to(rules, device)
    want = ops.apply_logit_rules(wide[:, 5:5 + vocab].contiguous(), on)
    tables = on._replace(**{n: torch.cat((getattr(on, n), getattr(on, n)), 1)[:, :getattr(on, n).shape[1]]
                            for n in ("tokens", "bias_ids", "bias_values", "allowed")})
    before = wide.clone()
    got = ops.apply_logit_rules(wide[:, 5:5 + vocab], tables, out=wide[:, 5:5 + vocab])
    assert torch.equal(got.logits, want.logits) and torch.equal(got.token_ids, want.token_ids)
    assert torch.equal(wide[:, :5], before[:, :5]) and torch.equal(wide[:, 5 + vocab:], before[:, 5 + vocab:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_rules_ties_and_special_values(device, dtype):
    """Without rules the logits come back bit for bit, and the ids are torch.argmax's."""
    say("logit rules special", dtype)
    inf, nan = float("inf"), float("nan")
    rows = [[0.0, -0.0, -1.0], [-0.0, 0.0, -1.0], [-inf, -inf, -inf], [1.0, nan, inf], [-inf, 2.0, 2.0], [nan, nan, 1.0]]
    logits = torch.tensor(rows).to(dtype).to(device)
    got = ops.apply_logit_rules(logits, ops.LogitRules())
    assert torch.equal(got.logits.view(torch.uint8), logits.view(torch.uint8))
    assert got.token_ids.tolist() == [0, 0, 0, 1, 1, 0]
    # An infinity or NaN that is not allowed does not come through.
    allowed = torch.tensor([[4]] * 6, dtype=torch.int32, device=device)
    got = ops.apply_logit_rules(logits, ops.LogitRules(allowed=allowed))
    assert got.token_ids.tolist() == [2] * 6
    assert torch.equal(got.logits[:, :2], torch.full_like(logits[:, :2], -inf))
    # Ties far apart: the first slice's, and the first within a row of equal logits.
    flat = torch.zeros(2, 9000, dtype=dtype, device=device)
    flat[1, [4095, 4096, 8999]] = 7
    assert ops.apply_logit_rules(flat, ops.LogitRules()).token_ids.tolist() == [0, 4095]


def test_lengths_beyond_the_table(device):
    """Lengths past the table are its width, negative ones 0; a prompt longer than the known
    tokens leaves nothing said."""
    say("logit rules lengths")
    logits = torch.ones(3, 40, device=device)
    tokens = torch.arange(30, dtype=torch.int32, device=device).view(1, 30).repeat(3, 1)
    rules = ops.LogitRules(
        tokens=tokens[:, :10], lengths=torch.tensor([100, -5, 10], dtype=torch.int32, device=device),
        prompt_lens=torch.tensor([0, 0, 99], dtype=torch.int32, device=device),
        repetition=torch.full((3,), 2.0, device=device), presence=torch.full((3,), 0.25, device=device))
    got = ops.apply_logit_rules(logits, rules).logits.cpu()
    assert got[0].tolist() == [0.25] * 10 + [1.0] * 30
    assert got[1].tolist() == [1.0] * 40
    assert got[2].tolist() == [0.5] * 10 + [1.0] * 30


@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_long_histories_and_bias_lists(device, shift):
    """More tokens and biases than a workgroup takes at once, token rows at every offset from a
    16-byte address."""
    say("logit rules long", shift)
    rules = _rules(3, 5000, 20001, 1300, True, seed=shift)
    rules = rules._replace(lengths=torch.tensor([20001, 8193 + shift, 2047], dtype=torch.int32))
    logits = torch.randn(3, 5000, generator=torch.Generator().manual_seed(shift)).to(torch.bfloat16)
    on = _to(rules, device)
    wide = torch.zeros(3, 20004 + shift, dtype=torch.int32, device=device)
    wide[:, shift:shift + 20001] = on.tokens
    on = on._replace(tokens=wide[:, shift:shift + 20001])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.apply_logit_rules(logits.to(device), on)
    torch.cuda.current_stream().wait_stream(side)
    _check(got, logits, rules)


def test_rows_past_32_bits(device):
    """A row that begins beyond 2^31 elements from the first."""
    say("logit rules far rows")
    wide = torch.empty(2 ** 31 + 8192, dtype=torch.bfloat16, device=device)
    far = wide.as_strided((2, 3000), (2 ** 31 + 24, 1), 40)
    rules = _rules(2, 3000, 40, 5, False, seed=9)
    logits = torch.randn(2, 3000, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    far.copy_(logits)
    _check(ops.apply_logit_rules(far, _to(rules, device), out=far), logits, rules)


def test_logit_rules_in_two_graphs(device):
    """Two captured calls of one pool of memory, replayed in turn with eager calls between."""
    say("logit rules graphs")
    logits = torch.randn(4, 9000, device=device).to(torch.bfloat16)
    rules = _to(_rules(4, 9000, 100, 8, True, seed=1), device)
    ops.apply_logit_rules(logits, rules)
    graphs, outs = [], []
    for part in (slice(0, 4), slice(1, 3)):
        on = ops.LogitRules(*(None if t is None else t[part].contiguous() for t in rules))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append((ops.apply_logit_rules(logits[part], on), on, part))
        graphs.append(graph)
    for seed in range(3):
        logits.copy_(torch.randn(4, 9000, generator=torch.Generator().manual_seed(seed)))
        for graph, (got, on, part) in zip(graphs, outs):
            graph.replay()
            want = ops.apply_logit_rules(logits[part], on)
            assert torch.equal(got.logits, want.logits) and torch.equal(got.token_ids, want.token_ids)


def test_logit_rules_refusals(device):
    logits = torch.zeros(2, 64, device=device)
    i32 = dict(dtype=torch.int32, device=device)
    tokens, lengths = torch.zeros(2, 5, **i32), torch.zeros(2, **i32)
    L = ops.LogitRules
    bad = [
        (logits.double(), L(), {}), (logits[0], L(), {}), (logits.t(), L(), {}), (logits[:1].expand(2, 64), L(), {}),
        (logits, L(tokens=tokens), {}), (logits, L(lengths=lengths), {}),
        (logits, L(repetition=torch.ones(2, device=device)), {}),
        (logits, L(tokens=tokens.long(), lengths=lengths), {}),
        (logits, L(tokens=tokens, lengths=lengths, repetition=torch.ones(3, device=device)), {}),
        (logits, L(tokens=tokens, lengths=lengths.cpu()), {}),
        (logits, L(bias_ids=tokens), {}),
        (logits, L(bias_ids=tokens, bias_values=torch.zeros(2, 4, device=device)), {}),
        (logits, L(allowed=torch.zeros(2, 1, **i32)), {}), (logits, L(allowed=torch.zeros(1, 2, **i32)), {}),
        (logits, L(), dict(out=logits.half())), (logits, L(), dict(out=logits[:, :32])),
    ]
    for x, rules, kw in bad:
        with pytest.raises(ValueError):
            ops.apply_logit_rules(x, rules, **kw)
    with pytest.raises(RuntimeError):
        ops.apply_logit_rules(logits.cpu(), L())
    assert ops.apply_logit_rules(logits[:0], L()).token_ids.shape == (0,)
