"""Timed cases of the operators of a long-context decode tick: 4-bit products, attention over
selected blocks of the paged cache, and the rules a request puts on its logits.

Five kinds of case:

``bounds``  ``ops.kv_block_bounds``: the elementwise lowest and highest key of every block that
            a tick's new tokens touched, per KV head.
``select``  ``ops.select_blocks``: the blocks that a query row's heads attend to, by an upper
            bound of their scores.
``sparse``  ``ops.block_sparse_attn``: attention of query rows over their selected blocks.
``int4``    ``ops.int4_linear``: a product with 4-bit weights and group scales, with RMSNorm
            before it and SwiGLU or a residual after it.
``rules``   ``ops.apply_logit_rules``: penalties, biases and allowed-token masks on the logits,
            and the greedy token ids.

Head shapes, widths and lengths are those of Qwen3-4B (32 query / 8 KV heads of 128, hidden
2560, ffn 9728, vocabulary 151936, pages of 256 tokens) unless the case says otherwise. Lengths
follow from the case; page placement and every value from the seed.
"""

from __future__ import annotations

import math
import random

import torch

PAGE = 256
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"
EPS = 1e-6

own = False  # the plain form (torch operations) or the framework's calls


# ------------------------------------------------------------------------- the cases
def listed():
    return [
        # The decode tick of a busy server: every request adds a token to its last block.
        dict(name="bounds_64_decoders", kind="bounds", dtype="bf16", hkv=8, d=128, block=64, decoders=64, lo=512,
             hi=4096, chunks="", lens=1),
        # Prompts prefilled in chunks, some of which begin and end inside a block; fp16 model.
        dict(name="bounds_chunks_fp16", kind="bounds", dtype="fp16", hkv=8, d=128, block=64, decoders=3, lo=700,
             hi=2000, chunks="4096@8192,2048@0,1001@333", lens=2),
        # One user with a book in the context: latency.
        dict(name="select_1_long", kind="select", dtype="bf16", hq=32, hkv=8, d=128, block=64, rows=1, lo=131000,
             hi=131000, budget=64, sink=1, recent=2, lens=3),
        # Long-document questions, a full batch.
        dict(name="select_64_decoders", kind="select", dtype="bf16", hq=32, hkv=8, d=128, block=64, rows=64, lo=16384,
             hi=40960, budget=64, sink=1, recent=2, lens=4),
        # One user: 2048 of 20000 keys.
        dict(name="sparse_1_decoder", kind="sparse", dtype="bf16", hq=32, hkv=8, d=128, block=64, rows=1, seqs=1,
             lo=20000, hi=20000, budget=32, lens=5),
        # A full batch with 4096 keys each, at 8000 to 16384 cached.
        dict(name="sparse_64_decoders", kind="sparse", dtype="bf16", hq=32, hkv=8, d=128, block=64, rows=64, seqs=64,
             lo=8000, hi=16384, budget=64, lens=6),
        # Another model's heads, small blocks, and drafted tokens: three rows to a sequence.
        dict(name="sparse_drafts_fp16", kind="sparse", dtype="fp16", hq=16, hkv=4, d=64, block=16, rows=21, seqs=7,
             lo=900, hi=9000, budget=96, lens=7),
        # The projections of one decoding request: the smallest product, latency.
        dict(name="int4_1_row_qkv", kind="int4", dtype="bf16", rows=1, cols=6144, k=2560, group=128, norm=True,
             form="plain"),
        # The gated half of the feed-forward block at eight requests.
        dict(name="int4_8_rows_gate_up", kind="int4", dtype="bf16", rows=8, cols=9728, k=2560, group=128, norm=True,
             form="swiglu"),
        # The way back to the residual stream at a full batch, finer groups.
        dict(name="int4_64_rows_down", kind="int4", dtype="fp16", rows=64, cols=2560, k=9728, group=64, norm=False,
             form="residual"),
        # A few chats: penalties over what they said, a bias list.
        dict(name="rules_4_rows", kind="rules", dtype="bf16", rows=4, vocab=151936, history=1500, bias=40,
             masked=False),
        # A full tick with structured output: long histories, biases, a grammar mask for every row.
        dict(name="rules_129_rows_masked", kind="rules", dtype="bf16", rows=129, vocab=151936, history=8192, bias=300,
             masked=True),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["bounds", "select", "sparse", "sparse", "int4", "int4", "rules"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    lens = rng.randrange(1 << 20)
    if kind == "bounds":
        form = rng.choice(["decode", "chunks", "mixed"])
        decoders = 0 if form == "chunks" else _log(rng, 1, 128)
        hi = _log(rng, 16, 8192)
        chunks = [] if form == "decode" else [
            "%d@%d" % (_log(rng, 2, 2048), rng.choice([0, _log(rng, 1, 8192)])) for _ in range(rng.randint(1, 3))]
        hkv, d = rng.choice([(8, 128), (8, 128), (4, 64), (1, 256), (2, 96), (1, 8)])
        return dict(kind=kind, dtype=dtype, hkv=hkv, d=d, block=rng.choice([16, 64, 64, 128, 256]), decoders=decoders,
                    lo=_log(rng, 1, hi), hi=hi, chunks=",".join(chunks), lens=lens)
    if kind in ("select", "sparse"):
        hq, hkv, d = rng.choice([(32, 8, 128), (32, 8, 128), (16, 4, 64), (12, 4, 96), (16, 1, 256), (8, 8, 128),
                                 (64, 4, 128), (2, 1, 8)])
        block = rng.choice([16, 64, 64, 128, 256])
        rows = _log(rng, 1, 64)
        if kind == "select":
            # More blocks than the budget takes, and some of that free to choose.
            hi = _log(rng, 24 * block, max(24 * block, min(65536, 700000 // rows)))
            lo = _log(rng, max(24 * block, hi // 6), hi)
            return dict(kind=kind, dtype=dtype, hq=hq, hkv=hkv, d=d, block=block, rows=rows, lo=lo, hi=hi,
                        budget=_log(rng, 6, lo // block // 2), sink=rng.randint(0, 1), recent=rng.randint(1, 2),
                        lens=lens)
        hi = _log(rng, 1, min(65536, 700000 // rows))
        lo = _log(rng, max(1, hi // 6), hi)
        budget = _log(rng, 3, max(4, 4096 // block))
        return dict(kind=kind, dtype=dtype, hq=hq, hkv=hkv, d=d, block=block, rows=rows,
                    seqs=max(1, rows // rng.choice([1, 1, 3])), lo=lo, hi=hi, budget=budget, lens=lens)
    if kind == "int4":
        cols, k = rng.choice([(6144, 2560), (2560, 4096), (9728, 2560), (2560, 9728), (4096, 4096), (1000, 576),
                              (16 * rng.randint(1, 300), 128 * rng.randint(1, 60)), (rng.randint(1, 3000), 2048)])
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 64), cols=cols, k=k,
                    group=rng.choice([128, 64, 32]) if k % 128 == 0 else 64 if k % 64 == 0 else 32,
                    norm=rng.random() < 0.5, form=rng.choice(["plain", "residual", "swiglu"]))
    return dict(kind="rules", dtype=rng.choice([dtype, "fp32"]), rows=_log(rng, 1, 96),
                vocab=rng.choice([151936, 151669, 32000, 50257, _log(rng, 500, 130000)]), history=_log(rng, 1, 8192),
                bias=rng.choice([0, _log(rng, 1, 300)]), masked=rng.random() < 0.5)


# ---------------------------------------------------------------- lengths and page tables
def _ticks(case):
    """(cached, new) tokens of every sequence: decoders, then chunks."""
    rng = random.Random(case["lens"])
    cached, new = [], []
    for _ in range(case["decoders"]):
        cached.append(rng.randint(case["lo"], case["hi"]) - 1)
        new.append(1)
    for part in filter(None, case["chunks"].split(",")):
        n, at = part.split("@")
        cached.append(int(at))
        new.append(int(n))
    return cached, new


def _key_counts(case):
    """Visible keys of every row, and the rows' sequences: drafted rows are consecutive positions."""
    rng = random.Random(case["lens"])
    seqs = case.get("seqs", case["rows"])
    ends = [rng.randint(case["lo"], case["hi"]) for _ in range(seqs)]
    of = [r * seqs // case["rows"] for r in range(case["rows"])]
    keys = [max(0, ends[s] - (sum(q == s for q in of[r + 1:]))) for r, s in enumerate(of)]
    return keys, of, ends


def _table(lengths, seed):
    """Page ids that cover each sequence, from one seeded permutation: [sequences, width], and
    the pool's pages. Entries past a sequence's pages are page 0."""
    need = [-(-n // PAGE) for n in lengths]
    order = list(range(sum(need) or 1))
    random.Random(seed).shuffle(order)
    table = torch.zeros((len(need), max(1, *need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, len(order)


def _blocks_of(case, keys, seed):
    """Selected blocks [rows, kv heads, budget], ascending, -1 behind them: the first block, the
    last two and random ones between, as a selection gives them."""
    g = torch.Generator().manual_seed(seed)
    count = torch.tensor([-(-n // case["block"]) for n in keys])
    most = int(count.max())
    budget = case["budget"]
    score = torch.rand((len(keys), case["hkv"], most), generator=g)
    at = torch.arange(most)
    last = count[:, None, None]
    score = torch.where((at == 0) | (at >= last - 2), score + 1, score).masked_fill(at >= last, -1)
    if most < budget:
        score = torch.nn.functional.pad(score, (0, budget - most), value=-1.0)
    top, index = score.topk(budget, dim=-1)
    index = index.masked_fill(top < 0, 1 << 30).sort(dim=-1).values
    return index.masked_fill(index == 1 << 30, -1).to(torch.int32)


# ----------------------------------------------------------------------------- prepare
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    state = dict(case=case, dtype=dt)

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype) * std

    def ints(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=DEVICE)

    if case["kind"] == "bounds":
        cached, new = _ticks(case)
        ends = [c + n for c, n in zip(cached, new)]
        table, pages = _table(ends, seed)
        h, d = case["hkv"], case["d"]
        state["k_pool"] = normal(pages, PAGE, h, d) + normal(h, d)  # keys have a mean of their own
        state["bounds"] = normal(pages, PAGE // case["block"], h, 2, d)
        state["table"] = table.to(DEVICE)
        state["cu_q"] = ints([0] + [sum(new[:i + 1]) for i in range(len(new))])
        state["used"] = ints(ends)
        state["max_q"] = max(new)
        return state

    if case["kind"] in ("select", "sparse"):
        keys, of, ends = _key_counts(case)
        table, pages = _table(ends, seed)
        state["table"] = table.to(DEVICE)
        state["keys"] = ints(keys)
        state["row_seq"] = None if of == list(range(len(of))) and len(ends) == len(of) else ints(of)
        h, d = case["hkv"], case["d"]
        state["q"] = normal(case["rows"], case["hq"], d)
        if case["kind"] == "select":
            # Bounds of 'block' keys each: the extremes of normal values, around the block's mean.
            mean = normal(pages, PAGE // case["block"], h, 1, d, std=0.5)
            half = 1.5 + 0.5 * normal(pages, PAGE // case["block"], h, 1, d).abs()
            state["bounds"] = torch.cat((mean - half, mean + half), dim=3)
            return state
        state["k_pool"] = normal(pages, PAGE, h, d)
        state["v_pool"] = normal(pages, PAGE, h, d)
        state["blocks"] = _blocks_of(case, keys, seed).to(DEVICE)
        return state

    if case["kind"] == "int4":
        n, k, group = case["cols"] * (2 if case["form"] == "swiglu" else 1), case["k"], case["group"]
        # Normal weights, quantised: most values lie around the zero point.
        values = (normal(n, k, dtype=torch.float32) * 3.2 + 8).round().clamp(0, 15).to(torch.uint8)
        scales = ((0.5 + torch.rand((k // group, n), generator=g, device=DEVICE)) * (0.3 * k ** -0.5)).to(dt)
        zeros = torch.randint(6, 11, (k // group, n), generator=g, device=DEVICE, dtype=torch.uint8)
        state["x"] = normal(case["rows"], k)
        state["norm"] = 1 + 0.1 * normal(k, dtype=torch.float32) if case["norm"] else None
        state["residual"] = normal(case["rows"], case["cols"]) if case["form"] == "residual" else None
        if own:
            from helios_amd import ops

            state["weight"] = ops.int4_pack(values, scales, zeros)
        else:  # two values to a byte, as they lie in a file
            state["packed"], state["scales"], state["zeros"] = values[:, ::2] | values[:, 1::2] << 4, scales, zeros
        return state

    rows, vocab = case["rows"], case["vocab"]
    state["logits"] = normal(rows, vocab, std=3.0)
    # Token ids are far from uniform: a few thousand make up most of a text.
    length = case["history"]
    ids = torch.rand((rows, length), generator=g, device=DEVICE) ** 4 * vocab
    state["tokens"] = ids.to(torch.int32).clamp_(0, vocab - 1)
    rng = random.Random(seed)
    lengths = [rng.randint(max(1, length // 4), length) for _ in range(rows)]
    state["lengths"] = ints(lengths)
    state["prompt_lens"] = ints([rng.randint(0, n) for n in lengths])
    state["repetition"] = 1 + torch.rand(rows, generator=g, device=DEVICE) * 0.5
    state["presence"] = torch.rand(rows, generator=g, device=DEVICE) * 2
    state["frequency"] = torch.rand(rows, generator=g, device=DEVICE)
    state["bias_ids"] = state["bias_values"] = state["allowed"] = None
    if case["bias"]:
        # Every id of a row once; ids past a row's own list are -1.
        step = max(1, vocab // case["bias"])
        at = torch.arange(case["bias"], device=DEVICE) * step
        at = at + torch.randint(0, step, (rows, case["bias"]), generator=g, device=DEVICE)
        used = torch.rand((rows, case["bias"]), generator=g, device=DEVICE) < 0.8
        state["bias_ids"] = torch.where(used & (at < vocab), at, -1).to(torch.int32)
        state["bias_values"] = normal(rows, case["bias"], std=4.0, dtype=torch.float32)
    if case["masked"]:
        # A grammar leaves some rows few tokens and others half of them.
        words = -(-vocab // 32)
        bits = torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device=DEVICE)
        keep = torch.rand((rows, words), generator=g, device=DEVICE) < torch.rand((rows, 1), generator=g, device=DEVICE)
        state["allowed"] = torch.where(keep, bits, 0).to(torch.int32)
    return state


# --------------------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    return (_own if own else _plain)[kind](state)


def _own_bounds(s):
    from helios_amd import ops

    ops.kv_block_bounds(s["k_pool"], s["bounds"], s["table"], s["cu_q"], s["used"], max_q=s["max_q"])
    return s["bounds"]


def _own_select(s):
    from helios_amd import ops

    c = s["case"]
    return ops.select_blocks(s["q"], s["bounds"], s["table"], s["keys"], c["budget"], block_size=c["block"],
                             sink=c["sink"], recent=c["recent"], row_seq=s["row_seq"])


def _own_sparse(s):
    from helios_amd import ops

    return ops.block_sparse_attn(s["q"], s["k_pool"], s["v_pool"], s["blocks"], s["table"], s["keys"],
                                 block_size=s["case"]["block"], row_seq=s["row_seq"])


def _own_int4(s):
    from helios_amd import ops

    return ops.int4_linear(s["x"], s["weight"], norm_weight=s["norm"], eps=EPS, residual=s["residual"],
                           swiglu=s["case"]["form"] == "swiglu")


def _own_rules(s):
    from helios_amd import ops

    rules = ops.LogitRules(tokens=s["tokens"], lengths=s["lengths"], prompt_lens=s["prompt_lens"],
                           repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                           bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"])
    got = ops.apply_logit_rules(s["logits"], rules)
    return got.logits, got.token_ids


_own = dict(bounds=_own_bounds, select=_own_select, sparse=_own_sparse, int4=_own_int4, rules=_own_rules)


def _plain_bounds(s):
    """lower / upper[block, head, d] = min / max over the block's keys so far."""
    block, used, bounds = s["case"]["block"], s["used"].long(), s["bounds"]
    per_page = PAGE // block
    first = (used - (s["cu_q"][1:] - s["cu_q"][:-1])) // block
    last = (used - 1) // block
    at = first[:, None] + torch.arange((s["max_q"] - 1) // block + 2, device=DEVICE)
    at = torch.minimum(at, last[:, None])  # a block named twice is written twice, alike
    page = s["table"].long().gather(1, at // per_page)
    pos = at[..., None] * block + torch.arange(block, device=DEVICE)
    keys = s["k_pool"].view(-1, block, *s["k_pool"].shape[2:])[page * per_page + at % per_page].float()
    seen = (pos < used[:, None, None])[..., None, None]
    low = keys.masked_fill(~seen, math.inf).amin(dim=2)
    high = keys.masked_fill(~seen, -math.inf).amax(dim=2)
    flat = bounds.view(-1, *bounds.shape[2:])
    flat[page * per_page + at % per_page] = torch.stack((low, high), dim=3).to(bounds.dtype)
    return bounds


def _plain_select(s):
    """score = sum over the group's heads and dims of max(q lower, q upper), in 64 bits: blocks
    at the border of the selection lie close together."""
    c = s["case"]
    block, budget, keys = c["block"], c["budget"], s["keys"].long()
    rows, hkv, d = s["q"].shape[0], c["hkv"], c["d"]
    bounds = s["bounds"].view(-1, hkv, 2, d)
    table = s["table"].long() if s["row_seq"] is None else s["table"].long()[s["row_seq"].long()]
    per_page = PAGE // block
    most = table.shape[1] * per_page
    at = torch.arange(most, device=DEVICE)
    q = s["q"].double().view(rows, hkv, -1, d)
    weight = torch.stack((q.clamp(max=0).sum(2), q.clamp(min=0).sum(2)), dim=2)  # of lower, of upper
    ids = table[:, at // per_page] * per_page + at % per_page
    score = (bounds[ids].double() * weight[:, None]).sum(dim=(3, 4)).transpose(1, 2)
    count = ((keys + block - 1) // block)[:, None, None]
    kept = (at < c["sink"]) | (at >= count - c["recent"])
    score = torch.where(kept, math.inf, score).masked_fill(at >= count, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    if most < budget:
        order = torch.nn.functional.pad(order, (0, budget - most), value=most)
    order = torch.where(order < count, order, 1 << 30).sort(dim=-1).values
    return torch.where(order == 1 << 30, -1, order).to(torch.int32)


def _plain_sparse(s):
    """softmax(q k / sqrt(d)) v over the keys of the row's selected blocks."""
    c = s["case"]
    block, blocks, keys = c["block"], s["blocks"].long(), s["keys"].long()
    rows, hkv, d = s["q"].shape[0], c["hkv"], c["d"]
    table = s["table"].long() if s["row_seq"] is None else s["table"].long()[s["row_seq"].long()]
    pos = blocks.clamp(min=0)[..., None] * block + torch.arange(block, device=DEVICE)
    seen = ((blocks[..., None] >= 0) & (pos < keys[:, None, None, None])).flatten(2)
    pos = torch.where(seen, pos.flatten(2), 0)
    page = table.gather(1, (pos // PAGE).flatten(1)).view_as(pos)
    slot = page * PAGE + pos % PAGE
    head = torch.arange(hkv, device=DEVICE)[:, None]
    k = s["k_pool"].view(-1, hkv, d)[slot, head].float()
    v = s["v_pool"].view(-1, hkv, d)[slot, head].float()
    q = s["q"].float().view(rows, hkv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    p = torch.exp(score - score.amax(dim=-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return out.reshape(rows, -1, d).to(s["dtype"])


def _plain_int4(s):
    """y = h W^T, W = scale (value - zero) by groups along k, h = x or its RMSNorm."""
    c, packed = s["case"], s["packed"]
    n, k, group = packed.shape[0], c["k"], c["group"]
    values = torch.stack((packed & 15, packed >> 4), dim=2).view(n, k // group, group).float()
    w = (values - s["zeros"].t().float()[..., None]) * s["scales"].t().float()[..., None]
    x = s["x"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + EPS) * s["norm"]
    y = x @ w.view(n, k).t()
    if c["form"] == "swiglu":
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1 + torch.exp(-gate)) * up
    if s["residual"] is not None:
        y = s["residual"].float() + y
    return y.to(s["dtype"])


def _plain_rules(s):
    """l / r or l r where a token was seen, - frequency count - presence, + bias; -inf where not
    allowed; the greedy ids of what is returned, -1 for a row that nothing is allowed in."""
    logits, tokens = s["logits"], s["tokens"].long()
    rows, vocab = logits.shape
    at = torch.arange(tokens.shape[1], device=DEVICE)
    known = at < s["lengths"][:, None]
    said = known & (at >= s["prompt_lens"][:, None])
    seen = torch.zeros((rows, vocab), device=DEVICE).scatter_add_(1, tokens, known.float()) > 0
    count = torch.zeros((rows, vocab), device=DEVICE).scatter_add_(1, tokens, said.float())
    x = logits.float()
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(count > 0, x - (s["frequency"][:, None] * count + s["presence"][:, None]), x)
    if s["bias_ids"] is not None:
        ids = s["bias_ids"].long()
        extra = torch.zeros((rows, vocab + 1), device=DEVICE)
        extra.scatter_(1, torch.where(ids < 0, vocab, ids), s["bias_values"])
        x = x + extra[:, :vocab]
    top = x.to(s["dtype"])
    if s["allowed"] is None:
        return top, top.argmax(dim=-1)
    at = torch.arange(vocab, device=DEVICE)
    allowed = (s["allowed"][:, at // 32] >> (at % 32).to(torch.int32)) & 1 != 0
    top = top.masked_fill(~allowed, -math.inf)
    best = allowed & (top == top.amax(dim=-1, keepdim=True))
    return top, torch.where(best.any(dim=-1), best.to(torch.uint8).argmax(dim=-1), -1)


_plain = dict(bounds=_plain_bounds, select=_plain_select, sparse=_plain_sparse, int4=_plain_int4, rules=_plain_rules)


# -------------------------------------------------------------------------------- work
def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind == "bounds":
        cached, new = _ticks(case)
        block, row = case["block"], case["hkv"] * case["d"] * size
        keys = sum(c + n - c // block * block for c, n in zip(cached, new))
        touched = sum((c + n - 1) // block - c // block + 1 for c, n in zip(cached, new))
        return dict(bytes=keys * row + touched * 2 * row, flops=2 * keys * row / size)
    if kind in ("select", "sparse"):
        keys, of, _ = _key_counts(case)
        row = case["hkv"] * case["d"]
        q = case["rows"] * case["hq"] * case["d"]
        counts = [-(-n // case["block"]) for n in keys]
        if kind == "select":
            # Drafted rows share their sequence's bounds.
            reads = sum({s: n for s, n in zip(of, counts)}.values())
            picks = case["rows"] * case["hkv"] * case["budget"]
            return dict(bytes=reads * 2 * row * size + q * size + picks * 4, flops=4 * sum(counts) * row)
        # Every row has blocks of its own, each head others: they share nothing.
        seen = sum(min(n, case["budget"] * case["block"]) for n in keys)
        return dict(bytes=2 * seen * row * size + 2 * q * size + case["rows"] * case["hkv"] * case["budget"] * 4,
                    flops=4 * seen * case["hq"] * case["d"])
    if kind == "int4":
        n = case["cols"] * (2 if case["form"] == "swiglu" else 1)
        weight = n * case["k"] // 2 + n * (case["k"] // case["group"]) * (size + 1)
        rows = case["rows"] * (case["k"] + case["cols"] * (2 if case["form"] == "residual" else 1)) * size
        return dict(bytes=weight + rows, flops=2 * case["rows"] * n * case["k"])
    rows, vocab = case["rows"], case["vocab"]
    return dict(bytes=rows * (2 * vocab * size + (vocab // 8 if case["masked"] else 0) + case["history"] * 5 // 8 * 4
                              + case["bias"] * 8), flops=4 * rows * vocab)


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    """What run returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return dict(bounds=_exact_bounds, select=_exact_select, sparse=_exact_sparse, int4=_exact_int4,
                rules=_exact_rules)[case["kind"]](case, s)


def _exact_bounds(case, s):
    cached, new = _ticks(case)
    out = s["bounds"].double()
    table, block = s["table"].tolist(), case["block"]
    for b, (c, n) in enumerate(zip(cached, new)):
        for j in range(c // block, (c + n - 1) // block + 1):
            page, at = table[b][j * block // PAGE], j * block % PAGE
            keys = s["k_pool"][page, at:at + min(block, c + n - j * block)].double()
            out[page, at // block, :, 0] = keys.min(dim=0).values
            out[page, at // block, :, 1] = keys.max(dim=0).values
    return out


def _exact_select(case, s):
    keys, of, _ = _key_counts(case)
    table, block = s["table"].long(), case["block"]
    out = torch.full((case["rows"], case["hkv"], case["budget"]), -1, dtype=torch.int32)
    group = case["hq"] // case["hkv"]
    for r, n in enumerate(keys):
        count = -(-n // block)
        if not count:
            continue
        of_row = s["bounds"][table[of[r]]].flatten(0, 1)[:count].double()
        q = s["q"][r].double().view(case["hkv"], group, 1, case["d"])
        both = q * of_row[:, :, 0].transpose(0, 1)[:, None], q * of_row[:, :, 1].transpose(0, 1)[:, None]
        score = torch.maximum(*both).sum(dim=(1, 3))
        score[:, :case["sink"]] = math.inf
        score[:, max(0, count - case["recent"]):] = math.inf
        take = min(count, case["budget"])
        order = (-score).argsort(dim=-1, stable=True)[:, :take].sort(dim=-1).values
        out[r, :, :take] = order.to(torch.int32).cpu()
    return out


def _exact_sparse(case, s):
    keys, of, _ = _key_counts(case)
    blocks, table = s["blocks"].long(), s["table"].long()
    block, group = case["block"], case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for r, n in enumerate(keys):
        for h in range(case["hkv"]):
            pos = blocks[r, h][blocks[r, h] >= 0][:, None] * block + torch.arange(block, device=DEVICE)
            pos = pos[pos < n]
            if not pos.numel():
                continue
            page = table[of[r]][pos // PAGE]
            k, v = (s[p][page, pos % PAGE, h].double() for p in ("k_pool", "v_pool"))
            heads = slice(h * group, (h + 1) * group)
            out[r, heads] = torch.softmax(s["q"][r, heads].double() @ k.t() / case["d"] ** 0.5, dim=-1) @ v
    return out


def _exact_int4(case, s):
    n, k, group = case["cols"] * (2 if case["form"] == "swiglu" else 1), case["k"], case["group"]
    values = torch.empty((n, k), dtype=torch.float64, device=DEVICE)
    values[:, 0::2] = (s["packed"] % 16).double()
    values[:, 1::2] = (s["packed"] // 16).double()
    w = (values - s["zeros"].double().repeat_interleave(group, dim=0).t()) \
        * s["scales"].double().repeat_interleave(group, dim=0).t()
    x = s["x"].double()
    if case["norm"]:
        x = x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / k + EPS) * s["norm"].double()
    y = torch.mm(x, w.t().contiguous())
    if case["form"] == "swiglu":
        y = torch.nn.functional.silu(y[:, :case["cols"]]) * y[:, case["cols"]:]
    return y + s["residual"].double() if case["form"] == "residual" else y


def _exact_rules(case, s):
    out = s["logits"].double()
    for r in range(case["rows"]):
        n, p, row = int(s["lengths"][r]), int(s["prompt_lens"][r]), out[r]
        known = s["tokens"][r, :n].long().unique()
        rep = s["repetition"][r].double()
        row[known] = torch.where(row[known] > 0, row[known] / rep, row[known] * rep)
        said, count = s["tokens"][r, p:n].long().unique(return_counts=True)
        row[said] -= s["frequency"][r].double() * count + s["presence"][r].double()
        if case["bias"]:
            keep = s["bias_ids"][r] >= 0
            row[s["bias_ids"][r][keep].long()] += s["bias_values"][r][keep].double()
        if case["masked"]:
            word = s["allowed"][r].long() & 0xffffffff
            bit = (word[:, None] >> torch.arange(32, device=DEVICE)) & 1
            row[bit.flatten()[:case["vocab"]] == 0] = -math.inf
    return out, None
