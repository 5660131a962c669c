"""Timed cases of a serving tick over a cache in 8 bits: keys and values quantised as they are
written, attention that reads them, pages read back, and tokens drawn from the logits.

Four kinds of case:

``write``   ``ops.kv8_append``, and ``ops.kv8_norm_rope_append`` with the norms and the position
            rotation of queries and keys in the same pass: a scale for each token and head, 8-bit
            codes into the pages.
``attn``    ``ops.Kv8AttnPlan.run``: attention of a tick's rows (one new token, a few drafted ones,
            chunks of prompts) over the paged 8-bit cache.
``read``    ``ops.kv8_gather``: a sequence's keys from its pages, as one 16-bit tensor.
``sample``  ``ops.sample_tokens``: temperature, top-k, top-p and min-p from given uniform numbers.

Head shapes and lengths are those of Qwen3-4B (32 query / 8 KV heads of 128, vocabulary 151936,
pages of 256 tokens) unless the case says otherwise. Lengths follow from the case; page placement
and every value from the seed.
"""

from __future__ import annotations

import math
import random

import torch

PAGE = 256
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
DEVICE = "cuda"
EPS = 1e-6
LEAST_SCALE = 2.0 ** -100

own = False  # the plain form (torch operations) or the framework's calls


# ------------------------------------------------------------------------- the cases
def listed():
    return [
        # The decode tick of a busy server: 64 new tokens, normalised, rotated and stored.
        dict(name="write_64_decoders", kind="write", rope=True, dtype="bf16", code="e4m3", hq=32, hkv=8, d=128, decoders=64,
             lo=512, hi=4096, chunks="", lens=1),
        # A prompt's chunk behind an earlier one, and a short prompt's.
        dict(name="write_chunks", kind="write", rope=True, dtype="bf16", code="e4m3", hq=32, hkv=8, d=128, decoders=0, lo=1,
             hi=1, chunks="2048@2048,333@0", lens=2),
        # Keys and values that are ready to be stored, another model's heads, whole numbers as codes.
        dict(name="write_ready_int8", kind="write", rope=False, dtype="fp16", code="int8", hq=16, hkv=4, d=64, decoders=32,
             lo=900, hi=2000, chunks="4096@100", lens=3),
        # One user with a long document: latency.
        dict(name="attn_1_decoder", kind="attn", dtype="bf16", code="e4m3", hq=32, hkv=8, d=128, decoders=1, rows=1, lo=32768,
             hi=32768, chunks="", left=-1, lens=4),
        # The decode tick of a busy server.
        dict(name="attn_64_decoders", kind="attn", dtype="bf16", code="e4m3", hq=32, hkv=8, d=128, decoders=64, rows=1,
             lo=512, hi=4096, chunks="", left=-1, lens=5),
        # Another model's heads and codes, three drafted tokens to a sequence.
        dict(name="attn_drafts_fp16_int8", kind="attn", dtype="fp16", code="int8", hq=16, hkv=4, d=64, decoders=16, rows=3,
             lo=900, hi=9000, chunks="", left=-1, lens=6),
        # A mixed tick: 32 decoders beside two prompts' chunks.
        dict(name="attn_mixed", kind="attn", dtype="bf16", code="int8", hq=32, hkv=8, d=128, decoders=32, rows=1, lo=300,
             hi=4000, chunks="1024@1500,333@0", left=-1, lens=7),
        # A long prompt's second chunk: the most arithmetic.
        dict(name="attn_prompt", kind="attn", dtype="bf16", code="e4m3", hq=32, hkv=8, d=128, decoders=0, rows=1, lo=1, hi=1,
             chunks="4096@4096", left=-1, lens=8),
        # One conversation's keys taken out of the pool, to be sent elsewhere.
        dict(name="read_1_sequence", kind="read", dtype="bf16", code="e4m3", hkv=8, d=128, tokens=1500),
        # A long document's.
        dict(name="read_long_fp16_int8", kind="read", dtype="fp16", code="int8", hkv=8, d=128, tokens=40001),
        # One conversation: latency.
        dict(name="sample_1_row", kind="sample", dtype="bf16", rows=1, vocab=151936, spread=3.0, top_k=50, top_p=0.95,
             min_p=0.0, greedy=0.0),
        # A full tick, every request with limits of its own, some of them greedy.
        dict(name="sample_96_rows", kind="sample", dtype="fp32", rows=96, vocab=151936, spread=3.0, top_k=1000, top_p=0.9,
             min_p=0.02, greedy=0.1),
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["write", "write", "attn", "attn", "attn", "read", "sample", "sample"])
    dtype, code = rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "int8"])
    lens = rng.randrange(1 << 20)
    hq, hkv, d = rng.choice([(32, 8, 128), (32, 8, 128), (16, 4, 64), (12, 4, 96), (16, 1, 256), (8, 8, 128), (64, 4, 128),
                             (5, 1, 16)])
    if kind == "write":
        # Rotated keys round at the codes' borders by the order of their sums: only codes whose
        # steps follow their size are compared there.
        rope = rng.random() < 0.6
        form = rng.choice(["decode", "chunks", "mixed"])
        hi = _log(rng, 16, 4096)
        chunks = [] if form == "decode" else [
            "%d@%d" % (_log(rng, 2, 2048), rng.choice([0, _log(rng, 1, 4096)])) for _ in range(rng.randint(1, 3))]
        return dict(kind=kind, rope=rope, dtype=dtype, code="e4m3" if rope else code, hq=hq, hkv=hkv, d=d,
                    decoders=0 if form == "chunks" else _log(rng, 1, 128), lo=_log(rng, 1, hi), hi=hi,
                    chunks=",".join(chunks), lens=lens)
    if kind == "attn":
        form = rng.choice(["decode", "decode", "chunks", "mixed"])
        decoders = 0 if form == "chunks" else _log(rng, 1, 64)
        hi = _log(rng, 8, max(8, min(65536, 250000 // max(1, decoders))))
        chunks = [] if form == "decode" else [
            "%d@%d" % (_log(rng, 2, 1500), rng.choice([0, _log(rng, 1, 4000)])) for _ in range(rng.randint(1, 2))]
        return dict(kind=kind, dtype=dtype, code=code, hq=hq, hkv=hkv, d=d, decoders=decoders,
                    rows=rng.choice([1, 1, 1, 3, 6]), lo=_log(rng, max(6, hi // 8), hi) if hi > 6 else hi, hi=hi,
                    chunks=",".join(chunks), left=rng.choice([-1, -1, -1, _log(rng, 1, 4096)]), lens=lens)
    if kind == "read":
        return dict(kind=kind, dtype=rng.choice([dtype, "fp32"]), code=code, hkv=hkv, d=d, tokens=_log(rng, 1, 65536))
    vocab = rng.choice([151936, 151669, 32000, 50257, _log(rng, 2, 130000)])
    return dict(kind=kind, dtype=rng.choice([dtype, "fp32"]), rows=_log(rng, 1, 96), vocab=vocab,
                spread=rng.choice([0.3, 3.0, 8.0]), top_k=rng.choice([0, 1, _log(rng, 1, vocab)]),
                top_p=rng.choice([1.0, 0.95, rng.random()]), min_p=rng.choice([0.0, 0.0, 0.05, rng.random()]),
                greedy=rng.choice([0.0, 0.2]))


# ---------------------------------------------------------------- lengths and page tables
def _ticks(case):
    """(cached, new) tokens of every sequence: decoders, then chunks. ``lo`` to ``hi`` are a
    decoder's tokens with its new ones."""
    rng = random.Random(case["lens"])
    cached, new = [], []
    rows = case.get("rows", 1)
    for _ in range(case["decoders"]):
        cached.append(max(0, rng.randint(case["lo"], case["hi"]) - rows))
        new.append(rows)
    for part in filter(None, case["chunks"].split(",")):
        n, at = part.split("@")
        cached.append(int(at))
        new.append(int(n))
    return cached, new


def _table(lengths, seed):
    """Page ids that cover each sequence, from one seeded permutation: [sequences, width], and
    the pool's pages. Entries past a sequence's pages are page 0."""
    need = [-(-n // PAGE) for n in lengths]
    order = list(range(sum(need) or 1))
    random.Random(seed).shuffle(order)
    table = torch.zeros((len(need), max(1, *need) if need else 1), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, len(order)


def _quantised(x, code):
    """Codes and scales of ``x`` [..., d], a scale for each row."""
    kind, most = CODES[code]
    x = x.float()
    scale = (x.abs().amax(dim=-1) / most).clamp(min=LEAST_SCALE)
    y = x / scale[..., None]
    return (y.round() if kind == torch.int8 else y).to(kind), scale


# ----------------------------------------------------------------------------- prepare
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    state = dict(case=case, dtype=dt)

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype) * std

    def ints(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=DEVICE)

    def pool(pages, h, d, spread):
        """A pool's codes [pages, PAGE, h, d] and scales [pages, h, PAGE]; tokens differ in size."""
        x = normal(pages, PAGE, h, d, dtype=torch.float32)
        x *= torch.exp(spread * torch.randn((pages, PAGE, h, 1), generator=g, device=DEVICE))
        codes, scales = _quantised(x, case["code"])
        return codes, scales.transpose(1, 2).contiguous()

    if case["kind"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        state["logits"] = normal(rows, vocab, std=case["spread"])
        state["u"] = torch.rand(rows, generator=g, device=DEVICE)
        # Every request has its own limits, around the case's.
        r = torch.rand((3, rows), generator=g, device=DEVICE)
        hot = torch.rand(rows, generator=g, device=DEVICE) >= case["greedy"]
        state["temperature"] = torch.where(hot, 0.5 + r[0], 0.0)
        state["top_k"] = (case["top_k"] * (0.5 + r[1])).ceil().to(torch.int32) if case["top_k"] else None
        state["top_p"] = 1 - (1 - case["top_p"]) * (0.5 + r[2]).clamp(max=1) if case["top_p"] < 1 else None
        state["min_p"] = torch.full((rows,), case["min_p"], device=DEVICE) if case["min_p"] else None
        return state

    h, d = case["hkv"], case["d"]
    if case["kind"] == "read":
        pages = -(-case["tokens"] // PAGE)
        state["codes"], state["scales"] = pool(pages + 3, h, d, 0.3)
        order = list(range(pages + 3))
        random.Random(seed).shuffle(order)
        state["pages"] = ints(order[:pages])
        return state

    cached, new = _ticks(case)
    ends = [c + n for c, n in zip(cached, new)]
    table, pages = _table(ends, seed)
    state["k"], state["k_scale"] = pool(pages, h, d, 0.2)
    state["v"], state["v_scale"] = pool(pages, h, d, 0.4)
    rows = sum(new)
    if case["kind"] == "write":
        at = [c + i for c, n in zip(cached, new) for i in range(n)]
        of = [b for b, n in enumerate(new) for _ in range(n)]
        position = ints(at, torch.int64)
        state["slots"] = table.to(DEVICE).long()[ints(of, torch.int64), position // PAGE] * PAGE + position % PAGE
        # Slices of one projection, as a model has them.
        both = normal(rows, (case["hq"] + 2 * h) * d)
        q, k, v = both.split([case["hq"] * d, h * d, h * d], dim=1)
        state["q"], state["keys"], state["values"] = q.unflatten(1, (-1, d)), k.unflatten(1, (-1, d)), v.unflatten(1, (-1, d))
        if case["rope"]:
            state["positions"] = position
            state["q_norm"], state["k_norm"] = (1 + 0.1 * normal(d, dtype=torch.float32) for _ in range(2))
            inv = 1e6 ** (-torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
            angle = torch.arange(max(ends) + 1, device=DEVICE, dtype=torch.float64)[:, None] * inv
            angle = torch.cat((angle, angle), dim=1)
            state["cos"], state["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        return state

    state["table"] = table.to(DEVICE)
    state["q"] = normal(rows, case["hq"], d)
    state["cu_q"] = ints([sum(new[:i]) for i in range(len(new) + 1)])
    state["used"] = ints(ends)
    if own:
        from helios_amd import ops

        state["cache"] = ops.Kv8Cache(state["k"], state["v"], state["k_scale"], state["v_scale"])
        # One plan for a tick's layers.
        state["plan"] = ops.Kv8AttnPlan(
            state["cu_q"], state["used"], total_q=rows, max_q=max(new), max_k=max(ends), n_q_heads=case["hq"],
            n_kv_heads=h, head_dim=d, page_size=PAGE, window=(case["left"], 0))
    return state


# --------------------------------------------------------------------------------- run
def run(state):
    kind = state["case"]["kind"]
    return (_own if own else _plain)[kind](state)


def _own_write(s):
    from helios_amd import ops

    cache = ops.Kv8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if not s["case"]["rope"]:
        ops.kv8_append(cache, s["slots"], s["keys"], s["values"])
        return cache
    q = ops.kv8_norm_rope_append(s["q"], s["keys"], s["values"], s["q_norm"], s["k_norm"], s["cos"], s["sin"],
                                 s["positions"], cache, s["slots"], EPS)
    return (*cache, q)


def _own_attn(s):
    return s["plan"].run(s["q"], s["cache"], s["table"])


def _own_read(s):
    from helios_amd import ops

    return ops.kv8_gather(s["codes"], s["scales"], s["pages"], s["case"]["tokens"], s["dtype"])


def _own_sample(s):
    from helios_amd import ops

    got = ops.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                            min_p=s["min_p"])
    return got.token_ids, got.logprobs


_own = dict(write=_own_write, attn=_own_attn, read=_own_read, sample=_own_sample)


def _plain_write(s):
    """scale = max |x| / most; code = round(x / scale); keys and queries normalised and rotated before."""
    c, q, keys, values = s["case"], s["q"], s["keys"].float(), s["values"].float()
    if c["rope"]:
        half = c["d"] // 2
        cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]

        def rotated(x, weight):
            x = x * torch.rsqrt(x.pow(2).mean(dim=-1, keepdim=True) + EPS) * weight
            return x * cos + torch.cat((-x[..., half:], x[..., :half]), dim=-1) * sin

        q, keys = rotated(q.float(), s["q_norm"]).to(s["dtype"]), rotated(keys, s["k_norm"])
    page, at = s["slots"] // PAGE, s["slots"] % PAGE
    for x, codes, scales in ((keys, s["k"], s["k_scale"]), (values, s["v"], s["v_scale"])):
        code, scale = _quantised(x, c["code"])
        codes.view(torch.uint8)[page, at] = code.view(torch.uint8)
        scales.transpose(1, 2)[page, at] = scale
    cache = s["k"], s["v"], s["k_scale"], s["v_scale"]
    return (*cache, q) if c["rope"] else cache


def _plain_attn(s):
    """softmax(q k / sqrt(d)) v, k = code scale: the decoders as one padded batch, the chunks as another."""
    c = s["case"]
    cached, new = _ticks(c)
    out = torch.empty_like(s["q"])
    n = c["decoders"]
    if n:
        _padded(s, out, 0, n, max(new[:n]), max(cached[b] + new[b] for b in range(n)))
    if len(new) > n:
        _padded(s, out, n, len(new), max(new[n:]), max(cached[b] + new[b] for b in range(n, len(new))))
    return out


def _padded(s, out, b0, b1, max_q, max_k):
    c, first, used = s["case"], s["cu_q"].long(), s["used"].long()[b0:b1]
    h, d = c["hkv"], c["d"]
    table = s["table"].long()[b0:b1, :-(-max_k // PAGE)]
    count = (first[1:] - first[:-1])[b0:b1]

    def dense(codes, scales):
        x = codes[table] if codes.dtype == torch.int8 else codes.view(torch.uint8)[table].view(codes.dtype)
        x = x.float() * scales[table].transpose(2, 3)[..., None]
        return x.flatten(1, 2).transpose(1, 2)  # [sequences, heads, keys, d]

    k, v = dense(s["k"], s["k_scale"]), dense(s["v"], s["v_scale"])
    row = torch.arange(max_q, device=DEVICE)
    real = row < count[:, None]
    at = first[b0:b1, None] + torch.minimum(row, (count - 1)[:, None])
    q = s["q"][at].float().unflatten(2, (h, -1))  # [sequences, rows, heads, group, d]
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)
    key = torch.arange(k.shape[2], device=DEVICE)
    place = (used - count)[:, None] + row
    seen = (key <= place[..., None]) & real[..., None]
    if c["left"] >= 0:
        seen &= key >= place[..., None] - c["left"]
    score = score.unflatten(2, (-1, max_q)).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(dim=-1, keepdim=True).clamp(min=-1e30))
    total = p.sum(dim=-1, keepdim=True)
    got = torch.matmul(p.flatten(2, 3), v.contiguous()).unflatten(2, (-1, max_q)) / torch.where(total > 0, total, 1.0)
    got = got.permute(0, 3, 1, 2, 4).flatten(2, 3).to(out.dtype)
    out[at[real]] = got[real]


def _plain_read(s):
    """x = code scale."""
    pages = s["pages"].long()
    x = s["codes"].view(torch.uint8)[pages].view(s["codes"].dtype).float() * s["scales"][pages].transpose(1, 2)[..., None]
    return x.flatten(0, 1)[:s["case"]["tokens"]].transpose(0, 1)[None].to(s["dtype"]).contiguous()


def _plain_sample(s):
    """weight = exp((l - max) / t); by falling logit (then index) the first n are kept; the first
    position whose cumulative weight passes u times theirs. In 64 bits: sums over the vocabulary,
    and cumulative weights next to a border."""
    logits = s["logits"]
    vocab = logits.shape[1]
    value, order = logits.sort(dim=-1, descending=True, stable=True)
    hot = s["temperature"] > 0
    t = torch.where(hot, s["temperature"], 1.0).double()[:, None]
    shift = (value.double() - value[:, :1].double()) / t
    weight = torch.exp(shift)
    total = weight.cumsum(dim=-1)
    keep = torch.full((logits.shape[0],), vocab, device=DEVICE)
    if s["top_k"] is not None:
        keep = torch.where(s["top_k"] > 0, s["top_k"].long(), vocab).clamp(max=vocab)
    if s["top_p"] is not None:
        of = total.gather(1, keep[:, None] - 1) * s["top_p"].double()[:, None]
        keep = torch.minimum(keep, (total < of).sum(dim=-1) + 1)
    if s["min_p"] is not None:
        keep = torch.minimum(keep, (weight >= s["min_p"].double()[:, None]).sum(dim=-1))
    keep = keep.clamp(min=1)
    kept = total.gather(1, keep[:, None] - 1)
    place = (total <= s["u"].double()[:, None] * kept).sum(dim=-1)
    place = torch.where(hot, torch.minimum(place, keep - 1), 0)[:, None]
    logprob = shift.gather(1, place) - torch.log(kept)
    return order.gather(1, place)[:, 0], torch.where(hot, logprob[:, 0], 0.0).float()


_plain = dict(write=_plain_write, attn=_plain_attn, read=_plain_read, sample=_plain_sample)


# -------------------------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * size + case["rows"] * 28, flops=4 * n)
    row = case["hkv"] * (case["d"] + 4)  # a token's codes and scales, keys or values
    if case["kind"] == "read":
        n = case["tokens"]
        return dict(bytes=n * (row + case["hkv"] * case["d"] * size), flops=n * case["hkv"] * case["d"])
    cached, new = _ticks(case)
    rows, q = sum(new), case["hq"] * case["d"] * size
    if case["kind"] == "write":
        each = 2 * case["hkv"] * case["d"] * size + 2 * row + 8
        tables = 2 * (max(c + n for c, n in zip(cached, new)) if case["rope"] else 0)
        return dict(bytes=rows * (each + (2 * q + 8 if case["rope"] else 0)) + min(tables, 2 * rows) * case["d"] * 4,
                    flops=rows * (2 * case["hkv"] + (case["hq"] if case["rope"] else 0)) * case["d"] * 4)
    keys = pairs = 0
    for c, n in zip(cached, new):
        lo = 0 if case["left"] < 0 else max(0, c - case["left"])
        keys += c + n - lo
        whole = n * c + n * (n + 1) // 2
        pairs += whole if case["left"] < 0 else sum(min(c + i + 1, case["left"] + 1) for i in range(n))
    return dict(bytes=2 * keys * row + 2 * rows * q, flops=4 * pairs * case["hq"] * case["d"])


# ------------------------------------------------------------------------------- exact
def exact(case, seed):
    """What run returns, from the definitions in 64 bits."""
    s = prepare(case, seed)
    return dict(write=_exact_write, attn=_exact_attn, read=_exact_read, sample=_exact_sample)[case["kind"]](case, s)


def _values(codes, scales):
    """codes [tokens, heads, d] of a page and its scales [heads, tokens], as they stand for values."""
    return codes.to(torch.float32).double() * scales.double().t()[..., None]


def _exact_write(case, s):
    most = CODES[case["code"]][1]
    outs = []
    for x, codes, scales, weight in ((s["keys"], s["k"], s["k_scale"], s.get("k_norm")), (s["values"], s["v"], s["v_scale"], None)):
        x = x.double()
        if case["rope"] and weight is not None:
            x = _exact_rotated(s, x, weight, case["d"])
        scale = torch.clamp(x.abs().max(dim=-1).values / most, min=LEAST_SCALE)
        flat, by = codes.to(torch.float32).double().flatten(0, 1), scales.double()
        if case["code"] == "e4m3":
            flat[s["slots"]] = (x / scale[..., None]).to(torch.float8_e4m3fn).to(torch.float32).double()
        by[s["slots"] // PAGE, :, s["slots"] % PAGE] = scale
        # Whole codes next to a border have no value of their own.
        outs.append((flat.view(codes.shape) if case["code"] == "e4m3" else None, by))
    out = outs[0][0], outs[1][0], outs[0][1], outs[1][1]
    return (*out, _exact_rotated(s, s["q"].double(), s["q_norm"], case["d"])) if case["rope"] else out


def _exact_rotated(s, x, weight, d):
    x = x / torch.sqrt((x * x).sum(dim=-1, keepdim=True) / d + EPS) * weight.double()
    a, b = x[..., :d // 2], x[..., d // 2:]
    cos, sin = s["cos"].double()[s["positions"]][:, None], s["sin"].double()[s["positions"]][:, None]
    return torch.cat((a * cos[..., :d // 2] - b * sin[..., :d // 2], b * cos[..., d // 2:] + a * sin[..., d // 2:]), dim=-1)


def _exact_attn(case, s):
    cached, new = _ticks(case)
    group, table = case["hq"] // case["hkv"], s["table"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        pages = table[b][:-(-(c + n) // PAGE)]
        k = torch.cat([_values(s["k"][p], s["k_scale"][p]) for p in pages])[:c + n]
        v = torch.cat([_values(s["v"][p], s["v_scale"][p]) for p in pages])[:c + n]
        behind = c + torch.arange(n, device=DEVICE)[:, None] - torch.arange(c + n, device=DEVICE)
        hidden = (behind < 0) | (behind > case["left"] if case["left"] >= 0 else False)
        for head in range(case["hq"]):
            score = torch.mm(s["q"][at:at + n, head].double(), k[:, head // group].t().contiguous()) * case["d"] ** -0.5
            score[hidden] = -math.inf
            out[at:at + n, head] = torch.mm(torch.softmax(score, dim=-1), v[:, head // group].contiguous())
        at += n
    return out


def _exact_read(case, s):
    x = torch.cat([_values(s["codes"][p], s["scales"][p]) for p in s["pages"].tolist()])
    return x[:case["tokens"]].transpose(0, 1)[None]


def _exact_sample(case, s):
    out = []
    for r in range(case["rows"]):
        t = float(s["temperature"][r])
        if t == 0:
            out.append(0.0)
            continue
        row = s["logits"][r].double()
        row, _ = torch.sort((row - row.max()) / t, descending=True)
        n = case["vocab"]
        if s["top_k"] is not None:
            n = min(n, int(s["top_k"][r]))
        weight = torch.exp(row)
        summed = torch.cumsum(weight, dim=0)
        if s["top_p"] is not None:
            n = min(n, 1 + int((summed < float(s["top_p"][r]) * summed[n - 1]).sum()))
        if s["min_p"] is not None:
            n = min(n, int((weight >= float(s["min_p"][r])).sum()))
        n = max(n, 1)
        at = min(n - 1, int((summed <= float(s["u"][r]) * summed[n - 1]).sum()))
        out.append(float(row[at] - torch.log(summed[n - 1])))
    return None, torch.tensor(out, dtype=torch.float64)
