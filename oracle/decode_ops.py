"""The operators of a long-context decode tick, restated in 64 bits on the CPU: key bounds of
cache blocks, the selection by them, attention over the selection, products with 4-bit
weights, and logit rules. No counterpart in the reference, which reads every key, keeps
16-bit weights and leaves its logits as they are."""

from __future__ import annotations

import math

import torch


def block_bounds(k_pool, bounds, table, cached, new):
    """``bounds`` (double) after a tick that appended ``new[b]`` tokens to ``cached[b]``: one
    block at a time. A NaN among a block's keys makes both bounds of its dim NaN."""
    page, per_page = k_pool.shape[1], bounds.shape[1]
    block = page // per_page
    out = bounds.double().clone()
    for b, (c, n) in enumerate(zip(cached, new)):
        for j in range(c // block, (c + n - 1) // block + 1) if n else ():
            p = int(table[b, j // per_page])
            at = j % per_page * block
            keys = k_pool[p, at:at + min(block, c + n - j * block)].double()
            out[p, j % per_page, :, 0] = keys.amin(0)
            out[p, j % per_page, :, 1] = keys.amax(0)
    return out


def block_scores(q, bounds, table_row, count, head, group):
    """Scores [count] of a query row ``q`` [heads, d] for KV head ``head``; NaN as +inf."""
    per_page = bounds.shape[1]
    heads = q[head * group:(head + 1) * group].double()
    out = torch.full((count,), -math.inf, dtype=torch.float64)
    for j in range(count):
        p = int(table_row[j // per_page])
        if 0 <= p < bounds.shape[0]:
            low, high = bounds[p, j % per_page, head].double()
            s = torch.maximum(heads * low, heads * high).sum()
            nan = torch.isnan(heads * low).any() or torch.isnan(heads * high).any()
            out[j] = math.inf if nan or torch.isnan(s) else s
    return out


def select(scores, count, budget, sink, recent):
    """The chosen blocks of one row and head, ascending, padded with -1."""
    if count <= budget:
        take = list(range(count))
    else:
        kept = set(range(sink)) | set(range(count - recent, count))
        rest = sorted((j for j in range(count) if j not in kept), key=lambda j: (-float(scores[j]), j))
        take = sorted(kept | set(rest[:budget - len(kept)]))
    return take + [-1] * (budget - len(take))


def sparse_attention(q, k_pool, v_pool, blocks, table, keys, seqs, block, scale):
    """[n, heads, d] in double: softmax over the listed blocks' keys, a block listed twice twice."""
    page, n_kv = k_pool.shape[1], k_pool.shape[2]
    group = q.shape[1] // n_kv
    out = torch.zeros(q.shape, dtype=torch.float64)
    for i, (n, s) in enumerate(zip(keys, seqs)):
        for h in range(n_kv):
            at = []
            for j in blocks[i, h].tolist():
                for t in range(j * block, min((j + 1) * block, n)) if j >= 0 else ():
                    p = int(table[s, t // page])
                    if 0 <= p < k_pool.shape[0]:
                        at.append((p, t % page))
            if not at:
                continue
            p, t = torch.tensor(at).t()
            k, v = k_pool[p, t, h].double(), v_pool[p, t, h].double()
            for g in range(h * group, (h + 1) * group):
                out[i, g] = torch.softmax(scale * (k @ q[i, g].double()), 0) @ v
    return out


def int4_matrix(values, scales, zeros):
    """W [rows, k] in double of values [rows, k] and scales / zeros [groups, rows]."""
    group = values.shape[1] // scales.shape[0]
    return (values.double() - zeros.double().t().repeat_interleave(group, 1)) \
        * scales.double().t().repeat_interleave(group, 1)


def logit_rules(row, known, prompt, repetition, presence, frequency, bias, allowed):
    """One row (double) after its rules, before the rounding: ``known`` the token list, the first
    ``prompt`` of them not said, ``bias`` pairs in order, ``allowed`` bools or None."""
    out = row.double().clone()
    vocab = out.numel()
    for v in {t for t in known if 0 <= t < vocab}:
        out[v] = out[v] / repetition if out[v] > 0 else out[v] * repetition
        c = sum(t == v for t in known[max(prompt, 0):])
        if c:
            out[v] -= frequency * c + presence
    for v, value in dict((v, x) for v, x in bias if 0 <= v < vocab).items():
        out[v] += value
    if allowed is not None:
        out[~allowed] = -math.inf
    return out
