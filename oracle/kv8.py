"""The operators of a serving tick over an 8-bit cache, restated on the CPU: quantising writes
(in fp32, as they are defined), norms and rotation, attention and drawn tokens (in 64 bits). No
counterpart in the reference, whose cache has the model's type and whose tokens are greedy."""

from __future__ import annotations

import math

import torch

MOST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}
LEAST_SCALE = 2.0 ** -100


def scale_of(rows, code):
    """Scales (fp32) of rows [..., d], NaN for one with an infinite or NaN element."""
    top = rows.float().abs().amax(dim=-1)
    scale = (top * torch.tensor(1.0 / MOST[code], dtype=torch.float32)).clamp(min=LEAST_SCALE)
    return torch.where(torch.isfinite(rows).all(dim=-1), scale, torch.nan)


def quantise(rows, code):
    """Codes and scales of rows [..., d]."""
    scale = scale_of(rows, code)
    y = rows.float() / scale[..., None]
    y = torch.where(torch.isnan(scale)[..., None], 0.0, y)
    return (y.round() if code == torch.int8 else y).to(code), scale


def rotate(x, weight, cos, sin, positions, eps):
    """RMSNorm and rotation of [rows, heads, d], in 64 bits."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + eps) * weight.double()
    at = positions.clamp(0, cos.shape[0] - 1)
    c, s = cos.double()[at][:, None], sin.double()[at][:, None]
    half = x.shape[-1] // 2
    return x * c + torch.cat((-x[..., half:], x[..., :half]), dim=-1) * s


def values(codes, scales):
    """codes [pages, page, heads, d] and scales [pages, heads, page] as fp32 values (one rounding)."""
    return codes.to(torch.float32) * scales.transpose(1, 2)[..., None]


def attention(q, keys, vals, table, cu_q, used, window, scale):
    """Attention of packed rows over dequantised pools (double), and of |values| with the same
    weights; the largest sum of |q| |k| of a row; the largest weight times |value| of a row; all
    [rows, heads, d] or [rows, heads, 1]. Rows without a key: zeros. A bad page has no keys."""
    rows, heads, d = q.shape
    n_kv, page = keys.shape[2], keys.shape[1]
    group = heads // n_kv
    out, mag = torch.zeros(2, rows, heads, d, dtype=torch.float64)
    reach, peak = torch.zeros(2, rows, heads, 1, dtype=torch.float64)
    for b in range(len(used)):
        q0, q1, L = int(cu_q[b]), int(cu_q[b + 1]), int(used[b])
        n = q1 - q0
        if n < 1 or L < 1:
            continue
        ids = [int(p) for p in table[b, :-(-L // page)]]
        there = torch.tensor([0 <= p < keys.shape[0] for p in ids]).repeat_interleave(page)[:L]
        safe = [p if 0 <= p < keys.shape[0] else 0 for p in ids]
        k, v = (t[safe].flatten(0, 1)[:L].double() for t in (keys, vals))
        behind = (L - n + torch.arange(n))[:, None] - torch.arange(L)
        seen = there[None].expand(n, L).clone()
        if window[1] >= 0:
            seen &= behind >= -window[1]
        if window[0] >= 0:
            seen &= behind <= window[0]
        k, v = (torch.where(there[:, None, None], t, 0.0) for t in (k, v))
        for h in range(heads):
            kh, vh, qh = k[:, h // group], v[:, h // group], q[q0:q1, h].double()
            s = (qh @ kh.t()) * scale
            s = torch.where(seen, s, -math.inf)
            top = s.amax(dim=1, keepdim=True)
            p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            total = p.sum(dim=1, keepdim=True)
            p = p / torch.where(total == 0, 1.0, total)
            hidden_nan = torch.where(torch.isnan(vh), 0.0, vh)
            has_nan = (seen & torch.isnan(vh).any(dim=1)[None]).any(dim=1, keepdim=True)
            got = p @ hidden_nan
            out[q0:q1, h] = torch.where(has_nan, torch.nan, got)
            mag[q0:q1, h] = p @ hidden_nan.abs()
            reach[q0:q1, h] = torch.where(seen, (qh.abs() @ kh.abs().t()) * scale, 0.0).amax(dim=1, keepdim=True)
            peak[q0:q1, h] = (p * hidden_nan.abs().amax(dim=1)[None]).amax(dim=1, keepdim=True)
    return out, mag, reach, peak


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    """Drawn tokens and their logprobs, a row at a time in 64 bits."""
    ids, logs = [], []
    for r in range(logits.shape[0]):
        row = logits[r].double().tolist()
        key = [math.inf if math.isnan(x) else x for x in row]  # a NaN counts as the largest
        nan = [math.isnan(x) for x in row]
        order = sorted(range(len(row)), key=lambda v: (not nan[v], -key[v], v))
        t = 1.0 if temperature is None else float(temperature[r])
        top = row[order[0]]
        if top == -math.inf:
            ids.append(-1)
            logs.append(-math.inf)
            continue
        if t <= 0 or not math.isfinite(top):
            ids.append(order[0])
            logs.append(0.0)
            continue
        weight = [math.exp((row[v] - top) / t) if row[v] > -math.inf else 0.0 for v in order]
        cum = torch.tensor(weight, dtype=torch.float64).cumsum(0).tolist()
        n = len(order)
        if top_k is not None and int(top_k[r]) > 0:
            n = min(n, int(top_k[r]))
        if top_p is not None and float(top_p[r]) < 1:
            border = float(top_p[r]) * cum[n - 1]
            n = min(n, 1 + sum(c < border for c in cum))
        if min_p is not None:
            n = min(n, sum(w >= float(min_p[r]) for w in weight))
        n = max(n, 1)
        x = min(max(float(u[r]), 0.0), 1.0) * cum[n - 1]
        at = next((i for i in range(n) if cum[i] > x), None)
        if at is None:
            at = max(i for i in range(n) if weight[i] > 2.0 ** -45)
        ids.append(order[at])
        logs.append((row[order[at]] - top) / t - math.log(cum[n - 1]))
    return torch.tensor(ids), torch.tensor(logs, dtype=torch.float64)
