"""The C entries of the decode tick's operators refuse what they cannot run, before any launch:
every call here returns an error or has no work."""

from __future__ import annotations

import pytest
import torch

from helios_amd import _capi, ops

BAD, NO, WS = _capi.HX_E_INVALID_ARG, _capi.HX_E_UNSUPPORTED, _capi.HX_E_WORKSPACE
P = 1 << 20  # an aligned address that no call here reads


def _call(name, base, **change):
    args = dict(base)
    assert set(change) <= set(args)
    args.update(change)
    return getattr(_capi.lib(), name)(*args.values())


INT4 = dict(x=P, x_row=256, rows=4, packed=P, steps=P, cols=16, k=256, group=64, dtype=0, norm=None, eps=0.0,
            residual=None, residual_row=16, swiglu=0, out=P, out_row=16, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), NO), (dict(group=16), NO), (dict(group=48), NO), (dict(rows=65), NO), (dict(rows=-1), BAD),
    (dict(cols=0), BAD), (dict(k=0), BAD), (dict(k=96), BAD), (dict(x=None), BAD), (dict(packed=None), BAD),
    (dict(steps=None), BAD), (dict(steps=P + 8), BAD), (dict(out=None), BAD), (dict(packed=P + 8), BAD),
    (dict(x=P + 2), BAD), (dict(x_row=255), BAD), (dict(x_row=252), BAD), (dict(norm=P, eps=-1.0), BAD),
    (dict(norm=P, eps=float("nan")), BAD), (dict(norm=P + 4), BAD), (dict(out=P + 1), BAD), (dict(out_row=15), BAD),
    (dict(residual=P, swiglu=1), BAD), (dict(residual=P, residual_row=15), BAD), (dict(rows=0), 0),
    (dict(norm=P, rows=17, ws=None), WS), (dict(norm=P, rows=17, ws=P + 8), WS), (dict(norm=P, rows=17, ws_bytes=16), WS),
    (dict(k=1 << 21, x_row=1 << 21), NO), (dict(x_row=1 << 27), NO), (dict(cols=1 << 26), NO)])
def test_int4_gemm(change, code):
    assert _call("hx_int4_gemm", INT4, **change) == code


DEQUANT = dict(packed=P, steps=P, rows=20, k=256, group=64, dtype=0, out=P, out_row=256, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=7), NO), (dict(group=0), NO), (dict(rows=0), BAD), (dict(k=100), BAD), (dict(out=None), BAD),
    (dict(out=P + 8), BAD), (dict(out_row=248), BAD), (dict(out_row=260), BAD), (dict(packed=P + 4), BAD),
    (dict(rows=1 << 30, k=4096, out_row=4096), NO)])
def test_int4_dequantize(change, code):
    assert _call("hx_int4_dequantize", DEQUANT, **change) == code


RULES = dict(logits=P, row=64, rows=2, vocab=64, dtype=0, tokens=P, token_row=8, cap=8, lengths=P, prompt=None, rep=None,
             pres=None, freq=None, bias_ids=P, bias_values=P, bias_row=4, n_bias=4, allowed=P, allowed_row=2, out=P,
             out_row=64, ids=P, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), NO), (dict(rows=-1), BAD), (dict(vocab=0), BAD), (dict(row=63), BAD), (dict(logits=None), BAD),
    (dict(ids=None), BAD), (dict(out_row=63), BAD), (dict(lengths=None), BAD), (dict(token_row=7), BAD),
    (dict(bias_values=None), BAD), (dict(bias_row=3), BAD), (dict(n_bias=-1), BAD), (dict(allowed_row=1), BAD),
    (dict(ws=None), WS), (dict(ws=P + 4), WS), (dict(ws_bytes=15), WS), (dict(rows=0), 0),
    (dict(logits=P + 1), BAD), (dict(dtype=2, out=P + 2), BAD),
    (dict(rows=1 << 31, ws_bytes=1 << 40), NO), (dict(rows=1 << 23, ws_bytes=1 << 40), NO)])
def test_logit_rules(change, code):
    assert _call("hx_logit_rules", RULES, **change) == code


BOUNDS = dict(k=P, bounds=P, pages=4, page=256, block=64, heads=8, dim=128, dtype=0, table=P, stride=4, width=4, cu=P,
              used=P, batch=2, max_q=1, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), NO), (dict(block=48), NO), (dict(block=8), NO), (dict(block=512), NO), (dict(dim=100), NO),
    (dict(dim=264), NO), (dict(pages=0), BAD), (dict(heads=0), BAD), (dict(k=None), BAD), (dict(bounds=P + 8), BAD),
    (dict(stride=3), BAD), (dict(width=0), BAD), (dict(cu=None), BAD), (dict(batch=-1), BAD), (dict(max_q=-1), BAD),
    (dict(batch=1 << 23), NO), (dict(batch=0), 0), (dict(max_q=0), 0)])
def test_kv_block_bounds(change, code):
    assert _call("hx_kv_block_bounds", BOUNDS, **change) == code


SELECT = dict(q=P, q_row=4096, q_head=128, q_rows=2, rows=None, row_seq=None, keys=P, n=2, hq=32, hkv=8, dim=128, dtype=0,
              bounds=P, pages=4, page=256, block=64, table=P, stride=4, batch=2, width=4, budget=8, sink=1, recent=2,
              blocks=P, ws=P, ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(ws=None), WS), (dict(ws=P + 4), WS), (dict(ws_bytes=2 * 8 * 16 * 8 - 1), WS), (dict(q=P + 8), BAD),
    (dict(q_row=4092), BAD), (dict(q_head=132), BAD),
    (dict(dtype=2), NO), (dict(block=24), NO), (dict(hq=30), BAD), (dict(budget=0), BAD), (dict(sink=-1), BAD),
    (dict(recent=0), BAD), (dict(sink=7, recent=2), BAD), (dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1), BAD),
    (dict(width=4097, stride=4097), NO), (dict(n=3), BAD), (dict(n=-1), BAD), (dict(q=None), BAD),
    (dict(bounds=P + 4), BAD), (dict(blocks=None), BAD), (dict(batch=1), BAD), (dict(n=0), 0),
    (dict(n=1 << 20, q_rows=1 << 20, batch=1 << 20, ws_bytes=1 << 40), NO)])
def test_select_blocks(change, code):
    assert _call("hx_select_blocks", SELECT, **change) == code


SPARSE = dict(q=P, q_row=4096, q_head=128, q_rows=2, rows=None, row_seq=None, keys=P, n=2, k=P, v=P, pages=4, page=256,
              block=64, blocks=P, budget=64, table=P, stride=4, batch=2, width=4, hq=32, hkv=8, dim=128, scale=1.0, dtype=0,
              out=P, out_row=4096, out_head=128, ws=P, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), NO), (dict(block=2048, page=2048), NO), (dict(dim=4), NO), (dict(hq=31), BAD), (dict(budget=0), BAD),
    (dict(n=3), BAD), (dict(batch=1), BAD), (dict(k=None), BAD), (dict(v=P + 2), BAD), (dict(q=P + 8), BAD),
    (dict(q_row=4092), BAD), (dict(q_head=132), BAD), (dict(out=P + 2), BAD), (dict(out_row=4097), BAD),
    (dict(blocks=None), BAD), (dict(ws=None), WS), (dict(ws=P + 8), WS), (dict(ws_bytes=64), WS), (dict(n=0), 0),
    (dict(hkv=1 << 18, hq=1 << 18), NO), (dict(budget=(1 << 24) + 1), BAD),
    (dict(n=1 << 20, q_rows=1 << 20, batch=1 << 20, ws_bytes=1 << 60), NO)])
def test_block_sparse_attn(change, code):
    assert _call("hx_block_sparse_attn", SPARSE, **change) == code


def test_workspace_sizes():
    lib = _capi.lib()
    # slices of 4096, a row's first up to 7 elements before it
    assert lib.hx_logit_rules_workspace_bytes(3, 4089) == 3 * 8
    assert lib.hx_logit_rules_workspace_bytes(3, 4090) == 3 * 2 * 8
    assert lib.hx_logit_rules_workspace_bytes(0, 10) == 0
    # normalised rows past one tile: two parts of each row tile of 16, k rounded up to 128
    assert lib.hx_int4_workspace_bytes(16, 2560, 1) == lib.hx_int4_workspace_bytes(64, 2560, 0) == 0
    assert lib.hx_int4_workspace_bytes(17, 200, 1) == 2 * 32 * 256 * 2
    # Few rows: their lists are split, each part with its sums and two statistics per head.
    small = lib.hx_block_sparse_workspace_bytes(1, 32, 8, 128, 32, 64)
    assert small > 0 and small % (32 * 130 * 4) == 0
    assert lib.hx_block_sparse_workspace_bytes(4096, 32, 8, 128, 2, 64) == 0  # one part each
    assert lib.hx_block_sparse_workspace_bytes(1, 31, 8, 128, 32, 64) == 0


def test_int4_quantize_at_the_ends_of_the_range():
    """A group from the type's lowest to its largest value, and one of its smallest: finite
    steps, the ends within half a step of the outer values."""
    for dtype in (torch.bfloat16, torch.float16):
        most, least = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
        w = torch.zeros(2, 32, dtype=dtype)
        w[0, :2] = torch.tensor([-most, most], dtype=dtype)
        w[1, :2] = torch.tensor([-least, 64 * least], dtype=dtype)
        q = ops.int4_quantize(w, 32)
        scale = (q.steps & 0xffff).to(torch.int16).view(dtype)[0, 0, :2, 0].double()
        zero = (q.steps >> 16).to(torch.int16).view(dtype)[0, 0, :2, 0].double() - 16
        assert torch.isfinite(scale).all() and (scale > 0).all()
        outer = torch.stack((-zero * scale, (15 - zero) * scale), dim=1)
        step = scale[:, None] * (0.5 + 15 * torch.finfo(dtype).eps)
        assert ((outer - w[:, :2].double()).abs() <= step).all()
