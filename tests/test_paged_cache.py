"""The paged 8-bit KV cache without a GPU: the oracle's own invariants, and what the host refuses."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from dsm import _lib
from dsm import paged_cache as pc
from oracle import paged_cache_oracle as po


# ------------------------------------------------------------------------------- the oracle
@pytest.mark.parametrize("seed", range(4))
def test_extend_then_trim_restores_the_stack(seed):
    r = random.Random(seed)
    page, b, most = 64, 9, 8
    lengths = [r.randint(0, 3 * page) for _ in range(b)]
    pool = list(range(60))
    r.shuffle(pool)
    table = [[-1] * most for _ in range(b)]
    for i, n in enumerate(lengths):
        for j in range(-(-n // page)):
            table[i][j] = pool.pop()
    free = pool + [-1] * (60 - len(pool))
    new = [r.choice([0, 1, 5, 64, 130]) for _ in range(b)]
    l2, t2, nf, cu, slots, pos, failed = po.paged_extend(lengths, new, table, free, len(pool), page, sum(new) + 3)
    assert not failed and l2 == [a + c for a, c in zip(lengths, new)] and slots[-3:] == [-1] * 3
    used = [t2[i][j] for i in range(b) for j in range(-(-l2[i] // page))]
    assert len(set(used)) == len(used) and not set(used) & set(free[:nf])
    live = [s for s in slots if s >= 0]
    assert len(set(live)) == sum(new)
    l3, f3, nf3, failed = po.paged_trim(l2, lengths, t2, free, nf, page)
    assert not failed and (l3, f3, nf3) == (lengths, free, len(pool))


def test_round_e4m3_agrees_with_torch():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(4000, generator=g) * s for s in (1e-3, 0.02, 1.0, 60.0)] + [po.e4m3_values().float()])
    x = x[x.abs() <= 448]
    ties = (po.e4m3_values()[:-1] + po.e4m3_values()[1:]).float() / 2  # halfway between neighbours
    x = torch.cat([x, ties[torch.isfinite(ties)]])
    assert torch.equal(po.round_e4m3(x.double()).float(), x.to(torch.float8_e4m3fn).float())


def test_scale_exponents_at_their_borders():
    assert po.kv8_scale_exp(0.0) == -120 and po.kv8_scale_exp(448.0) == 0
    assert po.kv8_scale_exp(449.0) == 1 and po.kv8_scale_exp(224.0) == -1 and po.kv8_scale_exp(3.3e38) == 120


def test_layouts_invert():
    x = torch.arange(2 * 128 * 128).reshape(2, 128, 128)
    assert torch.equal(po.load_keys(po.store_keys(x)), x) and torch.equal(po.load_values(po.store_values(x)), x)
    assert not torch.equal(po.store_keys(x), x)
    assert po.store_values(x)[1, 1, 5, 7] == x[1, 64 + 7, 5]


# ------------------------------------------------------------------------------- refusals
def _extend(L, batch=4, page=64, stride=8, most=8, n_pages=10, rows=16, ptr=1):
    return L.dsm_paged_extend(ptr, 1, batch, page, 1, stride, most, 1, 1, n_pages, 1, 1, 1, rows, None)


def _trim(L, batch=4, page=64, stride=8, most=8, n_pages=10, ptr=1):
    return L.dsm_paged_trim(ptr, 1, batch, page, 1, stride, most, 1, 1, n_pages, None)


def _append(L, dt=_lib.DT_BF16, rows=4, n_kv=2, hd=128, stride=128, page=64, n_pages=4, codes=16, slots=1):
    return L.dsm_kv8_append(1, 1, dt, rows, n_kv, hd, stride, 128, stride, 128, slots, page, n_pages, codes, 16, 1, 1,
                            None)


def _attn(L, ws=16, ws_bytes=1 << 30, blk=(1, 1), **over):
    f = dict(q_batch_stride=0, q_row_stride=128, q_head_stride=128, bk_batch_stride=0, bk_head_stride=0,
             bk_row_stride=0, bv_batch_stride=0, bv_head_stride=0, bv_row_stride=0, table_stride=8, k_codes=16,
             v_codes=16, dtype=_lib.DT_BF16, batch=2, block=3, n_heads=8, n_kv=2, head_dim=128, page_size=64,
             n_pages=4, max_pages=8, scale=0.1)
    f.update(over)
    d = _lib.KV8AttnDesc(**f)
    one = ctypes.cast(1, ctypes.POINTER(ctypes.c_float))
    d.k_scale = d.v_scale = ctypes.cast(one, ctypes.c_void_p)
    return L.dsm_gqa_attn_kv8(ctypes.byref(d), 1, 1, 1, blk[0], blk[1], 1, ws, ws_bytes, None)


@pytest.mark.parametrize("call", [
    lambda L: _extend(L, batch=-1), lambda L: _extend(L, batch=8193), lambda L: _extend(L, page=0),
    lambda L: _extend(L, page=96), lambda L: _extend(L, page=2048), lambda L: _extend(L, stride=7),
    lambda L: _extend(L, most=0), lambda L: _extend(L, stride=1 << 22, most=1 << 21),
    lambda L: _extend(L, n_pages=0), lambda L: _extend(L, rows=-1), lambda L: _extend(L, rows=1 << 31),
    lambda L: _extend(L, ptr=None),
    lambda L: _trim(L, batch=8193), lambda L: _trim(L, page=32), lambda L: _trim(L, stride=3),
    lambda L: _trim(L, n_pages=0), lambda L: _trim(L, ptr=None),
    lambda L: _append(L, dt=_lib.DT_F16), lambda L: _append(L, rows=-1), lambda L: _append(L, n_kv=0),
    lambda L: _append(L, hd=32), lambda L: _append(L, hd=96), lambda L: _append(L, stride=-1),
    lambda L: _append(L, page=100), lambda L: _append(L, n_pages=0), lambda L: _append(L, codes=8),
    lambda L: _append(L, slots=None),
    lambda L: _attn(L, n_heads=7), lambda L: _attn(L, head_dim=96), lambda L: _attn(L, page_size=48),
    lambda L: _attn(L, batch=8193), lambda L: _attn(L, block=0), lambda L: _attn(L, table_stride=7),
    lambda L: _attn(L, max_pages=0), lambda L: _attn(L, n_pages=0), lambda L: _attn(L, dtype=_lib.DT_F16),
    lambda L: _attn(L, q_row_stride=-1), lambda L: _attn(L, bk_row_stride=-1), lambda L: _attn(L, blk=(1, None)),
    lambda L: _attn(L, k_codes=None), lambda L: _attn(L, k_codes=8), lambda L: _attn(L, ws=8),
    lambda L: _attn(L, ws=None), lambda L: _attn(L, ws_bytes=0),
])
def test_entry_points_refuse_bad_arguments_on_the_host(call):
    L = _lib.lib()
    assert call(L) != 0
    assert L.dsm_last_error_message().decode()


def test_empty_calls_do_nothing():
    L = _lib.lib()
    assert _append(L, rows=0, slots=None) == 0
    assert _trim(L, batch=0, ptr=None) == 0
    assert _attn(L, batch=0) == 0
    assert L.dsm_gqa_attn_kv8_workspace_bytes(0, 1, 8, 2, 128) == 0
    assert L.dsm_gqa_attn_kv8_workspace_bytes(4, 1, 7, 2, 128) == 0
    assert L.dsm_gqa_attn_kv8_workspace_bytes(4, 1, 8, 2, 96) == 0
    assert L.dsm_gqa_attn_kv8_workspace_bytes(4, 7, 32, 8, 128) > 0


def test_desc_layout_matches_the_header():
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dsm.h")).read()
    body = text[text.index("typedef struct dsm_kv8_attn_desc"):text.index("} dsm_kv8_attn_desc;")]
    c_fields = re.findall(r"\*?\s*([a-z_0-9]+)\s*[,;]", body)
    assert c_fields == [f for f, _ in _lib.KV8AttnDesc._fields_]
    # what the calls pack is the same struct, byte for byte
    values = list(range(1, 11)) + [1 << 40, 1 << 41, 1 << 42, 1 << 43] + list(range(20, 29)) + [0.25]
    assert pc._DESC.pack(*values) == bytes(_lib.KV8AttnDesc(*values))


def test_python_functions_refuse_cpu_tensors_and_bad_settings():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA"):
        pc.paged_extend(i32(2), i32(2), i32(2, 4), i32(8), i32(1), 64, 4)
    with pytest.raises(ValueError, match="CUDA"):
        pc.paged_trim(i32(2), i32(2), i32(2, 4), i32(8), i32(1), 64)
    layer = pc.KV8Layer(torch.zeros(2, 1, 64, 128, dtype=torch.uint8), torch.zeros(2, 1, 1, 128, 64, dtype=torch.uint8),
                        torch.zeros(2, 1), torch.zeros(2, 1))
    with pytest.raises(ValueError, match="CUDA"):
        pc.kv8_append(layer, torch.zeros(3, 1, 128), torch.zeros(3, 1, 128), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        pc.gqa_attention_kv8(torch.zeros(1, 1, 4, 128), layer, i32(1, 2), i32(1))
    for kw in (dict(head_dim=96), dict(page_size=80), dict(page_size=2048), dict(batch=9000), dict(n_pages=0)):
        args = dict(n_layers=1, n_pages=4, n_kv=1, head_dim=128, batch=2, max_pages=2, device="cpu")
        args.update(kw)
        with pytest.raises(ValueError):
            pc.PagedKVCache(**args)


def test_attention_refuses_an_fp32_result_off_eight_bytes():
    L = _lib.lib()
    f = dict(q_row_stride=128, q_head_stride=128, table_stride=8, k_codes=16, v_codes=16, dtype=_lib.DT_F32, batch=2,
             block=3, n_heads=8, n_kv=2, head_dim=128, page_size=64, n_pages=4, max_pages=8, k_scale=4, v_scale=4)
    assert L.dsm_gqa_attn_kv8(ctypes.byref(_lib.KV8AttnDesc(**f)), 4, 4, 4, None, None, 4, 16, 1 << 30, None) != 0
    assert "out must be 8-byte aligned" in L.dsm_last_error_message().decode()


def test_attention_refuses_more_rows_than_32_bits_count():
    L = _lib.lib()
    assert L.dsm_gqa_attn_kv8_workspace_bytes(1, 1 << 16, 1 << 15, 1, 64) == 0
    assert L.dsm_gqa_attn_kv8_workspace_bytes(1, 1 << 16, (1 << 15) - 1, 1, 64) > 0
    assert _attn(L, block=1 << 16, n_heads=1 << 15, n_kv=1) != 0
    assert "too many rows" in L.dsm_last_error_message().decode()
