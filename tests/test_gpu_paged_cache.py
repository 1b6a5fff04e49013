"""The paged 8-bit KV cache on the GPU against its oracle (``oracle/paged_cache_oracle.py``).

Page tables and stored codes have to be equal. The attention's bound is derived from its
arithmetic. With u the type's half step (bf16 2^-8, fp32 2^-24), S = max sum_d |q_d k_d| * scale
and V = max |v| of a sequence:

* the result is rounded once: u |o|;
* a score that is off by ds moves each weight by a factor of e^ds, numerator and denominator alike:
  at most 2 ds V. bf16 calls split q into two e4m3 terms. A term's half step
  is 2^-4 of its value, so two leave 2^-8 |q_d|, and 2^-10 of e4m3's unit (its smallest step 2^-9,
  halved) of a row scaled to at least 224: 2^-17 max |q|; the products are exact and their fp32 sums
  add less than 2^-18 S. So ds <= (2^-8 + 2^-18) S in the worst case; but bf16's q has 8
  significant bits, a first term takes 4, the residual at most 4 with its sign, and is exact where it
  reaches e4m3's normals: 2^-17 max|q| sum|k| scale is what is left, held below 2^-17 * head_dim * S;
* the weights' terms leave less than 2^-8 of each, and 2^-18 of the largest of 64: at most
  (2^-8 + 2^-12) V, and their sum is taken before the rounding (three e5m2 terms of an f16 leave 2^-11 and 2^-29 of
  the largest: ``_close`` below holds each row to that);
* fp32 calls split into two f16 terms (2^-22 each), or use fp32 products: ds <= (2^-21 + (hd + 8)
  2^-24) S, weights 2^-21 + (n / 32 + 64) 2^-24 for n summed rows.
"""

from __future__ import annotations

import random

import pytest
import torch

import oracle
from dsm import _lib
from dsm import paged_cache as pc
from oracle import paged_cache_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------- page tables
def _tables_case(seed, b, page, longest, new_most, pool_extra, most=None, extra_cols=0):
    r = random.Random(seed)
    lengths = [r.choice([0, 1, page - 1, page, page + 1, r.randint(0, longest)]) for _ in range(b)]
    new = [r.choice([0, 0, 1, 2, page, r.randint(0, new_most)]) for _ in range(b)]
    need = [-(-n // page) for n in lengths]
    n_pages = sum(need) + pool_extra
    pool = list(range(n_pages))
    r.shuffle(pool)
    most = most or max(-(-(a + c) // page) for a, c in zip(lengths, new)) + 1
    table = [[-7] * most for _ in range(b)]
    for i, n in enumerate(need):
        for j in range(n):
            table[i][j] = pool.pop()
    free = pool + [-3] * (n_pages - len(pool))
    wide = torch.full((b, most + extra_cols), -9, dtype=torch.int32)
    wide[:, :most] = torch.tensor(table)
    return lengths, new, table, free, len(pool), wide.to(DEV)[:, :most]


def _run_extend(lengths, new, table_gpu, free, n_free, page, max_rows):
    L, F, N = i32(lengths), i32(free), i32([n_free])
    rows = pc.paged_extend(L, i32(new), table_gpu, F, N, page, max_rows)
    return L, F, N, rows


@pytest.mark.parametrize("b,page,longest,new_most,tail,extra_cols", [
    (1, 64, 300, 5, 0, 0), (1, 64, 0, 5000, 3, 0), (7, 128, 1000, 9, 5, 3), (61, 64, 700, 200, 40, 0),
    (513, 64, 300, 4, 1, 0), (1025, 256, 900, 300, 7, 5), (8192, 64, 130, 2, 100, 0),
])
def test_extend_and_trim_match_the_oracle(b, page, longest, new_most, tail, extra_cols):
    """One token to long prompts, one CTA and a cluster, one scan block and several, a strided table."""
    lengths, new, table, free, n_free, tg = _tables_case(b, b, page, longest, new_most, 3 * b + 200 + b * new_most // page,
                                                         extra_cols=extra_cols)
    max_rows = sum(new) + tail
    want = po.paged_extend(lengths, new, table, free, n_free, page, max_rows)
    assert not want[6]
    L, F, N, rows = _run_extend(lengths, new, tg, free, n_free, page, max_rows)
    assert L.tolist() == want[0] and tg.tolist() == want[1] and N.tolist() == [want[2]]
    assert rows.cu_rows.tolist() == want[3] and rows.slot_map.tolist() == want[4]
    assert rows.positions.tolist() == want[5] and F.tolist() == free
    # back to a mix of lengths: kept whole, cut, released, asked for more than there is
    r = random.Random(5)
    keep = [r.choice([n, n // 2, 0, n + 9, -4, max(0, n - 1)]) for n in want[0]]
    back = po.paged_trim(want[0], keep, want[1], free, want[2], page)
    pc.paged_trim(L, i32(keep), tg, F, N, page)
    assert L.tolist() == back[0] and F.tolist() == back[1] and N.tolist() == [back[2]] and not back[3]
    assert tg.tolist() == want[1]
    assert _lib.device_error() == 0


def test_extend_then_trim_to_the_old_lengths_restores_everything_but_the_table():
    lengths, new, table, free, n_free, tg = _tables_case(3, 40, 64, 500, 100, 200)
    L, F, N, _ = _run_extend(lengths, new, tg, free, n_free, 64, sum(new))
    pc.paged_trim(L, i32(lengths), tg, F, N, 64)
    assert (L.tolist(), F.tolist(), N.tolist()) == (lengths, free, [n_free])


@pytest.mark.parametrize("short", ["pages", "rows", "table", "negative length", "negative rows", "int32"])
def test_extend_leaves_out_what_does_not_fit(short):
    """Who finds no pages, rows or table keeps its length and gets no slots; those before it, and
    those after it that need nothing more, are served. The error word says so."""
    page = 64
    lengths, new, table, free, n_free, tg = _tables_case(11, 30, page, 300, 150, 60)
    new = [max(1, n) for n in new]
    lengths[4], new[4] = 10, 3  # fits its last page
    table[4][0] = table[4][0] if table[4][0] >= 0 else 0
    max_rows = sum(new)
    if short == "pages":
        n_free = 7
    elif short == "rows":
        max_rows = sum(new) // 2
    elif short == "table":
        most = 3
        lengths = [min(n, most * page) for n in lengths]
        table = [row[:most] for row in table]
    elif short == "negative length":
        lengths[2] = -5
    elif short == "negative rows":
        new[2] = -5
    else:
        new[2] = 2 ** 31 - 1
    tg = i32(table)
    want = po.paged_extend(lengths, new, table, free, n_free, page, max_rows)
    assert want[6]
    L, F, N, rows = _run_extend(lengths, new, tg, free, n_free, page, max_rows)
    assert L.tolist() == want[0] and tg.tolist() == want[1] and N.tolist() == [want[2]]
    assert rows.cu_rows.tolist() == want[3] and rows.slot_map.tolist() == want[4]
    assert rows.positions.tolist() == want[5]
    with pytest.raises(_lib.DsmError, match="ran out"):
        _lib.raise_device_error()


@pytest.mark.parametrize("short,page", [("pages", 64), ("pages", 192), ("rows", 1024), ("negative length", 128)])
def test_a_long_step_leaves_out_what_does_not_fit(short, page):
    """As above with more rows than one CTA writes; sequences without new rows lie between the others."""
    b = 90
    lengths, new, table, free, n_free, tg = _tables_case(7, b, page, 5 * page, 6 * page, 4 * b, most=14)
    new[3] = 5 * page
    max_rows = sum(new) + 11
    assert max_rows > 3000
    if short == "pages":
        n_free = 60
    elif short == "rows":
        max_rows = max_rows * 2 // 3
    else:
        lengths[3] = -1
    want = po.paged_extend(lengths, new, table, free, n_free, page, max_rows)
    assert want[6]
    L, F, N, rows = _run_extend(lengths, new, tg, free, n_free, page, max_rows)
    assert L.tolist() == want[0] and tg.tolist() == want[1] and N.tolist() == [want[2]]
    assert rows.cu_rows.tolist() == want[3] and rows.slot_map.tolist() == want[4]
    assert rows.positions.tolist() == want[5]
    with pytest.raises(_lib.DsmError, match="ran out"):
        _lib.raise_device_error()


def test_trim_refuses_more_pages_than_the_pool_holds():
    lengths, new, table, free, n_free, tg = _tables_case(2, 5, 64, 300, 1, 10)
    lengths = [64 * 3] * 5
    L, F, N = i32(lengths), i32(free), i32([len(free) - 2])
    pc.paged_trim(L, i32([0] * 5), tg, F, N, 64)
    assert L.tolist() == lengths and F.tolist() == free and N.tolist() == [len(free) - 2]
    with pytest.raises(_lib.DsmError):
        _lib.raise_device_error()


def test_empty_batch_and_no_rows():
    rows = pc.paged_extend(i32([]), i32([]), torch.empty(0, 4, dtype=torch.int32, device=DEV), i32([0, 1]), i32([2]), 64, 5)
    assert rows.cu_rows.tolist() == [0] and rows.slot_map.tolist() == [-1] * 5
    L, N = i32([3, 0]), i32([2])
    rows = pc.paged_extend(L, i32([0, 0]), i32([[0], [0]]), i32([0, 1]), N, 64, 0)
    assert L.tolist() == [3, 0] and rows.cu_rows.tolist() == [0, 0, 0] and rows.slot_map.numel() == 0
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------- append
def _pool(seed, n_pages, n_kv, page, hd, e_lo=-9, e_hi=3):
    """A pool by token: code values (no NaN), scales; and its stored form on the GPU."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        codes = po.round_e4m3((torch.randn(n_pages, n_kv, page, hd, generator=g) * 100).clamp(-448, 448).double())
        scale = torch.exp2(torch.randint(e_lo, e_hi, (n_pages, n_kv), generator=g).double())
        out.append((codes, scale))
    (k, ks), (v, vs) = out
    layer = pc.KV8Layer(_codes(po.store_keys(k)), _codes(po.store_values(v)), ks.float().to(DEV), vs.float().to(DEV))
    return k, ks, v, vs, layer


def _codes(values):
    """fp64 e4m3 values -> uint8 codes on the GPU."""
    return values.float().to(torch.float8_e4m3fn).view(torch.uint8).contiguous().to(DEV)


def _loaded(layer):
    f = lambda t: t.view(torch.float8_e4m3fn).float().double().cpu()  # noqa: E731
    return po.load_keys(f(layer.k_codes)), po.load_values(f(layer.v_codes)), layer.k_scale.double().cpu(), \
        layer.v_scale.double().cpu()


def _same(a, b):
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _check_append(layer, pool, k, v, slots):
    kc, ks, vc, vs = pool
    pc.kv8_append(layer, k.to(DEV) if not k.is_cuda else k, v.to(DEV) if not v.is_cuda else v,
                  torch.tensor(slots, dtype=torch.int64, device=DEV))
    wk, wks = po.kv8_append(kc, ks, k.double().cpu(), slots)
    wv, wvs = po.kv8_append(vc, vs, v.double().cpu(), slots)
    gk, gv, gks, gvs = _loaded(layer)
    assert torch.equal(gks, wks) and torch.equal(gvs, wvs)
    assert _same(gk, wk) and _same(gv, wv)
    return wk, wks, wv, wvs


def _runs(r, n_pages, page, n_runs, most, skip=0.1):
    """Slots of neighbouring rows page by page, as several sequences leave them, some rows without."""
    slots = []
    for pg in r.sample(range(n_pages), n_runs):
        first = r.choice([0, 0, r.randrange(page)])
        n = r.randint(1, min(most, page - first))
        slots += [pg * page + first + j for j in range(n)]
        if r.random() < skip:
            slots.append(-1)
    return slots


@pytest.mark.parametrize("dtype,hd,page,n_kv,n_runs,most", [
    (torch.bfloat16, 128, 64, 2, 1, 1), (torch.bfloat16, 128, 64, 8, 7, 64), (torch.bfloat16, 64, 128, 3, 6, 100),
    (torch.bfloat16, 256, 64, 1, 5, 9), (torch.float32, 128, 256, 2, 4, 256), (torch.float32, 64, 64, 1, 6, 3),
    (torch.float32, 256, 128, 2, 3, 128), (torch.bfloat16, 128, 1024, 1, 2, 700), (torch.bfloat16, 128, 64, 2, 40, 64),
])
def test_append_matches_the_oracle(dtype, hd, page, n_kv, n_runs, most):
    r = random.Random(hd + page + n_runs)
    n_pages = n_runs + 3
    k, ks, v, vs, layer = _pool(hd, n_pages, n_kv, page, hd)
    slots = _runs(r, n_pages, page, n_runs, most) + [-1, -1]
    g = torch.Generator().manual_seed(page)
    # rows from far below the pages' scales to far above them: kept, grown and fresh scales
    mag = torch.exp2(torch.randint(-14, 14, (len(slots), n_kv, 1), generator=g).float())
    rk = (torch.randn(len(slots), n_kv, hd, generator=g) * mag).to(dtype)
    rv = (torch.randn(len(slots), n_kv, hd, generator=g) * mag.flip(0)).to(dtype)
    pool = _check_append(layer, (k, ks, v, vs), rk, rv, slots)
    # the same rows again: nothing moves but pages that start afresh with the same rows
    _check_append(layer, (pool[0], pool[1], pool[2], pool[3]), rk, rv, slots)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype,hd,page,n_kv,longest", [
    (torch.bfloat16, 64, 64, 16, 1), (torch.bfloat16, 128, 64, 8, 40), (torch.float32, 64, 1024, 8, 1024),
    (torch.bfloat16, 64, 1024, 8, 1024), (torch.bfloat16, 256, 192, 8, 192),
])
def test_append_of_many_rows(dtype, hd, page, n_kv, longest):
    """Rows enough for windows of 64: runs of a row each, of a warp's size and longer ones side by side, and
    runs that pass the window and the 256 rows behind its start, in order and not."""
    r = random.Random(page + longest)
    rows = 64 * (4 * 148 // n_kv + 9)
    slots, n_pages = [], 0
    while len(slots) < rows:
        n = r.choice([1, 2, r.randint(1, longest), r.randint(1, longest), longest])
        first = r.randint(0, page - n)
        run = [n_pages * page + first + j for j in range(n)]
        if r.random() < 0.2:
            r.shuffle(run)
        slots += run + [-1] * (r.random() < 0.1)
        n_pages += 1
    k, ks, v, vs, layer = _pool(hd, n_pages, n_kv, page, hd)
    g = torch.Generator().manual_seed(page)
    mag = torch.exp2(torch.randint(-14, 14, (len(slots), 1, 1), generator=g).float())
    rk, rv = ((torch.randn(len(slots), n_kv, hd, generator=g) * mag).to(dtype) for _ in range(2))
    _check_append(layer, (k, ks, v, vs), rk, rv, slots)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("where", [0, 5, 8, 15, 16, 17, 63])
def test_append_infinities_anywhere_in_a_run(where):
    """An infinity or NaN takes no part in the scale, wherever its row and column fall in a run."""
    k, ks, v, vs, layer = _pool(2, 3, 2, 64, 128)
    g = torch.Generator().manual_seed(where)
    rk, rv = (torch.randn(70, 2, 128, generator=g).bfloat16() for _ in range(2))
    rk[where, 1, 127 - where], rk[where, 0, where] = float("inf"), float("nan")
    rv[where, 0, where], rv[where + 1, 1, 7] = float("-inf"), float("nan")
    _check_append(layer, (k, ks, v, vs), rk, rv, list(range(64)) + list(range(150, 156)))


@pytest.mark.parametrize("order", ["head first", "interleaved", "offset", "broadcast rows"])
def test_append_takes_any_row_and_head_strides(order):
    n, n_kv, hd, page = 70, 2, 128, 64
    k, ks, v, vs, layer = _pool(4, 4, n_kv, page, hd)
    slots = list(range(30, 64)) + list(range(128, 164))
    g = torch.Generator().manual_seed(0)
    base = torch.randn(2, 400, 400, generator=g).bfloat16().to(DEV)
    if order == "head first":
        rk, rv = (torch.randn(n_kv, n, hd, generator=g).bfloat16().to(DEV).transpose(0, 1) for _ in range(2))
    elif order == "interleaved":  # q | k | v columns of one projection
        rows = torch.randn(n, 3 * n_kv * hd, generator=g).bfloat16().to(DEV)
        rk, rv = (rows[:, c * n_kv * hd:(c + 1) * n_kv * hd].unflatten(1, (n_kv, hd)) for c in (1, 2))
    elif order == "offset":  # rows that start on two bytes
        rk, rv = (base[c, :, 1:].as_strided((n, n_kv, hd), (400, 129, 1), base[c].storage_offset() + 1) for c in (0, 1))
    else:
        rk, rv = (base[c, 0, :hd].expand(n, n_kv, hd) for c in (0, 1))
    _check_append(layer, (k, ks, v, vs), rk, rv, slots)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_borders_and_what_is_not_finite(dtype):
    """Maxima at 448 * 2^e and a step to either side, all-zero rows, the type's largest and smallest values,
    values halfway between codes, infinities and NaN."""
    hd, page, n_kv = 64, 64, 1
    tops = [448.0, 449.0, 450.0, 447.0, 3.5, 3.515625, 7 * 2.0 ** 100, 0.0, 1e-38, 2.0 ** -126, 2.0 ** -133,
            torch.finfo(dtype).max, float("inf"), float("nan"), 1.0]
    k, ks, v, vs, layer = _pool(9, len(tops), n_kv, page, hd)
    vals = po.e4m3_values()[:127]
    ties = (vals[:-1] + vals[1:]) / 2
    rows, slots = [], []
    for i, top in enumerate(tops):
        x = torch.zeros(2, n_kv, hd, dtype=torch.float64)
        x[0, 0, 0] = top
        x[1, 0, 1:] = ties[2 * torch.arange(63)] * (1.0 if 440 <= top <= 450 or not abs(top) < 1e39 else 0.0)
        x[1, 0, 3] = -top
        rows.append(x)
        slots += [i * page + (0 if i % 2 else 5), i * page + 6]
    rows = torch.cat(rows).to(dtype)
    _check_append(layer, (k, ks, v, vs), rows, rows.flip(2), slots)
    assert _lib.device_error() == 0


def test_append_skips_slots_outside_the_pool_and_says_so():
    n_kv, hd, page = 2, 128, 64
    k, ks, v, vs, layer = _pool(1, 2, n_kv, page, hd)
    rk = torch.randn(5, n_kv, hd).bfloat16()
    slots = [3, 2 * page, 2 ** 40, -5, page + 1]
    _check_append(layer, (k, ks, v, vs), rk, rk * 2, slots)
    with pytest.raises(_lib.DsmError, match="outside the pool"):
        _lib.raise_device_error()


def test_append_slots_past_32_bits():
    """A pool whose codes pass 2^32 bytes: the last page is written, the rest stays."""
    n_pages, n_kv, page, hd = 2200, 8, 1024, 256
    try:
        codes = torch.zeros(2, n_pages, n_kv, page, hd, dtype=torch.uint8, device=DEV)
    except torch.OutOfMemoryError:
        pytest.skip("no room for the pool")
    layer = pc.KV8Layer(codes[0], codes[1].view(n_pages, n_kv, page // 64, hd, 64),
                        torch.ones(n_pages, n_kv, device=DEV), torch.ones(n_pages, n_kv, device=DEV))
    rk = torch.randn(3, n_kv, hd, generator=torch.Generator().manual_seed(2)).bfloat16()
    slots = [(n_pages - 1) * page + j for j in range(3)]
    pc.kv8_append(layer, rk.to(DEV), rk.to(DEV), torch.tensor(slots, device=DEV))
    last = pc.KV8Layer(*(t[-1:] for t in layer))
    zero = torch.zeros(1, n_kv, page, hd, dtype=torch.float64)
    wk, wks = po.kv8_append(zero, torch.ones(1, n_kv, dtype=torch.float64), rk.double(), [0, 1, 2])
    gk, gv, gks, _ = _loaded(last)
    assert _same(gk, wk) and _same(gv, wk) and torch.equal(gks, wks)
    assert int(codes[:, :-1].max()) == 0


# ------------------------------------------------------------------------------- attention
def _attn_case(seed, lengths, s, n_kv, group, hd, page, dtype, with_block=True, q_mag=1.0, poison=True, cols=0, extra=2,
               e_lo=-9, e_hi=-4):
    """A pool of shuffled pages; whatever no sequence may read is NaN: codes behind the lengths, unused
    pages and their scales."""
    r = random.Random(seed)
    need = [-(-n // page) for n in lengths]
    n_pages = sum(need) + extra
    k, ks, v, vs, layer = _pool(seed, n_pages, n_kv, page, hd, e_lo, e_hi)
    pool = list(range(n_pages))
    r.shuffle(pool)
    most = max(1, max(need)) + 1
    table = [[-1] * most for _ in need]
    kept = torch.zeros(n_pages, page, dtype=torch.bool)
    for i, n in enumerate(lengths):
        for j in range(need[i]):
            table[i][j] = pool.pop()
            kept[table[i][j], :min(page, n - j * page)] = True
    if poison:
        nan = torch.full((), float("nan"), dtype=torch.float64)
        m = kept[:, None, :, None]
        k, v = torch.where(m, k, nan), torch.where(m, v, nan)
        ks[pool], vs[pool] = float("nan"), float("nan")
        layer = pc.KV8Layer(_codes(po.store_keys(k)), _codes(po.store_values(v)), ks.float().to(DEV),
                            vs.float().to(DEV))
    g = torch.Generator().manual_seed(seed + 1)
    b = len(lengths)
    q = (torch.randn(b, s, n_kv * group, hd, generator=g) * q_mag).to(dtype)
    blk = [torch.randn(b, n_kv, s, hd, generator=g).to(dtype) if with_block else None for _ in range(2)]
    wide = torch.full((b, most + cols), -1, dtype=torch.int32)
    wide[:, :most] = torch.tensor(table)
    return dict(q=q, layer=layer, table=table, tg=wide.to(DEV)[:, :most], lengths=lengths, blk=blk,
                k=k * ks[..., None, None], v=v * vs[..., None, None], hd=hd)


def _bound(dtype, ref, score, vmax, hd, n):
    s, v = score[:, None, None], vmax[:, None, None]
    if dtype == torch.bfloat16:
        ds = (2.0 ** -17 * hd + 2.0 ** -18) * s
        return 2.0 ** -8 * ref.abs() + (2 * ds + 2.0 ** -8 + 2.0 ** -12) * v
    ds = (2.0 ** -21 + (hd + 8) * 2.0 ** -24) * s
    return 2.0 ** -24 * ref.abs() + (2 * ds + 2.0 ** -21 + (n / 32 + 64) * 2.0 ** -24) * v


def _check_attn(c, scale=None, out=None, lengths=None, norm=None):
    scale = c["hd"] ** -0.5 if scale is None else scale
    lengths = c["lengths"] if lengths is None else lengths
    blk = [None if t is None else t.to(DEV) for t in c["blk"]]
    if out is None:
        out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(lengths), *blk, scale=scale)
    ref, score, vmax = po.kv8_attention(c["q"], c["k"], c["v"], c["table"], lengths, *c["blk"], scale)
    got = out.double().cpu()
    assert got.shape == ref.shape and out.dtype == c["q"].dtype
    assert torch.isfinite(got).all()
    err = (got - ref).abs()
    tol = _bound(c["q"].dtype, ref, score, vmax, c["hd"], max(lengths) + c["q"].shape[1])
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-30)).max())
    if norm is not None:
        assert float(err.norm()) <= norm * float(ref.norm()), float(err.norm() / ref.norm())
    return out


BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype,lengths,s,n_kv,group,hd,page,with_block", [
    (BF, [1], 1, 1, 1, 128, 64, False), (BF, [150], 1, 8, 4, 128, 64, True), (BF, [0], 7, 2, 4, 128, 64, True),
    (BF, [0, 5, 0], 1, 2, 4, 128, 64, False), (BF, [64, 63, 65, 128, 1, 0], 7, 2, 4, 128, 64, True),
    (BF, [700, 3, 1999, 0, 320], 7, 2, 4, 128, 64, True), (BF, [1000, 77], 7, 2, 8, 64, 64, True),
    (BF, [513, 300], 5, 1, 3, 256, 128, True), (BF, [256, 255, 257], 2, 2, 1, 64, 256, True),
    (BF, [2050], 16, 1, 8, 128, 128, True), (BF, [300, 90], 33, 1, 4, 128, 64, True),
    (BF, [600, 1], 70, 1, 2, 64, 64, True), (BF, [3000], 1, 2, 16, 128, 1024, False), (BF, [129] * 40, 3, 4, 2, 128, 64, True),
    (F32, [150, 0, 1], 1, 2, 4, 128, 64, True), (F32, [64, 63, 700], 5, 2, 4, 128, 64, True),
    (F32, [333, 2], 7, 1, 8, 64, 128, False), (F32, [500, 40], 5, 1, 4, 256, 64, True),
    (F32, [1300], 33, 1, 3, 128, 256, True),
])
def test_attention_matches_the_oracle(dtype, lengths, s, n_kv, group, hd, page, with_block):
    c = _attn_case(sum(lengths) + s, lengths, s, n_kv, group, hd, page, dtype, with_block)
    # over all values: a rounding's error is at most u and u / sqrt(3) on the average; the weights' terms and
    # sums stay below as much again (bf16 2^-8 each, of random sign; fp32 some 2^-22)
    out = _check_attn(c, norm=2.0 ** -8 if dtype == BF else 2.0 ** -20)
    if not with_block:
        for i, n in enumerate(lengths):
            assert n > 0 or int(out[i].count_nonzero()) == 0  # nothing to attend to: zeros
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype,q_mag,e_lo,e_hi,scale", [
    (BF, 30.0, -9, -4, None),   # peaked: a few keys carry everything
    (BF, 1.0, -30, 20, 2.0 ** -26),  # page scales fifty octaves apart
    (BF, 2.0 ** -100, -9, -4, 2.0 ** 95), (BF, 2.0 ** 100, -9, -4, 2.0 ** -105),
    (F32, 30.0, -9, -4, None), (F32, 1.0, -30, 20, 2.0 ** -26), (F32, 2.0 ** -100, -9, -4, 2.0 ** 95),
    (BF, 1.0, -9, -4, 0.0), (BF, 1.0, -9, -4, -0.7),
])
def test_attention_magnitudes(dtype, q_mag, e_lo, e_hi, scale):
    c = _attn_case(3, [500, 64, 1], 5, 2, 4, 128, 64, dtype, with_block=e_hi < 0 and q_mag < 2.0 ** 90, q_mag=q_mag,
                   e_lo=e_lo, e_hi=e_hi)
    _check_attn(c, scale)


def test_attention_rows_of_very_different_size():
    """Query rows 2^60 apart in one call: each row has its own scale."""
    c = _attn_case(5, [200, 90], 7, 2, 4, 128, 64, BF)
    c["q"] = (c["q"].float() * torch.exp2(-torch.arange(7.0) * 10)[None, :, None, None]).bfloat16()
    _check_attn(c)
    c["q"][:, 3] = 0
    _check_attn(c)


def test_attention_sink_over_a_long_tail():
    """One key 2^15 times heavier than each of 16384 others: the tail carries a third of the weight."""
    hd, n = 64, 16384
    c = _attn_case(8, [n], 1, 1, 2, hd, 64, BF, with_block=False, e_lo=-6, e_hi=-5)
    kd = torch.zeros(hd, dtype=torch.float64)
    kd[0] = 1.0
    k = torch.zeros_like(c["k"])
    sink = c["table"][0][0]
    k[sink, 0, 0] = kd
    c["k"] = k
    codes = po.round_e4m3(k * 2.0 ** 6)
    c["layer"].k_codes.copy_(_codes(po.store_keys(codes)))
    c["layer"].k_scale.fill_(2.0 ** -6)
    c["q"] = torch.zeros_like(c["q"])
    c["q"][..., 0] = 10.375  # e^10.375 ~ 2^15
    _check_attn(c, scale=1.0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_takes_strided_inputs(dtype):
    c = _attn_case(12, [300, 65, 1], 5, 2, 4, 128, 64, dtype, cols=3)
    b, s, nh, hd = c["q"].shape
    ref = _check_attn(c)
    rows = torch.zeros(b * s, nh * hd + 2 * 2 * hd + 1, dtype=dtype, device=DEV)  # q | k | v columns, odd row length
    rows[:, :nh * hd] = c["q"].reshape(b * s, -1).to(DEV)
    for j in (0, 1):
        rows[:, nh * hd + j * 2 * hd:][:, :2 * hd] = c["blk"][j].transpose(1, 2).reshape(b * s, -1).to(DEV)
    q = rows[:, :nh * hd].view(b, s, nh, hd)
    bk, bv = (rows[:, nh * hd + j * 2 * hd:][:, :2 * hd].view(b, s, 2, hd).transpose(1, 2) for j in (0, 1))
    out = pc.gqa_attention_kv8(q, c["layer"], c["tg"], i32(c["lengths"]), bk, bv)
    assert torch.equal(out, ref)
    one = c["q"][:1].to(DEV).expand(b, s, nh, hd)  # the same rows for every sequence
    want = pc.gqa_attention_kv8(one.contiguous(), c["layer"], c["tg"], i32(c["lengths"]), bk, bv)
    assert torch.equal(pc.gqa_attention_kv8(one, c["layer"], c["tg"], i32(c["lengths"]), bk, bv), want)


def test_attention_is_the_same_twice_and_on_another_stream():
    c = _attn_case(1, [1500, 3, 700, 0, 64], 7, 2, 4, 128, 64, BF)
    a = _check_attn(c)
    blk = [t.to(DEV) for t in c["blk"]]
    q, n = c["q"].to(DEV), i32(c["lengths"])
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(4):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                outs.append(pc.gqa_attention_kv8(q, c["layer"], c["tg"], n, *blk))
    torch.cuda.synchronize()
    assert all(torch.equal(o, a) for o in outs)


@pytest.mark.parametrize("dtype,s,group,hd", [
    (BF, 1, 7, 128), (BF, 3, 4, 64), (BF, 5, 4, 128), (BF, 3, 8, 128), (BF, 5, 8, 256), (BF, 6, 8, 64), (BF, 17, 2, 128),
    (BF, 16, 4, 128), (BF, 13, 6, 256), (BF, 31, 4, 64), (BF, 64, 1, 128), (BF, 64, 3, 64), (BF, 65, 1, 128), (BF, 130, 2, 64),
    (F32, 1, 7, 128), (F32, 9, 4, 64), (F32, 16, 8, 128), (F32, 43, 3, 64), (F32, 23, 3, 256), (F32, 70, 2, 128),
])
def test_attention_any_number_of_query_rows(dtype, s, group, hd):
    """One row of a KV head to several blocks of them, blocks of own rows that fill a step and more, over a
    sequence that many CTAs share, a short one, one of its own rows alone and one that ends at a page."""
    c = _attn_case(s * group + hd, [2500, 70, 0, 256], s, 2, group, hd, 64, dtype)
    _check_attn(c, norm=2.0 ** -8 if dtype == BF else 2.0 ** -20)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype,lengths,s,page,with_block", [
    (BF, [700, 0, 64, 1], 3, 64, True), (F32, [700, 0, 64, 1], 3, 128, True), (BF, [333], 1, 64, False),
])
def test_attention_on_the_cuda_cores(dtype, lengths, s, page, with_block):
    L = _lib.lib()
    c = _attn_case(9, lengths, s, 2, 4, 128, page, dtype, with_block)
    a = _check_attn(c)
    _lib.check(L.dsm_set_attn_kernel(1))
    try:
        b = _check_attn(c)
    finally:
        _lib.check(L.dsm_set_attn_kernel(_lib.ATTN_KERNEL_DEFAULT))
    assert not torch.equal(a, b)  # another kernel, other roundings


@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 256), (F32, 128), (F32, 256)])
def test_attention_of_the_largest_batch(dtype, hd):
    r = random.Random(hd)
    lengths = [r.choice([0, 0, 1, 5, 64, 65, 130]) for _ in range(8192)]
    c = _attn_case(5, lengths, 1, 1, 2, hd, 64, dtype)
    _check_attn(c)
    assert _lib.device_error() == 0


def test_attention_pages_of_unlike_scales_within_a_step():
    """A step takes two groups of 64 keys: pages with scales 2^25 apart, and pages that are none, in either half."""
    c = _attn_case(4, [640, 600, 200], 5, 2, 4, 128, 64, BF, e_lo=-24, e_hi=2)
    _check_attn(c, scale=2.0 ** -12)
    for i, cols in ((0, (1, 4)), (1, (0, 9)), (2, (2,))):
        for j in cols:
            c["table"][i][j] = -1 if j % 2 else 10 ** 6
    c["tg"].copy_(torch.tensor(c["table"], dtype=torch.int32))
    _check_attn(c, scale=2.0 ** -12)
    with pytest.raises(_lib.DsmError, match="outside the pool"):
        _lib.raise_device_error()


def test_two_captured_attentions_replay_side_by_side():
    """Two graphs, each with its own workspace, on two streams at once, over and over."""
    cases = [_attn_case(i, n, s, 2, 4, 128, 64, BF) for i, (n, s) in enumerate((([3000, 9], 7), ([700, 0, 4000], 3)))]
    want, graphs, outs = [], [], []
    for c in cases:
        want.append(_check_attn(c))
        args = [c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]), *[t.to(DEV) for t in c["blk"]]]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pc.gqa_attention_kv8(*args))
        graphs.append((g, args))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_attention_bad_tables_are_skipped_and_reported():
    """Pages outside the pool count as absent; a length past the table is cut to it."""
    c = _attn_case(7, [200, 130], 3, 1, 2, 128, 64, BF)
    c["table"][0][1] = 10 ** 6
    c["table"][1][0] = -2
    c["tg"] = i32(c["table"])
    _check_attn(c)
    with pytest.raises(_lib.DsmError, match="outside the pool"):
        _lib.raise_device_error()
    c = _attn_case(7, [200, 130], 3, 1, 2, 128, 64, BF)
    most = len(c["table"][0])
    for row in c["table"]:
        row[:] = [p if p >= 0 else row[0] for p in row]
    c["tg"] = i32(c["table"])
    c["k"], c["v"] = torch.nan_to_num(c["k"]), torch.nan_to_num(c["v"])
    for t in (c["layer"].k_codes, c["layer"].v_codes):
        t[(t & 127) == 127] = 0
    _check_attn(c, lengths=[most * 64 + 1000, 130])
    assert _lib.device_error() == 0x15
    _check_attn(c, lengths=[-3, 130])
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_passes_nan_of_its_own_rows_on(dtype):
    """A NaN among the rows that a sequence does read reaches its outputs, and no other sequence's."""
    c = _attn_case(2, [200, 90], 2, 1, 2, 128, 64, dtype)
    c["layer"].v_codes[c["table"][0][1], 0, 0, 5, 7] = 0x7F
    out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]),
                               *(t.to(DEV) for t in c["blk"])).view(2, 2, 2, 128)
    assert bool(out[0, :, :, 5].isnan().all()) and bool(torch.isfinite(out[1]).all())
    assert bool(torch.isfinite(out[0, :, :, :5]).all()) and bool(torch.isfinite(out[0, :, :, 6:]).all())
    q = c["q"].clone()
    q[1, 1, 0, 3] = float("inf")
    out = pc.gqa_attention_kv8(q.to(DEV), c["layer"], c["tg"], i32(c["lengths"]),
                               *(t.to(DEV) for t in c["blk"])).view(2, 2, 2, 128)
    assert bool(out[1, 1, 0].isnan().all()) and bool(torch.isfinite(out[1, 0]).all())
    assert bool(torch.isfinite(out[1, 1, 1]).all())


def test_attention_offsets_past_32_bits():
    """Pages behind 2^32 bytes of codes."""
    n_pages, n_kv, page, hd = 2200, 8, 1024, 256
    try:
        codes = torch.zeros(2, n_pages, n_kv, page, hd, dtype=torch.uint8, device=DEV)
    except torch.OutOfMemoryError:
        pytest.skip("no room for the pool")
    k, ks, v, vs, small = _pool(3, 2, n_kv, page, hd, -9, -4)
    layer = pc.KV8Layer(codes[0], codes[1].view(n_pages, n_kv, page // 64, hd, 64),
                        torch.full((n_pages, n_kv), float("nan"), device=DEV),
                        torch.full((n_pages, n_kv), float("nan"), device=DEV))
    for t, u in zip(layer, small):
        t[-2:] = u
    c = dict(q=torch.randn(1, 2, n_kv * 2, hd, generator=torch.Generator().manual_seed(0)).bfloat16(), layer=small,
             table=[[1, 0]], tg=i32([[1, 0]]), lengths=[1500], blk=[None, None], k=k * ks[..., None, None],
             v=v * vs[..., None, None], hd=hd)
    want = _check_attn(c)
    out = pc.gqa_attention_kv8(c["q"].to(DEV), layer, i32([[n_pages - 1, n_pages - 2]]), i32([1500]))
    assert torch.equal(out, want)


# ------------------------------------------------------------------------------- together
def test_a_run_of_steps_matches_the_oracle():
    """Five steps of a batch on one cache: extend, append, attend, trim, with a sequence that is released and its
    place taken by another, against a cache kept by the oracle."""
    r = random.Random(0)
    b, n_kv, group, hd, page, n_pages, most = 5, 2, 4, 128, 64, 24, 6
    cache = pc.PagedKVCache(2, n_pages, n_kv, hd, b, most, page_size=page)
    cache.k_codes.fill_(0xFF)
    cache.v_codes.fill_(0xFF)
    lengths, table = [0] * b, [[-1] * most for _ in range(b)]
    free, n_free = list(range(n_pages - 1, -1, -1)), n_pages
    state = {}
    for kind in ("k", "v"):
        state[kind] = (torch.full((n_pages, n_kv, page, hd), float("nan"), dtype=torch.float64),
                       torch.full((n_pages, n_kv), 2.0 ** -120, dtype=torch.float64))
    g = torch.Generator().manual_seed(1)
    for step in range(5):
        new = [r.choice([0, 1, 7, 70]) if step else r.randint(1, 130) for _ in range(b)]
        max_rows = sum(new) + 2
        rows = cache.extend(i32(new), max_rows)
        lengths, table, n_free, cu, slots, pos, failed = po.paged_extend(lengths, new, table, free, n_free, page, max_rows)
        assert not failed and rows.slot_map.tolist() == slots and cache.lengths.tolist() == lengths
        x = [torch.randn(max_rows, n_kv, hd, generator=g).bfloat16() * 2.0 ** step for _ in range(2)]
        cache.append(1, x[0].to(DEV), x[1].to(DEV), rows)
        for kind, t in zip(("k", "v"), x):
            state[kind] = po.kv8_append(*state[kind], t.double(), slots)
        k, v = (state[n][0] * state[n][1][..., None, None] for n in ("k", "v"))
        q = torch.randn(b, 3, n_kv * group, hd, generator=g).bfloat16() * 2.0 ** -step
        blk = [torch.randn(b, n_kv, 3, hd, generator=g).bfloat16() for _ in range(2)]
        out = cache.attend(1, q.to(DEV), *(t.to(DEV) for t in blk))
        _check_attn(dict(q=q, k=k, v=v, table=table, lengths=lengths, blk=blk, hd=hd), out=out)
        keep = [max(0, n - r.choice([0, 0, 3, 66])) for n in lengths]
        if step == 2:
            keep[1] = 0
        cache.trim(i32(keep))
        lengths, free, n_free, failed = po.paged_trim(lengths, keep, table, free, n_free, page)
        assert not failed and cache.lengths.tolist() == lengths and cache.n_free.tolist() == [n_free]
    assert _lib.device_error() == 0


def test_a_captured_step_replays_as_the_lengths_change():
    """extend, append, attend captured once; every replay grows the same cache, as eager calls grow another.
    Two graphs replay on one cache in turn."""
    b, n_kv, group, hd, page = 3, 2, 4, 128, 64
    caches = [pc.PagedKVCache(1, 30, n_kv, hd, b, 8, page_size=page) for _ in range(2)]
    g = torch.Generator(device=DEV).manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    new, x, q, blk = i32([0] * b), [mk(60, n_kv, hd) for _ in range(2)], mk(b, 4, n_kv * group, hd), \
        [mk(b, n_kv, 4, hd) for _ in range(2)]

    def step(cache):
        rows = cache.extend(new, 60)
        cache.append(0, *x, rows)
        return cache.attend(0, q, *blk)

    step(caches[0])  # kernels loaded; nothing is added
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(caches[0])
        graphs.append((gr, out))
    r = random.Random(3)
    for i in range(10):
        new.copy_(i32([r.randint(0, 20) for _ in range(b)]))
        for t in (*x, q, *blk):
            t.copy_(torch.randn(t.shape, generator=g, device=DEV))
        gr, out = graphs[i % 2]
        gr.replay()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert torch.equal(caches[0].lengths, caches[1].lengths) and torch.equal(caches[0].n_free, caches[1].n_free)
        assert torch.equal(caches[0].block_table, caches[1].block_table)
    assert int(caches[0].lengths.sum()) > 0 and _lib.device_error() == 0
    del graphs, gr


def test_a_captured_prefill_replays():
    """A step of more rows than one CTA writes, captured: extend's two kernels, append and attend, then a trim."""
    b, n_kv, hd, page, most = 40, 2, 64, 64, 4000
    caches = [pc.PagedKVCache(1, 400, n_kv, hd, b, 40, page_size=page) for _ in range(2)]
    g = torch.Generator(device=DEV).manual_seed(1)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    new, keep = i32([0] * b), i32([0] * b)
    x, q = [mk(most, n_kv, hd) for _ in range(2)], mk(b, 2, n_kv * 4, hd)

    def step(cache):
        rows = cache.extend(new, most)
        cache.append(0, *x, rows)
        out = cache.attend(0, q)
        cache.trim(keep)
        return out, rows

    step(caches[0])
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out, rows = step(caches[0])
    r = random.Random(8)
    for i in range(6):
        new.copy_(i32([r.choice([0, 1, r.randint(0, 130)]) for _ in range(b)]))
        keep.copy_(i32([r.choice([0, 70, 10 ** 6]) for _ in range(b)]))
        gr.replay()
        want, want_rows = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        assert all(torch.equal(a, c) for a, c in zip(rows, want_rows))
        assert torch.equal(caches[0].lengths, caches[1].lengths) and torch.equal(caches[0].n_free, caches[1].n_free)
        assert torch.equal(caches[0].free_pages, caches[1].free_pages)
    assert _lib.device_error() == 0
    del gr


@pytest.mark.parametrize("dtype", [BF, F32])
def test_qwen3_layer_over_the_paged_cache(dtype):
    """``append_paged`` + ``forward_paged`` of a Qwen3 draft layer for sequences of different lengths against the
    oracle's layer, one sequence at a time over the rows that the cache gives back: the 8-bit rounding of the context
    is in both. Tolerances are those of the dense layer's tests (bf16 2e-2, fp32 5e-3 of the largest value)."""
    from dsm.qwen3_attention import rope_tables
    from dsm.qwen3_layer import Qwen3DSparkLayer
    from helpers import max_rel_err

    b, s, h, nh, nkv, hd, inter, page, theta, eps = 3, 5, 256, 8, 2, 128, 256, 64, 1e6, 1e-6
    args = dict(hidden_size=h, num_attention_heads=nh, num_key_value_heads=nkv, head_dim=hd, rms_norm_eps=eps,
                intermediate_size=inter)
    g = torch.Generator().manual_seed(0)
    rnd = lambda *sh, std=1.0: (torch.randn(*sh, generator=g) * std).to(dtype)  # noqa: E731
    w = {"q_proj": rnd(nh * hd, h, std=h ** -0.5), "k_proj": rnd(nkv * hd, h, std=h ** -0.5),
         "v_proj": rnd(nkv * hd, h, std=h ** -0.5), "o_proj": rnd(h, nh * hd, std=(nh * hd) ** -0.5),
         "gate_proj": rnd(inter, h, std=h ** -0.5), "up_proj": rnd(inter, h, std=h ** -0.5),
         "down_proj": rnd(h, inter, std=inter ** -0.5)}
    layer = Qwen3DSparkLayer(args).to(DEV)
    for n in ("q_proj", "k_proj", "v_proj", "o_proj"):
        getattr(layer.self_attn, n).weight = torch.nn.Parameter(w[n].to(DEV), requires_grad=False)
    for n in ("gate_proj", "up_proj", "down_proj"):
        getattr(layer.mlp, n).weight = torch.nn.Parameter(w[n].to(DEV), requires_grad=False)
    cache = pc.PagedKVCache(1, 20, nkv, hd, b, 5, page_size=page)
    cos_t, sin_t = rope_tables(torch.arange(400), hd, theta)
    cos_t, sin_t = cos_t.to(DEV), sin_t.to(DEV)
    total = [0] * b
    for new in ([130, 0, 64], [3, 1, 0], [0, 0, 70]):
        max_rows = sum(new) + 1
        rows = cache.extend(i32(new), max_rows)
        pos = rows.positions.long()
        layer.append_paged(rnd(max_rows, h).to(DEV), cos_t[pos], sin_t[pos], cache, 0, rows)
        total = [a + c for a, c in zip(total, new)]
    assert cache.lengths.tolist() == total
    hidden = rnd(b, s, h)
    at = torch.tensor([[n + j for j in range(s)] for n in total])
    out = layer.forward_paged(hidden.to(DEV), cache, 0, cos_t[at.flatten().to(DEV)], sin_t[at.flatten().to(DEV)])
    p = {"self_attn": {n: w[n] for n in ("q_proj", "k_proj", "v_proj", "o_proj")}}
    p["self_attn"].update(q_norm=torch.ones(hd), k_norm=torch.ones(hd))
    params = dict(w, q_norm=torch.ones(hd), k_norm=torch.ones(hd), input_layernorm=torch.ones(h),
                  post_attention_layernorm=torch.ones(h))
    gk, gv, gks, gvs = _loaded(cache.layer(0))
    kd, vd = gk * gks[..., None, None], gv * gvs[..., None, None]
    table = cache.block_table.tolist()
    for i, n in enumerate(total):
        ck, cv = (torch.cat([x[table[i][j]] for j in range(-(-n // page))], 1)[None, :, :n].to(dtype) if n else None
                  for x in (kd, vd))
        ref = oracle.qwen3_layer_cached(params, nh, nkv, hd, eps, hidden[i:i + 1], ck, cv, cos_t[at[i].to(DEV)].cpu(),
                                        sin_t[at[i].to(DEV)].cpu())
        assert max_rel_err(out[i:i + 1], ref) < (2e-2 if dtype == BF else 5e-3), i
    assert _lib.device_error() == 0


def test_modules_refuse_caches_that_do_not_fit():
    from dsm.qwen3_attention import Qwen3DSparkAttention

    a = Qwen3DSparkAttention(dict(hidden_size=64, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                  rms_norm_eps=1e-6)).to(DEV)
    cache = pc.PagedKVCache(1, 4, 2, 64, 2, 2)
    cos = torch.zeros(6, 64)
    x = torch.zeros(2, 3, 64, device=DEV)
    rows = cache.extend(i32([1, 1]), 4)
    for bad in (lambda: a.attend_paged(x, pc.PagedKVCache(1, 4, 1, 64, 2, 2), 0, cos, cos),
                lambda: a.attend_paged(x, pc.PagedKVCache(1, 4, 2, 128, 2, 2), 0, cos, cos),
                lambda: a.attend_paged(x[:1], cache, 0, cos[:3], cos[:3]),
                lambda: a.attend_paged(x, cache, 0, cos[:3], cos[:3]),
                lambda: a.attend_paged(x.cpu(), cache, 0, cos, cos),
                lambda: a.append_paged(x[0], cos[:3], cos[:3], cache, 0, rows),
                lambda: a.append_paged(x, cos, cos, cache, 0, rows),
                lambda: cache.append(0, x[0].view(3, 1, 64), x[0].view(3, 1, 64), rows),
                lambda: cache.append(0, torch.zeros(4, 2, 64, device=DEV).half(),
                                     torch.zeros(4, 2, 64, device=DEV).half(), rows),
                lambda: cache.append(0, torch.zeros(4, 64, 2, device=DEV).transpose(1, 2),
                                     torch.zeros(4, 2, 64, device=DEV), rows),
                lambda: cache.attend(0, torch.zeros(2, 1, 3, 64, device=DEV)),
                lambda: cache.attend(0, torch.zeros(2, 1, 4, 64, device=DEV), torch.zeros(2, 2, 1, 64, device=DEV)),
                lambda: cache.attend(0, torch.zeros(2, 1, 4, 64, device=DEV, dtype=torch.float16)),
                lambda: cache.extend(i32([1]), 4), lambda: cache.extend(i32([1, 1]).long(), 4),
                lambda: cache.extend(i32([1, 1]), -1), lambda: cache.trim(i32([1, 1])[::2])):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------------------- alignment
def _placed(t, kind):
    """``t`` in memory that starts one element late, or whose rows are of odd length, or as it is."""
    if kind == "aligned":
        return t.contiguous()
    if kind == "late":
        return torch.zeros(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t)
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 1, dtype=t.dtype, device=t.device)
    return wide[..., :-1].copy_(t)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("q,bk,bv", [
    ("aligned", "aligned", "late"), ("aligned", "aligned", "odd"), ("aligned", "late", "aligned"),
    ("aligned", "odd", "aligned"), ("late", "aligned", "aligned"), ("odd", "aligned", "aligned"), ("odd", "late", "odd"),
])
def test_attention_inputs_aligned_apart(dtype, q, bk, bv):
    """q, the block's keys and its values each have an alignment of their own: whichever is off, the
    result is that of contiguous rows, bit for bit."""
    c = _attn_case(21, [300, 64, 0], 5, 2, 4, 128, 64, dtype)
    want = _check_attn(c)
    at = [_placed(t.to(DEV), kind) for t, kind in ((c["q"], q), (c["blk"][0], bk), (c["blk"][1], bv))]
    assert torch.equal(pc.gqa_attention_kv8(at[0], c["layer"], c["tg"], i32(c["lengths"]), at[1], at[2]), want)
    one = [t[:1].expand_as(t) for t in at]  # strides of zero: the same rows for every sequence
    want = pc.gqa_attention_kv8(*(one[0].contiguous(), c["layer"], c["tg"], i32(c["lengths"])),
                                *(t.contiguous() for t in one[1:]))
    assert torch.equal(pc.gqa_attention_kv8(one[0], c["layer"], c["tg"], i32(c["lengths"]), *one[1:]), want)
    assert _lib.device_error() == 0


def test_attention_results_past_32_bits():
    """A sequence's result of more than 2^31 values: one query row, read for every head and block row."""
    block, nh, hd = 64, 262150, 128
    k, ks, v, vs, layer = _pool(6, 2, 1, 64, hd, -9, -4)
    row = torch.randn(1, 1, 1, hd, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    table, n = i32([[1, 0]]), i32([100])
    try:
        out = pc.gqa_attention_kv8(row.expand(1, block, nh, hd), layer, table, n)
    except torch.OutOfMemoryError:
        pytest.skip("no room for the result")
    c = dict(q=row.cpu(), layer=layer, table=[[1, 0]], tg=table, lengths=[100], blk=[None, None],
             k=k * ks[..., None, None], v=v * vs[..., None, None], hd=hd)
    want = out[:, :1, :hd].clone()
    _check_attn(c, out=want)
    assert all(bool((part == want[0]).all()) for part in out.view(block, nh, hd))
    assert _lib.device_error() == 0


# ------------------------------------------------------------------------------- references and weights
def _all_negative(c):
    """Every score negative: q below zero, the keys above."""
    c["q"], c["k"] = -c["q"].abs(), c["k"].abs()
    c["layer"].k_codes.bitwise_and_(0x7F)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths,page,absent,scale", [
    ([640, 300], 64, (0, 1), 0.18), ([640, 300], 64, (0, 1, 2, 3), 1.8), ([640, 130], 128, (0,), 0.18),
    ([5000], 64, tuple(range(3, 70)), 0.18), ([5000, 900], 256, (0, 1, 2), 1.8),
])
def test_attention_where_the_first_pages_are_absent(dtype, lengths, page, absent, scale):
    """A unit, or a CTA's part of one, whose first keys lie on pages that are none: the rows' references
    come from the first keys that there are. Scores lie some 30 or 300 octaves below zero, so that
    weights relative to zero are nothing at all. Norm: bf16's rounding is at most 2^-8 and 2^-8.8 on the
    average, twice the scores' error at 300 octaves less than as much again (fp32: 2 * 2^-17 * 330)."""
    c = _attn_case(len(absent), lengths, 5, 2, 4, 128, page, dtype, with_block=False, e_lo=-6, e_hi=-5)
    _all_negative(c)
    for row in c["table"]:
        for j in absent:
            if j < len(row):
                row[j] = -1 if j % 2 else 10 ** 6
    c["tg"] = i32(c["table"])
    _check_attn(c, scale=scale, norm=2.0 ** -8)
    with pytest.raises(_lib.DsmError, match="outside the pool"):
        _lib.raise_device_error()


def _close(c, out, scale):
    """Every value within the sum of its roundings, per query row, in the order of its own weights. With A the
    mean of |v| under a row's weights, W the largest of these, n the keys, and Vs no less than 448 times any value
    scale that the row's unit meets (its own rows: 4 max |v|):

    * 2^-8 of the result, rounded once;
    * own keys and values as two e4m3 terms like q, exact but for 2^-10, half of e4m3's smallest step, of a row scaled
      to 224 or more: 2^-17 of the row's largest;
    * scores off by ds move the weights by 2 ds, hence 2 ds A. ds is q's second term below e4m3's normals,
      2^-17 max |q| sum |k| scale, and 2^-18 of S = sum |q k| scale for fp32 sums and the exponential's argument;
    * a weight is rounded to f16, 2^-11 of it, whose 11 bits three e5m2 terms hold, down to half of e5m2's
      smallest step, 2^-17 where the largest weight is 2^12 or more: 2^-11 A + n 2^-29 W Vs."""
    hd = c["hd"]
    b, s, nh, _ = c["q"].shape
    n_pages, n_kv, page, _ = c["k"].shape
    group = nh // n_kv
    got = out.double().cpu().view(b, s, nh, hd)
    assert torch.isfinite(got).all()
    sq, sr = 0.0, 0.0
    for i, n in enumerate(c["lengths"]):
        ids = c["table"][i][:-(-n // page)]
        for h in range(n_kv):
            k = torch.cat([c["k"][p, h] for p in ids])[:n]
            v = torch.cat([c["v"][p, h] for p in ids])[:n]
            vs = 448 * float(c["layer"].v_scale[ids, h].max())
            if c["blk"][0] is not None:
                k, v = (torch.cat([t, u[i, h].double()]) for t, u in ((k, c["blk"][0]), (v, c["blk"][1])))
                vs = max(vs, 4 * float(c["blk"][1][i, h].abs().max()))
            q = c["q"][i, :, h * group:(h + 1) * group].double()  # [s, group, hd]
            w = torch.softmax(q @ k.T * scale, -1)
            ref = w @ v
            a, top, m = w @ v.abs(), w.amax(-1, keepdim=True), len(k)
            big = (q.abs() @ k.abs().T).amax(-1, keepdim=True) * abs(scale)
            ds = 2.0 ** -17 * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1).max() * abs(scale) + 2.0 ** -18 * big
            own = 0.0
            if c["blk"][0] is not None:
                ds += 2.0 ** -17 * float(c["blk"][0][i, h].abs().max()) * q.abs().sum(-1, keepdim=True) * abs(scale)
                own = 2.0 ** -17 * float(c["blk"][1][i, h].abs().max())
            tol = 2.0 ** -8 * ref.abs() + (2 * ds + 2.0 ** -11) * a + own + m * 2.0 ** -29 * top * vs
            err = got[i, :, h * group:(h + 1) * group] - ref
            assert bool((err.abs() <= tol).all()), float((err.abs() / tol).max())
            sq, sr = sq + float(err.square().sum()), sr + float(ref.square().sum())
    return (sq / sr) ** 0.5


def _sinks(seed, dtype, n, s, n_kv, group, hd, page, q0, with_block=False):
    """Every 64th key draws q0 * 7 nats more than the others, whose scores are normal, and has a value of zero."""
    c = _attn_case(seed, [n], s, n_kv, group, hd, page, dtype, with_block=with_block, e_lo=-6, e_hi=-5,
                   q_mag=hd ** -0.5 / 1.5)
    k, v = c["k"] * 2.0 ** 6, c["v"] * 2.0 ** 6
    k[..., 0] = 0
    k[:, :, ::64], v[:, :, ::64] = 0, 0
    k[:, :, ::64, 0] = 448
    c["k"], c["v"] = torch.nan_to_num(k) * 2.0 ** -6, torch.nan_to_num(v) * 2.0 ** -6
    c["layer"] = pc.KV8Layer(_codes(po.store_keys(k)), _codes(po.store_values(v)),
                             torch.full_like(c["layer"].k_scale, 2.0 ** -6), torch.full_like(c["layer"].v_scale, 2.0 ** -6))
    c["q"][..., 0] = q0
    return c


SINKS = [(1.5, 700, 1, 1, 1, 64, 64), (1.5, 2048, 5, 2, 4, 128, 64), (2.0, 2048, 1, 2, 4, 128, 128),
         (2.0, 1500, 7, 1, 8, 64, 64), (2.0, 1000, 2, 1, 4, 256, 256)]


@pytest.mark.parametrize("q0,n,s,n_kv,group,hd,page", SINKS)
def test_attention_under_sinks(q0, n, s, n_kv, group, hd, page):
    """Keys 2^15 or 2^20 times heavier than the others that give nothing: the result is the others' alone. Norm: as far
    off as bf16's own rounding at most (2^-8; 2^-8.8 on the average), the weights' 2^-11 and 2^-29 of the
    largest, 2^-9 of one that is 2^-20 of it, taking the rest."""
    c = _sinks(4, BF, n, s, n_kv, group, hd, page, q0)
    out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]), scale=1.0)
    assert _close(c, out, 1.0) <= 2.0 ** -8
    assert _lib.device_error() == 0


@pytest.mark.parametrize("lower,s,hd", [(6, 1, 128), (12, 5, 128), (12, 2, 64), (14, 7, 256)])
def test_attention_to_pages_of_a_small_scale(lower, s, hd):
    """Every second page has values 2^lower times smaller, and all of the weight: 2^-40 is left for its neighbour. What
    the result owes to the small page is as exact as its distance leaves it: 2^-29 of the largest weight, in
    units of the large scale."""
    c = _attn_case(lower, [1024], s, 2, 4, hd, 64, BF, with_block=False, e_lo=-6, e_hi=-5, q_mag=hd ** -0.5 / 1.5,
                   poison=False)
    k = c["k"] * 2.0 ** 6
    for j, p in enumerate(c["table"][0][:16]):
        k[p, :, :, 0] = 448 if j % 2 else -448
        f = 2.0 ** -lower if j % 2 else 1.0
        c["v"][p] *= f
        c["layer"].v_scale[p] *= f
    c["k"] = k * 2.0 ** -6
    c["layer"].k_codes.copy_(_codes(po.store_keys(k)))
    c["q"][..., 0] = 2.0
    out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]), scale=1.0)
    assert _close(c, out, 1.0) <= 2.0 ** -8
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype,lengths,s,n_kv,group,hd,page", [
    (BF, [150, 0, 1], 1, 8, 4, 128, 64), (BF, [700, 3, 1999], 7, 2, 4, 128, 64), (BF, [1000, 77], 7, 2, 8, 64, 64),
    (BF, [513, 300], 5, 1, 3, 256, 128),
])
def test_attention_row_by_row(dtype, lengths, s, n_kv, group, hd, page):
    """The bound of each row by its own weights, own rows included. Norm: bf16's rounding alone is 2^-8.8 on the average
    (its half step's third root); 1.1 times it leaves half as much for all else."""
    c = _attn_case(sum(lengths) + 1, [n or 1 for n in lengths], s, n_kv, group, hd, page, dtype)
    out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]), *(t.to(DEV) for t in c["blk"]))
    norm = _close(c, out, hd ** -0.5)
    assert norm <= 1.1 * 2.0 ** -8 / 3 ** 0.5
    assert _lib.device_error() == 0


def _close_f32(c, out, scale):
    """The same for fp32 calls, whose factors are two f16 terms each; returns the norm of the error over what it may be.
    2^-24 of the result; scores off by ds <= (2^-21 + (hd + 8) 2^-24) S; a weight's second term is held times 2^11, so
    that both leave 2^-22 of a weight and 2^-36 where the largest is 2^6 or more, own values 2^-22, sums of n keys
    (n / 32 + 64) 2^-24: (2 ds + 2^-21 + (n / 32 + 64) 2^-24) A + n 2^-42 W Vs. Norm: 2^-20 for the terms, and
    2^-23 S, for the tensor cores cut off 2^-23 of a sum at each of the four steps that are added in them, a
    quarter of a row's products each, hence S 2^-23 for all of a row's at most."""
    hd = c["hd"]
    b, s, nh, _ = c["q"].shape
    n_pages, n_kv, page, _ = c["k"].shape
    group = nh // n_kv
    got = out.double().cpu().view(b, s, nh, hd)
    sq, sr, most = 0.0, 0.0, 0.0
    for i, n in enumerate(c["lengths"]):
        ids = c["table"][i][:-(-n // page)]
        for h in range(n_kv):
            k = torch.cat([c["k"][p, h] for p in ids])[:n]
            v = torch.cat([c["v"][p, h] for p in ids])[:n]
            vs = 448 * float(c["layer"].v_scale[ids, h].max())
            if c["blk"][0] is not None:
                k, v = (torch.cat([t, u[i, h].double()]) for t, u in ((k, c["blk"][0]), (v, c["blk"][1])))
                vs = max(vs, 4 * float(c["blk"][1][i, h].abs().max()))
            q = c["q"][i, :, h * group:(h + 1) * group].double()
            w = torch.softmax(q @ k.T * scale, -1)
            ref, a, top, m = w @ v, w @ v.abs(), w.amax(-1, keepdim=True), len(k)
            big = (q.abs() @ k.abs().T).amax(-1, keepdim=True) * abs(scale)
            ds = (2.0 ** -21 + (hd + 8) * 2.0 ** -24) * big
            tol = 2.0 ** -24 * ref.abs() + (2 * ds + 2.0 ** -21 + (m / 32 + 64) * 2.0 ** -24) * a + m * 2.0 ** -42 * top * vs
            err = got[i, :, h * group:(h + 1) * group] - ref
            assert bool((err.abs() <= tol).all()), float((err.abs() / tol).max())
            sq, sr, most = sq + float(err.square().sum()), sr + float(ref.square().sum()), max(most, float(big.max()))
    return (sq / sr) ** 0.5 / (2.0 ** -20 + 2.0 ** -23 * most)


@pytest.mark.parametrize("with_block", [False, True])
@pytest.mark.parametrize("q0,n,s,n_kv,group,hd,page", SINKS)
def test_fp32_attention_under_sinks(q0, n, s, n_kv, group, hd, page, with_block):
    c = _sinks(4, F32, n, s, n_kv, group, hd, page, q0, with_block)
    if with_block:  # own rows: the first draws as the sinks do and gives nothing
        c["blk"][0][..., 0] = 0
        c["blk"][0][:, :, 0] = 0
        c["blk"][0][:, :, 0, 0] = 7
        c["blk"][1][:, :, 0] = 0
    out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]),
                               *(None if t is None else t.to(DEV) for t in c["blk"]), scale=1.0)
    assert _close_f32(c, out, 1.0) <= 1
    assert _lib.device_error() == 0


@pytest.mark.parametrize("lengths,s,n_kv,group,hd,page", [
    ([150, 700], 5, 2, 4, 128, 64), ([500, 40], 5, 1, 4, 256, 64), ([1, 333], 1, 2, 8, 64, 128),
])
def test_fp32_attention_row_by_row(lengths, s, n_kv, group, hd, page):
    c = _attn_case(sum(lengths) + 1, lengths, s, n_kv, group, hd, page, F32)
    out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]), *(t.to(DEV) for t in c["blk"]))
    assert _close_f32(c, out, hd ** -0.5) <= 1
    assert _lib.device_error() == 0


@pytest.mark.parametrize("kernel", ["default", "cuda cores"])
@pytest.mark.parametrize("dtype,s", [(BF, 5), (BF, 65), (F32, 5), (F32, 65)])
@pytest.mark.parametrize("what", ["q", "keys", "values"])
@pytest.mark.parametrize("x", [float("inf"), float("-inf"), float("nan")])
def test_attention_counts_what_is_not_finite_as_nan(kernel, dtype, s, what, x):
    """As the append stores it: an infinity or NaN in q, the block's keys or its values gives NaN wherever it counts
    and nowhere else, whichever kernel takes the call."""
    c = _attn_case(13, [100, 70], s, 2, 2, 64, 64, dtype)
    t = {"q": c["q"], "keys": c["blk"][0], "values": c["blk"][1]}[what]
    t[(1, 3, 2, 9) if what == "q" else (1, 1, 3, 9)] = x  # sequence 1, row 3; query head 2 is of KV head 1
    want = torch.zeros(2, s, 4, 64, dtype=torch.bool)
    if what == "q":
        want[1, 3, 2] = True
    elif what == "keys":
        want[1, :, 2:] = True
    else:
        want[1, :, 2:, 9] = True
    L = _lib.lib()
    _lib.check(L.dsm_set_attn_kernel(1 if kernel == "cuda cores" else _lib.ATTN_KERNEL_DEFAULT))
    try:
        out = pc.gqa_attention_kv8(c["q"].to(DEV), c["layer"], c["tg"], i32(c["lengths"]),
                                   *(b.to(DEV) for b in c["blk"])).view(2, s, 4, 64).cpu()
    finally:
        _lib.check(L.dsm_set_attn_kernel(_lib.ATTN_KERNEL_DEFAULT))
    assert torch.equal(out.isnan(), want) and bool(torch.isfinite(out[~want]).all())


# ------------------------------------------------------------------------------- ids outside the pool
@pytest.mark.parametrize("b,longest,bad", [(5, 300, -1), (61, 700, 10 ** 6), (900, 300, -64), (8192, 500, -1)])
def test_trim_refuses_pages_outside_the_pool(b, longest, bad):
    """A table entry that is no page: nothing moves, and the error word says so. Entries that stay are not looked at."""
    page = 64
    lengths, new, table, free, n_free, tg = _tables_case(b, b, page, longest, 1, 3 * b)
    at = max(range(b), key=lambda i: lengths[i])
    last = -(-lengths[at] // page) - 1
    keep = [n // 2 for n in lengths]
    keep[at] = 0
    tg[at, last] = bad
    table[at][last] = bad
    assert po.paged_trim(lengths, keep, table, free, n_free, page) == (lengths, free, n_free, True)
    L, F, N = i32(lengths), i32(free), i32([n_free])
    pc.paged_trim(L, i32(keep), tg, F, N, page)
    assert L.tolist() == lengths and F.tolist() == free and N.tolist() == [n_free] and tg.tolist() == table
    with pytest.raises(_lib.DsmError, match="outside the pool"):
        _lib.raise_device_error()
    keep[at] = lengths[at]  # the entry stays where it is
    want = po.paged_trim(lengths, keep, table, free, n_free, page)
    pc.paged_trim(L, i32(keep), tg, F, N, page)
    assert not want[3] and L.tolist() == want[0] and F.tolist() == want[1] and N.tolist() == [want[2]]
    assert _lib.device_error() == 0


@pytest.mark.parametrize("b,new_most,where,bad", [
    (1, 5, 0, -1), (30, 150, 0, -2), (30, 150, 7, 10 ** 6), (30, 150, 40, -64), (90, 384, 100, -1), (700, 3, 60, 10 ** 9),
])
def test_extend_stops_at_a_page_outside_the_pool(b, new_most, where, bad):
    """A free page that is none ends the stack there: who would need it, or one below, is not served."""
    page = 64
    lengths, new, table, free, n_free, tg = _tables_case(b + where, b, page, 300, new_most, 60 + b * (new_most // page + 2))
    new = [max(1, n) for n in new]
    new[0] += page
    need = sum(-(-(n + a) // page) - -(-n // page) for n, a in zip(lengths, new))
    where = min(where, need - 1)
    free[n_free - 1 - where] = bad
    max_rows = sum(new) + 3
    want = po.paged_extend(lengths, new, table, free, n_free, page, max_rows)
    assert want[6] and want[2] >= n_free - where
    L, F, N, rows = _run_extend(lengths, new, tg, free, n_free, page, max_rows)
    assert L.tolist() == want[0] and tg.tolist() == want[1] and N.tolist() == [want[2]] and F.tolist() == free
    assert rows.cu_rows.tolist() == want[3] and rows.slot_map.tolist() == want[4]
    assert rows.positions.tolist() == want[5]
    with pytest.raises(_lib.DsmError, match="outside the pool"):
        _lib.raise_device_error()


# ------------------------------------------------------------------------------- host threads
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_host_thread_whose_first_cuda_call_is_the_attention(dtype):
    """The C entry point on a thread that has no context yet."""
    import ctypes
    import threading

    c = _attn_case(17, [100, 65], 1, 2, 2, 128, 64, dtype, with_block=False)
    L, q, n = _lib.lib(), c["q"].to(DEV), i32(c["lengths"])
    size = L.dsm_gqa_attn_kv8_workspace_bytes(2, 1, 4, 2, 128)
    ws, out = torch.empty(size, dtype=torch.uint8, device=DEV), torch.empty(2, 1, 512, dtype=dtype, device=DEV)
    layer = [t.data_ptr() for t in c["layer"]]
    desc = _lib.KV8AttnDesc(q_batch_stride=512, q_row_stride=512, q_head_stride=128, table_stride=c["tg"].stride(0),
                            k_codes=layer[0], v_codes=layer[1], k_scale=layer[2], v_scale=layer[3],
                            dtype=_lib.DT_BF16 if dtype == BF else _lib.DT_F32, batch=2, block=1, n_heads=4, n_kv=2,
                            head_dim=128, page_size=64, n_pages=c["layer"].k_codes.shape[0], max_pages=c["tg"].shape[1],
                            scale=128 ** -0.5)
    args = [t.data_ptr() for t in (q, c["tg"], n)] + [None, None, out.data_ptr(), ws.data_ptr(), size,
                                                      torch.cuda.current_stream().cuda_stream]
    torch.cuda.synchronize()
    rc = []

    def run():
        rc.append((L.dsm_gqa_attn_kv8(ctypes.addressof(desc), *args), L.dsm_last_error_message().decode()))

    t = threading.Thread(target=run)
    t.start()
    t.join()
    assert rc[0][0] == 0, rc[0][1]
    torch.cuda.synchronize()
    _check_attn(c, out=out)


@pytest.mark.parametrize("what", ["extend", "trim", "bf16 attention", "fp32 attention"])
def test_calls_of_unlike_sizes_from_two_threads(what):
    """Two host threads, each with a stream of its own, call the C entry points with batches that need unlike amounts of
    shared memory: what one sets must not take the other's launch."""
    import ctypes
    import threading

    L, kept = _lib.lib(), []

    def ptr(t):
        kept.append(t)
        return t.data_ptr()

    def setup(b, stream):
        zeros, table, pool, n = (ptr(torch.zeros(k, dtype=torch.int32, device=DEV)) for k in (b, 2 * b, 2, 1))
        lengths = ptr(torch.zeros(b, dtype=torch.int32, device=DEV))
        if what == "extend":
            cu, slots, pos = (ptr(torch.zeros(k, dtype=t, device=DEV)) for k, t in
                              ((b + 1, torch.int32), (1, torch.int64), (1, torch.int32)))
            return lambda: L.dsm_paged_extend(lengths, zeros, b, 64, table, 2, 2, pool, n, 2, cu, slots, pos, 1, stream)
        if what == "trim":
            return lambda: L.dsm_paged_trim(lengths, zeros, b, 64, table, 2, 2, pool, n, 2, stream)
        layer = [ptr(t) for t in _pool(0, 2, 1, 64, 128)[4]]
        dt, dtype = (_lib.DT_BF16, BF) if what[0] == "b" else (_lib.DT_F32, F32)
        q, out = (ptr(torch.zeros(b * 128, dtype=dtype, device=DEV)) for _ in range(2))
        size = L.dsm_gqa_attn_kv8_workspace_bytes(b, 1, 1, 1, 128)
        ws = ptr(torch.zeros(size, dtype=torch.uint8, device=DEV))
        desc = _lib.KV8AttnDesc(q_batch_stride=128, q_row_stride=128, q_head_stride=128, table_stride=2, k_codes=layer[0],
                                v_codes=layer[1], k_scale=layer[2], v_scale=layer[3], dtype=dt, batch=b, block=1,
                                n_heads=1, n_kv=1, head_dim=128, page_size=64, n_pages=2, max_pages=2, scale=1.0)
        kept.append(desc)
        d = ctypes.addressof(desc)
        return lambda: L.dsm_gqa_attn_kv8(d, q, table, lengths, None, None, out, ws, size, stream)

    streams = [torch.cuda.Stream() for _ in range(2)]
    sizes = (8192, 6500) if what in ("extend", "trim") else (8192, 2)
    calls = [setup(b, s.cuda_stream) for b, s in zip(sizes, streams)]
    torch.cuda.synchronize()
    errors, start = [], threading.Barrier(2)

    def run(call):
        start.wait()
        for _ in range(10000):
            if call():
                errors.append(L.dsm_last_error_message().decode())
                return

    threads = [threading.Thread(target=run, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]
    assert _lib.device_error() == 0
