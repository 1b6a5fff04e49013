"""CPU oracle for the paged 8-bit KV cache (test infrastructure only).

Plain restatements, one sequence, page and row at a time: the page tables in Python integers, the
quantising append and the attention in 64 bits. The cache is held by token here, codes as the
values they stand for (``[n_pages, n_kv, page_size, head_dim]`` float64, before the scale);
``store_*`` / ``load_*`` convert to and from the library's stored layout.
"""

from __future__ import annotations

from typing import List, Tuple

import torch

__all__ = ["paged_extend", "paged_trim", "kv8_append", "kv8_scale_exp", "kv8_attention", "e4m3_values", "round_e4m3",
           "load_keys", "load_values", "store_keys", "store_values"]

INT32_MAX = 2 ** 31 - 1


# ------------------------------------------------------------------------------- page tables
def paged_extend(lengths: List[int], new: List[int], table: List[List[int]], free: List[int], n_free: int, page: int,
                 max_rows: int):
    """Returns ``(lengths, table, n_free, cu_rows, slot_map, positions, failed)``; inputs unchanged."""
    lengths, table = list(lengths), [list(r) for r in table]
    n_free = min(max(n_free, 0), len(free))
    slots, pos = [-1] * max_rows, [0] * max_rows
    cu, wanted, failed, top = [0], 0, False, n_free
    usable = 0  # the stack ends at a page outside the pool
    while usable < n_free and 0 <= free[n_free - 1 - usable] < len(free):
        usable += 1
    for i, (n, add) in enumerate(zip(list(lengths), new)):
        rows = max(add, 0)
        first = cu[-1]
        cu.append(first + rows)
        if n < 0 or add < 0 or n + add > min(len(table[i]) * page, INT32_MAX):
            failed |= add != 0
            continue
        have, want = -(-n // page), -(-(n + add) // page)
        need = want - have
        wanted += need
        if first + rows > max_rows or (need and wanted > usable):
            failed |= rows > 0
            continue
        for j in range(have, want):
            top -= 1
            table[i][j] = free[top]
        for r in range(rows):
            p = n + r
            slots[first + r] = table[i][p // page] * page + p % page
            pos[first + r] = p
        lengths[i] = n + add
    return lengths, table, top, [min(c, INT32_MAX) for c in cu], slots, pos, failed


def paged_trim(lengths: List[int], keep: List[int], table: List[List[int]], free: List[int], n_free: int, page: int):
    """Returns ``(lengths, free, n_free, failed)``; inputs unchanged."""
    out, free = list(lengths), list(free)
    n_free = min(max(n_free, 0), len(free))
    back = []
    for i, (n, k) in enumerate(zip(lengths, keep)):
        n = min(max(n, 0), len(table[i]) * page)
        k = min(max(k, 0), n)
        back += [table[i][j] for j in range(-(-k // page), -(-n // page))]
        out[i] = k
    if n_free + len(back) > len(free) or any(not 0 <= p < len(free) for p in back):
        return list(lengths), free, n_free, True
    for j, p in enumerate(reversed(back)):
        free[n_free + j] = p
    return out, free, n_free + len(back), False


# ------------------------------------------------------------------------------- e4m3
def e4m3_values() -> torch.Tensor:
    """The value of each of the 256 codes, from its fields (sign, 4 exponent, 3 mantissa bits)."""
    t = []
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = float("nan") if (c & 127) == 127 else ((8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9)
        t.append(-x if c & 128 else x)
    return torch.tensor(t, dtype=torch.float64)


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """fp64 values to the nearest e4m3 value, ties to even; |x| <= 448 or NaN."""
    _, e = torch.frexp(x)
    step = torch.exp2((e.to(torch.float64) - 4).clamp_min(-9))
    return torch.round(x / step) * step


def kv8_scale_exp(amax: float) -> int:
    """The least e in [-120, 120] with amax <= 448 * 2^e."""
    e = -120
    while e < 120 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


# ------------------------------------------------------------------------------- layout
def _swizzle(x: torch.Tensor) -> torch.Tensor:
    page, hd = x.shape[-2:]
    if hd < 128:
        return x.clone()
    out = torch.empty_like(x)
    for t in range(page):
        for c in range(hd // 16):
            at = c ^ (t % 8)
            out[..., t, at * 16:at * 16 + 16] = x[..., t, c * 16:c * 16 + 16]
    return out


def store_keys(x: torch.Tensor) -> torch.Tensor:
    return _swizzle(x)


def load_keys(x: torch.Tensor) -> torch.Tensor:
    return _swizzle(x)


def store_values(x: torch.Tensor) -> torch.Tensor:
    """[..., page, hd] by token -> [..., page / 64, hd, 64]."""
    page, hd = x.shape[-2:]
    return x.reshape(*x.shape[:-2], page // 64, 64, hd).transpose(-1, -2).contiguous()


def load_values(x: torch.Tensor) -> torch.Tensor:
    groups, hd = x.shape[-3], x.shape[-2]
    return x.transpose(-1, -2).reshape(*x.shape[:-3], groups * 64, hd)


# ------------------------------------------------------------------------------- append
def kv8_append(codes: torch.Tensor, scale: torch.Tensor, rows: torch.Tensor, slots: List[int]) -> Tuple:
    """One of K and V: ``codes`` fp64 values by token, ``scale`` fp64 ``[n_pages, n_kv]``, ``rows``
    fp64 ``[n, n_kv, hd]``. Returns the new ``(codes, scale)``."""
    codes, scale = codes.clone(), scale.clone()
    n_pages, n_kv, page, _ = codes.shape
    at = [s // page if 0 <= s < n_pages * page else -1 for s in slots]
    r = 0
    while r < len(at):
        z = r + 1
        while z < len(at) and at[z] == at[r]:
            z += 1
        if at[r] >= 0:
            off = [s % page for s in slots[r:z]]
            for h in range(n_kv):
                x = rows[r:z, h]
                fin = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
                e = kv8_scale_exp(float(fin.max()))
                if 0 not in off:
                    old = int(round(torch.log2(scale[at[r], h]).item()))
                    if e > old:
                        codes[at[r], h] = round_e4m3(codes[at[r], h] * 2.0 ** (old - e))
                    e = max(e, old)
                scale[at[r], h] = 2.0 ** e
                x = torch.where(torch.isfinite(x), x, torch.full_like(x, float("nan")))
                codes[at[r], h, off] = round_e4m3(x / 2.0 ** e)
        r = z
    return codes, scale


# ------------------------------------------------------------------------------- attention
def kv8_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: List[List[int]], lengths: List[int],
                  blk_k, blk_v, scale: float):
    """``q [b, s, nh, hd]``; ``k``, ``v`` fp64 dequantised ``[n_pages, n_kv, page, hd]``; everything in
    64 bits. Returns ``(out [b, s, nh * hd], score [b], vmax [b])``: per sequence the largest
    ``sum_d |q_d k_d| * scale`` of a row and key, and the largest ``|v|``, for error bounds."""
    b, s, nh, hd = q.shape
    n_pages, n_kv, page, _ = k.shape
    group = nh // n_kv
    out = torch.zeros(b, s, nh, hd, dtype=torch.float64)
    score, vmax = torch.zeros(b, dtype=torch.float64), torch.zeros(b, dtype=torch.float64)
    for i in range(b):
        n = min(max(lengths[i], 0), len(table[i]) * page)
        for h in range(n_kv):
            ks, vs = [], []
            for j in range(-(-n // page)):
                p, m = table[i][j], min(page, n - j * page)
                if 0 <= p < n_pages:
                    ks.append(k[p, h, :m])
                    vs.append(v[p, h, :m])
            if blk_k is not None:
                ks.append(blk_k[i, h].double())
                vs.append(blk_v[i, h].double())
            if not ks:
                continue
            kk, vv = torch.cat(ks), torch.cat(vs)
            qq = q[i, :, h * group:(h + 1) * group].double().reshape(s * group, hd)
            x = qq @ kk.T * scale
            w = torch.softmax(x, -1)
            out[i, :, h * group:(h + 1) * group] = (w @ vv).reshape(s, group, hd)
            score[i] = max(score[i], (qq.abs() @ kk.abs().T).max() * scale)
            vmax[i] = max(vmax[i], vv.abs().max())
    return out.reshape(b, s, nh * hd), score, vmax
