"""64-bit CPU statement of the decode-step operators (test infrastructure only, never the product path).

Semantics: include/sh_ops_cuda.h, "decoding: paged 8-bit K / V cache and 4-bit weights". Written as plain loops over
requests, pages and groups.
"""
from __future__ import annotations

import numpy as np

QMAX = {"int8": 127.0, "fp8": 448.0}


# ---- e4m3 ------------------------------------------------------------------------------------------------------------
def e4m3_values() -> np.ndarray:
    """Value of each of the 256 codes (0x7F, 0xFF: NaN)."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >= 128, -v, v)


_E4M3 = e4m3_values()


def e4m3_encode(y) -> np.ndarray:
    """Nearest code, ties to the even one, |y| > 448 saturates."""
    y = np.clip(np.asarray(y, np.float64), -448.0, 448.0)
    a = np.abs(y)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -60))), -6.0) - 3.0)
    code = np.searchsorted(_E4M3[:127], np.rint(a / step) * step)
    return (code + np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def decode(codes, fmt: str) -> np.ndarray:
    codes = np.asarray(codes, np.uint8)
    return codes.view(np.int8).astype(np.float64) if fmt == "int8" else _E4M3[codes]


def encode(y, fmt: str) -> np.ndarray:
    if fmt == "int8":
        return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    return e4m3_encode(y)


def up8(x) -> np.ndarray:
    """The next value with 8 significant bits, x >= 0."""
    m, e = np.frexp(np.asarray(x, np.float64))
    return np.ldexp(np.ceil(m * 256.0), e - 8)


# ---- tables ------------------------------------------------------------------------------------------------------------
def kv_tables(lens, add, page: int, table, ring, pool, t_cap: int):
    """-> table, ring, pool_out[:3], lens_out, q_start, slots, pos (new arrays)."""
    table, ring = np.array(table, np.int64), np.array(ring, np.int64)
    R, ld = table.shape
    pages = ring.size
    head, count = int(pool[0]), int(pool[1])
    lens_out = np.array(lens, np.int64)
    slots, pos = np.full(t_cap, -1, np.int64), np.zeros(t_cap, np.int64)
    q_start = np.zeros(R + 1, np.int64)
    asked = taken = put_off = 0
    back = []
    for r in range(R):
        n, ln = int(add[r]), int(lens[r])
        q_start[r + 1] = q_start[r] + max(n, 0)
        have = -(-ln // page)
        if n < 0:
            back += [int(p) for p in table[r, :have]]
            lens_out[r] = 0
            continue
        need = -(-(ln + n) // page) - have
        served = have + need <= ld
        if served:
            asked += need
            served = need == 0 or asked <= count
        if served:
            for b in range(have, have + need):
                table[r, b] = ring[(head + taken) % pages]
                taken += 1
            lens_out[r] = ln + n
        elif n:
            put_off += 1
        for i in range(n):
            at = int(q_start[r]) + i
            if at < t_cap:
                pos[at] = ln + i
                if served:
                    slots[at] = table[r, (ln + i) // page] * page + (ln + i) % page
    for i, p in enumerate(back):
        ring[(head + count + i) % pages] = p
    return table, ring, np.array([(head + taken) % pages, count - taken + len(back), put_off]), lens_out, q_start, slots, pos


# ---- append ------------------------------------------------------------------------------------------------------------
def kv8_append(codes, scale, x, slots, page: int, fmt: str):
    """One of K and V: codes [pages, heads, page, dh] uint8, scale [pages, heads], x [T, heads * dh], slots [T]; tokens of one
    page follow one another with rising slots. -> new codes, scale."""
    codes, scale = np.array(codes), np.array(scale, np.float64)
    _, heads, _, dh = codes.shape
    x = np.nan_to_num(np.asarray(x, np.float64), nan=0.0, posinf=65504.0, neginf=-65504.0).reshape(-1, heads, dh)
    slots = np.asarray(slots, np.int64)
    i = 0
    while i < slots.size:
        if slots[i] < 0:
            i += 1
            continue
        j = i
        while j < slots.size and slots[j] >= 0 and slots[j] // page == slots[i] // page:
            j += 1
        p, off = int(slots[i] // page), slots[i:j] % page
        for h in range(heads):
            old = scale[p, h] if off[0] else 0.0
            new = max(old, float(up8(np.abs(x[i:j, h]).max() / QMAX[fmt])))
            if off[0] and new > old:
                codes[p, h, :off[0]] = encode(decode(codes[p, h, :off[0]], fmt) * old / new, fmt)
            codes[p, h, off] = encode(x[i:j, h] / new if new else np.zeros_like(x[i:j, h]), fmt)
            scale[p, h] = new
        i = j
    return codes, scale


# ---- attention -----------------------------------------------------------------------------------------------------------
def attention_kv8(q, codes_k, codes_v, ks, vs, table, lens, q_start, H: int, scale: float, fmt: str):
    """-> o [T, H * dh] (rows of no request: NaN) and, for tolerances, per output the weighted mean of |v|, and per row and
    head the largest scale sum |q k| among its keys and the number of keys."""
    q = np.asarray(q, np.float64)
    _, heads, page, dh = codes_k.shape
    G = H // heads
    o = np.full((q.shape[0], H * dh), np.nan)
    mean_abs = np.zeros_like(o)
    big = np.zeros((q.shape[0], H))
    keys = np.zeros(q.shape[0], np.int64)
    for r in range(len(lens)):
        a, e, n = int(q_start[r]), int(q_start[r + 1]), int(lens[r])
        ids = np.asarray(table[r, :-(-n // page)], np.int64)
        for h in range(heads):
            k = (decode(codes_k[ids, h], fmt) * np.asarray(ks, np.float64)[ids, h][:, None, None]).reshape(-1, dh)[:n]
            v = (decode(codes_v[ids, h], fmt) * np.asarray(vs, np.float64)[ids, h][:, None, None]).reshape(-1, dh)[:n]
            for i in range(a, e):
                m = min(max(n - (e - a) + (i - a) + 1, 0), n)
                keys[i] = m
                for g in range(h * G, (h + 1) * G):
                    col = slice(g * dh, (g + 1) * dh)
                    if m == 0:
                        o[i, col] = 0.0
                        continue
                    x = scale * (k[:m] @ q[i, col])
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    o[i, col] = p @ v[:m]
                    mean_abs[i, col] = p @ np.abs(v[:m])
                    big[i, g] = abs(scale) * (np.abs(k[:m]) @ np.abs(q[i, col])).max()
    return o, mean_abs, big, keys


# ---- 4-bit weights -----------------------------------------------------------------------------------------------------
def w4_weights(codes, scales, zeros, group: int, K: int) -> np.ndarray:
    """W [K, N] in 64 bits."""
    codes = np.asarray(codes, np.uint8)[:, :K // 2]
    q = np.stack([codes & 15, codes >> 4], 2).reshape(codes.shape[0], K).astype(np.float64)
    z = np.full(np.shape(scales), 8.0) if zeros is None else np.asarray(zeros, np.float64)
    return ((q - np.repeat(z, group, 1)) * np.repeat(np.asarray(scales, np.float64), group, 1)).T
