"""Float64 restatement of the paged serving operators, page by page on the host.

Pages are given as numbers: ``pages[i] = (K, V)`` float64 [T, heads_kv, dim] each, the values that
the page's stored bytes stand for (:func:`page_values`)."""
from __future__ import annotations

import numpy as np

from . import (PAGE_BF16, PAGE_FP8, PAGE_INT4, PAGE_INT8, fp8_decode, page_decode)


def bf16_to_f64(bits: np.ndarray) -> np.ndarray:
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def page_values(fmt: int, data: np.ndarray, T: int, heads: int, dim: int, outlier_cap: int = 0):
    """(K, V) of a page: ``data`` is its bf16 bit patterns (PAGE_BF16) or its slot bytes."""
    row = heads * dim
    E = 2 * T * row
    if fmt == PAGE_BF16:
        x = bf16_to_f64(np.asarray(data, np.uint16).reshape(-1))
    else:
        s = np.ascontiguousarray(data, dtype=np.uint8).reshape(-1)
        if fmt == PAGE_INT8:
            c0 = (4 * T + 15) // 16 * 16
            x = s[c0:c0 + E].view(np.int8).astype(np.float64).reshape(2 * T, row)
            x = x * s[:4 * T].copy().view(np.float16).astype(np.float64)[:, None] / 127.0
        elif fmt == PAGE_INT4:
            n = s[E // 32:E // 32 + E // 2]
            x = np.stack((n >> 4, n & 15), -1).astype(np.float64).reshape(E // 64, 64) - 8.0
            x = x * bf16_to_f64(s[:E // 32].copy().view(np.uint16))[:, None] / 7.0
        elif fmt == PAGE_FP8:
            x = bf16_to_f64(fp8_decode(s[:E]))  # every e4m3 number is a bf16 number
        else:
            x = bf16_to_f64(page_decode(fmt, s, T, row, outlier_cap=outlier_cap))
    x = x.reshape(2, T, heads, dim)
    return x[0], x[1]


def decode_attention(q, lists, lengths, T, scale, page_mass=None, decay=1.0):
    """q float64 [n, heads_q, dim]; ``lists[b][hk]`` = [(position, (K, V)), ...] of key head hk.

    Returns arrays: out, lse, mass, and for tolerances ``reach`` = sum_t P |v| per result element,
    ``size`` = max_t scale * sum |q||k|, ``wide`` = max_t scale * max|q| sum |k| and ``largest`` =
    max |v| per query head (0 without tokens)."""
    n, hq, d = q.shape
    hkv = len(lists[0])
    out, reach = np.zeros_like(q), np.zeros_like(q)
    lse, size, wide, largest = (np.full((n, hq), -np.inf), *(np.zeros((n, hq)) for _ in range(3)))
    mass = None if page_mass is None else page_mass.astype(np.float64).copy()
    for b in range(n):
        if mass is not None:
            used = -(-int(lengths[b]) // T)
            mass[b, :used] *= decay
        for h in range(hq):
            hk = h // (hq // hkv)
            entries = [(pos, K[:t, hk], V[:t, hk]) for pos, (K, V) in lists[b][hk]
                       if (t := min(T, int(lengths[b]) - pos * T)) > 0]
            if not entries:
                continue
            K, V = np.concatenate([e[1] for e in entries]), np.concatenate([e[2] for e in entries])
            s = scale * (K @ q[b, h])
            top = s.max()
            p = np.exp(s - (top if np.isfinite(top) else 0.0))
            with np.errstate(divide="ignore", invalid="ignore"):
                lse[b, h] = np.log(p.sum()) + (top if np.isfinite(top) else 0.0)
            p = p / p.sum() if p.sum() != 0 else p
            out[b, h], reach[b, h] = p @ V, p @ np.abs(V)
            size[b, h] = (abs(scale) * (np.abs(K) @ np.abs(q[b, h]))).max()
            wide[b, h] = abs(scale) * np.abs(K).sum(-1).max() * np.abs(q[b, h]).max()
            largest[b, h] = np.abs(V).max()
            if mass is not None:
                at = 0
                for pos, k, _ in entries:
                    mass[b, pos] += p[at:at + len(k)].sum()
                    at += len(k)
    return {"out": out, "lse": lse, "mass": mass, "reach": reach, "size": size, "wide": wide, "largest": largest}


def exponent(amax: float) -> int:
    """Smallest e >= -100 with amax <= 127 * 2^e."""
    e = -100
    while amax > 127.0 * 2.0 ** e:
        e += 1
    return e


def page_bounds(K: np.ndarray, valid: int):
    """K float64 [T, heads, dim] -> int8 codes [heads, 2, dim], exponents [heads]."""
    T, heads, dim = K.shape
    codes, exps = np.zeros((heads, 2, dim), np.int64), np.full(heads, -100)
    big = 3.3895313892515355e38
    for h in range(heads):
        x = np.clip(K[:valid, h], -big, big)
        lo, hi = np.zeros(dim), np.zeros(dim)
        for c in range(dim):
            col = x[:, c][~np.isnan(x[:, c])]
            if col.size:
                lo[c], hi[c] = col.min(), col.max()
        exps[h] = exponent(max(np.abs(lo).max(), np.abs(hi).max()))
        unit = 2.0 ** int(exps[h])
        codes[h, 0], codes[h, 1] = np.floor(lo / unit), np.ceil(hi / unit)
    return codes.astype(np.int8), exps.astype(np.int8)


def page_scores(q: np.ndarray, codes: np.ndarray, exps: np.ndarray) -> np.ndarray:
    """q float64 [group, dim] of one key head, its codes [pages, 2, dim] and exponents [pages] -> scores."""
    best = np.full(codes.shape[0], -np.inf)
    for x in q:
        x = np.where(np.isfinite(x), x, 0.0)
        f = exponent(np.abs(x).max())
        x8 = np.rint(x / 2.0 ** f)
        dots = np.maximum(x8 * codes[:, 0].astype(np.float64), x8 * codes[:, 1].astype(np.float64)).sum(-1)
        best = np.maximum(best, dots * 2.0 ** (f + exps.astype(np.float64)))
    return best


def keep_highest(score: np.ndarray, budget: int, sink: int, recent: int) -> list:
    """Ascending positions kept of a row of scores: first, last, then highest (ties: the lower position)."""
    n = len(score)
    if n <= budget:
        return list(range(n))
    middle = sorted(range(sink, n - recent),
                    key=lambda j: (-(score[j] if not np.isnan(score[j]) else -np.inf), np.isnan(score[j]), j))
    return sorted(list(range(sink)) + list(range(n - recent, n)) + middle[:budget - sink - recent])
