"""Grouped-query layers over 8-bit pages (oracle, test-only): the page format,
the cache write, the pages' mean keys, block selection and attention, as
``include/ernie_kv.h`` states them.

Codes, scales, summaries and selections are bit for bit what the kernels give
(fp32 steps where the rule has them, sums and products that are exact
otherwise); norm, rotation and attention are fp64.  The reference has no such
layer, so the pins are closed forms (``tests/test_oracle_gqa.py``).
"""

from __future__ import annotations

import numpy as np

from .fp8 import E4M3_MAX, bf16_round, decode_e4m3, encode_e4m3

PAGE = 64
FLOOR = np.float32(1e-10)


def page_bytes(kv_heads: int, dim: int) -> int:
    return (kv_heads * (2 * PAGE * dim + 8) + 15) // 16 * 16


def summary_bytes(kv_heads: int, dim: int) -> int:
    return (kv_heads * (dim + 4) + 15) // 16 * 16


def v_at(r):
    """Byte of token r within a channel's 64 of V."""
    r = np.asarray(r)
    return 16 * ((r // 4) % 4) + 4 * (r // 16) + r % 4


def pow2_scale(amax, top: float) -> np.ndarray:
    """2^ceil(log2(fl32(max(amax, 1e-10) * fl32(1 / top)))) as float32."""
    r = np.maximum(np.asarray(amax, np.float32), FLOOR) * np.float32(1.0 / top)
    m, e = np.frexp(r.astype(np.float32))
    return np.ldexp(np.float32(1.0), e - (m == 0.5)).astype(np.float32)


def k_codes(cache: np.ndarray, page: int, kv_heads: int, dim: int, h: int) -> np.ndarray:
    """View [64, dim] of a page's key codes."""
    at = h * PAGE * dim
    return cache[page, at:at + PAGE * dim].reshape(PAGE, dim)


def v_codes(cache: np.ndarray, page: int, kv_heads: int, dim: int, h: int) -> np.ndarray:
    """View [dim, 64] of a page's value codes, tokens in stored order."""
    at = (kv_heads + h) * PAGE * dim
    return cache[page, at:at + PAGE * dim].reshape(dim, PAGE)


def scales(cache: np.ndarray, page: int, kv_heads: int, dim: int) -> np.ndarray:
    """View [2, kv_heads] of a page's K and V scales."""
    at = 2 * kv_heads * PAGE * dim
    return cache[page, at:at + 8 * kv_heads].view(np.float32).reshape(2, kv_heads)


def summary_parts(summary: np.ndarray, page: int, kv_heads: int, dim: int):
    """Views: codes [kv_heads, dim] int8 and scales [kv_heads]."""
    rec = summary[page]
    return (rec[:kv_heads * dim].view(np.int8).reshape(kv_heads, dim),
            rec[kv_heads * dim:kv_heads * (dim + 4)].view(np.float32))


def _encode(x: np.ndarray) -> np.ndarray:
    return encode_e4m3(np.clip(x.astype(np.float32), -E4M3_MAX, E4M3_MAX))


def norm_rope(x, w, eps, cos_sin, positions, interleaved=False, offset=0) -> np.ndarray:
    """fp64 ``[T, heads, D]`` before the rounding to bf16."""
    x = np.array(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    if cos_sin is None:
        return x
    rope = cos_sin.shape[1]
    half = rope // 2
    for t, p in enumerate(positions):
        if not 0 <= p < cos_sin.shape[0]:
            continue
        c, s = cos_sin[p, :half].astype(np.float64), cos_sin[p, half:].astype(np.float64)
        i = np.arange(half)
        a, b = (offset + 2 * i, offset + 2 * i + 1) if interleaved else (offset + i, offset + half + i)
        u, v = x[t][:, a].copy(), x[t][:, b].copy()
        x[t][:, a], x[t][:, b] = u * c - v * s, v * c + u * s
    return x


def append(k, v, positions, qsl, block_table, cache, summary=None) -> None:
    """In place: bf16-valued rows ``k, v [T, kv_heads, D]`` into their pages."""
    _, KV, D = k.shape
    for b in range(len(qsl) - 1):
        t0, n = int(qsl[b]), int(qsl[b + 1] - qsl[b])
        if n <= 0 or positions[t0] < 0:
            continue
        p0 = int(positions[t0])
        for lp in range(p0 // PAGE, (p0 + n - 1) // PAGE + 1):
            page = int(block_table[b, lp]) if lp < block_table.shape[1] else -1
            if not 0 <= page < cache.shape[0]:
                continue
            lo, hi = max(p0, lp * PAGE), min(p0 + n, (lp + 1) * PAGE)
            first, end = lo - lp * PAGE, hi - lp * PAGE
            sc = scales(cache, page, KV, D)
            for h in range(KV):
                for i, x in enumerate((k, v)):
                    new = x[t0 + lo - p0:t0 + hi - p0, h].astype(np.float32)
                    s = pow2_scale(np.abs(new).max(), 448.0)
                    old = sc[i, h]
                    if first:
                        s = max(s, old)
                    grow = first and s > old
                    codes = (k_codes(cache, page, KV, D, h) if i == 0 else
                             v_codes(cache, page, KV, D, h).T)  # [token, D]; V in stored order
                    at = np.arange(PAGE) if i == 0 else v_at(np.arange(PAGE))
                    if grow:
                        codes[at[:first]] = _encode(decode_e4m3(codes[at[:first]]) * (old / s))
                    codes[at[first:end]] = _encode(new / s)
                    sc[i, h] = s
                if summary is not None:
                    mean = decode_e4m3(k_codes(cache, page, KV, D, h)[:end]).astype(np.float64).sum(0)
                    mean = mean.astype(np.float32) / np.float32(end)
                    e = pow2_scale(np.abs(mean).max(), 127.0)
                    cs, ss = summary_parts(summary, page, KV, D)
                    cs[h] = np.clip(np.rint(mean / e), -127, 127).astype(np.int8)
                    ss[h] = e * sc[0, h]


def tokens(cache, pages, kv_heads: int, dim: int, h: int):
    """fp64 keys and values ``[64 len(pages), dim]`` of one head."""
    ks, vs = [], []
    for p in pages:
        s = scales(cache, int(p), kv_heads, dim).astype(np.float64)
        ks.append(decode_e4m3(k_codes(cache, int(p), kv_heads, dim, h)).astype(np.float64) * s[0, h])
        vs.append(decode_e4m3(v_codes(cache, int(p), kv_heads, dim, h)).astype(np.float64).T[v_at(np.arange(PAGE))]
                  * s[1, h])
    return (np.concatenate(ks), np.concatenate(vs)) if ks else (np.zeros((0, dim)), np.zeros((0, dim)))


def attend(q, keys, vals, scale: float, sink=None):
    """One row ``q [D]`` over keys and values ``[n, D]``: (out, lse, sum of
    |weight * value|, sum over channels of |q k| at most); empty: zeros, -inf."""
    if not len(keys):
        z = np.zeros(vals.shape[1])
        return z, -np.inf, z, 0.0
    q = np.asarray(q, np.float64)
    s = keys @ q * scale
    m = s.max() if sink is None else max(s.max(), float(sink))
    e = np.exp(s - m)
    den = e.sum()
    lse = m + np.log(den) if den > 0 else s.max() + np.log(np.exp(s - s.max()).sum())
    if sink is not None:
        den = den + np.exp(float(sink) - m)
    return e @ vals / den, lse, e @ np.abs(vals) / den, float((np.abs(keys) @ np.abs(q)).max()) * abs(scale)


def select(q, summary, kv_heads: int, block_row, position: int, n: int, keep_first: int, keep_last: int) -> np.ndarray:
    """``[kv_heads, n]`` for one row ``q [H, D]`` (bf16 values)."""
    H, D = q.shape
    G = H // kv_heads
    out = np.full((kv_heads, n), -1, np.int32)
    nb = 0 if position < 0 else min(position // PAGE + 1, len(block_row))
    for h in range(kv_heads):
        x = np.asarray(q[h * G:(h + 1) * G], np.float32)
        e = pow2_scale(np.abs(x).max(), 127.0)
        codes = np.clip(np.rint(x / e), -127, 127).astype(np.int64)
        score = np.full(nb, -np.inf)
        for j in range(nb):
            page = int(block_row[j])
            if 0 <= page < summary.shape[0]:
                mc, ms = summary_parts(summary, page, kv_heads, D)
                score[j] = np.inf if j < keep_first or j >= nb - keep_last else float(
                    (codes @ mc[h].astype(np.int64)).max()) * float(ms[h])
        order = np.argsort(-score, kind="stable")[:n]
        order = np.sort(order[score[order] > -np.inf])
        out[h, :len(order)] = order
    return out


__all__ = ["append", "attend", "bf16_round", "norm_rope", "page_bytes", "select", "summary_bytes", "tokens"]
