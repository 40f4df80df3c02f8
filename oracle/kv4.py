"""The 4-bit KV cache (AMMON_KV4) restated in numpy -- TEST INFRASTRUCTURE.

Every step of the definition in include/ammon/ammon.h is computed in float64
and rounded where the definition rounds (fp32 unless it says fp16), element by
element; nothing is shared with the kernels.  Attention over the stored
numbers is float64.  A cache is the byte array the kernels read: codes, then
scales and biases.
"""
from __future__ import annotations

import numpy as np

LIMIT = 16384.0


def groups(head: int) -> int:
    return (head + 31) // 32


def cache_bytes(kv_heads: int, seq: int, head: int) -> int:
    return 20 * groups(head) * kv_heads * seq


def _f32(x):
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def _f16(x):
    return np.asarray(x, np.float64).astype(np.float16).astype(np.float64)


def quantise(x: np.ndarray):
    """Rows x [..., head] as (codes [..., head] in 0..15, s, b [..., groups] fp16)."""
    x = np.asarray(x, np.float32).astype(np.float64)
    n, head = groups(x.shape[-1]), x.shape[-1]
    codes = np.zeros(x.shape, np.uint8)
    s, b = (np.zeros(x.shape[:-1] + (n,), np.float16) for _ in range(2))
    with np.errstate(invalid="ignore", divide="ignore"):
        for j in range(n):
            y = x[..., 32 * j:min(head, 32 * j + 32)]
            bad = ~np.isfinite(y).all(-1)
            y = np.clip(y, -LIMIT, LIMIT)
            lo, hi = y.min(-1), y.max(-1)
            sj = _f16(_f32(_f32(hi - lo) / 15))
            bj = _f16(_f32(lo - 16 * sj))
            inv = np.where(sj > 0, _f32(1 / np.where(sj > 0, sj, 1)), 0)
            c = _f32(_f32(_f32(y - bj[..., None]) * inv[..., None]) - 16)
            c = np.clip(np.rint(c), 0, 15)
            codes[..., 32 * j:32 * j + 32] = np.where(bad[..., None], 0, c)
            s[..., j] = np.where(bad, np.nan, sj)
            b[..., j] = np.where(bad, np.nan, bj)
    return codes, s, b


def numbers(codes, s, b) -> np.ndarray:
    """What codes with their groups' s and b stand for (float64; fp16 numbers)."""
    j = np.arange(codes.shape[-1]) // 32
    s, b = (np.asarray(t, np.float64)[..., j] for t in (s, b))
    with np.errstate(invalid="ignore"):
        return _f16(s * (16.0 + codes) + b)


def stored(x: np.ndarray) -> np.ndarray:
    """What rows x read back as."""
    return numbers(*quantise(x))


def _place(d: int, n: int):
    """(word of the row, shift) of number d."""
    j, p, e = d // 32, d % 32 // 8, d % 8
    return p * n + j, 4 * (e // 2 + 4 * (e % 2))


def pack(cache: np.ndarray, kv_heads: int, seq: int, head: int, first: int, rows: np.ndarray):
    """Store rows [kv_heads, count, head] at positions first.. of `cache` (uint8)."""
    n, count = groups(head), rows.shape[1]
    codes, s, b = quantise(rows)
    words = np.zeros((kv_heads, count, 4 * n), np.uint32)
    for d in range(head):
        w, shift = _place(d, n)
        words[..., w] |= codes[..., d].astype(np.uint32) << np.uint32(shift)
    c, sb = views(cache, kv_heads, seq, head)
    c[:, first:first + count] = words
    sb[:, first:first + count] = s.view(np.uint16).astype(np.uint32) | \
        b.view(np.uint16).astype(np.uint32) << np.uint32(16)


def views(cache: np.ndarray, kv_heads: int, seq: int, head: int):
    """The words of a cache: codes [kv_heads, seq, 4 groups], s | b << 16 [kv_heads, seq, groups]."""
    n, w = groups(head), cache.view(np.uint32)
    k = kv_heads * seq * 4 * n
    return w[:k].reshape(kv_heads, seq, 4 * n), w[k:k + kv_heads * seq * n].reshape(kv_heads, seq, n)


def read(cache: np.ndarray, kv_heads: int, seq: int, head: int, first: int, count: int):
    """The numbers [kv_heads, count, head] of positions first.. (float64)."""
    n = groups(head)
    c, sb = (t[:, first:first + count] for t in views(cache, kv_heads, seq, head))
    codes = np.zeros((kv_heads, count, head), np.uint8)
    for d in range(head):
        w, shift = _place(d, n)
        codes[..., d] = (c[..., w] >> np.uint32(shift)) & np.uint32(15)
    s = (sb & np.uint32(0xffff)).astype(np.uint16).view(np.float16)
    b = (sb >> np.uint32(16)).astype(np.uint16).view(np.float16)
    return numbers(codes, s, b)


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, first: int) -> np.ndarray:
    """float64 attention of q [tokens, q_heads, head] at positions first.. over the numbers k, v
    [kv_heads, >= first + tokens, head]."""
    q = np.asarray(q, np.float64)
    tokens, heads, head = q.shape
    g, ctx = heads // k.shape[0], first + tokens
    seen = np.arange(ctx)[None, :] <= first + np.arange(tokens)[:, None]
    out = np.empty_like(q)
    with np.errstate(invalid="ignore"):
        for h in range(heads):
            kk, vv = k[h // g, :ctx], v[h // g, :ctx]
            s = np.where(seen, q[:, h] @ kk.T / np.sqrt(head), -np.inf)
            p = np.exp(s - s.max(-1, keepdims=True))  # NaN where a seen score is
            bad = ~np.isfinite(vv)
            o = p @ np.where(bad, 0, vv) / p.sum(-1, keepdims=True)
            # a number that is not finite is NaN (a group is), and so is its sum wherever it is seen
            out[:, h] = np.where(seen.astype(np.float64) @ bad > 0, np.nan, o)
    return out
