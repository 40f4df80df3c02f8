"""4-bit weights (AMMON_W4) and rows of 8-bit digits (AMMON_Q8, AMMON_Q24) restated in numpy --
TEST INFRASTRUCTURE.

Every step of the definitions in include/ammon/ammon.h is computed in float64 and rounded where
the definition rounds; nothing is shared with the kernels.  Products are float64 over the stored
numbers.  Matrices and rows are the byte arrays that the kernels read.
"""
from __future__ import annotations

import numpy as np

GROUP = 128


def groups(n: int) -> int:
    return -(-n // GROUP)


def w4_bytes(d: int, n: int) -> int:
    return -(-d // 16) * groups(n) * 1056


def q8_bytes(digits: int, tokens: int, n: int) -> int:
    return -(-tokens // 16) * groups(n) * (2048 * digits + 64)


def f32(x):
    with np.errstate(over="ignore"):
        return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def bf16(x):
    """fp32 numbers (float64) rounded to nearest even bf16."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = ((u + 0x7fff + ((u >> 16) & 1)) & 0xffff0000).astype(np.uint32)
    return np.where(np.isnan(x), np.nan, u.view(np.float32).astype(np.float64))


def blocks(x):
    """Rows [r, n] as [r, groups, 128], zeros past the end (float64)."""
    x = np.asarray(x, np.float64)
    out = np.zeros((x.shape[0], groups(x.shape[1]) * GROUP))
    out[:, :x.shape[1]] = x
    return out.reshape(x.shape[0], -1, GROUP)


def _ends(b):
    bad = ~np.isfinite(b).all(-1)
    return bad, np.abs(np.where(np.isfinite(b), b, 0)).max(-1), np.where(bad[..., None], 0, b)


def w4_quantise(w):
    """Codes [d, groups, 128] and scales [d, groups] of a matrix."""
    bad, top, b = _ends(blocks(w))
    s = bf16(f32(top / 7))
    s = np.where(s < 2.0**-126, 0, s)
    inv = np.where(s > 0, f32(1 / np.where(s > 0, s, 1)), 0)
    c = np.clip(np.rint(f32(b * inv[..., None])), -7, 7)
    return c.astype(np.int8), np.where(bad, np.nan, s)


def w4_numbers(codes, s, n):
    return (codes * s[..., None]).reshape(codes.shape[0], -1)[:, :n]


def w4_pack(codes, s):
    """The bytes of codes [d, groups, 128] and scales [d, groups]."""
    d, g = s.shape
    panels = -(-d // 16)
    c = np.zeros((panels * 16, g, GROUP), np.uint8)
    c[:d] = codes.astype(np.int8).view(np.uint8) & 15
    sc = np.zeros((panels * 16, g), np.float32)
    sc[:d] = s
    c = c.reshape(panels, 16, g, 4, 2, 16)  # panel, row, group, piece, half, byte
    byte = c[..., 0, :] | c[..., 1, :] << 4
    out = np.zeros((panels, g * 1056), np.uint8)
    out[:, :g * 1024] = byte.transpose(0, 2, 3, 1, 4).reshape(panels, -1)
    top = (sc.view(np.uint32) >> 16).astype("<u2").reshape(panels, 4, 4, g)
    out[:, g * 1024:] = np.ascontiguousarray(top.transpose(0, 1, 3, 2)).view(np.uint8).reshape(panels, -1)
    return out.reshape(-1)


def q_quantise(x, digits):
    """Whole numbers [tokens, blocks, 128] and scales [tokens, blocks] of rows."""
    bad, top, b = _ends(blocks(x))
    if digits == 1:
        s = f32(top / 127)
        s = np.where(s < 2.0**-120, 0, s)
        inv = np.where(s > 0, f32(1 / np.where(s > 0, s, 1)), 0)
        q = np.clip(np.rint(f32(b * inv[..., None])), -127, 127)
    else:
        s = np.full(top.shape, 2.0**-120)
        while (top >= 127 * 65536 * s).any():
            s = np.where(top >= 127 * 65536 * s, 2 * s, s)
        q = np.rint(b / s[..., None])
    return q.astype(np.int32), np.where(bad, np.nan, s)


def q_numbers(q, s, n):
    return f32(q * s[..., None]).reshape(q.shape[0], -1)[:, :n]


def q_pack(q, s, digits, into=None):
    """The bytes of rows; what a panel's tokens past the last one hold is kept from `into`."""
    t, b = s.shape
    panels = -(-t // 16)
    size = b * (2048 * digits + 64)
    out = (np.zeros(panels * size, np.uint8) if into is None else into.copy()).reshape(panels, size)
    scales = np.ascontiguousarray(s, "<f4")
    rest, low = np.asarray(q, np.int64), []
    for _ in range(digits):
        low.append((rest + 128) % 256 - 128)
        rest = (rest - low[-1]) // 256
    assert not rest.any()
    # token, block, digit, piece, half, byte
    numbers = np.stack(low, 2).astype(np.int8).view(np.uint8).reshape(t, b, digits, 4, 2, 16)
    for i in range(panels):
        n = min(16, t - 16 * i)
        at = out[i, :b * 2048 * digits].reshape(b, digits, 2, 4, 16, 16)  # .., token, byte
        at[:, :, :, :, :n] = numbers[16 * i:16 * i + n].transpose(1, 2, 4, 3, 0, 5)
        at = out[i, b * 2048 * digits:].reshape(b, 16, 4)
        at[:, :n] = np.ascontiguousarray(scales[16 * i:16 * i + n].T).view(np.uint8).reshape(b, n, 4)
    return out.reshape(-1)


def normed(x, w, eps):
    """RMSNorm as ammon_rmsnorm_q8 defines it: the mean and its root in 64 bits, the rest in 32."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        r = f32(1 / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))))
        return f32(np.asarray(w, np.float64) * f32(r * x))


def product_bar(x, w, exact_x):
    """How far fp32 results of rows x [t, n] (float64) times w [d, n] may be from float64's [t, d], a
    rounding being 2^-24 of its result.  With S = sum |w| |x|:

    Rows of digits (exact_x True).  A group's digits are joined by a conversion and an addition, at
    most 2^-24 of the group's part of S each, and added up with one more, of S: 2 + groups.  Waves
    (of which no more than groups have any), ranges and a residual add at most 16, 7 and 1 of S:
    2 groups + 16 in all, or less (groups + 3 + groups with fewer groups than waves).

    One token (exact_x False), whose x is made 32-bit whole numbers.  A number is off by half a step,
    2^-30.98 of its block's largest (2^-121 where that is below 2^-90).  The four digits' sums are
    added up apart, one rounding a group, then with each other (3) and over waves (16): again within
    2 groups + 16, but of the digits' sizes instead of |x|.  A digit's remainder is at most half a
    unit of the digit above, so that their sizes together are at most |x| + 6.1 times the remainder
    of the highest one, which is no larger than |x| and than 1 / 127 of the block's largest."""
    a, b = np.abs(x), np.abs(w)
    rounding = (2 * groups(x.shape[1]) + 16) * 2.0**-24
    if exact_x:
        return rounding * a @ b.T
    size = blocks(a)
    top = size.max(-1)  # [t, groups]
    size = (size + 6.1 * np.minimum(size, top[..., None] / 127)).reshape(len(a), -1)[:, :x.shape[1]]
    return rounding * size @ b.T + 2.0**-30.98 * top @ blocks(b).sum(-1).T
