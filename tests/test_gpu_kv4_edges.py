"""The 4-bit KV cache (AMMON_KV4) at the ends of its ranges.  The bar, and what it is
made of, is test_gpu_kv4's.
"""
import numpy as np
import pytest

import oracle
from ammon_amd import _abi
from ammon_amd._abi import F32, KV4, AmmonError, call, lib
from oracle import kv4
from test_gpu_kv4 import TOL, Cache, decode, off, prefill, rows_of, up

pytestmark = pytest.mark.gpu


# ---- query rows of subnormal numbers --------------------------------------------------------------
# Every score is within 2^-100 of 0, so a token's result is the mean of what it sees.
TINY = [2.0**-133, 2.0**-136, 2.0**-140, 2.0**-147]


@pytest.mark.parametrize("heads,kv_heads,head", [(8, 2, 128), (6, 2, 96), (4, 4, 48), (8, 1, 20)])
@pytest.mark.parametrize("scale", TINY)
def test_tiny_q_with_masked_positions(rt, heads, kv_heads, head, scale):
    # positions that end inside a wave's 64, so that scores are masked
    for pos in (0, 5, 200, 255, 299):
        a, b = (Cache(rt, kv_heads, 300, head, filled=n) for n in (pos + 1, pos))
        q = (oracle.normal(heads * head, 9).reshape(heads, head) * np.float32(scale)).astype(np.float32)
        q[:, 0] = scale * 2  # (no row is all zeros)
        want = kv4.attention(q[None], *a.numbers(pos + 1), pos)[0]
        for split in (300, 128):
            assert off(decode(rt, q, a, pos, split), want) <= TOL, (pos, split)
        k, v = rows_of(kv_heads, 1, head, 5), rows_of(kv_heads, 1, head, 50)
        got = decode(rt, q, b, pos, 128, new=(k, v))
        b.pack(pos, k, v)
        assert off(got, kv4.attention(q[None], *b.numbers(pos + 1), pos)[0]) <= TOL, pos


@pytest.mark.parametrize("scale", TINY)
@pytest.mark.parametrize("start,tokens", [(0, 1), (40, 9), (250, 13), (2000, 400)])  # units, and tiles
def test_tiny_q_of_a_prompt(rt, start, tokens, scale):
    c = Cache(rt, 2, 2600, 128, filled=start + tokens)
    q = (oracle.normal(tokens * 1024, 9).reshape(tokens, 8, 128) * np.float32(scale)).astype(np.float32)
    want = kv4.attention(q, *c.numbers(start + tokens), start)
    for split in (64, 1024):
        assert off(prefill(rt, q, c, start, split), want) <= TOL


# ---- scores too large for fp32 to hold their distance to a maximum exactly ------------------------
def huge(rt, heads, kv_heads, head, seq, tokens, start, size):
    """A cache of rows near the format's limit, and q: of each row of scores the largest is so far
    above the rest that its weight is 1 (the others' distances are above 100, while a score's error is
    at most 2^-21 of |q| |k| / sqrt(head), a tenth of them or less)."""
    c = Cache(rt, kv_heads, seq, head)
    rows = [rows_of(kv_heads, start + tokens, head, s) for s in (1, 11)]
    rows[0] *= np.float32(4000)
    c.pack(0, *rows)
    c.dev = [up(rt, h) for h in c.host]
    q = (oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head) * np.float32(size)).astype(np.float32)
    k, _ = c.numbers(start + tokens)
    for t in range(tokens):
        for h in range(heads):
            x = k[h // (heads // kv_heads), :start + t + 1]
            qh = q[t, h].astype(np.float64)
            s = np.sort(x @ qh) / np.sqrt(head)
            err = 2.0**-21 * np.linalg.norm(qh) * np.max(np.linalg.norm(x, axis=1)) / np.sqrt(head)
            if len(s) > 1 and s[-1] - s[-2] < max(100, 10 * err):
                q[t, h] = 0  # (rows of no clear winner are left out)
    assert (q != 0).any(-1).mean() > 0.7
    return c, q


SIZES = [30.0, 3e3, 1e4, 1e6, 1e9, 1e20]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("heads,kv_heads,head", [(8, 2, 128), (6, 2, 96), (4, 4, 48), (8, 1, 20)])
def test_scores_of_any_size(rt, heads, kv_heads, head, size):
    for pos in (63, 200, 299):
        c, q = huge(rt, heads, kv_heads, head, 300, 1, pos, size)
        want = kv4.attention(q, *c.numbers(pos + 1), pos)[0]
        for split in (300, 128, 16):
            assert off(decode(rt, q[0], c, pos, split), want) <= TOL, (pos, split)
        rows = [x[:, pos].astype(np.float32)[None] for x in c.numbers(pos + 1)]
        b = Cache(rt, kv_heads, 300, head)
        for h, x in zip(b.host, c.host):
            h[:] = x
        b.pack(pos, *rows)  # (stored numbers stored again)
        b.dev = [up(rt, h) for h in b.host]
        want = kv4.attention(q, *b.numbers(pos + 1), pos)[0]
        assert off(decode(rt, q[0], b, pos, 128, new=rows), want) <= TOL, pos


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("start,tokens", [(0, 6), (40, 9), (250, 13), (2000, 300)])  # units, and tiles
def test_scores_of_any_size_of_a_prompt(rt, start, tokens, size):
    c, q = huge(rt, 8, 2, 128, 2600, tokens, start, size)
    want = kv4.attention(q, *c.numbers(start + tokens), start)
    for split in (64, 1024):
        assert off(prefill(rt, q, c, start, split), want) <= TOL


# ---- groups with one word of scale and bias that is not finite ------------------------------------
@pytest.mark.parametrize("word", [0x7e000000, 0x00007e00, 0xfe00fe00])  # bias, scale, both (NaN)
@pytest.mark.parametrize("start,tokens", [(250, 13), (700, 400)])  # units, tiles
def test_half_of_a_group_not_finite(rt, start, tokens, word):
    """A later token's NaN does not reach an earlier one, whichever of the two it is in."""
    heads, kv_heads, head = 8, 4, 128
    last = start + tokens - 1
    for side in (0, 1):
        c = Cache(rt, kv_heads, 1200, head, filled=start + tokens)
        sb = kv4.views(c.host[side], kv_heads, 1200, head)[1]
        keep = 0xffff if word == 0x7e000000 else 0xffff0000 if word == 0x7e00 else 0
        for g, at, j in ((0, last, 1), (1, start + tokens // 2, 3), (2, start, 0)):
            sb[g, at, j] = (int(sb[g, at, j]) & keep) | word
        c.dev[side].upload(c.host[side])
        q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
        want = kv4.attention(q, *c.numbers(start + tokens), start)
        nan = np.isnan(want).any(-1)
        assert nan[-1, :6].all() and not nan[:-1, :2].any() and not nan[:tokens // 2, 2:4].any()
        assert nan[:, 4:6].all() and not nan[:, 6:].any()
        for split in (64, 1024):
            assert off(prefill(rt, q, c, start, split), want) <= TOL


# ---- which kernel a prompt gets -------------------------------------------------------------------
def prefill_scratch(rt, q, c, start, split, shift=0):
    """The result, and how much of the scratch was written: units write a part of every row for every
    `split` positions, tiles of ranges as long as they choose."""
    tokens, heads = q.shape[:2]
    ctx = start + tokens
    n = int(lib.ammon_attention_prefill_scratch_bytes(tokens, heads, c.head, ctx, split))
    part, out = rt.alloc(n + 4), rt.alloc(q.nbytes + 4)
    for buf, count in ((part, n // 4 + 1), (out, q.size + 1)):
        rt.fill(buf, F32, count, 7.0)
    dq = up(rt, np.concatenate([np.zeros(1, np.float32), q.ravel()]) if shift else q)
    call("ammon_attention_prefill", rt.handle, None, dq.offset(4 * shift), tokens, heads, *c.dev, KV4,
         c.kv_heads, c.head, c.seq, rt.step(0, start), ctx, split, part.offset(4 * shift), n,
         out.offset(4 * shift))
    got, used = out.download(q.size + 1), part.download(n // 4 + 1)
    assert got[0 if shift else -1] == 7.0 and used[0 if shift else -1] == 7.0
    return got[shift:shift + q.size].reshape(q.shape), np.mean(used != 7.0)


@pytest.mark.parametrize("heads,kv_heads,head,start,tokens", [(2, 1, 64, 131072, 200), (4, 1, 128, 131000, 73),
                                                              (2, 2, 40, 130950, 300), (1, 1, 32, 290001, 333)])
def test_tiles_past_131072_positions(rt, heads, kv_heads, head, start, tokens):
    c = Cache(rt, kv_heads, start + tokens + 3, head, filled=start + tokens)
    q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
    want = kv4.attention(q, *c.numbers(start + tokens), start)
    got, used = prefill_scratch(rt, q, c, start, 256)
    assert off(got, want) <= TOL
    assert used < 0.6  # units write nearly all of it


@pytest.mark.parametrize("heads,kv_heads,head", [(32, 8, 128), (18, 6, 96), (8, 8, 64), (6, 6, 33)])
@pytest.mark.parametrize("start,tokens", [(0, 700), (1500, 500)])
def test_tiles_of_rows_at_any_float(rt, heads, kv_heads, head, start, tokens):
    """q, the scratch and the output a float past 16 bytes: the same kernel, the same numbers."""
    c = Cache(rt, kv_heads, 2100, head, filled=start + tokens)
    q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
    want = kv4.attention(q, *c.numbers(start + tokens), start)
    got, used = prefill_scratch(rt, q, c, start, 64)
    shifted, used_shifted = prefill_scratch(rt, q, c, start, 64, shift=1)
    assert off(got, want) <= TOL
    np.testing.assert_array_equal(got, shifted)
    assert abs(used - used_shifted) < 1e-6 and used < 0.6


# ---- more rows than a launch takes (nothing is launched) --------------------------------------------
@pytest.mark.parametrize("rows,kv_heads,fits", [((1 << 28) - 16, 1, True), ((1 << 28) - 15, 1, False),
                                               ((1 << 25) - 2, 8, True), ((1 << 25) - 1, 8, False),
                                               (0xffffffff, 1, False)])
def test_rows_of_one_launch(rt, rows, kv_heads, fits):
    """16 lanes a row (of a load four rows), fewer than 2^32 lanes."""
    V, step = _abi.STREAM_VALIDATE, rt.step(0, 0)
    at = [1 << n for n in (50, 51, 52, 53)]  # (nothing is read or written)
    store = ("ammon_kv4_store", rt.handle, V, at[0], at[1], rows, kv_heads, 1, at[2], at[3], 100, step)
    load = ("ammon_kv4_load", rt.handle, V, at[2], at[3], kv_heads, 1, 0xffffffff, 0, min(4 * rows, 0xffffffff),
            at[0], at[1], F32)
    for c in (store, load):
        if fits:
            call(*c)
            continue
        with pytest.raises(AmmonError, match="too many rows") as e:
            call(*c)
        assert e.value.status == _abi.E_VALIDATION
