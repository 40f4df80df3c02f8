"""The 4-bit KV cache (AMMON_KV4) at the ends of its ranges.  The bar, and what it is
made of, is test_gpu_kv4's.
"""
import numpy as np
import pytest

import oracle
from oracle import kv4
from test_gpu_kv4 import TOL, Cache, decode, off, prefill, rows_of

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
