"""The prompt QKV of fp32 and bf16 weights at positions where the sum with the token's own passes
32 bits: no cache is touched, as at any position past it (4-bit weights share the epilogue)."""
import numpy as np
import pytest

import oracle
from ammon_amd._abi import BF16, F32, call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wd", [F32, BF16])
@pytest.mark.parametrize("t", [5, 40, 200])  # the tiles of few, of some and of many tokens
@pytest.mark.parametrize("first", [0xfffffffe, 0xffffffff - 150, 64, 20])
def test_positions_past_the_cache(rt, wd, t, first):
    heads, kv_heads, head, n, seq = 4, 2, 64, 256, 64
    dims = [heads * head, kv_heads * head, kv_heads * head]
    ws = [rt.upload(oracle.storage(oracle.normal(d * n, i), wd)) for i, d in enumerate(dims)]
    x, table = rt.upload(oracle.normal(t * n, 7)), rt.upload(oracle.rope_table(10000.0, head, seq))
    fits = max(0, min(t, seq - first))
    q = rt.alloc(t * dims[0] * 4)
    caches = [rt.upload(np.full(seq * dims[1], 3, np.float32)) for _ in "kv"]
    rows = [rt.alloc(t * dims[1] * 4) for _ in "kv"]
    front = [rt.handle, None, x, t, *ws, wd, n, heads, kv_heads, head, q]
    call("ammon_prefill_qkv_rope_store", *front, *caches, F32, seq, rt.step(0, first), table)
    got = q.download((t, dims[0]))
    assert np.isfinite(got[:fits]).all() and np.isnan(got[fits:]).all()
    call("ammon_prefill_qkv_rope", *front, *rows, seq, rt.step(0, first), table, None, 0)
    for cache, row in zip(caches, rows):
        c, r = cache.download((kv_heads, seq, head)), row.download((t, kv_heads, head))
        assert np.isfinite(r[:fits]).all() and np.isnan(r[fits:]).all()
        there = np.arange(seq) - min(first, seq)
        there = (there >= 0) & (there < fits)
        np.testing.assert_array_equal(c[:, there], r[:fits].transpose(1, 0, 2))
        assert (c[:, ~there] == 3).all()
