"""The 4-bit KV cache (AMMON_KV4) on the GPU: rows stored and read back, decode attention over
them, alone and with the new row stored, against the numpy restatement (oracle/kv4.py).

Stored rows are compared bit for bit: the definition fixes every rounding.  Attention is compared
with float64 over the stored numbers, normwise.  Its bar, 3e-6 of the largest output, is made of:
q in two fp16 parts and the weights in two fp16 parts (2^-22 each of the largest, 2.4e-7; a
score's error is the weight's relative one: |q| |k| / sqrt(head) < 4 in these inputs, so 4 x 2.4e-7
there), fp32 sums (scores: 4 matrix products and one addition, values: at most 32 products in a
chain, 2^-24 each at most: 2e-6) and 2^-23 of the base-2 exponential's argument (below 8).
"""
import ctypes

import numpy as np
import pytest

import oracle
from ammon_amd import _abi
from ammon_amd._abi import BF16, F32, KV4, AmmonError, call, lib
from oracle import kv4

pytestmark = pytest.mark.gpu
TOL = 3e-6
HEADS = [1, 2, 7, 16, 31, 32, 33, 48, 64, 65, 80, 96, 100, 112, 127, 128]
SHAPES = [(32, 8, 128), (16, 2, 128), (6, 6, 48), (6, 2, 96), (4, 1, 80), (5, 5, 32), (14, 2, 64),
          (3, 1, 127), (8, 8, 16), (2, 1, 1), (7, 7, 100)]


def up(rt, a):
    return rt.upload(np.ascontiguousarray(a))


def rows_of(kv_heads, n, head, seed):
    """Rows as rotated keys are: channels with sizes and means of their own."""
    x = oracle.normal(n * kv_heads * head, seed).reshape(n, kv_heads, head)
    size = 0.5 + np.abs(oracle.normal(kv_heads * head, seed + 1).reshape(kv_heads, head))
    return (x * size + oracle.normal(kv_heads * head, seed + 2).reshape(kv_heads, head)).astype(np.float32)


class Cache:
    """K and V caches on the host and the device; what is not written is 0xff (NaN)."""

    def __init__(self, rt, kv_heads, seq, head, filled=0, seed=1):
        self.rt, self.kv_heads, self.seq, self.head = rt, kv_heads, seq, head
        n = kv4.cache_bytes(kv_heads, seq, head)
        assert lib.ammon_kv_cache_bytes(KV4, kv_heads, seq, head) == n
        self.host = [np.full(n, 0xff, np.uint8) for _ in "kv"]
        for i, c in enumerate(self.host):
            if filled:
                rows = rows_of(kv_heads, filled, head, seed + 10 * i)
                kv4.pack(c, kv_heads, seq, head, 0, rows.transpose(1, 0, 2))
        self.dev = [up(rt, c) for c in self.host]

    def numbers(self, count, first=0):
        return [kv4.read(c, self.kv_heads, self.seq, self.head, first, count) for c in self.host]

    def pack(self, first, k, v):
        """Rows [tokens, kv_heads, head] into the host copies."""
        for c, rows in zip(self.host, (k, v)):
            kv4.pack(c, self.kv_heads, self.seq, self.head, first, rows.transpose(1, 0, 2))

    def same(self):
        for name, h, d in zip("kv", self.host, self.dev):
            np.testing.assert_array_equal(d.download(h.shape, np.uint8), h, err_msg=name)


def store(rt, cache, k, v, pos, stream=None):
    tokens = k.shape[0]
    call("ammon_kv4_store", rt.handle, stream, up(rt, k), up(rt, v), tokens, cache.kv_heads,
         cache.head, *cache.dev, cache.seq, rt.step(0, pos))
    rt.synchronize(stream)


# ---- rows ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("head", HEADS)
@pytest.mark.parametrize("tokens,kv_heads", [(1, 8), (19, 3)])
def test_store_is_the_definition(rt, head, tokens, kv_heads):
    c = Cache(rt, kv_heads, 40, head)
    k, v = (rows_of(kv_heads, tokens, head, s) for s in (5, 50))
    store(rt, c, k, v, 11)
    c.pack(11, k, v)
    c.same()  # every other row as it was


def test_store_long(rt):
    c = Cache(rt, 8, 2100, 128)
    k, v = (rows_of(8, 2048, 128, s) for s in (5, 50))
    store(rt, c, k, v, 52)
    c.pack(52, k, v)
    c.same()


def special_rows(head):
    rng = np.random.default_rng(3)
    rows = [np.zeros(head), np.full(head, -0.0), np.full(head, 3.25), np.full(head, 1e-30),
            rng.normal(size=head) * 1e-6, rng.normal(size=head) * 1e-8, rng.normal(size=head) * 1e4,
            rng.normal(size=head) * 1e30, 100 + 0.01 * rng.normal(size=head),
            np.where(np.arange(head) % 2, 65504.0, -65504.0), np.where(np.arange(head) % 3, 0, 1e38)]
    for bad in (np.nan, np.inf, -np.inf):
        r = rng.normal(size=head)
        r[head // 2] = bad
        rows.append(r)
    r = rng.normal(size=head)
    r[0], r[-1] = np.inf, -np.inf
    rows.append(r)
    # codes at and next to a border: multiples of half a step
    rows.append((np.arange(head) % 32) * 0.5)
    rows.append(np.nextafter(((np.arange(head) % 32) * 0.5).astype(np.float32), np.float32(100)))
    return np.array(rows, np.float32)


@pytest.mark.parametrize("head", [128, 100, 48, 33, 1])
def test_store_special_values(rt, head):
    rows = special_rows(head)
    k = rows[:, None, :]
    c = Cache(rt, 1, len(rows), head)
    store(rt, c, k, k[::-1].copy(), 0)
    c.pack(0, k, k[::-1])
    c.same()


def test_store_past_the_cache_is_left_out(rt):
    c = Cache(rt, 2, 20, 64)
    k, v = (rows_of(2, 6, 64, s) for s in (5, 50))
    store(rt, c, k, v, 17)
    c.pack(17, k[:3], v[:3])
    c.same()
    for pos in (20, 0xffffffff, 0xfffffffd):
        store(rt, c, k, v, pos)
        c.same()


@pytest.mark.parametrize("head", HEADS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_load_is_the_definition(rt, head, dtype):
    kv_heads, seq, first, count = 3, 50, 9, 33
    c = Cache(rt, kv_heads, seq, head, filled=seq)
    n = kv_heads * count * head
    out = [rt.alloc(n * 4 + 64) for _ in "kv"]
    for o in out:
        rt.fill(o, F32, n + 16, 7.0)
    call("ammon_kv4_load", rt.handle, None, *c.dev, kv_heads, head, seq, first, count, *out, dtype)
    es = 2 if dtype == BF16 else 4
    for o, want in zip(out, c.numbers(count, first)):
        got = o.download(n * 4 + 64, np.uint8)
        want = want.astype(np.float32)  # exact: fp16 numbers
        want = oracle.to_bf16(want) if dtype == BF16 else want
        np.testing.assert_array_equal(got[:n * es], want.reshape(-1).view(np.uint8))
        assert set(got[(n * es + 3) // 4 * 4:].view(np.float32)) == {7.0}  # nothing behind the last row


def test_load_keys_alone_and_nothing(rt):
    c = Cache(rt, 2, 8, 32, filled=8)
    out = rt.upload(np.full(2 * 8 * 32, 5, np.float32))
    call("ammon_kv4_load", rt.handle, None, c.dev[0], None, 2, 32, 8, 8, 0, out, None, F32)
    assert np.all(out.download(2 * 8 * 32) == 5)
    call("ammon_kv4_load", rt.handle, None, c.dev[1], None, 2, 32, 8, 0, 8, out, None, F32)
    np.testing.assert_array_equal(out.download((2, 8, 32)), c.numbers(8)[1])


def test_store_then_load_special_values(rt):
    rows = special_rows(96)
    c = Cache(rt, 1, len(rows), 96)
    store(rt, c, rows[:, None], rows[:, None], 0)
    out = [rt.alloc(rows.nbytes) for _ in "kv"]
    call("ammon_kv4_load", rt.handle, None, *c.dev, 1, 96, len(rows), 0, len(rows), *out, F32)
    for o in out:
        np.testing.assert_array_equal(o.download(rows.shape), kv4.stored(rows).astype(np.float32))


@pytest.mark.parametrize("heads,kv_heads,head", [s for s in SHAPES if s[2] % 2 == 0])
def test_rope_store_and_cache_store(rt, heads, kv_heads, head):
    seq, pos = 30, 13
    table = np.empty((seq, head // 2, 2), np.float32)
    call("ammon_rope_table_host", 10000.0, head, seq, table.ctypes.data)
    q = rows_of(heads, 1, head, 4)[0]
    k, v = rows_of(kv_heads, 1, head, 5), rows_of(kv_heads, 1, head, 50)
    c = Cache(rt, kv_heads, seq, head)
    dq, step = up(rt, q), rt.step(0, pos)
    call("ammon_rope_store", rt.handle, None, dq, heads, up(rt, k), kv_heads, head, c.dev[0], KV4,
         seq, step, up(rt, table))
    call("ammon_cache_store", rt.handle, None, up(rt, v), kv_heads, head, c.dev[1], KV4, seq, step)

    def rotate(x):  # fp32, products rounded before the sum
        cs, out = table[pos], np.empty_like(x)
        a, b = x[..., 0::2], x[..., 1::2]
        out[..., 0::2] = a * cs[:, 0] - b * cs[:, 1]
        out[..., 1::2] = a * cs[:, 1] + b * cs[:, 0]
        return out
    np.testing.assert_array_equal(dq.download(q.shape), rotate(q))
    c.pack(pos, rotate(k), v)
    c.same()
    call("ammon_rope_store", rt.handle, None, dq, heads, up(rt, k),
         kv_heads, head, c.dev[0], KV4, seq, rt.step(0, seq), up(rt, table))
    np.testing.assert_array_equal(dq.download(q.shape), rotate(q))  # out of range: as it was
    c.same()


# ---- decode attention -------------------------------------------------------------------------------
def decode(rt, q, c, pos, split, new=None, entry=None, stream=None, out=None):
    heads = q.shape[0]
    nbytes = int(lib.ammon_attention_scratch_bytes(heads, c.head, c.seq, split))
    part = rt.alloc(nbytes)
    rt.fill(part, F32, nbytes // 4, float("nan"))
    rt.synchronize()
    out = out or rt.alloc(q.nbytes)
    args = [rt.handle, stream, up(rt, q), heads]
    if new:
        args += [up(rt, x) for x in new]
    args += [*c.dev, KV4, c.kv_heads, c.head, c.seq, rt.step(0, pos), split]
    entry = entry or ("ammon_attention_decode_append" if new else "ammon_attention_decode")
    args += [out] if entry.endswith("noalloc") else [part, nbytes, out]
    call(entry, *args)
    rt.synchronize(stream)
    return out.download(q.shape)


def off(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    return np.max(np.abs(got - want)[fine], initial=0) / max(np.max(np.abs(want)[fine], initial=0), 1e-30)


@pytest.mark.parametrize("pos", [0, 1, 30, 31, 32, 127, 128, 300, 599])
@pytest.mark.parametrize("heads,kv_heads,head", SHAPES)
def test_decode(rt, heads, kv_heads, head, pos):
    c = Cache(rt, kv_heads, 600, head, filled=pos + 1)
    q = oracle.normal(heads * head, 9).reshape(heads, head)
    want = kv4.attention(q[None], *c.numbers(pos + 1), pos)[0]
    for split in (600, 128, 64, 33, 1):
        got = decode(rt, q, c, pos, split)
        assert off(got, want) <= TOL, split
    assert off(decode(rt, q, c, pos, 200, entry="ammon_attention_decode_noalloc"), want) <= TOL
    c.same()


@pytest.mark.parametrize("heads,kv_heads,head,seq,pos", [(32, 8, 128, 8192, 8191), (64, 8, 128, 8192, 5000),
                                                         (8, 4, 64, 16384, 16000), (3, 1, 96, 20000, 19999)])
def test_decode_long(rt, heads, kv_heads, head, seq, pos):
    c = Cache(rt, kv_heads, seq, head, filled=pos + 1)
    q = oracle.normal(heads * head, 9).reshape(heads, head)
    want = kv4.attention(q[None], *c.numbers(pos + 1), pos)[0]
    default = int(lib.ammon_attention_default_split_for(rt.handle, heads, kv_heads, head, KV4, seq))
    for split in (default, 1024, 500):
        assert off(decode(rt, q, c, pos, split), want) <= TOL, split


@pytest.mark.parametrize("pos", [0, 31, 32, 100, 127, 128, 255, 383])
@pytest.mark.parametrize("heads,kv_heads,head", SHAPES)
def test_append_is_store_then_decode(rt, heads, kv_heads, head, pos):
    a, b = (Cache(rt, kv_heads, 384, head, filled=pos) for _ in "ab")
    q = oracle.normal(heads * head, 9).reshape(heads, head)
    k, v = rows_of(kv_heads, 1, head, 5), rows_of(kv_heads, 1, head, 50)
    for split in (384, 128, 40):
        got = decode(rt, q, a, pos, split, new=(k, v))
        store(rt, b, k, v, pos)
        want = decode(rt, q, b, pos, split)
        np.testing.assert_array_equal(got, want)
    for c in (a, b):
        c.pack(pos, k, v)
        c.same()
    assert off(got, kv4.attention(q[None], *a.numbers(pos + 1), pos)[0]) <= TOL


def test_append_over_an_older_row_and_past_it(rt):
    # the position is stepped back: its row is replaced, later rows stay and are not attended to
    c = Cache(rt, 2, 300, 128, filled=300)
    q = oracle.normal(8 * 128, 9).reshape(8, 128)
    k, v = rows_of(2, 1, 128, 5), rows_of(2, 1, 128, 50)
    got = decode(rt, q, c, 140, 128, new=(k, v))
    c.pack(140, k, v)
    c.same()
    assert off(got, kv4.attention(q[None], *c.numbers(141), 140)[0]) <= TOL


@pytest.mark.parametrize("split", [64, 16])  # one split (direct output) and several
def test_position_out_of_range(rt, split):
    c = Cache(rt, 2, 64, 48, filled=64)
    q = oracle.normal(4 * 48, 9).reshape(4, 48)
    k = rows_of(2, 1, 48, 5)
    for pos in (64, 0xffffffff):
        assert np.all(np.isnan(decode(rt, q, c, pos, split)))
        assert np.all(np.isnan(decode(rt, q, c, pos, split, new=(k, k))))
        c.same()


@pytest.mark.parametrize("head", [128, 80])
def test_numbers_that_are_not_finite(rt, head):
    kv_heads, pos, at = 2, 200, 77
    q = oracle.normal(4 * head, 9).reshape(4, head)
    for side in (0, 1):
        c = Cache(rt, kv_heads, 400, head, filled=pos + 1)
        row = c.numbers(1, at)[side].astype(np.float32).transpose(1, 0, 2)
        row[0, 0, 40] = np.inf  # group 1 of kv head 0
        kv4.pack(c.host[side], kv_heads, 400, head, at, row.transpose(1, 0, 2))
        c.dev[side].upload(c.host[side])
        want = kv4.attention(q[None], *c.numbers(pos + 1), pos)[0]
        assert np.isnan(want[:2]).any() and not np.isnan(want[2:]).any()
        assert np.isnan(want[:2]).all() == (side == 0)  # a value's NaN stays in its group
        for split in (400, 128, 7):
            assert off(decode(rt, q, c, pos, split), want) <= TOL
        # ... and a position before it does not see it
        want = kv4.attention(q[None], *c.numbers(at), at - 1)[0]
        assert off(decode(rt, q, c, at - 1, 128), want) <= TOL


def test_q_of_any_size(rt):
    c = Cache(rt, 2, 256, 128, filled=256)
    q = oracle.normal(8 * 128, 9).reshape(8, 128)
    # 2^-20, 2^-130 (subnormal products) and a q of one large and many small numbers
    for scale in (2.0**-20, 2.0**-130):
        small = (q * np.float32(scale)).astype(np.float32)
        want = kv4.attention(small[None], *c.numbers(256), 255)[0]
        assert off(decode(rt, small, c, 255, 128), want) <= TOL
    mixed = q.copy()
    mixed[:, 5] = 300.0
    # scores are 300 / sqrt(128) |k| large: their fp32 rounding is 2^-24 of that, times ~6 roundings
    want = kv4.attention(mixed[None], *c.numbers(256), 255)[0]
    assert off(decode(rt, mixed, c, 255, 128), want) <= TOL + 6 * 2.0**-24 * 300 / np.sqrt(128) * 6
    assert np.all(decode(rt, np.zeros_like(q), c, 255, 128) != 0)
    bad = q.copy()
    bad[3, 7], bad[4, 0] = np.nan, np.inf
    got = decode(rt, bad, c, 255, 128)
    assert np.isnan(got[3:5]).all() and not np.isnan(got[[0, 1, 2, 5, 6, 7]]).any()


def test_decode_steps_in_a_graph(rt):
    """Append, merge and a replayed graph: the position is the only thing that changes."""
    heads, kv_heads, head, seq, split = 8, 2, 64, 320, 64
    c = Cache(rt, kv_heads, seq, head)
    stream = ctypes.c_void_p()
    call("ammon_stream_create", rt.handle, ctypes.byref(stream))
    q, k, v = (rt.alloc(n * head * 4) for n in (heads, kv_heads, kv_heads))
    nbytes = int(lib.ammon_attention_scratch_bytes(heads, head, seq, split))
    part, out, step = rt.alloc(nbytes), rt.alloc(heads * head * 4), rt.step(0, 0)
    rows = [rows_of(kv_heads, 200, head, s) for s in (5, 50)]
    qs = oracle.normal(200 * heads * head, 9).reshape(200, heads, head)
    rt.synchronize()
    call("ammon_capture_begin", rt.handle, stream)
    call("ammon_attention_decode_append", rt.handle, stream, q, heads, k, v, *c.dev, KV4, kv_heads,
         head, seq, step, split, part, nbytes, out)
    graph = ctypes.c_void_p()
    call("ammon_capture_end", rt.handle, stream, ctypes.byref(graph))
    for pos in range(0, 200):
        for buf, x in ((q, qs[pos]), (k, rows[0][pos]), (v, rows[1][pos])):
            buf.upload(x, stream)
        rt.deposit(step, 0, pos, stream)
        call("ammon_graph_launch", rt.handle, graph, stream)
        got = out.download((heads, head), stream=stream)
        c.pack(pos, rows[0][pos:pos + 1], rows[1][pos:pos + 1])
        if pos % 13 == 0 or pos > 190:
            want = kv4.attention(qs[pos:pos + 1], *c.numbers(pos + 1), pos)[0]
            assert off(got, want) <= TOL, pos
            eager = decode(rt, qs[pos], c, pos, split)
            np.testing.assert_array_equal(got, eager)
    c.same()
    call("ammon_graph_destroy", rt.handle, graph)
    call("ammon_stream_destroy", rt.handle, stream)


def prefill(rt, q, c, start, split, ctx=None, pad=64):
    tokens, heads = q.shape[:2]
    ctx = ctx or start + tokens
    nbytes = int(lib.ammon_attention_prefill_scratch_bytes(tokens, heads, c.head, ctx, split))
    part, out = rt.alloc(nbytes + pad * 4), rt.alloc(q.nbytes + pad * 4)
    for buf, n in ((part, nbytes // 4), (out, q.size)):
        rt.fill(buf, F32, n + pad, 7.0)
    call("ammon_attention_prefill", rt.handle, None, up(rt, q), tokens, heads, *c.dev, KV4,
         c.kv_heads, c.head, c.seq, rt.step(0, start), ctx, split, part, nbytes, out)
    got = out.download(q.size + pad)
    assert np.all(got[q.size:] == 7.0) and np.all(part.download(nbytes // 4 + pad)[nbytes // 4:] == 7.0)
    return got[:q.size].reshape(q.shape)


@pytest.mark.parametrize("heads,kv_heads,head", SHAPES)
@pytest.mark.parametrize("start,tokens", [(0, 1), (0, 5), (0, 70), (61, 40), (300, 3)])
def test_prefill(rt, heads, kv_heads, head, start, tokens):
    c = Cache(rt, kv_heads, 400, head, filled=start + tokens)
    q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
    want = kv4.attention(q, *c.numbers(start + tokens), start)
    for split in (16, 512):
        assert off(prefill(rt, q, c, start, split), want) <= TOL


# long enough for the tiles: one and several splits, rows that end inside a tile, a wave and a
# chunk, every number of groups, heads that are no multiple of 4
LONG = [(32, 8, 128, 0, 300), (32, 8, 128, 1500, 131), (8, 8, 128, 63, 1000), (16, 2, 128, 2500, 77),
        (8, 4, 64, 129, 700), (18, 6, 96, 1000, 200), (6, 6, 48, 1, 999), (5, 5, 32, 2000, 250),
        (12, 6, 100, 500, 333), (9, 3, 127, 700, 301), (12, 12, 30, 400, 500), (24, 3, 80, 64, 640)]


@pytest.mark.parametrize("heads,kv_heads,head,start,tokens", LONG)
def test_prefill_long(rt, heads, kv_heads, head, start, tokens):
    c = Cache(rt, kv_heads, 3000, head, filled=start + tokens)
    q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
    want = kv4.attention(q, *c.numbers(start + tokens), start)
    for split in (1024, 256, 64):
        assert off(prefill(rt, q, c, start, split), want) <= TOL, split


@pytest.mark.parametrize("head", [128, 80])
def test_prefill_numbers_that_are_not_finite(rt, head):
    """A later token's NaN does not reach an earlier one; a value's stays in its group."""
    heads, kv_heads, start, tokens = 8, 4, 700, 400
    for side in (0, 1):
        c = Cache(rt, kv_heads, 2000, head, filled=start + tokens)
        for at, g, d, bad in ((900, 0, 40, np.inf), (start + tokens - 1, 1, head - 1, np.nan), (5, 2, 0, -np.inf)):
            row = c.numbers(1, at)[side].astype(np.float32)
            row[g, 0, d] = bad
            kv4.pack(c.host[side], kv_heads, 2000, head, at, row)
        c.dev[side].upload(c.host[side])
        q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
        want = kv4.attention(q, *c.numbers(start + tokens), start)
        assert np.isnan(want[200:, 0]).any() and not np.isnan(want[:200, :2]).any()
        assert not np.isnan(want[:, 6:]).any() and np.isnan(want[:, 4:6]).any()
        for split in (1024, 64):
            assert off(prefill(rt, q, c, start, split), want) <= TOL


@pytest.mark.parametrize("tokens", [20, 700])
def test_prefill_positions_out_of_range(rt, tokens):
    # the last tokens are past ctx: NaN, and the others as they are
    c = Cache(rt, 4, 1000, 64, filled=1000)
    q = oracle.normal(tokens * 8 * 64, 9).reshape(tokens, 8, 64)
    start, ctx = 250, 250 + tokens - 7
    want = kv4.attention(q[:-7], *c.numbers(ctx), start)
    for split in (1024, 100):
        got = prefill(rt, q, c, start, split, ctx=ctx)
        assert off(got[:-7], want) <= TOL and np.all(np.isnan(got[-7:]))
    got = prefill(rt, q, c, 5000, 1024, ctx=ctx)
    assert np.all(np.isnan(got))


def test_prefill_in_a_graph(rt):
    c = Cache(rt, 8, 1500, 128, filled=1500)
    tokens, heads = 301, 32
    q = oracle.normal(tokens * heads * 128, 9).reshape(tokens, heads, 128)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    call("ammon_stream_create", rt.handle, ctypes.byref(stream))
    nbytes = int(lib.ammon_attention_prefill_scratch_bytes(tokens, heads, 128, 1500, 256))
    dq, part, out, step = up(rt, q), rt.alloc(nbytes), rt.alloc(q.nbytes), rt.step(0, 0)
    rt.synchronize()
    call("ammon_capture_begin", rt.handle, stream)
    call("ammon_attention_prefill", rt.handle, stream, dq, tokens, heads, *c.dev, KV4, 8, 128, 1500,
         step, 1500, 256, part, nbytes, out)
    call("ammon_capture_end", rt.handle, stream, ctypes.byref(graph))
    for start in (0, 700, 1199, 3):
        rt.deposit(step, 0, start, stream)
        call("ammon_graph_launch", rt.handle, graph, stream)
        got = out.download(q.shape, stream=stream)
        assert off(got, kv4.attention(q, *c.numbers(start + tokens), start)) <= TOL
        np.testing.assert_array_equal(got, prefill(rt, q, c, start, 256, ctx=1500))
    call("ammon_graph_destroy", rt.handle, graph)
    call("ammon_stream_destroy", rt.handle, stream)


# ---- a few tokens at a time: units of eight query rows of several tokens ------------------------
SETS = [(6, 6, 48), (12, 4, 80), (8, 8, 128), (10, 2, 64), (32, 8, 128), (14, 2, 96), (16, 2, 33)]


@pytest.mark.parametrize("heads,kv_heads,head", SETS)
@pytest.mark.parametrize("start,tokens", [(0, 2), (0, 17), (63, 3), (250, 13), (509, 9), (780, 19)])
def test_prefill_few_tokens(rt, heads, kv_heads, head, start, tokens):
    c = Cache(rt, kv_heads, 900, head, filled=start + tokens)
    q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
    want = kv4.attention(q, *c.numbers(start + tokens), start)
    for split in (256, 300, 1024):
        assert off(prefill(rt, q, c, start, split), want) <= TOL


@pytest.mark.parametrize("heads,kv_heads,head", SETS)
@pytest.mark.parametrize("start,at", [(0, 5), (60, 63), (60, 64), (250, 255), (250, 256), (250, 250)])
def test_prefill_few_tokens_not_finite(rt, heads, kv_heads, head, start, at):
    """A row that is not finite among the prompt's own: no token before it is touched."""
    tokens = 12
    for side in (0, 1):
        c = Cache(rt, kv_heads, 700, head, filled=start + tokens)
        for p, g, d in ((at, kv_heads - 1, head - 1), (start + tokens - 1, 0, 0)):
            row = c.numbers(1, p)[side].astype(np.float32)
            row[g, 0, d] = np.nan
            kv4.pack(c.host[side], kv_heads, 700, head, p, row)
        c.dev[side].upload(c.host[side])
        q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
        want = kv4.attention(q, *c.numbers(start + tokens), start)
        nan = np.isnan(want).any(-1)
        assert nan[at - start:, -1].all() and nan[-1, 0] and not nan[:at - start].any()
        for split in (128, 1024):
            assert off(prefill(rt, q, c, start, split), want) <= TOL


@pytest.mark.parametrize("heads,kv_heads,head", [(6, 6, 48), (12, 4, 80)])
@pytest.mark.parametrize("split", [64, 1024])
def test_prefill_few_tokens_out_of_range(rt, heads, kv_heads, head, split):
    """Tokens past ctx, and past the last position there is, give NaN; the others their rows."""
    c = Cache(rt, kv_heads, 300, head, filled=300)
    q = oracle.normal(10 * heads * head, 9).reshape(10, heads, head)
    got = prefill(rt, q, c, 297, split, ctx=300)
    assert off(got[:3], kv4.attention(q[:3], *c.numbers(300), 297)) <= TOL
    assert np.isnan(got[3:]).all()
    for start in (300, 2**32 - 4):
        assert np.isnan(prefill(rt, q, c, start, split, ctx=300)).all()


def test_prefill_past_the_last_position_there_is(rt):
    c = Cache(rt, 4, 1000, 64, filled=1000)
    q = oracle.normal(700 * 8 * 64, 9).reshape(700, 8, 64)
    for start in (2**32 - 1, 2**32 - 256, 2**32 - 700):
        for split in (1024, 100):
            assert np.isnan(prefill(rt, q, c, start, split, ctx=900)).all()


@pytest.mark.parametrize("heads,kv_heads,head", [(32, 8, 128), (8, 4, 64), (6, 2, 33)])
def test_rows_at_any_float(rt, heads, kv_heads, head):
    """q, the rows and the output a float past 16 bytes."""
    seq, tokens = 300, 5
    q = oracle.normal(tokens * heads * head, 9).reshape(tokens, heads, head)
    rows = [oracle.normal(tokens * kv_heads * head, s).reshape(tokens, kv_heads, head) for s in (1, 2)]
    kept = [up(rt, np.concatenate([np.zeros(1, np.float32), a.ravel()])) for a in (q, *rows)]
    dq, dk, dv = (b.offset(4) for b in kept)
    step = rt.step(0, 0)
    nbytes = int(lib.ammon_kv_cache_bytes(KV4, kv_heads, seq, head))
    caches = [up(rt, np.zeros(nbytes, np.uint8)) for _ in "kv"]
    call("ammon_kv4_store", rt.handle, None, dk, dv, tokens, kv_heads, head, *caches, seq, step)
    k, v = (kv4.stored(r).transpose(1, 0, 2) for r in rows)
    n = int(lib.ammon_attention_prefill_scratch_bytes(tokens, heads, head, tokens, 256))
    part, out = rt.alloc(n + 4), rt.alloc(q.nbytes + 4)
    call("ammon_attention_prefill", rt.handle, None, dq, tokens, heads, *caches, KV4, kv_heads, head,
         seq, step, tokens, 256, part.offset(4), n, out.offset(4))
    got = out.download(q.size + 1)[1:].reshape(q.shape)
    assert off(got, kv4.attention(q, k, v, 0)) <= TOL
    # the first token again at the next position, with its rows
    n = int(lib.ammon_attention_scratch_bytes(heads, head, seq, 100))
    part = rt.alloc(n + 4)
    call("ammon_attention_decode_append", rt.handle, None, dq, heads, dk, dv, *caches, KV4, kv_heads,
         head, seq, rt.step(0, tokens), 100, part.offset(4), n, out.offset(4))
    got = out.download(heads * head + 1)[1:].reshape(1, heads, head)
    k, v = (np.concatenate([x, x[:, :1]], 1) for x in (k, v))
    assert off(got, kv4.attention(q[:1], k, v, tokens)) <= TOL


def test_two_graphs_and_a_stream_share_a_cache(rt):
    """Decode graphs of two streams with scratch of their own, replayed in turn and at once."""
    heads, kv_heads, head, seq = 32, 8, 128, 2000
    c = Cache(rt, kv_heads, seq, head, filled=seq)
    n = int(lib.ammon_attention_scratch_bytes(heads, head, seq, 256))
    runs = []
    for seed in (1, 2):
        stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
        call("ammon_stream_create", rt.handle, ctypes.byref(stream))
        q = oracle.normal(heads * head, seed).reshape(1, heads, head)
        dq, part, out, step = up(rt, q), rt.alloc(n), rt.alloc(q.nbytes), rt.step(0, 0)
        rt.synchronize()
        call("ammon_capture_begin", rt.handle, stream)
        call("ammon_attention_decode", rt.handle, stream, dq, heads, *c.dev, KV4, kv_heads, head, seq,
             step, 256, part, n, out)
        call("ammon_capture_end", rt.handle, stream, ctypes.byref(graph))
        runs.append((stream, graph, q, step, out, (dq, part)))
    for at in ((0, 1999), (700, 3), (255, 256)):
        for (stream, graph, q, step, out, _), pos in zip(runs, at):
            rt.deposit(step, 0, pos, stream)
        for _ in range(3):
            for stream, graph, *_ in runs:
                call("ammon_graph_launch", rt.handle, graph, stream)
        for (stream, graph, q, step, out, _), pos in zip(runs, at):
            got = out.download(q.shape, stream=stream)
            assert off(got, kv4.attention(q, *c.numbers(pos + 1), pos)) <= TOL
    for stream, graph, *_ in runs:
        call("ammon_graph_destroy", rt.handle, graph)
        call("ammon_stream_destroy", rt.handle, stream)


# ---- borders of a wave's 64 positions, of a chunk's 256, of the ring's two chunks ----------------
@pytest.mark.parametrize("pos", [63, 64, 191, 192, 255, 256, 511, 512, 767, 768, 1030])
@pytest.mark.parametrize("heads,kv_heads,head", [(16, 2, 128), (6, 2, 96), (7, 7, 64), (2, 1, 20)])
def test_decode_and_append_at_borders(rt, heads, kv_heads, head, pos):
    a, b = (Cache(rt, kv_heads, 1100, head, filled=pos) for _ in "ab")
    q = oracle.normal(heads * head, 9).reshape(heads, head)
    k, v = rows_of(kv_heads, 1, head, 5), rows_of(kv_heads, 1, head, 50)
    store(rt, b, k, v, pos)
    b.pack(pos, k, v)
    want = kv4.attention(q[None], *b.numbers(pos + 1), pos)[0]
    for split in (1024, 768, 300, 256):
        got = decode(rt, q, a, pos, split, new=(k, v))
        np.testing.assert_array_equal(got, decode(rt, q, b, pos, split))
        assert off(got, want) <= TOL, split
    b.same()
    a.pack(pos, k, v)
    a.same()


def test_caches_past_32_bits(rt):
    """5 GB each: rows of the last heads at the last positions stored, read back, attended to."""
    heads = kv_heads = 64
    head, seq, tokens = 128, (1 << 20) - 3, 5
    nbytes = int(lib.ammon_kv_cache_bytes(KV4, kv_heads, seq, head))
    assert nbytes > 1 << 32
    caches = [rt.alloc(nbytes) for _ in "kv"]
    for c in caches:
        rt.fill(c, F32, nbytes // 4, 0.0)  # zeros
    k, v = rows_of(kv_heads, tokens, head, 5), rows_of(kv_heads, tokens, head, 50)
    v += np.arange(head, dtype=np.float32) % 2 * 8192  # (so that they show beside a million zeros)
    dk, dv = up(rt, k), up(rt, v)
    call("ammon_kv4_store", rt.handle, None, dk, dv, tokens, kv_heads, head, *caches, seq,
         rt.step(0, seq - tokens))
    bufs = [rt.alloc(kv_heads * (tokens + 2) * head * 4) for _ in "kv"]
    call("ammon_kv4_load", rt.handle, None, *caches, kv_heads, head, seq, seq - tokens - 2, tokens + 2,
         *bufs, F32)
    got = [b.download((kv_heads, tokens + 2, head)) for b in bufs]
    want = [kv4.stored(x).transpose(1, 0, 2) for x in (k, v)]
    for g, w in zip(got, want):
        assert not g[:, :2].any()
        np.testing.assert_array_equal(g[:, 2:], w)
    # softmax of seq - tokens zeros and the stored rows' scores
    q = oracle.normal(heads * head, 9).reshape(heads, head).astype(np.float64)
    s = np.einsum("hd,htd->ht", q, want[0]) / np.sqrt(head)
    e = np.exp(s)
    out64 = np.einsum("ht,htd->hd", e, want[1]) / (seq - tokens + e.sum(1))[:, None]
    n = int(lib.ammon_attention_scratch_bytes(heads, head, seq, 1024))
    part, out = rt.alloc(n), rt.alloc(heads * head * 4)
    call("ammon_attention_decode", rt.handle, None, up(rt, q.astype(np.float32)), heads, *caches, KV4,
         kv_heads, head, seq, rt.step(0, seq - 1), 1024, part, n, out)
    assert off(out.download((heads, head)), out64) <= TOL
    # the same through the append of the last row, over what stands there
    call("ammon_attention_decode_append", rt.handle, None, up(rt, q.astype(np.float32)), heads,
         dk.offset(4 * (tokens - 1) * kv_heads * head), dv.offset(4 * (tokens - 1) * kv_heads * head),
         *caches, KV4, kv_heads, head, seq, rt.step(0, seq - 1), 1024, part, n, out)
    assert off(out.download((heads, head)), out64) <= TOL
