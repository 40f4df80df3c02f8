"""4-bit weights (AMMON_W4) and rows of 8-bit digits (AMMON_Q8, AMMON_Q24) on the GPU against the
numpy restatement (oracle/w4.py).

Stored bytes are compared bit for bit: the definitions fix every rounding.  Products are compared
with float64 over the stored numbers, each result with a bar of its own (oracle.w4.product_bar:
the digits' half steps and the roundings of the fp32 sums, as if they all went one way).
"""
import ctypes

import numpy as np
import pytest

import oracle
from ammon_amd import _abi
from ammon_amd._abi import BF16, F32, KV4, Q8, Q24, W4, AmmonError, call, lib
from oracle import w4

pytestmark = pytest.mark.gpu
DIGITS = {Q8: 1, Q24: 3}
EPS = 1e-5
NORM = 40 * 2.0**-24  # of an fp32 norm: its sum's roundings (halved by the root) and three products


def up(rt, a):
    return rt.upload(np.ascontiguousarray(a))


def matrix(d, n, seed=1):
    """Weights, and a few groups of their own size."""
    w = oracle.normal(d * n, seed).reshape(d, n) * np.float32(0.05)
    w[d // 2, n // 2:] *= 300
    w[d // 3] *= np.float32(1e-3)
    return w


def stream(t, n, seed=2):
    """Rows of a residual stream: channels of their own size, one far larger."""
    size = np.exp(0.5 * oracle.normal(n, seed + 1))
    size[n // 3] *= 30
    return (oracle.normal(t * n, seed).reshape(t, n) * size).astype(np.float32)


class Weights:
    """A matrix as W4: on the device (packed by the restatement) and its numbers."""

    def __init__(self, rt, d, n, seed=1, w=None):
        codes, s = w4.w4_quantise(matrix(d, n, seed) if w is None else w)
        self.numbers = w4.w4_numbers(codes, s, n)
        self.bytes = w4.w4_pack(codes, s)
        self.dev = up(rt, self.bytes)


class Rows:
    def __init__(self, rt, x, dtype):
        t, n = x.shape
        q, s = w4.q_quantise(x, DIGITS[dtype])
        self.numbers = w4.q_numbers(q, s, n)
        # tokens past the last one hold anything
        junk = np.full(w4.q8_bytes(DIGITS[dtype], t, n), 0xff, np.uint8)
        self.bytes = w4.q_pack(q, s, DIGITS[dtype], into=junk)
        self.dev = up(rt, self.bytes)


def close(got, want, bar):
    got, want = np.asarray(got, np.float64), np.asarray(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    worst = np.nanmax(np.abs(got - want) / (bar + 1e-37), initial=0)
    assert worst <= 1, worst


# ---- matrices stored and read back ---------------------------------------------------------------
SHAPES = [(1, 1), (16, 128), (17, 129), (5, 300), (288, 288), (50, 96), (33, 1024), (100, 77)]


@pytest.mark.parametrize("d,n", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_w4_store_is_the_definition(rt, d, n, dtype):
    w = oracle.storage(matrix(d, n), dtype)
    want = w4.w4_pack(*w4.w4_quantise(oracle.widen(w, dtype).reshape(d, n)))
    assert lib.ammon_w4_bytes(d, n) == want.size
    out = rt.alloc(want.size + 64)
    rt.fill(out, F32, want.size // 4 + 16, 7.0)
    call("ammon_w4_store", rt.handle, None, up(rt, w), dtype, d, n, out)
    got = out.download(want.size + 64, np.uint8)
    np.testing.assert_array_equal(got[:want.size], want)
    assert set(got[want.size:].view(np.float32)) == {7.0}


def test_w4_store_at_any_float(rt):
    d, n = 20, 256
    w = matrix(d, n)
    buf = up(rt, np.concatenate([[0], w.reshape(-1)]).astype(np.float32))
    want = w4.w4_pack(*w4.w4_quantise(w))
    out = rt.alloc(want.size)
    call("ammon_w4_store", rt.handle, None, buf.offset(4), F32, d, n, out)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)


def test_w4_store_special_values(rt):
    w = matrix(24, 256)
    w[0] = 0
    w[1] = -0.0
    w[2, 5], w[3, 200], w[4, 0] = np.nan, np.inf, -np.inf
    w[5] = 1e-40
    w[6] *= np.float32(1e-35)
    w[7] = 3e38
    w[8] = np.where(np.arange(256) % 2, 7.0, 0.5)  # codes at a border: half a step
    w[9] = 2.0**-126
    want = w4.w4_pack(*w4.w4_quantise(w))
    out = rt.alloc(want.size)
    call("ammon_w4_store", rt.handle, None, up(rt, w), F32, 24, 256, out)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)
    back = rt.alloc(24 * 256 * 4)
    call("ammon_w4_load", rt.handle, None, out, 24, 256, back, F32)
    codes, s = w4.w4_quantise(w)
    np.testing.assert_array_equal(back.download((24, 256)), w4.w4_numbers(codes, s, 256).astype(np.float32))


@pytest.mark.parametrize("d,n", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_w4_load(rt, d, n, dtype):
    w = Weights(rt, d, n)
    es = 2 if dtype == BF16 else 4
    out = rt.alloc(d * n * 4 + 64)
    rt.fill(out, F32, d * n + 16, 7.0)
    call("ammon_w4_load", rt.handle, None, w.dev, d, n, out, dtype)
    got = out.download(d * n * 4 + 64, np.uint8)
    want = oracle.storage(w.numbers.astype(np.float32), dtype)
    np.testing.assert_array_equal(got[:d * n * es], want.reshape(-1).view(np.uint8))
    assert set(got[(d * n * es + 3) // 4 * 4:].view(np.float32)) == {7.0}


def test_codes_of_minus_eight(rt):
    # (store never writes them, other writers may)
    codes = np.full((16, 1, 128), -8, np.int8)
    codes[:, :, ::3] = 7
    s = np.full((16, 1), 0.5)
    dev = up(rt, w4.w4_pack(codes, s))
    out = rt.alloc(16 * 128 * 4)
    call("ammon_w4_load", rt.handle, None, dev, 16, 128, out, F32)
    np.testing.assert_array_equal(out.download((16, 128)), codes[:, 0] * 0.5)
    x = stream(1, 128)[0]
    y = rt.alloc(64)
    call("ammon_gemv", rt.handle, None, dev, W4, 16, 128, up(rt, x), y, None)
    want = x[None].astype(np.float64) @ (codes[:, 0] * 0.5).T
    close(y.download((1, 16)), want, w4.product_bar(x[None], codes[:, 0] * 0.5, False))


# ---- rows of digits --------------------------------------------------------------------------------
ROWS = [(1, 128), (1, 4096), (16, 256), (17, 300), (5, 1), (3, 2080), (40, 96), (2, 9000), (130, 77)]


@pytest.mark.parametrize("t,n", ROWS)
@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_q8_store_is_the_definition(rt, t, n, dtype):
    x = stream(t, n)
    size = w4.q8_bytes(DIGITS[dtype], t, n)
    before = np.full(size + 64, 0x5a, np.uint8)
    want = before.copy()
    want[:size] = w4.q_pack(*w4.q_quantise(x, DIGITS[dtype]), DIGITS[dtype], into=before[:size])
    out = up(rt, before)
    call("ammon_q8_store", rt.handle, None, up(rt, x), t, n, out, dtype)
    np.testing.assert_array_equal(out.download(size + 64, np.uint8), want)


@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_q8_special_values(rt, dtype):
    x = stream(12, 256)
    x[0] = 0
    x[1, 3], x[2, 200], x[3, 0] = np.nan, np.inf, -np.inf
    x[4] = 1e-40
    x[5] *= np.float32(1e-33)
    x[6] = 3.4e38
    x[7] = np.float32(127 * 65536)
    x[8] = np.nextafter(np.float32(127 * 65536), np.float32(0))
    x[9] = np.arange(256) % 32 * 0.5 + 0.25  # numbers at a border
    x[10] = 2.0**-98
    digits = DIGITS[dtype]
    q, s = w4.q_quantise(x, digits)
    want = w4.q_pack(q, s, digits, into=np.full(w4.q8_bytes(digits, 12, 256), 9, np.uint8))
    out = up(rt, np.full(want.size, 9, np.uint8))
    call("ammon_q8_store", rt.handle, None, up(rt, x), 12, 256, out, dtype)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)
    back = rt.alloc(x.nbytes)
    call("ammon_q8_load", rt.handle, None, out, dtype, 12, 256, back)
    np.testing.assert_array_equal(back.download(x.shape), w4.q_numbers(q, s, 256).astype(np.float32))


@pytest.mark.parametrize("t,n", ROWS)
@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_q8_load(rt, t, n, dtype):
    r = Rows(rt, stream(t, n), dtype)
    out = rt.alloc(t * n * 4 + 64)
    rt.fill(out, F32, t * n + 16, 7.0)
    call("ammon_q8_load", rt.handle, None, r.dev, dtype, t, n, out)
    got = out.download(t * n + 16)
    np.testing.assert_array_equal(got[:t * n].reshape(t, n), r.numbers.astype(np.float32))
    assert set(got[t * n:]) == {7.0}


def rmsnorm_q8(rt, x, r, w, wdt, dtype, out, into):
    t, n = x.shape
    dx, dr = up(rt, x), up(rt, r) if r is not None else None
    ds = {"new": rt.alloc(x.nbytes), "x": dx, "residual": dr}[into] if r is not None else None
    call("ammon_rmsnorm_q8", rt.handle, None, dx, dr, ds, up(rt, w), wdt, EPS, t, n, out, dtype)
    return ds.download(x.shape) if r is not None else None


@pytest.mark.parametrize("t,n", ROWS)
@pytest.mark.parametrize("dtype", [Q8, Q24])
@pytest.mark.parametrize("wdt,into", [(F32, "new"), (BF16, "x"), (F32, "residual"), (BF16, None)])
def test_rmsnorm_q8_is_the_definition(rt, t, n, dtype, wdt, into):
    x, r = stream(t, n), stream(t, n, 7) if into else None
    w = oracle.storage(1 + 0.2 * oracle.normal(n, 5), wdt)
    h = x + r if into else x
    v = w4.normed(h, oracle.widen(w, wdt), EPS)
    digits = DIGITS[dtype]
    before = np.full(w4.q8_bytes(digits, t, n), 0x5a, np.uint8)
    want = w4.q_pack(*w4.q_quantise(v, digits), digits, into=before)
    out = up(rt, before)
    got_h = rmsnorm_q8(rt, x, r, w, wdt, dtype, out, into)
    if into:
        np.testing.assert_array_equal(got_h, h)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)


def test_rmsnorm_q8_rows_that_are_not_finite(rt):
    x = stream(4, 300)
    x[1, 7], x[2, 100] = np.nan, np.inf
    x[3] = 0
    out = rt.alloc(w4.q8_bytes(3, 4, 300))
    rmsnorm_q8(rt, x, np.zeros_like(x), np.ones(300, np.float32), F32, Q24, out, "new")
    back = rt.alloc(x.nbytes)
    call("ammon_q8_load", rt.handle, None, out, Q24, 4, 300, back)
    got = back.download(x.shape)
    assert np.isfinite(got[0]).all() and not got[3].any()
    assert np.isnan(got[1]).all()  # the mean is NaN
    # inf: the others are 0 x w, itself inf x 0; its block of 128 is NaN
    assert np.isnan(got[2, :128]).all() and not got[2, 128:].any()


# ---- one token -----------------------------------------------------------------------------------
GEMV = [(1, 1), (16, 128), (17, 129), (288, 288), (70, 1000), (96, 4096), (33, 14336), (4128, 512),
        (20, 36864), (9000, 8192),
        # many groups a CU, of units that waves share: one unit and two, two groups a unit, no whole
        # pieces of x, more of x than a workgroup keeps
        (4100, 8300), (131072, 200), (4800, 9001), (4096, 20000)]


@pytest.mark.parametrize("d,n", GEMV)
@pytest.mark.parametrize("residual", [None, "y", "other"])
def test_gemv(rt, d, n, residual):
    w, x, r = Weights(rt, d, n), stream(1, n), oracle.normal(d, 9).reshape(1, d)
    want = x.astype(np.float64) @ w.numbers.T
    bar = w4.product_bar(x, w.numbers, False)
    y = rt.alloc(d * 4 + 64)
    rt.fill(y, F32, d + 16, 7.0)
    rt.synchronize()
    if residual == "y":
        y.upload(r)
    other = {"y": y, "other": up(rt, r), None: None}[residual]
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, x), y, other)
    got = y.download(d + 16)
    if residual:
        want, bar = want + r, bar + 2.0**-24 * (np.abs(want) + np.abs(r))
    close(got[None, :d], want, bar)
    assert set(got[d:]) == {7.0}


def test_gemv_x_at_any_float(rt):
    d, n = 40, 512
    w, x = Weights(rt, d, n), stream(1, n)
    buf = up(rt, np.concatenate([[0], x[0]]).astype(np.float32))
    y, z = rt.alloc(d * 4), rt.alloc(d * 4)
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, buf.offset(4), y, None)
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, x), z, None)
    np.testing.assert_array_equal(y.download(d), z.download(d))


def norm_of(x, w, wdt):
    h = x.astype(np.float64)
    return np.asarray(oracle.widen(w, wdt), np.float64) * h / np.sqrt((h * h).mean(-1, keepdims=True) + EPS)


@pytest.mark.parametrize("d,n", [(1, 1), (288, 288), (70, 1000), (200, 4096), (17, 9000), (8400, 256),
                                 (4100, 8300), (4800, 9001), (4096, 20000)])
@pytest.mark.parametrize("wdt", [F32, BF16])
def test_gemv_rmsnorm(rt, d, n, wdt):
    w, x = Weights(rt, d, n), stream(1, n)
    nw = oracle.storage(1 + 0.2 * oracle.normal(n, 5), wdt)
    xn = norm_of(x, nw, wdt)
    y = rt.alloc(d * 4)
    call("ammon_gemv_rmsnorm", rt.handle, None, up(rt, x), up(rt, nw), wdt, EPS, w.dev, W4, d, n, y)
    bar = w4.product_bar(xn, w.numbers, False) + NORM * np.abs(xn) @ np.abs(w.numbers).T
    close(y.download((1, d)), xn @ w.numbers.T, bar)


def swiglu_of(g, u, gbar, ubar):
    """silu(g) u and its bar: |silu'| <= 1.1, and a few roundings."""
    s = g / (1 + np.exp(-g))
    want = s * u
    return want, 1.1 * gbar * (np.abs(u) + ubar) + np.abs(s) * ubar + 6 * 2.0**-23 * np.abs(want)


@pytest.mark.parametrize("hidden,dim", [(1, 1), (8, 128), (40, 300), (768, 288), (24, 8192), (4200, 256),
                                        (2060, 8300), (7001, 1500)])
def test_gate_up_swiglu(rt, hidden, dim):
    a, b, x = Weights(rt, hidden, dim, 1), Weights(rt, hidden, dim, 11), stream(1, dim)
    nw = (1 + 0.2 * oracle.normal(dim, 5)).astype(np.float32)
    for norm in (False, True):
        xn = norm_of(x, nw, F32) if norm else x.astype(np.float64)
        hb = rt.alloc(hidden * 4 + 64)
        rt.fill(hb, F32, hidden + 16, 7.0)
        call("ammon_gate_up_swiglu", rt.handle, None, up(rt, x), up(rt, nw) if norm else None, F32, EPS,
             a.dev, b.dev, W4, dim, hidden, hb)
        bars = [w4.product_bar(xn, m.numbers, False) + norm * NORM * np.abs(xn) @ np.abs(m.numbers).T
                for m in (a, b)]
        got = hb.download(hidden + 16)
        close(got[None, :hidden], *swiglu_of(xn @ a.numbers.T, xn @ b.numbers.T, *bars))
        assert set(got[hidden:]) == {7.0}


def rotated(x, table, head):
    """Rows [t, heads * head] turned by table [t, head / 2, 2], and what 1 becomes of each bar."""
    p = x.reshape(x.shape[0], -1, head // 2, 2)
    c, s = table[:, None, :, 0].astype(np.float64), table[:, None, :, 1].astype(np.float64)
    return np.stack([p[..., 0] * c - p[..., 1] * s, p[..., 0] * s + p[..., 1] * c], -1).reshape(x.shape)


def turned_bar(bar, x, table, head):
    p, q = (t.reshape(x.shape[0], -1, head // 2, 2) for t in (bar, np.abs(x)))
    c, s = (np.abs(table[:, None, :, i]).astype(np.float64) for i in (0, 1))
    both = lambda t: np.stack([t[..., 0] * c + t[..., 1] * s, t[..., 0] * s + t[..., 1] * c], -1)  # noqa: E731
    return (both(p) + 3 * 2.0**-24 * both(p + q)).reshape(x.shape)


HEADS = [(32, 8, 128), (6, 6, 48), (4, 1, 80), (14, 2, 64), (8, 8, 2), (2, 1, 16)]


def qkv_weights(rt, heads, kv_heads, head, n):
    return [Weights(rt, h * head, n, s) for h, s in ((heads, 1), (kv_heads, 11), (kv_heads, 21))]


def qkv_of(xn, ws, table, head, extra):
    out = []
    for i, m in enumerate(ws):
        y, bar = xn @ m.numbers.T, w4.product_bar(xn, m.numbers, extra is None) + \
            (extra or 0) * np.abs(xn) @ np.abs(m.numbers).T
        out.append((rotated(y, table, head), turned_bar(bar, y, table, head)) if i < 2 else (y, bar))
    return out


@pytest.mark.parametrize("heads,kv_heads,head", HEADS)
def test_qkv_rope_rows(rt, heads, kv_heads, head):
    n, seq, pos = 300, 40, 13
    ws, x = qkv_weights(rt, heads, kv_heads, head, n), stream(1, n)
    nw = (1 + 0.2 * oracle.normal(n, 5)).astype(np.float32)
    table = oracle.rope_table(10000.0, head, seq)
    dims = [heads * head, kv_heads * head, kv_heads * head]
    out = [rt.alloc(d * 4) for d in dims]
    args = [rt.handle, None, up(rt, x), up(rt, nw), F32, EPS, *[m.dev for m in ws], W4, n, heads, kv_heads,
            head, *out, seq]
    call("ammon_qkv_rope", *args, rt.step(0, pos), up(rt, table))
    for o, d, (want, bar) in zip(out, dims, qkv_of(norm_of(x, nw, F32), ws, table[pos:pos + 1], head, NORM)):
        close(o.download((1, d)), want, bar)
    call("ammon_qkv_rope", *args, rt.step(0, seq), up(rt, table))
    assert all(np.isnan(o.download(d)).all() for o, d in zip(out, dims))


@pytest.mark.parametrize("kvd", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads,head", HEADS[:3])
def test_qkv_rope_store(rt, heads, kv_heads, head, kvd):
    n, seq, pos = 300, 20, 13
    ws, x = qkv_weights(rt, heads, kv_heads, head, n), stream(1, n)
    table = oracle.rope_table(10000.0, head, seq)
    kv = kv_heads * head
    rows = [rt.alloc(4 * kv) for _ in "kv"]
    q, q2 = rt.alloc(4 * heads * head), rt.alloc(4 * heads * head)
    caches = [up(rt, oracle.storage(np.full(seq * kv, 3, np.float32), kvd)) for _ in "kv"]
    front = [rt.handle, None, up(rt, x), None, F32, 0.0, *[m.dev for m in ws], W4, n, heads, kv_heads, head]
    call("ammon_qkv_rope", *front, q, *rows, seq, rt.step(0, pos), up(rt, table))
    call("ammon_qkv_rope_store", *front, q2, *caches, kvd, seq, rt.step(0, pos), up(rt, table))
    np.testing.assert_array_equal(q.download(heads * head), q2.download(heads * head))
    dt = np.uint16 if kvd == BF16 else np.float32
    for row, cache in zip(rows, caches):
        got = cache.download((kv_heads, seq, head), dt)
        want = oracle.storage(row.download((kv_heads, head)), kvd).reshape(kv_heads, head)
        np.testing.assert_array_equal(got[:, pos], want)
        rest = np.delete(got, pos, 1)
        assert np.all(rest == oracle.storage(np.array([3], np.float32), kvd)[0])
    before = [c.download((kv_heads, seq, head), dt) for c in caches]
    call("ammon_qkv_rope_store", *front, q2, *caches, kvd, seq, rt.step(0, 0xffffffff), up(rt, table))
    assert np.isnan(q2.download(heads * head)).all()
    for c, b in zip(caches, before):
        np.testing.assert_array_equal(c.download(b.shape, dt), b)


@pytest.mark.parametrize("vocab,dim", [(1, 64), (100, 300), (9000, 256), (70001, 500), (5000, 9000)])
def test_greedy_lm_head(rt, vocab, dim):
    w, x = Weights(rt, vocab, dim), stream(1, dim)
    nw = (1 + 0.2 * oracle.normal(dim, 5)).astype(np.float32)
    logits, plain = rt.alloc(vocab * 4), rt.alloc(vocab * 4)
    size = int(lib.ammon_greedy_lm_head_scratch_bytes(rt.handle))
    scratch, tokens, step = rt.alloc(size), rt.upload(np.full(8, -1, np.int32)), rt.step(3, 4)
    call("ammon_greedy_lm_head", rt.handle, None, up(rt, x), up(rt, nw), F32, EPS, w.dev, W4, vocab, dim,
         logits, scratch, size, None, 0, step, tokens, 8)
    call("ammon_gemv_rmsnorm", rt.handle, None, up(rt, x), up(rt, nw), F32, EPS, w.dev, W4, vocab, dim, plain)
    got = logits.download(vocab)
    np.testing.assert_array_equal(got, plain.download(vocab))
    assert rt.read_step(step) == (int(np.argmax(got)), 5)
    assert list(tokens.download(8, np.int32)) == [-1] * 4 + [int(np.argmax(got))] + [-1] * 3


def test_gemv_numbers_that_are_not_finite(rt):
    d, n = 40, 400
    m = matrix(d, n)
    m[7, 130] = np.nan
    w = Weights(rt, d, n, w=m)
    y = rt.alloc(d * 4)
    x = stream(1, n)
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, x), y, None)
    got = y.download(d)
    assert np.isnan(got[7]) and np.isfinite(np.delete(got, 7)).all()
    for bad in (np.nan, np.inf):
        x2 = x.copy()
        x2[0, 399] = bad
        call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, x2), y, None)
        assert np.isnan(y.download(d)).all()
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, 0 * x), y, None)
    assert np.all(np.delete(y.download(d), 7) == 0)


@pytest.mark.parametrize("scale", [2.0**-60, 2.0**40, 2.0**100])
def test_gemv_x_of_any_size(rt, scale):
    w, x = Weights(rt, 64, 512), stream(1, 512)
    y, z = rt.alloc(256), rt.alloc(256)
    call("ammon_gemv", rt.handle, None, w.dev, W4, 64, 512, up(rt, x), y, None)
    call("ammon_gemv", rt.handle, None, w.dev, W4, 64, 512, up(rt, x * np.float32(scale)), z, None)
    np.testing.assert_array_equal(y.download(64) * np.float32(scale), z.download(64))


def test_qkv_rope_of_many_groups(rt):
    """The q, k and v matrices' units shared by waves side by side: as the three products, turned."""
    n, seq, pos, heads, kv_heads, head = 4300, 30, 7, 36, 4, 96
    ws, x = qkv_weights(rt, heads, kv_heads, head, n), stream(1, n)
    table = oracle.rope_table(10000.0, head, seq)
    dims = [heads * head, kv_heads * head, kv_heads * head]
    assert sum(dims) // 16 >= 256
    out = [rt.alloc(d * 4) for d in dims]
    call("ammon_qkv_rope", rt.handle, None, up(rt, x), None, F32, 0.0, *[m.dev for m in ws], W4, n, heads,
         kv_heads, head, *out, seq, rt.step(0, pos), up(rt, table))
    for o, d, (want, bar) in zip(out, dims, qkv_of(x.astype(np.float64), ws, table[pos:pos + 1], head, 0)):
        close(o.download((1, d)), want, bar)


# ---- prompts -------------------------------------------------------------------------------------
def workspace(rt, rows, tokens, size=None):
    size = int(lib.ammon_prefill_gemm_workspace_bytes(rows, tokens)) if size is None else size
    buf = rt.alloc(size)
    rt.fill(buf, F32, size // 4, float("nan"))
    return buf, size


GEMM = [(1, 1, 1), (16, 128, 16), (17, 129, 3), (300, 288, 17), (70, 1000, 33), (1030, 512, 65),
        (96, 4096, 5), (260, 300, 130), (48, 14336, 64), (512, 2080, 301), (4100, 256, 40),
        # 16 rows of sixteen waves; 32 and 64 rows to a workgroup, tokens of one and two panels; long tiles
        (90, 14000, 5), (9001, 300, 37), (20000, 260, 5), (4200, 2100, 130), (3000, 1000, 600)]


@pytest.mark.parametrize("d,n,t", GEMM)
@pytest.mark.parametrize("dtype", [Q8, Q24])
@pytest.mark.parametrize("residual,ws", [(None, True), ("y", True), ("other", False)])
def test_prefill_gemm(rt, d, n, t, dtype, residual, ws):
    w, x = Weights(rt, d, n), Rows(rt, stream(t, n), dtype)
    r = oracle.normal(t * d, 9).reshape(t, d)
    want, bar = x.numbers @ w.numbers.T, w4.product_bar(x.numbers, w.numbers, True)
    y = rt.alloc(t * d * 4 + 64)
    rt.fill(y, F32, t * d + 16, 7.0)
    rt.synchronize()
    if residual == "y":
        y.upload(r)
    other = {"y": y, "other": up(rt, r), None: None}[residual]
    call("ammon_prefill_gemm_w4", rt.handle, None, w.dev, d, n, x.dev, dtype, t, y, other,
         *(workspace(rt, d, t) if ws else (None, 0)))
    got = y.download(t * d + 16)
    if residual:
        want, bar = want + r, bar + 2.0**-24 * (np.abs(want) + np.abs(r))
    close(got[:t * d].reshape(t, d), want, bar)
    assert set(got[t * d:]) == {7.0}


@pytest.mark.parametrize("hidden,n,t", [(1, 1, 1), (8, 128, 16), (40, 300, 17), (768, 288, 33), (1000, 512, 70),
                                        (24, 8192, 5), (2100, 256, 130), (7000, 300, 20), (3001, 900, 150),
                                        (9000, 300, 33)])
@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_prefill_gate_up_swiglu(rt, hidden, n, t, dtype):
    a, b = Weights(rt, hidden, n, 1), Weights(rt, hidden, n, 11)
    x = Rows(rt, stream(t, n), dtype)
    hb = rt.alloc(t * hidden * 4 + 64)
    rt.fill(hb, F32, t * hidden + 16, 7.0)
    call("ammon_prefill_gate_up_swiglu_w4", rt.handle, None, x.dev, dtype, t, a.dev, b.dev, n, hidden, hb)
    bars = [w4.product_bar(x.numbers, m.numbers, True) for m in (a, b)]
    got = hb.download(t * hidden + 16)
    close(got[:t * hidden].reshape(t, hidden),
          *swiglu_of(x.numbers @ a.numbers.T, x.numbers @ b.numbers.T, *bars))
    assert set(got[t * hidden:]) == {7.0}


@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_prefill_qkv_rope_of_long_rows(rt, dtype):
    n, seq, pos, t, heads, head = 13000, 30, 4, 5, 6, 48
    ws, x = qkv_weights(rt, heads, heads, head, n), Rows(rt, stream(t, n), dtype)
    table = oracle.rope_table(10000.0, head, seq)
    out = [rt.alloc(t * heads * head * 4) for _ in "qkv"]
    call("ammon_prefill_qkv_rope_w4", rt.handle, None, x.dev, dtype, t, *[m.dev for m in ws], n, heads, heads, head,
         *out, seq, rt.step(0, pos), up(rt, table), None, 0)
    for o, (want, bar) in zip(out, qkv_of(x.numbers, ws, table[pos:pos + t], head, None)):
        close(o.download((t, heads * head)), want, bar)


@pytest.mark.parametrize("t", [1, 16, 20, 70])
@pytest.mark.parametrize("heads,kv_heads,head", HEADS)
def test_prefill_qkv_rope(rt, heads, kv_heads, head, t):
    n, seq, pos = 300, 100, 13
    ws = qkv_weights(rt, heads, kv_heads, head, n)
    table = oracle.rope_table(10000.0, head, seq)
    dims = [heads * head, kv_heads * head, kv_heads * head]
    for dtype in (Q8, Q24):
        x = Rows(rt, stream(t, n), dtype)
        for space in (workspace(rt, sum(dims), t), (None, 0)):
            out = [rt.alloc(t * d * 4) for d in dims]
            args = [rt.handle, None, x.dev, dtype, t, *[m.dev for m in ws], n, heads, kv_heads, head, *out, seq]
            call("ammon_prefill_qkv_rope_w4", *args, rt.step(0, pos), up(rt, table), *space)
            for o, d, (want, bar) in zip(out, dims, qkv_of(x.numbers, ws, table[pos:pos + t], head, None)):
                close(o.download((t, d)), want, bar)


@pytest.mark.parametrize("kvd", [F32, BF16])
@pytest.mark.parametrize("t", [7, 30])
def test_prefill_qkv_rope_store(rt, kvd, t):
    heads, kv_heads, head, n, seq, pos = 6, 2, 48, 300, 32, 10
    ws, x = qkv_weights(rt, heads, kv_heads, head, n), Rows(rt, stream(t, n), Q24)
    table, kv, fits = up(rt, oracle.rope_table(10000.0, head, seq)), kv_heads * head, min(t, seq - pos)
    rows = [rt.alloc(4 * kv * t) for _ in "kv"]
    q, q2 = rt.alloc(4 * heads * head * t), rt.alloc(4 * heads * head * t)
    caches = [up(rt, oracle.storage(np.full(seq * kv, 3, np.float32), kvd)) for _ in "kv"]
    front = [rt.handle, None, x.dev, Q24, t, *[m.dev for m in ws], n, heads, kv_heads, head]
    dt = np.uint16 if kvd == BF16 else np.float32
    for first in (pos, 0xfffffffe):
        step = rt.step(0, first)
        call("ammon_prefill_qkv_rope_w4", *front, q, *rows, seq, step, table, None, 0)
        call("ammon_prefill_qkv_rope_store_w4", *front, q2, *caches, kvd, seq, step, table, None, 0)
        got = q2.download((t, heads * head))
        np.testing.assert_array_equal(got, q.download((t, heads * head)))
        n_ok = fits if first == pos else 0
        assert np.isfinite(got[:n_ok]).all() and np.isnan(got[n_ok:]).all()
        for row, cache in zip(rows, caches):
            r = row.download((t, kv_heads, head))
            assert np.isfinite(r[:n_ok]).all() and np.isnan(r[n_ok:]).all()
            c = cache.download((kv_heads, seq, head), dt)
            if n_ok:
                want = oracle.storage(r[:fits].reshape(-1), kvd).reshape(fits, kv_heads, head)
                np.testing.assert_array_equal(c[:, pos:pos + fits], want.transpose(1, 0, 2))
            rest = np.delete(c, np.s_[pos:pos + fits], 1)
            assert np.all(rest == oracle.storage(np.array([3], np.float32), kvd)[0])
        if n_ok:
            before = [c.download((kv_heads, seq, head), dt) for c in caches]
    for c, b in zip(caches, before):
        np.testing.assert_array_equal(c.download(b.shape, dt), b)


def test_prompt_tokens_do_not_touch_each_other(rt):
    """A NaN token is NaN alone, and a token's result does not depend on its neighbours."""
    d, n, t = 80, 400, 40
    w, x = Weights(rt, d, n), stream(t, n)
    bad = x.copy()
    bad[5, 3], bad[20, 399] = np.nan, np.inf
    for dtype in (Q8, Q24):
        out = []
        for rows in (x, bad):
            y = rt.alloc(t * d * 4)
            call("ammon_prefill_gemm_w4", rt.handle, None, w.dev, d, n, Rows(rt, rows, dtype).dev, dtype, t, y,
                 None, None, 0)
            out.append(y.download((t, d)))
        assert np.isnan(out[1][[5, 20]]).all()
        keep = np.delete(np.arange(t), [5, 20])
        np.testing.assert_array_equal(out[0][keep], out[1][keep])


# ---- as they are used together ---------------------------------------------------------------------
def test_a_block_in_a_graph(rt):
    """Residual + norm + digits, gate/up, digits, down: captured once, replayed on new rows, equal
    to the eager calls, with eager work between the replays."""
    t, dim, hidden = 21, 288, 768
    gate, upw, down = Weights(rt, hidden, dim, 1), Weights(rt, hidden, dim, 11), Weights(rt, dim, hidden, 21)
    nw = up(rt, (1 + 0.2 * oracle.normal(dim, 5)).astype(np.float32))
    x, r = rt.alloc(t * dim * 4), rt.alloc(t * dim * 4)
    xq = rt.alloc(int(lib.ammon_q8_bytes(Q24, t, dim)))
    hq = rt.alloc(int(lib.ammon_q8_bytes(Q24, t, hidden)))
    hb = rt.alloc(t * hidden * 4)
    ws, size = workspace(rt, dim, t)
    s = ctypes.c_void_p()
    call("ammon_stream_create", rt.handle, ctypes.byref(s))

    def block(st):
        call("ammon_rmsnorm_q8", rt.handle, st, x, r, x, nw, F32, EPS, t, dim, xq, Q24)
        call("ammon_prefill_gate_up_swiglu_w4", rt.handle, st, xq, Q24, t, gate.dev, upw.dev, dim, hidden, hb)
        call("ammon_q8_store", rt.handle, st, hb, t, hidden, hq, Q24)
        call("ammon_prefill_gemm_w4", rt.handle, st, down.dev, dim, hidden, hq, Q24, t, x, x, ws, size)

    call("ammon_capture_begin", rt.handle, s)
    block(s)
    graph = ctypes.c_void_p()
    call("ammon_capture_end", rt.handle, s, ctypes.byref(graph))
    for seed in range(4):
        a, b = stream(t, dim, 30 + seed), stream(t, dim, 60 + seed)
        x.upload(a), r.upload(b)
        block(None)
        want = x.download((t, dim))
        x.upload(a)
        call("ammon_graph_launch", rt.handle, graph, s)
        rt.synchronize(s)
        np.testing.assert_array_equal(x.download((t, dim)), want)
        # and the formula, over the stored numbers
        h = (a + b).astype(np.float64)
        xn = norm_of(a + b, np.asarray(nw.download(dim)), F32)
        g, u = xn @ gate.numbers.T, xn @ upw.numbers.T
        ref = h + (g / (1 + np.exp(-g)) * u) @ down.numbers.T
        assert np.max(np.abs(want - ref)) <= 2e-6 * np.max(np.abs(ref)) * 10
    call("ammon_graph_destroy", rt.handle, graph)
    call("ammon_stream_destroy", rt.handle, s)


# ---- refusals ------------------------------------------------------------------------------------
def refused(match, name, *args):
    with pytest.raises(AmmonError, match=match):
        call(name, *args)


def test_refusals(rt):
    h, b = rt.handle, rt.alloc(1 << 20)
    o = lambda k: b.offset(k)  # noqa: E731
    step, f, z = rt.step(0, 0), 1e-5, None
    for name, args in (("ammon_w4_store", (b, F32, 16, 16, o(4096))),
                       ("ammon_q8_store", (b, 2, 16, o(4096), Q8))):
        call(name, h, _abi.STREAM_VALIDATE, *args)
    refused("NULL", "ammon_w4_store", h, z, z, F32, 16, 16, b)
    refused("unknown dtype", "ammon_w4_store", h, z, b, W4, 16, 16, o(4096))
    refused("empty", "ammon_w4_store", h, z, b, F32, 0, 16, o(4096))
    refused("empty", "ammon_w4_store", h, z, b, F32, 16, 0, o(4096))
    refused("16-byte", "ammon_w4_store", h, z, b, F32, 16, 16, o(4104))
    refused("overlaps", "ammon_w4_store", h, z, b, F32, 16, 16, o(512))
    refused("too many", "ammon_w4_store", h, z, b, F32, 0xffffffff, 1, o(4096))
    refused("too long", "ammon_w4_store", h, z, b, F32, 1, 0xffffffff, o(4096))
    refused("output dtype", "ammon_w4_load", h, z, b, 16, 16, o(4096), Q8)
    refused("16-byte", "ammon_w4_load", h, z, o(4), 16, 16, o(4096), F32)
    refused("overlaps", "ammon_w4_load", h, z, b, 16, 16, o(512), F32)
    refused("AMMON_Q8 or", "ammon_q8_store", h, z, b, 2, 16, o(4096), F32)
    refused("empty", "ammon_q8_store", h, z, b, 0, 16, o(4096), Q8)
    refused("16-byte", "ammon_q8_store", h, z, b, 2, 16, o(4100), Q8)
    refused("overlap", "ammon_q8_store", h, z, b, 2, 16, o(64), Q8)
    refused("AMMON_Q8 or", "ammon_q8_load", h, z, b, BF16, 2, 16, o(8192))
    refused("overlaps", "ammon_q8_load", h, z, b, Q8, 2, 16, o(16))
    norm = (o(16384), F32, f, 2, 16, o(8192), Q8)
    call("ammon_rmsnorm_q8", h, _abi.STREAM_VALIDATE, b, o(1024), o(1024), *norm)
    refused("go together", "ammon_rmsnorm_q8", h, z, b, o(1024), z, *norm)
    refused("go together", "ammon_rmsnorm_q8", h, z, b, z, o(1024), *norm)
    refused("partially", "ammon_rmsnorm_q8", h, z, b, o(1024), o(1056), *norm)
    refused("partially", "ammon_rmsnorm_q8", h, z, b, o(1024), o(32), *norm)
    refused("NULL", "ammon_rmsnorm_q8", h, z, b, z, z, z, F32, f, 2, 16, o(8192), Q8)
    refused("weight dtype", "ammon_rmsnorm_q8", h, z, b, z, z, o(16384), W4, f, 2, 16, o(8192), Q8)
    refused("eps", "ammon_rmsnorm_q8", h, z, b, z, z, o(16384), F32, -1.0, 2, 16, o(8192), Q8)
    refused("weight overlaps", "ammon_rmsnorm_q8", h, z, b, z, z, o(8192), F32, f, 2, 16, o(8192), Q8)
    # one token
    refused("16-byte", "ammon_gemv", h, z, o(8), W4, 16, 16, o(8192), o(16384), z)
    refused("overlaps x", "ammon_gemv", h, z, b, W4, 16, 16, o(8192), o(8200), z)
    refused("LDS", "ammon_gemv", h, z, b, W4, 16, 100000, o(8192), o(512000), z)
    refused("no W4", "ammon_gemv_at_position", h, z, b, W4, 16, 16, o(8192), o(16384), 4, step)
    refused("multiple of 16", "ammon_qkv_rope", h, z, o(16384), z, F32, f, b, b, b, W4, 16, 2, 1, 8, o(20480),
            o(24576), o(28672), 4, step, b)
    refused("table dtype", "ammon_embed", h, z, b, W4, 16, 16, step, o(8192))
    refused("rows of digits", "ammon_prefill_gemm", h, z, b, W4, 16, 16, o(8192), 2, o(16384), z)
    # prompts
    g = lambda *a: ("ammon_prefill_gemm_w4", h, z, *a)  # noqa: E731
    x, y = o(8192), o(32768)
    call("ammon_prefill_gemm_w4", h, _abi.STREAM_VALIDATE, b, 16, 16, x, Q8, 2, y, y, z, 0)
    refused("NULL", *g(z, 16, 16, x, Q8, 2, y, z, z, 0))
    refused("rows of digits", *g(b, 16, 16, x, F32, 2, y, z, z, 0))
    refused("empty", *g(b, 16, 16, x, Q8, 0, y, z, z, 0))
    refused("empty", *g(b, 0, 16, x, Q8, 2, y, z, z, 0))
    refused("16-byte", *g(o(8), 16, 16, x, Q8, 2, y, z, z, 0))
    refused("16-byte", *g(b, 16, 16, o(8200), Q8, 2, y, z, z, 0))
    refused("overlaps x", *g(b, 16, 16, x, Q8, 2, o(8256), z, z, 0))
    refused("overlaps weights", *g(b, 16, 16, x, Q8, 2, o(64), z, z, 0))
    refused("partially", *g(b, 16, 16, x, Q8, 2, y, o(32772), z, 0))
    refused("workspace", *g(b, 16, 16, x, Q8, 2, y, z, y, 64))
    refused("workspace", *g(b, 16, 16, x, Q8, 2, y, z, o(40968), 64))
    refused("NULL w1", "ammon_prefill_gate_up_swiglu_w4", h, z, x, Q8, 2, b, z, 16, 16, y)
    qkv = lambda heads, kvh, head, kvd, k, v: (  # noqa: E731
        "ammon_prefill_qkv_rope_store_w4", h, z, x, Q8, 2, b, b, b, 16, heads, kvh, head, y, k, v, kvd, 4, step,
        b, z, 0)
    k, v = o(36864), o(40960)
    call(*qkv(1, 1, 16, F32, k, v))
    refused("KV4", *qkv(1, 1, 16, KV4, k, v))
    refused("kv dtype", *qkv(1, 1, 16, Q8, k, v))
    refused("even", *qkv(16, 16, 1, F32, k, v))
    refused("multiple of 16", *qkv(1, 1, 24, F32, k, v))
    refused("wider", *qkv(1, 2, 16, F32, k, v))
    refused("caches overlap", *qkv(1, 1, 16, F32, k, o(36880)))
    refused("overlaps x or q", *qkv(1, 1, 16, F32, k, y))
    refused("pairs", *qkv(1, 1, 16, F32, o(36868), v))
    rt.synchronize()
