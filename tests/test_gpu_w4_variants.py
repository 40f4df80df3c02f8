"""Every kernel of the 4-bit weights' products against float64: each tile of the prompt products, whole
and with its reduction in ranges, and each way of the one-token products, in every mode.

A product takes the variant that ammon_w4_choose named, or is refused; so a test runs the kernel that it
names.  What the library takes by itself is compared with the named variant bit for bit.
"""
import numpy as np
import pytest

import oracle
from ammon_amd import AmmonError
from ammon_amd._abi import BF16, F32, Q8, Q24, W4, call, lib
from oracle import w4
from test_gpu_w4 import EPS, NORM, Rows, Weights, close, matrix, norm_of, qkv_of, stream, swiglu_of, up, workspace

pytestmark = pytest.mark.gpu
TILES = {Q8: ["t16", "t16_deep", "t16_x4", "t32_x2", "t64", "long"],
         Q24: ["t16", "t16_deep", "t16_x2", "t16_x4", "t64", "long"]}
WAYS = ["k8_one", "k8", "k2", "k8_wide", "flat"]
KINDS = [(q, tile) for q in (Q8, Q24) for tile in TILES[q]]
# panels of rows (gated: of results, half as many where big) and tokens of a tile
SIZE = {(Q8, "t16"): (1, 16), (Q8, "t16_deep"): (1, 16), (Q8, "t16_x4"): (4, 16), (Q8, "t32_x2"): (2, 32),
        (Q8, "t64"): (8, 64), (Q8, "long"): (8, 128), (Q24, "t16"): (1, 16), (Q24, "t16_deep"): (1, 16),
        (Q24, "t16_x2"): (2, 16), (Q24, "t16_x4"): (4, 16), (Q24, "t64"): (8, 64), (Q24, "long"): (16, 64)}


@pytest.fixture
def tuned(rt):
    """The runtime, its products taking the variant named, or again the library's."""

    def get(tile=None, way=None):
        call("ammon_w4_choose", rt.handle, *[None if name is None else name.encode() for name in (tile, way)])
        return rt

    yield get
    get()


class Panels(Weights):
    """A matrix of d rows that repeats 7 panels of their own: every unit's neighbours differ."""

    def __init__(self, rt, d, n, seed=1):
        codes, s = w4.w4_quantise(matrix(112, n, seed))
        self.seven = w4.w4_numbers(codes, s, n)
        panels = -(-d // 16)
        size = w4.w4_bytes(112, n) // 7
        self.dev = up(rt, np.resize(w4.w4_pack(codes, s).reshape(7, size), (panels, size)))
        self.d = d

    def rows(self, y):
        """Columns [.., 112] of the seven panels as the whole matrix's [.., d]."""
        return np.concatenate([y] * (-(-self.d // 112)), -1)[..., :self.d]


def gemm(rt, w, d, n, x, dtype, t, residual=None, ws=(None, 0)):
    """ammon_prefill_gemm_w4 with what lies behind its result; residual: in place."""
    y = rt.alloc(t * d * 4 + 64)
    rt.fill(y, F32, t * d + 16, 7.0)
    rt.synchronize()
    if residual is not None:
        y.upload(residual)
    call("ammon_prefill_gemm_w4", rt.handle, None, w, d, n, x, dtype, t, y, None if residual is None else y, *ws)
    got = y.download(t * d + 16)
    assert set(got[t * d:]) == {7.0}
    return got[:t * d].reshape(t, d)


def check_gemm(rt, d, n, t, dtype, ws=None):
    w, x = Weights(rt, d, n), Rows(rt, stream(t, n), dtype)
    want, bar = x.numbers @ w.numbers.T, w4.product_bar(x.numbers, w.numbers, True)
    space = ws() if ws else (None, 0)
    close(gemm(rt, w.dev, d, n, x.dev, dtype, t, ws=space), want, bar)
    r = oracle.normal(t * d, 9).reshape(t, d)
    got = gemm(rt, w.dev, d, n, x.dev, dtype, t, r, space)
    close(got, want + r, bar + 2.0**-24 * (np.abs(want) + np.abs(r)))


# ---- prompts: every tile --------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,tile", KINDS)
@pytest.mark.parametrize("n", [96, 300, 400, 520, 1100])  # 1, 3, 4, 5 and 9 groups
def test_tiles(tuned, dtype, tile, n):
    """One token, part of a panel of tokens, part of a tile; part of a panel of rows, two row blocks."""
    rt = tuned(tile=tile)
    panels, tokens = SIZE[dtype, tile]
    check_gemm(rt, 5, n, 1, dtype)
    check_gemm(rt, 16 * panels + 21, n, tokens + 19, dtype)


@pytest.mark.parametrize("dtype,tile", KINDS)
def test_tiles_of_more_blocks_than_xcds(tuned, dtype, tile):
    rt = tuned(tile=tile)
    panels, tokens = SIZE[dtype, tile]
    check_gemm(rt, 16 * panels * 9 + 5, 200, 2 * tokens + 3, dtype)


@pytest.mark.parametrize("dtype,tile", [k for k in KINDS if k[1] != "t16_deep"])
@pytest.mark.parametrize("n", [96, 300, 400, 1100])
def test_gated_tiles(tuned, dtype, tile, n):
    rt = tuned(tile=tile)
    panels, tokens = SIZE[dtype, tile]
    for hidden, t in ((3, 1), (16 * panels + 21, tokens + 19)):
        a, b, x = Weights(rt, hidden, n, 1), Weights(rt, hidden, n, 11), Rows(rt, stream(t, n), dtype)
        hb = rt.alloc(t * hidden * 4 + 64)
        rt.fill(hb, F32, t * hidden + 16, 7.0)
        call("ammon_prefill_gate_up_swiglu_w4", rt.handle, None, x.dev, dtype, t, a.dev, b.dev, n, hidden, hb)
        got = hb.download(t * hidden + 16)
        bars = [w4.product_bar(x.numbers, m.numbers, True) for m in (a, b)]
        close(got[:t * hidden].reshape(t, hidden), *swiglu_of(x.numbers @ a.numbers.T, x.numbers @ b.numbers.T, *bars))
        assert set(got[t * hidden:]) == {7.0}


def check_qkv(rt, dtype, heads, kv_heads, head, n, t, ws=None):
    """Rows, then both kinds of caches, which have the rows' numbers; the last tokens past the caches."""
    seq, pos = 13 + t - min(2, t - 1), 13
    table = oracle.rope_table(10000.0, head, seq)
    dims = [heads * head, kv_heads * head, kv_heads * head]
    weights = [Weights(rt, d, n, s) for d, s in zip(dims, (1, 11, 21))]
    x, fits, tab = Rows(rt, stream(t, n), dtype), seq - pos, up(rt, table)
    out = [rt.alloc(t * d * 4) for d in dims]
    front = [rt.handle, None, x.dev, dtype, t, *[m.dev for m in weights], n, heads, kv_heads, head]
    call("ammon_prefill_qkv_rope_w4", *front, *out, seq, rt.step(0, pos), tab, *(ws() if ws else (None, 0)))
    rows = [o.download((t, d)) for o, d in zip(out, dims)]
    for got, (want, bar) in zip(rows, qkv_of(x.numbers[:fits], weights, table[pos:pos + fits], head, None)):
        close(got[:fits], want, bar)
        assert np.isnan(got[fits:]).all()
    for kvd in (F32, BF16):
        dt = np.uint16 if kvd == BF16 else np.float32
        filler = oracle.storage(np.full(seq * dims[1], 3, np.float32), kvd)
        caches = [up(rt, filler) for _ in "kv"]
        call("ammon_prefill_qkv_rope_store_w4", *front, out[0], *caches, kvd, seq, rt.step(0, pos), tab,
             *(ws() if ws else (None, 0)))
        np.testing.assert_array_equal(out[0].download((t, dims[0])), rows[0])
        for cache, r in zip(caches, rows[1:]):
            got = cache.download((kv_heads, seq, head), dt)
            want = oracle.storage(r[:fits].reshape(-1), kvd).reshape(fits, kv_heads, head)
            np.testing.assert_array_equal(got[:, pos:], want.transpose(1, 0, 2))
            assert (got[:, :pos] == filler[0]).all()


@pytest.mark.parametrize("dtype,tile", KINDS)
@pytest.mark.parametrize("heads,kv_heads,head,n", [(6, 2, 48, 300), (14, 2, 64, 400), (2, 1, 16, 1100)])
def test_qkv_tiles(tuned, dtype, tile, heads, kv_heads, head, n):
    rt = tuned(tile=tile)
    for t in (1, SIZE[dtype, tile][1] + 19):
        check_qkv(rt, dtype, heads, kv_heads, head, n, t)


# ---- prompts: the reduction in ranges ----------------------------------------------------------------
RANGES = [(q, tile, k) for q in (Q8, Q24) for tile in ("t64", "long") for k in (2, 4, 8)]


def nan_workspace(rt, rows, t, k, made):
    """A workspace for eight ranges, the k ranges' part of which has to be written, and no more."""
    def get():
        made.append(workspace(rt, rows, t))
        return made[-1]

    def written():
        for buf, size in made:
            got = buf.download(size // 4)
            assert not np.isnan(got[:k * t * rows]).any() and np.isnan(got[k * t * rows:]).all()
    return get, written


@pytest.mark.parametrize("dtype,tile,k", RANGES)
@pytest.mark.parametrize("n", [4200, 4096, 5000])  # 33 groups (of eight ranges the last has none), 32, 40
def test_ranges(tuned, dtype, tile, k, n):
    rt, made = tuned(tile=f"{tile}/{k}"), []
    panels, tokens = SIZE[dtype, tile]
    d, t = 16 * panels + 21, tokens + 19
    get, written = nan_workspace(rt, d, t, k, made)
    check_gemm(rt, d, n, t, dtype, get)
    written()


@pytest.mark.parametrize("dtype,tile,k", RANGES)
def test_qkv_ranges(tuned, dtype, tile, k):
    rt, made = tuned(tile=f"{tile}/{k}"), []
    t = SIZE[dtype, tile][1] + 19
    get, written = nan_workspace(rt, 10 * 48, t, k, made)
    check_qkv(rt, dtype, 6, 2, 48, 4200, t, get)
    written()


@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_ranges_go_by_the_workspace(tuned, rt, dtype):
    """As many ranges as the workspace holds: nothing behind it is written, and fewer are right too."""
    d, n, t = 288, 8192, 700
    w, x = Panels(rt, d, n), Rows(rt, stream(t, n), dtype)
    seven = x.numbers @ w.seven.T
    want, bar = w.rows(seven), w.rows(w4.product_bar(x.numbers, w.seven, True))
    tile = "t64" if dtype == Q8 else "long"
    for k in (8, 4, 2):
        size = k * t * d * 4
        buf = rt.alloc(size + 64)
        rt.fill(buf, F32, size // 4 + 16, float("nan"))
        tuned(f"{tile}/{k}")
        got = gemm(rt, w.dev, d, n, x.dev, dtype, t, ws=(buf, size))
        close(got, want, bar)
        words = buf.download(size // 4 + 16)
        assert not np.isnan(words[:-16]).any() and np.isnan(words[-16:]).all()
        for space in ((buf, size - 4), (None, 0)):
            tuned(f"{tile}/{k}")
            with pytest.raises(AmmonError, match="does not take"):
                gemm(rt, w.dev, d, n, x.dev, dtype, t, ws=space)
            tuned()
            rt.fill(buf, F32, size // 4 + 16, float("nan"))
            close(gemm(rt, w.dev, d, n, x.dev, dtype, t, ws=space), want, bar)
            assert np.isnan(buf.download(size // 4 + 16)[-17:]).all()


# ---- prompts: what the rule takes ----------------------------------------------------------------
@pytest.mark.parametrize("dtype,d,n,t,variant", [
    (Q24, 2048, 300, 1500, "long/1"), (Q24, 8200, 300, 300, "long/1"), (Q24, 3000, 1000, 600, "t64/1"),
    (Q24, 288, 8192, 700, "long/8"), (Q24, 256, 5120, 600, "t64/8"), (Q24, 520, 8300, 301, "t64/8"),
    (Q24, 4200, 2100, 130, "t16_x4/1"), (Q24, 512, 14336, 100, "t16_deep/1"), (Q24, 512, 14336, 130, "t16_x2/1"),
    (Q8, 8200, 300, 1100, "long/1"), (Q8, 9001, 300, 2100, "long/1"), (Q8, 288, 8192, 700, "t64/8"),
    (Q8, 3000, 1000, 600, "t64/1"), (Q8, 256, 5120, 600, "t32_x2/1")])
def test_the_rule_takes(tuned, rt, dtype, d, n, t, variant):
    """At 256 compute units, with a workspace: bit for bit the variant named, and right."""
    w, x = Panels(rt, d, n), Rows(rt, stream(t, n), dtype)
    made = []
    get, written = nan_workspace(rt, d, t, int(variant.split("/")[1]), made)
    got = gemm(rt, w.dev, d, n, x.dev, dtype, t, ws=get())
    if not variant.endswith("/1"):
        written()
    else:
        assert np.isnan(made[0][0].download(made[0][1] // 4)).all()
    tuned(variant)
    np.testing.assert_array_equal(got, gemm(rt, w.dev, d, n, x.dev, dtype, t, ws=workspace(rt, d, t)))
    close(got, w.rows(x.numbers @ w.seven.T), w.rows(w4.product_bar(x.numbers, w.seven, True)))


@pytest.mark.parametrize("dtype,hidden,n,t,variant", [(Q24, 4000, 300, 300, "long"), (Q24, 9000, 300, 200, "t64"),
                                                      (Q8, 8000, 300, 1000, "long"), (Q8, 8000, 300, 520, "t64"),
                                                      (Q24, 7000, 300, 20, "t16_x4"), (Q8, 7000, 300, 20, "t32_x2")])
def test_the_rule_takes_gated(tuned, rt, dtype, hidden, n, t, variant):
    a, b, x = Panels(rt, hidden, n, 1), Panels(rt, hidden, n, 11), Rows(rt, stream(t, n), dtype)
    out = []
    for tile in (None, variant):
        tuned(tile)
        hb = rt.alloc(t * hidden * 4)
        call("ammon_prefill_gate_up_swiglu_w4", rt.handle, None, x.dev, dtype, t, a.dev, b.dev, n, hidden, hb)
        out.append(hb.download((t, hidden)))
    np.testing.assert_array_equal(*out)
    bars = [w4.product_bar(x.numbers, m.seven, True) for m in (a, b)]
    want, bar = swiglu_of(x.numbers @ a.seven.T, x.numbers @ b.seven.T, *bars)
    close(out[0], a.rows(want), a.rows(bar))


# ---- prompts: the digits' ends ---------------------------------------------------------------------
@pytest.mark.parametrize("dtype,tile", KINDS)
def test_digits_at_their_ends(tuned, dtype, tile):
    """Every digit and code at its least or largest: a group's sums as large as they get, exactly.
    (y = s_w s_x sum c q is below 2^24 times a power of two where q is one digit or +-65536 of them.)"""
    rt = tuned(tile=tile)
    panels, tokens = SIZE[dtype, tile]
    d, n, t, digits = 16 * panels, 256, tokens, 1 if dtype == Q8 else 3
    codes = np.where(np.arange(d)[:, None, None] % 3 == 1, 7, -8) * np.ones((1, 2, 128), np.int64)
    s = np.full((d, 2), 0.5)
    lowest = -128 * (1 + 256 + 65536) if digits == 3 else -128
    largest = 127 * (1 + 256 + 65536) if digits == 3 else 127
    q = np.where(np.arange(t)[:, None, None] % 2 == 1, largest, lowest) * np.ones((1, 2, 128), np.int64)
    sx = np.full((t, 2), 2.0**-3)
    w, x = up(rt, w4.w4_pack(codes, s)), up(rt, w4.q_pack(q, sx, digits))
    got = gemm(rt, w, d, n, x, dtype, t)
    a, b = w4.w4_numbers(codes, s, n), (q * sx[..., None]).reshape(t, n)
    want = b @ a.T
    if digits == 1:
        np.testing.assert_array_equal(got, want)
    else:  # two groups' sums and digits' sums of 24 bits and more: four roundings
        assert np.max(np.abs(got / want - 1)) <= 4 * 2.0**-24


@pytest.mark.parametrize("tile,k", [(tile, 0) for tile in TILES[Q24]] + [("t64", 8), ("long", 8)])
@pytest.mark.parametrize("size", [2.0**-22, 2.0**-15, 2.0**-8])
def test_the_lower_digits_of_rows(tuned, tile, k, size):
    """A block's one large number meets code 0; the others are `size` times that, so that the result
    is in the lower digits alone."""
    rt = tuned(tile=f"{tile}/{k}" if k else tile)
    panels, tokens = SIZE[Q24, tile]
    d, n, t = 16 * panels + 5, 4200 if k else 700, tokens + 3
    w, x = lower(rt, d, n, size, t)
    rows = Rows(rt, x, Q24)
    assert np.all(rows.numbers[:, 5::128] == 1)
    want, bar = rows.numbers @ w.numbers.T, w4.product_bar(rows.numbers[:, keep(n)], w.numbers[:, keep(n)], True)
    close(gemm(rt, w.dev, d, n, rows.dev, Q24, t, ws=workspace(rt, d, t)), want, bar)
    assert np.all(np.abs(want) > 1000 * bar)


def keep(n):
    return np.arange(n) % 128 != 5


def lower(rt, d, n, size, t=1):
    """Weights with code 0 at number 5 of every group, where rows x [t, n] are 1; elsewhere both are
    positive, x between `size` / 2 and `size`."""
    g = np.random.default_rng(4)
    m = g.uniform(0.3, 1.0, (d, n)).astype(np.float32)
    m[:, 5::128] = 0
    x = (size * g.uniform(0.5, 1.0, (t, n))).astype(np.float32)
    x[:, 5::128] = 1
    return Weights(rt, d, n, w=m), x


# ---- one token: every way ------------------------------------------------------------------------
def gemv_bar(x, w, norm):
    return w4.product_bar(x, w, False) + norm * NORM * np.abs(x) @ np.abs(w).T


# rows and numbers: fewer than a unit; units and chunks that end inside; several units of several chunks;
# groups fewer than waves; the longest row
ONE = [(5, 3), (70, 300), (1030, 1000), (8300, 300), (530, 4300), (9000, 5000), (300, 14400), (33, 36864)]


def takes(way, d, n):
    if way == "k8_one":
        return n <= 4096 and -(-d // 16) <= 512
    return way != "flat" or -(-d // 16) <= 32 * 256


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("d,n", ONE)
def test_ways(tuned, way, d, n):
    rt = tuned(way=way)
    w, x = Panels(rt, d, n), stream(1, n)
    nw, r = (1 + 0.2 * oracle.normal(n, 5)).astype(np.float32), oracle.normal(d, 9).reshape(1, d)
    y, dx = rt.alloc(d * 4 + 64), up(rt, x)
    if not takes(way, d, n):
        with pytest.raises(AmmonError, match="does not take"):
            call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, dx, y, None)
        return
    for res, norm in ((None, False), (r, False), (None, True)):
        rt.fill(y, F32, d + 16, 7.0)
        rt.synchronize()
        if res is not None:
            y.upload(res)
        if norm:
            call("ammon_gemv_rmsnorm", rt.handle, None, dx, up(rt, nw), F32, EPS, w.dev, W4, d, n, y)
        else:
            call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, dx, y, None if res is None else y)
        got = y.download(d + 16)
        xn = norm_of(x, nw, F32) if norm else x.astype(np.float64)
        want, bar = w.rows(xn @ w.seven.T), w.rows(gemv_bar(xn, w.seven, norm))
        if res is not None:
            want, bar = want + res, bar + 2.0**-24 * (np.abs(want) + np.abs(res))
        close(got[None, :d], want, bar)
        assert set(got[d:]) == {7.0}


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("hidden,n", [(3, 5), (29, 300), (520, 1000), (4300, 260), (4600, 4300), (300, 14400)])
def test_gated_ways(tuned, way, hidden, n):
    if not takes(way, 2 * hidden, n):
        return
    rt = tuned(way=way)
    a, b, x = Panels(rt, hidden, n, 1), Panels(rt, hidden, n, 11), stream(1, n)
    nw = oracle.storage(1 + 0.2 * oracle.normal(n, 5), BF16)
    xn = norm_of(x, nw, BF16)
    hb = rt.alloc(hidden * 4 + 64)
    rt.fill(hb, F32, hidden + 16, 7.0)
    call("ammon_gate_up_swiglu", rt.handle, None, up(rt, x), up(rt, nw), BF16, EPS, a.dev, b.dev, W4, n, hidden, hb)
    got = hb.download(hidden + 16)
    want, bar = swiglu_of(xn @ a.seven.T, xn @ b.seven.T, *[gemv_bar(xn, m.seven, True) for m in (a, b)])
    close(got[None, :hidden], a.rows(want), a.rows(bar))
    assert set(got[hidden:]) == {7.0}


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("heads,kv_heads,head,n", [(6, 2, 48, 300), (36, 4, 96, 1000), (90, 9, 80, 4300)])
def test_qkv_ways(tuned, way, heads, kv_heads, head, n):
    if not takes(way, (heads + 2 * kv_heads) * head, n):
        return
    rt, seq, pos = tuned(way=way), 30, 7
    dims = [heads * head, kv_heads * head, kv_heads * head]
    weights, x = [Weights(rt, d, n, s) for d, s in zip(dims, (1, 11, 21))], stream(1, n)
    nw = (1 + 0.2 * oracle.normal(n, 5)).astype(np.float32)
    table = oracle.rope_table(10000.0, head, seq)
    out = [rt.alloc(d * 4) for d in dims]
    front = [rt.handle, None, up(rt, x), up(rt, nw), F32, EPS, *[m.dev for m in weights], W4, n, heads, kv_heads, head]
    call("ammon_qkv_rope", *front, *out, seq, rt.step(0, pos), up(rt, table))
    rows = [o.download((1, d)) for o, d in zip(out, dims)]
    for got, (want, bar) in zip(rows, qkv_of(norm_of(x, nw, F32), weights, table[pos:pos + 1], head, NORM)):
        close(got, want, bar)
    caches = [up(rt, np.zeros(seq * dims[1], np.float32)) for _ in "kv"]
    call("ammon_qkv_rope_store", *front, out[0], *caches, F32, seq, rt.step(0, pos), up(rt, table))
    for cache, r in zip(caches, rows[1:]):
        got = cache.download((kv_heads, seq, head))
        np.testing.assert_array_equal(got[:, pos], r.reshape(kv_heads, head))
        assert not np.delete(got, pos, 1).any()


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("vocab,dim", [(5, 64), (1030, 1000), (9001, 5000), (100003, 300)])
def test_greedy_ways(tuned, way, vocab, dim):
    rt = tuned(way=way)
    if not takes(way, vocab, dim):
        return
    w, x = Panels(rt, vocab, dim), stream(1, dim)
    nw = (1 + 0.2 * oracle.normal(dim, 5)).astype(np.float32)
    xn, logits = norm_of(x, nw, F32), rt.alloc(vocab * 4)
    size = int(lib.ammon_greedy_lm_head_scratch_bytes(rt.handle))
    scratch, tokens, step = rt.alloc(size), rt.upload(np.full(8, -1, np.int32)), rt.step(3, 4)
    call("ammon_greedy_lm_head", rt.handle, None, up(rt, x), up(rt, nw), F32, EPS, w.dev, W4, vocab, dim, logits,
         scratch, size, None, 0, step, tokens, 8)
    got = logits.download(vocab)
    close(got[None], w.rows(xn @ w.seven.T), w.rows(gemv_bar(xn, w.seven, True)))
    assert rt.read_step(step) == (int(np.argmax(got)), 5)


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("d,n", [(70, 300), (600, 4000), (4200, 4300)])
@pytest.mark.parametrize("size", [2.0**-24, 2.0**-15, 2.0**-7])
def test_the_lower_digits_of_a_token(tuned, way, d, n, size):
    """As for rows: with a result that is in the lower digits alone, a lost digit shows.  x's numbers
    are 2^-30.98 of 1 off, 2^-6.98 of those of 2^-24."""
    if not takes(way, d, n):
        return
    rt = tuned(way=way)
    w, x = lower(rt, 112, n, size)
    panels, one = -(-d // 16), w.bytes.size // 7
    dev, y = up(rt, np.resize(w.bytes.reshape(7, one), (panels, one))), rt.alloc(4 * d)
    call("ammon_gemv", rt.handle, None, dev, W4, d, n, up(rt, x), y, None)
    a, b = x[:, keep(n)].astype(np.float64), w.numbers[:, keep(n)]
    half = 2.0**-30.98 * b.sum(-1)  # (every block's largest number is 1)
    bar = 7 * w4.product_bar(a, b, True) + half  # (a small number's digits may be 7 times as large)
    want = np.resize(a @ b.T, d)
    close(y.download((1, d)), want[None], np.resize(bar, d)[None])
    assert np.all(want > 60 * np.resize(bar, d))


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("size", [2.0**-125, 2.0**-110, 2.0**-92, 2.0**90])
def test_tokens_of_any_size(tuned, way, size):
    """x's numbers are at most 2^-121 off where they are smaller than 2^-90 (the weights are some 2^30,
    so that results are normal numbers)."""
    rt, d, n = tuned(way=way), 112, 300
    w = Weights(rt, d, n, w=np.ldexp(matrix(d, n), 30))
    x = (size * np.random.default_rng(2).uniform(-1, 1, (1, n))).astype(np.float32)
    y = rt.alloc(4 * d)
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, x), y, None)
    x = x.astype(np.float64)
    bar = w4.product_bar(x, w.numbers, False) + 2.0**-121 * np.abs(w.numbers).sum(-1)
    close(y.download((1, d)), x @ w.numbers.T, bar)


@pytest.mark.parametrize("d,n,way", [(288, 288, "k8_one"), (4096, 4096, "k8_one"), (9000, 2000, "k8"),
                                     (131072, 128, "k2"), (128256, 1700, "k2"), (20, 36864, "k8_wide"),
                                     (4112, 36864, "flat"), (4096, 14336, "flat"), (131072, 200, "flat"),
                                     (9000, 8192, "flat"), (60000, 4096, "k8"), (57344, 8192, "k8")])
def test_the_rule_takes_the_way(tuned, rt, d, n, way):
    """At 256 compute units: bit for bit the way named, and right."""
    w, x = Panels(rt, d, n), stream(1, n)
    y, z = rt.alloc(d * 4), rt.alloc(d * 4)
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, x), y, None)
    tuned(way=way)
    call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, x), z, None)
    got = y.download((1, d))
    np.testing.assert_array_equal(got, z.download((1, d)))
    close(got, w.rows(x.astype(np.float64) @ w.seven.T), w.rows(w4.product_bar(x, w.seven, False)))


def test_names_that_are_none(tuned, rt):
    """Refused, and what was chosen stays."""
    tuned("long/2", "flat")
    for tile, way, match in (("t17", None, "no tile"), ("", None, "no tile"), ("/2", None, "no tile"),
                             ("long/3", None, "ranges"), ("long/", None, "ranges"), ("long/16", None, "ranges"),
                             (None, "k3", "no way"), ("t16", "", "no way")):
        with pytest.raises(AmmonError, match=match):
            tuned(tile, way)
    w, x = Weights(rt, 40, 300), Rows(rt, stream(5, 300), Q8)
    with pytest.raises(AmmonError, match="does not take"):  # (3 groups are not split)
        gemm(rt, w.dev, 40, 300, x.dev, Q8, 5, ws=workspace(rt, 40, 5))
    for tile, dtype in (("t16_x2", Q8), ("t32_x2", Q24)):
        tuned(tile)
        with pytest.raises(AmmonError, match="does not take"):
            gemm(rt, w.dev, 40, 300, x.dev if dtype == Q8 else Rows(rt, stream(5, 300), Q24).dev, dtype, 5)
    tuned("t16_deep")
    hb = rt.alloc(5 * 40 * 4)
    with pytest.raises(AmmonError, match="does not take"):
        call("ammon_prefill_gate_up_swiglu_w4", rt.handle, None, x.dev, Q8, 5, w.dev, w.dev, 300, 40, hb)
