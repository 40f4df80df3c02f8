"""Rows of digits and matrices where the tests by size leave off: rows longer than a workgroup keeps in
registers (16384 numbers), reductions past 65536, numbers at any address."""
import numpy as np
import pytest

import oracle
from ammon_amd._abi import BF16, F32, Q8, Q24, call
from oracle import w4
from test_gpu_w4 import DIGITS, EPS, Rows, Weights, close, matrix, stream, up
from test_gpu_w4_edges import shifted
from test_gpu_w4_variants import gemm, tuned  # noqa: F401

pytestmark = pytest.mark.gpu
LONG = [(3, 16384), (2, 16385), (3, 20000), (2, 28672), (17, 28700), (1, 70001)]


def rows_of(x, digits, fill=0x5a):
    before = np.full(w4.q8_bytes(digits, *x.shape) + 64, fill, np.uint8)
    want = before.copy()
    want[:-64] = w4.q_pack(*w4.q_quantise(x, digits), digits, into=before[:-64])
    return before, want


@pytest.mark.parametrize("t,n", LONG)
@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_long_rows(rt, t, n, dtype):
    x, digits = stream(t, n), DIGITS[dtype]
    before, want = rows_of(x, digits)
    out, back = up(rt, before), rt.alloc(x.nbytes)
    call("ammon_q8_store", rt.handle, None, up(rt, x), t, n, out, dtype)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)
    call("ammon_q8_load", rt.handle, None, out, dtype, t, n, back)
    np.testing.assert_array_equal(back.download(x.shape), w4.q_numbers(*w4.q_quantise(x, digits), n).astype(np.float32))


@pytest.mark.parametrize("t,n", LONG)
@pytest.mark.parametrize("dtype", [Q8, Q24])
@pytest.mark.parametrize("wdt,into", [(F32, "new"), (BF16, "x"), (F32, "residual"), (BF16, None)])
def test_long_rows_normed(rt, t, n, dtype, wdt, into):
    x, r = stream(t, n), stream(t, n, 7)
    w = oracle.storage(1 + 0.2 * oracle.normal(n, 5), wdt)
    h = x + r if into else x
    before, want = rows_of(w4.normed(h, oracle.widen(w, wdt), EPS).astype(np.float32), DIGITS[dtype])
    out, dx, dr = up(rt, before), up(rt, x), up(rt, r) if into else None
    ds = {"new": rt.alloc(x.nbytes), "x": dx, "residual": dr, None: None}[into]
    call("ammon_rmsnorm_q8", rt.handle, None, dx, dr, ds, up(rt, w), wdt, EPS, t, n, out, dtype)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)
    if into:
        np.testing.assert_array_equal(ds.download(x.shape), h)


@pytest.mark.parametrize("t,n", [(3, 300), (18, 4096), (2, 9001), (2, 20000)])
@pytest.mark.parametrize("dtype", [Q8, Q24])
@pytest.mark.parametrize("wdt,by", [(F32, 4), (BF16, 2), (BF16, 6)])
def test_rows_at_any_number(rt, t, n, dtype, wdt, by):
    x, r = stream(t, n), stream(t, n, 7)
    w = oracle.storage(1 + 0.2 * oracle.normal(n, 5), wdt)
    before, want = rows_of(w4.normed(x + r, oracle.widen(w, wdt), EPS).astype(np.float32), DIGITS[dtype])
    held = [shifted(rt, x, 4), shifted(rt, r, 12), shifted(rt, w, by)]
    out, ds = up(rt, before), rt.alloc(x.nbytes + 64)
    rt.fill(ds, F32, t * n + 16, 7.0)
    call("ammon_rmsnorm_q8", rt.handle, None, held[0][0], held[1][0], ds.offset(8), held[2][0], wdt, EPS, t, n, out, dtype)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)
    got = ds.download(t * n + 16)
    np.testing.assert_array_equal(got[2:t * n + 2].reshape(t, n), x + r)
    assert set(got[:2]) == set(got[t * n + 2:]) == {7.0}
    before, want = rows_of(x, DIGITS[dtype])
    out = up(rt, before)
    call("ammon_q8_store", rt.handle, None, held[0][0], t, n, out, dtype)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)
    rt.fill(ds, F32, t * n + 16, 7.0)
    call("ammon_q8_load", rt.handle, None, out, dtype, t, n, ds.offset(4))
    got = ds.download(t * n + 16)
    want = w4.q_numbers(*w4.q_quantise(x, DIGITS[dtype]), n).astype(np.float32)
    np.testing.assert_array_equal(got[1:t * n + 1].reshape(t, n), want)
    assert got[0] == 7.0 and set(got[t * n + 1:]) == {7.0}


@pytest.mark.parametrize("d,n", [(20, 300), (33, 129), (16, 128)])
@pytest.mark.parametrize("dtype,by", [(F32, 4), (BF16, 2), (BF16, 4)])
def test_matrices_at_any_number(rt, d, n, dtype, by):
    w = oracle.storage(matrix(d, n), dtype)
    codes, s = w4.w4_quantise(oracle.widen(w, dtype).reshape(d, n))
    want, (at, held) = w4.w4_pack(codes, s), shifted(rt, w, by)
    out = rt.alloc(want.size)
    call("ammon_w4_store", rt.handle, None, at, dtype, d, n, out)
    np.testing.assert_array_equal(out.download(want.size, np.uint8), want)
    back = rt.upload(np.full(d * n * 4 + 64, 0x5a, np.uint8))
    call("ammon_w4_load", rt.handle, None, out, d, n, back.offset(by), dtype)
    got = back.download(d * n * 4 + 64, np.uint8)
    numbers = oracle.storage(w4.w4_numbers(codes, s, n).astype(np.float32), dtype).reshape(-1).view(np.uint8)
    np.testing.assert_array_equal(got[by:by + numbers.size], numbers)
    assert set(got[:by]) == set(got[by + numbers.size:]) == {0x5a}
    del held


@pytest.mark.parametrize("dtype,tile", [(Q8, "t16"), (Q24, "t16_deep"), (Q8, "t64"), (Q24, "long"), (Q24, "long/8")])
def test_reductions_past_65536(tuned, rt, dtype, tile):  # noqa: F811
    d, n, t = 37, 70100, 5
    w, x = Weights(rt, d, n), Rows(rt, stream(t, n), dtype)
    tuned(tile)
    ws = rt.alloc(8 * t * d * 4)
    got = gemm(rt, w.dev, d, n, x.dev, dtype, t, ws=(ws, 8 * t * d * 4))
    close(got, x.numbers @ w.numbers.T, w4.product_bar(x.numbers, w.numbers, True))
