"""4-bit weights and rows of digits at the ends of their ranges: numbers at any address, ties,
graphs that share a workspace, matrices and rows past 4 GiB."""
import ctypes

import numpy as np
import pytest

import oracle
from ammon_amd._abi import BF16, COPY_D2H, COPY_H2D, F32, Q8, Q24, W4, call, lib
from oracle import w4
from test_gpu_w4 import EPS, NORM, Rows, Weights, close, matrix, norm_of, stream, up, workspace

pytestmark = pytest.mark.gpu


def shifted(rt, a, by):
    """The bytes of a, `by` bytes into a buffer; the pointer and what holds it."""
    raw = np.ascontiguousarray(a).view(np.uint8).ravel()
    buf = rt.upload(np.concatenate([np.full(by, 0xff, np.uint8), raw, np.full(16, 0xff, np.uint8)]))
    return buf.offset(by), buf


@pytest.mark.parametrize("d,n", [(40, 300), (33, 1001), (288, 4096), (4100, 8320), (6000, 9004)])
@pytest.mark.parametrize("wdt,by", [(F32, 4), (BF16, 2), (BF16, 4)])
def test_gemv_rmsnorm_at_any_number(rt, d, n, wdt, by):
    w, x = Weights(rt, d, n), stream(1, n)
    nw = oracle.storage(1 + 0.2 * oracle.normal(n, 5), wdt)
    xn = norm_of(x, nw, wdt)
    (px, bx), (pw, bw), y = shifted(rt, x, 4), shifted(rt, nw, by), rt.alloc(d * 4 + 64)
    rt.fill(y, F32, d + 16, 7.0)
    call("ammon_gemv_rmsnorm", rt.handle, None, px, pw, wdt, EPS, w.dev, W4, d, n, y.offset(12))
    got = y.download(d + 16)
    bar = w4.product_bar(xn, w.numbers, False) + NORM * np.abs(xn) @ np.abs(w.numbers).T
    close(got[3:d + 3].reshape(1, d), xn @ w.numbers.T, bar)
    assert set(got[:3]) == set(got[d + 3:]) == {7.0}
    del bx, bw


@pytest.mark.parametrize("d,n,t,dtype", [(40, 300, 5, Q24), (6144, 520, 20, Q24), (5001, 260, 33, Q8)])
def test_prefill_gemm_at_any_number(rt, d, n, t, dtype):
    w, x, r = Weights(rt, d, n), Rows(rt, stream(t, n), dtype), oracle.normal(t * d, 9)
    (pr, br), y = shifted(rt, r, 4), rt.alloc(t * d * 4 + 64)
    rt.fill(y, F32, t * d + 16, 7.0)
    call("ammon_prefill_gemm_w4", rt.handle, None, w.dev, d, n, x.dev, dtype, t, y.offset(12), pr, None, 0)
    got = y.download(t * d + 16)
    want, bar = x.numbers @ w.numbers.T, w4.product_bar(x.numbers, w.numbers, True)
    res = r.reshape(t, d).astype(np.float64)
    close(got[3:t * d + 3].reshape(t, d), want + res, bar + 2.0**-24 * np.abs(want + res))
    assert set(got[:3]) == set(got[t * d + 3:]) == {7.0}
    del br


@pytest.mark.parametrize("exact", [False, True])
@pytest.mark.parametrize("vocab,dim", [(50, 256), (5000, 256), (4800, 9000), (100001, 130)])
def test_ties_go_to_the_lowest_token(rt, vocab, dim, exact):
    """Equal rows wherever a unit, a wave, a workgroup or a round ends; NaN rows never win.  Their sums
    may be added up in another order; exact: x is ones, so that no sum rounds (m groups of 7 x 128
    times a bf16 scale: 18 bits at m = 71)."""
    w = np.abs(matrix(vocab, dim, 3)) * 0.01
    x = np.ones((1, dim), np.float32) if exact else np.abs(stream(1, dim)) + 0.1
    places = sorted({vocab - 1, vocab // 2, vocab // 2 + 1, min(vocab - 2, 4097), 33, 31})
    for p in places:
        w[p] = 1.0
    w[7, 3] = np.nan
    dev = Weights(rt, vocab, dim, w=w).dev
    logits, size = rt.alloc(vocab * 4), int(lib.ammon_greedy_lm_head_scratch_bytes(rt.handle))
    scratch, step = rt.alloc(size), rt.step(0, 0)
    args = [rt.handle, None, up(rt, x), up(rt, np.ones(dim, np.float32)), F32, EPS, dev, W4, vocab, dim, logits,
            scratch, size, None, 0, step, None, 0]
    call("ammon_greedy_lm_head", *args)
    got = logits.download(vocab)
    assert np.isnan(got[7]) and np.isfinite(np.delete(got, 7)).all()
    assert int(np.nanargmax(got)) in places
    assert rt.read_step(step) == (int(np.nanargmax(got)), 1)
    if exact:
        assert len({got[p] for p in places}) == 1 and rt.read_step(step)[0] == places[0]


def test_graphs_that_share_a_workspace(rt):
    """Two captured prompts whose reductions are split, one workspace, replayed in turn on a stream
    with eager products of a third between them: each as alone."""
    d, n, tokens = 512, 14336, (100, 130, 70)
    w = Weights(rt, d, n)
    rows = [Rows(rt, stream(t, n) * (i + 1), Q24) for i, t in enumerate(tokens)]
    size = max(int(lib.ammon_prefill_gemm_workspace_bytes(d, t)) for t in tokens)
    ws, ys = rt.alloc(size), [rt.alloc(t * d * 4) for t in tokens]
    s, graphs = ctypes.c_void_p(), []
    call("ammon_stream_create", rt.handle, ctypes.byref(s))

    def product(i, out):
        call("ammon_prefill_gemm_w4", rt.handle, s, w.dev, d, n, rows[i].dev, Q24, tokens[i], out, None, ws, size)

    alone = []
    for i, t in enumerate(tokens):
        product(i, ys[i])
        alone.append(ys[i].download(t * d, stream=s))
    for i in range(2):
        g = ctypes.c_void_p()
        call("ammon_capture_begin", rt.handle, s)
        product(i, ys[i])
        call("ammon_capture_end", rt.handle, s, ctypes.byref(g))
        graphs.append(g)
    for turn in range(6):
        for y, t in zip(ys, tokens):
            rt.fill(y, F32, t * d, 7.0, stream=s)
        for i in (0, 1) if turn % 2 else (1, 0):
            call("ammon_graph_launch", rt.handle, graphs[i], s)
            product(2, ys[2])
        for y, t, want in zip(ys, tokens, alone):
            np.testing.assert_array_equal(y.download(t * d, stream=s), want)
    for g in graphs:
        call("ammon_graph_destroy", rt.handle, g)
    call("ammon_stream_destroy", rt.handle, s)


@pytest.mark.parametrize("d", [4096, 300])
def test_one_token_in_a_graph(rt, d):
    n = 8320
    w, (x, y) = Weights(rt, d, n), (rt.alloc(4 * n), rt.alloc(4 * d))
    s, g = ctypes.c_void_p(), ctypes.c_void_p()
    call("ammon_stream_create", rt.handle, ctypes.byref(s))
    call("ammon_capture_begin", rt.handle, s)
    call("ammon_gemv", rt.handle, s, w.dev, W4, d, n, x, y, y)
    call("ammon_capture_end", rt.handle, s, ctypes.byref(g))
    other = rt.alloc(4 * d)
    for turn in range(4):
        row = stream(1, n, 30 + turn)
        x.upload(row, stream=s)
        y.upload(np.zeros(d, np.float32), stream=s)
        call("ammon_graph_launch", rt.handle, g, s)
        got = y.download(d, stream=s)
        call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, up(rt, row), other, None)
        np.testing.assert_array_equal(got, other.download(d))
    call("ammon_graph_destroy", rt.handle, g)
    call("ammon_stream_destroy", rt.handle, s)


def test_a_matrix_past_4_gib(rt):
    """Zeros but for panels at its start and end; every product reads both."""
    n, d = 14336, 600 * 1024
    assert int(lib.ammon_w4_bytes(d, n)) > 2**32
    big = rt.alloc(int(lib.ammon_w4_bytes(d, n)))
    rt.fill(big, F32, big.nbytes // 4, 0.0)
    rt.synchronize()
    first, last = Weights(rt, 16, n, 1), Weights(rt, 16, n, 2)
    for part, at in ((first, 0), (last, big.nbytes - first.bytes.size)):
        call("ammon_memcpy", rt.handle, big.offset(at), part.bytes.ctypes.data, part.bytes.size, COPY_H2D, None)
    rt.synchronize()
    x = stream(1, n)
    dx, y = up(rt, x), rt.alloc(4 * d)

    def compare(got, run):
        for part, sl in ((first, slice(0, 16)), (last, slice(d - 16, d))):
            want, bar = run(part)
            close(got[..., sl], want, bar)
        assert not got[..., 16:d - 16].any()

    call("ammon_gemv", rt.handle, None, big, W4, d, n, dx, y, None)
    compare(y.download((1, d)), lambda m: (x.astype(np.float64) @ m.numbers.T, w4.product_bar(x, m.numbers, False)))
    for t in (3, 40):
        rows = Rows(rt, stream(t, n), Q8)
        out = rt.alloc(4 * t * d)
        call("ammon_prefill_gemm_w4", rt.handle, None, big, d, n, rows.dev, Q8, t, out, None, None, 0)
        compare(out.download((t, d)),
                lambda m: (rows.numbers @ m.numbers.T, w4.product_bar(rows.numbers, m.numbers, True)))


def test_rows_past_4_gib(rt):
    n, t = 14336, 110000
    size = int(lib.ammon_q8_bytes(Q24, t, n))
    assert size > 2**32 and t * n * 4 > 2**32
    x, q = rt.alloc(t * n * 4), rt.alloc(size)
    rt.fill(x, F32, t * n, 0.0)
    rt.synchronize()
    tail = stream(16, n)
    call("ammon_memcpy", rt.handle, x.offset((t - 16) * n * 4), tail.ctypes.data, tail.nbytes, COPY_H2D, None)
    rt.synchronize()
    call("ammon_q8_store", rt.handle, None, x, t, n, q, Q24)
    w, few, y = Weights(rt, 48, n), Rows(rt, tail, Q24), rt.alloc(t * 48 * 4)
    call("ammon_prefill_gemm_w4", rt.handle, None, w.dev, 48, n, q, Q24, t, y, None, None, 0)
    got = y.download((t, 48))
    assert not got[:t - 16].any()
    close(got[t - 16:], few.numbers @ w.numbers.T, w4.product_bar(few.numbers, w.numbers, True))
    rt.fill(x, F32, t * n, 7.0)
    call("ammon_q8_load", rt.handle, None, q, Q24, t, n, x)
    back = np.empty((17, n), np.float32)
    rt.synchronize()
    call("ammon_memcpy", rt.handle, back.ctypes.data, x.offset((t - 17) * n * 4), back.nbytes, COPY_D2H, None)
    rt.synchronize()
    assert not back[0].any()
    np.testing.assert_array_equal(back[1:], few.numbers.astype(np.float32))


@pytest.mark.parametrize("d,n", [(20, 36864), (4112, 36864), (4096, 4096), (6144, 4096), (4096, 14336), (10240, 8192),
                                 (70000, 1000), (9000, 8192), (300, 300)])
def test_the_same_in_every_call(rt, d, n):
    w, x = Weights(rt, d, n, w=matrix(64, n).repeat((d + 63) // 64, 0)[:d]), up(rt, stream(1, n))
    ys = [rt.alloc(4 * d) for _ in range(24)]
    for y in ys * 2:
        call("ammon_gemv", rt.handle, None, w.dev, W4, d, n, x, y, None)
    first = ys[0].download(d)
    for y in ys[1:]:
        np.testing.assert_array_equal(y.download(d), first)


@pytest.mark.parametrize("dtype", [Q8, Q24])
@pytest.mark.parametrize("d,n,t", [(4096, 4096, 5), (96, 14336, 5), (6144, 1024, 20), (6144, 1024, 41), (1024, 8192, 200),
                                   (3000, 1000, 600)])
def test_prompts_the_same_in_every_call(rt, d, n, t, dtype):
    w, x = Weights(rt, d, n, w=matrix(64, n).repeat((d + 63) // 64, 0)[:d]), Rows(rt, stream(t, n), dtype)
    ws, ys = workspace(rt, d, t), [rt.alloc(4 * t * d) for _ in range(8)]
    for y in ys * 2:
        call("ammon_prefill_gemm_w4", rt.handle, None, w.dev, d, n, x.dev, dtype, t, y, None, *ws)
    first = ys[0].download(t * d)
    for y in ys[1:]:
        np.testing.assert_array_equal(y.download(t * d), first)
