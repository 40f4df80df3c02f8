"""The 4-bit KV cache in the model and the blocks' launches: rows of the QKV fronts, whole decode
steps, prompt prefill, the greedy loops, refusals.

The model is compared with a float64 forward that takes the cached numbers from the device's own
cache, so that both sides attend to the same numbers: a code at a border may go either way when
its row differs by fp32 summation order.  The rows themselves are then compared with the forward's
own, before quantising: half a step and what is said at the bar below.  Logits, normwise: 1e-5 x
the two or three layers' amplification, 1e-4.
"""
import dataclasses
import os
import subprocess

import numpy as np
import pytest

import oracle
from ammon_amd import AmmonError, LlamaModel, _abi
from ammon_amd._abi import BF16, F32, KV4, call, lib
from oracle import kv4

pytestmark = pytest.mark.gpu
LOGITS_TOL = 1e-4


def Config(**kw):
    return oracle.LlamaConfig(**dict(dict(w_dtype=F32, kv_dtype=KV4), **kw))


CONFIGS = {
    "gqa64": Config(dim=512, n_layers=2, n_heads=8, n_kv_heads=2, hidden=640, vocab=400, max_seq=700),
    "mha48": Config(dim=288, n_layers=3, n_heads=6, n_kv_heads=6, hidden=768, vocab=500, max_seq=256),
    "gqa128_bf16": Config(dim=512, n_layers=2, n_heads=4, n_kv_heads=1, hidden=512, vocab=300,
                          max_seq=1500, w_dtype=BF16),
    # a layer's cache is 255 rows of 20 bytes: no multiple of 16
    "odd_cache": Config(dim=64, n_layers=3, n_heads=2, n_kv_heads=1, hidden=96, vocab=100, max_seq=255),
}


def weights_of(c, seed=7):
    return oracle.random_weights(c, seed=seed, std=0.06)


def norm(x, w, eps):
    return np.asarray(w, np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def forward(c, w, ids, first, caches):
    """Logits [n, vocab] in float64 of ids at positions first.., and the rows [layer][k, v] [n,
    kv_heads, head] before quantising; attention over `caches` [layer][k, v] [>= first + n,
    kv_heads, head]."""
    g = {n: np.asarray(oracle.widen(w[n], c.w_dtype if not n.startswith("rms") else F32), np.float64)
         for n in w}
    head = c.dim // c.n_heads
    table = oracle.rope_table(c.theta, head, c.max_seq).astype(np.float64)
    n = len(ids)

    def rotate(x):
        cs, out = table[first:first + n][:, None], np.empty_like(x)
        a, b = x[..., 0::2], x[..., 1::2]
        out[..., 0::2] = a * cs[..., 0] - b * cs[..., 1]
        out[..., 1::2] = a * cs[..., 1] + b * cs[..., 0]
        return out

    x, rows = g["tok_emb"][np.asarray(ids)], []
    for l in range(c.n_layers):
        xn = norm(x, g["rms_att"][l], c.eps)
        q = rotate((xn @ g["wq"][l].T).reshape(n, -1, head))
        rows.append([rotate((xn @ g["wk"][l].T).reshape(n, -1, head)),
                     (xn @ g["wv"][l].T).reshape(n, -1, head)])
        k, v = (t.astype(np.float64).transpose(1, 0, 2) for t in caches[l])
        x = x + kv4.attention(q, k, v, first).reshape(n, -1) @ g["wo"][l].T
        xn = norm(x, g["rms_ffn"][l], c.eps)
        a = xn @ g["w1"][l].T
        x = x + (a / (1 + np.exp(-a)) * (xn @ g["w3"][l].T)) @ g["w2"][l].T
    return norm(x, g["rms_final"], c.eps) @ g["wcls"].T, rows


def rows_close(got, want):
    """Stored numbers against the rows before quantising: half a step of the group, 15 roundings
    of the scale (2^-11), fp16 roundings of bias and number, and the row's own 1e-5."""
    head = want.shape[-1]
    for j in range(0, head, 32):
        y = want[..., j:j + 32]
        step = (y.max(-1, keepdims=True) - y.min(-1, keepdims=True)) / 15
        size = np.abs(y).max()
        bar = (0.5 + 15 * 2.0**-11 + 1e-3) * step + 3 * 2.0**-11 * size + 1e-5 * np.abs(want).max()
        assert np.all(np.abs(got[..., j:j + 32] - y) <= bar)


def rel(got, want):
    return np.max(np.abs(got - want)) / np.max(np.abs(want))


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("use_graph", [True, False])
def test_steps(rt, name, use_graph):
    c, w = CONFIGS[name], weights_of(CONFIGS[name])
    m = LlamaModel.from_host(rt, c, w, use_graph=use_graph)
    ids = np.random.default_rng(3).integers(0, c.vocab, 40)
    got = [m.step(int(t), p) for p, t in enumerate(ids)]
    caches = [m.kv_layer(l) for l in range(c.n_layers)]
    want, rows = forward(c, w, ids, 0, caches)
    for p in range(len(ids)):
        assert rel(got[p], want[p]) <= LOGITS_TOL, p
    for l in range(c.n_layers):
        for got_rows, want_rows in zip(caches[l], rows[l]):
            rows_close(got_rows[:40].astype(np.float64), want_rows)
            assert not got_rows[40:].any()  # the cache starts as zeros
    m.close()


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("n,start", [(1, 0), (33, 0), (130, 60), (500, 150)])
def test_prefill(rt, name, n, start):
    c, w = CONFIGS[name], weights_of(CONFIGS[name])
    if (c.dim // c.n_heads) % 16 or start + n > c.max_seq:
        n = c.max_seq - start
    m = LlamaModel.from_host(rt, c, w)
    ids = np.random.default_rng(5).integers(0, c.vocab, start + n)
    if start:
        m.prefill(ids[:start], 0)
        before = [m.kv_layer(l) for l in range(c.n_layers)]
    logits = m.prefill(ids[start:], start)
    caches = [m.kv_layer(l) for l in range(c.n_layers)]
    want, rows = forward(c, w, ids[start:], start, caches)
    assert rel(logits, want[-1]) <= LOGITS_TOL
    for l in range(c.n_layers):
        for i in range(2):
            rows_close(caches[l][i][start:start + n].astype(np.float64), rows[l][i])
            assert not caches[l][i][start + n:].any()
            if start:
                np.testing.assert_array_equal(caches[l][i][:start], before[l][i][:start])
    # ... and decode goes on from it
    if start + n < c.max_seq:
        got = m.step(int(ids[0]), start + n)
        caches = [m.kv_layer(l) for l in range(c.n_layers)]
        want, _ = forward(c, w, ids[:1], start + n, caches)
        assert rel(got, want[0]) <= LOGITS_TOL
    m.close()


@pytest.mark.parametrize("name", CONFIGS)
def test_greedy_loops_agree(rt, name):
    c, w = CONFIGS[name], weights_of(CONFIGS[name])
    a = LlamaModel.from_host(rt, c, w)
    b = LlamaModel.from_host(rt, c, w)
    prompt = [3, 17, 99, 5, 42]
    host, logits_h, _ = a.generate_tokens(prompt, 60)
    device, logits_d, _ = b.generate_tokens_device(prompt, 60)
    np.testing.assert_array_equal(host, device)
    np.testing.assert_array_equal(logits_h, logits_d)
    for l in range(c.n_layers):
        for x, y in zip(a.kv_layer(l), b.kv_layer(l)):
            np.testing.assert_array_equal(x, y)
    pre, _, _ = b.generate_tokens_prefill(prompt, 60)
    assert len(pre) == len(host) and list(pre[:4]) == list(host[:4])  # (the forced ones)
    a.close()
    b.close()


def test_launches_are_the_other_caches(rt):
    c = CONFIGS["mha48"]
    w = weights_of(c)
    m = LlamaModel.from_host(rt, c, w)
    n = LlamaModel.from_host(rt, dataclasses.replace(c, kv_dtype=F32), w)
    assert m.launches == n.launches
    m.close()
    n.close()


# ---- the QKV fronts' rows -----------------------------------------------------------------------
def up(rt, a):
    return rt.upload(np.ascontiguousarray(a))


@pytest.mark.parametrize("w_dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv_heads,head,dim", [(8, 2, 64, 512), (6, 6, 48, 288), (4, 1, 128, 300)])
def test_qkv_rows_are_the_cache_rows(rt, heads, kv_heads, head, dim, w_dtype):
    seq, pos = 40, 17
    q_dim, kv_dim = heads * head, kv_heads * head
    std = oracle.storage
    wq, wk, wv = (up(rt, std(oracle.normal(r * dim, s, std=0.05), w_dtype)) for r, s in
                  ((q_dim, 1), (kv_dim, 2), (kv_dim, 3)))
    x, nw = up(rt, oracle.normal(dim, 4)), up(rt, oracle.normal(dim, 5, mean=1.0, std=0.1))
    table = up(rt, oracle.rope_table(10000.0, head, seq))
    q1, q2 = (rt.alloc(q_dim * 4) for _ in "qq")
    kc, vc = (rt.alloc(kv_heads * seq * head * 4) for _ in "kv")
    k, v = (rt.alloc(kv_dim * 4 + 16) for _ in "kv")
    for buf in (k, v):
        rt.fill(buf, F32, kv_dim + 4, 7.0)
    step = rt.step(0, pos)
    front = (rt.handle, None, x, nw, F32, 1e-5, wq, wk, wv, w_dtype, dim, heads, kv_heads, head)
    call("ammon_qkv_rope_store", *front, q1, kc, vc, F32, seq, step, table)
    call("ammon_qkv_rope", *front, q2, k, v, seq, step, table)
    np.testing.assert_array_equal(q1.download(q_dim), q2.download(q_dim))
    for cache, rows in ((kc, k), (vc, v)):
        got = rows.download(kv_dim + 4)
        np.testing.assert_array_equal(got[:kv_dim].reshape(kv_heads, head),
                                      cache.download((kv_heads, seq, head))[:, pos])
        assert np.all(got[kv_dim:] == 7.0)
    call("ammon_qkv_rope", *front, q2, k, v, seq, rt.step(0, seq), table)
    for buf, n in ((q2, q_dim), (k, kv_dim), (v, kv_dim)):
        assert np.isnan(buf.download(n)).all()
    assert np.all(k.download(kv_dim + 4)[kv_dim:] == 7.0)


@pytest.mark.parametrize("w_dtype", [F32, BF16])
@pytest.mark.parametrize("tokens", [1, 9, 40, 200])
@pytest.mark.parametrize("ws", [False, True])
def test_prefill_qkv_rows_are_the_cache_rows(rt, tokens, w_dtype, ws):
    heads, kv_heads, head, dim, seq, pos = 8, 2, 64, 1024, 300, 30
    q_dim, kv_dim = heads * head, kv_heads * head
    wq, wk, wv = (up(rt, oracle.storage(oracle.normal(r * dim, s, std=0.05), w_dtype)) for r, s in
                  ((q_dim, 1), (kv_dim, 2), (kv_dim, 3)))
    x = up(rt, oracle.normal(tokens * dim, 4))
    table = up(rt, oracle.rope_table(10000.0, head, seq))
    q1, q2 = (rt.alloc(tokens * q_dim * 4) for _ in "qq")
    kc, vc = (rt.alloc(kv_heads * seq * head * 4) for _ in "kv")
    k, v = (rt.alloc(tokens * kv_dim * 4 + 16) for _ in "kv")
    for buf in (k, v):
        rt.fill(buf, F32, tokens * kv_dim + 4, 7.0)
    n = int(lib.ammon_prefill_gemm_workspace_bytes(q_dim + 2 * kv_dim, tokens))
    work = (rt.alloc(n), n) if ws else (None, 0)
    step = rt.step(0, pos)
    front = (rt.handle, None, x, tokens, wq, wk, wv, w_dtype, dim, heads, kv_heads, head)
    call("ammon_prefill_qkv_rope_store_ws", *front, q1, kc, vc, F32, seq, step, table, *work)
    call("ammon_prefill_qkv_rope", *front, q2, k, v, seq, step, table, *work)
    np.testing.assert_array_equal(q1.download((tokens, q_dim)), q2.download((tokens, q_dim)))
    for cache, rows in ((kc, k), (vc, v)):
        got = rows.download(tokens * kv_dim + 4)
        want = cache.download((kv_heads, seq, head))[:, pos:pos + tokens].transpose(1, 0, 2)
        np.testing.assert_array_equal(got[:-4].reshape(want.shape), want)
        assert np.all(got[-4:] == 7.0)
    # the last three tokens past the cache
    call("ammon_prefill_qkv_rope", *front, q2, k, v, seq, rt.step(0, seq - tokens + 3), table, *work)
    for buf, width in ((q2, q_dim), (k, kv_dim), (v, kv_dim)):
        got = np.isnan(buf.download((tokens, width)))
        assert got[max(tokens - 3, 0):].all() and not got[:max(tokens - 3, 0)].any()


# ---- refusals (nothing is launched: the stream only checks) ---------------------------------------
def test_refusals(rt):
    b = rt.alloc(1 << 20)  # any device memory
    at = lambda n: b.offset(n)  # noqa: E731
    step, V = rt.step(0, 0), _abi.STREAM_VALIDATE
    k, v, kc, vc = at(0), at(4096), at(65536), at(262144)

    def bad(match, name, *args):
        with pytest.raises(AmmonError, match=match) as e:
            call(name, rt.handle, V, *args)
        assert e.value.status == _abi.E_VALIDATION

    call("ammon_kv4_store", rt.handle, V, k, v, 4, 2, 64, kc, vc, 100, step)
    bad("NULL", "ammon_kv4_store", None, v, 4, 2, 64, kc, vc, 100, step)
    bad("NULL", "ammon_kv4_store", k, v, 4, 2, 64, kc, None, 100, step)
    bad("NULL", "ammon_kv4_store", k, v, 4, 2, 64, kc, vc, 100, None)
    bad("empty", "ammon_kv4_store", k, v, 4, 0, 64, kc, vc, 100, step)
    bad("empty", "ammon_kv4_store", k, v, 4, 2, 64, kc, vc, 0, step)
    bad("exceeds", "ammon_kv4_store", k, v, 4, 2, 129, kc, vc, 100, step)
    bad("aligned", "ammon_kv4_store", k, v, 4, 2, 64, at(65544), vc, 100, step)
    bad("caches overlap", "ammon_kv4_store", k, v, 4, 2, 64, kc, at(65536 + 16), 100, step)
    bad("rows overlap", "ammon_kv4_store", k, at(65536 + 64), 4, 2, 64, kc, vc, 100, step)
    bad("too many", "ammon_kv4_store", k, v, 1 << 30, 2, 64, kc, vc, 100, step)
    call("ammon_kv4_load", rt.handle, V, kc, vc, 2, 64, 100, 60, 40, k, at(32768), F32)
    bad("exceed", "ammon_kv4_load", kc, vc, 2, 64, 100, 61, 40, k, at(32768), F32)
    bad("exceed", "ammon_kv4_load", kc, vc, 2, 64, 100, 0xffffffff, 1, k, at(32768), F32)
    bad("go together", "ammon_kv4_load", kc, vc, 2, 64, 100, 0, 40, k, None, F32)
    bad("output dtype", "ammon_kv4_load", kc, vc, 2, 64, 100, 0, 40, k, at(32768), KV4)
    bad("aligned", "ammon_kv4_load", kc, vc, 2, 64, 100, 0, 40, at(8), at(32768), F32)
    bad("outputs overlap", "ammon_kv4_load", kc, vc, 2, 64, 100, 0, 40, k, at(64), F32)
    bad("overlaps a cache", "ammon_kv4_load", kc, vc, 2, 64, 100, 0, 40, k, at(65536), F32)
    part, out, q = at(524288), at(16384), at(20480)
    n = int(lib.ammon_attention_scratch_bytes(8, 64, 100, 64))
    append = lambda **kw: [kw.get("q", q), kw.get("heads", 8), kw.get("k", k), kw.get("v", v),  # noqa: E731
                           kw.get("kc", kc), kw.get("vc", vc), kw.get("dt", KV4), kw.get("kv", 2),
                           kw.get("head", 64), 100, kw.get("step", step), kw.get("split", 64), part,
                           kw.get("n", n), out]
    call("ammon_attention_decode_append", rt.handle, V, *append())
    for match, kw in (("only a KV4", dict(dt=F32)), ("only a KV4", dict(dt=BF16)), ("NULL", dict(k=None)),
                      ("NULL", dict(vc=None)), ("NULL", dict(q=None)), ("NULL", dict(step=None)),
                      ("multiple", dict(heads=7)), ("exceeds 8", dict(heads=18, n=4 * n)),
                      ("exceeds", dict(head=130, n=4 * n)), ("scratch", dict(n=n - 4)), ("split length", dict(split=2048, n=4 * n)),
                      ("aligned", dict(kc=at(65540))), ("caches overlap", dict(vc=at(65552))),
                      ("overlap a cache", dict(q=at(65536))), ("overlap a cache", dict(v=at(262144))),
                      ("overlap the output", dict(k=at(16384))), ("overlap the output", dict(v=at(524288))),
                      ("cache overlaps the output", dict(kc=at(16384 - 4096)))):
        bad(match, "ammon_attention_decode_append", *append(**kw))
    bad("aligned", "ammon_attention_decode", q, 8, at(65540), vc, KV4, 2, 64, 100, step, 64, part, n, out)
    bad("aligned", "ammon_attention_prefill", q, 3, 8, at(65540), vc, KV4, 2, 64, 100, step, 50, 64, part,
        1 << 18, at(32768))
    bad("unknown kv dtype", "ammon_attention_decode", q, 8, kc, vc, 3, 2, 64, 100, step, 64, part, n, out)
    # entries that do not take such a cache
    w, table = at(600000 // 16 * 16), at(700000 // 16 * 16)
    bad("takes rows", "ammon_qkv_rope_store", q, None, F32, 1e-5, w, w, w, F32, 64, 8, 2, 64, out, kc, vc,
        KV4, 100, step, table)
    bad("takes rows", "ammon_prefill_qkv_rope_store", q, 2, w, w, w, F32, 64, 8, 2, 64, out, kc, vc, KV4, 100,
        step, table)
    bad("in place", "ammon_rope", q, 8, 2, 64, kc, KV4, 100, step, table)
    bad("dtype", "ammon_fill", kc, KV4, 16, 0.0)
    bad("dtype", "ammon_gemv", kc, KV4, 16, 16, q, out, None)
    front = (q, None, F32, 1e-5, w, w, w, F32, 64, 8, 2, 64)
    bad("rows overlap", "ammon_qkv_rope", *front, out, k, k, 100, step, table)
    bad("overlap x or q", "ammon_qkv_rope", *front, out, out, v, 100, step, table)
    bad("8-byte", "ammon_qkv_rope", *front, out, at(4), v, 100, step, table)
    bad("NULL", "ammon_qkv_rope", *front, out, None, v, 100, step, table)
    with pytest.raises(AmmonError, match="dtype"):
        LlamaModel.from_host(rt, dataclasses.replace(CONFIGS["mha48"], kv_dtype=3),
                             weights_of(CONFIGS["mha48"]))


def test_cpp_cache(rt):
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_bin", "kv4_test")
    r = subprocess.run([path], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 failed" in r.stdout, r.stdout + r.stderr
