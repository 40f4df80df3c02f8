"""4-bit weights in the model: decode steps, prompt prefill, the greedy loops and checkpoints.

The model is compared with a float64 forward over the numbers that the W4 matrices stand for, with
attention over the device's own caches (so that a rounding of a cached row is on both sides).
Logits, normwise: every product is fp32-grade, 1e-5 x the two or three layers' amplification: 1e-4.
"""
import ctypes
import dataclasses

import numpy as np
import pytest

import oracle
from ammon_amd import AmmonError, LlamaModel, _abi
from ammon_amd._abi import BF16, F32, KV4, W4, call
from oracle import kv4, llama2c, w4

pytestmark = pytest.mark.gpu
TOL = 1e-4


def Config(**kw):
    return oracle.LlamaConfig(**dict(dict(w_dtype=W4, kv_dtype=F32), **kw))


CONFIGS = {
    "gqa64": Config(dim=512, n_layers=2, n_heads=8, n_kv_heads=2, hidden=640, vocab=400, max_seq=700),
    "mha48_kv4": Config(dim=288, n_layers=3, n_heads=6, n_kv_heads=6, hidden=768, vocab=500, max_seq=256,
                        kv_dtype=KV4),
    "gqa128_bf16": Config(dim=512, n_layers=2, n_heads=4, n_kv_heads=1, hidden=500, vocab=301, max_seq=900,
                          kv_dtype=BF16),
    # widths that are no multiple of a group or a panel
    "odd": Config(dim=80, n_layers=2, n_heads=5, n_kv_heads=5, hidden=107, vocab=77, max_seq=120),
}


def weights_of(c, seed=7):
    """fp32 weights as given, and the numbers that a W4 model has in their place."""
    given = oracle.random_weights(dataclasses.replace(c, w_dtype=F32), seed=seed, std=0.06)
    numbers = {}
    for name, a in given.items():
        a = np.asarray(a, np.float32)
        if name.startswith("rms"):
            numbers[name] = a.astype(np.float64)
        elif name == "tok_emb":
            numbers[name] = oracle.from_bf16(oracle.to_bf16(a)).astype(np.float64)
        else:
            m = a.reshape(-1, a.shape[-1])
            numbers[name] = w4.w4_numbers(*w4.w4_quantise(m), a.shape[-1]).reshape(a.shape)
    return given, numbers


def norm(x, w, eps):
    return w * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)


def forward(c, g, ids, first, caches):
    """Logits [n, vocab] in float64 of ids at positions first.., and the key and value rows [layer];
    attention over `caches` [layer][k, v] [>= first + n, kv_heads, head]."""
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
        rows.append([rotate((xn @ g["wk"][l].T).reshape(n, -1, head)), (xn @ g["wv"][l].T).reshape(n, -1, head)])
        k, v = (t.astype(np.float64).transpose(1, 0, 2) for t in caches[l])
        x = x + kv4.attention(q, k, v, first).reshape(n, -1) @ g["wo"][l].T
        xn = norm(x, g["rms_ffn"][l], c.eps)
        a = xn @ g["w1"][l].T
        x = x + (a / (1 + np.exp(-a)) * (xn @ g["w3"][l].T)) @ g["w2"][l].T
    return norm(x, g["rms_final"], c.eps) @ g["wcls"].T, rows


def rel(got, want):
    return np.max(np.abs(got - want)) / np.max(np.abs(want))


def caches_of(m, c):
    out = [m.kv_layer(l) for l in range(c.n_layers)]
    return [[oracle.from_bf16(t) if c.kv_dtype == BF16 else t for t in kv] for kv in out]


def rows_close(c, got, want):
    """Cached rows against the forward's: fp32-grade, bf16 rounded, or half a step of a group of 32."""
    bar = {F32: 1e-5, BF16: 2.0**-8 + 1e-5, KV4: 0}[c.kv_dtype] * np.max(np.abs(want))
    if c.kv_dtype == KV4:  # (the range of a group over 15, and fp16 roundings)
        bar = (0.5 + 15 * 2.0**-11) * 2 * np.max(np.abs(want)) / 15 + 3 * 2.0**-11 * np.max(np.abs(want))
    assert np.max(np.abs(got - want)) <= bar


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("use_graph", [True, False])
def test_steps(rt, name, use_graph):
    c = CONFIGS[name]
    given, g = weights_of(c)
    m = LlamaModel.from_host(rt, c, given, use_graph=use_graph)
    ids = np.random.default_rng(3).integers(0, c.vocab, 24)
    got = [m.step(int(t), p) for p, t in enumerate(ids)]
    caches = caches_of(m, c)
    want, rows = forward(c, g, ids, 0, caches)
    for p in range(len(ids)):
        assert rel(got[p], want[p]) <= TOL, p
    for kv, r in zip(caches, rows):
        for a, b in zip(kv, r):
            rows_close(c, a[:len(ids)].astype(np.float64), b)
    m.close()


@pytest.mark.parametrize("name", CONFIGS)
@pytest.mark.parametrize("n,start", [(1, 0), (2, 5), (33, 0), (90, 20), (400, 150)])
def test_prefill(rt, name, n, start):
    c = CONFIGS[name]
    n = min(n, c.max_seq - start)
    if n <= 0:
        pytest.skip("the cache is shorter")
    given, g = weights_of(c)
    m = LlamaModel.from_host(rt, c, given)
    ids = np.random.default_rng(5).integers(0, c.vocab, start + n)
    if start:
        m.prefill(ids[:start], 0)
    logits = m.prefill(ids[start:], start)
    caches = caches_of(m, c)
    want, rows = forward(c, g, ids[start:], start, caches)
    assert rel(logits, want[-1]) <= TOL
    for kv, r in zip(caches, rows):
        for a, b in zip(kv, r):
            rows_close(c, a[start:start + n].astype(np.float64), b)
    m.close()


def test_a_shorter_prefill_after_a_longer_one(rt):
    c = CONFIGS["gqa64"]
    given, _ = weights_of(c)
    ids = np.random.default_rng(6).integers(0, c.vocab, 300)
    m, fresh = LlamaModel.from_host(rt, c, given), LlamaModel.from_host(rt, c, given)
    m.prefill(ids, 0)
    np.testing.assert_array_equal(m.prefill(ids[:13], 0), fresh.prefill(ids[:13], 0))
    np.testing.assert_array_equal(m.step(7, 13), fresh.step(7, 13))
    m.close()
    fresh.close()


@pytest.mark.parametrize("name", ["gqa64", "mha48_kv4"])
def test_greedy_loops(rt, name):
    c = CONFIGS[name]
    given, _ = weights_of(c)
    m = LlamaModel.from_host(rt, c, given)
    prompt = [3, 9, 27, 81]
    host, logits_h, _ = m.generate_tokens(prompt, 40)
    device, logits_d, _ = m.generate_tokens_device(prompt, 40)
    np.testing.assert_array_equal(host, device)
    np.testing.assert_array_equal(logits_h, logits_d)
    pre, _, _ = m.generate_tokens_prefill(prompt, 40)
    assert len(pre) == len(host) and list(pre[:3]) == list(host[:3])  # (the forced ones)
    m.close()


def test_launches_are_the_other_weights(rt):
    c = CONFIGS["gqa64"]
    given, _ = weights_of(c)
    m = LlamaModel.from_host(rt, c, given)
    n = LlamaModel.from_host(rt, dataclasses.replace(c, w_dtype=F32), given)
    assert m.launches == n.launches
    m.close()
    n.close()


@pytest.mark.parametrize("version", [0, 1])
@pytest.mark.parametrize("shared", [False, True])
def test_checkpoint(rt, tmp_path, version, shared):
    c = dataclasses.replace(CONFIGS["gqa64"], max_seq=40)
    given, _ = weights_of(c, seed=11)
    if shared:
        given["wcls"] = given["tok_emb"].copy()
    path = tmp_path / "m.bin"
    llama2c.write(path, dataclasses.replace(c, w_dtype=F32), given, version=version, shared=shared)
    loaded = LlamaModel.from_checkpoint(rt, str(path), w_dtype=W4)
    assert loaded.cfg.w_dtype == W4
    direct = LlamaModel.from_host(rt, dataclasses.replace(c, theta=10000.0), given)
    for pos, tok in enumerate([1, 399, 37, 37, 5]):
        np.testing.assert_array_equal(loaded.step(tok, pos), direct.step(tok, pos))
    np.testing.assert_array_equal(loaded.prefill([4, 5, 6], 5), direct.prefill([4, 5, 6], 5))
    loaded.close()
    direct.close()


def test_synthetic_and_bf16_weights(rt):
    c = CONFIGS["odd"]
    m = LlamaModel.synthetic(rt, c, seed=3)
    assert np.isfinite(m.step(1, 0)).all() and np.abs(m.step(1, 0)).max() > 0
    m.close()
    given, _ = weights_of(c)
    bf = {k: a if k.startswith("rms") else oracle.to_bf16(a).reshape(a.shape) for k, a in given.items()}
    wide = {k: a if k.startswith("rms") else oracle.from_bf16(oracle.to_bf16(a)).reshape(a.shape)
            for k, a in given.items()}
    a, b = LlamaModel.from_host(rt, c, bf), LlamaModel.from_host(rt, c, wide)
    np.testing.assert_array_equal(a.step(2, 0), b.step(2, 0))
    a.close()
    b.close()


def test_rows_that_no_panel_begins_are_refused(rt):
    c = Config(dim=40, n_layers=1, n_heads=5, n_kv_heads=5, hidden=64, vocab=20, max_seq=16)
    given, _ = weights_of(c)
    with pytest.raises(AmmonError, match="multiple of 16"):
        LlamaModel.from_host(rt, c, given)


def test_two_streams_and_another_models_work(rt):
    """Steps of one model while another's prompt runs: their buffers and streams are their own."""
    c = CONFIGS["gqa64"]
    given, _ = weights_of(c)
    a, b = LlamaModel.from_host(rt, c, given), LlamaModel.from_host(rt, c, given)
    ids = np.random.default_rng(8).integers(0, c.vocab, 200)
    alone = [a.prefill(ids, 0).copy(), a.step(5, 200).copy()]
    a.decode(3, 0, 30)
    both = [b.prefill(ids, 0), b.step(5, 200)]
    for x, y in zip(alone, both):
        np.testing.assert_array_equal(x, y)
    a.synchronize()
    a.close()
    b.close()


def test_stream_of_ones_own(rt):
    """The entries on a stream that the runtime does not own, twice at once with buffers apart."""
    d, n = 512, 1024
    w = w4.w4_quantise(oracle.normal(d * n, 1).reshape(d, n))
    dev = rt.upload(w4.w4_pack(*w))
    xs = [rt.upload(oracle.normal(n, 20 + i)) for i in range(2)]
    ys = [rt.alloc(4 * d) for _ in range(4)]
    streams = []
    for i in range(2):
        s = ctypes.c_void_p()
        call("ammon_stream_create", rt.handle, ctypes.byref(s))
        streams.append(s)
    for _ in range(20):
        for i, s in enumerate(streams):
            call("ammon_gemv", rt.handle, s, dev, W4, d, n, xs[i], ys[i], None)
    for s in streams:
        rt.synchronize(s)
    for i in range(2):
        call("ammon_gemv", rt.handle, None, dev, W4, d, n, xs[i], ys[2 + i], None)
        np.testing.assert_array_equal(ys[i].download(d), ys[2 + i].download(d))
    for s in streams:
        call("ammon_stream_destroy", rt.handle, s)
    assert _abi.W4 == W4
