"""4-bit weights as they are used together: captured products that share a workspace for their
reduction ranges, prompts of a model through each tile, a prompt against the same tokens in steps."""
import ctypes

import numpy as np
import pytest

from ammon_amd import LlamaModel
from ammon_amd._abi import BF16, F32, KV4, Q8, Q24, call, lib
from test_gpu_w4 import Rows, stream
from test_gpu_w4_model import CONFIGS, TOL, Config, caches_of, forward, rel, rows_close, weights_of
from test_gpu_w4_variants import Panels, tuned  # noqa: F401

pytestmark = pytest.mark.gpu
# its prompts of 700 tokens: QKV by 64-token tiles, gate/up by long ones, down by 64-token tiles in four ranges
WIDE = Config(dim=1280, n_layers=2, n_heads=10, n_kv_heads=2, hidden=4200, vocab=300, max_seq=760)


@pytest.mark.parametrize("dtype", [Q8, Q24])
def test_ranges_of_graphs_that_share_a_workspace(tuned, rt, dtype):  # noqa: F811
    """Two captured products whose reductions are split and an eager third, in turn on one stream over
    one workspace: each as alone, and the workspace written by each."""
    d, n, calls = 288, 8192, (("t64/8", 600), ("long/4", 333), (None, 560))
    w = Panels(rt, d, n)
    rows = [Rows(rt, stream(t, n) * (i + 1), dtype) for i, (_, t) in enumerate(calls)]
    size = max(int(lib.ammon_prefill_gemm_workspace_bytes(d, t)) for _, t in calls)
    ws, ys = rt.alloc(size), [rt.alloc(t * d * 4) for _, t in calls]
    s, graphs = ctypes.c_void_p(), []
    call("ammon_stream_create", rt.handle, ctypes.byref(s))

    def product(i):
        tuned(calls[i][0])
        call("ammon_prefill_gemm_w4", rt.handle, s, w.dev, d, n, rows[i].dev, dtype, calls[i][1], ys[i], None, ws, size)

    alone = []
    for i, (variant, t) in enumerate(calls):
        rt.fill(ws, F32, size // 4, float("nan"), stream=s)
        product(i)
        alone.append(ys[i].download(t * d, stream=s))
        used = int(variant[-1]) if variant else 8
        got = np.isnan(ws.download(size // 4, stream=s))
        assert not got[:used * t * d].any() and got[used * t * d:].all()
    for i in range(2):
        g = ctypes.c_void_p()
        call("ammon_capture_begin", rt.handle, s)
        product(i)
        call("ammon_capture_end", rt.handle, s, ctypes.byref(g))
        graphs.append(g)
    for turn in range(6):
        for y, (_, t) in zip(ys, calls):
            rt.fill(y, F32, t * d, 7.0, stream=s)
        for i in (0, 1) if turn % 2 else (1, 0):
            call("ammon_graph_launch", rt.handle, graphs[i], s)
            product(2)
        for y, (_, t), want in zip(ys, calls, alone):
            np.testing.assert_array_equal(y.download(t * d, stream=s), want)
    for g in graphs:
        call("ammon_graph_destroy", rt.handle, g)
    call("ammon_stream_destroy", rt.handle, s)


def check_prompt(rt, c, n, start, choose=None):
    given, g = weights_of(c)
    m = LlamaModel.from_host(rt, c, given)
    ids = np.random.default_rng(5).integers(0, c.vocab, start + n)
    if choose:
        choose()
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


@pytest.mark.parametrize("name,tile", [("gqa64", "t64"), ("gqa64", "long"), ("mha48_kv4", "long"), ("odd", "t64"),
                                       ("gqa128_bf16", "t16_x4"), ("gqa128_bf16", "t16_x2"), ("odd", "long")])
def test_prompts_through_a_tile(tuned, rt, name, tile):  # noqa: F811
    c = CONFIGS[name]
    check_prompt(rt, c, min(200, c.max_seq - 20), 20, lambda: tuned(tile))


@pytest.mark.parametrize("kvd", [F32, BF16, KV4])
def test_a_long_prompt(rt, kvd):
    check_prompt(rt, Config(**{**WIDE.__dict__, "kv_dtype": kvd}), 700, 45)


@pytest.mark.parametrize("c,n", [(CONFIGS["gqa64"], 40), (CONFIGS["odd"], 40), (WIDE, 60), (WIDE, 333)])
def test_a_prompt_and_its_tokens_in_steps(rt, c, n):
    """The logits behind a prompt and of five tokens after it.  Both are within TOL of the float64
    forward over their own caches; those agree within 1e-5, which weights of at most 1 pass on."""
    given, _ = weights_of(c)
    a, b = LlamaModel.from_host(rt, c, given), LlamaModel.from_host(rt, c, given)
    ids = [int(i) for i in np.random.default_rng(9).integers(0, c.vocab, n + 5)]
    for p in range(n):
        step = a.step(ids[p], p)
    assert rel(b.prefill(np.array(ids[:n]), 0), step) <= 3 * TOL
    for x, y in zip(sum(caches_of(a, c), []), sum(caches_of(b, c), [])):
        assert np.max(np.abs(x[:n] - y[:n])) <= 2e-5 * np.max(np.abs(x[:n]))
    for p in range(n, n + 5):
        assert rel(b.step(ids[p], p), a.step(ids[p], p)) <= 3 * TOL
    a.close()
    b.close()


@pytest.mark.parametrize("name", ["gqa64", "odd"])
def test_free_tokens_behind_a_prompt(rt, name):
    """Tokens generated behind a prompt taken at once and in steps: equal as long as the steps' best
    logit leads by more than what the two may differ by."""
    c = CONFIGS[name]
    given, _ = weights_of(c)
    m = LlamaModel.from_host(rt, c, given)
    prompt = [3, 9, 27, 61]
    steps, _, _ = m.generate_tokens(prompt, 30)
    whole, _, _ = m.generate_tokens_prefill(prompt, 30)
    assert len(whole) == len(steps)
    ids, free = [int(t) for t in steps], 0
    tokens = [prompt[0]] + ids
    for p, t in enumerate(ids):
        logits = np.sort(m.step(tokens[p], p))
        if p < len(prompt) - 1:  # (forced)
            assert t == int(whole[p]) == prompt[p + 1]
            continue
        if logits[-1] - logits[-2] <= 6 * TOL * np.max(np.abs(logits)):
            break
        assert int(whole[p]) == t
        free += 1
    assert free >= 5
    m.close()
