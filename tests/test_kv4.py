"""The 4-bit KV cache (AMMON_KV4) without a device: sizes, refusals before a runtime is touched,
the C++ layer's shapes, and the numpy restatement's own properties."""
import os
import subprocess

import numpy as np
import pytest

import ammon_amd
import oracle
from ammon_amd import _abi
from ammon_amd._abi import BF16, F32, KV4, lib
from oracle import kv4

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_bin", "kv4_test")


@pytest.mark.parametrize("head", [1, 31, 32, 33, 64, 80, 100, 128])
def test_cache_bytes(head):
    rows = 3 * 17
    assert lib.ammon_kv_cache_bytes(F32, 3, 17, head) == rows * head * 4
    assert lib.ammon_kv_cache_bytes(BF16, 3, 17, head) == rows * head * 2
    assert lib.ammon_kv_cache_bytes(KV4, 3, 17, head) == kv4.cache_bytes(3, 17, head)
    assert lib.ammon_kv_cache_bytes(7, 3, 17, head) == 0
    # past 32 bits
    assert lib.ammon_kv_cache_bytes(KV4, 1 << 10, 1 << 20, 128) == 80 << 30


def test_calls_without_a_runtime_are_refused():
    z = None
    assert lib.ammon_kv4_store(z, z, z, z, 1, 1, 32, z, z, 4, z) == _abi.E_VALIDATION
    assert lib.ammon_kv4_load(z, z, z, z, 1, 32, 4, 0, 1, z, z, F32) == _abi.E_VALIDATION
    assert lib.ammon_attention_partial_append(z, z, z, 1, z, z, z, z, KV4, 1, 32, 4, z, 4, z) == \
        _abi.E_VALIDATION
    assert lib.ammon_attention_decode_append(z, z, z, 1, z, z, z, z, KV4, 1, 32, 4, z, 4, z, 0, z) == \
        _abi.E_VALIDATION
    assert lib.ammon_qkv_rope(z, z, z, z, F32, 1e-5, z, z, z, F32, 32, 1, 1, 32, z, z, z, 4, z, z) == \
        _abi.E_VALIDATION
    assert lib.ammon_prefill_qkv_rope(z, z, z, 1, z, z, z, F32, 32, 1, 1, 32, z, z, z, 4, z, z, z, 0) == \
        _abi.E_VALIDATION
    assert "runtime" in _abi.last_error()
    assert ammon_amd.KV4 == KV4


def test_cpp_shapes():
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} is not built (run __graft_entry__.build())")
    r = subprocess.run([BIN, "storage_bytes_of_kv4", "views_of_kv4"], capture_output=True, text=True,
                       timeout=120)
    assert r.returncode == 0 and "0 failed" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("head", [128, 80, 33, 1])
def test_restatement_is_within_half_a_step(head):
    x = oracle.normal(200 * head, 3).reshape(200, head) * 3 + 1
    codes, s, b = kv4.quantise(x)
    assert codes.max() <= 15
    step = np.asarray(s, np.float64)[..., np.arange(head) // 32]
    # half a step; a scale rounded down by 2^-11 leaves the largest number up to 15 of that short;
    # then the bias's and the number's own rounding to fp16, of numbers below 64
    bar = (0.5 + 15 * 2.0**-11) * step + 2 * 64 * 2.0**-12
    assert np.all(np.abs(kv4.numbers(codes, s, b) - x) <= bar)


def test_restatement_of_special_groups():
    x = np.zeros((6, 64), np.float32)
    x[1] = 5.5
    x[2, 3], x[2, 40] = np.nan, 1.0
    x[3, 40] = np.inf
    x[4, :32] = 1e30 * np.where(np.arange(32) % 2, 1, -1)
    x[5] = -1e-9
    got = kv4.stored(x)
    np.testing.assert_array_equal(got[:2], x[:2])
    assert np.isnan(got[2, :32]).all() and got[2, 40] == 1.0
    assert np.isnan(got[3, 32:]).all() and not got[3, :32].any()
    assert set(np.abs(got[4, :32])) == {16384.0} or np.max(np.abs(np.abs(got[4, :32]) - 16384)) <= 16
    assert np.max(np.abs(got[5])) <= 2.0**-25 + 1e-9


def test_pack_and_read_are_inverse():
    cache = np.full(kv4.cache_bytes(3, 20, 100), 0xff, np.uint8)
    rows = oracle.normal(3 * 7 * 100, 4).reshape(3, 7, 100)
    kv4.pack(cache, 3, 20, 100, 5, rows)
    np.testing.assert_array_equal(kv4.read(cache, 3, 20, 100, 5, 7), kv4.stored(rows))
    assert np.isnan(kv4.read(cache, 3, 20, 100, 12, 8)).all()


def test_attention_restatement_against_the_oracle():
    k, v = (oracle.normal(2 * 40 * 64, s).reshape(2, 40, 64) for s in (1, 2))
    q = oracle.normal(6 * 64, 3).reshape(1, 6, 64)
    got = kv4.attention(q, k.astype(np.float64), v.astype(np.float64), 39)[0]
    for h in range(6):
        s = k[h // 3].astype(np.float64) @ q[0, h] / 8.0
        p = np.exp(s) / np.exp(s).sum()
        np.testing.assert_allclose(got[h], p @ v[h // 3], rtol=1e-12, atol=1e-12)
