"""4-bit weights and rows of 8-bit digits without a device: sizes, refusals before a runtime is
touched, and the numpy restatement's own properties."""
import os
import subprocess

import numpy as np
import pytest

import ammon_amd
import oracle
from ammon_amd import _abi
from ammon_amd._abi import BF16, F32, KV4, Q8, Q24, W4, lib
from oracle import w4


@pytest.mark.parametrize("d,n", [(1, 1), (16, 128), (17, 129), (288, 288), (5003, 2080), (128256, 4096)])
def test_sizes(d, n):
    assert lib.ammon_w4_bytes(d, n) == w4.w4_bytes(d, n)
    for dtype, digits in ((Q8, 1), (Q24, 3)):
        assert lib.ammon_q8_bytes(dtype, d, n) == w4.q8_bytes(digits, d, n)
    for dtype in (F32, BF16, KV4, W4, 8):
        assert lib.ammon_q8_bytes(dtype, d, n) == 0
    assert lib.ammon_w4_bytes(1 << 20, 1 << 20) == (1 << 16) * (1 << 13) * 1056  # past 32 bits
    for dtype in (W4, Q8, Q24):
        assert lib.ammon_kv_cache_bytes(dtype, 1, 1, 1) == 0


def test_calls_without_a_runtime_are_refused():
    z = None
    for st in (lib.ammon_w4_store(z, z, z, F32, 1, 1, z), lib.ammon_w4_load(z, z, z, 1, 1, z, F32),
               lib.ammon_q8_store(z, z, z, 1, 1, z, Q8), lib.ammon_q8_load(z, z, z, Q8, 1, 1, z),
               lib.ammon_rmsnorm_q8(z, z, z, z, z, z, F32, 1e-5, 1, 1, z, Q8),
               lib.ammon_prefill_gemm_w4(z, z, z, 1, 1, z, Q8, 1, z, z, z, 0),
               lib.ammon_prefill_gate_up_swiglu_w4(z, z, z, Q8, 1, z, z, 1, 1, z),
               lib.ammon_prefill_qkv_rope_w4(z, z, z, Q8, 1, z, z, z, 1, 1, 1, 16, z, z, z, 1, z, z, z, 0),
               lib.ammon_prefill_qkv_rope_store_w4(z, z, z, Q8, 1, z, z, z, 1, 1, 1, 16, z, z, z, F32, 1,
                                                   z, z, z, 0)):
        assert st == _abi.E_VALIDATION
        assert "runtime" in _abi.last_error()
    assert (ammon_amd.W4, ammon_amd.Q8, ammon_amd.Q24) == (W4, Q8, Q24)


@pytest.mark.parametrize("n", [1, 127, 128, 300])
def test_w4_is_within_half_a_step(n):
    w = oracle.normal(40 * n, 3).reshape(40, n)
    codes, s = w4.w4_quantise(w)
    assert np.abs(codes).max() <= 7
    step = np.repeat(s, 128, 1)[:, :n]
    # half a step; a scale rounded down by 2^-9 leaves the largest number 7 / 2^9 of one short
    assert np.all(np.abs(w4.w4_numbers(codes, s, n) - w) <= 0.515 * step)


@pytest.mark.parametrize("digits", [1, 3])
@pytest.mark.parametrize("scale", [1.0, 1e-30, 1e30])
def test_digits_are_within_half_a_step(digits, scale):
    x = (oracle.normal(20 * 300, 4).reshape(20, 300) * np.float32(scale)).astype(np.float32)
    q, s = w4.q_quantise(x, digits)
    assert np.abs(q).max() <= (127 if digits == 1 else 127 * 65536)
    step = np.repeat(s, 128, 1)[:, :300]
    # (Q8: the reciprocal and the product round, 2 x 127 x 2^-24 of a step)
    assert np.all(np.abs(w4.q_numbers(q, s, 300) - x) <= 0.50004 * step)
    if digits == 3 and scale == 1.0:
        top = np.repeat(np.abs(w4.blocks(x)).max(-1), 128, 1)[:, :300]
        assert np.all(0.5 * step <= 2.0**-22.98 * top)


def test_rows_that_are_not_finite_or_tiny():
    x = np.zeros((4, 256), np.float32)
    x[0, 3], x[1, 200], x[2, 5], x[3, 6] = np.nan, -np.inf, 1e-40, 3e38
    for digits in (1, 3):
        q, s = w4.q_quantise(x, digits)
        assert np.isnan(s[0, 0]) and np.isnan(s[1, 1]) and np.isfinite(s[2:]).all()
        assert not q[:2].any() and not q[2].any() and q[3].any()
    codes, s = w4.w4_quantise(x)
    assert np.isnan(s[0, 0]) and np.isnan(s[1, 1]) and not s[2].any() and np.isfinite(s[3]).all()


def run_cpp(*tests):
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "_bin", "w4_test")
    if not os.path.exists(path):
        pytest.fail(f"{path} is not built (run __graft_entry__.build())")
    r = subprocess.run([path, *tests], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 failed" in r.stdout, r.stdout + r.stderr


def test_cpp_shapes():
    run_cpp("storage_bytes_of_w4", "views_of_w4")


@pytest.mark.gpu
def test_cpp_linear():
    run_cpp("linear_over_w4")
