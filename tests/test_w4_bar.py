"""The bar of the 4-bit weights' one-token products (oracle.w4.product_bar): x as whole numbers of four
digits lies within, with any digit lost it does not."""
import numpy as np
import pytest

import oracle
from oracle import w4


def four_digits(x):
    """x [t, n] as digits [4, t, n] times their units, as the products take them."""
    b = w4.blocks(x)
    top = np.abs(b).max(-1)
    s = np.full(top.shape, 2.0**-120)
    while (top >= 127 * 2**24 * s).any():
        s = np.where(top >= 127 * 2**24 * s, 2 * s, s)
    rest, out = np.rint(b / s[..., None]).astype(np.int64), []
    for k in range(4):
        low = (rest + 128) % 256 - 128 if k < 3 else rest
        rest = (rest - low) // 256
        out.append((low * 256.0**k * s[..., None]).reshape(len(x), -1)[:, :x.shape[1]])
    return np.stack(out)


def rows(kind, n):
    x = np.asarray(oracle.normal(3 * n, 5).reshape(3, n), np.float64)
    if kind == "stream":
        x[:, n // 3] *= 30
    if kind == "borders":  # the highest digit rounds up: sizes far above |x|
        x = np.sign(x) * (2.0**23 * 255 / 256 + 2.0**15 + 128) * 2.0**-30
        x[:, ::128] = 1.0
    return x.astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("kind", ["normal", "stream", "borders"])
@pytest.mark.parametrize("n", [100, 300, 4096])
def test_sizes_of_digits(kind, n):
    x = rows(kind, n)
    d = four_digits(x)
    top = np.abs(w4.blocks(x)).max(-1, keepdims=True)
    half = np.broadcast_to(2.0**-30.98 * top, w4.blocks(x).shape).reshape(3, -1)[:, :n]
    assert np.all(np.abs(d.sum(0) - x) <= half)
    rest = np.minimum(np.abs(w4.blocks(x)), top / 127).reshape(3, -1)[:, :n]
    assert np.all(np.abs(d).sum(0) <= np.abs(x) * (1 + 1e-6) + 6.1 * rest + half)


@pytest.mark.parametrize("lost,size", [(0, 2.0**-24), (1, 2.0**-16), (2, 2.0**-8), (3, 1.0)])
def test_a_lost_digit_is_outside(lost, size):
    n = 700
    g = np.random.default_rng(1)
    w, x = g.uniform(0.3, 1.0, (20, n)), size * g.uniform(0.5, 1.0, (2, n))
    x[:, 5::128], w[:, 5::128] = 1.0, 0.0  # a block's one large number meets zeros
    d = four_digits(x)
    want, bar = x @ w.T, w4.product_bar(x, w, False)
    assert np.all(np.abs(d.sum(0) @ w.T - want) <= bar)
    assert np.all(np.abs(np.delete(d, lost, 0).sum(0) @ w.T - want) > bar)
