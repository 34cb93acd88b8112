"""The bounds on whole outputs of 4-bit products (w4_bounds.py): what has the accuracy that is claimed lies within, what has lost bits does not. Mistakes are
made here, in plain arithmetic."""
import numpy as np
import pytest

import w4_bounds as bounds
import w4_plain as plain

N, ROWS = 400, 64


def case(k, group, dtype, with_zeros, seed):
    rng = np.random.default_rng([seed, k, group])
    codes = rng.integers(0, 16, (N, k))
    scales = plain.to_bf16(np.exp(0.7 * rng.standard_normal((k // group, N))) * 0.3 / np.sqrt(k))
    zeros = rng.integers(0, 16, (k // group, N)) if with_zeros else None
    x = rng.standard_normal((ROWS, k)).astype(np.float32).astype(np.float64)
    return plain.to_bf16(x) if dtype == "bf16" else x, plain.dequantize(codes, scales, zeros, group)


def with_bits(w, bits):
    m, e = np.frexp(w)
    return np.ldexp(np.rint(np.ldexp(m, bits)), e - bits)


def upper(x):
    """A value's first eight bits, cut off."""
    return (x.astype(np.float32).view(np.uint32) & np.uint32(0xffff0000)).view(np.float32).astype(np.float64)


def chains(x, w, per, group=None):
    """f32 sums that go through `per` products at a time, each step cut off at 24 bits; of groups, whose ends are added."""
    def cut(v):
        m, e = np.frexp(v)
        return np.ldexp(np.trunc(np.ldexp(m, 24)), e - 24)

    k = w.shape[1]
    group = group or k
    total = np.zeros((x.shape[0], w.shape[0]))
    for g in range(0, k, group):
        part = np.zeros_like(total)
        for j in range(g, g + group, per):
            part = cut(part + x[:, j:j + per] @ w[:, j:j + per].T)
        total = (total + part).astype(np.float32).astype(np.float64)
    return total


def passes(got, x, w, group, dtype, tiles, step=0.0):
    try:
        bounds.check(bounds.rounded(got, dtype), x @ w.T, bounds.error(x, w, group, dtype, tiles, step), dtype)
    except AssertionError:
        return False
    return True


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k", [512, 4096, 8192])
def test_terms_of_f32_tokens(k, group):
    for with_zeros in (False, True):
        x, w = case(k, group, "f32", with_zeros, 1)
        hi = upper(x)
        mid = upper(x - hi)
        lo = upper(x - hi - mid)
        assert np.array_equal(hi + mid + lo, x)
        assert passes(x @ w.T, x, w, group, "f32", False)
        assert passes(chains(np.stack([hi, mid, lo], 1).reshape(ROWS * 3, k), w, 16, group).reshape(ROWS, 3, N).sum(1), x, w, group, "f32", False)
        assert not passes((hi + mid) @ w.T, x, w, group, "f32", False)
        assert not passes(hi @ w.T, x, w, group, "f32", False)


@pytest.mark.parametrize("k", [512, 4096, 8192])
def test_bits_of_weights(k):
    x, w = case(k, 128, "bf16", False, 2)
    for tiles in (False, True):
        assert passes(x @ w.T, x, w, 128, "bf16", tiles) and passes(chains(x, w, 16, None if tiles else 128), x, w, 128, "bf16", tiles)
        assert np.array_equal(with_bits(w, 11), w)
        assert not any(passes(x @ with_bits(w, bits).T, x, w, 128, "bf16", tiles) for bits in (8, 9, 10))
    x, w = case(k, 128, "bf16", True, 3)
    step = 2.0 ** -12
    assert passes(x @ with_bits(w, 11).T, x, w, 128, "bf16", True, step)
    assert not passes(x @ with_bits(w, 11).T, x, w, 128, "bf16", False)
    assert not any(passes(x @ with_bits(w, bits).T, x, w, 128, "bf16", True, step) for bits in (8, 9))


def test_rounding():
    v = np.array([0.0, 1.0, 1.0 + 2.0 ** -9, 1.0 + 3 * 2.0 ** -9, -2.0 ** -126, 2.0 ** -133, 2.0 ** -134, 3 * 2.0 ** -135])
    np.testing.assert_array_equal(bounds.rounded(v, "bf16"), [0.0, 1.0, 1.0, 1.0 + 2.0 ** -7, -2.0 ** -126, 2.0 ** -133, 0.0, 2.0 ** -133])
    r = np.random.default_rng(0).standard_normal(1000) * np.exp2(np.arange(1000) % 40 - 20)
    np.testing.assert_array_equal(bounds.rounded(r, "f32"), r.astype(np.float32))
    np.testing.assert_array_equal(bounds.rounded(r, "bf16"), plain.to_bf16(r))
