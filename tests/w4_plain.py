"""Plain 64-bit forms of the 4-bit operators, in numpy, and the bounds that the tests hold the kernels to."""
import numpy as np

SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)


def to_bf16(x):
    """f64 -> the nearest bf16 value (ties to even), one rounding; normal numbers, zero and non-finite values."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        m, e = np.frexp(x)
        r = np.ldexp(np.rint(m * 256.0), e - 8)
    return np.where(np.isfinite(x), r, x)


def pack(codes):
    codes = codes.astype(np.uint32).reshape(codes.shape[0], -1, 8)
    words = np.zeros(codes.shape[:2], np.uint32)
    for i, s in enumerate(SHIFTS):
        words |= codes[:, :, i] << np.uint32(s)
    return words.view(np.int32)


def unpack(words):
    words = np.ascontiguousarray(words).view(np.uint32)
    return np.stack([(words >> np.uint32(s)) & 15 for s in SHIFTS], axis=-1).reshape(words.shape[0], -1).astype(np.int64)


def dequantize(codes, scales, zeros, group):
    """[n, k] f64 from codes [n, k], scales [k / group, n], zeros likewise or None."""
    z = 8.0 if zeros is None else np.repeat(np.asarray(zeros, np.float64).T, group, axis=1)
    return (codes - z) * np.repeat(np.asarray(scales, np.float64).T, group, axis=1)


def quantize(w, group, with_zeros):
    """(codes [n, k], scales [k / group, n], zeros or None) of f64 values that f32 holds."""
    n, k = w.shape
    v = np.asarray(w, np.float64).reshape(n, k // group, group)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[:, :, None], 0.0, v)
    if with_zeros:
        lo, hi = np.minimum(v.min(-1), 0.0), np.maximum(v.max(-1), 0.0)
        scale = to_bf16((hi - lo) / 15.0)
    else:
        scale = to_bf16(np.abs(v).max(-1) / 7.0)
    scale = np.where(scale < 2.0 ** -126, 0.0, scale)
    per = np.where(scale > 0, scale, np.inf)
    zero = np.clip(np.rint(-lo / per), 0, 15) if with_zeros else np.full(scale.shape, 8.0)
    codes = np.clip(np.rint(v / per[:, :, None]) + zero[:, :, None], 0, 15)
    scale = np.where(bad, np.nan, scale)
    if with_zeros:
        zero = np.where(bad, 0.0, zero)
        codes = np.where(bad[:, :, None], 0.0, codes)
    return codes.reshape(n, k).astype(np.int64), scale.T, zero.T if with_zeros else None


def weight_step(rows, dtype, zeros):
    """How far, relative to its size, a weight may be rounded. The kernels for many rows of bf16 hold (code - zero) * scale in f16. A code less 8 is at most 8 in
    size: three bits, or one, times the eight of a bf16 scale are at most 11, which f16 holds. A code less any other zero is at most 15: four bits times eight
    are at most 12, and rounding to 11 is off by at most half a step, 2^-12. Everywhere else codes and scales are not multiplied before the sum."""
    return 2.0 ** -12 if rows > 16 and dtype == "bf16" and zeros is not None else 0.0


def product(x, w, step=0.0):
    """(x w^T, bound of the error of its f32 sum): k additions, each off by at most a unit in the last place of the sum of magnitudes, of weights that are off
    by `step`."""
    with np.errstate(invalid="ignore", over="ignore"):
        return x @ w.T, ((w.shape[1] + 8) * 2.0 ** -23 + step) * (np.abs(x) @ np.abs(w.T))


def activate(name, g):
    """(f(g), bound of the relative error of its evaluation). silu: the argument enters the exponential as it is, the fast exponential is off by
    2 + 1.2 |g| units of 2^-23, and the quotient and products by a few more. gelu: the argument takes some roundings of its own."""
    with np.errstate(over="ignore", invalid="ignore"):
        a = g if name == "silu" else np.sqrt(8.0 / np.pi) * (g + 0.044715 * g ** 3)
        f = g / (1.0 + np.exp(-a))
    return f, (8.0 + 6.0 * np.abs(a)) * 2.0 ** -23


def gated(name, x, wg, wu, gate_step=0.0, up_step=0.0):
    (g, dg), (u, du) = product(x, wg, gate_step), product(x, wu, up_step)
    f, rel = activate(name, g)
    df = 1.13 * dg + rel * np.abs(f)  # neither function is steeper than 1.13
    return f * u, df * np.abs(u) + np.abs(f) * du + df * du + 2.0 ** -23 * np.abs(f * u)


def half_step(dtype):
    return {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}[dtype]


def check(got, want, bound, dtype, what=""):
    """Non-finite values where the plain form has them, and the others within the bound of the sum plus the rounding to the output's type."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    inf = ~finite & ~np.isnan(want)
    assert np.array_equal(got[inf], want[inf]), what
    with np.errstate(invalid="ignore"):
        over = np.abs(got - want) - (half_step(dtype) * (np.abs(want) + bound) + bound + 1e-37)
    worst = np.max(over[finite], initial=-1.0)
    assert worst <= 0, f"{what}: off by {worst} more than the bound"
