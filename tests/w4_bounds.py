"""Bounds on the error of 4-bit products over a whole output, beside the elementwise worst cases of w4_plain.py, which grow with the length of a sum.

Let q = sqrt(sum of (x w)^2) of an output. Products of random signs sum up to about q, and after j of n steps to about sqrt(j / n) q. A step of the tensor
cores (16 products) cuts the running sum off at its 24 bits: by at most 2^-23 of it, always towards zero. So a chain of n steps is off by at most
2^-23 q (sum of sqrt(j / n)) = 2/3 n 2^-23 q, all in one direction. Chains are a group's (few rows; three terms for each f32 value), whose ends are off by
that share of the group's sum and so, together, of the whole sum; or all of k (many rows of bf16). What is added in f32 beyond them, m sums, is rounded to
the nearest: sqrt(m) 2^-24 q, with a few sums more of parts of k. Weights that are rounded by up to `step` of themselves, each in a direction of its own, make
step / sqrt(3) q.

An output v that is off by d before it is rounded to its type, with spacing u there, ends in another place than v with probability |d| / u and is then off by u: on
average by |d|, whatever the spacing. So the sum of |got - round(want)| over all outputs is that of |d|, with a variance V of at most sum |d| u. Where |d| is far
below u few outputs change place, and the sum is not normally distributed: by Bernstein's inequality it exceeds its mean by t with a probability of at most
exp(-t^2 / (2 V + 2 t U / 3)), U the largest u, and that is e^-16 for t = 16 U / 3 + sqrt((16 U / 3)^2 + 32 V)."""
import numpy as np

import w4_plain as plain

TILE_PRODUCTS = 1e9  # csrc/w4_api.cu: products beyond which bf16 rows run in tiles


def in_tiles(rows, weight_rows, k, dtype):
    """Whether a product runs in the kernel for many rows."""
    return dtype == "bf16" and rows > 16 and k >= 256 and max(rows, 48) * weight_rows * k > TILE_PRODUCTS


def splits(rows, weight_rows, k):
    """CTAs of a cluster that share the k of a tile of the kernel for 17 to 128 rows, and the k of its stages (csrc/w4_tiles.cu: make_plan)."""
    assert rows <= 128
    stage = 256 if rows <= 64 else 128
    resident = (0, 148, 144, 132, 128, 120, 126, 105, 112)
    stages, tiles_w = -(-k // stage), -(-weight_rows // 128)
    best = (1e300, 0)
    tokens = -(-rows // 32) * 32
    for parts in range(1, min(8, stages) + 1):
        if parts > 1 and tiles_w * parts > resident[parts]:
            continue
        rounds = -(-tiles_w * parts // 148)
        cost = rounds * (-(-stages // parts) * max(4.0 * tokens, 450.0) * (stage // 128) + 3000.0) + (2000.0 if parts > 1 else 0.0)
        best = min(best, (cost, parts))
    return best[1], stage


def spacing(v, dtype):
    """From a value of a type to the next."""
    bits, lowest = {"bf16": (8, -133), "f32": (24, -149)}[dtype]
    return np.exp2(np.maximum(np.frexp(np.where(v == 0, 1.0, v))[1] - bits, lowest).astype(np.float64)) * (v != 0) + 2.0 ** lowest * (v == 0)


def rounded(v, dtype):
    """The nearest value of the type, ties to even, subnormal numbers among them."""
    step = spacing(v, dtype)
    return np.rint(v / step) * step


def error(x, w, group, dtype, tiles, step=0.0):
    """What an output of x w^T is off by before it is rounded: see above."""
    k = w.shape[1]
    chain = k // 16 if tiles else group // 16 * (3 if dtype == "f32" else 1)
    sums = 0 if tiles else k // group
    return (2.0 / 3.0 * chain * 2.0 ** -23 + (np.sqrt(sums) + 8.0) * 2.0 ** -24 + step / np.sqrt(3.0)) * np.sqrt((x ** 2) @ (w ** 2).T)


def gated_error(name, x, wg, wu, group, dtype, tiles, gate_step=0.0, up_step=0.0):
    g, u = x @ wg.T, x @ wu.T
    f, rel = plain.activate(name, g)
    dg, du = error(x, wg, group, dtype, tiles, gate_step), error(x, wu, group, dtype, tiles, up_step)
    return f * u, 1.13 * dg * np.abs(u) + np.abs(f) * du + dg * du + (rel + 2.0 ** -23) * np.abs(f * u)


def check(got, want, bound, dtype, what=""):
    """The outputs as a whole: sum |got - round(want)| against the sum of their bounds."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape and np.isfinite(want).all()
    u = spacing(want, dtype)
    rare = 16.0 / 3.0 * u.max()
    off, most = np.abs(got - rounded(want, dtype)).sum(), bound.sum() + rare + np.sqrt(rare ** 2 + 32.0 * (bound * u).sum())
    assert off <= most, f"{what}: {off / most:.3g} times the bound"
