"""Products with 4-bit weights at the ends of the range of scales, tokens and results: every row of weights counts in powers of two of its own, as does every
token, and what is in range in the end has to come out, whatever stands between."""
import numpy as np
import pytest

import w4_bounds as bounds
import w4_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GROUP = 64


@pytest.fixture(scope="module")
def backend(pkg):
    return pkg.CudaBackend(0)


def device(x, dtype):
    return torch.tensor(x, dtype=torch.float64).to(DTYPES[dtype]).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def sizes(rows):
    """(n, k) that runs in tiles where there are more than 16 rows of bf16: of one CTA each to 128 rows, of pairs beyond."""
    return (140, 512) if rows <= 16 else (5602, 4160) if rows <= 64 else (2602, 4160) if rows <= 128 else (1002, 4160)


def values(rng, shape, bits):
    """Of either sign, 1 to 2 in size, with so many significant bits."""
    return np.floor(np.exp2(bits - 1) * (1.0 + rng.random(shape))) * 2.0 ** (1 - bits) * rng.choice([-1.0, 1.0], shape)


def scales_near(rng, groups, n, power):
    return plain.to_bf16(np.exp2(power + rng.random((groups, n))))


def handle(pkg, codes, scales):
    return pkg.W4Weight(torch.tensor(plain.pack(codes)).cuda(), device(scales, "bf16"), None, GROUP)


def compare(pkg, backend, x, codes, scales, dtype, size):
    """A projection, and a gated feed-forward whose gate brings tokens of 2^size to ordinary values."""
    rows, (n, k) = x.shape[0], codes.shape
    w, weight = plain.dequantize(codes, scales, None, GROUP), handle(pkg, codes, scales)
    tiles = bounds.in_tiles(rows, n, k, dtype)
    bounds.check(host(pkg.linear_w4(backend, device(x, dtype), weight)), x @ w.T, bounds.error(x, w, GROUP, dtype, tiles), dtype, "linear")
    back = np.full((k // GROUP, n), 2.0 ** (-9 - size))
    gate, plain_gate = handle(pkg, codes, back), plain.dequantize(codes, back, None, GROUP)
    tiles = bounds.in_tiles(rows, 2 * n, k, dtype)
    bounds.check(host(pkg.gated_w4(backend, device(x, dtype), gate, weight)), *bounds.gated_error("silu", x, plain_gate, w, GROUP, dtype, tiles), dtype, "gated")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("power", [-126, -124, -118, -60, 0, 60])
@pytest.mark.parametrize("rows", [3, 20, 100, 300])
def test_groups_of_scale_zero_have_no_weights(pkg, backend, rows, power, dtype):
    """Whatever their codes, and however small the largest scale of the row is."""
    rng = np.random.default_rng([31, rows, 200 + power])
    n, k = sizes(rows)
    codes = rng.integers(0, 16, (n, k))
    scales = scales_near(rng, k // GROUP, n, power)
    scales[np.arange(k // GROUP)[:, None] % 8 != np.arange(n)[None, :] % 8] = 0.0  # one group in eight is left
    size = 40 if power < 0 else 0
    compare(pkg, backend, values(rng, (rows, k), {"bf16": 8, "f32": 24}[dtype]) * 2.0 ** size, codes, scales, dtype, size)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale, token, rest", [(118, -100, 0), (124, -110, 0), (-126, 110, 0), (-120, 118, -24), (99, 48, -30), (60, 70, -20), (115, -120, -4), (-90, -20, 0)])
@pytest.mark.parametrize("rows", [3, 20, 100, 300])
def test_scales_and_tokens_of_opposite_ends(pkg, backend, rows, scale, token, rest, dtype):
    """Scales of 2^scale, a largest token of 2^token whose weights are 0, others of 2^(token + rest), with codes that keep the largest sums finite. f32 tokens are
    taken as multiples of 2^-133: those of less than 2^-109 have fewer than 24 bits, and here eight."""
    rng = np.random.default_rng([32, rows, 200 + scale, 200 + token])
    n, k = sizes(rows)
    codes = rng.integers(7, 10, (n, k))
    codes[:, 77] = 8
    x = values(rng, (rows, k), 24 if dtype == "f32" and token + rest >= -109 else 8) * 2.0 ** (token + rest)
    x[:, 77] = 2.0 ** token
    compare(pkg, backend, x, codes, scales_near(rng, k // GROUP, n, scale), dtype, token + rest)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("power", [-126, -122, -116])
@pytest.mark.parametrize("rows", [1, 8, 12, 40])
def test_small_f32_results_keep_their_bits(pkg, backend, rows, power, group):
    """Results of about 2^power: f32 has their 24 bits down to 2^-126."""
    rng = np.random.default_rng([33, rows, 200 + power, group])
    n, k = 140, 1024
    codes = rng.integers(7, 10, (n, k))
    scales = scales_near(rng, k // group, n, power + 60)
    x = values(rng, (rows, k), 24) * 2.0 ** -65  # sums of 1024 random signs: five powers of two
    w = plain.dequantize(codes, scales, None, group)
    weight = pkg.W4Weight(torch.tensor(plain.pack(codes)).cuda(), device(scales, "bf16"), None, group)
    bounds.check(host(pkg.linear_w4(backend, device(x, "f32"), weight)), x @ w.T, bounds.error(x, w, group, "f32", False), "f32")
