"""The precision of products with 4-bit weights: single products bit for bit, and the error of whole outputs (w4_bounds.py), in every kernel."""
import numpy as np
import pytest

import w4_bounds as bounds
import w4_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def backend(pkg):
    return pkg.CudaBackend(0)


def device(x, dtype):
    return torch.tensor(x, dtype=torch.float64).to(DTYPES[dtype]).cuda()


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def values(rng, shape, dtype, std=1.0):
    x = (rng.standard_normal(shape) * std).astype(np.float32).astype(np.float64)
    return plain.to_bf16(x) if dtype == "bf16" else x


class Weight:
    def __init__(self, pkg, rng, n, k, group, with_zeros, codes=None, scales=None):
        self.group, self.with_zeros = group, with_zeros
        codes = rng.integers(0, 16, (n, k)) if codes is None else codes
        self.scales = plain.to_bf16(np.exp(0.7 * rng.standard_normal((k // group, n))) * 0.3 / np.sqrt(k)) if scales is None else scales
        zeros = rng.integers(0, 16, (k // group, n)) if with_zeros else None
        self.w = plain.dequantize(codes, self.scales, zeros, group)
        self.handle = pkg.W4Weight(torch.tensor(plain.pack(codes)).cuda(), device(self.scales, "bf16"),
                                   torch.tensor(zeros, dtype=torch.uint8).cuda() if with_zeros else None, group)

    def step(self, tiles):
        """A weight with a zero point other than 8 is rounded to eleven bits in the tiles."""
        return 2.0 ** -12 if tiles and self.with_zeros else 0.0


def check_linear(pkg, backend, x, w, dtype, what=""):
    tiles = bounds.in_tiles(x.shape[0], w.w.shape[0], w.w.shape[1], dtype)
    got = host(pkg.linear_w4(backend, device(x, dtype), w.handle))
    bounds.check(got, x @ w.w.T, bounds.error(x, w.w, w.group, dtype, tiles, w.step(tiles)), dtype, f"linear {what}")


def check_gated(pkg, backend, x, gate, up, dtype, act, what=""):
    tiles = bounds.in_tiles(x.shape[0], 2 * up.w.shape[0], up.w.shape[1], dtype)
    got = host(pkg.gated_w4(backend, device(x, dtype), gate.handle, up.handle, activation=act))
    bounds.check(got, *bounds.gated_error(act, x, gate.w, up.w, up.group, dtype, tiles, gate.step(tiles), up.step(tiles)), dtype, f"gated {what}")


ROWS = [1, 7, 8, 9, 16, 17, 32, 33, 64, 65, 128, 130, 300]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", ROWS)
def test_single_f32_products_bit_for_bit(pkg, backend, rows, group):
    """One value of 24 bits in a row, weights that are powers of two: a product is exact, and so is the output."""
    for n, k in ((37, 128), (300, 1152)):
        rng = np.random.default_rng([41, rows, group, n])
        codes = 8 + rng.choice([-8, -4, -2, -1, 1, 2, 4], (n, k))
        w = Weight(pkg, rng, n, k, group, False, codes, 2.0 ** rng.integers(-20, 20, (k // group, n)).astype(np.float64))
        x = np.zeros((rows, k))
        x[np.arange(rows), rng.integers(0, k, rows)] = rng.integers(1 << 23, 1 << 24, rows) * 2.0 ** rng.integers(-60, 40, rows) * rng.choice([-1.0, 1.0], rows)
        got = host(pkg.linear_w4(backend, device(x, "f32"), w.handle))
        np.testing.assert_array_equal(got, x @ w.w.T)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", ROWS)
def test_single_bf16_products_are_rounded_once(pkg, backend, rows, group):
    """One value in a row: code, scale and value make 19 bits, which f32 holds; the output is the nearest bf16 number. Zero points other than 8 likewise in the
    kernel for few rows."""
    for n, k, with_zeros in ((37, 128, True), (300, 1152, True), (5602, 4224, False), (2602, 4224, False)):
        rng = np.random.default_rng([42, rows, group, n])
        w = Weight(pkg, rng, n, k, group, with_zeros)
        assert not (with_zeros and bounds.in_tiles(rows, n, k, "bf16"))
        x = np.zeros((rows, k))
        x[np.arange(rows), rng.integers(0, k, rows)] = values(rng, rows, "bf16")
        np.testing.assert_array_equal(host(pkg.linear_w4(backend, device(x, "bf16"), w.handle)), bounds.rounded(x @ w.w.T, "bf16"))


@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", ROWS)
def test_errors_of_sums(pkg, backend, rows, dtype, group, with_zeros):
    """Short, ordinary and long sums; the last of them run in tiles where rows and type allow it."""
    for n, k in ((257, 256), (1030, 4224), (150, 14336), (5602 if rows <= 64 else 2602, 4224)):
        rng = np.random.default_rng([43, rows, group, n, with_zeros])
        w = Weight(pkg, rng, n, k, group, with_zeros)
        check_linear(pkg, backend, values(rng, (rows, k), dtype), w, dtype, f"{rows} x {k} to {n}")


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", ROWS)
def test_errors_of_gated_products(pkg, backend, rows, dtype, group):
    act = ("silu", "gelu_tanh")[(rows + group // 32) % 2]
    for n, k in ((130, 256), (515, 4224), (2802 if rows <= 64 else 1302, 4224)):
        rng = np.random.default_rng([44, rows, group, n])
        gate, up = (Weight(pkg, rng, n, k, group, with_zeros) for with_zeros in (rows % 2 == 0, rows % 3 == 0))
        check_gated(pkg, backend, values(rng, (rows, k), dtype, 0.5), gate, up, dtype, act, f"{rows} x {k} to {n}")


SPLITS = [(50, 5642, 3616, 2, 256), (61, 4398, 4192, 3, 256), (63, 3802, 4192, 4, 256), (61, 3006, 5568, 5, 256), (50, 2254, 8992, 6, 256), (64, 1762, 8960, 7, 256),
          (62, 1790, 9056, 8, 256), (61, 1166, 14368, 8, 256), (90, 5642, 2080, 2, 128), (113, 4398, 2336, 3, 128), (100, 3786, 2720, 4, 128), (97, 3002, 3616, 5, 128),
          (113, 2254, 4256, 6, 128), (65, 1806, 8992, 7, 128), (113, 1790, 5600, 8, 128), (128, 1088, 7264, 8, 128)]


@pytest.mark.parametrize("rows, weight_rows, k, parts, stage", SPLITS)
def test_parts_of_k_in_the_tiles(pkg, backend, rows, weight_rows, k, parts, stage):
    """A tile's k dealt to clusters of every size, in stages of either length."""
    assert bounds.in_tiles(rows, weight_rows, k, "bf16") and bounds.splits(rows, weight_rows, k) == (parts, stage)
    rng = np.random.default_rng([45, rows, weight_rows])
    x = values(rng, (rows, k), "bf16", 0.5)
    for with_zeros in (False, True):
        w = Weight(pkg, rng, weight_rows, k, 32, with_zeros)
        check_linear(pkg, backend, x, w, "bf16")
        half = weight_rows // 2
        gate, up = Weight(pkg, rng, half, k, 32, with_zeros), Weight(pkg, rng, half, k, 32, False)
        check_gated(pkg, backend, x, gate, up, "bf16", "silu")
