"""4-bit weights on the device: quantiser, projection, gated feed-forward, against plain 64-bit forms."""
import functools

import numpy as np
import pytest

import w4_plain as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def backend(pkg):
    return pkg.CudaBackend(0)


def values(rng, shape, dtype, std=1.0):
    """f64 values that `dtype` holds."""
    x = (rng.standard_normal(shape) * std).astype(np.float32).astype(np.float64)
    return plain.to_bf16(x) if dtype == "bf16" else x


def device(x, dtype):
    return torch.tensor(x, dtype=torch.float64).to(DTYPES[dtype]).cuda()


class Weight:
    def __init__(self, pkg, rng, n, k, group, zeros):
        self.codes = rng.integers(0, 16, (n, k))
        self.scales = plain.to_bf16(np.exp(0.7 * rng.standard_normal((k // group, n))) * 0.3 / np.sqrt(k))
        self.zeros = rng.integers(0, 16, (k // group, n)) if zeros else None
        self.w = plain.dequantize(self.codes, self.scales, self.zeros, group)
        self.handle = pkg.W4Weight(torch.tensor(plain.pack(self.codes)).cuda(), device(self.scales, "bf16"),
                                   None if self.zeros is None else torch.tensor(self.zeros, dtype=torch.uint8).cuda(), group)


    def step(self, rows, dtype):
        return plain.weight_step(rows, dtype, self.zeros)


def host(t):
    torch.cuda.synchronize()
    return t.double().cpu().numpy()


def sizes(rows):
    """(n, k) of a product that runs in tiles where its rows are more than 16, or 100 of more than 64: of one CTA each to 128 rows, of pairs beyond."""
    return (140, 512) if rows <= 16 else (5602, 4160) if rows <= 64 else (2602, 4160) if rows <= 128 else (1002, 4160)


ROWS = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 130, 257, 300]
SHAPES = [(1, 32, 32), (15, 128, 128), (17, 96, 32), (33, 64, 64), (100, 352, 32), (256, 1024, 128), (1001, 4160, 64), (130, 8192, 128), (2051, 2752, 64), (1400, 4384, 32)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", ROWS)
def test_linear(pkg, backend, rows, dtype):
    for i, (n, k, group) in enumerate(SHAPES):
        rng = np.random.default_rng([rows, i, dtype == "f32"])
        w = Weight(pkg, rng, n, k, group, zeros=(rows + i) % 2 == 0)
        x = values(rng, (rows, k), dtype)
        bias = values(rng, n, "f32") if i % 3 else None
        got = pkg.linear_w4(backend, device(x, dtype), w.handle, bias=None if bias is None else device(bias, "f32"))
        want, bound = plain.product(x, w.w, w.step(rows, dtype))
        if bias is not None:
            want, bound = want + bias, bound + 2.0 ** -23 * (np.abs(want) + np.abs(bias))
        assert got.dtype == DTYPES[dtype]
        plain.check(host(got), want, bound, dtype, f"{rows} x {k} to {n}, groups of {group}")


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", ROWS)
def test_gated(pkg, backend, rows, dtype, act):
    for i, (n, k, group) in enumerate(SHAPES):
        rng = np.random.default_rng([rows, i, dtype == "f32", len(act)])
        gate, up = (Weight(pkg, rng, n, k, group, zeros=(rows + i + j) % 2 == 0) for j in range(2))
        x = values(rng, (rows, k), dtype, 0.5)
        got = pkg.gated_w4(backend, device(x, dtype), gate.handle, up.handle, activation=act)
        plain.check(host(got), *plain.gated(act, x, gate.w, up.w, gate.step(rows, dtype), up.step(rows, dtype)), dtype, f"{rows} x {k} to {n}, groups of {group}")


@pytest.mark.parametrize("n, k", [(10880, 1536), (6528, 2560), (5376, 6144), (4608, 3584)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 12, 40])
def test_clusters_of_any_size(pkg, backend, rows, dtype, n, k):
    """k dealt to 3, 5, 6 and 7 CTAs and to other numbers of them."""
    rng = np.random.default_rng([22, rows, n])
    w = Weight(pkg, rng, n, k, 128, zeros=rows == 12)
    x = values(rng, (rows, k), dtype)
    plain.check(host(pkg.linear_w4(backend, device(x, dtype), w.handle)), *plain.product(x, w.w, w.step(rows, dtype)), dtype)
    half = n // 2
    top, low = (pkg.W4Weight(w.handle.packed[i:i + half], w.handle.scales[:, i:i + half].contiguous(), None if w.zeros is None else w.handle.zeros[:, i:i + half].contiguous(), 128)
                for i in (0, half))
    step = w.step(rows, dtype)
    plain.check(host(pkg.gated_w4(backend, device(x, dtype), top, low)), *plain.gated("silu", x, w.w[:half], w.w[half:], step, step), dtype)


@functools.lru_cache(maxsize=None)
def large_weight(pkg, n, k, group, zeros, seed):
    return Weight(pkg, np.random.default_rng([n, zeros, seed]), n, k, group, zeros)


LARGE = [(5602, 4128, 32), (3001, 7488, 64), (4097, 5504, 128)]


@pytest.mark.parametrize("n, k, group", LARGE)
@pytest.mark.parametrize("rows", [17, 33, 64, 65, 100, 128, 130])
def test_linear_of_large_matrices(pkg, backend, rows, n, k, group):
    rng = np.random.default_rng([20, rows, n])
    for zeros in (False, True):
        w = large_weight(pkg, n, k, group, zeros, 0)
        x, bias = values(rng, (rows, k), "bf16"), values(rng, n, "f32")
        got = pkg.linear_w4(backend, device(x, "bf16"), w.handle, bias=device(bias, "f32"))
        want, bound = plain.product(x, w.w, w.step(rows, "bf16"))
        plain.check(host(got), want + bias, bound + 2.0 ** -23 * (np.abs(want) + np.abs(bias)), "bf16")


@pytest.mark.parametrize("n, k, group", LARGE)
@pytest.mark.parametrize("rows", [17, 64, 65, 128, 130])
def test_gated_of_large_matrices(pkg, backend, rows, n, k, group):
    x = values(np.random.default_rng([21, rows, n]), (rows, k), "bf16", 0.5)
    for act, zeros in (("silu", (False, True)), ("gelu_tanh", (True, False)), ("silu", (False, False))):
        gate, up = (large_weight(pkg, n, k, group, z, i) for i, z in enumerate(zeros))
        got = pkg.gated_w4(backend, device(x, "bf16"), gate.handle, up.handle, activation=act)
        plain.check(host(got), *plain.gated(act, x, gate.w, up.w, gate.step(rows, "bf16"), up.step(rows, "bf16")), "bf16")


@pytest.mark.parametrize("rows, n, k", [(3, 38000, 160), (14, 39001, 128), (30, 38001, 288), (100, 39000, 256), (129, 20001, 384), (1100, 6001, 512), (520, 20000, 160),
                                        (30, 78001, 288), (100, 42000, 288), (129, 22001, 384)])
def test_more_tiles_than_the_device_takes_at_once(pkg, backend, rows, n, k):
    """Resident CTAs go from tile to tile, their rings running on."""
    rng = np.random.default_rng([rows, n])
    w = Weight(pkg, rng, n, k, 32, zeros=rows % 2 == 0)
    x = values(rng, (rows, k), "bf16")
    plain.check(host(pkg.linear_w4(backend, device(x, "bf16"), w.handle)), *plain.product(x, w.w, w.step(rows, "bf16")), "bf16")
    half = n // 2
    top, low = (pkg.W4Weight(w.handle.packed[i:i + half].clone(), w.handle.scales[:, i:i + half].contiguous(),
                             None if w.zeros is None else w.handle.zeros[:, i:i + half].contiguous(), 32) for i in (0, half))
    step = w.step(rows, "bf16")
    plain.check(host(pkg.gated_w4(backend, device(x, "bf16"), top, low)), *plain.gated("silu", x, w.w[:half], w.w[half:2 * half], step, step), "bf16")


@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n, k, group", [(1, 32, 32), (3, 128, 128), (31, 96, 32), (33, 64, 64), (70, 1120, 32), (257, 4096, 128), (513, 2112, 64)])
def test_quantize(pkg, backend, n, k, group, dtype, with_zeros):
    rng = np.random.default_rng([n, k, with_zeros])
    w = values(rng, (n, k), dtype, 0.02) + 0.0
    w[0, :group] = 0.0  # a group of zeros
    if n > 2:  # whole multiples and halves of a scale of 2^-6: every other quotient lies on a border
        w[1, :group] = (np.arange(group) % 29 - 14) * 2.0 ** -7
        w[2, :group] = np.abs(w[2, :group])  # one sign only
        w[2, group - 1] = 0.0
    got = pkg.quantize_w4(backend, device(w, dtype), group=group, zeros=with_zeros)
    codes, scales, zeros = plain.quantize(w, group, with_zeros)
    assert got.packed.dtype == torch.int32 and got.group == group and (got.zeros is not None) == with_zeros
    np.testing.assert_array_equal(host(got.scales), scales)
    np.testing.assert_array_equal(plain.unpack(got.packed.cpu().numpy()), codes)
    if with_zeros:
        np.testing.assert_array_equal(host(got.zeros), zeros)


@pytest.mark.parametrize("with_zeros", [False, True])
def test_quantize_extremes(pkg, backend, with_zeros):
    """Infinities and NaN, the largest and the smallest numbers, and values next to a border between two codes."""
    rng = np.random.default_rng(5)
    w = values(rng, (12, 64), "f32")
    w[0, 5], w[1, 40], w[2, 3] = np.inf, np.nan, -np.inf
    w[3, :32] *= 2.0 ** 125
    w[3, 1], w[3, 2] = np.float32(3.4028234e38), np.float32(-3.4028234e38)
    w[4, :32] *= 2.0 ** -130  # scales below the smallest normal number
    w[5, :32] *= 2.0 ** -115
    w[6, :32] = np.nextafter(np.float32(0.5), np.float32(1))
    w[6, 0] = 7.0
    w[7, :32] = np.nextafter(np.float32(2.5), np.float32(0))
    w[7, 0] = -7.0
    w[8, :32], w[8, 0], w[8, 1] = 1.5, 15.0, 0.5
    w[9, :32], w[9, 0], w[9, 1] = -3.5, -7.5, 7.5
    w[10, :32] = np.nextafter(np.float32(1.5), np.float32(0))
    w[10, 0] = 15.0
    w = w.astype(np.float32).astype(np.float64)
    got = pkg.quantize_w4(backend, device(w, "f32"), group=32, zeros=with_zeros)
    codes, scales, zeros = plain.quantize(w, 32, with_zeros)
    np.testing.assert_array_equal(host(got.scales), scales)
    np.testing.assert_array_equal(plain.unpack(got.packed.cpu().numpy()), codes)
    if with_zeros:
        np.testing.assert_array_equal(host(got.zeros), zeros)


def test_quantize_strided_rows(pkg, backend):
    rng = np.random.default_rng(6)
    w = values(rng, (40, 256), "bf16")
    wide = device(w, "bf16")
    a, b = pkg.quantize_w4(backend, wide[3:30, 64:192], group=64), pkg.quantize_w4(backend, wide[3:30, 64:192].contiguous(), group=64)
    assert torch.equal(a.packed, b.packed) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 5, 20, 50, 100, 300])
def test_infinities_and_nan_stay_in_their_rows(pkg, backend, rows, dtype):
    rng = np.random.default_rng([7, rows])
    n, k = sizes(rows)
    w, up = Weight(pkg, rng, n, k, 64, True), Weight(pkg, rng, n, k, 64, False)
    x = values(rng, (rows, k), dtype)
    clean = host(pkg.linear_w4(backend, device(x, dtype), w.handle))
    x[0, 3] = np.inf
    if rows > 2:
        x[1, 70], x[2, 5], x[2, 9] = np.nan, np.inf, -np.inf
    with np.errstate(invalid="ignore"):
        # a code that equals its zero point makes the product of an infinity a NaN
        want = np.stack([(r[None, :] * w.w).sum(1) for r in x[:3]] + [np.zeros(n)] * (rows - 3))
    got = host(pkg.linear_w4(backend, device(x, dtype), w.handle))
    assert np.array_equal(np.isnan(got[:3]), np.isnan(want[:3]))
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    np.testing.assert_array_equal(got[3:], clean[3:])
    y = host(pkg.gated_w4(backend, device(x, dtype), w.handle, up.handle))
    assert not np.isfinite(y[0]).any() or rows == 0
    assert np.isfinite(y[3:]).all()


@pytest.mark.parametrize("rows", [3, 20, 100, 300])
@pytest.mark.parametrize("scale", [1e-30, 1e-4, 1e4, 1e30])
def test_rows_of_any_magnitude(pkg, backend, rows, scale):
    """Rows and outputs whose sizes differ by many powers of ten come out as exact as others."""
    rng = np.random.default_rng([8, rows])
    n, k = sizes(rows)
    w = Weight(pkg, rng, n, k, 64 if k % 128 else 128, True)
    x = values(rng, (rows, k), "bf16")
    x[0] = plain.to_bf16(x[0] * scale)
    x[1, 17] = plain.to_bf16(np.float64(1e5))
    x[2] = 0.0
    want, bound = plain.product(x, w.w, w.step(rows, "bf16"))
    plain.check(host(pkg.linear_w4(backend, device(x, "bf16"), w.handle)), want, bound, "bf16")


@pytest.mark.parametrize("rows", [1, 20, 100, 300])
def test_outputs_of_any_magnitude(pkg, backend, rows):
    rng = np.random.default_rng([9, rows])
    n, k = sizes(rows)
    w = Weight(pkg, rng, n, k, 64, True)
    w.scales[:, 0] = plain.to_bf16(w.scales[:, 0] * 2.0 ** -60)
    w.scales[:, 1] = plain.to_bf16(w.scales[:, 1] * 2.0 ** 60)
    w.scales[1, 2] = 0.0
    w.scales[:, 3] = 0.0
    w.scales[2, 4] *= 2.0 ** -20
    handle = pkg.W4Weight(w.handle.packed, device(w.scales, "bf16"), w.handle.zeros, 64)
    x = values(rng, (rows, k), "bf16")
    want, bound = plain.product(x, plain.dequantize(w.codes, w.scales, w.zeros, 64), w.step(rows, "bf16"))
    plain.check(host(pkg.linear_w4(backend, device(x, "bf16"), handle)), want, bound, "bf16")


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows", [1, 20, 100, 300])
def test_groups_of_any_magnitude(pkg, backend, rows, zeros):
    """Groups of a row whose scales differ by up to 2^19 and whose tokens make up for it, so that every group counts as much."""
    rng = np.random.default_rng([17, rows])
    n, k = sizes(rows)
    w = Weight(pkg, rng, n, k, 32, zeros)
    power = np.arange(k // 32) * 7 % 20
    scales = w.scales * 2.0 ** -power[:, None]
    handle = pkg.W4Weight(w.handle.packed, device(scales, "bf16"), w.handle.zeros, 32)
    x = values(rng, (rows, k), "bf16") * np.repeat(2.0 ** power, 32)
    want, bound = plain.product(x, plain.dequantize(w.codes, scales, w.zeros, 32), w.step(rows, "bf16"))
    plain.check(host(pkg.linear_w4(backend, device(x, "bf16"), handle)), want, bound, "bf16")


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 20, 100, 300])
def test_an_infinite_scale_reaches_its_output_alone(pkg, backend, rows, dtype, zeros):
    """The last group's, behind which a tile of k is not filled; a scale of NaN likewise."""
    rng = np.random.default_rng([18, rows])
    n, k = sizes(rows)
    w = Weight(pkg, rng, n, k, 32, zeros)
    x = values(rng, (rows, k), dtype)
    x[:, -32:] = np.abs(x[:, -32:]) + 1.0
    clean = host(pkg.linear_w4(backend, device(x, dtype), w.handle))
    w.codes[[3, 4], -32:] = [[15], [0]]
    if zeros:
        w.zeros[-1, [3, 4]] = 7
    w.scales[-1, [3, 4]] = np.inf
    w.scales[1, 5] = np.nan
    handle = pkg.W4Weight(torch.tensor(plain.pack(w.codes)).cuda(), device(w.scales, "bf16"), None if w.zeros is None else torch.tensor(w.zeros, dtype=torch.uint8).cuda(), 32)
    got = host(pkg.linear_w4(backend, device(x, dtype), handle))
    assert (got[:, 3] == np.inf).all() and (got[:, 4] == -np.inf).all() and np.isnan(got[:, 5]).all()
    clean[:, 3:6] = got[:, 3:6] = 0.0
    np.testing.assert_array_equal(got, clean)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 6, 14, 40, 120, 270])
def test_strided_rows_and_neighbours_of_the_output(pkg, backend, rows, dtype):
    rng = np.random.default_rng([10, rows])
    n, k = sizes(rows)
    n -= 3
    w = Weight(pkg, rng, n, k, 64, True)
    x = values(rng, (rows, k), dtype)
    wide = torch.full((rows, k + 32), float("nan"), dtype=DTYPES[dtype], device="cuda")
    wide[:, 16:k + 16] = device(x, dtype)
    out = torch.full((rows + 2, n + 22), -7.0, dtype=DTYPES[dtype], device="cuda")
    got = pkg.linear_w4(backend, wide[:, 16:k + 16], w.handle, out=out[1:rows + 1, 11:n + 11])
    assert got.data_ptr() == out[1:, 11:].data_ptr()
    plain.check(host(got), *plain.product(x, w.w, w.step(rows, dtype)), dtype)
    rest = host(out)
    rest[1:rows + 1, 11:n + 11] = -7.0
    assert (rest == -7.0).all()


@pytest.mark.parametrize("rows", [1, 12, 100, 290])
def test_captured_and_replayed(pkg, backend, rows):
    """A run of the operators as a feed-forward uses them, in two graphs that are replayed in turn with new inputs, on a stream of its own."""
    rng = np.random.default_rng([11, rows])
    width, hidden = (256, 320) if rows <= 16 else (1088, 2624)
    gate, up, down = (pkg.quantize_w4(backend, device(values(rng, s, "bf16", 0.05), "bf16"), group=64, zeros=z)
                      for s, z in (((hidden + 32, width), True), ((hidden + 32, width), True), ((width, hidden), False)))
    stream = torch.cuda.Stream()
    x = [device(values(rng, (rows, width), "bf16"), "bf16") for _ in range(2)]

    def block(v):
        return pkg.linear_w4(backend, pkg.gated_w4(backend, v, gate, up)[:, :hidden], down)

    with torch.cuda.stream(stream):
        block(x[0])
    stream.synchronize()
    graphs, outs = [], []
    for v in x:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(block(v))
        graphs.append(g)
    for turn in range(3):
        fresh = [device(values(rng, (rows, width), "bf16"), "bf16") for _ in x]
        for v, f in zip(x, fresh):
            v.copy_(f)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, f in zip(outs, fresh):
            assert torch.equal(o, block(f))


@pytest.mark.parametrize("rows", [1, 30, 128, 500])
def test_feed_forward_of_quantized_weights(pkg, backend, rows):
    """quantise three matrices, gated product, down projection: against the same in 64 bits with the codes that the quantiser must give."""
    rng = np.random.default_rng([12, rows])
    width, hidden = (256, 448) if rows <= 16 else (1088, 2624)
    shapes = ((hidden, width), (hidden, width), (width, hidden))
    raw = [values(rng, s, "f32", s[1] ** -0.5) for s in shapes]
    w = [pkg.quantize_w4(backend, device(r, "f32"), group=64, zeros=True) for r in raw]
    wide = [plain.dequantize(*plain.quantize(r, 64, True)[:2], plain.quantize(r, 64, True)[2], 64) for r in raw]
    x = values(rng, (rows, width), "bf16")
    h = pkg.gated_w4(backend, device(x, "bf16"), w[0], w[1])
    step = plain.weight_step(rows, "bf16", True)
    want, bound = plain.gated("silu", x, wide[0], wide[1], step, step)
    plain.check(host(h), want, bound, "bf16")
    y = pkg.linear_w4(backend, h, w[2])
    plain.check(host(y), *plain.product(host(h), wide[2], step), "bf16")


@pytest.mark.parametrize("n, zeros", [(600, False), (601, True), (4002, True), (4004, False), (11201, True), (11204, False)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [1, 6, 12, 40, 260])
def test_same_results_every_run_and_on_two_streams(pkg, backend, rows, dtype, n, zeros):
    rng = np.random.default_rng([13, rows])
    w = Weight(pkg, rng, n, 2048, 128, zeros)
    x = device(values(rng, (rows, 2048), dtype), dtype)
    first = pkg.linear_w4(backend, x, w.handle)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(pkg.linear_w4(backend, x, w.handle))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


def test_offsets_beyond_32_bits(pkg, backend):
    """Matrices of more than 2^33 weights, rows of activations and of outputs more than 2^32 bytes apart in all: what repeats in one comes back repeated."""
    period, times, k = 1024, 520, 16384
    rng = np.random.default_rng(19)
    base = torch.randn((period, k), generator=torch.Generator("cuda").manual_seed(19), device="cuda").to(torch.bfloat16)
    n = period * times
    w = pkg.quantize_w4(backend, base.repeat(times, 1), group=64, zeros=True)
    one = pkg.quantize_w4(backend, base, group=64, zeros=True)
    assert w.packed.numel() * 4 > 1 << 32
    for whole, part in ((w.packed.view(times, period, -1), one.packed), (w.scales.view(-1, times, period).transpose(0, 1), one.scales),
                        (w.zeros.view(-1, times, period).transpose(0, 1), one.zeros)):
        assert all(torch.equal(v, part) for v in whole)
    plain_w = plain.dequantize(plain.unpack(one.packed.cpu().numpy()), host(one.scales), host(one.zeros), 64)
    for rows, apart in ((3, 1 << 30), (20, 1 << 27), (140, 1 << 24)):
        x = values(rng, (rows, k), "bf16")
        wide = torch.empty(((rows - 1) * apart + k,), dtype=torch.bfloat16, device="cuda").as_strided((rows, k), (apart, 1))
        wide.copy_(device(x, "bf16"))
        room = torch.empty(((rows - 1) * apart + n,), dtype=torch.bfloat16, device="cuda").as_strided((rows, n), (apart, 1))
        got = pkg.linear_w4(backend, wide, w, out=room)
        first = got[:, :period]
        assert all(torch.equal(got[:, i * period:(i + 1) * period], first) for i in range(times))
        plain.check(host(first), *plain.product(x, plain_w, plain.weight_step(rows, "bf16", True)), "bf16", f"{rows} rows")
        del wide, room, got, first


def test_no_rows_and_values_written_in_place(pkg, backend):
    rng = np.random.default_rng(14)
    w = Weight(pkg, rng, 64, 128, 32, False)
    assert pkg.linear_w4(backend, torch.empty((0, 128), dtype=torch.bfloat16, device="cuda"), w.handle).shape == (0, 64)
    assert pkg.gated_w4(backend, torch.empty((0, 128), device="cuda"), w.handle, w.handle).shape == (0, 64)
    x = values(rng, (4, 128), "f32")
    w.handle.scales.mul_(2.0)  # a weight's values may change between calls
    plain.check(host(pkg.linear_w4(backend, device(x, "f32"), w.handle)), *plain.product(x, 2.0 * w.w), "f32")


def test_codes_of_other_formats(pkg, backend):
    rng = np.random.default_rng(15)
    w = Weight(pkg, rng, 50, 256, 128, True)
    again = pkg.W4Weight.from_codes(torch.tensor(w.codes).cuda(), w.handle.scales, w.handle.zeros, 128)
    assert torch.equal(again.packed, w.handle.packed)


def test_refusals(pkg, backend):
    rng = np.random.default_rng(16)
    w, other = Weight(pkg, rng, 64, 128, 32, False).handle, Weight(pkg, rng, 64, 128, 64, False).handle
    x = torch.zeros((4, 128), dtype=torch.bfloat16, device="cuda")
    bad = pytest.raises(pkg.InvalidRequest)
    for v in (x.half(), x.cpu(), x[0], x[:, :96], x.t().contiguous().t(), torch.zeros((4, 256), device="cuda")[:, ::2],
              torch.zeros((4, 129), device="cuda")[:, 1:], torch.zeros((4, 136), dtype=torch.bfloat16, device="cuda")[:, 4:132],
              x.expand(1, 4, 128), x[:1].expand(4, 128), np.zeros((4, 128)), x.float().requires_grad_()):
        with bad:
            pkg.linear_w4(backend, v, w)
        with bad:
            pkg.gated_w4(backend, v, w, w)
    for out in (torch.zeros((4, 64), device="cuda"), torch.zeros((4, 65), dtype=torch.bfloat16, device="cuda"), torch.zeros((4, 64), dtype=torch.bfloat16),
                torch.zeros((64, 4), dtype=torch.bfloat16, device="cuda").t()):
        with bad:
            pkg.linear_w4(backend, x, w, out=out)
    square = Weight(pkg, rng, 128, 128, 32, False).handle
    room = torch.zeros((12, 128), dtype=torch.bfloat16, device="cuda")
    for a, b in ((room[:4], room[:4]), (room[:4], room[3:7]), (room[4:8], room[1:5]), (room[2:10:2], room[4:12:2])):
        with bad:
            pkg.linear_w4(backend, a, square, out=b)
    wide = torch.zeros((4, 256), dtype=torch.bfloat16, device="cuda")
    for a, b in ((room[:4], room[4:8]), (room[2:10:2], room[3:11:2]), (wide[:, :128], wide[:, 128:]), (wide[:, 128:], wide[:, :128])):
        pkg.linear_w4(backend, a, square, out=b)
    for bias in (torch.zeros(64, dtype=torch.bfloat16, device="cuda"), torch.zeros(64, device="cuda", requires_grad=True), torch.zeros(63, device="cuda"), torch.zeros(64), torch.zeros(128, device="cuda")[::2]):
        with bad:
            pkg.linear_w4(backend, x, w, bias=bias)
    with bad:
        pkg.gated_w4(backend, x, w, other)
    with bad:
        pkg.gated_w4(backend, x, w, w, activation="relu")
    for args in ((w.packed, w.scales, None, 64), (w.packed, w.scales, None, 16), (w.packed, w.scales.float(), None, 32), (w.packed.long(), w.scales, None, 32),
                 (w.packed.cpu(), w.scales, None, 32), (w.packed, w.scales, w.scales, 32), (w.packed[:, :15], w.scales, None, 32),
                 (w.packed, w.scales[:, :63], None, 32), (w.packed[0], w.scales, None, 32), (w.packed, w.scales.t().contiguous().t(), None, 32)):
        with bad:
            pkg.W4Weight(*args)
    learned = w.scales.clone().requires_grad_()
    with bad:
        pkg.W4Weight(w.packed, learned, None, 32)
    with bad:
        pkg.quantize_w4(backend, x.float().requires_grad_(), group=32)
    with torch.no_grad():
        pkg.W4Weight(w.packed, learned, None, 32)
        pkg.quantize_w4(backend, x.float().requires_grad_(), group=32)
    with bad:
        pkg.W4Weight.from_codes(torch.full((64, 128), 16, device="cuda"), w.scales, None, 32)
    for v, g in ((x.half(), 32), (x.cpu(), 32), (x, 48), (x[:, :96].contiguous(), 64), (x[0], 32), (x[:0], 32), (x.t(), 4)):
        with bad:
            pkg.quantize_w4(backend, v, group=g)
