"""What the entry points of the 4-bit operators refuse before they touch a device, and the plain forms that the device tests compare with."""
import ctypes as C

import numpy as np
import pytest

import w4_plain as plain

P = 1 << 20  # stands for a device pointer: nothing here gets as far as using one


def weight(pkg, **over):
    f = dict(packed=P, scales=P, zeros=0, out_features=64, in_features=128, group=32)
    f.update(over)
    return pkg._ffi.OrionW4Weight(f["packed"], f["scales"], f["zeros"], f["out_features"], f["in_features"], f["group"])


def linear(pkg, w=None, dtype=2, x=P, rows=4, stride=128, bias=0, out=P, out_stride=64, space=0, size=0):
    w = weight(pkg) if w is None else w
    return pkg._ffi.lib().orion_cuda_w4_linear(0, dtype, x, rows, stride, C.addressof(w) if w else None, bias, out, out_stride, space, size, None)


def gated(pkg, gate=None, up=None, dtype=2, act=0, x=P, rows=4, stride=128, out=P, out_stride=64, space=0, size=0):
    gate, up = gate or weight(pkg), up or weight(pkg)
    return pkg._ffi.lib().orion_cuda_w4_gated(0, dtype, x, rows, stride, C.addressof(gate), C.addressof(up), act, out, out_stride, space, size, None)


def quantize(pkg, dtype=2, w=P, n=64, k=128, stride=128, group=32, packed=P, scales=P, zeros=0):
    return pkg._ffi.lib().orion_cuda_w4_quantize(0, dtype, w, n, k, stride, group, packed, scales, zeros, None)


BAD_WEIGHTS = [dict(packed=0), dict(scales=0), dict(packed=P + 8), dict(scales=P + 1), dict(scales=P + 2), dict(zeros=P + 2), dict(group=0), dict(group=16), dict(group=48), dict(group=256),
               dict(in_features=0), dict(in_features=130), dict(in_features=1 << 31), dict(out_features=0), dict(out_features=1 << 31)]
BAD_ROWS = [dict(dtype=1), dict(dtype=4), dict(dtype=-1), dict(x=0), dict(x=P + 2), dict(x=P + 8), dict(stride=127), dict(stride=0), dict(stride=132),
            dict(stride=1 << 50), dict(rows=1 << 31), dict(out=0), dict(out=P + 1), dict(out_stride=63), dict(out_stride=1 << 50)]


@pytest.mark.parametrize("over", BAD_WEIGHTS)
def test_weights_that_are_refused(pkg, over):
    bad = pkg._ffi.ERR_INVALID_REQUEST
    assert linear(pkg, weight(pkg, **over)) == bad and pkg._ffi.last_error()
    assert gated(pkg, weight(pkg, **over)) == bad
    assert gated(pkg, None, weight(pkg, **over)) == bad
    assert linear(pkg, weight(pkg, **over), rows=0) == bad


@pytest.mark.parametrize("over", BAD_ROWS)
def test_rows_that_are_refused(pkg, over):
    assert linear(pkg, **over) == pkg._ffi.ERR_INVALID_REQUEST and pkg._ffi.last_error()
    assert gated(pkg, **over) == pkg._ffi.ERR_INVALID_REQUEST


def test_other_refusals(pkg):
    bad = pkg._ffi.ERR_INVALID_REQUEST
    assert pkg._ffi.lib().orion_cuda_w4_linear(0, 2, P, 4, 128, None, None, P, 64, None, 0, None) == bad
    assert linear(pkg, bias=P + 2) == bad
    assert gated(pkg, act=2) == bad and gated(pkg, act=-1) == bad
    for over in (dict(out_features=65), dict(in_features=160), dict(group=64)):
        assert gated(pkg, None, weight(pkg, **over)) == bad
    for over in (dict(dtype=1), dict(w=0), dict(w=P + 4), dict(n=0), dict(n=1 << 31), dict(k=0), dict(k=100), dict(stride=96), dict(stride=129), dict(group=8),
                 dict(packed=0), dict(packed=P + 4), dict(scales=0), dict(scales=P + 2), dict(zeros=P + 1), dict(n=1 << 30, k=1 << 20, stride=1 << 20)):
        assert quantize(pkg, **over) == bad, over


@pytest.mark.parametrize("is_gated", [0, 1])
def test_workspaces(pkg, is_gated):
    """What a call for many rows needs, and that it is refused with less; few rows and f32 need nothing."""
    lib, bad, w, need = pkg._ffi.lib(), pkg._ffi.ERR_INVALID_REQUEST, weight(pkg, in_features=512, out_features=4096), C.c_uint64(5)
    for dtype, rows in ((0, 1), (0, 5000), (2, 1), (2, 8), (2, 0)):
        assert lib.orion_cuda_w4_workspace(dtype, rows, C.addressof(w), is_gated, C.byref(need)) == pkg._ffi.ORION_OK and need.value == 0
    last = 0
    for rows in (600, 1000, 5000, 70000):
        assert lib.orion_cuda_w4_workspace(2, rows, C.addressof(w), is_gated, C.byref(need)) == pkg._ffi.ORION_OK
        assert need.value >= rows * 512 * 2 and need.value > last
        last, call = need.value, gated if is_gated else linear
        for space, size in ((0, 0), (0, last), (P, last - 1), (P + 128, last)):
            assert call(pkg, w, rows=rows, stride=512, out_stride=4096, space=space, size=size, **({"up": w} if is_gated else {})) == bad
    assert lib.orion_cuda_w4_workspace(1, 8, C.addressof(w), 0, C.byref(need)) == bad
    assert lib.orion_cuda_w4_workspace(2, 1 << 31, C.addressof(w), 0, C.byref(need)) == bad
    assert lib.orion_cuda_w4_workspace(2, 8, None, 0, C.byref(need)) == bad
    assert lib.orion_cuda_w4_workspace(2, 8, C.addressof(w), 0, None) == bad
    assert lib.orion_cuda_w4_workspace(2, 8, C.addressof(weight(pkg, group=5)), 0, C.byref(need)) == bad


def test_no_rows_need_no_device(pkg):
    assert linear(pkg, rows=0, x=0, out=0) == pkg._ffi.ORION_OK
    assert gated(pkg, rows=0, x=0, out=0) == pkg._ffi.ORION_OK


def test_tensors_that_are_not_on_a_device_are_refused(pkg):
    torch = pytest.importorskip("torch")
    packed, scales = torch.zeros((8, 16), dtype=torch.int32), torch.zeros((4, 8), dtype=torch.bfloat16)
    for args in ((packed, scales, None, 32), (packed, scales, None, 16), (np.zeros((8, 16)), scales, None, 32), (packed[0], scales, None, 32)):
        with pytest.raises(pkg.InvalidRequest):
            pkg.W4Weight(*args)
    with pytest.raises(pkg.InvalidRequest):
        pkg.W4Weight.from_codes(torch.zeros((8, 12)), scales, None, 32)


def test_plain_forms_agree_with_one_another():
    rng = np.random.default_rng(3)
    w = rng.standard_normal((6, 256)).astype(np.float32).astype(np.float64)
    for zeros in (False, True):
        codes, scales, z = plain.quantize(w, 64, zeros)
        np.testing.assert_array_equal(plain.unpack(plain.pack(codes)), codes)
        step = np.repeat(scales.T, 64, axis=1)
        # half a step, and where the two ends of a group both round outward half a step more, plus the rounding of the scale over 15 steps
        assert (np.abs(plain.dequantize(codes, scales, z, 64) - w) <= step * (1.0 + 15 * 2.0 ** -8)).all()
    assert plain.to_bf16(1.0 + 2.0 ** -8) == 1.0 and plain.to_bf16(1.0 + 3 * 2.0 ** -8) == 1.0 + 2.0 ** -6
