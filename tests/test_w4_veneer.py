"""What the torch veneer of the 4-bit operators refuses, on tensors of the host: the checks come ahead of any device."""
import copy
import types

import pytest

torch = pytest.importorskip("torch")

HOST = types.SimpleNamespace(_ordinal=-1)  # the "device" of a tensor that is on the host


@pytest.fixture
def w4(pkg):
    import sys

    module = sys.modules[pkg.linear_w4.__module__]
    module._load()
    return module


def weight(w4, n=8, k=64, group=32, zeros=False):
    w = w4.W4Weight.__new__(w4.W4Weight)
    w._hold(torch.zeros((n, k // 8), dtype=torch.int32), torch.zeros((k // group, n), dtype=torch.bfloat16),
            torch.zeros((k // group, n), dtype=torch.uint8) if zeros else None, group, n, k, -1)
    return w


@pytest.fixture
def no_device(w4, monkeypatch):
    """Calls that end where the library would be called."""
    for name in ("_linear", "_gated"):
        monkeypatch.setattr(w4, name, lambda *args: 0)
    monkeypatch.setattr(w4, "_stream", lambda device: 0)


def test_what_a_weight_holds_stays(w4):
    """The kernels are given the addresses that its tensors had when it was made."""
    w = weight(w4, zeros=True)
    for name in ("packed", "scales", "zeros", "group", "out_features", "in_features", "device_index", "other"):
        before = getattr(w, name, None)
        with pytest.raises(AttributeError):
            setattr(w, name, before)
        with pytest.raises(AttributeError):
            delattr(w, name)
        assert getattr(w, name, None) is before
    assert copy.copy(w) is w
    assert w._desc.packed == w.packed.data_ptr() and w._desc.zeros == w.zeros.data_ptr()


def test_scales_that_need_a_gradient_are_refused_at_the_call(pkg, w4, no_device):
    """A weight may be made under no_grad, or its scales may need a gradient later."""
    x = torch.zeros((3, 64), dtype=torch.bfloat16)
    w, learned = weight(w4), weight(w4)
    learned.scales.requires_grad_()
    for call in (lambda: pkg.linear_w4(HOST, x, learned), lambda: pkg.gated_w4(HOST, x, learned, w), lambda: pkg.gated_w4(HOST, x, w, learned)):
        with pytest.raises(pkg.InvalidRequest, match="gradient"):
            call()
    with torch.no_grad():
        assert pkg.linear_w4(HOST, x, learned).shape == (3, 8)


def test_forward_mode_tangents_are_refused(pkg, w4):
    """Under no_grad too, which leaves them on."""
    import torch.autograd.forward_ad as fw

    x, w, dual = torch.zeros((3, 64)), weight(w4), weight(w4)
    with fw.dual_level():
        for t in (x, w.scales):  # other tensors of a dual level are as good as ever
            w4._unrecorded(t, None)
        held = {name: getattr(dual, name) for name in ("packed", "scales", "zeros")}
        held["scales"] = fw.make_dual(held["scales"], torch.ones_like(held["scales"]))
        dual._hold(**held, group=32, n=8, k=64, device_index=-1)
        tangent, bias = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(torch.zeros(8), torch.ones(8))
        calls = (lambda: pkg.linear_w4(HOST, tangent, w), lambda: pkg.linear_w4(HOST, x, dual), lambda: pkg.linear_w4(HOST, x, w, bias=bias),
                 lambda: pkg.gated_w4(HOST, tangent, w, w), lambda: pkg.gated_w4(HOST, x, w, dual), lambda: pkg.gated_w4(HOST, x, dual, w),
                 lambda: pkg.quantize_w4(HOST, tangent, group=32))
        for call in calls:
            with pytest.raises(pkg.InvalidRequest, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(pkg.InvalidRequest, match="forward-mode"):
                call()


def test_traces_are_refused(pkg, w4):
    x, w = torch.zeros((3, 64)), weight(w4)
    for call in (lambda x: pkg.linear_w4(HOST, x, w), lambda x: pkg.gated_w4(HOST, x, w, w), lambda x: pkg.quantize_w4(HOST, x, group=32).scales):
        with pytest.raises(pkg.InvalidRequest, match="traced"):
            torch.jit.trace(call, (x,))


def test_two_first_calls_at_once(pkg, w4, monkeypatch):
    """What one thread's first call loads is there in full before another thread's takes it for loaded."""
    names = ("_forward_ad", "_empty", "_linear", "_gated", "_quantize", "_is_tracing", "_torch")
    for name in names:
        monkeypatch.setattr(w4, name, None)
    seen, real = [], w4._raw_stream

    def watched(*args):
        seen.append(w4._torch)
        return real(*args)

    monkeypatch.setattr(w4, "_raw_stream", watched)
    w4._load()
    assert seen == [None] and all(getattr(w4, name) is not None for name in names)


def test_outputs_that_a_backward_pass_has_kept(pkg, w4, no_device):
    """Written by a call, they no longer serve it."""
    x, w = torch.zeros((3, 64)), weight(w4)
    for call in (lambda out: pkg.linear_w4(HOST, x, w, out=out), lambda out: pkg.gated_w4(HOST, x, w, w, out=out)):
        whole = torch.ones((4, 12))
        learned = torch.ones((4, 12), requires_grad=True)
        loss = (learned * whole).sum()
        before = whole._version
        assert call(whole[1:, 2:10]).data_ptr() == whole[1:, 2:].data_ptr()
        assert whole._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        with torch.inference_mode():
            call(torch.zeros((3, 8)))


def test_outputs_that_overlap_a_bias_or_a_weight_are_refused(pkg, w4, no_device, monkeypatch):
    """CTAs that have ended write while others still read."""
    monkeypatch.setattr(w4, "_on_device", lambda *args: None)  # which asks for a CUDA tensor
    room = torch.zeros(4096, dtype=torch.uint8)
    room = room[-room.data_ptr() % 16:]

    def piece(start, shape, dtype):
        size = torch.empty((), dtype=dtype).element_size()
        n = 1
        for d in shape:
            n *= d
        return room[start:start + n * size].view(dtype).view(shape)

    def made(packed, scales, zeros):
        w = w4.W4Weight.__new__(w4.W4Weight)
        w._hold(packed, scales, zeros, 32, 8, 64, -1)
        return w

    x, bias = torch.zeros((3, 64)), torch.zeros(8)
    inside = made(piece(512, (8, 8), torch.int32), piece(1024, (2, 8), torch.bfloat16), piece(1280, (2, 8), torch.uint8))
    apart = weight(w4)
    for start, length in ((512, 256), (1024, 32), (1280, 16)):
        for at in (start - 64, start - 96 + 4, start, start + length - 4):  # three rows of 32 bytes
            for call in (lambda out: pkg.linear_w4(HOST, x, inside, out=out), lambda out: pkg.gated_w4(HOST, x, inside, apart, out=out),
                         lambda out: pkg.gated_w4(HOST, x, apart, inside, out=out)):
                with pytest.raises(pkg.InvalidRequest, match="overlaps"):
                    call(piece(at, (3, 8), torch.float32))
        for at in (start - 96, start + length):
            pkg.linear_w4(HOST, x, inside, out=piece(at, (3, 8), torch.float32))
    wide = piece(2048, (4, 24), torch.float32)
    for out in (wide[:3, :8], wide[1:4, 16:], wide[::2, 8:16][:2]):
        lone = x[:out.shape[0]]
        pkg.linear_w4(HOST, lone, apart, bias=wide[3, :8], out=out)  # between the rows, or behind them
        pkg.linear_w4(HOST, lone, apart, bias=wide[1, :8] if out.shape[0] == 2 else wide[0, 8:16], out=out)
        for row in range(out.shape[0]):
            with pytest.raises(pkg.InvalidRequest, match="overlaps"):
                pkg.linear_w4(HOST, lone, apart, bias=out[row], out=out)
    pkg.linear_w4(HOST, x[:1], apart, bias=bias, out=torch.zeros((1, 8)))


def test_codes_of_any_strides_are_packed(pkg, w4, monkeypatch):
    gen = torch.Generator().manual_seed(5)
    codes = torch.randint(0, 16, (64, 24), generator=gen)
    monkeypatch.setattr(w4, "_on_device", lambda *args: None)  # which asks for a CUDA tensor
    scales, shifts = torch.zeros((2, 24), dtype=torch.bfloat16), torch.tensor([0, 16, 4, 20, 8, 24, 12, 28])
    for dtype in (torch.uint8, torch.int8, torch.int32, torch.int64):
        for c in (codes.to(dtype).t(), codes.to(dtype).t().contiguous(), torch.cat([codes.to(dtype).t()] * 2, dim=1)[:, ::1][:, 64:], codes.to(dtype).t().repeat_interleave(2, 1)[:, ::2]):
            words = pkg.W4Weight.from_codes(c, scales, None, 32).packed
            assert torch.equal((words[:, :, None] >> shifts) & 15, codes.t().reshape(24, 8, 8).to(torch.int32))


def test_codes_that_are_refused(pkg, w4):
    scales = torch.zeros((2, 24), dtype=torch.bfloat16)
    for c in (torch.zeros((24, 64)), torch.zeros((24, 64), dtype=torch.complex64), torch.zeros((24, 60), dtype=torch.int32), torch.zeros((0, 64), dtype=torch.int32), torch.zeros((24, 0), dtype=torch.int32),
              torch.full((24, 64), 16), torch.full((24, 64), -1), torch.zeros(64, dtype=torch.int32)):
        with pytest.raises(pkg.InvalidRequest):
            pkg.W4Weight.from_codes(c, scales, None, 32)
