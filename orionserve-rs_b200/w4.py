"""4-bit weights: a quantiser, projections and gated feed-forwards over torch tensors on the GPU.

``W[n][k] = (code - zero) * scale`` with a bf16 scale, and in the asymmetric form a zero point, per group of 32, 64 or 128 consecutive ``k`` of a row.
Codes are packed eight to an int32: of eight consecutive ``k``, number ``2i`` is in bits ``4i .. 4i + 3``, number ``2i + 1`` in bits ``16 + 4i ..
19 + 4i``. The functions stand beside ``ops.linear`` and ``ops.swiglu`` for tensors that are on the device already: they run on torch's current
stream of the tensors' device, allocate what they return and, for many rows, a workspace, and can be captured into a CUDA graph once a call of
the same kind and size has been made outside of one. Activations are f32 or bf16. Nothing here has a gradient; tensors that require
one are refused, unless gradients are off (``torch.no_grad()``), as are tensors with a forward-mode tangent and calls under ``torch.jit.trace``, which
would not see the kernels.
"""
from __future__ import annotations

import ctypes as C

from . import _ffi
from .backend import CudaBackend
from .errors import InvalidRequest, check

GROUPS = (32, 64, 128)
_ACTIVATIONS = {"silu": _ffi.GATE_SILU, "gelu_tanh": _ffi.GATE_GELU_TANH}
_torch = _forward_ad = None
_dtypes = {}  # torch dtype -> OrionDType
_empty = _linear = _gated = _quantize = _is_tracing = None  # torch.empty_strided, the fastest of its kind, entry points of the library, torch.jit.is_tracing


def _load():
    """torch and the library, at the first call: the rest of the package does without torch."""
    global _torch, _forward_ad, _empty, _linear, _gated, _quantize, _stream, _is_tracing
    import torch
    import torch.autograd.forward_ad

    lib = _ffi.lib()
    _linear, _gated, _quantize = lib.orion_cuda_w4_linear, lib.orion_cuda_w4_gated, lib.orion_cuda_w4_quantize
    _dtypes.update({torch.float32: 0, torch.bfloat16: 2})
    _forward_ad, _empty = torch.autograd.forward_ad, torch.empty_strided
    _stream = _raw_stream(torch)
    _is_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)
    _torch = torch  # last: calls on other threads take it for a sign that the others are there


def _unrecorded(*tensors):
    """Refuses what torch records by other means than ``requires_grad``: forward-mode derivatives, which ``torch.no_grad()`` leaves on, and traces."""
    if _is_tracing():
        raise InvalidRequest("4-bit operators cannot be traced")
    for t in tensors:
        if isinstance(t, _torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise InvalidRequest("4-bit operators have no forward-mode derivative")


def _on_device(name, t, dtype, shape=None):
    if not isinstance(t, _torch.Tensor) or not t.is_cuda:
        raise InvalidRequest(f"{name}: a CUDA tensor is needed")
    if t.dtype != dtype:
        raise InvalidRequest(f"{name}: {dtype} is needed, got {t.dtype}")
    if shape is not None and tuple(t.shape) != shape:
        raise InvalidRequest(f"{name}: shape {shape} is needed, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise InvalidRequest(f"{name}: not contiguous")
    if t.requires_grad and _torch.is_grad_enabled():
        raise InvalidRequest(f"{name}: 4-bit operators have no gradient")


class W4Weight:
    """A matrix of 4-bit codes ``[out_features, in_features]``, kept by a program for as long as it uses the matrix.

    ``packed`` is int32 ``[out, in / 8]``, ``scales`` bf16 ``[in / group, out]``, ``zeros`` uint8 like ``scales`` with values of at most 15, or None:
    8 everywhere. The tensors are kept for good, as is everything else of the handle, since the kernels are given their addresses: they must not be resized
    or given other storage; their values may be written."""

    # One tuple, which the calls take apart and nothing else writes: packed, scales, zeros, group, out_features, in_features, device_index, the descriptor of
    # the library, its address, and the sizes of workspaces by key.
    __slots__ = ("_held",)

    packed, scales, zeros, group, out_features, in_features, device_index, _desc = (property(lambda self, i=i: self._held[i]) for i in range(8))

    def __init__(self, packed, scales, zeros=None, group: int = 128):
        if _torch is None:
            _load()
        if group not in GROUPS:
            raise InvalidRequest(f"groups of 4-bit weights hold 32, 64 or 128 values, got {group}")
        if not isinstance(packed, _torch.Tensor) or packed.dim() != 2:
            raise InvalidRequest("packed: a matrix is needed")
        n, k = packed.shape[0], packed.shape[1] * 8
        if n == 0 or k == 0 or k % group != 0:
            raise InvalidRequest(f"a matrix of {n} x {k} has no whole groups of {group}")
        _on_device("packed", packed, _torch.int32)
        _on_device("scales", scales, _torch.bfloat16, (k // group, n))
        if zeros is not None:
            _on_device("zeros", zeros, _torch.uint8, (k // group, n))
        if scales.device != packed.device or (zeros is not None and zeros.device != packed.device):
            raise InvalidRequest("packed, scales and zeros are on different devices")
        if packed.data_ptr() % 16:
            raise InvalidRequest("packed: must start on a 16-byte boundary")
        self._hold(packed, scales, zeros, group, n, k, packed.device.index)

    def _hold(self, packed, scales, zeros, group, n, k, device_index):
        desc = _ffi.OrionW4Weight(packed.data_ptr(), scales.data_ptr(), None if zeros is None else zeros.data_ptr(), n, k, group)
        self._held = packed, scales, zeros, group, n, k, device_index, desc, C.addressof(desc), {}

    def __copy__(self):
        return self

    @classmethod
    def from_codes(cls, codes, scales, zeros=None, group: int = 128) -> "W4Weight":
        """Packs codes ``[out, in]`` of 0..15, as other formats hold them, on their device; ``scales`` and ``zeros`` as in the constructor."""
        if _torch is None:
            _load()
        if not isinstance(codes, _torch.Tensor) or codes.dim() != 2 or codes.shape[1] % 8 or codes.dtype.is_floating_point or codes.dtype.is_complex:
            raise InvalidRequest("codes: a matrix of whole numbers is needed, with a multiple of 8 columns")
        if codes.numel() and (int(codes.min()) < 0 or int(codes.max()) > 15):
            raise InvalidRequest("codes: values of 0 to 15 are needed")
        at = _torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=_torch.int32, device=codes.device)
        words = (codes.to(_torch.int32).reshape(codes.shape[0], codes.shape[1] // 8, 8) << at).sum(-1, dtype=_torch.int32)
        return cls(words, scales, zeros, group)


def _rows(backend: CudaBackend, x, scales, in_features, device_index):
    """Checks a call's activations and its weight's place; returns (dtype, rows, row stride)."""
    if x.__class__ is not _torch.Tensor and not isinstance(x, _torch.Tensor):
        raise InvalidRequest("x: a CUDA tensor is needed")
    dtype = _dtypes.get(x.dtype)
    if dtype is None:
        raise InvalidRequest(f"x: float32 or bfloat16 is needed, got {x.dtype}")
    if x.dim() != 2 or x.shape[1] != in_features:
        raise InvalidRequest(f"x: shape [rows, {in_features}] is needed, got {tuple(x.shape)}")
    if x.get_device() != backend._ordinal or device_index != backend._ordinal:
        raise InvalidRequest(f"x and the weight must be on the backend's device {backend._ordinal}")
    if (x.requires_grad or scales.requires_grad) and _torch.is_grad_enabled():
        raise InvalidRequest("x and the weight's scales: 4-bit operators have no gradient")
    stride, unit = x.stride()
    if unit != 1:
        raise InvalidRequest("x: the values of a row must be neighbours")
    return dtype, x.shape[0], stride


def _overlap(a, b):
    """Whether two matrices of one type, their rows' values neighbours, share a byte; those of unequal row strides also where one lies between the other's rows."""
    size = a.element_size()
    at, bt = a.data_ptr(), b.data_ptr()
    if bt >= at + ((a.shape[0] - 1) * a.stride(0) + a.shape[1]) * size or at >= bt + ((b.shape[0] - 1) * b.stride(0) + b.shape[1]) * size:
        return False
    stride = a.stride(0) * size
    if stride != b.stride(0) * size or a.shape[0] == 1:
        return True
    apart = (bt - at) % stride
    return apart < a.shape[1] * size or apart + b.shape[1] * size > stride


def _meets(rows, row, apart, at, length):
    """Whether one of `rows` pieces of `row` bytes, `apart` bytes from one to the next, shares a byte with `length` bytes that begin `at` bytes behind the first's
    beginning."""
    first = max(0, (at - row) // apart + 1) if apart > 0 else 0  # the first that ends behind the beginning of the others
    return first < rows and first * apart < at + length and first * apart + row > at


def _output(x, out, rows, n, bias, *weights):
    if out is None:
        return _empty((rows, n), (n, 1), dtype=x.dtype, device=x.device), n
    if not isinstance(out, _torch.Tensor) or out.dtype != x.dtype or out.device != x.device or tuple(out.shape) != (rows, n) or (n > 1 and out.stride(1) != 1):
        raise InvalidRequest(f"out: a {x.dtype} tensor of shape [{rows}, {n}] on {x.device} is needed, its rows' values neighbours")
    if out.requires_grad and _torch.is_grad_enabled():
        raise InvalidRequest("out: 4-bit operators have no gradient")
    if rows:
        if _overlap(x, out):
            raise InvalidRequest("out: overlaps x")
        size, apart, begin = out.element_size(), out.stride(0), out.data_ptr()
        end = begin + ((rows - 1) * apart + n) * size
        others = [] if bias is None else [(bias.data_ptr(), 4 * n)]
        for _, _, _, group, w_n, k, _, desc, _, _ in weights:
            others += (desc.packed, w_n * k // 2), (desc.scales, w_n * (k // group) * 2)
            if desc.zeros is not None:
                others.append((desc.zeros, w_n * (k // group)))
        for at, length in others:
            if at < end and at + length > begin and _meets(rows, n * size, apart * size, at - begin, length):
                raise InvalidRequest("out: overlaps the bias or a weight")
    return out, out.stride(0)


def _written(out):
    """Tells torch that a tensor of the caller's was written: a backward pass that has kept it has to fail, as after torch's own writes."""
    _torch.autograd.graph.increment_version(out)


def _stream(device: int) -> int:
    return _torch.cuda.current_stream(device).cuda_stream


def _raw_stream(torch):
    """torch's own lookup of the current stream's handle, without a Stream object around it (1.2 us of a call), where this torch has it."""
    return getattr(torch._C, "_cuda_getCurrentRawStream", _stream)


def _workspace(x, dtype, rows, address, spaces, gated):
    """(tensor or None, address, bytes) of what a call needs beside its arguments, from torch's allocator: its own until later work of the stream. The sizes
    are kept with the weight."""
    key = rows << 3 | dtype << 1 | gated
    need = spaces.get(key)
    if need is None:
        size = C.c_uint64()
        check(_ffi.lib().orion_cuda_w4_workspace(dtype, rows, address, gated, C.byref(size)))
        if len(spaces) >= 256:
            spaces.clear()
        need = spaces[key] = size.value
    if need == 0:
        return None, None, 0
    t = _empty((need,), (1,), dtype=_torch.uint8, device=x.device)
    return t, t.data_ptr(), need


def linear_w4(backend: CudaBackend, x, weight: W4Weight, bias=None, out=None):
    """``x W^T + bias`` (tensor.rs:96-130) over ``x`` ``[rows, in]``, f32 or bf16; ``bias`` f32 ``[out]``. Sums are f32, rounded once to the type of
    ``x``. Rows may be apart (any stride that keeps them on 16-byte boundaries); ``out``, if given, overlaps none of
    the others, is written and returned.

    f32 values count as multiples of 2^-133, with all of their bits from 2^-109 on. With many rows of bf16 a weight has 11 bits: all of them with a zero point
    of 8, else off by up to 2^-12 of itself; scales below 2^-21 of their row's largest, and values below 2^-30 of their row's, lose bits. A bounded wait of
    those kernels that gives up leaves outputs of no use and sets bit 0 of ``CudaBackend.poll_wait_timeouts()``, which a program reads when it has waited for the
    stream: the call itself has returned by then."""
    if _torch is None:
        _load()
    held = weight._held
    _, scales, _, _, n, k, device_index, _, address, spaces = held
    dtype, rows, stride = _rows(backend, x, scales, k, device_index)
    if rows.__class__ is not int or _forward_ad._current_level >= 0:  # under a trace sizes are tensors
        _unrecorded(x, scales, bias, out)
    if bias is not None:
        _on_device("bias", bias, _torch.float32, (n,))
        if bias.get_device() != backend._ordinal:
            raise InvalidRequest(f"bias must be on the backend's device {backend._ordinal}")
    given = out
    out, out_stride = _output(x, out, rows, n, bias, held)
    space, at, size = _workspace(x, dtype, rows, address, spaces, 0)
    check(_linear(backend._ordinal, dtype, x.data_ptr(), rows, stride, address, None if bias is None else bias.data_ptr(), out.data_ptr(), out_stride, at, size,
                  _stream(backend._ordinal)))
    if given is not None:
        _written(given)
    return out


def gated_w4(backend: CudaBackend, x, gate: W4Weight, up: W4Weight, activation: str = "silu", out=None):
    """``f(x Wgate^T) * (x Wup^T)`` in one kernel, ``f`` = "silu" or "gelu_tanh" (tensor.rs:96-130, 175-189); the matrices have the same sizes and
    groups. Otherwise as ``linear_w4``."""
    if _torch is None:
        _load()
    kind = _ACTIVATIONS.get(activation)
    if kind is None:
        raise InvalidRequest(f"unknown activation {activation!r}")
    held, up_held = gate._held, up._held
    _, scales, _, _, n, k, device_index, _, address, spaces = held
    up_scales = up_held[1]
    dtype, rows, stride = _rows(backend, x, scales, k, device_index)
    if up_held[6] != backend._ordinal:
        raise InvalidRequest(f"x and the weight must be on the backend's device {backend._ordinal}")
    if up_scales.requires_grad and _torch.is_grad_enabled():
        raise InvalidRequest("the weight's scales: 4-bit operators have no gradient")
    if rows.__class__ is not int or _forward_ad._current_level >= 0:
        _unrecorded(x, scales, up_scales, out)
    given = out
    out, out_stride = _output(x, out, rows, n, None, held, up_held)
    space, at, size = _workspace(x, dtype, rows, address, spaces, 1)
    check(_gated(backend._ordinal, dtype, x.data_ptr(), rows, stride, address, up_held[8], kind, out.data_ptr(), out_stride, at, size,
                 _stream(backend._ordinal)))
    if given is not None:
        _written(given)
    return out


def quantize_w4(backend: CudaBackend, weight, group: int = 128, zeros: bool = False) -> W4Weight:
    """Codes, scales and (``zeros``) zero points of ``weight`` ``[out, in]``, f32 or bf16.

    Symmetric: scale = max|w| / 7, code = 8 + round(w / scale). With zero points: lo = min(w, 0), hi = max(w, 0), scale = (hi - lo) / 15, zero =
    round(-lo / scale), code = round(w / scale) + zero within 0..15. Scales are rounded to bf16 first, one below 2^-126 is 0; ties go to the even
    number. A group with an infinity or a NaN gets a scale of NaN."""
    if _torch is None:
        _load()
    if not isinstance(weight, _torch.Tensor) or weight.dim() != 2 or weight.dtype not in _dtypes:
        raise InvalidRequest("weight: a float32 or bfloat16 matrix is needed")
    if weight.get_device() != backend._ordinal:
        raise InvalidRequest(f"weight must be on the backend's device {backend._ordinal}")
    n, k = weight.shape
    if group not in GROUPS or n == 0 or k == 0 or k % group != 0:
        raise InvalidRequest(f"a matrix of {n} x {k} has no whole groups of {group} (32, 64 or 128)")
    if weight.requires_grad and _torch.is_grad_enabled():
        raise InvalidRequest("weight: 4-bit operators have no gradient")
    if n.__class__ is not int or _forward_ad._current_level >= 0:
        _unrecorded(weight)
    if weight.stride(1) != 1:
        raise InvalidRequest("weight: the values of a row must be neighbours")
    w = W4Weight.__new__(W4Weight)
    groups, device = k // group, weight.device
    w._hold(_empty((n, k // 8), (k // 8, 1), dtype=_torch.int32, device=device), _empty((groups, n), (n, 1), dtype=_torch.bfloat16, device=device),
            _empty((groups, n), (n, 1), dtype=_torch.uint8, device=device) if zeros else None, group, n, k, backend._ordinal)
    d = w._held[7]
    check(_quantize(backend._ordinal, _dtypes[weight.dtype], weight.data_ptr(), n, k, weight.stride(0), group, d.packed, d.scales, d.zeros,
                    _stream(backend._ordinal)))
    return w
